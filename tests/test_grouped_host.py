"""Refusals of the expert-mixture entry points, on the host and without a GPU: the C ABI checks its
arguments before any launch, the Python calls refuse CPU tensors."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from flash_uma_b200 import _native, build
    build.build()
    return _native.load()


P = 4096   # a 16-byte aligned non-null address that no check reads


@pytest.mark.parametrize("change,message", [
    (dict(G=0), b"G=0"), (dict(G=4097), b"G=4097"), (dict(T=-1), b"T=-1"), (dict(T=2 ** 31), b"out of range"),
    (dict(N=0), b"positive"), (dict(K=0), b"positive"), (dict(ldw=8), b"ldw=8"), (dict(ldw=20), b"ldw=20"), (dict(dtype=3), b"dtype=3"),
    (dict(ldx=8), b"ldx=8"), (dict(ldx=20), b"ldx=20"), (dict(bias=P, bias_rows=2), b"bias_rows=2"),
    (dict(x=None), b"null pointer"), (dict(dtype=0, xs=None), b"null pointer"), (dict(dtype=0, ldx=24), b"planes"), (dict(offsets=None), b"one group only"),
    (dict(T=2 ** 31 - 512, N=2 ** 20, G=1), b"too many output tiles"), (dict(G=4096, N=2 ** 20), b"too large"),
])
def test_grouped_linear_refusals(lib, change, message):
    a = dict(x=P, ldx=16, xs=P, W=P, ldw=16, ws=P, offsets=P, G=3, bias=None, bias_rows=0, T=10, N=24, K=16, dtype=1, y=P)
    a.update(change)
    assert lib.fuma_grouped_linear(*a.values(), None, None) == -1
    assert message in lib.fuma_last_error()


def test_alignment_refused(lib):
    assert lib.fuma_grouped_linear(P + 8, 16, None, P, 16, None, P, 3, None, 0, 10, 24, 16, 1, P, None, None) == -2
    assert lib.fuma_grouped_linear_dgrad(P, 24, None, P + 2, 16, None, P, 3, 10, 24, 16, 1, P, None, None) == -2
    assert lib.fuma_quantize_rows_fp8(P, 16, 4, 16, 1, P + 4, 16, P, None) == -2
    assert lib.fuma_mix_experts(P, 4, 1, P + 4, 2, 4, 64, 0, P, None, None) == -2


def test_other_refusals(lib):
    f = lib
    assert f.fuma_grouped_linear_dgrad(P, 16, None, P, 16, None, P, 3, 10, 24, 16, 1, P, None, None) == -1   # lddy < N
    assert f.fuma_split_blocks(P, 8, 4, 12, P, 1, 0, 0, P, P, None) == -1                            # ldx
    assert f.fuma_pad_rows(P, 12, 4, 12, P, 12, None, 0, 0, 0, None) == -1                        # ldo
    assert f.fuma_pad_rows(P, 12, 5, 12, P, 16, P, 2, 2, 9, None) == -1                           # rows != G * mat_rows
    assert f.fuma_split_blocks(P, 16, 10, 16, None, 0, 4, 0, P, P, None) == -1                       # mat_rows
    assert f.fuma_split_blocks(P, 16, 10, 16, None, 2, 0, 0, P, P, None) == -1                       # no offsets
    assert f.fuma_quantize_rows_fp8(P, 16, 4, 16, 1, P, 24, P, None) == -1                        # ldq
    assert f.fuma_quantize_weight_fp8(P, 1, 24, 16, P, 16, P, P, 24, P, None) == -1               # ldt
    assert f.fuma_grouped_linear_fp8(P, 16, P, P, None, 2, None, 0, 10, 24, 16, 1, P, P, 1 << 20, None, None) == -1
    assert f.fuma_grouped_linear_fp8(P, 16, P, P, P, 2, None, 0, 10, 24, 16, 1, P, P, 100, None, None) == -1   # work space
    assert f.fuma_mix_experts(P, 4, 1, P, 2, 0, 64, 0, P, None, None) == -1
    assert f.fuma_mix_experts_bwd(P, P, 4, 1, P, 2, 4, 64, 5, P, P, P, 1 << 20, None, None) == -1
    assert f.fuma_mix_experts_bwd(P, P, 4, 1, P, 2, 4, 64, 0, P, P, P, 4, None, None) == -1                # work space
    assert f.fuma_mix_experts_bwd(P, P, 4, 1, P, 2, 4, 64, 0, None, None, P, 1 << 20, None, None) == -1
    # nothing to do: no launch, no device needed
    assert f.fuma_grouped_linear(None, 16, None, None, 16, None, None, 3, None, 0, 0, 24, 16, 1, None, None, None) == 0
    assert f.fuma_mix_experts(None, 4, 1, None, 0, 4, 64, 0, None, None, None) == 0


def test_work_sizes(lib):
    """The weight gradient's work space holds the parts of cut groups; none for short batches."""
    n = lib.fuma_grouped_wgrad_work_bytes
    assert n(0, 64, 64, 1) == 0 and n(2048, 64, 64, 1) == 0
    assert n(2049, 64, 64, 1) >= 2 * 64 * 64 * 4
    assert lib.fuma_grouped_bias_grad_work_bytes(1000, 64, 5) >= (2 + 5) * 64 * 4
    assert lib.fuma_mix_experts_work_bytes(3, 4, 1000, 0) >= 3 * 4 * 4


def test_part_slots_never_meet():
    """The slot rule of the weight gradient's partial matrices, restated: over random group lengths no two parts share a
    slot, all stay inside the work space, and the parts cover each group's blocks of 128 rows once."""
    g = torch.Generator().manual_seed(0)
    for trial in range(400):
        cap = int(torch.randint(2, 30, (1,), generator=g))
        lens = (torch.rand(12, generator=g) ** 3 * 128 * cap * 5).long().tolist()
        T, a, used = sum(lens), 0, set()
        for n in lens:
            blocks = -(-n // 128)
            if blocks > cap:
                parts = -(-blocks // cap)
                each = -(-blocks // parts)
                assert each <= cap
                for c in range(parts):
                    s = 2 * (a // 128) // cap + c
                    assert s not in used and 0 <= s < 2 * (T // 128) // cap + 2
                    used.add(s)
            a += n


def test_row_block_slots_never_meet():
    """The slot rule of the fp32 split's block scales (group start / 128 + group + tile), restated: distinct, in range,
    and found again by the kernel's search."""
    g = torch.Generator().manual_seed(1)
    for _ in range(300):
        lens = (torch.rand(15, generator=g) ** 2 * 500).long().tolist()
        starts = [sum(lens[:i]) for i in range(len(lens))]
        slots, used = sum(lens) // 128 + len(lens), set()
        for k, (a, n) in enumerate(zip(starts, lens)):
            for i in range(-(-n // 128)):
                s = a // 128 + k + i
                assert s not in used and s < slots
                used.add(s)
                found = max(j for j in range(len(lens)) if starts[j] // 128 + j <= s)
                assert found == k and s - (starts[found] // 128 + found) == i


def test_cpu_tensors_refused():
    from flash_uma_b200.fp8 import Fp8Weight, quantize_rows
    from flash_uma_b200.grouped import grouped_linear, mix_experts
    x = torch.zeros(4, 8)
    for call in (lambda: grouped_linear(x, torch.zeros(1, 8, 8), torch.tensor([0, 4])),
                 lambda: mix_experts(torch.zeros(2, 3), torch.zeros(3, 8)),
                 lambda: quantize_rows(x), lambda: Fp8Weight(x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_widths_that_32_bit_sums_do_not_hold_are_refused(lib):
    wide = 2 ** 30 + 8
    f = lib
    assert f.fuma_grouped_linear(P, 16, None, P, 16, None, P, 1, None, 0, 10, wide, 16, 1, P, None, None) == -1
    assert b"at most" in f.fuma_last_error()
    assert f.fuma_grouped_linear_dgrad(P, wide, None, P, 16, None, P, 1, 10, wide, 16, 1, P, None, None) == -1
    assert f.fuma_grouped_linear(P, wide, None, P, wide, None, P, 1, None, 0, 10, 24, wide, 1, P, None, None) == -1
    assert f.fuma_quantize_rows_fp8(P, wide, 4, wide, 1, P, wide, P, None) == -1
    assert f.fuma_grouped_bias_grad(P, 2 ** 24, P, 1, 1, 10, 2 ** 24, 1, P, P, 1 << 40, None) == -1
    assert b"too large" in f.fuma_last_error()


def test_launches_of_the_calls_that_vary(lib):
    from flash_uma_b200 import _native as nat

    def wgrad(T):
        return nat.launches_of("fuma_grouped_linear_wgrad", (P, 64, P, P, 64, P, P, 1, T, 64, 64, 0, P, P, 0, None, None))

    def mix(S, E, dtype, dc, dx):
        return nat.launches_of("fuma_mix_experts_bwd", (P, P, E, 1, P, S, E, 1000, dtype, dc, dx, P, 0, None, None))
    assert [wgrad(0), wgrad(2048), wgrad(2049)] == [0, 1, 2]
    assert [nat.launches_of("fuma_grouped_bias_grad", (P, 8, P, 1, 0, T, 8, 0, P, P, 0, None)) for T in (0, 5)] == [1, 2]
    assert [mix(128, 128, d, P, P) for d in (0, 1, 2)] == [2, 2, 2]
    assert [mix(129, 2, 1, P, P), mix(2, 129, 1, P, P)] == [3, 3]
    assert [mix(4, 4, 1, P, None), mix(4, 4, 1, None, P)] == [2, 1]
