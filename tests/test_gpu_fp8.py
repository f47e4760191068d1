"""Block-scaled fp8 dense maps (``flash_uma_b200.fp8``) against the definition in fp64.

The oracle rounds each value to e4m3 under its block's power-of-two scale by counting (no float8
type), so codes and scales have to agree exactly; the products of codes are exact in fp32 and the
sums obey the bound of the grouped maps: |error| <= eps/2 |y| + (n / 32 + n / 128 + 8) 2^-23 S.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _scale(amax):
    s = torch.full_like(amax, 2.0 ** -126)
    for k in range(-125, 121):
        s = torch.where(amax > 448.0 * 2.0 ** (k - 1), torch.full_like(s, 2.0 ** k), s)
    return s


def _round(v):
    """fp64 -> the nearest e4m3 value, ties to even mantissas."""
    _, e = torch.frexp(v.abs().clamp(min=2.0 ** -6))
    step = torch.ldexp(torch.ones_like(v), e - 4)
    return torch.round(v / step) * step


def _rows64(x):
    out, scales = torch.empty(x.shape, dtype=torch.float64, device=x.device), []
    for a in range(0, x.shape[1], 128):
        b = x[:, a:a + 128].double()
        s = _scale(b.abs().amax(1, keepdim=True))
        out[:, a:a + 128] = _round(b / s) * s
        scales.append(s[:, 0])
    return out, torch.stack(scales)


def _weight64(w):
    out = torch.empty(w.shape, dtype=torch.float64, device=w.device)
    for n in range(0, w.shape[1], 128):
        for k in range(0, w.shape[2], 128):
            b = w[:, n:n + 128, k:k + 128].double()
            s = _scale(b.abs().amax((1, 2), keepdim=True))
            out[:, n:n + 128, k:k + 128] = _round(b / s) * s
    return out


def _values(T, K, dt, seed=0):
    """Rows of very unlike magnitudes, with blocks of zeros, exact borders and tiny values."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(T, K, device=DEV, generator=g) * torch.exp2(torch.randint(-12, 6, (T, 1), device=DEV, generator=g).float())
    x[::5, : K // 2] = 0.0
    x[1::7, 0] = 448.0
    x[2::7, -1] = -448.5
    x[3::7, K // 3] = 1.75 * 2.0 ** -7
    return x.to(dt)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T,K", [(1, 8), (1, 128), (17, 136), (130, 520), (33, 13), (7, 1), (300, 535), (1000, 1024)])
def test_quantize_rows(T, K, dt):
    from flash_uma_b200.fp8 import quantize_rows
    x = _values(T, K, dt)
    codes, scales = quantize_rows(x)
    want, ws = _rows64(x)
    got = codes.view(torch.float8_e4m3fn).double()[:, :K] * scales.double().repeat_interleave(128, 0).t()[:, :K]
    assert torch.equal(scales.double(), ws)
    assert torch.equal(got, want)
    assert not codes[:, K:].any()


def test_quantize_rows_not_finite_and_tiny():
    from flash_uma_b200.fp8 import quantize_rows
    x = torch.ones(6, 256, device=DEV)
    x[0, 3], x[1, 200], x[2, 0] = float("inf"), float("nan"), -float("inf")
    x[3, :128], x[3, 128:] = 0.0, 1e-44
    x[4, :128] = 3e38
    codes, scales = quantize_rows(x)
    bad = torch.isnan(scales)
    want = torch.zeros(2, 6, dtype=torch.bool, device=DEV)
    want[0, 0] = want[1, 1] = want[0, 2] = True
    assert torch.equal(bad, want)
    assert scales[0, 3] == 2.0 ** -126 and scales[1, 3] == 2.0 ** -126 and not codes[3].any()
    assert torch.equal(codes.view(torch.float8_e4m3fn).double()[4, :128] * scales[0, 4].double(),
                       _rows64(x[4:5])[0][0, :128])


@pytest.mark.parametrize("G,N,K", [(1, 8, 8), (2, 130, 264), (3, 7, 13), (1, 640, 768)])
def test_quantize_weight(G, N, K):
    from flash_uma_b200.fp8 import Fp8Weight
    w = _values(G * N, K, torch.float32, 2).view(G, N, K)
    q = Fp8Weight(w)
    want = _weight64(w)
    assert torch.equal(q.dequantize().double(), want)
    t = q.codes_t.view(torch.float8_e4m3fn).double()[:, :K, :N]
    s = q.scales_t.double().repeat_interleave(128, 1).repeat_interleave(128, 2)[:, :K, :N]
    assert torch.equal((t * s).transpose(1, 2), want)
    assert not q.codes[..., K:].any() and not q.codes_t[..., N:].any()


def _close(got, want, S, n, dt, what):
    tol = torch.finfo(dt).eps / 2 * want.abs() + (n / 32 + n / 128 + 8) * 2.0 ** -23 * S + \
        torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    bad = ~((got.double() - want).abs() <= tol)
    assert got.dtype == dt and got.shape == want.shape
    assert not bad.any(), (what, int(bad.sum()), float(((got.double() - want).abs() / tol).max()))


SHAPES = [([1], 8, 8, 0, 0), ([1], 512, 512, 0, 0), ([0, 5, 0, 130, 1, 127, 128, 0], 136, 264, 0, 0),
          ([300, 20], 768, 640, 7, 200), ([17, 0, 40], 13, 7, 2, 1), ([200], 1032, 136, 0, 0), ([9, 1], 1, 1, 1, 0),
          ([40, 0, 300], 535, 583, 1, 0), ([31], 260, 131, 0, 0),
          ([9001, 0, 257, 8000, 128, 129], 136, 640, 3, 77)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("bias", [None, "shared", "group"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"K{s[1]}N{s[2]}T{sum(s[0])}")
def test_linear_and_input_gradient(shape, bias, dt):
    from flash_uma_b200 import linear
    from flash_uma_b200.fp8 import Fp8Weight, fp8_linear
    lens, K, N, head, tail = shape
    G, T = len(lens), head + sum(lens) + tail
    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(T, K, device=DEV, generator=g).to(dt).requires_grad_(True)
    w = torch.randn(G, N, K, device=DEV, generator=g) * K ** -0.5
    w[:, N // 2:] *= 40.0
    b = None if bias is None else torch.randn(*((N,) if bias == "shared" else (G, N)), device=DEV, generator=g)
    gy = (torch.randn(T, N, device=DEV, generator=g) * 0.01).to(dt)
    off = torch.tensor([head] + lens, device=DEV).cumsum(0)
    y = fp8_linear(x, Fp8Weight(w), off, b)
    (dx,) = torch.autograd.grad(y, [x], gy)
    torch.cuda.synchronize()
    linear.check_errors()
    X, GY, W = _rows64(x.detach())[0], _rows64(gy)[0], _weight64(w)
    Y, Sy = torch.zeros(T, N, device=DEV).double(), torch.zeros(T, N, device=DEV).double()
    D, Sd = torch.zeros(T, K, device=DEV).double(), torch.zeros(T, K, device=DEV).double()
    o = off.tolist()
    for i in range(G):
        s = slice(o[i], o[i + 1])
        Y[s], Sy[s] = X[s] @ W[i].T, X[s].abs() @ W[i].abs().T
        if b is not None:
            Y[s] += (b if b.dim() == 1 else b[i]).double()
            Sy[s] += (b if b.dim() == 1 else b[i]).double().abs()
        D[s], Sd[s] = GY[s] @ W[i], GY[s].abs() @ W[i].abs()
    _close(y.detach(), Y, Sy, K, dt, "y")
    _close(dx, D, Sd, N, dt, "dx")


def test_one_matrix_without_offsets_and_one_row():
    from flash_uma_b200.fp8 import Fp8Weight, fp8_linear
    g = torch.Generator(device=DEV).manual_seed(5)
    w = torch.randn(72, 136, device=DEV, generator=g)
    q = Fp8Weight(w)
    x = torch.randn(70, 136, device=DEV, generator=g)
    off = torch.tensor([0, 70], device=DEV)
    y = fp8_linear(x, q)
    assert torch.equal(y, fp8_linear(x, q, off))
    assert torch.equal(y[5:6], fp8_linear(x[5:6], q))
    assert torch.equal(y, fp8_linear(x.t().contiguous().t(), q))
    assert fp8_linear(x[:0], q).shape == (0, 72)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fp8_linear(x, q)
    x.mul_(-0.3)
    graph.replay()
    assert torch.equal(out, fp8_linear(x, q))


def test_not_finite_rows_stay_alone():
    from flash_uma_b200.fp8 import Fp8Weight, fp8_linear
    g = torch.Generator(device=DEV).manual_seed(6)
    q = Fp8Weight(torch.randn(2, 72, 264, device=DEV, generator=g))
    x = torch.randn(90, 264, device=DEV, generator=g)
    off = torch.tensor([0, 40, 90], device=DEV)
    want = fp8_linear(x, q, off)
    x2 = x.clone()
    x2[7, 3], x2[50, 263] = float("inf"), float("nan")
    got = fp8_linear(x2, q, off)
    keep = [i for i in range(90) if i not in (7, 50)]
    assert torch.equal(got[keep], want[keep])
    assert torch.isnan(got[[7, 50]]).all()


def test_refusals():
    from flash_uma_b200.fp8 import Fp8Weight, fp8_linear, quantize_rows
    w = torch.randn(2, 72, 136, device=DEV)
    q = Fp8Weight(w)
    x = torch.randn(9, 136, device=DEV)
    off = torch.tensor([0, 4, 9], device=DEV)
    with pytest.raises(ValueError):
        fp8_linear(x, q)                                   # two matrices, no offsets
    with pytest.raises(TypeError):
        fp8_linear(x, w, off)
    with pytest.raises(TypeError):
        fp8_linear(x.double(), q, off)
    with pytest.raises(TypeError):
        fp8_linear(x, q, off, torch.zeros(72, device=DEV).bfloat16())
    with pytest.raises(ValueError):
        fp8_linear(x, q, off, torch.zeros(72, device=DEV, requires_grad=True))
    with pytest.raises(ValueError):
        fp8_linear(x[:, :8], q, off)
    with pytest.raises(RuntimeError, match="CUDA"):
        fp8_linear(x.cpu(), q, off)
    with pytest.raises(RuntimeError, match="CUDA"):
        Fp8Weight(w.cpu())
    with pytest.raises(ValueError):
        Fp8Weight(w[0, 0])
    with pytest.raises(TypeError):
        quantize_rows(x.double())


@pytest.mark.parametrize("dt", DTYPES)
def test_strides_alignment_streams_and_replay(dt):
    """Rows that are strided, transposed or off 16 bytes, another stream and a captured call on new data give the bits of the
    contiguous eager call."""
    from flash_uma_b200.fp8 import Fp8Weight, fp8_linear
    g = torch.Generator(device=DEV).manual_seed(5)
    T, G, N, K = 140, 3, 72, 200
    w8 = Fp8Weight(torch.randn(G, N, K, device=DEV, generator=g))
    off = torch.tensor([1, 60, 60, 139], device=DEV)
    b = torch.randn(G, N, device=DEV, generator=g)
    x = torch.randn(T, K, device=DEV, generator=g).to(dt)
    gy = torch.randn(T, N, device=DEV, generator=g).to(dt)

    def run(x, gy):
        x = x.detach().requires_grad_(True)
        y = fp8_linear(x, w8, off, b)
        return y.detach(), torch.autograd.grad(y, x, gy)[0]
    want = run(x, gy)
    wide = torch.zeros(T, K + 3, device=DEV, dtype=dt)[:, 1:K + 1].copy_(x)
    gt = gy.t().contiguous().t()
    for xi, gi in ((wide, gt), (x.t().contiguous().t(), gy.flip(0).flip(0)[:, :N])):
        assert all(torch.equal(p, q) for p, q in zip(run(xi, gi), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(x, gy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x, gy)
    x.mul_(3.0)
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(out, run(x, gy)))


def test_rows_past_32_bit_offsets():
    from flash_uma_b200.fp8 import Fp8Weight, fp8_linear
    T, K, N, n = 2 ** 21 + 5, 1032, 8, 300
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.zeros(T, K, device=DEV, dtype=torch.bfloat16)
    x[-n:] = torch.randn(n, K, device=DEV, generator=g).bfloat16()
    w8 = Fp8Weight(torch.randn(N, K, device=DEV, generator=g))
    y = fp8_linear(x, w8)
    assert torch.equal(y[-n:], fp8_linear(x[-n:].contiguous(), w8)) and not y[:-n].any()


@pytest.mark.parametrize("dt", DTYPES)
def test_scales_whose_product_leaves_the_fp32_range(dt):
    """Blocks of the largest magnitudes whose products are all zero add nothing; blocks of the smallest add what they hold."""
    from flash_uma_b200.fp8 import Fp8Weight, fp8_linear
    g = torch.Generator(device=DEV).manual_seed(8)
    T, K, N = 40, 384, 72
    x = torch.randn(T, K, device=DEV, generator=g).to(dt)
    w = torch.randn(N, K, device=DEV, generator=g)
    x[:, :128], w[:, :128] = 0.0, 0.0
    want = fp8_linear(x, Fp8Weight(w))
    x[::2, 0], w[:, 1] = torch.finfo(dt).max, 3e38    # scales 2^120 (fp16 2^8) and 2^120; every product is 0
    assert torch.equal(fp8_linear(x, Fp8Weight(w)), want)
    x[3, 200] = float("nan")
    got = fp8_linear(x, Fp8Weight(w))
    keep = torch.arange(T, device=DEV) != 3
    assert torch.isnan(got[3]).all() and torch.equal(got[keep], want[keep])
    if dt != torch.float16:                           # 2^-126 and 2^-24: 128 products of 2^-134
        y = fp8_linear(torch.full((T, 128), 2.0 ** -118, device=DEV, dtype=dt), Fp8Weight(torch.full((N, 128), 2.0 ** -16, device=DEV)))
        assert (y.double() == 2.0 ** -127).all()
