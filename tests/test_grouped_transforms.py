"""The expert-mixture calls under torch's transformations, on the CPU with the C entry points replaced by a record of their
names: what would leave the kernels or the derivative out without a word goes through the autograd function or is refused."""
import pytest
import torch
from torch.autograd import forward_ad


@pytest.fixture
def calls(monkeypatch):
    from flash_uma_b200 import _native as nat
    from flash_uma_b200 import fp8, grouped
    seen = []
    monkeypatch.setattr(nat, "call", lambda name, *a: seen.append(name))
    monkeypatch.setattr(nat, "require_cuda", lambda *t: None)
    for mod in (grouped, fp8):
        monkeypatch.setattr(mod, "guard_capture", lambda *t: False)
        monkeypatch.setattr(mod, "error_flag", lambda dev: torch.zeros(1, dtype=torch.int32))
        monkeypatch.setattr(mod, "stream_of", lambda t: 0)
    return seen


def _cases():
    from flash_uma_b200.fp8 import Fp8Weight, fp8_linear
    from flash_uma_b200.grouped import grouped_linear, mix_experts
    off = torch.tensor([0, 3, 5])
    w8 = Fp8Weight(torch.randn(2, 8, 16))
    return {"grouped": (lambda x: grouped_linear(x, torch.ones(2, 8, 16), off), torch.randn(5, 16), "fuma_grouped_linear"),
            "mix": (lambda c: mix_experts(c, torch.ones(4, 8)), torch.randn(3, 4), "fuma_mix_experts"),
            "fp8": (lambda x: fp8_linear(x, w8, off), torch.randn(5, 16), "fuma_grouped_linear_fp8")}


NAMES = ["grouped", "mix", "fp8"]


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(calls, name):
    """A dual input without requires_grad must not come back without its tangent."""
    f, x, _ = _cases()[name]
    with forward_ad.dual_level():
        with pytest.raises((NotImplementedError, RuntimeError)):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
        f(x)                                               # no tangent: nothing to lose
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))


@pytest.mark.parametrize("name", NAMES)
def test_jit_trace_records_the_call(calls, name):
    f, x, entry = _cases()[name]
    traced = torch.jit.trace(f, (x,), check_trace=False)
    calls.clear()
    out = traced(x)
    assert entry in calls and out.shape == f(x).shape


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [False, True])
def test_fx_trace_is_refused(calls, name, grad):
    """A traced graph would hold the empty outputs alone."""
    from torch.fx.experimental.proxy_tensor import make_fx
    f, x, _ = _cases()[name]
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(f)(x.requires_grad_(grad))


def test_quantisation_in_a_trace_is_refused(calls):
    from flash_uma_b200.fp8 import Fp8Weight, quantize_rows
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.randn(5, 16)
    for f in (quantize_rows, lambda x: Fp8Weight(x).codes):
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(f)(x)
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(f, (x,), check_trace=False)


@pytest.mark.parametrize("name", NAMES)
def test_other_transforms_raise(calls, name):
    f, x, _ = _cases()[name]
    for transform, arg in ((torch.func.vmap(f), x[None]), (torch.func.grad(lambda x: f(x).sum()), x), (torch.func.functionalize(f), x)):
        with pytest.raises((NotImplementedError, RuntimeError, ValueError)):
            transform(arg)
