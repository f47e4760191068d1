"""Dense maps on block-scaled 8-bit operands (e4m3, one scale for each block of 128).

The step below the ``"f16"`` mode of :mod:`flash_uma_b200.linear`: frozen weights at one byte per
value, products on the fp8 tensor cores, fp32 sums; about 4 significant bits per operand, for
screening and other uses that bear errors of a few percent per product. :class:`Fp8Weight` holds
a frozen matrix (or one per system) in 128 x 128 blocks, laid out once; :func:`fp8_linear` rounds the
activations in blocks of 128 along each row and multiplies. A scale is the smallest power of two
(at least 2^-126) that brings its block's largest magnitude to 448 or below, so a value is rounded
once, to nearest even.
"""
from __future__ import annotations

import torch

from . import _native as nat
from ._native import ptr, stream_of
from .grouped import (_DTYPES, MAX_GROUPS, _apply, _check_dtype, _once, _opaque, _same_device, _unit_stride, check_groups,
                      guard_capture, refuse_fx_trace)
from .linear import error_flag

_BLOCK = 128


def _ceil16(n: int) -> int:
    return (n + 15) // 16 * 16


def _blocks(n: int) -> int:
    return (n + _BLOCK - 1) // _BLOCK


def _refuse_trace() -> None:
    refuse_fx_trace()
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError("quantisation to fp8 cannot be traced: a traced graph would hold the empty codes alone")


class Fp8Weight:
    """Frozen weights [N, K] or [G, N, K] (float32, bfloat16 or float16, on a GPU) as e4m3 codes and scales, and
    the same of the transposed matrices for the input gradient: two bytes per weight in all."""

    def __init__(self, weight: torch.Tensor):
        _refuse_trace()
        nat.require_cuda(weight)
        if weight.dim() not in (2, 3):
            raise ValueError(f"weight must be [N, K] or [groups, N, K] (got {tuple(weight.shape)})")
        _check_dtype("weight", weight)
        w = weight.detach()
        w = w[None] if w.dim() == 2 else w
        self.G, self.N, self.K = w.shape
        if not 1 <= self.G <= MAX_GROUPS:
            raise ValueError(f"the number of groups must be from 1 to {MAX_GROUPS} (got {self.G})")
        if self.N < 1 or self.K < 1:
            raise ValueError(f"weight needs N >= 1 and K >= 1 (got {tuple(weight.shape)})")
        w = w.float().contiguous()
        dev, G, N, K = w.device, self.G, self.N, self.K
        self.device = dev
        self.codes = w.new_empty((G, N, _ceil16(K)), dtype=torch.uint8)
        self.scales = w.new_empty((G, _blocks(N), _blocks(K)))
        self.codes_t = w.new_empty((G, K, _ceil16(N)), dtype=torch.uint8)
        self.scales_t = w.new_empty((G, _blocks(K), _blocks(N)))
        nat.call("fuma_quantize_weight_fp8", ptr(w), G, N, K, ptr(self.codes), _ceil16(K), ptr(self.scales),
                 ptr(self.codes_t), _ceil16(N), ptr(self.scales_t), stream_of(w))

    def dequantize(self) -> torch.Tensor:
        """The values that the codes stand for, fp32 [G, N, K]."""
        v = self.codes.view(torch.float8_e4m3fn).float()[:, : self.N, : self.K]
        s = self.scales.repeat_interleave(_BLOCK, 1).repeat_interleave(_BLOCK, 2)
        return v * s[:, : self.N, : self.K]


def quantize_rows(x: torch.Tensor):
    """x [T, K] -> (codes uint8 [T, K rounded up to 16], scales float32 [ceil(K / 128), T]): e4m3 in
    blocks of 128 along each row (``fuma_quantize_rows_fp8``)."""
    _refuse_trace()
    nat.require_cuda(x)
    code = _check_dtype("x", x)
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"x must be [rows, K] with K >= 1 (got {tuple(x.shape)})")
    T, K = x.shape
    x = _unit_stride(x)
    codes = x.new_empty((T, _ceil16(K)), dtype=torch.uint8)
    scales = x.new_empty((_blocks(K), T), dtype=torch.float32)
    if T:
        nat.call("fuma_quantize_rows_fp8", ptr(x), x.stride(0), T, K, code, ptr(codes), _ceil16(K), ptr(scales),
                 stream_of(x))
    return codes, scales


def _product(x, w_codes, w_scales, offsets, bias, N, K):
    T, G = x.shape[0], w_codes.shape[0]
    y = x.new_empty((T, N))
    if T:
        x = _unit_stride(x)
        nbytes = nat.load().fuma_fp8_work_bytes(T, K)   # the quantised rows and their scales
        work = x.new_empty(nbytes, dtype=torch.uint8)
        nat.call("fuma_grouped_linear_fp8", ptr(x), x.stride(0), ptr(w_codes), ptr(w_scales), ptr(offsets), G, ptr(bias),
                 0 if bias is None else (1 if bias.dim() == 1 else G), T, N, K, _DTYPES[x.dtype], ptr(y), ptr(work),
                 nbytes, ptr(error_flag(x.device)), stream_of(x))
    return y


class _Fp8LinearFn(torch.autograd.Function):
    @staticmethod
    def compute(x, weight, offsets, bias):
        if bias is not None:
            bias = bias.contiguous()
        return _product(x, weight.codes, weight.scales, offsets, bias, weight.N, weight.K)

    @staticmethod
    def forward(ctx, x, weight, offsets, bias):
        ctx.weight = weight
        ctx.save_for_backward(*(() if offsets is None else (offsets,)))
        return _Fp8LinearFn.compute(x, weight, offsets, bias)

    @staticmethod
    @_once
    def backward(ctx, g):
        weight = ctx.weight
        offsets = ctx.saved_tensors[0] if ctx.saved_tensors else None
        return _product(g, weight.codes_t, weight.scales_t, offsets, None, weight.K, weight.N), None, None, None


def fp8_linear(x: torch.Tensor, weight: Fp8Weight, offsets: torch.Tensor | None = None,
               bias: torch.Tensor | None = None) -> torch.Tensor:
    """``y = x_q W_q^T (+ bias)`` with x rounded to e4m3 in row blocks of 128; y has x's type
    (float32, bfloat16 or float16), sums are fp32.

    ``offsets`` [G + 1] int64 gives the rows of each of the weight's G matrices, as in
    :func:`flash_uma_b200.grouped.grouped_linear`; None: all rows through the one matrix. ``bias``
    float32 [N] or [G, N]. Weights and bias are frozen (a bias that requires a gradient is refused);
    the gradient of x is ``g_q W_q`` with the output's gradient rounded the same way (for forces). A block
    with a value that is not finite makes the results that depend on it NaN."""
    if torch.compiler.is_compiling():
        return _opaque(fp8_linear, x, weight, offsets, bias)
    nat.require_cuda(x, offsets, bias)
    if not isinstance(weight, Fp8Weight):
        raise TypeError(f"weight must be an Fp8Weight (got {type(weight).__name__})")
    _check_dtype("x", x)
    if bias is not None and bias.dtype != torch.float32:
        raise TypeError(f"bias must be float32 (got {bias.dtype})")
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        raise ValueError("fp8_linear has frozen weights: the bias must not require a gradient")
    if offsets is None and weight.G != 1:
        raise ValueError(f"offsets are needed for the weight's {weight.G} matrices")
    check_groups(x, weight.G, weight.N, weight.K, offsets, bias)
    _same_device(x.device, weight=weight, offsets=offsets, bias=bias)
    return _apply(_Fp8LinearFn, guard_capture(x), x, weight, None if offsets is None else offsets.contiguous(), bias)
