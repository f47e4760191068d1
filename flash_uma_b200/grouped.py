"""Dense layers of a mixture of linear experts: per-system weights and the grouped dense map.

FAIRChem's UMA models keep E expert matrices per dense layer and give a system the mean of them
under its own coefficients. The reference (and :class:`~flash_uma_b200.wrapper.ZeroAllocBackbone`)
takes a model whose experts were merged for one composition (``readme.md:35-72``). For a batch of
unlike systems, and for training, every system keeps its own matrix:

* :func:`mix_experts`: ``W[s] = sum_e coeff[s, e] experts[e]``, with both gradients;
* :func:`grouped_linear`: ``y[t] = W[g(t)] x[t] + b`` for rows grouped by system, with the
  gradients of ``x``, ``W`` and ``b``;
* :class:`MoleLinear`: the two together, a layer.

Counterpart of :class:`~flash_uma_b200.linear.FrozenLinear` (one frozen matrix for all rows) on
the same tensor cores. Types: fp32 (two fp16 planes per operand under a scale for each block, three products:
22 bits, or 2^-39 of the block's largest magnitude where that is more; the whole fp32 range, no range error), bf16 and fp16 (fp32 sums, one rounding at the end).
:func:`flash_uma_b200.fp8.fp8_linear` is the map on frozen 8-bit weights.
"""
from __future__ import annotations

import threading
import weakref

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _native as nat
from ._native import ptr, stream_of
from .linear import _err_flags, error_flag

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_GROUPS = 4096


def _check_dtype(name: str, t: torch.Tensor) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32, bfloat16 or float16 (got {t.dtype})")
    return code


def _same_device(dev: torch.device, **others) -> None:
    for name, t in others.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the call's other tensors on {dev}")


# autograd nodes of eager calls, while their graph is alive
_live_nodes: "weakref.WeakSet" = weakref.WeakSet()
_live_lock = threading.Lock()


def _leaves_below(nodes) -> list:
    """The leaf tensors that the autograd graphs of ``nodes`` end in."""
    found, seen, stack = [], set(), list(nodes)
    while stack:
        node = stack.pop()
        if node is None or node in seen:
            continue
        seen.add(node)
        leaf = getattr(node, "variable", None)
        if leaf is not None:
            found.append(leaf)
        stack.extend(n for n, _ in node.next_functions)
    return found


def guard_capture(*inputs) -> bool:
    """True if the current stream is capturing. Refuses to put a call on leaf tensors into a CUDA graph capture
    while an eager graph of the same leaves is alive: autograd keeps one gradient node per leaf, bound to the
    stream it was made on, and a captured backward pass that meets a node of an uncaptured stream
    invalidates the capture or ends the process. Seen are the eager calls of this module and of fp8."""
    if not torch.cuda.is_current_stream_capturing():
        return False
    if inputs[0].device.index not in _err_flags:   # it would be made in the graph's memory, and cleared by every replay
        raise RuntimeError("the first call on a device cannot be captured into a CUDA graph: run one before the capture")
    if torch.is_grad_enabled():
        leaves = [t for t in inputs if t is not None and t.requires_grad and t.is_leaf]
        leaves += _leaves_below(t.grad_fn for t in inputs if t is not None and t.grad_fn is not None)
        with _live_lock:
            nodes = list(_live_nodes)
        held = {id(t) for t in _leaves_below(nodes)} if leaves else ()
        if any(id(t) in held for t in leaves):
            raise RuntimeError("a CUDA graph capture of this call needs the results of earlier eager calls on the same "
                               "leaf tensors to be released or detached first (their autograd graph is alive)")
    return True


_dispatch_mode, _PROXY = torch._C._get_dispatch_mode, torch._C._TorchDispatchModeKey.PROXY
_tracing_state, _functorch_active = torch._C._get_tracing_state, torch._C._are_functorch_transforms_active


def refuse_fx_trace() -> None:
    """A graph traced by ``make_fx`` would hold the empty outputs and none of the kernels, which torch does not see."""
    if _dispatch_mode(_PROXY) is not None:
        raise RuntimeError("the expert-mixture calls cannot be traced by make_fx or torch.export (their kernels are not "
                           "torch operators)")


def _apply(fn, capturing: bool, *args):
    """``fn.apply`` where a gradient may be asked for, else its forward alone. Under torch's transformations always the
    former: ``torch.jit.trace`` records it, and forward mode and ``torch.func`` find no rule and raise, where they would take
    outputs of the bare forward for constants."""
    if _dispatch_mode(_PROXY) is not None:
        refuse_fx_trace()
    recorded = forward_ad._current_level >= 0 or _tracing_state() is not None or _functorch_active()
    if not recorded and torch.is_grad_enabled():
        for t in args:
            if isinstance(t, torch.Tensor) and t.requires_grad:
                recorded = True
                break
    if recorded:
        out = fn.apply(*args)
        if not capturing and out.grad_fn is not None:
            with _live_lock:
                _live_nodes.add(out.grad_fn)
        return out
    return fn.compute(*args)


def _once(backward):
    """``once_differentiable`` only where a second derivative may be asked for: its bookkeeping costs 5 us a call."""
    checked = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return checked(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


@torch.compiler.disable
def _opaque(fn, *args):
    """A traced call: the kernels sit behind ctypes, so torch.compile runs the call eagerly."""
    return fn(*args)


def _unit_stride(x: torch.Tensor) -> torch.Tensor:
    """``x`` [rows, cols] with contiguous rows (any pitch); a copy only where it is not that already."""
    ld, one = x.stride()
    return x if (one == 1 or x.shape[1] == 1) and ld >= x.shape[1] else x.clone(memory_format=torch.contiguous_format)


def _ceil8(n: int) -> int:
    return (n + 7) // 8 * 8


def _split(x: torch.Tensor, offsets, G: int, mat_rows: int, T: int):
    """One array with the two fp16 planes [2, rows, cols rounded up to 8] of an fp32 operand [rows, cols] and, behind
    them, their block scales (``fuma_split_blocks``), and the scales' address: of ragged rows, or (``mat_rows`` > 0) of
    matrices of that many rows, those of groups with rows (of T)."""
    rows, cols = x.shape
    planes = rows * _ceil8(cols)   # two of 2 bytes: as many floats
    blocks = rows // mat_rows * ((mat_rows + 127) // 128) if mat_rows else rows // 128 + G
    out = x.new_empty(planes + (cols + 127) // 128 * blocks)
    at = out.data_ptr()
    nat.call("fuma_split_blocks", ptr(x), x.stride(0), rows, cols, ptr(offsets), G, mat_rows, T, at, at + 4 * planes,
             stream_of(x))
    return out, at + 4 * planes


def _operand(x: torch.Tensor, offsets, G: int):
    """(tensor, leading dimension, address of the scales) of a row operand for the C ABI: 16-bit rows a multiple of 16 bytes apart and
    aligned to that (a copy where they are not), fp32 as planes."""
    x = _unit_stride(x)
    rows, cols = x.shape
    if x.dtype == torch.float32:
        planes, scales = _split(x, offsets, G, 0, rows)
        return planes, _ceil8(cols), scales
    ld = x.stride(0)
    if ld % 8 or x.data_ptr() % 16:
        out = x.new_empty((rows, _ceil8(cols)))
        nat.call("fuma_pad_rows", ptr(x), ld, rows, cols, ptr(out), _ceil8(cols), None, 0, 0, 0, stream_of(x))
        return out, _ceil8(cols), None
    return x, ld, None


def _weight_operand(w: torch.Tensor, offsets, T: int):
    """(tensor, leading dimension, address of the scales) of the matrices [G, N, K] for the C ABI, likewise; a copy leaves out the
    matrices of groups without rows."""
    if not w.is_contiguous():
        w = w.contiguous()
    G, N, K = w.shape
    if w.dtype == torch.float32:
        planes, scales = _split(w.view(G * N, K), offsets, G, N, T)
        return planes, _ceil8(K), scales
    if K % 8 or w.data_ptr() % 16:
        out = w.new_empty((G, N, _ceil8(K)))
        nat.call("fuma_pad_rows", ptr(w), K, G * N, K, ptr(out), _ceil8(K), ptr(offsets), G, N, T, stream_of(w))
        return out, _ceil8(K), None
    return w, K, None


class _GroupedLinearFn(torch.autograd.Function):
    @staticmethod
    def compute(x, weight, offsets, bias, keep_x=False, keep_w=False):
        """y; with ``keep_x`` or ``keep_w``, y and those of the two operands as the kernels read them: the same bytes that
        the backward pass needs again (fp32: planes instead of the values), laid out once."""
        T = x.shape[0]
        G, N, K = weight.shape
        y = x.new_empty((T, N))
        a, w = (x, _ceil8(K), None), (weight, _ceil8(K), None)
        if T:
            bias_rows = 0
            if bias is not None:
                bias_rows = 1 if bias.dim() == 1 else G
                bias = bias.contiguous()
            a, w = _operand(x, offsets, G), _weight_operand(weight, offsets, T)
            nat.call("fuma_grouped_linear", ptr(a[0]), a[1], a[2], ptr(w[0]), w[1], w[2], ptr(offsets), G,
                     ptr(bias), bias_rows, T, N, K, _DTYPES[x.dtype], ptr(y), ptr(error_flag(x.device)), stream_of(x))
        if keep_x or keep_w:
            return y, a if keep_x else (None, 0), w if keep_w else (None, 0)
        return y

    @staticmethod
    def forward(ctx, x, weight, offsets, bias):
        want_x, want_w, _, _ = ctx.needs_input_grad
        a = w = (None, 0)
        out = _GroupedLinearFn.compute(x, weight, offsets, bias, want_w, want_x)
        if want_w or want_x:
            out, a, w = out
        ctx.save_for_backward(a[0], w[0], offsets)
        ctx.lds = a[1], w[1]
        ctx.shapes = x.shape[0], weight.shape, None if bias is None else bias.shape
        return out

    @staticmethod
    @_once
    def backward(ctx, g):
        b, w, offsets = ctx.saved_tensors
        ldb, ldw = ctx.lds
        T, (G, N, K), bias_shape = ctx.shapes
        dev, dt = g.device, g.dtype
        code = _DTYPES[dt]
        want_x, want_w, _, want_b = ctx.needs_input_grad
        dx = dw = db = None
        s, err = stream_of(g), ptr(error_flag(dev))
        g = _unit_stride(g)
        a, lda, a_s = _operand(g, offsets, G) if T and (want_x or want_w) else (g, _ceil8(N), None)
        if want_x:
            dx = g.new_empty((T, K))
            if T:
                w_s = w.data_ptr() + 4 * G * N * ldw if code == 0 else None
                nat.call("fuma_grouped_linear_dgrad", ptr(a), lda, a_s, ptr(w), ldw, w_s, ptr(offsets), G, T, N, K, code,
                         ptr(dx), err, s)
        if want_w:
            dw = g.new_empty((G, N, K))
            nbytes = nat.load().fuma_grouped_wgrad_work_bytes(T, N, K, code)
            work = g.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
            b_s = b.data_ptr() + 4 * T * ldb if code == 0 else None
            nat.call("fuma_grouped_linear_wgrad", ptr(a), lda, a_s, ptr(b), ldb, b_s, ptr(offsets), G, T, N, K, code,
                     ptr(dw), ptr(work), nbytes, err, s)
        if want_b:
            shared = len(bias_shape) == 1
            db = g.new_empty(bias_shape)
            nbytes = nat.load().fuma_grouped_bias_grad_work_bytes(T, N, 1 if shared else G)
            work = g.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
            nat.call("fuma_grouped_bias_grad", ptr(g), g.stride(0) if T else N, ptr(offsets), G, 1 if shared else 0, T, N,
                     code, ptr(db), ptr(work), nbytes, s)
        return dx, dw, None, db


def check_groups(x: torch.Tensor, G: int, N: int, K: int, offsets: torch.Tensor | None, bias: torch.Tensor | None):
    """The argument checks that the grouped dense maps share."""
    shape = x.shape
    if len(shape) != 2 or shape[1] != K:
        raise ValueError(f"x must be [rows, {K}] (got {tuple(shape)})")
    if not 1 <= G <= MAX_GROUPS:
        raise ValueError(f"the number of groups must be from 1 to {MAX_GROUPS} (got {G})")
    if N < 1 or K < 1:
        raise ValueError(f"the matrices need N >= 1 and K >= 1 (got {N} and {K})")
    if offsets is not None:
        if offsets.dtype != torch.int64:
            raise TypeError(f"offsets must be int64 (got {offsets.dtype})")
        if offsets.shape != (G + 1,):
            raise ValueError(f"offsets must be [{G + 1}] for {G} groups (got {tuple(offsets.shape)})")
    if bias is not None and bias.shape not in ((N,), (G, N)):
        raise ValueError(f"bias must be [{N}] or [{G}, {N}] (got {tuple(bias.shape)})")


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor,
                   bias: torch.Tensor | None = None) -> torch.Tensor:
    """``y[t] = weight[g] @ x[t] (+ bias)`` for the rows ``offsets[g] <= t < offsets[g + 1]``.

    x [T, K]; weight [G, N, K]; offsets [G + 1] int64 on the same GPU, not decreasing, within
    [0, T] (groups may be empty; the values are read on the device, so the call does not
    synchronise); bias [N] (one for all groups) or [G, N]. All of one type: float32, bfloat16 or
    float16. Returns [T, N]; rows outside [offsets[0], offsets[G]) come back as zeros and get zero
    gradients. Differentiable in x, weight and bias (once); repeated calls give the same bits.

    16-bit operands whose rows are not contiguous, aligned to 16 bytes and a multiple of 16 bytes apart (an
    odd K, say) run on a copy. Bad offset values are recorded in the device error flag
    (:func:`flash_uma_b200.linear.check_errors`).

    fp32: each operand is taken to 2^-22 of itself or, in a 128 x 128 block (128 rows of one group, from its first row,
    and 128 columns) of widely different magnitudes, to 2^-39 of the block's largest; an infinite input may give NaN
    where fp32 arithmetic gives an infinity. A training call keeps the operands as the kernels read them for the backward
    pass: fp32 planes take the place of x and weight, at the same size."""
    if torch.compiler.is_compiling():
        return _opaque(grouped_linear, x, weight, offsets, bias)
    nat.require_cuda(x, weight, offsets, bias)
    if weight.dim() != 3:
        raise ValueError(f"weight must be [groups, N, K] (got {tuple(weight.shape)})")
    G, N, K = weight.shape
    _check_dtype("x", x)
    if weight.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype):
        raise TypeError("x, weight and bias must have the same dtype")
    check_groups(x, G, N, K, offsets, bias)
    _same_device(x.device, weight=weight, offsets=offsets, bias=bias)
    if not offsets.is_contiguous():
        offsets = offsets.contiguous()
    return _apply(_GroupedLinearFn, guard_capture(x, weight, bias), x, weight, offsets, bias)


class _MixFn(torch.autograd.Function):
    @staticmethod
    def compute(coeff, experts):
        S, E = coeff.shape
        stride_s, stride_e = coeff.stride()
        x = _flat(experts)
        out = experts.new_empty((S, *experts.shape[1:]))
        nat.call("fuma_mix_experts", coeff.data_ptr(), stride_s, stride_e, x.data_ptr(), S, E, x.numel() // E,
                 _DTYPES[experts.dtype], ptr(out), ptr(error_flag(experts.device)), stream_of(experts))
        return out

    @staticmethod
    def forward(ctx, coeff, experts):
        ctx.save_for_backward(coeff, experts)
        return _MixFn.compute(coeff, experts)

    @staticmethod
    @_once
    def backward(ctx, g):
        coeff, experts = ctx.saved_tensors
        S, E = coeff.shape
        P = experts.numel() // E
        want_c, want_e = ctx.needs_input_grad
        dev, code = experts.device, _DTYPES[experts.dtype]
        if S == 0 or P == 0:
            return (torch.zeros_like(coeff) if want_c else None), (torch.zeros_like(experts) if want_e else None)
        dc = de = work = None
        nbytes = 0
        if want_c:
            dc = coeff.new_empty((S, E))
            nbytes = nat.load().fuma_mix_experts_work_bytes(S, E, P, code)
            work = coeff.new_empty(nbytes, dtype=torch.uint8)
        if want_e:
            de = torch.empty_like(experts, memory_format=torch.contiguous_format)
        g, x = _flat(g), _flat(experts)
        nat.call("fuma_mix_experts_bwd", ptr(g), ptr(coeff), coeff.stride(0), coeff.stride(1), ptr(x), S, E, P, code,
                 ptr(dc), ptr(de), ptr(work), nbytes, ptr(error_flag(dev)), stream_of(g))
        return dc, de


def _flat(t: torch.Tensor) -> torch.Tensor:
    if not t.is_contiguous():
        t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def mix_experts(coeff: torch.Tensor, experts: torch.Tensor) -> torch.Tensor:
    """``W[s] = sum_e coeff[s, e] experts[e]``: coeff [S, E] float32 (any strides), experts [E, ...]
    float32, bfloat16 or float16 -> [S, ...] of the experts' type, summed in fp32. Differentiable
    (once) in both; the gradient of coeff is float32, its sum over a matrix in fp64 after at most 4,096 values. Large fp32 mixes run
    on the tensor cores with the precision of :func:`grouped_linear`'s fp32 maps, a block being the same 64 values
    of all matrices; a value that is not finite makes the results that depend on it not finite."""
    if torch.compiler.is_compiling():
        return _opaque(mix_experts, coeff, experts)
    nat.require_cuda(coeff, experts)
    _check_dtype("experts", experts)
    if coeff.dtype != torch.float32:
        raise TypeError(f"coeff must be float32 (got {coeff.dtype})")
    c_shape, e_shape = coeff.shape, experts.shape
    if not e_shape or len(c_shape) != 2 or c_shape[1] != e_shape[0] or e_shape[0] < 1:
        raise ValueError(f"coeff must be [systems, experts] for experts [experts, ...] (got {tuple(c_shape)} and "
                         f"{tuple(e_shape)})")
    if coeff.device != experts.device:
        _same_device(experts.device, coeff=coeff)
    return _apply(_MixFn, guard_capture(coeff, experts), coeff, experts)


class MoleLinear(nn.Module):
    """Mixture-of-linear-experts layer: experts [E, N, K] and one bias [N], trainable;
    ``forward(x, coeff, offsets)`` maps the rows of system s (``offsets[s] <= t < offsets[s + 1]``)
    with ``sum_e coeff[s, e] experts[e]``. ``coeff`` [systems, E] float32 comes from the model's
    router (a softmax over the system embedding, say) and gets its gradient."""

    def __init__(self, experts: torch.Tensor, bias: torch.Tensor | None = None):
        super().__init__()
        if experts.dim() != 3:
            raise ValueError(f"experts must be [experts, N, K] (got {tuple(experts.shape)})")
        self.experts = nn.Parameter(experts.detach().clone())
        self.bias = None if bias is None else nn.Parameter(bias.detach().clone())

    def forward(self, x: torch.Tensor, coeff: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
        return grouped_linear(x, mix_experts(coeff, self.experts), offsets, self.bias)

    def extra_repr(self) -> str:
        E, N, K = self.experts.shape
        return f"experts={E}, N={N}, K={K}, bias={self.bias is not None}"
