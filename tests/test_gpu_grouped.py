"""Grouped dense maps and mixed expert weights (``flash_uma_b200.grouped``) against plain fp64 sums.

Tolerances are per element and derived, not fitted. With S = sum of |products| of an element:
the tensor core truncates one addition per 16 products to 24 bits (2^-23 of a partial sum, which is
at most S), the epilogue rounds once per segment (2^-24 S each), the fp32 planes drop products below
3 * 2^-24 S and the result is rounded to its type once (half an eps of it):
    |error| <= eps/2 |y| + (n / 16 + 12) 2^-23 S       for a contraction of n values.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _half(dt):
    return torch.finfo(dt).eps / 2


def _close(got, want, S, n, dt, what):
    tol = _half(dt) * want.abs() + (n / 16 + 12) * 2.0 ** -23 * S + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    bad = ((got.double() - want).abs() > tol) | ~torch.isfinite(got.double())
    assert got.dtype == dt and got.shape == want.shape
    assert not bad.any(), (what, int(bad.sum()), float(((got.double() - want).abs() / tol).max()))


def _make(lens, K, N, dt, bias=None, head=0, tail=0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    T, G = head + sum(lens) + tail, len(lens)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g).to(dt)   # noqa: E731
    x, w, gy = r(T, K), r(G, N, K), r(T, N)
    b = None if bias is None else r(N) if bias == "shared" else r(G, N)
    off = torch.tensor([head] + lens, device=DEV).cumsum(0)
    return x, w, off, b, gy


def _oracle(x, w, off, b, gy):
    """fp64 results and the sums of |products|: y, dx, dw, db, and S of the first three."""
    X, W, GY = x.double(), w.double(), gy.double()
    G, N, K = w.shape
    y, Sy = X.new_zeros(x.shape[0], N), X.new_zeros(x.shape[0], N)
    dx, Sx = torch.zeros_like(X), torch.zeros_like(X)
    dw, Sw, db, Sb = torch.zeros_like(W), torch.zeros_like(W), X.new_zeros(G, N), X.new_zeros(G, N)
    o = off.tolist()
    for g in range(G):
        s = slice(o[g], o[g + 1])
        y[s], Sy[s] = X[s] @ W[g].T, X[s].abs() @ W[g].abs().T
        if b is not None:
            bg = (b if b.dim() == 1 else b[g]).double()
            y[s] += bg
            Sy[s] += bg.abs()
        dx[s], Sx[s] = GY[s] @ W[g], GY[s].abs() @ W[g].abs()
        dw[g], Sw[g] = GY[s].T @ X[s], GY[s].abs().T @ X[s].abs()
        db[g], Sb[g] = GY[s].sum(0), GY[s].abs().sum(0)
    if b is not None and b.dim() == 1:
        db, Sb = db.sum(0), Sb.sum(0)
    return y, Sy, dx, Sx, dw, Sw, db, Sb


def _check(x, w, off, b, gy, dt):
    from flash_uma_b200 import linear
    from flash_uma_b200.grouped import grouped_linear
    leaves = [t.detach().clone().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = grouped_linear(leaves[0], leaves[1], off, leaves[2])
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], gy)
    torch.cuda.synchronize()
    linear.check_errors()
    Y, Sy, DX, Sx, DW, Sw, DB, Sb = _oracle(x, w, off, b, gy)
    K, N = x.shape[1], w.shape[1]
    longest = int((off[1:] - off[:-1]).max())
    _close(y.detach(), Y, Sy, K, dt, "y")
    _close(grads[0], DX, Sx, N, dt, "dx")
    _close(grads[1], DW, Sw, longest, dt, "dw")
    if b is not None:
        _close(grads[2], DB, Sb, 16 * 512, dt, "db")   # 512 fp32 additions per piece
    return y.detach(), grads


SHAPES = [
    # lens, K, N, head, tail
    ([1], 64, 64, 0, 0),
    ([1], 8, 8, 0, 0),
    ([3], 768, 640, 0, 0),
    ([0, 5, 0, 130, 1, 0, 127, 128, 0], 72, 136, 0, 0),
    ([300, 20], 256, 264, 7, 200),
    ([33, 200, 64], 520, 392, 0, 3),
    ([17, 0, 40], 13, 7, 2, 1),          # odd widths
    ([9, 1], 1, 1, 1, 0),
    ([50, 130, 0, 2], 65, 129, 0, 3),
    ([40, 0, 300], 535, 583, 1, 0),
    ([31], 260, 131, 0, 0),
    ([129], 1032, 520, 0, 0),
]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("bias", [None, "shared", "group"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"K{s[1]}N{s[2]}T{sum(s[0])}")
def test_forward_and_gradients(shape, bias, dt):
    lens, K, N, head, tail = shape
    x, w, off, b, gy = _make(lens, K, N, dt, bias, head, tail)
    y, grads = _check(x, w, off, b, gy, dt)
    dead = torch.ones(x.shape[0], dtype=torch.bool, device=DEV)
    dead[head:head + sum(lens)] = False
    assert not y[dead].any() and not grads[0][dead].any()
    for g, n in enumerate(lens):
        if n == 0:
            assert not grads[1][g].any()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("K,N", [(72, 40), (71, 33), (70, 44)])
def test_long_groups_cut_over_the_contraction(dt, K, N):
    """Groups longer than one chunk of the weight gradient, next to short and empty ones, with chunk
    ends inside tiles."""
    x, w, off, b, gy = _make([2047, 5001, 0, 2049, 6200, 3], K, N, dt, "group", 1, 5)
    _check(x, w, off, b, gy, dt)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("lens,K,N,head,tail", [([20000], 72, 256, 0, 0), ([9001, 0, 257, 8000, 128, 129], 136, 640, 3, 77),
                                                ([5000, 5100], 520, 392, 0, 0), ([60000, 60001], 264, 264, 0, 0),
                                                ([30001, 0, 20000, 257, 25128, 129], 520, 640, 3, 77)])
def test_long_groups_on_cta_pairs(lens, K, N, head, tail, dt):
    """Groups long enough for the 256-row tiles of CTA pairs, with last tiles of 1, 128, 129 and 256 rows."""
    x, w, off, b, gy = _make(lens, K, N, dt, "shared", head, tail)
    _check(x, w, off, b, gy, dt)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("G", [700, 4096])
def test_many_groups(dt, G):
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 9, (G,), generator=g).tolist()
    x, w, off, b, gy = _make(lens, 40, 24, dt, "group")
    _check(x, w, off, b, gy, dt)


@pytest.mark.parametrize("dt", DTYPES)
def test_groups_do_not_see_each_other(dt):
    """NaN and infinities in one group's rows, matrix and bias, and in rows outside all groups, stay there."""
    from flash_uma_b200.grouped import grouped_linear
    lens, K, N = [70, 50, 90], 72, 40
    x, w, off, b, gy = _make(lens, K, N, dt, "group", 3, 9)
    lo, hi = int(off[1]), int(off[2])
    clean = _oracle(x, w, off, b, gy)
    x2, w2, b2, gy2 = x.clone(), w.clone(), b.clone(), gy.clone()
    for t in (x2, gy2):
        t[lo:hi] = float("nan")
        t[lo + 3] = float("inf")
        t[:3] = float("inf")
        t[-9:] = float("nan")
    w2[1] = float("inf")
    b2[1] = float("nan")
    for t in (x2, w2, b2):
        t.requires_grad_(True)
    y = grouped_linear(x2, w2, off, b2)
    dx, dw, db = torch.autograd.grad(y, [x2, w2, b2], gy2)
    y = y.detach()
    keep = [s for s in range(3, 3 + sum(lens)) if not lo <= s < hi]
    _close(y[keep], clean[0][keep], clean[1][keep], K, dt, "y")
    _close(dx[keep], clean[2][keep], clean[3][keep], N, dt, "dx")
    _close(dw[[0, 2]], clean[4][[0, 2]], clean[5][[0, 2]], 90, dt, "dw")
    _close(db[[0, 2]], clean[6][[0, 2]], clean[7][[0, 2]], 16 * 512, dt, "db")
    assert torch.isnan(y[lo:hi]).all()
    assert not y[:3].any() and not y[-9:].any() and not dx[:3].any() and not dx[-9:].any()


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e5, 1e15])
def test_fp32_whole_range(scale):
    """fp32 operands far outside fp16's range keep their 24 bits."""
    x, w, off, b, gy = _make([70, 33], 136, 72, torch.float32)
    _check(x * scale, w, off, None, gy * scale, torch.float32)


@pytest.mark.parametrize("dt", DTYPES)
def test_strides_and_alignment(dt):
    from flash_uma_b200.grouped import grouped_linear
    x, w, off, b, gy = _make([70, 33], 136, 72, dt, "shared")
    want = grouped_linear(x, w, off, b)
    wide = torch.full((x.shape[0], 200), float("nan"), device=DEV, dtype=dt)
    for c in (8, 5):                                  # aligned and not aligned column slices
        v = wide[:, c:c + 136]
        v.copy_(x)
        assert torch.equal(grouped_linear(v, w, off, b), want)
    assert torch.equal(grouped_linear(x.t().contiguous().t(), w, off, b), want)
    assert torch.equal(grouped_linear(x, w.transpose(1, 2).contiguous().transpose(1, 2), off, b), want)
    assert torch.equal(grouped_linear(x, w, off.repeat_interleave(2)[::2], b), want)
    row = x[:1].expand(x.shape[0], -1)                # a broadcast input: its gradient is the sum over rows
    leaf = x[:1].detach().clone().requires_grad_(True)
    y = grouped_linear(leaf.expand(x.shape[0], -1), w, off, b)
    assert torch.equal(y.detach(), grouped_linear(row, w, off, b))
    (gl,) = torch.autograd.grad(y, [leaf], gy)
    X, W = leaf.detach().double(), w.double()
    o = off.tolist()
    each = torch.cat([gy[o[g]:o[g + 1]].double() @ W[g] for g in range(2)])
    S = torch.cat([gy[o[g]:o[g + 1]].double().abs() @ W[g].abs() for g in range(2)])
    n = x.shape[0]
    # each row's gradient rounded to dt, then torch's own sum over the n rows
    tol = (2 * _half(dt) * each.abs().sum(0) + (72 / 16 + 12 + n) * 2.0 ** -23 * S.sum(0)) + \
        _half(dt) * each.sum(0).abs()
    assert ((gl[0].double() - each.sum(0)).abs() <= tol).all()


@pytest.mark.parametrize("dt", DTYPES)
def test_no_rows(dt):
    from flash_uma_b200.grouped import grouped_linear
    x = torch.empty(0, 16, device=DEV, dtype=dt, requires_grad=True)
    w = torch.randn(3, 24, 16, device=DEV).to(dt).requires_grad_(True)
    b = torch.randn(24, device=DEV).to(dt).requires_grad_(True)
    off = torch.zeros(4, dtype=torch.int64, device=DEV)
    y = grouped_linear(x, w, off, b)
    assert y.shape == (0, 24)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty(0, 24, device=DEV, dtype=dt))
    assert dx.shape == (0, 16) and not dw.any() and not db.any() and torch.isfinite(dw).all()
    # rows, but every group empty
    x = torch.randn(5, 16, device=DEV).to(dt).requires_grad_(True)
    y = grouped_linear(x, w, off + 2, b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.ones(5, 24, device=DEV, dtype=dt))
    assert not y.any() and not dx.any() and not dw.any() and not db.any()


@pytest.mark.parametrize("dt", DTYPES)
def test_same_bits_and_graph_replay(dt):
    """Repeated calls, a captured and replayed call on new data, and another stream give the same bits. A
    capture while an eager graph of the same leaves lives is refused."""
    from flash_uma_b200.grouped import grouped_linear
    x, w, off, b, gy = _make([2500, 0, 300, 2100], 72, 136, dt, "shared")
    for t in (x, w, b):
        t.requires_grad_(True)

    def step():
        y = grouped_linear(x, w, off, b)
        return (y.detach(), *torch.autograd.grad(y, [x, w, b], gy))
    first, again = step(), step()
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first, other))
    held = grouped_linear(x, w, off, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="eager"):
            step()
        torch.zeros(1, device=DEV)
    del held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.mul_(0.5)
        off[1:3] -= 100
    graph.replay()
    fresh = step()
    assert all(torch.equal(p, q) for p, q in zip(out, fresh))


def test_bad_offsets_are_recorded():
    from flash_uma_b200 import linear
    from flash_uma_b200.grouped import grouped_linear
    x, w, off, b, gy = _make([70, 33], 136, 72, torch.bfloat16)
    for bad in ([0, 80, 70], [-1, 50, 103], [0, 50, 104], [2 ** 40, 2 ** 41, 2 ** 42]):
        grouped_linear(x, w, torch.tensor(bad, device=DEV))
        with pytest.raises(RuntimeError, match="offsets"):
            linear.check_errors()
    grouped_linear(x, w, off)
    linear.check_errors()


def test_refusals():
    from flash_uma_b200.grouped import grouped_linear, mix_experts
    x, w, off, b, gy = _make([70, 33], 136, 72, torch.bfloat16, "shared")
    with pytest.raises(TypeError):
        grouped_linear(x.float(), w, off)
    with pytest.raises(TypeError):
        grouped_linear(x.double(), w.double(), off)
    with pytest.raises(TypeError):
        grouped_linear(x, w, off.int())
    with pytest.raises(TypeError):
        grouped_linear(x, w, off, b.float())
    for bad in (off[:2], off[None]):
        with pytest.raises(ValueError):
            grouped_linear(x, w, bad)
    with pytest.raises(ValueError):
        grouped_linear(x[:, :8], w, off)
    with pytest.raises(ValueError):
        grouped_linear(x, w[0], off)
    with pytest.raises(ValueError):
        grouped_linear(x, w, off, b[:8])
    with pytest.raises(ValueError):
        grouped_linear(x[:, :8], torch.zeros(4097, 8, 8, device=DEV, dtype=x.dtype),
                       torch.zeros(4098, device=DEV, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        grouped_linear(x.cpu(), w, off)
    with pytest.raises(RuntimeError, match="CUDA"):
        grouped_linear(x, w, off.cpu())
    c = torch.rand(3, 4, device=DEV)
    with pytest.raises(TypeError):
        mix_experts(c.bfloat16(), torch.zeros(4, 8, device=DEV))
    with pytest.raises(ValueError):
        mix_experts(c, torch.zeros(5, 8, device=DEV))
    y = grouped_linear(x.requires_grad_(True), w, off)
    (g,) = torch.autograd.grad(y.float().sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), [x])


# ---- mixed weights ---------------------------------------------------------------------------------

@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("S,E,shape", [(1, 1, (4,)), (1, 8, (16, 24)), (5, 3, (7, 9)), (33, 70, (24, 40)),
                                       (130, 64, (520,)), (64, 32, (37, 111)), (9, 130, (8, 1000)), (65, 2, (1,))])
def test_mix(S, E, shape, dt):
    """Sums of n products in fp32: n 2^-24 of S = the sum of |products|, and one rounding of the result. The tensor
    core truncates (2^-23 S) up to three additions per 16 products. fp32 matrices and coefficients are two fp16 planes each:
    hi is within 2^-11 of x, so lo = fp16(x - hi) within 2^-22 of it, for both operands, and the product lo lo <= 2^-22
    is dropped: 3 * 2^-22 = 12 * 2^-24 of S more. dc sums up to 4096 products in fp32 before the fp64 join."""
    from flash_uma_b200.grouped import mix_experts
    g = torch.Generator(device=DEV).manual_seed(1)
    c = torch.randn(S, E, device=DEV, generator=g).requires_grad_(True)
    x = torch.randn(E, *shape, device=DEV, generator=g).to(dt).requires_grad_(True)
    gw = torch.randn(S, *shape, device=DEV, generator=g).to(dt)
    w = mix_experts(c, x)
    dc, dx = torch.autograd.grad(w, [c, x], gw)
    C, X, GW = c.detach().double(), x.detach().double().flatten(1), gw.double().flatten(1)

    def check(got, want, S_, n, t):
        steps = n + 1 + 6 * -(-n // 16) + (12 if dt == torch.float32 else 0)
        tol = _half(t) * want.abs() + steps * 2.0 ** -24 * S_ + torch.finfo(t).smallest_normal * torch.finfo(t).eps
        assert got.dtype == t and (got.double().reshape(want.shape) - want).abs().le(tol).all()
    check(w.detach(), C @ X, C.abs() @ X.abs(), E, dt)
    check(dx, C.T @ GW, C.T.abs() @ GW.abs(), S, dt)
    check(dc, GW @ X.T, GW.abs() @ X.T.abs(), 2 * min(X.shape[1], 4096), torch.float32)
    assert torch.equal(mix_experts(c.detach().t().contiguous().t(), x.detach()), w.detach())


def test_mix_empty():
    from flash_uma_b200.grouped import mix_experts
    x = torch.randn(3, 8, device=DEV, requires_grad=True)
    c = torch.zeros(0, 3, device=DEV, requires_grad=True)
    w = mix_experts(c, x)
    dc, dx = torch.autograd.grad(w, [c, x], torch.empty(0, 8, device=DEV))
    assert w.shape == (0, 8) and dc.shape == (0, 3) and not dx.any()


@pytest.mark.parametrize("dt", DTYPES)
def test_mole_layer(dt):
    """Router coefficients -> mixed weights -> grouped map, with all gradients, against the same layer in
    fp64 (the mixed weights rounded to the type as the layer stores them) and against differences."""
    from flash_uma_b200.grouped import MoleLinear
    g = torch.Generator(device=DEV).manual_seed(3)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g)   # noqa: E731
    lens, E, N, K = [40, 0, 129, 7], 6, 72, 56
    off = torch.tensor([0] + lens, device=DEV).cumsum(0)
    layer = MoleLinear((r(E, N, K) * K ** -0.5).to(dt), r(N).to(dt))
    x = r(sum(lens), K).to(dt).requires_grad_(True)
    logits = r(len(lens), E).requires_grad_(True)
    gy = r(sum(lens), N).to(dt)
    y = layer(x, torch.softmax(logits, 1), off)
    got = torch.autograd.grad(y, [x, logits, layer.experts, layer.bias], gy)

    L = logits.detach().double().requires_grad_(True)
    X64 = x.detach().double().requires_grad_(True)
    E64 = layer.experts.detach().double().requires_grad_(True)
    B64 = layer.bias.detach().double().requires_grad_(True)

    def f64(L, E64, X64, B64):
        W = torch.einsum("se,enk->snk", torch.softmax(L, 1), E64)
        return torch.cat([X64[a:z] @ W[s].T + B64 for s, (a, z) in
                          enumerate(zip(off.tolist()[:-1], off.tolist()[1:]))])
    Y = f64(L, E64, X64, B64)
    want = torch.autograd.grad(Y, [X64, L, E64, B64], gy.double())
    # mixed weights, results and weight gradients are each rounded to dt: a few half-eps of the norms
    for p, q in zip((y.detach(), *got), (Y.detach(), *want)):
        assert (p.double() - q).norm() <= (4 * _half(dt) + 2.0 ** -20) * max(q.norm(), 1e-30)
    # directional differences of the fp64 layer
    d = [torch.randn_like(t) for t in (L, E64, X64, B64)]
    h = 1e-6
    with torch.no_grad():
        up = (f64(*[t + h * u for t, u in zip((L, E64, X64, B64), d)]) * gy.double()).sum()
        dn = (f64(*[t - h * u for t, u in zip((L, E64, X64, B64), d)]) * gy.double()).sum()
    grads = (got[1], got[2], got[0], got[3])
    slope = sum((gr.double() * u).sum() for gr, u in zip(grads, d))
    size = sum((gr.double() * u).norm() for gr, u in zip(grads, d))
    assert abs(slope - (up - dn) / (2 * h)) <= (8 * _half(dt) + 1e-6) * size * 4


# ---- what a user may do with them ------------------------------------------------------------------

def test_fp32_blocks_of_mixed_magnitudes():
    """Rows, columns and matrices whose magnitudes differ by up to 2^40 within a block. A block is scaled so that its largest
    magnitude M is below 2^15, where the second plane's smallest step is 2^-24 and its rounding 2^-25: 2^-39 M, or 2^-22 of
    the value itself. So besides the bound of :func:`_close` (with 12 2^-24 of S for the planes in it) each product
    may be off by 2^-39 (M_x |w| + |x| M_w); M over the whole operand is at least a block's."""
    lens, K, N = [300, 20, 129], 200, 136
    x, w, off, b, gy = _make(lens, K, N, torch.float32, None, 0, 0, 7)
    g = torch.Generator(device=DEV).manual_seed(8)
    mag = lambda n: 2.0 ** torch.randint(-20, 21, (n, 1), device=DEV, generator=g)   # noqa: E731
    x, gy = x * mag(x.shape[0]), gy * mag(x.shape[0])
    w = w * mag(N)
    from flash_uma_b200.grouped import grouped_linear
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = grouped_linear(xl, wl, off)
    dx, dw = torch.autograd.grad(y, [xl, wl], gy)
    Y, Sy, DX, Sx, DW, Sw, _, _ = _oracle(x, w, off, b, gy)
    X, W, GY = x.double().abs(), w.double().abs(), gy.double().abs()
    Mx, Mw, Mg = X.max(), W.max(), GY.max()
    o = off.tolist()
    for i in range(len(lens)):
        r = slice(o[i], o[i + 1])
        for got, want, S, n, extra in (
                (y.detach()[r], Y[r], Sy[r], K, Mx * W[i].sum(1)[None] + Mw * X[r].sum(1)[:, None]),
                (dx[r], DX[r], Sx[r], N, Mg * W[i].sum(0)[None] + Mw * GY[r].sum(1)[:, None]),
                (dw[i], DW[i], Sw[i], lens[i], Mg * X[r].sum(0)[None] + Mx * GY[r].sum(0)[:, None])):
            tol = (n / 16 + 12) * 2.0 ** -23 * S + 2.0 ** -39 * extra
            assert (got.double() - want).abs().le(tol).all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("S,E,P", [(3, 5, 304), (40, 33, 304), (40, 33, 305), (70, 70, 640)])
def test_mix_not_finite_values_stay_in_their_column(S, E, P, dt):
    """NaN or an infinity in expert e0 at p0 reaches W[:, p0] and dc[:, e0]; in the gradient of W[s0] at p1, dX[:, p1]
    and dc[s0, :]; everything else keeps its value to the rounding of the results."""
    from flash_uma_b200.grouped import mix_experts
    g = torch.Generator(device=DEV).manual_seed(2)
    c = torch.rand(S, E, device=DEV, generator=g) + 0.5
    x = torch.randn(E, P, device=DEV, generator=g).to(dt)
    gw = torch.randn(S, P, device=DEV, generator=g).to(dt)
    e0, p0, s0, p1 = E // 2, 65, S // 2, P - 1

    def run(x, gw):
        cl, xl = c.clone().requires_grad_(True), x.clone().requires_grad_(True)
        w = mix_experts(cl, xl)
        return (w.detach(), *torch.autograd.grad(w, [cl, xl], gw))
    w0, dc0, dx0 = run(x, gw)
    for bad in (float("nan"), float("inf")):
        x1, gw1 = x.clone(), gw.clone()
        x1[e0, p0], gw1[s0, p1] = bad, bad
        w, dc, dx = run(x1, gw1)
        assert not w[:, p0].isfinite().any() and not dx[:, p1].isfinite().any()
        assert not dc[:, e0].isfinite().any() and not dc[s0].isfinite().any()
        for got, want, dim, i in ((w, w0, 1, p0), (dx, dx0, 1, p1)):
            keep = torch.arange(P, device=DEV) != i
            # a tile's scale may change with its largest finite value: the planes' bound on either side
            tol = 4 * _half(dt) * want.abs() + 2.0 ** -16
            assert (got - want).abs().le(tol).index_select(dim, keep.nonzero()[:, 0]).all()
        keep_s, keep_e = torch.arange(S, device=DEV) != s0, torch.arange(E, device=DEV) != e0
        assert torch.allclose(dc[keep_s][:, keep_e], dc0[keep_s][:, keep_e], rtol=1e-4, atol=1e-3)


@pytest.mark.parametrize("dt", DTYPES)
def test_mix_operands_of_any_layout_and_single_gradients(dt):
    """Expanded and strided coefficients, experts and gradients that are not contiguous or aligned, and each gradient
    alone, against the contiguous call with both."""
    from flash_uma_b200.grouped import mix_experts
    g = torch.Generator(device=DEV).manual_seed(4)
    S, E, N, K = 12, 34, 24, 40
    c = torch.randn(S, E, device=DEV, generator=g)
    x = torch.randn(E, N, K, device=DEV, generator=g).to(dt)
    gw = torch.randn(S, N, K, device=DEV, generator=g).to(dt)

    def run(c, x, gw, grads=(True, True)):
        c, x = c.detach().requires_grad_(grads[0]), x.detach().requires_grad_(grads[1])
        w = mix_experts(c, x)
        got = torch.autograd.grad(w, [t for t in (c, x) if t.requires_grad], gw)
        return (w.detach(), *got)
    w, dc, dx = run(c, x, gw)
    xt = x.permute(1, 2, 0).contiguous().permute(2, 0, 1)
    off = torch.empty(x.numel() + 1, device=DEV, dtype=dt)[1:].view(x.shape).copy_(x)
    gt = gw.transpose(1, 2).contiguous().transpose(1, 2)
    ct = torch.empty(E, 2 * S, device=DEV).t()[::2].copy_(c)
    for xi in (xt, off):
        for p, q in zip(run(ct, xi, gt), (w, dc, dx)):
            assert torch.equal(p, q)
    # one gradient alone may take another kernel: fp32 sums in another order
    s_c = gw.double().abs().flatten(1) @ x.double().abs().flatten(1).T
    s_x = torch.einsum("se,snk->enk", c.double().abs(), gw.double().abs())
    assert (run(c, x, gw, (True, False))[1] - dc).double().abs().le((2 * N * K + 40) * 2.0 ** -24 * s_c).all()
    assert (run(c, x, gw, (False, True))[1].double() - dx.double()).abs().le(
        2 * _half(dt) * dx.double().abs() + (S + 60) * 2.0 ** -24 * s_x).all()
    one = torch.randn(1, E, device=DEV, generator=g).expand(S, E).requires_grad_(True)
    y = mix_experts(one, x)
    assert torch.equal(y[0], y[-1])


@pytest.mark.parametrize("dt", DTYPES)
def test_two_captured_layers_replayed_in_turn(dt):
    """A layer's training step, small and with groups long enough for CTA pairs and for cut weight gradients, captured twice in
    one memory pool and replayed alternately on new data, gives the eager call's bits."""
    from flash_uma_b200.grouped import MoleLinear
    g = torch.Generator(device=DEV).manual_seed(6)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g)   # noqa: E731
    steps = []
    for lens, E, N, K in (([5, 0, 130], 3, 72, 40), ([9000, 31000], 40, 520, 136)):
        off = torch.tensor([0] + lens, device=DEV).cumsum(0)
        layer = MoleLinear((r(E, N, K) * K ** -0.5).to(dt), r(N).to(dt))
        x, gy = r(sum(lens), K).to(dt).requires_grad_(True), r(sum(lens), N).to(dt)
        coeff = torch.rand(len(lens), E, device=DEV, generator=g).requires_grad_(True)

        def step(layer=layer, x=x, coeff=coeff, off=off, gy=gy):
            y = layer(x, coeff, off)
            return (y.detach(), *torch.autograd.grad(y, [x, coeff, layer.experts, layer.bias], gy))
        steps.append((step, x, coeff))
    for step, _, _ in steps:
        step()
    pool = torch.cuda.graph_pool_handle()
    graphs, outs = [], []
    for step, _, _ in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(step())
        graphs.append(graph)
    for i in (0, 1, 0, 1):
        step, x, coeff = steps[i]
        with torch.no_grad():
            x.mul_(-0.5)
            coeff.add_(0.25)
        graphs[i].replay()
        got = [t.clone() for t in outs[i]]
        assert all(torch.equal(p, q) for p, q in zip(got, step()))


def test_layer_under_torch_compile():
    """The layer's calls are opaque to a trace and run eagerly, with gradients."""
    from flash_uma_b200.grouped import MoleLinear
    g = torch.Generator(device=DEV).manual_seed(9)
    off = torch.tensor([0, 40, 57], device=DEV)
    layer = MoleLinear(torch.randn(4, 24, 16, device=DEV, generator=g), torch.randn(24, device=DEV, generator=g))
    x = torch.randn(57, 16, device=DEV, generator=g).requires_grad_(True)
    c = torch.rand(2, 4, device=DEV, generator=g).requires_grad_(True)
    f = lambda x, c: layer(x * 2, torch.softmax(c, 1), off) + 1   # noqa: E731
    want = f(x, c)
    got = torch.compile(f, backend="eager")(x, c)
    assert torch.equal(got, want)
    for p, q in zip(torch.autograd.grad(got.sum(), [x, c]), torch.autograd.grad(want.sum(), [x, c])):
        assert torch.equal(p, q)


def test_first_call_in_a_capture_is_refused():
    """The device's error flag would be made in the graph's memory."""
    from flash_uma_b200 import linear
    from flash_uma_b200.grouped import mix_experts
    c, x = torch.rand(2, 4, device=DEV), torch.rand(4, 8, device=DEV)
    mix_experts(c, x)
    held = dict(linear._err_flags)
    linear._err_flags.clear()
    try:
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            with pytest.raises(RuntimeError, match="first call"):
                mix_experts(c, x)
            torch.zeros(1, device=DEV)
    finally:
        linear._err_flags.update(held)


def test_gradient_of_an_expanded_bias_and_of_a_row_taken_twice():
    """Autograd joins what the operator gives for inputs that were broadcast or used twice."""
    from flash_uma_b200.grouped import grouped_linear
    x, w, off, b, gy = _make([33, 0, 90], 48, 40, torch.float32, "shared", 1, 2)
    X, W, B = (t.clone().requires_grad_(True) for t in (x[:1], w[:1], b))
    y = grouped_linear(X.expand(x.shape[0], -1), W.expand(3, -1, -1), off, B.expand(3, -1))
    got = torch.autograd.grad(y, [X, W, B], gy)
    live = gy.double()[1:124]
    assert torch.allclose(got[0].double(), (live @ w[0].double()).sum(0, keepdim=True), rtol=1e-5, atol=1e-4)
    assert torch.allclose(got[1][0].double(), live.sum(0)[:, None] * x[0].double()[None], rtol=1e-5, atol=1e-4)
    assert torch.allclose(got[2].double(), live.sum(0), rtol=1e-5, atol=1e-4)


def test_rows_past_32_bit_offsets():
    """2^21 + 5 rows of 1032 values: the last group starts behind element 2^31 of x and of dx."""
    from flash_uma_b200 import linear
    from flash_uma_b200.grouped import grouped_linear
    T, K, N, n = 2 ** 21 + 5, 1032, 16, 300
    dt = torch.bfloat16
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.zeros(T, K, device=DEV, dtype=dt)
    x[-n:] = torch.randn(n, K, device=DEV, generator=g).to(dt)
    gy = torch.zeros(T, N, device=DEV, dtype=dt)
    gy[-n:] = torch.randn(n, N, device=DEV, generator=g).to(dt)
    w = torch.randn(2, N, K, device=DEV, generator=g).to(dt)
    off = torch.tensor([0, T - n + 100, T - 1], device=DEV)
    xl, wl = x.requires_grad_(True), w.clone().requires_grad_(True)
    y = grouped_linear(xl, wl, off)
    dx, dw = torch.autograd.grad(y, [xl, wl], gy)
    linear.check_errors()
    small = _oracle(x.detach()[-n:], w, torch.tensor([0, 100, n - 1], device=DEV), None, gy[-n:])
    _close(y.detach()[-n:], small[0], small[1], K, dt, "y")
    _close(dx[-n:], small[2], small[3], N, dt, "dx")
    _close(dw, small[4], small[5], T, dt, "dw")
    assert not y.detach()[:-n].any() and not dx[:-n].any()


def test_mix_past_32_bit_offsets():
    """Matrices of 2^31 + 8 values, more than a tensor map addresses."""
    from flash_uma_b200.grouped import mix_experts
    P, dt = 2 ** 31 + 8, torch.bfloat16
    c = torch.tensor([[0.75, -1.5]], device=DEV).requires_grad_(True)
    x = torch.zeros(2, P, device=DEV, dtype=dt)
    x[0, -3:], x[1, -5:] = 2.0, 0.5
    x[0, :7] = 1.0
    x.requires_grad_(True)
    w = mix_experts(c, x)
    gw = torch.zeros(1, P, device=DEV, dtype=dt)
    gw[0, -4:], gw[0, 0] = 1.0, 8.0
    dc, dx = torch.autograd.grad(w, [c, x], gw)
    assert w.detach()[0, -6:].tolist() == [0.0, -0.75, -0.75, 0.75, 0.75, 0.75] and w.detach()[0, :8].tolist() == [0.75] * 7 + [0]
    assert dc.tolist() == [[14.0, 2.0]]
    assert dx[0, -5:].tolist() == [0.0] + [0.75] * 4 and dx[1, -5:].tolist() == [0.0] + [-1.5] * 4
    assert dx[:, 0].tolist() == [6.0, -12.0] and int((dx != 0).sum()) == 10


def test_capture_while_an_eager_graph_of_the_layer_lives_is_refused():
    """Also where the shared leaf is behind another operator (the router's logits, behind a softmax)."""
    from flash_uma_b200.grouped import MoleLinear
    g = torch.Generator(device=DEV).manual_seed(9)
    off = torch.tensor([0, 40, 57], device=DEV)
    layer = MoleLinear(torch.randn(4, 24, 16, device=DEV, generator=g)).requires_grad_(False)
    x = torch.randn(57, 16, device=DEV, generator=g)
    logits = torch.randn(2, 4, device=DEV, generator=g).requires_grad_(True)

    def step():
        y = layer(x, torch.softmax(logits, 1), off)
        return torch.autograd.grad(y.sum(), logits)[0]
    want = step()
    held = layer(x, torch.softmax(logits, 1), off)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="eager"):
            step()
        torch.zeros(1, device=DEV)
    del held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    assert torch.equal(got, want)


def test_two_threads_on_two_streams():
    from flash_uma_b200.grouped import MoleLinear
    import threading
    g = torch.Generator(device=DEV).manual_seed(9)
    off = torch.tensor([0, 400, 457], device=DEV)
    layer = MoleLinear(torch.randn(4, 72, 56, device=DEV, generator=g), torch.randn(72, device=DEV, generator=g))
    x = torch.randn(457, 56, device=DEV, generator=g)
    c = torch.rand(2, 4, device=DEV, generator=g)

    def step():
        xl = x.clone().requires_grad_(True)
        y = layer(xl, c, off)
        return (y.detach(), *torch.autograd.grad(y.sum(), [xl, layer.experts, layer.bias]))   # an expanded gradient
    want, bad = step(), []
    torch.cuda.synchronize()

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = step()
                s.synchronize()
                if not all(torch.equal(p, q) for p, q in zip(got, want)):
                    bad.append(1)
    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_default_dtype_of_64_bits():
    """The work arrays do not follow torch's default type."""
    from flash_uma_b200.fp8 import Fp8Weight, fp8_linear
    from flash_uma_b200.grouped import MoleLinear
    g = torch.Generator(device=DEV).manual_seed(3)
    off = torch.tensor([0, 130, 257], device=DEV)
    layer = MoleLinear(torch.randn(4, 72, 130, device=DEV, generator=g))
    x = torch.randn(257, 130, device=DEV, generator=g).requires_grad_(True)
    c = torch.rand(2, 4, device=DEV, generator=g).requires_grad_(True)
    w8 = torch.randn(72, 130, device=DEV, generator=g)

    def run():
        y = layer(x, c, off)
        return (y.detach(), *torch.autograd.grad(y.sum(), [x, c, layer.experts]), fp8_linear(x, Fp8Weight(w8)).detach())
    want = run()
    torch.set_default_dtype(torch.float64)
    try:
        got = run()
    finally:
        torch.set_default_dtype(torch.float32)
    assert all(p.dtype == q.dtype and torch.equal(p, q) for p, q in zip(got, want))


def test_rows_of_2_31_bytes_outside_all_groups_are_zeros():
    from flash_uma_b200.grouped import grouped_linear
    T, N, K, dt = 3, 2 ** 30, 8, torch.bfloat16
    w = torch.zeros(1, N, K, device=DEV, dtype=dt)
    w[0, -5:] = 1.0
    poison = torch.full((T, N), float("nan"), device=DEV, dtype=dt)   # the memory that the result is likely to get
    del poison
    y = grouped_linear(torch.ones(T, K, device=DEV, dtype=dt), w, torch.tensor([1, 2], device=DEV))
    assert not y[0].any() and not y[2].any() and not y[1, :-5].any() and (y[1, -5:] == K).all()


def test_launches_are_counted_as_they_happen():
    from flash_uma_b200 import _native as nat
    from flash_uma_b200.fp8 import Fp8Weight, fp8_linear
    from flash_uma_b200.grouped import grouped_linear, mix_experts

    def grouped(lens, dt):
        x, w, off, b, gy = _make(lens, 72, 40, dt, "shared")
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        return lambda: torch.autograd.grad(grouped_linear(x, w, off, b), leaves, gy)

    def mix(S, E, grads):
        c, x = torch.rand(S, E, device=DEV), torch.rand(E, 1000, device=DEV)
        leaves = [t.requires_grad_(True) for t, g in zip((c, x), grads) if g]
        return lambda: torch.autograd.grad(mix_experts(c, x), leaves, torch.ones(S, 1000, device=DEV))
    x, w8 = torch.rand(40, 136, device=DEV), Fp8Weight(torch.rand(72, 136, device=DEV))
    for f in (grouped([40, 3], torch.bfloat16), grouped([40, 3], torch.float32), grouped([2047, 9], torch.bfloat16),
              mix(5, 4, (1, 1)), mix(5, 4, (1, 0)), mix(5, 4, (0, 1)), mix(129, 4, (1, 1)), lambda: fp8_linear(x, w8)):
        f()
        torch.cuda.synchronize()
        probe = nat.LaunchProbe()
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
            nat.set_probe(probe)
            try:
                f()
            finally:
                nat.set_probe(None)
            torch.cuda.synchronize()
        assert probe.launches == sum("fuma::" in e.name for e in prof.events()), probe.counts
