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
def test_many_groups(dt):
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 9, (700,), generator=g).tolist()
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
