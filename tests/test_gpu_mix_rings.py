"""Large expert mixes against fp64: 8 tiles and more for every thread block, so that each ring of the tensor-core kernel (operand
stages, raw tiles, accumulators, tile scales, the drain of dc) goes round, at each depth that the shapes come to. The
columns' magnitudes change from tile to tile, so that values or a scale of another tile show.

Bounds, in units of 2^-24 of S = the sum of |products|: the tensor core truncates (2) up to three additions per 16
products; two fp16 planes on each side leave 12 (fp32); a rounded addition is 1. Then half an eps of the result's type.
dc: 16 steps of 16 columns stay in the tensor core's sum, one addition per such sum and thread block, a few in fp64."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ALIGNED, ODD = 160000, 160003


def _check(got, want, S, steps, what):
    t = got.dtype
    tol = torch.finfo(t).eps / 2 * want.abs() + steps * 2.0 ** -24 * S + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[0].tolist())


def _compare(S, E, P, dt):
    from flash_uma_b200 import linear
    from flash_uma_b200.grouped import mix_experts
    g = torch.Generator(device=DEV).manual_seed(S * 1000 + E)
    tile = 64 if dt == torch.float32 else 128
    steps_of = 12 if dt == torch.float32 else 0
    n_tiles = -(-P // tile)

    def matrices(n):
        mag = 2.0 ** torch.randint(-6, 7, (n_tiles,), device=DEV, generator=g)
        return (torch.randn(n, P, device=DEV, generator=g) * mag.repeat_interleave(tile)[:P]).to(dt)
    c = torch.randn(S, E, device=DEV, generator=g).requires_grad_(True)
    x, gw = matrices(E).requires_grad_(True), matrices(S)

    def run():
        w = mix_experts(c, x)
        return (w.detach(), *torch.autograd.grad(w, [c, x], gw))
    w, dc, dx = run()
    linear.check_errors()
    C, X, GW = c.detach().double(), x.detach().double(), gw.double()
    _check(w, C @ X, C.abs() @ X.abs(), 6 * -(-E // 16) + steps_of + 2, "w")
    _check(dx, C.T @ GW, C.T.abs() @ GW.abs(), 6 * -(-S // 16) + steps_of + 2, "dx")
    sms = torch.cuda.get_device_properties(DEV).multi_processor_count
    _check(dc, GW @ X.T, GW.abs() @ X.abs().T, 6 * 16 + -(-n_tiles // sms) + steps_of + 4, "dc")
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(run(), (w, dc, dx)))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("S,E,P", [(64, 32, ALIGNED), (64, 32, ODD), (70, 70, ALIGNED), (70, 70, ODD), (128, 64, ALIGNED),
                                   (128, 64, ODD), (112, 97, ODD), (128, 128, ODD)])
def test_stages_of_the_operand_ring(S, E, P, dt):
    """One to four operand stages, filled by two warpgroups in turn."""
    _compare(S, E, P, dt)


@pytest.mark.parametrize("S,E", [(128, 80), (100, 96), (128, 96), (112, 97), (128, 128)])
@pytest.mark.parametrize("dt", DTYPES)
def test_one_raw_tile(S, E, dt):
    """Shapes at which fp32 has room for one raw tile beside one operand stage."""
    _compare(S, E, ALIGNED, dt)


@pytest.mark.parametrize("both", [True, False])
def test_long_sums_of_one_sign(both):
    """dc over 3 * 2^23 columns. Every product is a little more than 1, by an amount that an fp32 sum of a thread's whole share would
    drop at each addition once it is large (460 and 3,600 units, by where the share ends). fp32 sums end after 4,096 columns: 64
    sums of 64 columns from the tensor core (24 units inside each, 12 for the planes), or 1,024 sums of 4."""
    from flash_uma_b200.grouped import mix_experts
    P = 3 * 2 ** 23
    step = 2.0 ** -13 if both else 2.0 ** -10
    x = torch.full((1, P), 1.0 + step * (1.0 - 2.0 ** -6), device=DEV).requires_grad_(both)
    c = torch.ones(1, 1, device=DEV, requires_grad=True)
    dc = torch.autograd.grad(mix_experts(c, x), [c, x] if both else [c], torch.ones(1, P, device=DEV))[0]
    want = float(x.detach()[0, 0].double()) * P
    steps = 64 + 24 + 12 + 4 if both else 1024 + 4 + 2
    assert abs(float(dc) - want) <= steps * 2.0 ** -24 * want


@pytest.mark.parametrize("up,down", [(120, -100), (-100, 120)])
def test_coefficients_and_matrices_at_the_ends_of_the_fp32_range(up, down):
    """Coefficients about 2^up and matrices about 2^down: results about 2^20."""
    from flash_uma_b200.grouped import mix_experts
    S, E, P = 64, 32, 1000
    g = torch.Generator(device=DEV).manual_seed(3)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g)   # noqa: E731
    c = (r(S, E) * 2.0 ** up).requires_grad_(True)
    x, gw = (r(E, P) * 2.0 ** down).requires_grad_(True), r(S, P) * 2.0 ** down
    w = mix_experts(c, x)
    dx, = torch.autograd.grad(w, [x], gw, retain_graph=True)
    both = torch.autograd.grad(w, [c, x], gw)[1]
    C, X, GW = c.detach().double(), x.detach().double(), gw.double()
    _check(w.detach(), C @ X, C.abs() @ X.abs(), 6 * 2 + 14, "w")
    for got in (dx, both):
        _check(got, C.T @ GW, C.T.abs() @ GW.abs(), 6 * 4 + 14, "dx")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("S,E,P", [(160, 96, 20000), (96, 160, 20003), (130, 129, 9000)])
def test_more_than_128_systems_or_experts(S, E, P, dt):
    """The vector kernels, in several rounds over systems and experts: n rounded additions for a contraction of n, for dc 1,024 of 4
    products (5 units each way) before fp64."""
    from flash_uma_b200.grouped import mix_experts
    g = torch.Generator(device=DEV).manual_seed(5)
    c = torch.randn(S, E, device=DEV, generator=g).requires_grad_(True)
    x = torch.randn(E, P, device=DEV, generator=g).to(dt).requires_grad_(True)
    gw = torch.randn(S, P, device=DEV, generator=g).to(dt)
    w = mix_experts(c, x)
    dc, dx = torch.autograd.grad(w, [c, x], gw, retain_graph=True)
    C, X, GW = c.detach().double(), x.detach().double(), gw.double()
    planes = 12 if dt == torch.float32 else 0   # the forward may take the tensor cores
    _check(w.detach(), C @ X, C.abs() @ X.abs(), max(E, 6 * -(-E // 16) + planes) + 2, "w")
    _check(dx, C.T @ GW, C.T.abs() @ GW.abs(), max(S, 6 * -(-S // 16) + planes) + 2, "dx")
    _check(dc, GW @ X.T, GW.abs() @ X.abs().T, 1024 + 8, "dc")
    assert torch.equal(torch.autograd.grad(w, [c], gw, retain_graph=True)[0], dc)
    assert torch.equal(torch.autograd.grad(w, [x], gw)[0], dx)


def test_systems_and_experts_of_unlike_magnitudes():
    """fp32, systems and experts 2^-20 to 2^20 apart. A scale for a row of coefficients, and one for 64 columns of all matrices,
    brings the largest magnitude M below 2^15, where a second plane's rounding is 2^-25: 2^-39 M (2^-40 of the largest at its
    least, half a unit more for the division's power of two), or 2^-22 of the value. So each product may be off by
    2^-39 (M_c |x| + |c| M_x) beside the planes' 12 2^-24 |c x|."""
    from flash_uma_b200.grouped import mix_experts
    S, E, P = 70, 40, 3000
    g = torch.Generator(device=DEV).manual_seed(11)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g)   # noqa: E731
    mag = lambda n: 2.0 ** torch.randint(-20, 21, (n, 1), device=DEV, generator=g)   # noqa: E731
    c = (r(S, E) * mag(S) * mag(E).T).requires_grad_(True)
    x, gw = (r(E, P) * mag(E)).requires_grad_(True), r(S, P) * mag(S)
    w = mix_experts(c, x)
    dc, dx = torch.autograd.grad(w, [c, x], gw)
    C, X, GW = c.detach().double(), x.detach().double(), gw.double()

    def check(got, A, B, Ma, Mb, steps, what):
        """got = A @ B; Ma, Mb: the magnitudes that the rows' scales of A and the columns' of B go by, broadcast."""
        S_ = A.abs() @ B.abs()
        extra = Ma * B.abs().sum(0)[None] + A.abs().sum(1)[:, None] * Mb
        tol = steps * 2.0 ** -24 * S_ + 2.0 ** -39 * extra + 2.0 ** -24 * (A @ B).abs()
        assert ((got.double() - A @ B).abs() <= tol).all(), what
    check(w.detach(), C, X, C.abs().amax(1, keepdim=True), X.abs().max(), 6 * 3 + 14, "w")
    check(dx, C.T, GW, C.abs().amax(0)[:, None], GW.abs().max(), 6 * 5 + 14, "dx")
    check(dc, GW, X.T, GW.abs().max(), X.abs().max(), 6 * 4 + 1 + 16, "dc")


@pytest.mark.parametrize("dt", DTYPES)
def test_large_mixes_on_two_streams_and_replayed(dt):
    """Two mixes of several tiles a thread block in flight at once, and a captured one on new data, give the eager calls' bits."""
    from flash_uma_b200.grouped import mix_experts
    g = torch.Generator(device=DEV).manual_seed(13)

    def make(S, E, P):
        c = torch.rand(S, E, device=DEV, generator=g).requires_grad_(True)
        x = torch.randn(E, P, device=DEV, generator=g).to(dt).requires_grad_(True)
        gw = torch.randn(S, P, device=DEV, generator=g).to(dt)

        def run():
            w = mix_experts(c, x)
            return (w.detach(), *torch.autograd.grad(w, [c, x], gw))
        return run, x
    (a, xa), (b, _) = make(70, 70, ALIGNED), make(128, 96, ODD)
    want = a(), b()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            got_b = b()
        got_a = a()
        torch.cuda.current_stream().wait_stream(side)
        for got, w in ((got_a, want[0]), (got_b, want[1])):
            assert all(torch.equal(p, q) for p, q in zip(got, w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = a()
    with torch.no_grad():
        xa.mul_(-3.0)
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(out, a()))
