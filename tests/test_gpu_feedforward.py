"""The gated feed-forward block and its backward pass against the definition in 64 bits.

Each element is held to its own bound, from the rounding steps on its way: half a step of the
type (u) for the output and for the gated row / the gate adjoints that feed a product, and for an
fp32 sum of K products GAMMA(K) = (K + 16) 2^-23 of the sum of their magnitudes (every addition
may round toward zero; fp32 operands are carried to 2^-22 each)."""
import pytest
import torch

from tt_atom import _lib as L
from tt_atom.feedforward import gated_ff, gated_ff_bwd

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
# bounds of |act'| and |act''|: SiLU 1.0999 and 1/2, sigmoid 1/4 and 0.0963, GELU 1.1290 and
# sqrt(2 / pi) = 0.7979
SLOPES = {"silu": (1.1, 0.5), "sigmoid": (0.25, 0.097), "gelu": (1.13, 0.8)}


def gamma(k):
    return (k + 16) * 2.0 ** -23


def half_step(t):
    return 0.0 if t == torch.float32 else torch.finfo(t).eps / 2


def least(t):
    """What a rounding may be off by below the type's normal range."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def make(M, D, F, O, t, seed=0, spread=2.0):  # noqa: E741
    g = torch.Generator(device="cuda").manual_seed(seed)

    def n(*shape, s=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * s).to(t)
    return (n(M, D), n(F, D, s=spread / D ** 0.5), n(F, D, s=spread / D ** 0.5),
            n(O, F, s=1 / F ** 0.5), n(M, O))


def reference(x, wg, wu, wd, dy, act):
    """Every value in 64 bits and the bound of each output's error."""
    t = x.dtype
    u, lo, out_step = half_step(t), least(t), torch.finfo(t).eps / 2
    x, wg, wu, wd, dy = (v.double() for v in (x, wg, wu, wd, dy))
    (M, D), F, O = x.shape, wg.shape[0], wd.shape[0]  # noqa: E741
    g, up = x @ wg.T, x @ wu.T
    eg, eu = gamma(D) * (x.abs() @ wg.abs().T), gamma(D) * (x.abs() @ wu.abs().T)
    gg = g.clone().requires_grad_()
    a = {"silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid,
         "gelu": torch.nn.functional.gelu}[act](gg)
    (da,) = torch.autograd.grad(a.sum(), gg)
    a = a.detach()
    s1, s2 = SLOPES[act]
    few = 2.0 ** -20                    # the activation's own arithmetic, a few steps of fp32
    h = a * up
    # |a| <= s1 |g| + 1/2 bounds what the exponential's rounding leaves of it in absolute terms
    eh = s1 * eg * up.abs() + (a.abs() + s1 * eg) * eu + few * (g.abs() + 1) * up.abs() \
        + u * h.abs() + lo
    y = h @ wd.T
    dh = dy @ wd
    edh = gamma(O) * (dy.abs() @ wd.abs())
    edu = edh * (a.abs() + s1 * eg) + dh.abs() * (s1 * eg + few * (g.abs() + 1))
    ada = da.abs() + s2 * eg + few * (g.abs() + 1) ** 2
    edg = edh * (up.abs() + eu) * ada + dh.abs() * eu * ada \
        + (dh * up).abs() * (s2 * eg + few * (g.abs() + 1) ** 2)
    dg, du = dh * up * da, dh * a
    edg, edu = edg + u * dg.abs() + lo, edu + u * du.abs() + lo

    def both(A, eA, B, eB=None):
        """A @ B and the bound of its error."""
        e = eA @ B.abs() + gamma(A.shape[1]) * ((A.abs() + eA) @ B.abs())
        if eB is not None:
            e = e + (A.abs() + eA) @ eB
        return A @ B, e
    z = torch.zeros_like
    vy = both(h, eh, wd.T)
    v1, v2 = both(dg, edg, wg), both(du, edu, wu)
    out = {"y": (y, vy[1]), "dx": (v1[0] + v2[0], (v1[1] + v2[1]) * 2),
           "dwg": both(dg.T, edg.T, x), "dwu": both(du.T, edu.T, x),
           "dwd": both(dy.T, z(dy.T), h, eh)}
    return {k: (v, e * 1.01 + (out_step * 1.01) * v.abs() + lo + 1e-30) for k, (v, e) in out.items()}


def check(got, want, names):
    for name, v in zip(names, got):
        ref, bound = want[name]
        assert v.shape == ref.shape
        off = (v.double() - ref).abs()
        assert torch.isfinite(v).all(), name
        bad = off > bound
        assert not bad.any(), (name, int(bad.sum()), float((off / bound).max()))


SIZES = [(1, 64, 128, 64), (3, 33, 70, 45), (8, 256, 512, 256), (17, 128, 64, 128),
         (33, 1, 1, 1), (130, 40, 264, 24), (257, 512, 384, 136), (300, 129, 1000, 65),
         (1000, 256, 1024, 256), (2100, 64, 136, 200)]


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_against_the_definition(size, t):
    M = size[0]
    act = ("silu", "sigmoid", "gelu")[M % 3]
    x, wg, wu, wd, dy = make(*size, t)
    want = reference(x, wg, wu, wd, dy, act)
    names = ("dx", "dwg", "dwu", "dwd")
    y, kept = gated_ff(x, wg, wu, wd, act=act, keep=True)
    check([y], want, ["y"])
    assert torch.equal(y, gated_ff(x, wg, wu, wd, act=act))
    check(gated_ff_bwd(x, wg, wu, wd, dy, act=act, kept=kept), want, names)
    grads = gated_ff_bwd(x, wg, wu, wd, dy, act=act)
    check(grads, want, names)
    alone = gated_ff_bwd(x, wg, wu, wd, dy, act=act, weight_grads=False)
    assert alone[1:] == (None, None, None) and torch.equal(alone[0], grads[0])


@pytest.mark.parametrize("act", ["silu", "sigmoid", "gelu"])
def test_activations_over_their_range(act):
    # gates from -30 to 30: the tails, where a SiLU or GELU derivative is all but lost
    x = torch.linspace(-30, 30, 513, device="cuda")[:, None] * torch.tensor([[1.0, 0.0]], device="cuda")
    x[:, 1] = 1.0
    wg = torch.tensor([[1.0, 0.0]], device="cuda")
    wu = torch.tensor([[0.0, 1.0]], device="cuda")
    wd = torch.ones(1, 1, device="cuda")
    dy = torch.ones(513, 1, device="cuda")
    want = reference(x, wg, wu, wd, dy, act)
    check([gated_ff(x, wg, wu, wd, act=act)], want, ["y"])
    check(gated_ff_bwd(x, wg, wu, wd, dy, act=act), want, ("dx", "dwg", "dwu", "dwd"))


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_gradient_against_differences(t):
    # along one direction of the rows, in 64 bits: (f(x + s v) - f(x - s v)) / 2 s
    x, wg, wu, wd, dy = make(40, 48, 72, 56, t, seed=3)
    dx = gated_ff_bwd(x, wg, wu, wd, dy)[0].double()
    v = torch.randn(x.shape, dtype=torch.double, device="cuda")

    def f(z):
        g, u = z @ wg.double().T, z @ wu.double().T
        return ((torch.nn.functional.silu(g) * u) @ wd.double().T * dy.double()).sum()
    step = 1e-5
    slope = (f(x.double() + step * v) - f(x.double() - step * v)) / (2 * step)
    bound = (reference(x, wg, wu, wd, dy, "silu")["dx"][1] * v.abs()).sum()
    assert abs(float((dx * v).sum() - slope)) <= float(bound) + 1e-6 * abs(float(slope))


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_row_strides_and_what_lies_between_the_rows(t):
    M, D, F, O = 150, 72, 136, 40  # noqa: E741
    x, wg, wu, wd, dy = make(M, D, F, O, t, seed=1)
    for pad in (3, 8):
        wide_x = torch.full((M, D + pad), float("nan"), dtype=t, device="cuda")
        wide_dy = torch.full((M, O + pad), float("nan"), dtype=t, device="cuda")
        xs, dys = wide_x[:, 1:D + 1] if pad == 3 else wide_x[:, :D], wide_dy[:, :O]
        xs.copy_(x)
        dys.copy_(dy)
        assert torch.equal(gated_ff(xs, wg, wu, wd), gated_ff(x, wg, wu, wd))
        for a, b in zip(gated_ff_bwd(xs, wg, wu, wd, dys), gated_ff_bwd(x, wg, wu, wd, dy)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("M", [5, 200])
def test_outputs_with_a_leading_dimension_through_the_c_interface(M):
    D, F, O, t = 64, 96, 24, torch.bfloat16  # noqa: E741
    x, wg, wu, wd, dy = make(M, D, F, O, t, seed=2)
    n = (L.c_size_t * 3)()
    L.call("atom_gated_ff_bytes", 1, M, D, F, O, n)
    ws = torch.empty(max(n[0], n[1]), dtype=torch.uint8, device="cuda")
    y = torch.full((M + 2, O + 5), 7.0, dtype=t, device="cuda")
    dx = torch.full((M + 2, D + 3), 7.0, dtype=t, device="cuda")
    L.call("atom_gated_ff_fwd", 1, x.data_ptr(), D, M, D, F, O, wg.data_ptr(), wu.data_ptr(),
           wd.data_ptr(), 0, y.data_ptr(), O + 5, None, ws.data_ptr(), n[0], L.stream_ptr())
    L.call("atom_gated_ff_bwd", 1, x.data_ptr(), D, M, D, F, O, wg.data_ptr(), wu.data_ptr(),
           wd.data_ptr(), 0, dy.data_ptr(), O, None, dx.data_ptr(), D + 3, None, None, None,
           ws.data_ptr(), n[1], L.stream_ptr())
    assert torch.equal(y[:M, :O], gated_ff(x, wg, wu, wd))
    assert torch.equal(dx[:M, :D], gated_ff_bwd(x, wg, wu, wd, dy, weight_grads=False)[0])
    assert (y[M:] == 7).all() and (y[:, O:] == 7).all()
    assert (dx[M:] == 7).all() and (dx[:, D:] == 7).all()


def test_no_rows():
    x, wg, wu, wd, dy = make(0, 32, 64, 32, torch.bfloat16)
    y, kept = gated_ff(x, wg, wu, wd, keep=True)
    assert y.shape == (0, 32)
    dx, *dw = gated_ff_bwd(x, wg, wu, wd, dy, kept=kept)
    assert dx.shape == (0, 32) and all((w == 0).all() for w in dw)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M", [4, 300])
def test_a_row_that_is_not_finite_stays_alone(M, t):
    x, wg, wu, wd, dy = make(M, 96, 160, 80, t, seed=5)
    y, dx = gated_ff(x, wg, wu, wd), gated_ff_bwd(x, wg, wu, wd, dy)[0]
    for value in (float("nan"), float("inf")):
        bad = x.clone()
        bad[1, 3] = value
        yb, dxb = gated_ff(bad, wg, wu, wd), gated_ff_bwd(bad, wg, wu, wd, dy, weight_grads=False)[0]
        keep = [i for i in range(M) if i != 1]
        assert torch.equal(yb[keep], y[keep]) and torch.equal(dxb[keep], dx[keep])
        assert not torch.isfinite(yb[1]).all()


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_rows_do_not_depend_on_their_neighbours_size(t):
    # one row many times larger than the others leaves their accuracy as it is (in fp16 the large
    # row itself is out of range: its gated values are some 100^2 g u, and g and u pass 3)
    x, wg, wu, wd, dy = make(70, 64, 128, 64, t, seed=6)
    big = x.clone()
    big[0] *= 100
    first = 1 if t == torch.float16 else 0
    want = reference(big[first:], wg, wu, wd, dy[first:], "silu")
    check([gated_ff(big, wg, wu, wd)[first:]], want, ["y"])
    if t == torch.float32:
        big[0] *= 1e15
        want = reference(big[1:], wg, wu, wd, dy[1:], "silu")
        check([gated_ff(big, wg, wu, wd)[1:]], want, ["y"])
        check([gated_ff_bwd(big, wg, wu, wd, dy, weight_grads=False)[0][1:]], want, ["dx"])


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_other_streams_and_repeats(t):
    args = [make(500, 128, 256, 128, t, seed=s) for s in (7, 8)]
    want = [(gated_ff(*a[:4]), *gated_ff_bwd(*a)) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = [[], []]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append((gated_ff(*args[k][:4]), *gated_ff_bwd(*args[k])))
    torch.cuda.synchronize()
    for k in range(2):
        for r in got[k]:
            assert all(torch.equal(p, q) for p, q in zip(r, want[k]))


@pytest.mark.parametrize("M", [2, 400])
def test_captured_and_replayed(M):
    x, wg, wu, wd, dy = make(M, 128, 256, 128, torch.bfloat16, seed=9)
    gated_ff(x, wg, wu, wd)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):       # two graphs at a time, each with its own workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y, kept = gated_ff(x, wg, wu, wd, keep=True)
            outs.append((y, *gated_ff_bwd(x, wg, wu, wd, dy, kept=kept)))
        graphs.append(g)
    x.copy_(make(M, 128, 256, 128, torch.bfloat16, seed=10)[0])
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    y, kept = gated_ff(x, wg, wu, wd, keep=True)
    want = (y, *gated_ff_bwd(x, wg, wu, wd, dy, kept=kept))
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(o, want))


def test_wide_and_long():
    # more rows than one pass of the GPU's blocks, a width of several tiles, both odd
    x, wg, wu, wd, dy = make(20011, 136, 264, 72, torch.bfloat16, seed=11)
    want = reference(x, wg, wu, wd, dy, "silu")
    check([gated_ff(x, wg, wu, wd)], want, ["y"])
    check(gated_ff_bwd(x, wg, wu, wd, dy), want, ("dx", "dwg", "dwu", "dwd"))
    x, wg, wu, wd, dy = make(70, 2056, 4104, 1032, torch.bfloat16, seed=12)
    want = reference(x, wg, wu, wd, dy, "silu")
    check([gated_ff(x, wg, wu, wd)], want, ["y"])
    check(gated_ff_bwd(x, wg, wu, wd, dy), want, ("dx", "dwg", "dwu", "dwd"))


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M, D, F, O", [(1, 7, 9, 300), (2, 1000, 33, 5), (9, 65, 700, 136),
                                        (16, 264, 130, 1), (13, 40, 2000, 24), (17, 264, 130, 8)])
def test_few_rows_both_ways(M, D, F, O, t):  # noqa: E741
    test_against_the_definition((M, D, F, O), t)


@pytest.mark.parametrize("act", ["silu", "sigmoid", "gelu"])
def test_fp32_rows_far_below_their_bound(act):
    """fp32 rows of H and of dG | dU are two 16-bit planes scaled by a bound of the row, below
    (8 D max|x| max|w|) for g and u (each factor rounded up to a power of two): a plane's last
    place is 2^-36 where the bound is 2^15, so a value is off by at most 2^-51 of it. Outliers in x
    and in rows of the weights, and gates that are closed, bring rows far below it."""
    M, D, F, O = 40, 512, 264, 64  # noqa: E741
    x, wg, wu, wd, dy = make(M, D, F, O, torch.float32, seed=31)
    x[:, 5] *= 300
    x[::4] *= 2.0 ** -20
    wg[3], wu[7] = wg[3] * 50, wu[7] * 50
    wg[:, 5] = 0.02 * wg[:, 5].sign() - 0.01
    dy[::3, 1] *= 100
    want = reference(x, wg, wu, wd, dy, act)
    X, WG, WU, WD, DY = (v.double() for v in (x, wg, wu, wd, dy))
    top = torch.maximum(WG.abs().max(), WU.abs().max())
    g = 8 * D * X.abs().amax(1, keepdim=True) * top
    dh = 8 * O * DY.abs().amax(1, keepdim=True) * WD.abs().max()
    one = torch.ones_like(g)
    eh = (2.0 ** -51 * (g if act == "sigmoid" else g * g)).expand(M, F)
    eg = (2.0 ** -51 * dh * (torch.maximum(g, one) if act == "sigmoid" else 2 * g)).expand(M, F)
    wx = 2.0 ** -51 * M * (eg[:, :1] * 2.0 ** 51 * 2 * X.abs().amax(1, keepdim=True)).max()
    wy = 2.0 ** -51 * M * (eh[:, :1] * 2.0 ** 51 * 2 * DY.abs().amax(1, keepdim=True)).max()
    more = {"y": eh @ WD.abs().T, "dx": eg @ (WG.abs() + WU.abs()), "dwg": eg.T @ X.abs() + wx,
            "dwu": eg.T @ X.abs() + wx, "dwd": DY.abs().T @ eh + wy}
    want = {k: (v, e + 1.01 * more[k]) for k, (v, e) in want.items()}
    check([gated_ff(x, wg, wu, wd, act=act)], want, ["y"])
    y, kept = gated_ff(x, wg, wu, wd, act=act, keep=True)
    for k in (None, kept):
        check(gated_ff_bwd(x, wg, wu, wd, dy, act=act, kept=k), want, ("dx", "dwg", "dwu", "dwd"))
