"""Where the typed operators could lose what the definition keeps: a NaN in a gate's weights, gates
that are closed or open, fp32 values far below others of their row, weight or call, and the same
call with 16 rows and with more (which other kernels take)."""
import pytest
import torch

import test_gpu_adapters as ad
import test_gpu_feedforward as ff
from tt_atom import _lib as L
from tt_atom.adapters import adapted_linear, adapted_linear_bwd
from tt_atom.feedforward import gated_ff, gated_ff_bwd

pytestmark = pytest.mark.gpu

ACTS = ["silu", "sigmoid", "gelu"]


def closed_gates(M, D, F, O, t, level, seed=0):  # noqa: E741
    """A block whose gates all lie around ``level``, through a constant feature of the rows."""
    x, wg, wu, wd, dy = ff.make(M, D, F, O, t, seed=seed, spread=0.25)
    x[:, 0] = 1
    wg[:, 0] = level
    return x, wg, wu, wd, dy


def derivatives(g, act):
    """act and act' in 64 bits, their tails from functions of the tail."""
    if act == "gelu":
        phi = torch.special.erfc(-g * 0.5 ** 0.5) / 2
        return g * phi, phi + g * torch.exp(-g * g / 2) / (2 * torch.pi) ** 0.5
    s, r = torch.sigmoid(g), torch.sigmoid(-g)
    return (s, s * r) if act == "sigmoid" else (g * s, s * (1 + g * r))


def exact(x, wg, wu, wd, dy, act, dtype=torch.double):
    """Everything in 64 bits, or (dtype float32) the plain form in separate steps."""
    x, wg, wu, wd, dy = (v.to(dtype) for v in (x, wg, wu, wd, dy))
    g, u = x @ wg.T, x @ wu.T
    a, da = derivatives(g, act)
    h, dh = a * u, dy @ wd
    dg, du = dh * u * da, dh * a
    return {"y": h @ wd.T, "dx": dg @ wg + du @ wu, "dwg": dg.T @ x, "dwu": du.T @ x, "dwd": dy.T @ h}


def run(x, wg, wu, wd, dy, act):
    """The block's outputs with what its forward pass kept and without."""
    y, kept = gated_ff(x, wg, wu, wd, act=act, keep=True)
    for k in (kept, None):
        yield dict(zip(("y", "dx", "dwg", "dwu", "dwd"),
                       (y, *gated_ff_bwd(x, wg, wu, wd, dy, act=act, kept=k))))


def off(got, want):
    """Relative 2-norm of the difference, whole and of the worst row."""
    d, w = (got.double() - want).norm(dim=1), want.norm(dim=1)
    return float(d.norm() / w.norm()), float((d / w.clamp_min(1e-300)).max())


@pytest.mark.parametrize("t", ff.TYPES, ids=str)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [4, 16, 17, 300])
def test_nan_in_a_gates_weights(M, act, t):
    # row 3 of Wg makes column 3 of g NaN: y and dx, sums over the columns, are NaN as a whole, and
    # of the weights' gradients what belongs to the column
    x, wg, wu, wd, dy = ff.make(M, 48, 72, 40, t, seed=1)
    good = list(run(x, wg, wu, wd, dy, act))
    wg[3, 2] = float("nan")
    for got, was in zip(run(x, wg, wu, wd, dy, act), good):
        for name in ("y", "dx"):
            assert got[name].isnan().all(), name
        for name in ("dwg", "dwu", "dwd"):
            a, b = (v[name].T if name == "dwd" else v[name] for v in (got, was))
            rest = [i for i in range(72) if i != 3]
            assert a[3].isnan().all() and torch.equal(a[rest], b[rest]), name


@pytest.mark.parametrize("M", [16, 40])
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float32], ids=str)
def test_sigmoid_gates_that_are_closed(t, M):
    # sigmoid(-50) = 2e-22. A product's error in g, gamma(D) of its terms' magnitudes (64 at most),
    # is a relative error of the sigmoid; beside it half steps of the type for h and y, both ways
    args = closed_gates(M, 32, 64, 24, t, -50.0)
    y = gated_ff(*args[:4], act="sigmoid")
    bound = 64 * ff.gamma(32) + 3 * torch.finfo(t).eps
    assert off(y, exact(*args, "sigmoid")["y"])[0] <= bound


@pytest.mark.parametrize("M", [5, 40])
def test_sigmoid_gates_that_are_open(M):
    # sigmoid'(14) = 8e-7 = s (1 - s), where 1 - s has no more than 4 bits left in fp32 once s is
    # rounded; dwg is proportional to it. Bound as above, with the terms' magnitudes below 20.
    args = closed_gates(M, 32, 64, 24, torch.float32, 14.0)
    want = exact(*args, "sigmoid")["dwg"]
    for got in run(*args, "sigmoid"):
        assert off(got["dwg"], want)[0] <= 20 * ff.gamma(32) + 2.0 ** -20


@pytest.mark.parametrize("M", [5, 40])
@pytest.mark.parametrize("level", [-3.0, -6.0, -9.0])
def test_gelu_gates_that_are_closed(level, M):
    # a Gaussian's tail: an error e in g is one of |g| e in it (1 + g^2 / 2 steps of fp32 for the
    # exponential's own argument), |g| below 1.5 |level| and its terms' magnitudes below 2 |level|
    args = closed_gates(M, 32, 64, 24, torch.float32, level)
    want = exact(*args, "gelu")
    top = 1.5 * abs(level)
    bound = (top + 1) * 2 * abs(level) * ff.gamma(32) + (4 + top * top) * 2.0 ** -23
    for got in run(*args, "gelu"):
        for name in ("y", "dwu", "dwd"):
            assert off(got[name], want[name])[0] <= bound, name


def outliers(kind, M, D, F, O):  # noqa: E741
    x, wg, wu, wd, dy = ff.make(M, D, F, O, torch.float32, seed=4)
    if kind == "a weight of 16":
        wg[5, 7] = 16
    elif kind == "a weight of 100 and a feature of 100":
        wg[5, 7] = 100
        x[:, 9] *= 100
    elif kind == "a feature of 1,000 with small weights":
        x[:, 9] *= 1000
        wg[:, 9] /= 1000
        wu[:, 9] /= 1000
    elif kind == "a constant feature without weights":
        x[:, 9] = 1e4
        wg[:, 9] = wu[:, 9] = 0
    elif kind == "closed gates":
        x[:, 9] = 1
        wg[:, 9] = -12
    elif kind == "a large row":
        x[1] *= 1e5
        dy[1] = 0
    elif kind == "a large weight beside small ones":
        wd[0, 0] = 1e6
        dy[:, 0] = 0
    return x, wg, wu, wd, dy


@pytest.mark.parametrize("kind", [
    "a weight of 16", "a weight of 100 and a feature of 100", "a feature of 1,000 with small weights",
    "a constant feature without weights", "closed gates", "a large row",
    "a large weight beside small ones"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [16, 17, 130])
def test_fp32_keeps_fp32s_accuracy_beside_outliers(M, act, kind):
    """Every output keeps its bound of fp32, element by element, and is as a whole (y and dx, whose rows
    sum over all gates, also in the worst row; a row of dwg may hang on one gate, and is then as far
    off as chance has it) at most twice as far off as the same formulas in fp32 steps: an addition
    here may be off by a whole step (the tensor core's, toward zero) where those are off by half.
    Beside it what the activation's own arithmetic may add, 8 + g^2 steps (|g| <= 20 where a gate is
    neither 0 nor 1 nor the value itself)."""
    args = outliers(kind, M, 1024, 264, 72)
    bounds = ff.reference(*args, act)
    want, plain = exact(*args, act), exact(*args, act, torch.float32)
    g = float((args[0] @ args[1].T).abs().max().clamp_max(20))
    own = (8 + g * g) * 2.0 ** -23
    for got in run(*args, act):
        ff.check(got.values(), bounds, got)
        for name, v in got.items():
            a, b = off(v, want[name]), off(plain[name], want[name])
            assert a[0] <= 2 * b[0] + own, (name, a, b)
            assert name[:2] == "dw" or a[1] <= 2 * b[1] + own, (name, a, b)


@pytest.mark.parametrize("size", [1e3, 1e9, 1e15])
@pytest.mark.parametrize("R", [8, 72])
@pytest.mark.parametrize("rows", [3, 70])
def test_an_adapters_size_stays_with_its_requests(rows, R, size):
    # fp32: one adapter many times larger than the others; the other requests keep their bounds
    args = ad.make([rows] * 3, [0, 1, 2], 3, R, 64, 96, torch.float32, seed=5)
    x, w, a, b, scale, ptr, ids, dy = args
    a[1] *= size
    b[1] *= size
    want = ad.reference(*args)
    rest = [i for i in range(3 * rows) if not rows <= i < 2 * rows]
    y, kept = adapted_linear(*args[:7], keep=True)
    ad.check([y[rest]], {"y": [v[rest] for v in want["y"]]}, ["y"])
    want = {k: [v[rest if k == "dx" else [0, 2]] for v in want[k]] for k in ("dx", "da", "db")}
    for k in (kept, None):
        dx, da, db = adapted_linear_bwd(*args, kept=k)
        ad.check([dx[rest], da[[0, 2]], db[[0, 2]]], want, ("dx", "da", "db"))


def test_a_row_without_an_adapter_beside_large_ones_and_an_old_workspace():
    # fp32, the workspace full of 3.4e38, adapters of 2^16: nothing of either reaches a row that has
    # no adapter
    M, D, O, R = 40, 64, 96, 8  # noqa: E741
    x, w, a, b, scale, ptr, ids, dy = ad.make([15, 10], [0, -1], 2, R, D, O, torch.float32, seed=6,
                                              tail=15)
    b *= 2.0 ** 16
    n = (L.c_size_t * 3)()
    L.call("atom_adapted_linear_bytes", 0, M, D, O, 2, R, 2, n)
    ws = torch.full((n[0],), 0x7F, dtype=torch.uint8, device="cuda")
    y = torch.empty(M, O, device="cuda")
    L.call("atom_adapted_linear_fwd", 0, x.data_ptr(), D, M, D, O, w.data_ptr(), a.data_ptr(),
           b.data_ptr(), scale.data_ptr(), 2, R, ptr.data_ptr(), ids.data_ptr(), 2, y.data_ptr(), O,
           None, ws.data_ptr(), n[0], L.stream_ptr())
    want = ad.reference(x, w, a, b, scale, ptr, ids, dy)
    ad.check([y[15:]], {"y": [v[15:] for v in want["y"]]}, ["y"])


def test_fp32_captured_and_replayed():
    # two graphs at a time, each with its own workspace, on rows that change under them
    a, b = ff.make(400, 128, 256, 128, torch.float32, seed=9), ff.make(400, 128, 256, 128, torch.float32, seed=8)
    p = ad.make([90] * 4, [0, 1, 2, -1], 3, 72, 128, 64, torch.float32, seed=7)

    def everything():
        y, kept = gated_ff(*a[:4], keep=True)
        z, kept2 = adapted_linear(*p[:7], keep=True)
        return (y, *gated_ff_bwd(*a, kept=kept), z, *adapted_linear_bwd(*p, kept=kept2))
    everything()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(everything())
        graphs.append(g)
    a[0].copy_(b[0])
    p[6].copy_(torch.tensor([2, 2, -1, 0], dtype=torch.int32))
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    want = everything()
    for o in outs:
        assert all(torch.equal(u, v) for u, v in zip(o, want))


def test_fp32_offsets_past_32_bits():
    # 2.2e9 values of H: the last rows against the definition of those rows alone
    M, D, F, O, last = 540_000, 64, 4104, 32, 300  # noqa: E741
    x, wg, wu, wd, dy = ff.make(M, D, F, O, torch.float32, seed=5)
    want = ff.reference(x[-last:], wg, wu, wd, dy[-last:], "silu")
    ff.check([gated_ff(x, wg, wu, wd)[-last:]], want, ["y"])
    dx = gated_ff_bwd(x, wg, wu, wd, dy, weight_grads=False)[0]
    ff.check([dx[-last:]], want, ["dx"])
