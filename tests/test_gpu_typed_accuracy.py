"""Where the typed operators could lose what the definition keeps, with 16 rows and with more (which
other kernels take)."""
import pytest
import torch

import test_gpu_adapters as ad
import test_gpu_feedforward as ff
from tt_atom import _lib as L
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
@pytest.mark.parametrize("t", [torch.bfloat16], ids=str)
def test_sigmoid_gates_that_are_closed(t, M):
    # sigmoid(-50) = 2e-22. A product's error in g, gamma(D) of its terms' magnitudes (64 at most),
    # is a relative error of the sigmoid; beside it half steps of the type for h and y, both ways
    args = closed_gates(M, 32, 64, 24, t, -50.0)
    y = gated_ff(*args[:4], act="sigmoid")
    bound = 64 * ff.gamma(32) + 3 * torch.finfo(t).eps
    assert off(y, exact(*args, "sigmoid")["y"])[0] <= bound


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
