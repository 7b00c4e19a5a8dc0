"""Low-rank adapters of many requests beside a shared projection, and their backward pass,
against the definition in 64 bits (the bounds are built as in test_gpu_feedforward.py: half a
step of the type for an output and for the low-rank row that feeds a product, (K + 16) 2^-23 of
the summed magnitudes for an fp32 sum of K products)."""
import pytest
import torch

from test_gpu_feedforward import TYPES, gamma, half_step, least
from tt_atom.adapters import adapted_linear, adapted_linear_bwd
from tt_atom.feedforward import gated_ff, gated_ff_bwd

pytestmark = pytest.mark.gpu


def make(lengths, ids, n, R, D, O, t, seed=0, tail=0, head=0):  # noqa: E741
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*shape, s=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * s).to(t)
    ptr = [head]
    for k in lengths:
        ptr.append(ptr[-1] + k)
    M = ptr[-1] + tail
    i32 = dict(dtype=torch.int32, device="cuda")
    return (r(M, D), r(O, D, s=D ** -0.5), r(n, R, D, s=D ** -0.5), r(n, O, R, s=R ** -0.5),
            torch.rand(n, generator=g, device="cuda") * 2 - 0.5, torch.tensor(ptr, **i32),
            torch.tensor(ids, **i32), r(M, O))


def reference(x, w, a, b, scale, ptr, ids, dy):
    t = x.dtype
    u, lo, step = half_step(t), least(t), torch.finfo(t).eps / 2
    x, w, a, b, scale, dy = (v.double() for v in (x, w, a, b, scale, dy))
    (M, D), O, (n, R) = x.shape, w.shape[0], a.shape[:2]  # noqa: E741
    y, ey = x @ w.T, gamma(D + R) * (x.abs() @ w.abs().T)
    dx, edx = dy @ w, gamma(O + R) * (dy.abs() @ w.abs())
    da, eda, db, edb = (torch.zeros_like(v) for v in (a, a, b, b))
    p = ptr.tolist()
    for lo_, hi, k in zip(p, p[1:], ids.tolist()):
        if not 0 <= k < n or hi <= lo_:
            continue
        s, rows, g = scale[k], x[lo_:hi], dy[lo_:hi]
        S, T = rows @ a[k].T, g @ b[k]
        # the low-rank rows, scaled or not, are rounded to the type on their way
        eS = gamma(D) * (rows.abs() @ a[k].abs().T) + u * S.abs() + lo
        eT = gamma(O) * (g.abs() @ b[k].abs()) + u * T.abs() + lo
        y[lo_:hi] += s * S @ b[k].T
        ey[lo_:hi] += s.abs() * (eS + gamma(D + R) * S.abs()) @ b[k].abs().T + lo * b[k].abs().sum(1)
        dx[lo_:hi] += s * T @ a[k]
        edx[lo_:hi] += s.abs() * (eT + gamma(O + R) * T.abs()) @ a[k].abs() + lo * a[k].abs().sum(0)
        da[k] += s * T.T @ rows
        db[k] += s * g.T @ S
        m = gamma(M)
        eda[k] += s.abs() * ((eT + m * (T.abs() + eT)).T @ rows.abs()) + lo * rows.abs().sum(0)
        edb[k] += s.abs() * (g.abs().T @ (eS + m * (S.abs() + eS))) + lo * g.abs().sum(0)[:, None]
    out = {"y": (y, ey), "dx": (dx, edx), "da": (da, eda), "db": (db, edb)}
    return {k: (v, e * 1.01 + step * 1.01 * v.abs() + lo + 1e-30) for k, (v, e) in out.items()}


def check(got, want, names):
    for name, v in zip(names, got):
        ref, bound = want[name]
        assert v.shape == ref.shape
        assert torch.isfinite(v).all(), name
        off = (v.double() - ref).abs()
        assert not (off > bound).any(), (name, int((off > bound).sum()), float((off / bound).max()))


def both(args):
    want = reference(*args)
    y, kept = adapted_linear(*args[:7], keep=True)
    check([y], want, ["y"])
    assert torch.equal(y, adapted_linear(*args[:7]))
    check(adapted_linear_bwd(*args, kept=kept), want, ("dx", "da", "db"))
    grads = adapted_linear_bwd(*args)
    check(grads, want, ("dx", "da", "db"))
    alone = adapted_linear_bwd(*args, adapter_grads=False)
    assert alone[1] is None and torch.equal(alone[0], grads[0])


CASES = [
    # lengths, adapter ids, n, R, D, O
    ([1], [0], 1, 8, 64, 64),
    ([1] * 16, list(range(16)), 16, 16, 128, 256),
    ([1] * 40, [i % 7 - 1 for i in range(40)], 6, 4, 72, 40),
    ([5, 0, 30, 1, 0], [2, 1, 2, -1, 0], 3, 1, 33, 45),
    ([100, 200, 3, 0, 77], [1, 0, 1, 5, -7], 2, 20, 256, 136),
    ([300, 17, 290, 64], [0, 2, 1, 1], 4, 64, 136, 520),
    ([700], [0], 1, 128, 64, 72),
    ([3] * 200, [i * 5 % 11 for i in range(200)], 11, 12, 96, 64),
    ([1000, 1, 1, 900], [0, 1, 2, 1], 3, 16, 512, 256),
]


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_the_definition(case, t):
    both(make(*CASES[case], t, seed=case))


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_rows_of_no_request(t):
    # rows before the first request and behind the last have the projection alone
    args = make([20, 150, 9], [1, 0, 1], 2, 16, 64, 96, t, seed=20, head=37, tail=290)
    both(args)
    x, w, ptr = args[0], args[1], args[5].tolist()
    none = torch.full_like(args[6], -1)
    plain = adapted_linear(*args[:6], none)
    y = adapted_linear(*args[:7])
    assert torch.equal(y[:ptr[0]], plain[:ptr[0]]) and torch.equal(y[ptr[-1]:], plain[ptr[-1]:])


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_no_requests_and_no_adapters_and_no_rows(t):
    x, w, a, b, scale, ptr, ids, dy = make([10, 20], [0, 1], 2, 8, 64, 32, t, seed=21)
    plain = adapted_linear(x, w, a, b, scale, ptr, torch.full_like(ids, -1))
    assert torch.equal(adapted_linear(x, w, a, b, scale, ptr[:1], ids[:0]), plain)
    assert torch.equal(adapted_linear(x, w, a[:0], b[:0], scale[:0], ptr, ids), plain)
    dx, da, db = adapted_linear_bwd(x, w, a, b, scale, ptr[:1], ids[:0], dy)
    assert (da == 0).all() and (db == 0).all()
    e = adapted_linear(x[:0], w, a, b, scale, ptr * 0, ids)
    assert e.shape == (0, 32)
    dx, da, db = adapted_linear_bwd(x[:0], w, a, b, scale, ptr * 0, ids, dy[:0])
    assert dx.shape == (0, 64) and (da == 0).all() and (db == 0).all()


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_a_bound_outside_the_rows_is_kept_within_them(t):
    args = list(make([10, 40, 30], [0, 1, 0], 2, 8, 64, 64, t, seed=22))
    good = adapted_linear(*args[:7])
    args[5] = torch.tensor([-5, 10, 50, 10 ** 6], dtype=torch.int32, device="cuda")
    assert torch.equal(adapted_linear(*args[:7]), good)
    for v in adapted_linear_bwd(*args):
        assert torch.isfinite(v).all()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("size", [(3, 2, 4), (180, 150, 333)])
def test_what_is_not_finite_stays_with_its_request(size, t):
    args = make(size, [0, 1, 2], 3, 16, 128, 64, t, seed=23)
    y, grads = adapted_linear(*args[:7]), adapted_linear_bwd(*args)
    lo, hi = args[5].tolist()[1:3]
    rest = [i for i in range(args[0].shape[0]) if not lo <= i < hi]
    for which in ("x", "a", "b", "dy"):
        for value in (float("nan"), float("inf")):
            bad = [v.clone() for v in args]
            i = {"x": 0, "a": 2, "b": 3, "dy": 7}[which]
            bad[i][(1 if which in "ab" else lo + 1), 3] = value
            yb, gb = adapted_linear(*bad[:7]), adapted_linear_bwd(*bad)
            assert torch.equal(yb[rest], y[rest]), which
            assert torch.equal(gb[0][rest], grads[0][rest]), which
            for k in (1, 2):
                assert torch.equal(gb[k][0], grads[k][0]) and torch.equal(gb[k][2], grads[k][2])


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_strides_streams_and_repeats(t):
    args = list(make([100, 30, 200], [1, 0, 1], 2, 16, 72, 104, t, seed=24))
    want = (adapted_linear(*args[:7]), *adapted_linear_bwd(*args))
    torch.cuda.synchronize()
    M = args[0].shape[0]
    for pad in (3, 8):
        wide = [torch.full((M, v.shape[1] + pad), float("nan"), dtype=t, device="cuda")
                for v in (args[0], args[7])]
        xs, dys = wide[0][:, :72], wide[1][:, pad - 1:pad - 1 + 104]
        xs.copy_(args[0])
        dys.copy_(args[7])
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got = [(adapted_linear(xs, *args[1:7]), *adapted_linear_bwd(xs, *args[1:7], dys))
                   for _ in range(3)]
        st.synchronize()
        for r in got:
            assert all(torch.equal(p, q) for p, q in zip(r, want))


@pytest.mark.parametrize("rows", [1, 90])
def test_a_replayed_graph_sees_new_requests(rows):
    args = list(make([rows] * 4, [0, 1, 2, -1], 3, 16, 128, 64, torch.bfloat16, seed=25))
    adapted_linear(*args[:7])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, kept = adapted_linear(*args[:7], keep=True)
        out = (y, *adapted_linear_bwd(*args, kept=kept))
    args[6].copy_(torch.tensor([2, 2, -1, 0], dtype=torch.int32))
    args[5].copy_(torch.tensor([0, rows // 2, rows, 2 * rows, 4 * rows], dtype=torch.int32))
    g.replay()
    torch.cuda.synchronize()
    y, kept = adapted_linear(*args[:7], keep=True)
    for p, q in zip(out, (y, *adapted_linear_bwd(*args, kept=kept))):
        assert torch.equal(p, q)


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_adapted_projection_then_gated_block(t):
    """The two together, as a fine-tuned block runs them: forward, and the adjoint back through
    both, against one differentiation in 64 bits. The bound: the two operators' own relative
    errors in the 2-norm (each below 4 half steps of the type, fp32 below 2^-18), added, with
    the growth that the block's slope gives to an error of its rows."""
    x, w, a, b, scale, ptr, ids, _ = make([60, 1, 140], [1, -1, 0], 2, 16, 64, 96, t, seed=26)
    g = torch.Generator(device="cuda").manual_seed(27)
    wg, wu, wd, dy = ((torch.randn(*s, generator=g, device="cuda") * k).to(t) for s, k in
                      (((256, 96), 0.1), ((256, 96), 0.1), ((96, 256), 0.06), ((201, 96), 1.0)))
    h, kept1 = adapted_linear(x, w, a, b, scale, ptr, ids, keep=True)
    y, kept2 = gated_ff(h, wg, wu, wd, keep=True)
    dh, *dw = gated_ff_bwd(h, wg, wu, wd, dy, kept=kept2)
    dx, da, db = adapted_linear_bwd(x, w, a, b, scale, ptr, ids, dh, kept=kept1)
    leaves = [v.double().requires_grad_() for v in (x, a, b, wg, wu, wd)]
    X, A, B, G, U, D = leaves
    parts, p = [], ptr.tolist()
    for lo, hi, k in zip(p, p[1:], ids.tolist()):
        r = X[lo:hi] @ w.double().T
        parts.append(r if k < 0 else r + scale[k].double() * (X[lo:hi] @ A[k].T) @ B[k].T)
    H = torch.cat(parts)
    Y = (torch.nn.functional.silu(H @ G.T) * (H @ U.T)) @ D.T
    want = (Y.detach(), *torch.autograd.grad(Y, leaves, dy.double()))
    u = max(torch.finfo(t).eps / 2, 2.0 ** -20)
    for got, ref in zip((y, dx, da, db, *dw), want):
        assert float((got.double() - ref).norm() / ref.norm()) <= 4 * u * 4


MANY = [
    # requests of a tile that share adapters, in and out of order, with empty ones between them
    ([1] * 300, [i % 3 for i in range(300)], 3, 16, 64, 72),
    ([2, 0] * 400, [(i * 7 // 3) % 9 - 1 for i in range(800)], 8, 8, 40, 136),
    ([0] * 700 + [30, 0, 30] + [0] * 600 + [40], [i % 2 for i in range(1304)], 2, 4, 64, 64),
    ([1] * 100 + [400] + [1] * 100, [0, 1] * 50 + [1] + [1, 0] * 50, 2, 40, 72, 64),
    ([7] * 60, [i % 4 for i in range(60)], 4, 33, 128, 96),
    ([7] * 60, [i % 4 for i in range(60)], 4, 72, 136, 64),
    ([5] * 104, list(range(104)), 104, 20, 64, 200),
]


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("case", range(len(MANY)))
def test_requests_that_share_a_tile_and_an_adapter(case, t):
    both(make(*MANY[case], t, seed=60 + case))


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("R", [12, 72])
def test_rows_do_not_depend_on_how_requests_cut_them(R, t):
    # Blocks that have other requests' rows add zeros to a row's sums, which change nothing. In fp32
    # the sums leave tensor memory after every second stage of four slices of 16 ranks: a block of
    # several slices that does not begin on a stage has them cut elsewhere, and its rounding (not
    # its bound, gamma) depends on that.
    args = make([600], [1], 2, R, 64, 96, t, seed=70)
    x, w, a, b, scale, ptr, ids, dy = args
    y, dx = adapted_linear(*args[:7]), adapted_linear_bwd(*args, adapter_grads=False)[0]
    i32 = dict(dtype=torch.int32, device="cuda")
    want = reference(*args)
    for lengths in ([1] * 600, [250, 20, 330], [0] * 300 + [3, 0] * 200):
        p = torch.tensor([0] + lengths, **i32).cumsum(0).to(torch.int32)
        q = torch.ones(len(lengths), **i32)
        y2 = adapted_linear(x, w, a, b, scale, p, q)
        dx2 = adapted_linear_bwd(x, w, a, b, scale, p, q, dy, adapter_grads=False)[0]
        check([y2, dx2], want, ("y", "dx"))
        if t != torch.float32 or R <= 16:
            same = torch.equal(y2, y) and torch.equal(dx2, dx)
            assert same


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("M", [1, 7, 16, 17])
@pytest.mark.parametrize("R, D, O", [(1, 7, 300), (20, 1000, 33), (128, 72, 136), (9, 264, 8)])
def test_few_rows_both_ways(M, R, D, O, t):  # noqa: E741
    lengths = [M // 3, 0, M - M // 3]
    both(make(lengths, [1, 0, 2 if M > 1 else -1], 4, R, D, O, t, seed=80 + M))


def test_offsets_past_32_bits():
    # 2.2e9 outputs: the last rows and their adapter against the definition of those rows alone
    M, D, O, R, last = 1_050_000, 64, 2104, 16, 300  # noqa: E741
    t, g = torch.bfloat16, torch.Generator(device="cuda").manual_seed(5)

    def r(*shape, s=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * s).to(t)
    x, w, a, b = r(M, D), r(O, D, s=D ** -0.5), r(2, R, D, s=D ** -0.5), r(2, O, R, s=R ** -0.5)
    scale = torch.tensor([0.5, 1.5], device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    ptr, ids = torch.tensor([0, 500, M - last, M], **i32), torch.tensor([0, -1, 1], **i32)
    dy = r(M, O)
    want = reference(x[-last:], w, a, b, scale, torch.tensor([0, last], **i32), ids[2:], dy[-last:])
    check([adapted_linear(x, w, a, b, scale, ptr, ids)[-last:]], want, ["y"])
    dx, da, db = adapted_linear_bwd(x, w, a, b, scale, ptr, ids, dy)
    want = {"dx": want["dx"], **{k: tuple(v[1] for v in want[k]) for k in ("da", "db")}}
    check([dx[-last:], da[1], db[1]], want, ("dx", "da", "db"))
