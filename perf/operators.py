"""Cases of the gated feed-forward block and of the low-rank adapters beside a shared projection:
what a program has in hand, the operators in plain torch operations, and the framework's calls."""
import math
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one row through a block, as a program does that evaluates a single system's head
        {"name": "ff token bf16", "op": "ff", "dir": "fwd", "type": "bf16", "act": "silu",
         "M": 1, "D": 1024, "F": 4096, "O": 1024},
        # the nodes of a 1,002-atom cell through a 256-wide block, in the framework's own type
        {"name": "ff nodes f32", "op": "ff", "dir": "fwd", "type": "f32", "act": "silu",
         "M": 1002, "D": 256, "F": 1024, "O": 256},
        # the edges of a 2,000-atom cell (30 a receiver) through the same block
        {"name": "ff edges bf16", "op": "ff", "dir": "fwd", "type": "bf16", "act": "silu",
         "M": 60000, "D": 256, "F": 1024, "O": 256},
        # forces: the adjoint of the rows alone, weights fixed; odd rows and widths
        {"name": "ff forces f16", "op": "ff", "dir": "vjp", "type": "f16", "act": "gelu",
         "M": 3001, "D": 500, "F": 1333, "O": 500},
        # training in the framework's type: every gradient, 9 coefficients of 2,000 atoms, 128 wide
        {"name": "ff train f32", "op": "ff", "dir": "train", "type": "f32", "act": "silu",
         "M": 18000, "D": 128, "F": 512, "O": 128},
        # training a wide block
        {"name": "ff train bf16", "op": "ff", "dir": "train", "type": "bf16", "act": "silu",
         "M": 8192, "D": 2048, "F": 8192, "O": 2048},
        # 16 requests with one row each, an adapter each
        {"name": "adapters tokens bf16", "op": "ad", "dir": "fwd", "type": "bf16",
         "M": 16, "requests": 16, "adapters": 16, "R": 16, "D": 2048, "O": 2048},
        # a screening batch: 512 molecules of 24 atoms or so, 40 fine-tunes, the framework's type
        {"name": "adapters screen f32", "op": "ad", "dir": "fwd", "type": "f32",
         "M": 12011, "requests": 512, "adapters": 40, "R": 8, "D": 256, "O": 1024},
        # requests of mixed lengths beside a wide projection
        {"name": "adapters mixed bf16", "op": "ad", "dir": "fwd", "type": "bf16",
         "M": 8192, "requests": 48, "adapters": 24, "R": 32, "D": 2048, "O": 4096},
        # the adapters' training step: rows' and adapters' gradients, the projection fixed
        {"name": "adapters train bf16", "op": "ad", "dir": "train", "type": "bf16",
         "M": 6007, "requests": 24, "adapters": 8, "R": 16, "D": 2048, "O": 2048},
        {"name": "adapters train f32", "op": "ad", "dir": "train", "type": "f32",
         "M": 4000, "requests": 200, "adapters": 20, "R": 20, "D": 256, "O": 256},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    n = _log(rng, low, high)
    return n if rng.random() < 0.25 else max(low, n // 8 * 8)


def draw(rng):
    type_ = rng.choice(["f32", "bf16", "bf16", "f16"])
    if rng.random() < 0.5:
        dir_ = rng.choice(["fwd", "fwd", "vjp", "train"])
        D, F = _width(rng, 64, 2048), _width(rng, 128, 8192)
        O = D if rng.random() < 0.8 else _width(rng, 64, 2048)  # noqa: E741
        most = 8192 * 2048 * 8192 // (max(D, O) * F * (4 if type_ == "f32" else 1))
        return {"op": "ff", "dir": dir_, "type": type_, "act": rng.choice(["silu", "silu", "sigmoid", "gelu"]),
                "M": _log(rng, 1, min(60000, max(2, most))), "D": D, "F": F, "O": O}
    dir_ = rng.choice(["fwd", "fwd", "train"])
    D, O = _width(rng, 64, 4096), _width(rng, 64, 4096)  # noqa: E741
    M = _log(rng, 1, 12000)
    requests = min(512, _log(rng, 1, max(2, M)))
    return {"op": "ad", "dir": dir_, "type": type_, "M": M, "requests": requests,
            "adapters": _log(rng, 1, min(64, max(2, requests))), "R": rng.choice([4, 8, 8, 12, 16, 16, 20, 32, 64]),
            "D": D, "O": O}


def _lengths(case, seed):
    """Rows of each request: ragged, some empty, all of them together M (decoding: one each)."""
    r, n, M = random.Random(seed * 7919 + 1), case["requests"], case["M"]
    if n == M:
        return [1] * n
    share = [0.0 if r.random() < 0.05 and n > 1 else r.uniform(0.2, 1.8) for _ in range(n)]
    share[r.randrange(n)] += 0.2
    total, at, cuts = sum(share), 0.0, [0]
    for s in share:
        at += s
        cuts.append(min(M, int(round(at / total * M))))
    return [b - a for a, b in zip(cuts, cuts[1:])]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(t)

    def weight(*shape):  # uniform, scaled by the fan-in
        return ((torch.rand(*shape, generator=g, device="cuda") * 2 - 1) / math.sqrt(shape[-1])).to(t)

    M, D, O = case["M"], case["D"], case["O"]  # noqa: E741
    s = {"case": case, "x": normal(M, D)}
    if case["op"] == "ff":
        F = case["F"]
        # weights spread a little wider than at their start, so that the gates are not all near a half
        s.update(wg=weight(F, D) * 2, wu=weight(F, D) * 2, wd=weight(O, F) * 2)
        if case["dir"] != "fwd":
            s["dy"] = normal(M, O, std=0.1)
        return s
    n, R, nreq = case["adapters"], case["R"], case["requests"]
    r = random.Random(seed * 104729 + 3)
    lengths = _lengths(case, seed)
    ptr = [0]
    for k in lengths:
        ptr.append(ptr[-1] + k)
    ids = [-1 if r.random() < 0.08 else r.randrange(n) for _ in range(nreq)]
    if nreq == n:
        ids = list(range(n))
    s.update(w=weight(O, D), a=weight(n, R, D), b=weight(n, O, R) * 0.5,
             scale=torch.rand(n, generator=g, device="cuda") * 1.5 + 0.5,
             req_ptr=torch.tensor(ptr, dtype=torch.int32, device="cuda"),
             req_adapter=torch.tensor(ids, dtype=torch.int32, device="cuda"))
    if case["dir"] != "fwd":
        s["dy"] = normal(M, O, std=0.1)
    return s


def _act(g, act):
    """The activation and its derivative."""
    if act == "gelu":
        phi = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    p = 1 / (1 + torch.exp(-g))
    if act == "sigmoid":
        return p, p * (1 - p)
    return g * p, p * (1 + g * (1 - p))


def _plain_ff(s):
    case, t = s["case"], s["x"].dtype
    x, wg, wu, wd = (s[k].float() for k in ("x", "wg", "wu", "wd"))
    g, u = x @ wg.T, x @ wu.T
    a, da = _act(g, case["act"])
    h = a * u
    if case["dir"] == "fwd":
        return {"y": (h @ wd.T).to(t)}
    dy = s["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * da, dh * a
    out = {"dx": dg @ wg + du @ wu}
    if case["dir"] == "train":
        out.update(y=h @ wd.T, dwg=dg.T @ x, dwu=du.T @ x, dwd=dy.T @ h)
    return {k: v.to(t) for k, v in out.items()}


def _plain_ad(s):
    case, t = s["case"], s["x"].dtype
    x, w, a, b = (s[k].float() for k in ("x", "w", "a", "b"))
    n, R, D = a.shape
    O = w.shape[0]  # noqa: E741
    # every adapter's product for every row, and a mask of which row has which
    rows = torch.arange(x.shape[0], device=x.device)
    request = torch.bucketize(rows, s["req_ptr"][1:].long(), right=True)
    request = request.clamp(max=case["requests"] - 1)
    mask = (s["req_adapter"][request][:, None] == torch.arange(n, device=x.device)) * s["scale"]
    mask = mask[:, :, None].expand(-1, n, R).reshape(-1, n * R)
    flat_a, flat_b = a.reshape(n * R, D), b.transpose(1, 2).reshape(n * R, O)
    xa = (x @ flat_a.T) * mask
    out = {"y": x @ w.T + xa @ flat_b}
    if case["dir"] == "train":
        dy = s["dy"].float()
        tb = (dy @ flat_b.T) * mask
        out.update(dx=dy @ w + tb @ flat_a, da=(tb.T @ x).reshape(n, R, D),
                   db=(dy.T @ xa).reshape(O, n, R).transpose(0, 1))
    return {k: v.to(t) for k, v in out.items()}


def run(s):
    case = s["case"]
    if not own:
        return _plain_ff(s) if case["op"] == "ff" else _plain_ad(s)
    if "tt-atom_b200" not in sys.path:
        sys.path.insert(0, "tt-atom_b200")
    if case["op"] == "ff":
        from tt_atom.feedforward import gated_ff, gated_ff_bwd
        weights = s["wg"], s["wu"], s["wd"]
        if case["dir"] == "fwd":
            return {"y": gated_ff(s["x"], *weights, act=case["act"])}
        if case["dir"] == "vjp":
            return {"dx": gated_ff_bwd(s["x"], *weights, s["dy"], act=case["act"], weight_grads=False)[0]}
        y, kept = gated_ff(s["x"], *weights, act=case["act"], keep=True)
        dx, dwg, dwu, dwd = gated_ff_bwd(s["x"], *weights, s["dy"], act=case["act"], kept=kept)
        return {"y": y, "dx": dx, "dwg": dwg, "dwu": dwu, "dwd": dwd}
    from tt_atom.adapters import adapted_linear, adapted_linear_bwd
    args = s["x"], s["w"], s["a"], s["b"], s["scale"], s["req_ptr"], s["req_adapter"]
    if case["dir"] == "fwd":
        return {"y": adapted_linear(*args)}
    y, kept = adapted_linear(*args, keep=True)
    dx, da, db = adapted_linear_bwd(*args, s["dy"], kept=kept)
    return {"y": y, "dx": dx, "da": da, "db": db}


def work(case):
    size = 4 if case["type"] == "f32" else 2
    M, D, O = case["M"], case["D"], case["O"]  # noqa: E741
    if case["op"] == "ff":
        F = case["F"]
        weights, forward = F * (2 * D + O), 2 * M * F * (2 * D + O)
        if case["dir"] == "fwd":
            return {"bytes": size * (M * (D + O) + weights), "flops": forward}
        # the adjoint of the rows needs the gates again, which come from the rows
        vjp = 2 * M * F * (2 * D + O + 2 * D)
        if case["dir"] == "vjp":
            return {"bytes": size * (M * (2 * D + O) + weights), "flops": vjp}
        return {"bytes": size * (M * (2 * D + 2 * O) + 2 * weights), "flops": 2 * M * F * O + vjp + forward}
    # adapters that no request can have need not be read
    n, R = min(case["adapters"], case["requests"]), case["R"]
    adapters = n * R * (D + O)
    flops, values = 2 * M * (D * O + R * (D + O)), M * (D + O) + D * O + adapters
    if case["dir"] == "train":
        flops += 2 * M * (D * O + R * (D + O)) + 2 * M * R * (D + O)
        values += M * (D + O) + case["adapters"] * R * (D + O)
    return {"bytes": size * values, "flops": flops}


def exact(case, seed):
    """From the definitions in 64 bits: each request by itself, gradients by differentiation."""
    s = prepare(case, seed)
    train = case["dir"] != "fwd"
    if case["op"] == "ff":
        x, wg, wu, wd = leaves = [s[k].double().requires_grad_(train) for k in ("x", "wg", "wu", "wd")]
        g = torch.einsum("md,fd->mf", x, wg)
        gate = {"silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid, "gelu": torch.nn.functional.gelu}
        y = torch.einsum("mf,of->mo", gate[case["act"]](g) * torch.einsum("md,fd->mf", x, wu), wd)
        if not train:
            return {"y": y}
        grads = torch.autograd.grad(y, leaves[:1] if case["dir"] == "vjp" else leaves, s["dy"].double())
        if case["dir"] == "vjp":
            return {"dx": grads[0]}
        return dict(zip(("y", "dx", "dwg", "dwu", "dwd"), (y.detach(), *grads)))
    x, a, b = leaves = [s[k].double().requires_grad_(train) for k in ("x", "a", "b")]
    w, scale = s["w"].double(), s["scale"].double()
    ptr, ids, parts = s["req_ptr"].tolist(), s["req_adapter"].tolist(), []
    for lo, hi, k in zip(ptr, ptr[1:], ids):
        rows = x[lo:hi]
        y = rows.matmul(w.t())
        if k >= 0:
            y = y + rows.matmul(a[k].t()).matmul(b[k].t()).mul(scale[k])
        parts.append(y)
    y = torch.cat(parts)
    if not train:
        return {"y": y}
    grads = torch.autograd.grad(y, leaves, s["dy"].double(), allow_unused=True)
    grads = [torch.zeros_like(v) if q is None else q for v, q in zip(leaves, grads)]
    return {"y": y.detach(), "dx": grads[0], "da": grads[1], "db": grads[2]}
