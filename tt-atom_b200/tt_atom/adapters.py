"""Low-rank adapters of many requests beside one shared projection, and their backward pass.

A batch of systems is stored back to back (as in ``evaluate_batch``), and each of them, a
request, may have a fine-tuned variant of the model: y = x W^T + s (x A^T) B^T with the request's
own A, B and s beside the W that all of them share. No counterpart in the reference, which bakes
one set of weights per composition (tt_atom/bundle_cache.py) and refuses a mixed batch. The
kernels are behind ``atom_adapted_linear_fwd`` / ``atom_adapted_linear_bwd``.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib as L
from .feedforward import buffer, check_like, check_rows, dtype_code, row_stride


def _int32(name, t, x, n=None):
    if t.dtype != torch.int32 or t.device != x.device or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a dense int32 vector on {x.device}")
    if n is not None and t.numel() != n:
        raise ValueError(f"{name} has {t.numel()} entries: expected {n}")


def _shapes(x, w, a, b, scale, req_ptr, req_adapter):
    check_rows("x", x)
    code = dtype_code("x", x)
    if w.dim() != 2 or a.dim() != 3:
        raise ValueError("w must be [O, D], a [n, R, D] and b [n, O, R]")
    (M, D), O, (n, R) = x.shape, w.shape[0], a.shape[:2]  # noqa: E741
    check_like("w", w, (O, D), x)
    check_like("a", a, (n, R, D), x)
    check_like("b", b, (n, O, R), x)
    if scale.dtype != torch.float32 or scale.device != x.device or tuple(scale.shape) != (n,) \
            or not scale.is_contiguous():
        raise ValueError(f"scale must be a dense float32 vector of {n} on {x.device}")
    _int32("req_adapter", req_adapter, x)
    _int32("req_ptr", req_ptr, x, req_adapter.numel() + 1)
    return code, M, D, O, n, R, req_adapter.numel()


def _bytes(code, M, D, O, n, R, nreq):  # noqa: E741
    out = (ctypes.c_size_t * 3)()
    L.call("atom_adapted_linear_bytes", code, M, D, O, n, R, nreq, out)
    return out


def adapted_linear(x, w, a, b, scale, req_ptr, req_adapter, keep=False):
    """y [M, O]: for the rows req_ptr[r] .. req_ptr[r + 1] - 1 of request r, with
    k = req_adapter[r], y = x w^T + scale[k] (x a[k]^T) b[k]^T; a request whose k is not in
    0 .. n - 1 (-1, say) and rows of no request have x w^T alone. x [M, D] with any row stride,
    w [O, D], a [n, R, D], b [n, O, R], scale [n] float32, req_ptr [nreq + 1] ascending and
    req_adapter [nreq] int32, all on x's device: a replayed graph sees what they hold then.
    Requests may be empty and may share an adapter. Sums in float32. With ``keep`` returns
    (y, kept): what ``adapted_linear_bwd`` needs to spare the product x a^T."""
    code, M, D, O, n, R, nreq = _shapes(x, w, a, b, scale, req_ptr, req_adapter)  # noqa: E741
    with torch.cuda.device(x.device):
        nb = _bytes(code, M, D, O, n, R, nreq)
        y = torch.empty(M, O, dtype=x.dtype, device=x.device)
        ws, kept = buffer(nb[0], x), buffer(nb[2], x) if keep else None
        L.call("atom_adapted_linear_fwd", code, x.data_ptr(), row_stride(x), M, D, O,
               w.data_ptr(), a.data_ptr(), b.data_ptr(), scale.data_ptr(), n, R,
               req_ptr.data_ptr(), req_adapter.data_ptr(), nreq, y.data_ptr(), O, L.ptr(kept),
               L.ptr(ws), nb[0], L.stream_ptr())
    return (y, kept) if keep else y


def adapted_linear_bwd(x, w, a, b, scale, req_ptr, req_adapter, dy, kept=None,
                       adapter_grads=True):
    """(dx, da, db) of ``adapted_linear`` from dy [M, O], in the inputs' type; the shared w has
    no gradient here (it is what the adapters leave fixed). An adapter of no request has zeros.
    Without ``adapter_grads`` the last two are None. ``kept``: what
    ``adapted_linear(..., keep=True)`` returned for the same inputs."""
    code, M, D, O, n, R, nreq = _shapes(x, w, a, b, scale, req_ptr, req_adapter)  # noqa: E741
    check_rows("dy", dy, x, (M, O))
    with torch.cuda.device(x.device):
        nb = _bytes(code, M, D, O, n, R, nreq)
        if kept is not None and (kept.dtype != torch.uint8 or kept.numel() != nb[2]
                                 or kept.device != x.device):
            raise ValueError("kept is not what adapted_linear(..., keep=True) returns for these "
                             "inputs")
        dx = torch.empty(M, D, dtype=x.dtype, device=x.device)
        da = torch.empty_like(a) if adapter_grads else None
        db = torch.empty_like(b) if adapter_grads else None
        ws = buffer(nb[1], x)
        L.call("atom_adapted_linear_bwd", code, x.data_ptr(), row_stride(x), M, D, O,
               w.data_ptr(), a.data_ptr(), b.data_ptr(), scale.data_ptr(), n, R,
               req_ptr.data_ptr(), req_adapter.data_ptr(), nreq, dy.data_ptr(), row_stride(dy),
               L.ptr(kept), dx.data_ptr(), D, L.ptr(da), L.ptr(db), L.ptr(ws), nb[1],
               L.stream_ptr())
    return dx, da, db
