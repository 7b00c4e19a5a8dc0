"""Low-rank adapters of many requests beside one shared projection, and their backward pass.

A batch of systems is stored back to back (as in ``evaluate_batch``), and each of them, a
request, may have a fine-tuned variant of the model: y = x W^T + s (x A^T) B^T with the request's
own A, B and s beside the W that all of them share. No counterpart in the reference, which bakes
one set of weights per composition (tt_atom/bundle_cache.py) and refuses a mixed batch. The
kernels are behind ``atom_adapted_linear_fwd`` / ``atom_adapted_linear_bwd``.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib as L
from .feedforward import buffer, check_kept, check_like, on_device, row_stride, rows_code


def _vector(name, t, dtype, n, x):
    if t.dtype != dtype or t.device != x.device or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a dense {dtype} vector of {n} on {x.device}")


def _shapes(x, w, a, b, scale, req_ptr, req_adapter):
    code = rows_code(x)
    if w.dim() != 2 or a.dim() != 3 or req_adapter.dim() != 1:
        raise ValueError("w must be [O, D], a [n, R, D], b [n, O, R] and req_adapter a vector")
    (M, D), O, (n, R, _) = x.shape, w.shape[0], a.shape  # noqa: E741
    nreq = req_adapter.shape[0]
    check_like("w", w, (O, D), x)
    check_like("a", a, (n, R, D), x)
    check_like("b", b, (n, O, R), x)
    _vector("scale", scale, torch.float32, n, x)
    _vector("req_adapter", req_adapter, torch.int32, nreq, x)
    _vector("req_ptr", req_ptr, torch.int32, nreq + 1, x)
    return code, M, D, O, n, R, nreq


@functools.lru_cache(maxsize=1024)
def _bytes(device, *sizes):
    """Workspace and kept sizes, by sizes and the GPU they are for."""
    out = (ctypes.c_size_t * 3)()
    L.call("atom_adapted_linear_bytes", *sizes, out)
    return tuple(out)


def adapted_linear(x, w, a, b, scale, req_ptr, req_adapter, keep=False):
    """y [M, O]: for the rows req_ptr[r] .. req_ptr[r + 1] - 1 of request r, with
    k = req_adapter[r], y = x w^T + scale[k] (x a[k]^T) b[k]^T; a request whose k is not in
    0 .. n - 1 (-1, say) and rows of no request have x w^T alone. x [M, D] with any row stride from
    D on, w [O, D], a [n, R, D], b [n, O, R], scale [n] float32, req_ptr [nreq + 1] ascending and
    req_adapter [nreq] int32, all on x's device: a replayed graph sees what they hold then.
    Requests may be empty and may share an adapter; 1 <= R <= 128, at most 2^14 adapters and
    2^22 requests (a little less above 112 ranks: include/atom_b200.h has the sum that has to fit).
    What is not finite in an adapter stays with its requests (whose rows may be NaN as a whole).
    Sums in float32; 16-bit types round the low-rank row, scale and all, before the product with b
    (above 16 rows). With ``keep`` returns (y, kept): what ``adapted_linear_bwd`` needs to spare
    the product x a^T. Does not synchronise; ``tt_atom.check_device`` tells whether a kernel gave up
    a wait."""
    sizes = code, M, D, O, n, R, nreq = _shapes(x, w, a, b, scale, req_ptr,  # noqa: E741
                                                req_adapter)
    ldx = row_stride("x", x)
    here, stream = on_device(x)
    with here:
        nb = _bytes(x.device.index, *sizes)
        y = torch.empty(M, O, dtype=x.dtype, device=x.device)
        ws, at = buffer(nb[0], x)
        kept, kept_at = buffer(nb[2], x) if keep else (None, None)
        L.call("atom_adapted_linear_fwd", code, x.data_ptr(), ldx, M, D, O, w.data_ptr(),
               a.data_ptr(), b.data_ptr(), scale.data_ptr(), n, R, req_ptr.data_ptr(),
               req_adapter.data_ptr(), nreq, y.data_ptr(), O, kept_at, at, nb[0], stream)
    return (y, kept) if keep else y


def adapted_linear_bwd(x, w, a, b, scale, req_ptr, req_adapter, dy, kept=None,
                       adapter_grads=True):
    """(dx, da, db) of ``adapted_linear`` from dy [M, O], in the inputs' type; the shared w has
    no gradient here (it is what the adapters leave fixed). An adapter of no request has zeros.
    Without ``adapter_grads`` the last two are None. 16-bit types round the low-rank rows before
    the products that take them (above 16 rows). ``kept``: what
    ``adapted_linear(..., keep=True)`` returned for the same inputs."""
    sizes = code, M, D, O, n, R, nreq = _shapes(x, w, a, b, scale, req_ptr,  # noqa: E741
                                                req_adapter)
    check_like("dy", dy, (M, O), x, dense=False)
    ldx, lddy = row_stride("x", x), row_stride("dy", dy)
    here, stream = on_device(x)
    with here:
        nb = _bytes(x.device.index, *sizes)
        if kept is not None:
            check_kept(kept, nb[2], x, "adapted_linear")
        dx = torch.empty(M, D, dtype=x.dtype, device=x.device)
        da = torch.empty_like(a) if adapter_grads else None
        db = torch.empty_like(b) if adapter_grads else None
        ws, at = buffer(nb[1], x)
        L.call("atom_adapted_linear_bwd", code, x.data_ptr(), ldx, M, D, O, w.data_ptr(),
               a.data_ptr(), b.data_ptr(), scale.data_ptr(), n, R, req_ptr.data_ptr(),
               req_adapter.data_ptr(), nreq, dy.data_ptr(), lddy, L.ptr(kept), dx.data_ptr(), D,
               L.ptr(da), L.ptr(db), at, nb[1], stream)
    return dx, da, db
