"""The gated feed-forward block y = (act(x Wg^T) * (x Wu^T)) Wd^T and its backward pass.

The block that the spectral feed-forward's gate (``atom_spectral_gate_fwd``) is the fixed-shape
case of, for any widths, in fp32, bf16 and fp16, with the gradients of its weights: what a
program needs to train or fine-tune a block and to run it in 16 bits. No counterpart in the
reference, whose feed-forwards are ungated MLPs (tt_atom/grid.py) or the spectral block
(tt_atom/spectral.py). The kernels are behind ``atom_gated_ff_fwd`` / ``atom_gated_ff_bwd``.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib as L

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTS = {"silu": 0, "sigmoid": 1, "gelu": 2}


def dtype_code(name, t):
    """The C ABI's type code of a tensor; ValueError for a type it does not have."""
    code = DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} is {t.dtype}: expected float32, bfloat16 or float16")
    return code


def check_like(name, t, shape, x):
    """A dense operand of ``shape`` with x's type, on x's device."""
    if t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{name} is {t.dtype} on {t.device}, x is {x.dtype} on {x.device}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}: expected {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def check_rows(name, t, x=None, shape=None):
    """A matrix whose rows are dense (any row stride of at least their width)."""
    if t.dim() != 2:
        raise ValueError(f"{name} must be a matrix [rows, width], got {t.dim()} dimensions")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device")
    if x is not None and (t.dtype != x.dtype or t.device != x.device):
        raise ValueError(f"{name} is {t.dtype} on {t.device}, x is {x.dtype} on {x.device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}: expected {tuple(shape)}")
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{name} must have dense rows (strides {t.stride()})")


def row_stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def buffer(nbytes, x):
    """A scratch tensor on x's device, from the current stream's pool (None for 0 bytes)."""
    return torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None


def _shapes(x, wg, wu, wd, act):
    check_rows("x", x)
    code = dtype_code("x", x)
    if act not in ACTS:
        raise ValueError(f"unknown activation {act!r}: expected one of {', '.join(ACTS)}")
    if wg.dim() != 2 or wd.dim() != 2:
        raise ValueError("wg, wu [F, D] and wd [O, F] must be matrices")
    (M, D), F, O = x.shape, wg.shape[0], wd.shape[0]  # noqa: E741
    check_like("wg", wg, (F, D), x)
    check_like("wu", wu, (F, D), x)
    check_like("wd", wd, (O, F), x)
    return code, M, D, F, O


def _bytes(code, M, D, F, O):  # noqa: E741
    out = (ctypes.c_size_t * 3)()
    L.call("atom_gated_ff_bytes", code, M, D, F, O, out)
    return out


def gated_ff(x, wg, wu, wd, act="silu", keep=False):
    """y [M, O] = (act(x wg^T) * (x wu^T)) wd^T for x [M, D], wg and wu [F, D], wd [O, F]; act:
    "silu", "sigmoid" or "gelu" (the erf form). x may have any row stride; the weights are
    dense. float32, bfloat16 or float16, sums in float32; the gated row h is rounded to the
    inputs' type before the second product (float32: it is not). With ``keep`` returns
    (y, kept): what ``gated_ff_bwd`` needs to spare the first two products. Runs on the current
    stream of x's device, without synchronising."""
    code, M, D, F, O = _shapes(x, wg, wu, wd, act)  # noqa: E741
    with torch.cuda.device(x.device):
        n = _bytes(code, M, D, F, O)
        y = torch.empty(M, O, dtype=x.dtype, device=x.device)
        ws, kept = buffer(n[0], x), buffer(n[2], x) if keep else None
        L.call("atom_gated_ff_fwd", code, x.data_ptr(), row_stride(x), M, D, F, O, wg.data_ptr(),
               wu.data_ptr(), wd.data_ptr(), ACTS[act], y.data_ptr(), O, L.ptr(kept), L.ptr(ws),
               n[0], L.stream_ptr())
    return (y, kept) if keep else y


def gated_ff_bwd(x, wg, wu, wd, dy, act="silu", kept=None, weight_grads=True):
    """(dx, dwg, dwu, dwd) of ``gated_ff`` from dy [M, O], in the inputs' type; the last three
    are None without ``weight_grads`` (the adjoint of the rows alone, as forces need it).
    ``kept`` is what ``gated_ff(..., keep=True)`` returned for the same inputs; without it the
    first two products are computed again."""
    code, M, D, F, O = _shapes(x, wg, wu, wd, act)  # noqa: E741
    check_rows("dy", dy, x, (M, O))
    with torch.cuda.device(x.device):
        n = _bytes(code, M, D, F, O)
        if kept is not None and (kept.dtype != torch.uint8 or kept.numel() != n[2]
                                 or kept.device != x.device):
            raise ValueError("kept is not what gated_ff(..., keep=True) returns for these inputs")
        dx = torch.empty(M, D, dtype=x.dtype, device=x.device)
        dw = [torch.empty_like(w) for w in (wg, wu, wd)] if weight_grads else [None] * 3
        ws = buffer(n[1], x)
        L.call("atom_gated_ff_bwd", code, x.data_ptr(), row_stride(x), M, D, F, O, wg.data_ptr(),
               wu.data_ptr(), wd.data_ptr(), ACTS[act], dy.data_ptr(), row_stride(dy),
               L.ptr(kept), dx.data_ptr(), D, *map(L.ptr, dw), L.ptr(ws), n[1], L.stream_ptr())
    return (dx, *dw)
