"""The gated feed-forward block y = (act(x Wg^T) * (x Wu^T)) Wd^T and its backward pass.

For any widths, in fp32, bf16 and fp16, with the gradients of its weights: what a program needs
to train or fine-tune such a block and to run it in 16 bits. It stands beside the feed-forwards
of the models, which have gates of their own in fixed shapes and fp32
(``atom_spectral_gate_fwd``) and do not call it. No counterpart in the reference, whose
feed-forwards are ungated MLPs (tt_atom/grid.py) or the spectral block (tt_atom/spectral.py).
The kernels are behind ``atom_gated_ff_fwd`` / ``atom_gated_ff_bwd``.
As everywhere in this package gradients are functions of their own: autograd does not see them.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools

import torch

from . import _lib as L

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTS = {"silu": 0, "sigmoid": 1, "gelu": 2}
_SAME = contextlib.nullcontext()


def rows_code(x):
    """Checks the matrix x of rows and returns the C ABI's code of its type."""
    if x.dim() != 2:
        raise ValueError(f"x must be a matrix [rows, width], got {x.dim()} dimensions")
    if not x.is_cuda:
        raise ValueError("x must be on a CUDA device")
    code = DTYPES.get(x.dtype)
    if code is None:
        raise ValueError(f"x is {x.dtype}: expected float32, bfloat16 or float16")
    return code


def row_stride(name, t):
    """The stride of a matrix's rows, which have to be dense."""
    rows, width = t.shape
    if rows <= 1:
        if width > 1 and t.stride(1) != 1:
            raise ValueError(f"{name} must have dense rows (strides {t.stride()})")
        return width
    s0, s1 = t.stride()
    if width > 1 and s1 != 1 or s0 < width:
        raise ValueError(f"{name} must have dense rows (strides {t.stride()})")
    return s0


def check_like(name, t, shape, x, dense=True):
    """An operand of ``shape`` with x's type, on x's device."""
    if t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{name} is {t.dtype} on {t.device}, x is {x.dtype} on {x.device}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}: expected {tuple(shape)}")
    if dense and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def on_device(x):
    """Context with x's device current, and x's current stream there."""
    i = x.device.index
    return (_SAME if i == torch.cuda.current_device() else torch.cuda.device(i),
            torch._C._cuda_getCurrentRawStream(i))


def buffer(nbytes, x):
    """Scratch on x's device from the current stream's pool, and its address."""
    t = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    return t, t.data_ptr()


def check_kept(kept, nbytes, x, maker):
    if kept.dtype != torch.uint8 or kept.numel() != nbytes or kept.device != x.device:
        raise ValueError(f"kept is not what {maker}(..., keep=True) returns for these inputs")


def _shapes(x, wg, wu, wd, act):
    code = rows_code(x)
    if act not in ACTS:
        raise ValueError(f"unknown activation {act!r}: expected one of {', '.join(ACTS)}")
    if wg.dim() != 2 or wd.dim() != 2:
        raise ValueError("wg, wu [F, D] and wd [O, F] must be matrices")
    (M, D), F, O = x.shape, wg.shape[0], wd.shape[0]  # noqa: E741
    check_like("wg", wg, (F, D), x)
    check_like("wu", wu, (F, D), x)
    check_like("wd", wd, (O, F), x)
    return code, M, D, F, O


@functools.lru_cache(maxsize=1024)
def _bytes(device, *sizes):
    """Workspace and kept sizes, by sizes and the GPU they are for."""
    out = (ctypes.c_size_t * 3)()
    L.call("atom_gated_ff_bytes", *sizes, out)
    return tuple(out)


def gated_ff(x, wg, wu, wd, act="silu", keep=False):
    """y [M, O] = (act(x wg^T) * (x wu^T)) wd^T for x [M, D], wg and wu [F, D], wd [O, F]; act:
    "silu", "sigmoid" or "gelu" (the erf form). x may have any row stride from its width on; the
    weights are dense. float32, bfloat16 or float16, sums in float32; the gated row h is rounded to the
    inputs' type before the second product (float32: it is not). With ``keep`` returns
    (y, kept): what ``gated_ff_bwd`` needs to spare the first two products. Runs on the current
    stream of x's device, without synchronising: call ``tt_atom.check_device`` where results are
    read back, which raises if a kernel gave up a wait."""
    code, M, D, F, O = _shapes(x, wg, wu, wd, act)  # noqa: E741
    ldx = row_stride("x", x)
    here, stream = on_device(x)
    with here:
        n = _bytes(x.device.index, code, M, D, F, O)
        y = torch.empty(M, O, dtype=x.dtype, device=x.device)
        ws, at = buffer(n[0], x)
        kept, kept_at = buffer(n[2], x) if keep else (None, None)
        L.call("atom_gated_ff_fwd", code, x.data_ptr(), ldx, M, D, F, O, wg.data_ptr(),
               wu.data_ptr(), wd.data_ptr(), ACTS[act], y.data_ptr(), O, kept_at, at, n[0], stream)
    return (y, kept) if keep else y


def gated_ff_bwd(x, wg, wu, wd, dy, act="silu", kept=None, weight_grads=True):
    """(dx, dwg, dwu, dwd) of ``gated_ff`` from dy [M, O], in the inputs' type; the last three
    are None without ``weight_grads`` (the adjoint of the rows alone, as forces need it).
    ``kept`` is what ``gated_ff(..., keep=True)`` returned for the same inputs; without it the
    first two products are computed again. 16-bit types round h and the gradients of the gate's
    two factors before the products that take them (a few rows: not)."""
    code, M, D, F, O = _shapes(x, wg, wu, wd, act)  # noqa: E741
    check_like("dy", dy, (M, O), x, dense=False)
    ldx, lddy = row_stride("x", x), row_stride("dy", dy)
    here, stream = on_device(x)
    with here:
        n = _bytes(x.device.index, code, M, D, F, O)
        if kept is not None:
            check_kept(kept, n[2], x, "gated_ff")
        dx = torch.empty(M, D, dtype=x.dtype, device=x.device)
        dw = [torch.empty_like(w) for w in (wg, wu, wd)] if weight_grads else [None] * 3
        ws, at = buffer(n[1], x)
        L.call("atom_gated_ff_bwd", code, x.data_ptr(), ldx, M, D, F, O, wg.data_ptr(),
               wu.data_ptr(), wd.data_ptr(), ACTS[act], dy.data_ptr(), lddy, L.ptr(kept),
               dx.data_ptr(), D, *map(L.ptr, dw), at, n[1], stream)
    return (dx, *dw)
