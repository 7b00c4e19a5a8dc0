"""What the typed operators (gated feed-forward, adapters) refuse, before any work on a GPU: the
C interface's checks through the built library, the Python wrappers' on CPU tensors."""
import ctypes

import pytest
import torch

from tt_atom import _lib as L
from tt_atom.adapters import adapted_linear, adapted_linear_bwd
from tt_atom.feedforward import gated_ff, gated_ff_bwd

P = ctypes.c_void_p(256)      # never read: every call here is refused on the host


def status(name, *args):
    return getattr(L.lib(), name)(*args), L.last_error()


def ff(dtype=1, ldx=8, M=4, D=8, F=16, O=8, act=0, ldy=8, x=P, ws=P, nbytes=1 << 40):  # noqa: E741
    return status("atom_gated_ff_fwd", dtype, x, ldx, M, D, F, O, P, P, P, act, P, ldy, None, ws,
                  nbytes, None)


def ff_bwd(lddy=8, lddx=8, nbytes=1 << 40, dy=P, act=0):
    return status("atom_gated_ff_bwd", 1, P, 8, 4, 8, 16, 8, P, P, P, act, dy, lddy, None, P, lddx,
                  P, P, P, P, nbytes, None)


def ad(dtype=1, M=4, D=8, O=8, n=2, R=8, nreq=2, ldx=8, ldy=8, a=P, ptr=P, nbytes=1 << 40):  # noqa: E741
    return status("atom_adapted_linear_fwd", dtype, P, ldx, M, D, O, P, a, P, P, n, R, ptr, P,
                  nreq, P, ldy, None, P, nbytes, None)


def ad_bwd(lddy=8, lddx=8, R=8, nbytes=1 << 40):
    return status("atom_adapted_linear_bwd", 1, P, 8, 4, 8, 8, P, P, P, P, 2, R, P, P, 2, P, lddy,
                  None, P, lddx, P, P, P, nbytes, None)


@pytest.mark.parametrize("call, words", [
    (lambda: ff(dtype=3), "type"), (lambda: ff(dtype=-1), "type"), (lambda: ff(M=-1), "sizes"),
    (lambda: ff(M=1 << 31), "sizes"), (lambda: ff(D=0), "sizes"), (lambda: ff(F=0), "sizes"),
    (lambda: ff(O=0), "sizes"), (lambda: ff(D=1 << 25, ldx=1 << 25), "2^24"),
    (lambda: ff(act=3), "act"), (lambda: ff(ldx=7), "operand"), (lambda: ff(ldy=7), "operand"),
    (lambda: ff(x=None), "operand"), (lambda: ff(ws=None), "workspace"),
    (lambda: ff(nbytes=16), "workspace"), (lambda: ff_bwd(lddy=7), "operand"),
    (lambda: ff_bwd(lddx=7), "operand"), (lambda: ff_bwd(dy=None), "operand"),
    (lambda: ff_bwd(act=-1), "act"), (lambda: ff_bwd(nbytes=16), "workspace"),
    (lambda: ad(dtype=9), "type"), (lambda: ad(M=-1), "sizes"), (lambda: ad(D=0), "sizes"),
    (lambda: ad(O=-3), "sizes"), (lambda: ad(n=-1), "sizes"), (lambda: ad(nreq=-1), "sizes"),
    (lambda: ad(R=0), "rank"), (lambda: ad(R=129), "rank"), (lambda: ad(ldx=7), "operand"),
    (lambda: ad(ldy=7), "operand"), (lambda: ad(a=None), "operand"),
    (lambda: ad(ptr=None), "operand"), (lambda: ad(nbytes=16), "workspace"),
    (lambda: ad_bwd(lddy=7), "operand"), (lambda: ad_bwd(lddx=7), "operand"),
    (lambda: ad_bwd(R=500), "rank"), (lambda: ad_bwd(nbytes=16), "workspace"),
])
def test_c_interface_refuses(call, words):
    code, message = call()
    assert code == 1 and words in message, message


def test_size_queries():
    n = (L.c_size_t * 3)()
    L.call("atom_gated_ff_bytes", 1, 100, 64, 128, 64, n)
    assert all(v > 0 for v in n)
    big = (L.c_size_t * 3)()
    L.call("atom_gated_ff_bytes", 1, 1 << 20, 4096, 16384, 4096, big)      # past 32 bits
    assert big[1] > 1 << 32
    L.call("atom_adapted_linear_bytes", 0, 100, 64, 128, 4, 8, 3, n)
    assert all(v > 0 for v in n)
    assert status("atom_gated_ff_bytes", 1, 4, 8, 8, 8, None)[0] == 1
    assert status("atom_adapted_linear_bytes", 1, 4, 8, 8, 2, 8, 1, None)[0] == 1


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_python_wrappers_refuse():
    w = t(16, 8), t(16, 8), t(8, 16)
    for call in (lambda: gated_ff(t(4, 8), *w),                       # not on a CUDA device
                 lambda: gated_ff(t(8), *w),
                 lambda: gated_ff(t(4, 8, dtype=torch.float64), *w),
                 lambda: gated_ff_bwd(t(4, 8), *w, t(4, 8)),
                 lambda: adapted_linear(t(4, 8), t(8, 8), t(2, 4, 8), t(2, 8, 4), t(2),
                                        t(2, dtype=torch.int32), t(1, dtype=torch.int32)),
                 lambda: adapted_linear_bwd(t(4, 8), t(8, 8), t(2, 4, 8), t(2, 8, 4), t(2),
                                            t(2, dtype=torch.int32), t(1, dtype=torch.int32),
                                            t(4, 8))):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_python_wrappers_refuse_on_the_gpu():
    def c(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=dtype, device="cuda")
    i32 = torch.int32
    x, w = c(4, 8), (c(16, 8), c(16, 8), c(8, 16))
    ok = dict(x=x, w=c(8, 8), a=c(2, 4, 8), b=c(2, 8, 4), scale=c(2, dtype=torch.float32),
              req_ptr=c(3, dtype=i32), req_adapter=c(2, dtype=i32))
    adapted_linear(**ok)
    bad = [dict(x=c(8, 4).T), dict(x=c(4, 8, dtype=torch.float64)), dict(w=c(8, 9)),
           dict(a=c(2, 4, 9)), dict(b=c(2, 8, 5)), dict(b=c(2, 4, 8).transpose(1, 2)),
           dict(scale=c(2)), dict(scale=c(3, dtype=torch.float32)), dict(req_ptr=c(2, dtype=i32)),
           dict(req_adapter=c(2, dtype=torch.int64)), dict(a=c(2, 4, 8, dtype=torch.float16)),
           dict(w=torch.zeros(8, 8, dtype=torch.bfloat16))]
    for change in bad:
        with pytest.raises(ValueError):
            adapted_linear(**{**ok, **change})
    for call in (lambda: gated_ff(x, *w, act="relu"), lambda: gated_ff(x, w[0], w[1], c(8, 15)),
                 lambda: gated_ff(x, w[0], c(15, 8), w[2]), lambda: gated_ff(x[:, ::2], *w),
                 lambda: gated_ff(x, w[0].T.contiguous().T, w[1], w[2]),
                 lambda: gated_ff_bwd(x, *w, c(5, 8)), lambda: gated_ff_bwd(x, *w, c(4, 8), act=""),
                 lambda: gated_ff_bwd(x, *w, c(4, 8), kept=c(3, dtype=torch.uint8)),
                 lambda: adapted_linear_bwd(**ok, dy=c(4, 9)),
                 lambda: adapted_linear_bwd(**ok, dy=c(4, 8), kept=c(3, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            call()
    assert torch.cuda.current_device() == 0


def test_pair_wait_selftest_rejects_bad_budget():
    for budget in (0, 2_000_000_001):
        with pytest.raises(L.AtomError):
            L.call("atom_pair_wait_selftest", budget, None)


@pytest.mark.gpu
def test_expired_pair_wait_is_reported_and_cleared():
    """A product's bounded wait gives up, records its code, and the context stays usable."""
    st, code = L.stream_ptr(), ctypes.c_int(-1)
    L.call("atom_device_error", ctypes.byref(code), st)
    L.call("atom_pair_wait_selftest", 2_000_000, st)          # ~1 ms
    L.call("atom_device_error", ctypes.byref(code), st)
    assert code.value == 9
    L.call("atom_device_error", ctypes.byref(code), st)
    assert code.value == 0
    x = torch.ones(40, 64, device="cuda", dtype=torch.bfloat16)
    y = gated_ff(x, x, x, x.T.contiguous(), act="sigmoid")
    assert torch.equal(y, torch.full_like(y, float(y[0, 0])))
