"""Where the typed operators end: alignments that a kernel would fault on are refused on the host, before
any work, and the largest sizes that the header names are taken."""
import ctypes

import pytest
import torch

from tt_atom import _lib as L

P = ctypes.c_void_p(1 << 20)      # never read: every call here is refused on the host
ODD = [ctypes.c_void_p((1 << 20) + k) for k in (2, 16, 128)]


def refused(words, name, *args):
    code, message = getattr(L.lib(), name)(*args), L.last_error()
    assert code == 1 and words in message, (code, message)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("odd", ODD, ids=lambda p: str(p.value & 255))
def test_workspace_and_kept_have_to_be_aligned(odd, dtype):
    n = 1 << 40
    for M, ws, kept in ((40, odd, P), (40, P, odd), (4, odd, None)):
        refused("256-byte", "atom_gated_ff_fwd", dtype, P, 8, M, 8, 16, 8, P, P, P, 0, P, 8, kept, ws, n,
                None)
        refused("256-byte", "atom_gated_ff_bwd", dtype, P, 8, M, 8, 16, 8, P, P, P, 0, P, 8, kept, P, 8,
                P, P, P, ws, n, None)
        refused("256-byte", "atom_adapted_linear_fwd", dtype, P, 8, M, 8, 8, P, P, P, P, 2, 8, P, P, 2, P,
                8, kept, ws, n, None)
        refused("256-byte", "atom_adapted_linear_bwd", dtype, P, 8, M, 8, 8, P, P, P, P, 2, 8, P, P, 2, P,
                8, kept, P, 8, P, P, ws, n, None)


@pytest.mark.parametrize("n, R, nreq, fits", [
    (1 << 14, 8, 1 << 22, True), ((1 << 14) + 1, 8, 5, False), (5, 8, (1 << 22) + 1, False),
    # (T + requests) ceil(R / 16) + 4 T < 2^25 - 4 with T = 1
    (5, 128, (1 << 22) - 3, True), (5, 128, (1 << 22) - 2, False)])
def test_the_most_adapters_and_requests(n, R, nreq, fits):
    size = (L.c_size_t * 3)()
    code = L.lib().atom_adapted_linear_bytes(1, 40, 8, 8, n, R, nreq, size)
    assert code == (0 if fits else 1)
    assert fits or "2^14 adapters, 2^22 requests" in L.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("M", [4, 60])
def test_as_many_adapters_as_there_may_be(M, t):
    import test_gpu_adapters as ad
    n = 1 << 14
    args = ad.make([1] * M, [(n - 1 - 37 * i) % n for i in range(M)], n, 128, 8, 16, t, seed=M)
    ad.both(args)


@pytest.mark.gpu
def test_a_wait_that_ran_out_raises_where_results_are_read_back():
    import tt_atom
    from tt_atom.feedforward import gated_ff
    x = torch.ones(40, 64, device="cuda", dtype=torch.bfloat16)
    gated_ff(x, x, x, x.T.contiguous())
    tt_atom.check_device()
    L.call("atom_pair_wait_selftest", 2_000_000, L.stream_ptr())          # ~1 ms
    gated_ff(x, x, x, x.T.contiguous())
    with pytest.raises(RuntimeError, match="bounded device-side wait"):
        tt_atom.check_device()
    y = gated_ff(x, x, x, x.T.contiguous())
    tt_atom.check_device()
    assert (y == y[0, 0]).all()
