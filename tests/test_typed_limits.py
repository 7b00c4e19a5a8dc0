"""Where the typed operators' C entries end: alignments that a kernel would fault on are refused on the
host, before any work."""
import ctypes

import pytest

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
