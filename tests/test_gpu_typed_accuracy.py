"""Where the typed operators could lose what the definition keeps."""
import pytest
import torch

import test_gpu_adapters as ad
from tt_atom import _lib as L

pytestmark = pytest.mark.gpu


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
