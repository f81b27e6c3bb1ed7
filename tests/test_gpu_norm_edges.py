"""GPU: rms_norm's backward pass at the ends of its tensors, against 64 bits."""
import numpy as np
import pytest

import _lm_ref as R
from test_gpu_norm import inputs, within
from vectorcore_b200 import backend as B

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [33, 131, 1030, 2047, 5003, 8189])
@pytest.mark.parametrize("spare", [0, 1, 2, 3])
def test_the_last_row_of_odd_lengths(backend, cols, spare):
    """The last row's columns past its last whole 16 bytes come another way than
    the others. The tensors end inside a larger buffer of NaN, so nothing beyond
    their end may be used, and the last row's gradients are by far the largest:
    a column lost there shows in dw. Every residue of the rows modulo 4."""
    rows = (4 * 148 * 16 if cols < 1000 else 4 * 148 * 4) + spare
    rng, x, _, w = inputs(rows, cols, 5)
    gy, gh = (rng.normal(size=(rows, cols)).astype(np.float32) for _ in range(2))
    gy[-1] *= 1e3
    at, keep = {}, []
    for name, v in (("h", x), ("gy", gy), ("gh", gh)):
        keep.append(backend.upload(np.concatenate([v.ravel(), np.full(64, np.nan, np.float32)])))
        at[name] = B.CudaStorage.borrow(keep[-1].ptr, v.size)
    dw_ = backend.upload(w)
    _, _, rstd = backend.rms_norm(at["h"], dw_, rows, cols)
    edh, edw, bdh, bdw = R.rms_norm_backward(x, w, 1e-6, gy, gh)
    for _ in range(3):
        dh, dw = backend.rms_norm_backward(at["h"], dw_, rstd, at["gy"], rows, cols, gh=at["gh"])
        within(backend.download(dh).reshape(rows, cols), edh, bdh, "dh")
        within(backend.download(dw), edw, bdw, "dw")
