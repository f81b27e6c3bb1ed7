"""GPU: the 8-bit product with scales whose product is no normal float, though
the results are floats, against 64 bits."""
import numpy as np
import pytest

import _lm_ref as R
from test_gpu_matmul_q8 import matrix
from vectorcore_b200 import backend as B

pytestmark = pytest.mark.gpu

# every kernel: weights to registers, a tile shared by a cluster, one CTA a tile, pairs
SIZES = [(3, 40, 64), (14, 100, 300), (40, 200, 5000), (200, 9000, 300), (300, 2000, 640), (300, 20000, 100), (70, 20001, 130)]


@pytest.mark.parametrize("m,n,k", SIZES + [(5, 7, 0)])
@pytest.mark.parametrize("ea,eb", [(-66, -66), (-100, -45), (-75, -75), (-149, 10), (64, 64), (100, 90), (-149, -149)])
def test_products_of_scales_outside_the_floats(backend, m, n, k, ea, eb):
    rng = np.random.default_rng(m + n + k)
    pitch, up = max(16, B.q8_pitch(k)), backend.upload
    a, b = matrix(rng, m, k, pitch), matrix(rng, n, k, pitch)
    a[m // 2] = 0  # sums of 0 stay 0
    b[n // 3] = 0
    sa, sb = (rng.uniform(1, 2, m) * 2.0 ** ea).astype(np.float32), (rng.uniform(1, 2, n) * 2.0 ** eb).astype(np.float32)
    sa[0], sb[0] = 1.0, 2.0 ** -20  # ordinary ones beside them
    sa[1] = 0.0
    bias = rng.normal(size=n).astype(np.float32) if ea == eb else None
    out = backend.matmul_q8(up(a, np.int8), up(sa), up(b, np.int8), up(sb), m, n, k,
                            bias=None if bias is None else up(bias), a_pitch=pitch, b_pitch=pitch)
    got = backend.download(out).reshape(m, n).astype(np.float64)
    want, bound = R.matmul_q8(a[:, :k], sa, b[:, :k], sb, bias)
    far = np.abs(want) > np.finfo(np.float32).max  # too large for the result too
    assert (got[far] == np.sign(want[far]) * np.inf).all()
    assert not got[1].any() if bias is None else (got[1] == bias).all()
    # the smallest float is the step of what lies below the normal ones
    assert (np.abs(got - want)[~far] <= (bound + 2.0 ** -149)[~far]).all()


@pytest.mark.parametrize("m,n,k", SIZES)
def test_odd_scales_reach_their_own_outputs(backend, m, n, k):
    rng = np.random.default_rng(m)
    pitch, up = B.q8_pitch(k), backend.upload
    a, b = matrix(rng, m, k, pitch), matrix(rng, n, k, pitch)
    sa, sb = rng.uniform(1, 2, m).astype(np.float32), rng.uniform(1, 2, n).astype(np.float32)
    sa[0], sb[1], sb[2] = np.nan, np.inf, 0.0
    out = backend.download(backend.matmul_q8(up(a, np.int8), up(sa), up(b, np.int8), up(sb), m, n, k)).reshape(m, n)
    with np.errstate(invalid="ignore"):
        want, bound = R.matmul_q8(a[:, :k], sa, b[:, :k], sb, None)
    ordinary = np.isfinite(want)
    assert ordinary.sum() == (m - 1) * (n - 1)
    assert np.array_equal(out[~ordinary], want[~ordinary].astype(np.float32), equal_nan=True)
    assert (np.abs(out[ordinary] - want[ordinary]) <= bound[ordinary]).all()
