"""GPU: the C++ forms of the language-model operators against 64 bits, and
their refusals on the device's own storages."""
import ctypes

import numpy as np
import pytest

import _host_forms as H
import _lm_ref as R
from vectorcore_b200 import backend as B
from vectorcore_b200.build import library_path

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib(backend, tmp_path_factory):
    return H.build(tmp_path_factory.mktemp("forms"), library_path())


def at(a):
    return None if a is None else a.ctypes.data_as(ctypes.c_void_p)


def close(got, want, bound):
    return (np.abs(got.astype(np.float64) - want) <= bound).all()


@pytest.mark.parametrize("rows,cols", [(5, 33), (64, 256)])
@pytest.mark.parametrize("full", [True, False])
def test_norm(lib, rows, cols, full):
    rng = np.random.default_rng(cols)
    x, r, gy, gh = (rng.normal(size=(rows, cols)).astype(np.float32) for _ in range(4))
    w = rng.normal(size=cols).astype(np.float32)
    if not full:
        r = gh = None
    y, h, dh = (np.zeros((rows, cols), np.float32) for _ in range(3))
    rstd, dw = np.zeros(rows, np.float32), np.zeros(cols, np.float32)
    n = ctypes.c_size_t
    assert lib.form_rms_norm(at(x), at(r), at(w), n(rows), n(cols), ctypes.c_float(1e-5), at(gy), at(gh), at(y), at(h),
                             at(rstd), at(dh), at(dw)) == 0
    stream = x if r is None else x + r
    assert np.array_equal(h, stream if full else np.zeros_like(h))
    want, s = R.rms_norm(stream, w, 1e-5)
    edh, edw, bdh, bdw = R.rms_norm_backward(stream, w, 1e-5, gy, gh)
    assert close(y, want, R.rms_norm_bound(want)) and close(rstd, s, 6 * R.U * s)
    assert close(dh, edh, bdh) and close(dw, edw, bdw)


@pytest.mark.parametrize("rows,cols,n", [(3, 33, 40), (40, 256, 130)])
@pytest.mark.parametrize("form", ["norm and residual", "norm", "rows"])
def test_8_bit_rows_and_their_product(lib, rows, cols, n, form):
    rng = np.random.default_rng(rows)
    x, r = (rng.normal(size=(rows, cols)).astype(np.float32) for _ in range(2))
    b, w, bias = (rng.normal(size=s).astype(np.float32) for s in ((n, cols), cols, n))
    if form != "norm and residual":
        r = None
    if form == "rows":
        w = bias = None
    pitch = B.q8_pitch(cols)
    q, scale = np.zeros((rows, pitch), np.int8), np.zeros(rows, np.float32)
    h, out = np.zeros((rows, cols), np.float32), np.zeros((rows, n), np.float32)
    size = ctypes.c_size_t
    assert lib.form_q8(at(x), at(r), at(w), size(rows), size(cols), at(b), size(n), at(bias), at(q), at(scale), at(h),
                       at(out)) == 0
    stream = x if r is None else x + r
    if r is not None:
        assert np.array_equal(h, stream)
    eq, step = R.q8(stream if w is None else stream * w)
    if w is not None:
        step = step * R.rms_norm(stream, w, 1e-6)[1]
    assert np.array_equal(q[:, :cols], eq) and not q[:, cols:].any() and close(scale, step, 10 * R.U * step)
    qb, step_b = R.q8(b)
    product = (eq.astype(np.int64) @ qb.astype(np.int64).T) * (step[:, None] * step_b)
    want = product if bias is None else product + bias
    # scales: 10 and 3 roundings, the product and the bias 4
    assert close(out, want, 20 * R.U * (np.abs(product) + np.abs(want)) + 1e-44)


@pytest.mark.parametrize("settings", [{}, {"temperature": 0.7, "top_k": 9, "top_p": 0.8, "min_p": 0.01}])
def test_sample(lib, settings):
    rng = np.random.default_rng(7)
    rows, vocab = 9, 1000
    x, noise = rng.normal(0, 2, size=(rows, vocab)).astype(np.float32), rng.exponential(size=(rows, vocab)).astype(np.float32)
    of = [None if name not in settings else np.full(rows, settings[name], np.int64 if name == "top_k" else np.float32)
          for name in ("temperature", "top_k", "top_p", "min_p")]
    token, logprob, n = np.zeros(rows, np.int64), np.zeros(rows, np.float32), ctypes.c_size_t
    assert lib.form_sample(at(x), at(noise), n(rows), n(vocab), *map(at, of), at(token), at(logprob)) == 0
    for i in range(rows):
        R.Row(x[i], noise[i], **settings).check(int(token[i]), float(logprob[i]), f"row {i}")


def test_short_storages_and_other_types_are_refused(lib):
    assert H.refusals(lib) == H.REFUSALS
