"""The language-model operators' host side: argument checks that need no GPU,
borrowed storages, and the 64-bit references themselves (the gradient against
differences, the sampling rules against a direct walk)."""
import numpy as np
import pytest

import _lm_ref as R
from vectorcore_b200 import backend as B


def fake(elements, dtype=np.float32):
    return B.CudaStorage.borrow(1 << 20, elements, np.dtype(dtype))


@pytest.fixture(scope="module")
def be():
    return B.CudaBackend.instance()


def test_borrowed_storage_is_a_storage_and_frees_nothing():
    s = fake(12, np.int8)
    assert isinstance(s, B.CudaStorage) and (s.ptr, s.size, s.nbytes, s.version) == (1 << 20, 12, 12, 0)
    s.bump_version()
    assert s.version == 1
    del s  # an attempt to free the fake address would fail in the library


def test_pitch():
    assert [B.q8_pitch(k) for k in (0, 1, 15, 16, 17, 4100)] == [0, 16, 16, 16, 32, 4112]


def test_short_storages_are_refused(be):
    ok, short, w = fake(60), fake(59), fake(10)
    for kw in ({"x": short}, {"residual": short}, {"weight": fake(9)}, {"out": (ok, short, fake(6))},
               {"out": (ok, ok, fake(5))}, {"x_stride": 11}, {"residual_stride": 12, "residual": ok}):
        a = {"x": ok, "weight": w, "residual": None, "out": (ok, ok, fake(6)), **kw}
        with pytest.raises(IndexError):
            be.rms_norm(a.pop("x"), a.pop("weight"), 6, 10, **a)
    with pytest.raises(IndexError):
        be.rms_norm_backward(ok, w, fake(5), ok, 6, 10, out=(ok, w))
    with pytest.raises(IndexError):
        be.rms_norm_q8(ok, w, 6, 10, out=(fake(95, np.int8), fake(6), None))
    with pytest.raises(IndexError):
        be.quantize_q8(short, 6, 10, out=(fake(96, np.int8), fake(6)))
    a, b, sa, sb = fake(2 * 32, np.int8), fake(3 * 32, np.int8), fake(2), fake(3)
    with pytest.raises(IndexError):
        be.matmul_q8(a, sa, b, sb, 2, 3, 33, out=fake(6))
    with pytest.raises(IndexError):
        be.matmul_q8(a, sa, b, sb, 2, 3, 32, out=fake(5))
    with pytest.raises(IndexError):
        be.matmul_q8(a, sa, b, sb, 2, 3, 32, b_pitch=48, out=fake(6))
    with pytest.raises(IndexError):
        be.sample(ok, fake(59), 6, 10, out=(fake(6, np.int64), fake(6)))
    with pytest.raises(IndexError):
        be.sample(ok, ok, 6, 10, row_stride=11, out=(fake(6, np.int64), fake(6)))
    with pytest.raises(IndexError):
        be.sample(ok, ok, 6, 10, temperature=fake(5), out=(fake(6, np.int64), fake(6)))


def test_other_types_are_refused(be):
    ok = fake(60)
    with pytest.raises(ValueError):
        be.rms_norm(fake(60, np.int64), fake(10), 6, 10, out=(ok, None, None))
    with pytest.raises(ValueError):
        be.matmul_q8(ok, fake(2), fake(60, np.int8), fake(3), 2, 3, 10, out=fake(6))
    with pytest.raises(ValueError):
        be.sample(ok, ok, 6, 10, top_k=fake(6), out=(fake(6, np.int64), fake(6)))
    with pytest.raises(ValueError):
        be.sample(ok, ok, 6, 10, out=(fake(6), fake(6)))
    with pytest.raises(ValueError):
        be.rms_norm(ok, fake(10), -1, 10, out=(ok, None, None))


def test_norm_gradient_against_differences():
    rng = np.random.default_rng(3)
    h, w = rng.normal(size=(5, 9)), rng.normal(size=9)
    gy, gh = rng.normal(size=(5, 9)), rng.normal(size=(5, 9))

    def loss(h, w):
        return (R.rms_norm(h, w, 1e-3)[0] * gy).sum() + (h * gh).sum()

    dh, dw, _, _ = R.rms_norm_backward(h, w, 1e-3, gy, gh)
    step = 1e-5
    for i in np.ndindex(h.shape):
        e = np.zeros_like(h)
        e[i] = step
        assert abs((loss(h + e, w) - loss(h - e, w)) / (2 * step) - dh[i]) < 1e-7
    for j in range(9):
        e = np.zeros_like(w)
        e[j] = step
        assert abs((loss(h, w + e) - loss(h, w - e)) / (2 * step) - dw[j]) < 1e-7


def test_sampling_rules_against_a_walk():
    rng = np.random.default_rng(4)
    for trial in range(200):
        n = int(rng.integers(1, 12))
        x = rng.integers(-3, 4, n).astype(np.float32)
        x[rng.random(n) < 0.2] = -np.inf
        k, p, least = int(rng.integers(0, n + 2)), float(rng.choice([1.0, 0.3, 0.8])), float(rng.choice([0.0, 0.2]))
        noise = rng.exponential(size=n).astype(np.float32)
        r = R.Row(x, noise, 0.7, k, p, least)
        if not r.play.any():
            continue
        alive = sorted(np.flatnonzero(r.play), key=lambda i: (-x[i], i))
        w = {i: np.exp((float(x[i]) - float(x[alive[0]])) / float(np.float32(0.7))) for i in alive}
        if k > 0:
            alive = alive[:k]
        mass, run, left = sum(w[i] for i in alive), 0.0, []
        for i in alive:
            if left and not (p >= 1 or run < float(np.float32(p)) * mass):
                break
            left.append(i)
            run += w[i]
        left = [i for i in left if i == left[0] or w[i] >= float(np.float32(least))]
        # equal weights can sit on a limit: the walk's set lies between the two
        sure, may = set(r.order[r.sure]), set(r.order[r.may])
        assert sure <= set(left) <= may, (x, k, p, least)
        token = max(left, key=lambda i: (w[i] / float(noise[i]), -i))
        r.check(int(token), np.log(w[token]) - np.log(r.total))
