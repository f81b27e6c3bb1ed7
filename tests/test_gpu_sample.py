"""GPU: the next token from logits with temperature, top-k, top-p and min-p,
against the same rules in 64 bits (_lm_ref.Row: a class within rounding of a
filter's limit, or of the race's winner, may go either way)."""
import numpy as np
import pytest

import _lm_ref as R
from vectorcore_b200 import _abi

pytestmark = pytest.mark.gpu

SETTINGS = [{}, {"temperature": 0.7}, {"top_k": 1}, {"top_k": 5}, {"top_k": 50, "top_p": 0.9}, {"top_p": 0.5},
            {"top_p": 0.98, "temperature": 1.3}, {"min_p": 0.05}, {"top_k": 40, "top_p": 0.95, "min_p": 0.01},
            {"top_p": 0.0}, {"temperature": 0.0}, {"top_k": 1 << 40}, {"min_p": 5.0}, {"temperature": 1e-3},
            {"temperature": 1e30}, {"temperature": float("inf")}, {"temperature": float("nan")}, {"top_p": float("nan")},
            {"min_p": float("nan")}, {"top_k": -3, "top_p": 0.999999}, {"top_k": 700, "top_p": 0.3}]


def run(be, x, noise, settings, stride=None, noise_stride=None, vocab=None):
    rows = len(settings)
    up = be.upload
    column = lambda name, off, dtype: up(np.array([s.get(name, off) for s in settings], dtype))  # noqa: E731
    vocab = x.shape[1] if vocab is None else vocab
    token, logprob = be.sample(up(x), up(noise), rows, vocab, temperature=column("temperature", 1.0, np.float32),
                               top_k=column("top_k", 0, np.int64), top_p=column("top_p", 1.0, np.float32),
                               min_p=column("min_p", 0.0, np.float32), row_stride=stride, noise_stride=noise_stride)
    return be.download(token), be.download(logprob)


def verify(be, x, noise, settings, **kw):
    token, logprob = run(be, x, noise, settings, **kw)
    vocab = kw.get("vocab") or x.shape[1]
    for i, s in enumerate(settings):
        R.Row(x[i, :vocab], noise[i, :vocab], **s).check(int(token[i]), float(logprob[i]), f"row {i} {s}")
    return token


def draw(rng, rows, vocab, kind):
    if kind == "normal":
        x = rng.normal(0, 2, size=(rows, vocab))
    elif kind == "peaked":
        x = rng.normal(0, 1, size=(rows, vocab))
        x[np.arange(rows), rng.integers(0, vocab, rows)] += 12
    elif kind == "flat":  # every class equal: only the order by index decides
        x = np.full((rows, vocab), 1.5)
    elif kind == "few":  # long runs of equal logits
        x = rng.integers(-2, 3, size=(rows, vocab)).astype(float)
    elif kind == "narrow":  # the same leading bits for all
        x = 100 + rng.normal(0, 1e-4, size=(rows, vocab))
    else:  # wide: most weights vanish
        x = rng.normal(0, 60, size=(rows, vocab))
    return x.astype(np.float32)


@pytest.mark.parametrize("kind", ["normal", "peaked", "flat", "few", "narrow", "wide"])
@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 64, 1000, 4097, 32000])
def test_every_setting(backend, vocab, kind):
    rng = np.random.default_rng(vocab + len(kind))
    x = draw(rng, len(SETTINGS), vocab, kind)
    verify(backend, x, rng.exponential(size=x.shape).astype(np.float32), SETTINGS)


@pytest.mark.parametrize("vocab", [50257, 65536, 128000, 200001, 600000])
def test_long_rows(backend, vocab):
    rng = np.random.default_rng(vocab)
    settings = [{}, {"top_k": 50, "top_p": 0.95}, {"top_p": 0.98}, {"top_p": 0.9, "min_p": 0.001}, {"temperature": 0.0}]
    for kind in ("normal", "flat", "few"):
        x = draw(rng, len(settings), vocab, kind)
        verify(backend, x, rng.exponential(size=x.shape).astype(np.float32), settings)


@pytest.mark.parametrize("vocab", [7, 1000, 40000])
def test_masked_rows(backend, vocab):
    """-inf and NaN logits are never drawn; +inf ones share the row; a row with
    nothing left says so."""
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, 2, size=(8, vocab)).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, :] = -np.inf
    x[2, vocab // 2] = -5.0
    x[3, rng.random(vocab) < 0.5] = -np.inf
    x[3, 0] = 0.25
    x[4, rng.random(vocab) < 0.3] = np.nan
    x[4, 1] = 0.5
    x[5, [1, vocab - 1]] = np.inf
    x[6] = np.finfo(np.float32).min
    x[7] = np.where(np.arange(vocab) % 2, np.float32(0.0), np.float32(-0.0))
    for s in ({}, {"top_k": 3}, {"top_p": 0.6}, {"top_k": 4, "top_p": 0.7, "min_p": 0.1}, {"temperature": 0.0}):
        noise = rng.exponential(size=x.shape).astype(np.float32)
        token = verify(backend, x, noise, [s] * 8)
        assert token[0] == token[1] == -1 and token[2] == vocab // 2
        assert token[5] in (1, vocab - 1)
        if s.get("temperature", 1.0) == 0.0:
            assert token[6] == token[7] == 0 and token[5] == 1


def test_strides_and_short_rows_of_a_long_buffer(backend):
    rng = np.random.default_rng(5)
    settings = [{"top_k": 9}, {"top_p": 0.8}, {}, {"temperature": 0.0}, {"min_p": 0.1}]
    for vocab, ls, ns in ((1000, 1003, 1000), (1000, 1024, 1001), (4099, 4100, 4103)):
        x = np.full((5, ls), 50, np.float32)  # past the row: larger than everything in it
        x[:, :vocab] = rng.normal(size=(5, vocab))
        noise = np.zeros((5, ns), np.float32)
        noise[:, :vocab] = rng.exponential(size=(5, vocab))
        verify(backend, x, noise, settings, stride=ls, noise_stride=ns, vocab=vocab)


def test_odd_noise(backend):
    """A zero wins the race, an infinity and a NaN lose it, also in the only
    class that is left."""
    x = np.zeros((4, 100), np.float32)
    noise = np.ones((4, 100), np.float32)
    noise[0, 70] = 0.0
    noise[1] = np.inf
    noise[1, 30] = 3.0
    noise[2] = np.nan
    noise[2, 99] = 8.0
    noise[3] = np.nan
    token, logprob = run(backend, x, noise, [{}] * 4)
    assert token.tolist() == [70, 30, 99, 0]
    assert np.allclose(logprob, -np.log(100), rtol=1e-6)


def test_draws_follow_the_distribution(backend):
    """65536 draws from 6 classes: each count within 6 standard deviations."""
    rng = np.random.default_rng(11)
    logits = np.array([1.0, 0.0, -1.0, 2.0, -np.inf, 0.5], np.float32)
    rows = 65536
    x, noise = np.tile(logits, (rows, 1)), rng.exponential(size=(rows, 6)).astype(np.float32)
    for s, left in (({"temperature": 0.8}, range(6)), ({"top_k": 3}, (0, 3, 5)), ({"top_p": 0.7}, (0, 3))):
        token, _ = run(backend, x, noise, [s] * rows)
        w = np.where(np.isin(np.arange(6), list(left)), np.exp(logits.astype(float) / s.get("temperature", 1.0)), 0)
        p = w / w.sum()
        counts = np.bincount(token, minlength=6)
        assert (np.abs(counts - rows * p) <= 6 * np.sqrt(rows * p * (1 - p)) + 1e-9).all(), (s, counts, rows * p)


def test_settings_may_be_missing(backend):
    rng = np.random.default_rng(2)
    x, noise = (f(size=(3, 500)).astype(np.float32) for f in (rng.normal, rng.exponential))
    token, logprob = backend.sample(backend.upload(x), backend.upload(noise), 3, 500)
    token, logprob = backend.download(token), backend.download(logprob)
    for i in range(3):
        R.Row(x[i], noise[i]).check(int(token[i]), float(logprob[i]))
    assert backend.download(backend.sample(backend.allocate(0), backend.allocate(0), 0, 500)[0]).size == 0


def test_repeatable(backend):
    rng = np.random.default_rng(3)
    x = draw(rng, 20, 30000, "normal")
    noise = rng.exponential(size=x.shape).astype(np.float32)
    settings = [SETTINGS[i % len(SETTINGS)] for i in range(20)]
    first = run(backend, x, noise, settings)
    for _ in range(3):
        again = run(backend, x, noise, settings)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


def test_refusals(backend):
    f, i = backend.allocate(64), backend.allocate(64, np.int64)
    with pytest.raises(ValueError, match="at least one class"):
        backend.sample(f, f, 4, 0)
    with pytest.raises(OverflowError, match="2\\^23"):
        _abi.call("vc_cuda_sample", f.ptr, 1 << 24, f.ptr, 1 << 24, None, None, None, None, 1, (1 << 23) + 1, i.ptr, f.ptr)
    with pytest.raises(OverflowError, match="rows"):
        _abi.call("vc_cuda_sample", f.ptr, 8, f.ptr, 8, None, None, None, None, 1 << 40, 8, i.ptr, f.ptr)
    for gone in range(4):
        ptrs = [f.ptr, f.ptr, i.ptr, f.ptr]
        ptrs[gone] = None
        with pytest.raises(ValueError, match="null"):
            _abi.call("vc_cuda_sample", ptrs[0], 8, ptrs[1], 8, None, None, None, None, 4, 8, ptrs[2], ptrs[3])
