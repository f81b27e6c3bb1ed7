"""GPU: sampling of more rows than SMs, against the rules in 64 bits
(_lm_ref.Row): small CTAs for short rows, one CTA a row that shares its SM, and
clusters for long filtered ones."""
import numpy as np
import pytest

import _lm_ref as R
from test_gpu_sample import SETTINGS, draw, run

pytestmark = pytest.mark.gpu

FILTERS = [{}, {"top_k": 50, "top_p": 0.95}, {"top_p": 0.98}, {"top_p": 0.6}, {"top_p": 0.9, "min_p": 0.001},
           {"min_p": 0.02}, {"temperature": 0.0}, {"top_k": 700, "top_p": 0.8}, {"top_k": 6000}, {"min_p": 1e-6}]


def verify(backend, x, noise, settings, look):
    """The rows in `look` by the rules, the rest by being the same twice."""
    first = run(backend, x, noise, settings)
    for i in look:
        R.Row(x[i], noise[i], **settings[i]).check(int(first[0][i]), float(first[1][i]), f"row {i} {settings[i]}")
    again = run(backend, x, noise, settings)
    assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1], equal_nan=True)


@pytest.mark.parametrize("kind", ["normal", "flat", "few"])
@pytest.mark.parametrize("vocab", [6, 1000, 2500, 4097, 16384, 16385, 50257])
def test_every_setting(backend, vocab, kind):
    rows = 12 * len(SETTINGS)
    rng = np.random.default_rng(vocab)
    x = draw(rng, rows, vocab, kind)
    noise = rng.exponential(size=x.shape).astype(np.float32)
    x[5::7, rng.integers(0, vocab, vocab // 3)] = -np.inf  # masked, and rows with nothing left
    x[8] = np.nan
    look = range(rows) if vocab < 5000 else [*range(len(SETTINGS)), *range(len(SETTINGS), rows, 19)]
    verify(backend, x, noise, [SETTINGS[i % len(SETTINGS)] for i in range(rows)], look)


@pytest.mark.parametrize("kind", ["normal", "few"])
@pytest.mark.parametrize("vocab", [4097, 12001, 16384])
def test_lists_that_overflow_in_small_ctas(backend, vocab, kind):
    """min-p that leaves more classes than a CTA lists, k beyond both lists."""
    rng = np.random.default_rng(vocab)
    rows = 30 * len(FILTERS)
    settings = [{**FILTERS[i % len(FILTERS)], **({"min_p": 1e-6, "top_p": 0.3} if i % 7 == 3 else {})} for i in range(rows)]
    x = draw(rng, rows, vocab, kind)
    verify(backend, x, rng.exponential(size=x.shape).astype(np.float32), settings, range(0, rows, 3))


@pytest.mark.parametrize("rows,vocab", [(160, 100003), (150, 128000), (149, 400001)])
def test_clusters_of_long_rows(backend, rows, vocab):
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal(size=(rows, vocab), dtype=np.float32) * 2
    x[np.arange(rows), rng.integers(0, vocab, rows)] += 8
    noise = rng.standard_exponential(size=x.shape, dtype=np.float32)
    verify(backend, x, noise, [FILTERS[i % len(FILTERS)] for i in range(rows)], [*range(len(FILTERS)), rows - 1, rows - 3])


@pytest.mark.parametrize("rows,vocab", [(300, 50), (300, 16000), (200, 30000), (149, 200000)])
def test_no_settings_at_all(backend, rows, vocab):
    rng = np.random.default_rng(rows)
    x = rng.standard_normal(size=(rows, vocab), dtype=np.float32) * 3
    noise = rng.standard_exponential(size=x.shape, dtype=np.float32)
    up = backend.upload
    token, logprob = (backend.download(v) for v in backend.sample(up(x), up(noise), rows, vocab))
    for i in range(0, rows, 11):
        R.Row(x[i], noise[i]).check(int(token[i]), float(logprob[i]), f"row {i}")
