"""GPU: sampling at the ends of its ranges, against the rules in 64 bits
(_lm_ref.Row)."""
import numpy as np
import pytest

import _lm_ref as R
from test_gpu_sample import draw, run

pytestmark = pytest.mark.gpu

COLD = [1e-45, 1e-39, 4.2e-39, 4.3e-39, 1.1e-38, 2.0 ** -126, 1e-37]


@pytest.mark.parametrize("filters", [{}, {"min_p": 0.05}, {"min_p": 1.0}, {"top_k": 5, "top_p": 0.9}, {"top_p": 0.9},
                                     {"top_k": 700, "top_p": 0.9}, {"top_p": 0.7, "min_p": 0.01}])
@pytest.mark.parametrize("kind", ["normal", "few", "flat"])
@pytest.mark.parametrize("vocab", [5, 1000, 20000])
def test_temperatures_near_zero(backend, vocab, kind, filters):
    """Down to the smallest float the largest logits share the row; 160 rows
    reach the other launch shapes too."""
    for rows in (len(COLD), 160):
        rng = np.random.default_rng(vocab + rows)
        settings = [{"temperature": COLD[i % len(COLD)], **filters} for i in range(rows)]
        x = draw(rng, rows, vocab, kind)
        noise = rng.exponential(size=x.shape).astype(np.float32)
        token, logprob = run(backend, x, noise, settings)
        for i in range(0, rows, 1 if rows < 20 else 9):
            R.Row(x[i], noise[i], **settings[i]).check(int(token[i]), float(logprob[i]), f"row {i} {settings[i]}")


def test_temperatures_below_the_normal_floats_count_as_the_smallest(backend):
    """Shown by logits whose distances are as small as the temperature."""
    rng = np.random.default_rng(1)
    x = (rng.normal(size=(6, 500)) * 2.0 ** -126).astype(np.float32)
    noise = rng.exponential(size=x.shape).astype(np.float32)
    cold = [1e-45, 1e-40, 4e-39, 2.0 ** -127, 2.0 ** -126, 2.0 ** -125]
    for filters in ({}, {"min_p": 0.3}, {"top_k": 9}):
        token, logprob = run(backend, x, noise, [{"temperature": t, **filters} for t in cold])
        for i, t in enumerate(cold):
            R.Row(x[i], noise[i], max(t, 2.0 ** -126), **filters).check(int(token[i]), float(logprob[i]), f"{t} {filters}")


@pytest.mark.parametrize("steps", [1, 5, 7, 11, 13, 17, 23, 29])
def test_a_maximum_that_grows_all_along_a_long_row(backend, steps):
    """The longest rows, one CTA a row, every batch of classes above the one
    before it. An early class and a late one are 3e-6 apart in the race, where
    the definition's e^d (2^-22), division and the noise's own rounding (2^-24
    each) leave 4e-7; d is exact."""
    rows, vocab, batch = 149, 1 << 23, 4096
    batches = vocab // batch
    step = steps * 2.0 ** -11  # all distances exact
    x = (np.arange(vocab) // batch * step).astype(np.float32)
    up, early, late = backend.upload, 40, vocab - batch + 40
    dx = up(x)
    total = batch * np.exp(-step * np.arange(batches)).sum()
    for winner, factor in ((early, 1 - 3e-6), (late, 1 + 3e-6)):
        noise = np.full(vocab, 1e9, np.float32)
        noise[late], noise[early] = 1.0, np.exp(-step * (batches - 1)) * factor
        token, logprob = backend.sample(dx, up(noise), rows, vocab, row_stride=0, noise_stride=0)
        assert (backend.download(token) == winner).all()
        # rounding as in _lm_ref.Row.check, no distance above the longest
        want = (step * (batches - 1) if winner == early else 0.0) * -1.0 - np.log(total)
        worst = step * (batches - 1)
        bound = R.U * (8 * worst + 8 + 4 * np.log(total) + abs(want))
        assert (np.abs(backend.download(logprob) - want) <= bound).all()


@pytest.mark.parametrize("vocab", [10, 300, 4097, 20000, 50000])
@pytest.mark.parametrize("setting", [{"temperature": 0.0}, {}, {"top_k": 1}, {"top_k": 2}, {"top_k": 600},
                                     {"top_k": 600, "top_p": 0.4}, {"top_p": 0.4}, {"min_p": 0.5},
                                     {"top_p": 0.4, "min_p": 0.5}])
def test_infinity_counts_as_the_largest_float(backend, vocab, setting):
    """Equal ones are ordered by index alone, near to each other and far apart."""
    rng = np.random.default_rng(vocab)
    big, rows = np.finfo(np.float32).max, 6
    x = rng.normal(size=(rows, vocab)).astype(np.float32)
    x[0, 0], x[0, -1] = big, np.inf
    x[1, 0], x[1, -1] = np.inf, big
    x[2, 1:3] = np.inf, big
    x[3, -3:-1] = big, np.inf
    x[4, ::2], x[4, 1::2] = big, np.inf
    x[5, ::3] = np.where(rng.random(x[5, ::3].size) < 0.5, big, np.inf)
    noise = rng.exponential(size=x.shape).astype(np.float32)
    for rows_again in (1, 30):  # 180 rows take the other launch shapes
        xs, es = np.tile(x, (rows_again, 1)), np.tile(noise, (rows_again, 1))
        token, logprob = run(backend, xs, es, [setting] * len(xs))
        for i in range(rows):
            R.Row(np.minimum(x[i], big), noise[i], **setting).check(int(token[i]), float(logprob[i]), f"row {i}")
        assert (token.reshape(-1, rows) == token[:rows]).all()
