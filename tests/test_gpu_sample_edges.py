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
