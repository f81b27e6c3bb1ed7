"""GPU: the operators together, as examples/next_token.py uses them -- the
norm trained through the device's cross-entropy, then norm, 8-bit head product
and sampling from one graph replay -- against 64 bits."""
import sys
from pathlib import Path

import numpy as np
import pytest

import _lm_ref as R

pytestmark = pytest.mark.gpu

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


@pytest.mark.parametrize("rows,cols,classes", [(64, 256, 1000), (3, 130, 5003)])
def test_example(backend, rows, cols, classes):
    import next_token

    r = next_token.main(rows, cols, classes)
    assert r["losses"][-1] < 0.9 * r["losses"][0]
    # the graph's logits: the 8-bit rule on the same stream and weights
    h = r["x"] + r["residual"]
    q, step = R.q8(h * r["weight"])
    _, rstd = R.rms_norm(h, r["weight"], 1e-6)
    qh, step_h = R.q8(r["head"])
    logits = (q.astype(np.int64) @ qh.astype(np.int64).T) * ((step * rstd)[:, None] * step_h)
    # scales: 10 and 3 roundings, the product 4
    assert (np.abs(r["logits"] - logits) <= 20 * R.U * np.abs(logits) + 1e-44).all()
    for i in range(rows):
        R.Row(r["logits"][i], r["noise"][i], 0.5, 20, 0.9).check(int(r["token"][i]), float(r["logprob"][i]), f"row {i}")
