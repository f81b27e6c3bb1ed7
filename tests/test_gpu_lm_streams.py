"""GPU: the language-model operators beside another library's work, on whatever
stream that library is using: use_stream follows it."""
import numpy as np
import pytest

import _lm_ref as R
from vectorcore_b200 import backend as B

pytestmark = pytest.mark.gpu


def test_on_the_owner_s_stream_of_the_moment(backend):
    torch = pytest.importorskip("torch")
    rows, cols, classes = 64, 1024, 5000
    gen = torch.Generator(device="cuda").manual_seed(0)
    base = torch.randn((rows, cols), device="cuda", generator=gen)
    weight = torch.rand(cols, device="cuda", generator=gen) + 0.5
    head = torch.randn((classes, cols), device="cuda", generator=gen)
    noise = torch.empty((rows, classes), device="cuda").exponential_(generator=gen)
    busy = torch.randn((4096, 4096), device="cuda", generator=gen)

    def st(t, dtype=np.float32):
        return B.CudaStorage.borrow(t.data_ptr(), t.numel(), np.dtype(dtype))

    def step(scale):
        """x comes late on torch's stream, and torch reads the results there."""
        backend.use_stream(torch.cuda.current_stream().cuda_stream)
        wait = busy
        for _ in range(4):
            wait = wait @ busy * 1e-2
        x = base * scale + 0 * wait.nan_to_num(0, 0, 0)[:rows, :cols].clamp(-1, 1)
        q, s, _ = backend.rms_norm_q8(st(x), st(weight), rows, cols)
        hq, hs = backend.quantize_q8(st(head), classes, cols)
        logits = torch.empty((rows, classes), device="cuda")
        backend.matmul_q8(q, s, hq, hs, rows, classes, cols, out=st(logits))
        token, logprob = torch.empty(rows, dtype=torch.int64, device="cuda"), torch.empty(rows, device="cuda")
        backend.sample(st(logits), st(noise), rows, classes, out=(st(token, np.int64), st(logprob)))
        # torch reads them, and keeps its memory until the stream is done with it
        return (token + 0, logprob * 1, logits * 1), (x, logits, token, logprob)

    streams, results, held = [torch.cuda.default_stream(), torch.cuda.Stream(), torch.cuda.Stream()], [], []
    try:
        torch.cuda.synchronize()
        for turn in range(6):
            with torch.cuda.stream(streams[turn % 3]):
                kept, record = step(1.0 + turn % 2)
                results.append(kept)
                held.append(record)
        torch.cuda.synchronize()
    finally:
        backend.use_stream(None)
    for token, logprob, logits in results:
        token, logprob, logits = (t.cpu().numpy() for t in (token, logprob, logits))
        for i in range(0, rows, 9):
            R.Row(logits[i], noise[i].cpu().numpy()).check(int(token[i]), float(logprob[i]), f"row {i}")
    # the norm does not depend on the scale of its rows, but for eps
    want = results[0][2]
    for other in results[1:]:
        assert torch.allclose(other[2], want, rtol=1e-3, atol=1e-3 * float(want.abs().max()))
