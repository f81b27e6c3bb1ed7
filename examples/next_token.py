"""From a residual stream to the next token on the CUDA device.

    python examples/next_token.py

A final norm's weight is trained for a few steps (rms_norm -> head product ->
cross_entropy, and the gradients back), the head is brought to 8 bits once, and
tokens are then drawn the way a server does it at every step:
rms_norm_q8 -> matmul_q8 -> sample, captured into one graph and replayed.
"""
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from vectorcore_b200 import backend as B  # noqa: E402


def train_norm(be, x, residual, weight, head, targets, steps=20, rate=2.0):
    """SGD on the norm's weight; returns the losses. x, residual [rows, cols],
    head [classes, cols] and targets live on the device."""
    rows, cols = targets.size, weight.size
    classes = head.size // cols
    one = be.fill(1, 1.0)
    losses = []
    for _ in range(steps):
        y, h, rstd = be.rms_norm(x, weight, rows, cols, residual=residual)
        logits = be.matmul(y, head, rows, cols, classes, [0], [0], trans_b=True)
        loss, row_max, row_sum, _ = be.cross_entropy(logits, targets, rows, classes)
        g_logits = be.cross_entropy_backward(logits, targets, row_max, row_sum, one, rows, classes)
        gy = be.matmul(g_logits, head, rows, classes, cols, [0], [0])
        _, dw = be.rms_norm_backward(h, weight, rstd, gy, rows, cols, out=(None, be.allocate(cols)))
        be.axpy_inplace(weight, dw, cols, -rate)
        losses.append(float(be.download(loss)[0]))
    return losses


class Decoder:
    """The last layers of a model at decode time, for a fixed batch: buffers
    made once, one graph launch a step."""

    def __init__(self, be, weight, head, rows, temperature, top_k, top_p):
        self.be, self.rows, self.cols = be, rows, weight.size
        self.classes = head.size // self.cols
        self.weight = weight
        self.head = be.quantize_q8(head, self.classes, self.cols)
        self.settings = {"temperature": be.fill(rows, temperature), "top_k": be.upload(np.full(rows, top_k, np.int64)),
                         "top_p": be.fill(rows, top_p)}
        self.x, self.residual = be.allocate(rows * self.cols), be.allocate(rows * self.cols)
        self.noise = be.allocate(rows * self.classes)
        self.step()  # kernels are loaded before the capture
        be.synchronize()
        self.graph, (self.token, self.logprob, self.logits) = be.capture(self.step)

    def step(self):
        be = self.be
        q, scale, _ = be.rms_norm_q8(self.x, self.weight, self.rows, self.cols, residual=self.residual)
        logits = be.matmul_q8(q, scale, *self.head, self.rows, self.classes, self.cols)
        token, logprob = be.sample(logits, self.noise, self.rows, self.classes, **self.settings)
        return token, logprob, logits

    def __call__(self, x, residual, noise):
        """(token, logprob) for host arrays x, residual [rows, cols] and noise
        [rows, classes]."""
        for storage, values in ((self.x, x), (self.residual, residual), (self.noise, noise)):
            B._abi.call("vc_cuda_upload", storage.ptr, values.ctypes.data, values.nbytes)
        self.graph.launch()
        return self.be.download(self.token), self.be.download(self.logprob)


def main(rows=64, cols=256, classes=1000, seed=0):
    be = B.CudaBackend.instance()
    rng = np.random.default_rng(seed)
    x, residual = (rng.normal(size=(rows, cols)).astype(np.float32) for _ in range(2))
    head = (rng.normal(size=(classes, cols)) / np.sqrt(cols)).astype(np.float32)
    # classes that follow from a rescaled stream: what the weight can learn
    hidden = (x + residual) * np.exp(rng.normal(size=cols)).astype(np.float32)
    targets = (hidden @ head.T).argmax(1).astype(np.int64)
    weight, d_head = be.fill(cols, 1.0), be.upload(head)
    losses = train_norm(be, be.upload(x), be.upload(residual), weight, d_head, be.upload(targets))
    decoder = Decoder(be, weight, d_head, rows, temperature=0.5, top_k=20, top_p=0.9)
    hits = 0
    for _ in range(4):
        noise = rng.exponential(size=(rows, classes)).astype(np.float32)
        token, logprob = decoder(x, residual, noise)
        hits += int((token == targets).sum())
    return {"losses": losses, "token": token, "logprob": logprob, "hits": hits / (4 * rows), "targets": targets,
            "x": x, "residual": residual, "noise": noise, "weight": be.download(weight), "head": head,
            "logits": be.download(decoder.logits).reshape(rows, classes)}


if __name__ == "__main__":
    r = main()
    print(f"loss {r['losses'][0]:.3f} -> {r['losses'][-1]:.3f}; {100 * r['hits']:.0f}% of drawn tokens are the target; "
          f"first tokens {r['token'][:8].tolist()}")
