"""Cases of the operators on the way from a model's residual stream to its
next token, and of the norm's training step:

* ``rms_norm``      residual addition and root-mean-square norm, forward and
                    backward (a training step of the norm);
* ``rms_norm_q8``   the same norm with its output in 8 bits and a scale for
                    each token (serving);
* ``matmul_q8``     the product of 8-bit rows, with a scale for each token and
                    for each output channel;
* ``sample``        the next token from logits, with temperature, top-k,
                    top-p and min-p, from given exponential random numbers.

``run`` computes a case in plain torch operations, or through
``vectorcore_b200.backend.CudaBackend`` where ``own`` is true; ``exact``
computes it in 64 bits.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
F32, I64, I8 = np.dtype(np.float32), np.dtype(np.int64), np.dtype(np.int8)


# ---- cases --------------------------------------------------------------------

def listed():
    return [
        # fine-tuning a small model on short odd-sized sentences
        {"name": "norm-train-37x1030", "kind": "rms_norm", "rows": 37, "cols": 1030},
        # one microbatch of 2048 tokens of a mid-sized model
        {"name": "norm-train-2048x4096", "kind": "rms_norm", "rows": 2048, "cols": 4096},
        # a long-context batch of a wide model
        {"name": "norm-train-8192x8192", "kind": "rms_norm", "rows": 8192, "cols": 8192},
        # decoding: one new token
        {"name": "norm-q8-1x4096", "kind": "rms_norm_q8", "rows": 1, "cols": 4096},
        # a decode batch, hidden size off the vector width
        {"name": "norm-q8-250x5003", "kind": "rms_norm_q8", "rows": 250, "cols": 5003},
        # a prompt of 8192 tokens
        {"name": "norm-q8-8192x8192", "kind": "rms_norm_q8", "rows": 8192, "cols": 8192},
        # decoding one token through the 32000-class head
        {"name": "matmul-q8-1x32000x4096", "kind": "matmul_q8", "m": 1, "n": 32000, "k": 4096, "bias": False},
        # a decode batch through an odd-sized projection with a bias
        {"name": "matmul-q8-70x11009x4100", "kind": "matmul_q8", "m": 70, "n": 11009, "k": 4100, "bias": True},
        # a prompt through a square projection
        {"name": "matmul-q8-8192x8192x8192", "kind": "matmul_q8", "m": 8192, "n": 8192, "k": 8192, "bias": False},
        # one stream, temperature alone
        {"name": "sample-1x32000", "kind": "sample", "rows": 1, "vocab": 32000, "pad": 0, "temperature": 0.8,
         "top_k": 0, "top_p": 1.0, "min_p": 0.0, "masked": 0.0},
        # a serving batch with the usual settings, logits on a padded vocabulary
        {"name": "sample-48x50257-k-p", "kind": "sample", "rows": 48, "vocab": 50257, "pad": 47, "temperature": 0.9,
         "top_k": 50, "top_p": 0.95, "min_p": 0.0, "masked": 0.25},
        # many rollouts with a nucleus over the whole large vocabulary
        {"name": "sample-256x128000-p-min", "kind": "sample", "rows": 256, "vocab": 128000, "pad": 0,
         "temperature": 1.0, "top_k": 0, "top_p": 0.98, "min_p": 0.0005, "masked": 0.0},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    kind = rng.choice(["rms_norm", "rms_norm_q8", "matmul_q8", "sample"])
    if kind in ("rms_norm", "rms_norm_q8"):
        cols = _log_int(rng, 64, 16384)
        return {"kind": kind, "rows": _log_int(rng, 1, min(32768, (1 << 26) // cols)), "cols": cols}
    if kind == "matmul_q8":
        n, k = _log_int(rng, 64, 32768), _log_int(rng, 64, 16384)
        return {"kind": kind, "m": _log_int(rng, 1, max(1, min(8192, (1 << 39) // (n * k)))), "n": n, "k": k,
                "bias": rng.random() < 0.5}
    vocab = _log_int(rng, 1000, 200000)
    return {"kind": kind, "rows": _log_int(rng, 1, min(512, 32768000 // vocab)), "vocab": vocab,
            "pad": rng.choice([0, 0, rng.randint(1, 64)]), "temperature": round(rng.uniform(0.5, 1.5), 3),
            "top_k": rng.choice([0, 0, _log_int(rng, 1, 1000)]), "top_p": rng.choice([1.0, round(rng.uniform(0.5, 0.99), 3)]),
            "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.0005, 0.1), 4)]), "masked": rng.choice([0.0, 0.5])}


# ---- inputs ---------------------------------------------------------------------

def _pitch(k):
    """8-bit rows start on 16-byte boundaries; the bytes past k are zero."""
    return (k + 15) // 16 * 16


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    s = dict(case)
    if case["kind"] in ("rms_norm", "rms_norm_q8"):
        rows, cols = case["rows"], case["cols"]
        # a residual stream: channels of different widths, a block's output added to it
        wide = normal(cols).mul_(0.7).exp_()
        s["residual"] = normal(rows, cols).mul_(wide)
        s["x"] = normal(rows, cols).mul_(0.5)
        s["weight"] = 1.0 + 0.1 * normal(cols)
        if case["kind"] == "rms_norm":
            s["gy"] = normal(rows, cols).mul_(0.01)
            s["gh"] = normal(rows, cols).mul_(0.01)
    elif case["kind"] == "matmul_q8":
        m, n, k = case["m"], case["n"], case["k"]

        def q8(r):
            q = torch.zeros((r, _pitch(k)), dtype=torch.int8, device="cuda")
            q[:, :k] = normal(r, k).mul_(32.0).round_().clamp_(-127, 127).to(torch.int8)
            return q

        s["a"], s["b"] = q8(m), q8(n)
        s["a_scale"] = torch.rand(m, device="cuda", generator=gen).mul_(0.05).add_(0.01)
        s["b_scale"] = torch.rand(n, device="cuda", generator=gen).mul_(1e-3).add_(1e-4)
        s["bias"] = normal(n) if case["bias"] else None
    else:
        rows, vocab, width = case["rows"], case["vocab"], case["vocab"] + case["pad"]
        logits = normal(rows, width).mul_(2.0)
        # a model's row has a few likely classes over a broad floor
        likely = torch.randint(0, vocab, (rows, 24), device="cuda", generator=gen)
        logits.scatter_add_(1, likely, normal(rows, 24).mul_(2.0).add_(8.0))
        if case["masked"]:
            logits[torch.rand((rows, width), device="cuda", generator=gen) < case["masked"]] = -math.inf
            logits[:, vocab // 2] = 3.0  # no row is left empty
        s["logits"] = logits
        s["noise"] = torch.empty((rows, vocab), device="cuda").exponential_(generator=gen)
        # every request has its own settings: around the case's, some greedy or untruncated
        at = torch.arange(rows, device="cuda")
        t = torch.full((rows,), case["temperature"], device="cuda") * (1.0 + 0.1 * (at % 3))
        s["temperature"] = torch.where(at % 8 == 5, 0.0, t)
        s["top_k"] = torch.where(at % 8 == 3, 0, case["top_k"] + at % 4) if case["top_k"] else None
        s["top_p"] = torch.where(at % 8 == 6, 1.0, case["top_p"] - 0.01 * (at % 4)) if case["top_p"] < 1 else None
        s["min_p"] = torch.where(at % 8 == 7, 0.0, case["min_p"] * (1.0 + at % 2)) if case["min_p"] else None
    return s


# ---- the plain form ---------------------------------------------------------------

def _plain_rms_norm(s):
    h = s["x"] + s["residual"]
    rstd = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    y = h * rstd * s["weight"]
    t = s["gy"] * s["weight"]
    dh = rstd * (t - h * (rstd * rstd * (t * h).mean(1, keepdim=True))) + s["gh"]
    dw = (s["gy"] * (h * rstd)).sum(0)
    return {"h": h, "y": y, "dh": dh, "dw": dw}


def _plain_rms_norm_q8(s):
    # rstd is a factor of the whole row, so the 8-bit values do not depend on it
    h = s["x"] + s["residual"]
    rstd = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    u = h * s["weight"]
    most = u.abs().amax(1, keepdim=True)
    q = torch.round(u * (torch.full_like(most, 127.0) / most))
    scale = most * torch.full_like(most, 1.0 / 127.0) * rstd
    return {"h": h, "values": q * scale, "scale": scale[:, 0]}


def _plain_matmul_q8(s):
    a, b = s["a"][:, : s["k"]].float(), s["b"][:, : s["k"]].float()
    out = torch.matmul(a, b.T) * s["a_scale"][:, None] * s["b_scale"]
    return {"out": out if s["bias"] is None else out + s["bias"]}


def _plain_sample(s):
    x = s["logits"][:, : s["vocab"]]
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.amax(1, keepdim=True)
    greedy = s["temperature"][:, None] <= 0
    t = torch.where(greedy, 1.0, s["temperature"][:, None])
    d = torch.where(x == top, 0.0, (x - top) / t)
    w = torch.where(x == -math.inf, 0.0, torch.exp(d))
    total = w.sum(1, keepdim=True)
    # most likely first, equal logits by index
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(s["vocab"], device=x.device)[None]
    keep = (rank == 0) | ~greedy
    if s["top_k"] is not None:
        k = s["top_k"][:, None]
        keep = keep & ((rank < k) | (k <= 0))
    if s["top_p"] is not None:
        p = s["top_p"][:, None]
        mass = torch.where(keep, ws, 0.0)
        before = torch.cumsum(mass, 1) - mass
        keep = keep & ((before < p * mass.sum(1, keepdim=True)) | (p >= 1) | (rank == 0))
    if s["min_p"] is not None:
        keep = keep & (ws >= s["min_p"][:, None])
    race = torch.where(keep, ws / s["noise"].gather(1, order), -1.0)
    race = torch.empty_like(race).scatter_(1, order, race)
    token = race.argmax(1)
    logprob = d.gather(1, token[:, None])[:, 0] - torch.log(total[:, 0])
    return {"token": token, "logprob": logprob}


# ---- the framework's operators ------------------------------------------------------

_backend = None


def _device():
    """The framework's device, enqueuing on torch's stream."""
    global _backend
    if _backend is None:
        from vectorcore_b200.backend import CudaBackend, CudaStorage

        be = CudaBackend.instance()
        be.use_stream(torch.cuda.current_stream().cuda_stream)
        _backend = be, CudaStorage.borrow
    return _backend


def _own_rms_norm(s):
    be, st = _device()
    x, rows, cols = s["x"], s["rows"], s["cols"]
    y, h, dh, dw = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), torch.empty_like(s["weight"])
    rstd = torch.empty(rows, device=x.device)
    n, w = x.numel(), st(s["weight"].data_ptr(), cols)
    hs, rs = st(h.data_ptr(), n), st(rstd.data_ptr(), rows)
    be.rms_norm(st(x.data_ptr(), n), w, rows, cols, eps=EPS, residual=st(s["residual"].data_ptr(), n),
                out=(st(y.data_ptr(), n), hs, rs))
    be.rms_norm_backward(hs, w, rs, st(s["gy"].data_ptr(), n), rows, cols, gh=st(s["gh"].data_ptr(), n),
                         out=(st(dh.data_ptr(), n), st(dw.data_ptr(), cols)))
    return {"h": h, "y": y, "dh": dh, "dw": dw}


def _own_rms_norm_q8(s):
    be, st = _device()
    x, rows, cols = s["x"], s["rows"], s["cols"]
    h, scale = torch.empty_like(x), torch.empty(rows, device=x.device)
    q = torch.empty((rows, _pitch(cols)), dtype=torch.int8, device=x.device)
    n = x.numel()
    be.rms_norm_q8(st(x.data_ptr(), n), st(s["weight"].data_ptr(), cols), rows, cols, eps=EPS,
                   residual=st(s["residual"].data_ptr(), n),
                   out=(st(q.data_ptr(), q.numel(), I8), st(scale.data_ptr(), rows), st(h.data_ptr(), n)))
    return {"h": h, "values": q[:, :cols] * scale[:, None], "scale": scale}


def _own_matmul_q8(s):
    be, st = _device()
    m, n, k, a, b, bias = s["m"], s["n"], s["k"], s["a"], s["b"], s["bias"]
    out = torch.empty((m, n), device=a.device)
    be.matmul_q8(st(a.data_ptr(), a.numel(), I8), st(s["a_scale"].data_ptr(), m), st(b.data_ptr(), b.numel(), I8),
                 st(s["b_scale"].data_ptr(), n), m, n, k, bias=None if bias is None else st(bias.data_ptr(), n),
                 out=st(out.data_ptr(), m * n))
    return {"out": out}


def _own_sample(s):
    be, st = _device()
    x, noise, rows, vocab = s["logits"], s["noise"], s["rows"], s["vocab"]
    token = torch.empty(rows, dtype=torch.int64, device=x.device)
    logprob = torch.empty(rows, device=x.device)
    k, p, least = s["top_k"], s["top_p"], s["min_p"]
    be.sample(st(x.data_ptr(), x.numel()), st(noise.data_ptr(), noise.numel()), rows, vocab,
              row_stride=vocab + s["pad"], temperature=st(s["temperature"].data_ptr(), rows),
              top_k=None if k is None else st(k.data_ptr(), rows, I64), top_p=None if p is None else st(p.data_ptr(), rows),
              min_p=None if least is None else st(least.data_ptr(), rows),
              out=(st(token.data_ptr(), rows, I64), st(logprob.data_ptr(), rows)))
    return {"token": token, "logprob": logprob}


_PLAIN = {"rms_norm": _plain_rms_norm, "rms_norm_q8": _plain_rms_norm_q8, "matmul_q8": _plain_matmul_q8,
          "sample": _plain_sample}
_OWN = {"rms_norm": _own_rms_norm, "rms_norm_q8": _own_rms_norm_q8, "matmul_q8": _own_matmul_q8,
        "sample": _own_sample}


def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


# ---- what a pass cannot do without ----------------------------------------------------

def work(case):
    if case["kind"] == "rms_norm":
        # x, residual, gy, gh in; h, y, dh out; weight in, dw out
        rows, cols = case["rows"], case["cols"]
        return {"bytes": 4 * (7 * rows * cols + 2 * cols), "flops": 16 * rows * cols}
    if case["kind"] == "rms_norm_q8":
        # x, residual, weight in; h, the values and the scales out
        rows, cols = case["rows"], case["cols"]
        return {"bytes": 4 * (4 * rows * cols + cols + rows), "flops": 8 * rows * cols}
    if case["kind"] == "matmul_q8":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * k + 4 * m * n + 4 * (m + n) + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    # the logits, and the random numbers of the classes that stay in the race
    rows, vocab = case["rows"], case["vocab"]
    raced = vocab if not case["top_k"] and case["top_p"] >= 1 and not case["min_p"] else min(vocab, case["top_k"] or vocab // 100)
    return {"bytes": 4 * rows * (vocab + raced) + 28 * rows, "flops": 8 * rows * vocab}


# ---- in 64 bits -------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("rms_norm", "rms_norm_q8"):
        h = s["x"].double().add_(s["residual"])
        w = s["weight"].double()
        norm = (h.square().sum(1).div_(case["cols"]).add_(EPS)).sqrt_()
        if case["kind"] == "rms_norm":
            unit = h / norm[:, None]
            g = s["gy"].double()
            dw = torch.einsum("rc,rc->c", g, unit)
            g *= w
            along = torch.einsum("rc,rc->r", g, unit) / case["cols"]
            g -= unit * along[:, None]
            g /= norm[:, None]
            return {"h": h, "y": unit * w, "dh": g.add_(s["gh"]), "dw": dw}
        u = h * w
        step = u.abs().max(1).values / 127.0
        q = torch.round(u / step[:, None])
        step /= norm
        return {"h": h, "values": q * step[:, None], "scale": step}
    if case["kind"] == "matmul_q8":
        k = case["k"]
        a = s["a"][:, :k].double() * s["a_scale"].double()[:, None]
        b = s["b"][:, :k].double() * s["b_scale"].double()[:, None]
        out = a @ b.T
        return {"out": out if s["bias"] is None else out.add_(s["bias"])}
    # the race in its additive form: log w - log noise, over what the filters leave
    rows, vocab = case["rows"], case["vocab"]
    x = s["logits"][:, :vocab].double()
    greedy = s["temperature"] <= 0
    z = x / torch.where(greedy, 1.0, s["temperature"].double())[:, None]
    lp = torch.log_softmax(z, 1)
    value, index = torch.sort(lp, dim=1, descending=True, stable=True)
    value[torch.isnan(value)] = -math.inf
    left = torch.ones((rows, vocab), dtype=torch.bool, device=x.device)
    if s["top_k"] is not None:
        k = torch.where(s["top_k"] > 0, s["top_k"], vocab)
        left &= torch.arange(1, vocab + 1, device=x.device)[None] <= k[:, None]
    if s["top_p"] is not None:
        mass = value.exp() * left
        run_up = torch.cumsum(mass, 1)
        run_up = torch.nn.functional.pad(run_up[:, :-1], (1, 0))
        left &= (run_up < (s["top_p"].double() * mass.sum(1))[:, None]) | (s["top_p"] >= 1)[:, None]
    if s["min_p"] is not None:
        left &= value - value[:, :1] >= s["min_p"].double().log()[:, None]
    left[:, 0] = True
    left[greedy, 1:] = False
    score = torch.where(left, value - s["noise"].double().gather(1, index).log(), -math.inf)
    best = index.gather(1, score.max(1).indices[:, None])
    return {"token": None, "logprob": lp.gather(1, best)[:, 0]}
