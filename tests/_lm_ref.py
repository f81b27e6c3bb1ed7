"""Plain 64-bit forms of the language-model operators (norm, 8-bit product,
sampling), and the error bounds their tests use. U is half an ulp of 1 in
float32, the relative error of one rounding."""
import numpy as np

U = 2.0 ** -24


def f64(a):
    return np.asarray(a, np.float64)


# ---- norm -----------------------------------------------------------------------

def rms_norm(h, w, eps):
    """(y, rstd) in 64 bits of the float32 residual stream h."""
    h = f64(h)
    rstd = 1.0 / np.sqrt((h * h).mean(1) + eps)
    return h * rstd[:, None] * f64(w), rstd


# y: squares summed by fours in float (4 roundings of positive terms), the
# square root halves that to 2; mean to float and + eps (half of 1 each), square
# root, division, two products: 7 roundings at most. One spare.
def rms_norm_bound(y):
    return 8 * U * np.abs(y) + 1e-44


def rms_norm_backward(h, w, eps, gy, gh):
    """(dh, dw) in 64 bits and the bounds of their float32 forms."""
    h, w, gy = f64(h), f64(w), f64(gy)
    gh = np.zeros_like(h) if gh is None else f64(gh)
    cols = h.shape[1]
    s = (1.0 / np.sqrt((h * h).mean(1) + eps))[:, None]
    t = gy * w
    along = (t * h).mean(1, keepdims=True)
    dh = s * (t - h * (s * s * along)) + gh
    # t 1 rounding; along at most 6 of its absolute terms; s 5 (twice in s * s);
    # products and sums: below 32 of the absolute terms
    reach = s * (np.abs(t) + np.abs(h) * (s * s * (np.abs(t * h)).mean(1, keepdims=True))) + np.abs(gh)
    terms = gy * (h * s)
    # dw: 7 roundings a term, up to 64 float additions before double ones
    return dh, terms.sum(0), 32 * U * reach + 1e-44, 96 * U * np.abs(terms).sum(0) + 1e-44


def q8(u):
    """8-bit rows of float32 u by the operators' rule (float32 products, so the
    integers are exact), with the unscaled step in 64 bits."""
    u = np.asarray(u, np.float32)
    m = np.abs(u).max(1)
    q = np.zeros(u.shape, np.int8)
    step = np.zeros(u.shape[0])
    for i in range(u.shape[0]):
        if not np.isfinite(m[i]):
            step[i] = np.nan
        elif m[i] >= np.float32(2.0) ** -100:
            q[i] = np.rint(u[i] * (np.float32(127) / m[i])).astype(np.int8)
            step[i] = float(m[i]) / 127.0
    return q, step


# ---- 8-bit product -----------------------------------------------------------------

def matmul_q8(a, sa, b, sb, bias):
    """The product in 64 bits and its bound: the sum's conversion, sa * sb and
    their product round (3), the bias' addition once more."""
    prod = (a.astype(np.int64) @ b.astype(np.int64).T) * (f64(sa)[:, None] * f64(sb))
    out = prod if bias is None else prod + f64(bias)
    reach = np.abs(prod) + (0.0 if bias is None else np.abs(f64(bias)))
    return out, 4 * U * reach + 1e-44


# ---- sampling -------------------------------------------------------------------------

class Row:
    """One row's sampling in 64 bits."""

    def __init__(self, x, noise, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        x = np.asarray(x, np.float32)
        self.play = x > -np.inf
        if not self.play.any():
            return
        x = f64(x)
        top = x[self.play].max()
        self.greedy = not temperature > 0
        t = 1.0 if self.greedy else float(np.float32(temperature))
        with np.errstate(invalid="ignore", divide="ignore"):
            d = np.where(x == top, 0.0, (x - top) / t)
            self.w = np.where(self.play, np.exp(d), 0.0)
        self.d = d
        # in order: larger logits first, equal ones (-0 and +0 too) by index
        self.order = np.lexsort((np.arange(x.size), np.where(self.play, -x, np.inf)))
        self.total = self.w.sum()
        w = self.w[self.order]
        rank = np.arange(x.size)
        count = int(self.play.sum())
        in_k = rank < (top_k if 0 < top_k < count else count)
        mass = np.where(in_k, w, 0.0)
        self.before = np.concatenate([[0.0], np.cumsum(mass)[:-1]])
        p = float(np.float32(top_p)) if top_p < 1 else np.inf
        limit = p * mass.sum()
        # the operator's masses are float32 weights in steps of 2^-40; a class
        # this near a limit may fall on either side
        slack = 1e-6 * mass.sum()
        least = -1.0 if np.isnan(min_p) else float(np.float32(min_p))
        sure = in_k & (self.before < limit - slack) & (w >= least * (1 + 1e-5))
        may = in_k & (self.before < limit + slack) & (w >= least * (1 - 1e-5))
        sure[0] = may[0] = True
        if self.greedy:
            sure[1:] = may[1:] = False
        with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
            score = w / f64(noise)[self.order]
        score[np.isnan(score)] = -1.0
        self.sure, self.may, self.score = sure, may, score

    def check(self, token, logprob, what=""):
        if not self.play.any():
            assert token == -1 and np.isnan(logprob), (what, token, logprob)
            return
        at = int(np.flatnonzero(self.order == token)[0]) if 0 <= token < self.d.size else -1
        assert at >= 0, (what, token)
        assert self.may[at], f"{what}: class {token} (place {at}) was filtered out"
        if not self.greedy:
            # d has two roundings of its size, e^d two of its own, the division one
            best = self.score[self.sure].max()
            d = abs(self.d[token])
            assert self.score[at] >= best * (1 - (4 * d + 16) * U), (what, token, self.score[at], best)
        want = self.d[token] - np.log(self.total)
        # d: 2 roundings; the total: 4 a term (and d's); the log and the difference 1 each
        heavy = self.w > 0
        worst = float((self.w[heavy] * np.abs(self.d[heavy])).sum() / self.total)
        bound = U * (4 * abs(self.d[token]) + 4 * worst + 8 + 4 * abs(np.log(self.total)) + abs(want))
        assert abs(logprob - want) <= bound, (what, logprob, want, bound)
