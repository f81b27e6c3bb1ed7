"""GPU: rms_norm with the residual's addition, its backward pass and its 8-bit
output, against 64 bits (bounds derived in _lm_ref). Row lengths cover a warp a
row, several warps, the register limit (32768) and rows beyond it, on and off
the vector width."""
import numpy as np
import pytest

import _lm_ref as R
from vectorcore_b200 import _abi
from vectorcore_b200 import backend as B

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (3, 1), (5, 7), (64, 33), (9, 64), (1, 128), (130, 257), (37, 1030), (300, 1024), (2, 2049),
          (1, 4096), (1000, 4096), (40, 5003), (7, 8192), (700, 8192), (3, 16384), (2, 16385), (2, 32768), (3, 32769),
          (2, 32772), (2, 70001), (20000, 64), (5000, 100)]


def inputs(rows, cols, seed=0):
    rng = np.random.default_rng(rows * 131 + cols + seed)
    x = rng.normal(size=(rows, cols)).astype(np.float32)
    r = (rng.normal(size=(rows, cols)) * np.exp(rng.normal(size=cols))).astype(np.float32)
    w = (1 + 0.1 * rng.normal(size=cols)).astype(np.float32)
    return rng, x, r, w


def within(got, want, bound, what):
    err = np.abs(np.asarray(got, np.float64) - want)
    worst = np.argmax(err - bound)
    assert (err <= bound).all(), f"{what}: {err.flat[worst]:.3e} over {np.broadcast_to(bound, err.shape).flat[worst]:.3e}"


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_and_backward(backend, rows, cols):
    rng, x, r, w = inputs(rows, cols)
    gy, gh = (rng.normal(size=(rows, cols)).astype(np.float32) for _ in range(2))
    up = backend.upload
    dw_, dx, dr = up(w), up(x), up(r)
    y, h, rstd = backend.rms_norm(dx, dw_, rows, cols, eps=1e-5, residual=dr)
    h32 = x + r
    assert np.array_equal(backend.download(h).reshape(rows, cols), h32)
    want, s = R.rms_norm(h32, w, 1e-5)
    within(backend.download(y).reshape(rows, cols), want, R.rms_norm_bound(want), "y")
    within(backend.download(rstd), s, 6 * R.U * s, "rstd")
    y0, h0, rstd0 = backend.rms_norm(dx, dw_, rows, cols, eps=1e-5)  # no residual
    assert h0 is None
    want0, _ = R.rms_norm(x, w, 1e-5)
    within(backend.download(y0).reshape(rows, cols), want0, R.rms_norm_bound(want0), "y without residual")
    for g in (gh, None):
        dh, dw = backend.rms_norm_backward(h, dw_, rstd, up(gy), rows, cols, gh=None if g is None else up(g))
        edh, edw, bdh, bdw = R.rms_norm_backward(h32, w, 1e-5, gy, g)
        within(backend.download(dh).reshape(rows, cols), edh, bdh, "dh")
        within(backend.download(dw), edw, bdw, "dw")
    dh, none = backend.rms_norm_backward(h, dw_, rstd, up(gy), rows, cols, need_w=False)
    assert none is None
    edh, _, bdh, _ = R.rms_norm_backward(h32, w, 1e-5, gy, None)
    within(backend.download(dh).reshape(rows, cols), edh, bdh, "dh alone")


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_q8(backend, rows, cols):
    _, x, r, w = inputs(rows, cols, 1)
    x[rows // 2] *= 1e-20
    r[rows // 2] *= 1e-20
    q, scale, h = backend.rms_norm_q8(backend.upload(x), backend.upload(w), rows, cols, residual=backend.upload(r))
    h32 = x + r
    assert np.array_equal(backend.download(h).reshape(rows, cols), h32)
    pitch = B.q8_pitch(cols)
    got = backend.download(q).reshape(rows, pitch)
    eq, step = R.q8(h32 * w)
    assert np.array_equal(got[:, :cols], eq)
    assert not got[:, cols:].any()
    _, s = R.rms_norm(h32, w, 1e-6)
    # M / 127 rounds twice, rstd 6 times, their product once
    within(backend.download(scale), step * s, 10 * R.U * step * s, "scale")
    q, scale = backend.quantize_q8(backend.upload(x), rows, cols)
    eq, step = R.q8(x)
    assert np.array_equal(backend.download(q).reshape(rows, pitch)[:, :cols], eq)
    within(backend.download(scale), step, 3 * R.U * step, "scale of quantize_q8")


@pytest.mark.parametrize("cols", [96, 97, 4096, 40000])
def test_strided_rows_and_in_place(backend, cols):
    rows, xs, rs = 6, 3 * cols + 5, cols + 4
    rng = np.random.default_rng(cols)
    bx, br = rng.normal(size=rows * xs).astype(np.float32), rng.normal(size=rows * rs).astype(np.float32)
    w = rng.normal(size=cols).astype(np.float32)
    x = np.stack([bx[i * xs:i * xs + cols] for i in range(rows)])
    r = np.stack([br[i * rs:i * rs + cols] for i in range(rows)])
    y, h, _ = backend.rms_norm(backend.upload(bx), backend.upload(w), rows, cols, residual=backend.upload(br),
                               x_stride=xs, residual_stride=rs)
    assert np.array_equal(backend.download(h).reshape(rows, cols), x + r)
    want, _ = R.rms_norm(x + r, w, 1e-6)
    within(backend.download(y).reshape(rows, cols), want, R.rms_norm_bound(want), "strided")
    # a stride of 0 repeats one row
    y, _, _ = backend.rms_norm(backend.upload(x[0]), backend.upload(w), rows, cols, x_stride=0)
    want, _ = R.rms_norm(np.repeat(x[:1], rows, 0), w, 1e-6)
    within(backend.download(y).reshape(rows, cols), want, R.rms_norm_bound(want), "repeated")
    # the residual stream updated in place, from an address off the vector width
    for off in (0, 1):
        stream = backend.upload(np.concatenate([np.zeros(off, np.float32), r.ravel()]))
        at = B.CudaStorage.borrow(stream.ptr + 4 * off, rows * cols)
        out = backend.allocate(rows * B.q8_pitch(cols), np.int8), backend.allocate(rows), at
        backend.rms_norm_q8(backend.upload(x.ravel()), backend.upload(w), rows, cols, residual=at, out=out)
        assert np.array_equal(backend.download(stream)[off:].reshape(rows, cols), x + r)
        eq, _ = R.q8((x + r) * w)
        assert np.array_equal(backend.download(out[0]).reshape(rows, -1)[:, :cols], eq)


@pytest.mark.parametrize("cols", [5, 256, 5000, 33000])
def test_odd_rows(backend, cols):
    """Zero, tiny, infinite and NaN rows beside an ordinary one."""
    rng = np.random.default_rng(cols)
    x = rng.normal(size=(7, cols)).astype(np.float32)
    x[1] = 0.0
    x[2] = 1e-35 * x[0]
    x[3, cols - 1] = np.inf
    x[4, cols // 2] = np.nan
    x[5] = 0.0
    x[5, cols - 1] = -3.0
    w = np.ones(cols, np.float32)
    for kind in ("rms_norm_q8", "quantize_q8"):
        if kind == "rms_norm_q8":
            q, scale, _ = backend.rms_norm_q8(backend.upload(x), backend.upload(w), 7, cols)
            _, s = R.rms_norm(x[[0, 1, 2, 5, 6]], w, 1e-6)
        else:
            q, scale = backend.quantize_q8(backend.upload(x), 7, cols)
            s = np.ones(5)
        q, scale = backend.download(q).reshape(7, -1)[:, :cols], backend.download(scale)
        eq, step = R.q8(x)
        assert np.array_equal(q, eq)
        assert np.isnan(scale[3]) and np.isnan(scale[4]) and not q[3].any() and not q[4].any()
        assert scale[1] == 0 and scale[2] == 0
        within(scale[[0, 1, 2, 5, 6]], step[[0, 1, 2, 5, 6]] * s, 10 * R.U * step[[0, 1, 2, 5, 6]] * s, kind)
    y, _, _ = backend.rms_norm(backend.upload(x), backend.upload(w), 7, cols)
    y = backend.download(y).reshape(7, cols)
    assert not y[1].any() and np.isnan(y[4]).any()
    want, _ = R.rms_norm(x[[0, 5, 6]], w, 1e-6)
    within(y[[0, 5, 6]], want, R.rms_norm_bound(want), "rows beside odd ones")


@pytest.mark.parametrize("rows,cols", [(50, 1030), (50, 4096), (3000, 1024), (1000, 4096), (700, 8192), (3, 40000)])
@pytest.mark.parametrize("over", ["gy", "gh", "h"])
def test_gradient_in_place(backend, rows, cols, over):
    """dh written over one of the tensors it is computed from, which dw reads too."""
    rng, x, _, w = inputs(rows, cols, 2)
    gy, gh = (rng.normal(size=(rows, cols)).astype(np.float32) for _ in range(2))
    d = {"h": backend.upload(x), "gy": backend.upload(gy), "gh": backend.upload(gh)}
    dw_ = backend.upload(w)
    _, _, rstd = backend.rms_norm(d["h"], dw_, rows, cols)
    dw = backend.allocate(cols)
    backend.rms_norm_backward(d["h"], dw_, rstd, d["gy"], rows, cols, gh=d["gh"], out=(d[over], dw))
    edh, edw, bdh, bdw = R.rms_norm_backward(x, w, 1e-6, gy, gh)
    within(backend.download(d[over]).reshape(rows, cols), edh, bdh, "dh")
    within(backend.download(dw), edw, bdw, "dw")


@pytest.mark.parametrize("rows,cols", [(160000, 64), (2049, 33), (5000, 1030), (90000, 128)])
def test_long_sums_over_rows(backend, rows, cols):
    """dw over more rows than one run of float additions takes."""
    rng, x, _, w = inputs(rows, cols, 3)
    gy = rng.normal(size=(rows, cols)).astype(np.float32)
    dx, dw_ = backend.upload(x), backend.upload(w)
    _, _, rstd = backend.rms_norm(dx, dw_, rows, cols)
    dh, dw = backend.rms_norm_backward(dx, dw_, rstd, backend.upload(gy), rows, cols)
    edh, edw, bdh, bdw = R.rms_norm_backward(x, w, 1e-6, gy, None)
    within(backend.download(dh).reshape(rows, cols), edh, bdh, "dh")
    within(backend.download(dw), edw, bdw, "dw")


@pytest.mark.parametrize("rows,cols", [(7105, 1), (7107, 131), (7111, 33), (3600, 1000), (1801, 1030), (900, 2051),
                                       (893, 4093), (449, 4099), (450, 8189), (450, 8191), (1000, 8192), (225, 8196),
                                       (300, 12000), (230, 16380), (4800, 8200), (250, 16384), (250, 16388)])
@pytest.mark.parametrize("shifted,over", [((), None), ((), "h"), (("dh",), None), (("gh", "w"), "gy"), ((), "gh")])
def test_gradient_of_many_odd_rows(backend, rows, cols, shifted, over):
    """Rows, or tensors beside h and gy, that start off the 16-byte grid."""
    rng, x, _, w = inputs(rows, cols, 4)
    host = {"h": x, "w": w, **{n: rng.normal(size=(rows, cols)).astype(np.float32) for n in ("gy", "gh")}}
    host["dh"] = np.zeros((rows, cols), np.float32)
    on, at = {}, {}
    for name, v in host.items():
        off = int(name in shifted)
        on[name] = backend.upload(np.concatenate([np.zeros(off, np.float32), v.ravel()]))
        at[name] = B.CudaStorage.borrow(on[name].ptr + 4 * off, v.size)
    _, _, rstd = backend.rms_norm(at["h"], backend.upload(w), rows, cols)
    dw, to = backend.allocate(cols), over or "dh"
    backend.rms_norm_backward(at["h"], at["w"], rstd, at["gy"], rows, cols, gh=at["gh"], out=(at[to], dw))
    edh, edw, bdh, bdw = R.rms_norm_backward(x, w, 1e-6, host["gy"], host["gh"])
    within(backend.download(on[to])[int(to in shifted):].reshape(rows, cols), edh, bdh, "dh")
    within(backend.download(dw), edw, bdw, "dw")


def test_no_rows_and_repeatable(backend):
    w = backend.upload(np.ones(40, np.float32))
    empty = backend.allocate(0)
    backend.rms_norm(empty, w, 0, 40)
    backend.rms_norm_q8(empty, w, 0, 40)
    dw = backend.upload(np.full(40, 7, np.float32))
    backend.rms_norm_backward(empty, w, empty, empty, 0, 40, out=(empty, dw))
    assert not backend.download(dw).any()
    _, x, r, w = inputs(3000, 1000)
    a = [backend.upload(v) for v in (x, r, w)]
    _, h, rstd = backend.rms_norm(a[0], a[2], 3000, 1000, residual=a[1])
    first = [backend.download(v) for v in backend.rms_norm_backward(h, a[2], rstd, a[1], 3000, 1000, gh=a[0])]
    for _ in range(3):
        again = [backend.download(v) for v in backend.rms_norm_backward(h, a[2], rstd, a[1], 3000, 1000, gh=a[0])]
        assert all(np.array_equal(p, q) for p, q in zip(first, again))


def test_refusals(backend):
    x, w = backend.upload(np.ones(64, np.float32)), backend.upload(np.ones(16, np.float32))
    y = backend.allocate(64)
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            backend.rms_norm(x, w, 4, 16, eps=eps)
        with pytest.raises(ValueError, match="eps"):
            backend.rms_norm_q8(x, w, 4, 16, eps=eps)
    with pytest.raises(ValueError, match="at least one column"):
        backend.rms_norm(x, w, 4, 0)
    with pytest.raises(ValueError, match="null"):
        backend.rms_norm(x, None, 4, 16)
    with pytest.raises(ValueError, match="null"):
        backend.rms_norm_backward(x, w, None, x, 4, 16)
    q, s = backend.allocate(64, np.int8), backend.allocate(4)
    for args in ((x.ptr, 16, 4, 16, q.ptr, 15, s.ptr), (x.ptr, 16, 4, 16, q.ptr, 24, s.ptr),
                 (x.ptr, 16, 4, 16, q.ptr + 8, 16, s.ptr), (x.ptr, 16, 4, 16, None, 16, s.ptr)):
        with pytest.raises(ValueError, match="pitch|null"):
            _abi.call("vc_cuda_quantize_q8", *args)
    for name in ("vc_cuda_rms_norm", "vc_cuda_rms_norm_q8"):  # rows of x that overlap rows of h unlike
        tail = (y.ptr, None) if name == "vc_cuda_rms_norm" else (q.ptr, 16, s.ptr)
        with pytest.raises(ValueError, match="contiguous"):
            _abi.call(name, x.ptr, 12, None, 0, w.ptr, 4, 16, 1e-6, x.ptr, *tail)
        with pytest.raises(ValueError, match="contiguous"):
            _abi.call(name, y.ptr, 16, x.ptr, 12, w.ptr, 4, 16, 1e-6, x.ptr, *tail)
    with pytest.raises(OverflowError):
        _abi.call("vc_cuda_rms_norm", x.ptr, 16, None, 0, w.ptr, 1 << 62, 16, 1e-6, None, x.ptr, None)
    with pytest.raises(OverflowError):
        _abi.call("vc_cuda_rms_norm", x.ptr, 16, None, 0, w.ptr, 1, 1 << 40, 1e-6, None, x.ptr, None)
