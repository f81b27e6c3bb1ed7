"""GPU: the product of 8-bit rows with scales, against exact integers in 64
bits. Sizes cover both sides of every rule that picks a kernel or a tile, and
lengths around the 16-byte and 128-byte steps."""
import numpy as np
import pytest

import _lm_ref as R
from vectorcore_b200 import _abi
from vectorcore_b200 import backend as B

pytestmark = pytest.mark.gpu

SIZES = [(1, 1, 1), (1, 5, 16), (2, 16, 17), (3, 33, 127), (4, 64, 128), (5, 100, 129), (7, 129, 255), (8, 128, 256),
         (9, 200, 500), (15, 257, 1024), (16, 31, 2048), (17, 64, 1030), (31, 300, 640), (32, 32, 31), (33, 1000, 333),
         (48, 130, 4096), (63, 96, 5000), (64, 64, 64), (65, 4097, 96), (100, 40, 16384), (127, 127, 127),
         (128, 128, 128), (129, 129, 129), (200, 513, 4100), (256, 256, 512), (257, 300, 1000), (300, 2000, 640),
         (511, 512, 2048), (1000, 1000, 1000), (1030, 2050, 520), (2048, 2048, 256), (5000, 70, 300), (33, 20000, 160),
         (1, 4096, 4096), (1, 32000, 1024), (2, 11009, 4100), (640, 11009, 200)]


def matrix(rng, rows, k, pitch, low=-127):
    """An 8-bit matrix whose bytes past k are garbage."""
    full = rng.integers(-128, 128, size=(rows, pitch)).astype(np.int8)
    full[:, :k] = rng.integers(low, 128, size=(rows, k))
    return full


def check(backend, a, b, k, sa, sb, bias, got, what):
    want, bound = R.matmul_q8(a[:, :k], sa, b[:, :k], sb, bias)
    err = np.abs(got.astype(np.float64) - want)
    bad = np.argwhere(~(err <= bound))
    assert not len(bad), f"{what}: {len(bad)} of {err.size} off, first at {bad[0]}: {got[tuple(bad[0])]} for {want[tuple(bad[0])]}"


@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(backend, m, n, k):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    up = backend.upload
    for extra, with_bias in ((0, False), (16, True)):
        pitch = B.q8_pitch(k) + extra
        a, b = matrix(rng, m, k, pitch, -128), matrix(rng, n, k, pitch)
        sa, sb = rng.uniform(0.5, 2, m).astype(np.float32), rng.uniform(1e-3, 2e-3, n).astype(np.float32)
        bias = rng.normal(size=n).astype(np.float32) if with_bias else None
        out = backend.matmul_q8(up(a, np.int8), up(sa), up(b, np.int8), up(sb), m, n, k,
                                bias=None if bias is None else up(bias), a_pitch=pitch, b_pitch=pitch)
        check(backend, a, b, k, sa, sb, bias, backend.download(out).reshape(m, n), f"{m}x{n}x{k} pitch {pitch}")


@pytest.mark.parametrize("m,n,k", [(17, 18944, 40), (33, 18945, 130), (70, 20001, 300), (200, 19500, 64), (256, 38001, 16)])
def test_wide_products_of_one_tile_of_tokens(backend, m, n, k):
    """More weight rows than one tile a pair of CTAs: tiles have fewer than 128."""
    test_product(backend, m, n, k)


@pytest.mark.parametrize("m,n", [(1, 3), (9, 130), (70, 40), (300, 260)])
def test_largest_sums(backend, m, n):
    """The longest rows of the largest values: 131071 * 2^14 < 2^31."""
    k = 131071
    pitch = B.q8_pitch(k)
    a, b = np.full((m, pitch), -128, np.int8), np.full((n, pitch), -128, np.int8)
    b[::2] = 127
    one_m, one_n = np.ones(m, np.float32), np.ones(n, np.float32)
    up = backend.upload
    out = backend.matmul_q8(up(a, np.int8), up(one_m), up(b, np.int8), up(one_n), m, n, k)
    row = np.where(np.arange(n) % 2 == 0, -128 * 127 * k, 128 * 128 * k).astype(np.float32)
    assert np.array_equal(backend.download(out).reshape(m, n), np.tile(row, (m, 1)))


@pytest.mark.parametrize("m,n", [(1, 40), (20, 70), (150, 300)])
def test_no_length_and_no_rows(backend, m, n):
    up = backend.upload
    sa, sb, bias = np.ones(m, np.float32), np.ones(n, np.float32), np.arange(n, dtype=np.float32)
    none = backend.allocate(0, np.int8)
    out = backend.matmul_q8(none, up(sa), none, up(sb), m, n, 0, bias=up(bias))
    assert np.array_equal(backend.download(out).reshape(m, n), np.tile(bias, (m, 1)))
    out = backend.matmul_q8(none, up(sa), none, up(sb), m, n, 0)
    assert not backend.download(out).any()
    q = backend.allocate(n * 16, np.int8)
    empty = backend.allocate(0)
    backend.matmul_q8(none, empty, q, up(sb), 0, n, 16, out=empty)
    backend.matmul_q8(q, up(sb), none, empty, n, 0, 16, out=empty)


def test_poisoned_scale_shows(backend):
    """A NaN scale (a row that held an infinity) reaches its outputs alone."""
    for m in (3, 40, 200):
        rng = np.random.default_rng(m)
        a, b = matrix(rng, m, 64, 64), matrix(rng, 96, 64, 64)
        sa = np.ones(m, np.float32)
        sa[m // 2] = np.nan
        up = backend.upload
        out = backend.matmul_q8(up(a, np.int8), up(sa), up(b, np.int8), up(np.ones(96, np.float32)), m, 96, 64)
        bad = np.isnan(backend.download(out).reshape(m, 96))
        assert bad[m // 2].all() and bad.sum() == 96


def test_repeatable_and_on_another_stream(backend):
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(0)
    up = backend.upload
    side = torch.cuda.Stream()
    for m in (4, 90, 500):
        a, b = matrix(rng, m, 1000, 1008), matrix(rng, 777, 1000, 1008)
        args = (up(a, np.int8), up(np.ones(m, np.float32)), up(b, np.int8), up(np.ones(777, np.float32)), m, 777, 1000)
        first = backend.download(backend.matmul_q8(*args))
        for _ in range(3):
            assert np.array_equal(first, backend.download(backend.matmul_q8(*args)))
        try:
            backend.use_stream(side.cuda_stream)
            assert np.array_equal(first, backend.download(backend.matmul_q8(*args)))
            backend.use_stream(0)
            assert np.array_equal(first, backend.download(backend.matmul_q8(*args)))
        finally:
            backend.use_stream(None)


def test_refusals(backend):
    q, s, out = backend.allocate(64 * 64, np.int8), backend.allocate(64), backend.allocate(64 * 64)
    with pytest.raises(OverflowError, match="131071"):
        _abi.call("vc_cuda_matmul_q8", q.ptr, 131072, s.ptr, q.ptr, 131072, s.ptr, None, 1, 1, 131072, out.ptr)
    for ap, bp, a, b in ((48, 64, q.ptr, q.ptr), (64, 72, q.ptr, q.ptr), (64, 64, q.ptr + 4, q.ptr),
                         (64, 64, q.ptr, q.ptr + 1)):
        with pytest.raises(ValueError, match="pitch"):
            _abi.call("vc_cuda_matmul_q8", a, ap, s.ptr, b, bp, s.ptr, None, 8, 8, 64, out.ptr)
    for gone in range(5):
        ptrs = [q.ptr, s.ptr, q.ptr, s.ptr, out.ptr]
        ptrs[gone] = None
        with pytest.raises(ValueError, match="null"):
            _abi.call("vc_cuda_matmul_q8", ptrs[0], 64, ptrs[1], ptrs[2], 64, ptrs[3], None, 8, 8, 64, ptrs[4])
    with pytest.raises(OverflowError):
        _abi.call("vc_cuda_matmul_q8", q.ptr, 64, s.ptr, q.ptr, 64, s.ptr, None, 1 << 40, 8, 64, out.ptr)
