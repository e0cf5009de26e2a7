"""The 8-bit row operators on the GPU against the formulas in 64 bits (oracle/rows8.py).

Tolerances are counted from the roundings: U is half a step of fp32 (2^-24 of a value), B half a step of bf16 (2^-8). A sum
of n products is off by at most n of its own roundings (2 U each, whatever the order) times the sum of the magnitudes."""
import numpy as np
import pytest

from grilly_b200 import DeviceTensor, Rows8
from grilly_b200 import _lib as L
from oracle import rows8 as R

pytestmark = pytest.mark.gpu
U, B = 2.0 ** -24, 2.0 ** -8
EPS = 1e-5


def rng_for(*key):
    return np.random.default_rng([int(k) for k in key])


def acts(rng, rows, features):
    """Hidden states: tokens of different size, a few loud channels."""
    x = rng.standard_normal((rows, features)) * (0.5 + rng.random((rows, 1)))
    return (x * np.where(rng.random(features) < 0.02, 8.0, 1.0)).astype(np.float32)


def put(b, x, dtype):
    """(DeviceTensor, the values it holds)."""
    t = b.device.upload(x, dtype)
    return t, (R.bf16(x) if dtype == "bf16" else np.asarray(x, np.float32))


def put_rows8(b, q, s, shape=None, junk=None, extra=0):
    """Rows8 of integers q (rows, features) and scales; the bytes past the features hold ``junk``."""
    rows, f = q.shape
    buf = np.zeros((rows, (f + 15) // 16 * 16 + extra), np.int8)
    if junk is not None:
        buf[:] = junk.integers(-128, 128, buf.shape)
    buf[:, :f] = q
    return Rows8(b.device.upload(buf, "i8"), b.device.upload(np.asarray(s, np.float32)), shape or (rows, f))


def check_quantised(r8, want, rel):
    """8-bit rows against 64-bit values known to a relative ``rel`` of the row's largest: half a step, the two roundings of
    x / scale (up to 127 steps in size) and what the values themselves are off."""
    q, s = r8.q.numpy()[:, : r8.features].astype(np.float64), r8.scale.numpy().astype(np.float64)
    amax = np.abs(want).max(-1)
    assert np.all(np.abs(s - np.maximum(amax / 127, float(R.TINY))) <= (rel + 3 * U) * amax / 127 + 1e-45)
    assert np.all(np.abs(q) <= 127)
    assert np.all(np.abs(q * s[:, None] - want) <= s[:, None] * (0.5 + 127 * (rel + 6 * U)))
    assert np.all(r8.q.numpy()[:, r8.features:] == 0)


WIDTHS = [1, 2, 15, 16, 17, 100, 384, 1001, 1024, 4095, 4096, 9000]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("features", WIDTHS + [33000])
@pytest.mark.parametrize("rows", [1, 77])
def test_quantize_and_read_back(backend, rows, features, dtype):
    rng = rng_for(1, rows, features)
    xd, x = put(backend, acts(rng, rows, features) * np.exp(rng.uniform(-20, 20, (rows, 1))).astype(np.float32), dtype)
    r8 = backend.fnn.quantize_rows(xd)
    q, s = R.quantize(x)
    assert np.array_equal(r8.scale.numpy(), s)                       # one division: the same fp32 number
    check_quantised(r8, x.astype(np.float64), 0.0)
    got = r8.q.numpy()[:, :features].astype(np.float64)
    assert np.mean(got != q) < 1e-3                                  # only next to ties
    want = got * s[:, None].astype(np.float64)
    assert np.array_equal(r8.numpy(), want.astype(np.float32))
    back = backend.fnn.dequantize_rows(r8)
    assert back.shape == (rows, features) and np.array_equal(back.numpy(), want.astype(np.float32))
    half = backend.fnn.dequantize_rows(r8, "bf16").numpy()
    assert np.array_equal(half, R.bf16(want.astype(np.float32)))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("features", [384, 1001, 17000])
def test_ties_go_to_the_even_integer(backend, features, dtype):
    """Rows whose scale is m 2^j: every second value on half its grid is an exact tie of x / scale."""
    rng = rng_for(27, features)
    ms = [1, 1, 1, 1] if dtype == "bf16" else [1, 3, 5, 7, 11, 13, 23, 101, 641, 8191]     # 127 m 2^j is a bf16 number for m = 1
    x = np.stack([m * (rng.integers(-253, 254, features) / 2.0) * 2.0 ** (3 * i - 20) for i, m in enumerate(ms)]).astype(np.float32)
    if dtype == "bf16":
        x = R.bf16(x)
    for i, m in enumerate(ms):
        x[i, rng.integers(features)] = 127 * m * 2.0 ** (3 * i - 20)
    q, s = R.quantize(x)
    assert np.array_equal(s, [np.float32(m * 2.0 ** (3 * i - 20)) for i, m in enumerate(ms)])
    assert np.mean(np.abs(x / s[:, None] % 1) == 0.5) > 0.2
    xd = backend.device.upload(x, dtype)
    got = backend.fnn.rmsnorm_residual_q8(xd, backend.device.upload(np.zeros_like(x), dtype), keep=True).h8
    for r8 in (backend.fnn.quantize_rows(xd), got):
        assert np.array_equal(r8.scale.numpy(), s) and np.array_equal(r8.q.numpy()[:, :features], q)


@pytest.mark.parametrize("features", [384, 1001, 17000])
def test_half_of_the_largest_value(backend, features):
    """x = amax / 2 is 127 / 2 steps, a tie, however the scale itself is rounded: q = 64."""
    b, ms = backend, np.arange(128, 256)
    x = rng_for(28, features).uniform(-128, 128, (128, features))
    x[:, 1::7] = ms[:, None] * np.where(np.arange(len(x[0, 1::7])) % 2, 1.0, -1.0)
    x[:, 3::7] = x[:, 1::7][:, :x[:, 3::7].shape[1]] / 2
    x = R.bf16((x * np.exp2(ms % 60 - 30.0)[:, None]).astype(np.float32))
    want, s = R.quantize(x)
    assert np.all(np.abs(want[:, 3::7]) == 64)
    xd = b.device.upload(x, "bf16")
    kept = b.fnn.rmsnorm_residual_q8(xd, b.device.upload(np.zeros_like(x), "bf16"), keep=True).h8
    for r8 in (b.fnn.quantize_rows(xd), kept, b.fnn.quantize_rows(b.device.upload(x))):
        assert np.array_equal(r8.scale.numpy(), s) and np.array_equal(r8.q.numpy()[:, :features], want)


def test_rows_that_are_zero_tiny_or_not_finite(backend):
    x = acts(rng_for(2), 12, 130)
    x[0] = 0
    x[1] *= 1e-40            # below the smallest normal number
    x[2] = 0
    x[2, 7] = 3e38
    x[3, 129] = np.nan
    x[4, 0] = np.inf
    x[5, 64] = -np.inf
    x[6] = -x[6, 0]
    r8 = backend.fnn.quantize_rows(backend.device.upload(x))
    q, s = R.quantize(x)
    assert np.array_equal(r8.scale.numpy(), s, equal_nan=True)
    got = r8.numpy()
    assert np.isnan(got[3:6]).all() and np.all(r8.q.numpy()[3:6] == 0) and np.all(got[0] == 0)
    ok = [0, 1, 2, 6, 7, 8, 9, 10, 11]
    assert np.all(np.abs(got[ok].astype(np.float64) - x[ok]) <= 0.5001 * s[ok, None].astype(np.float64))
    assert np.isnan(backend.fnn.dequantize_rows(r8, "bf16").numpy()[3:6]).all()


def test_strange_rows_through_the_norm_and_the_product(backend):
    """A row that is not finite poisons itself and no other row; a zero row is zero."""
    rng = rng_for(3)
    x, r = acts(rng, 9, 200), acts(rng, 9, 200)
    x[0] = r[0] = 0
    x[2, 5], x[4, 199], r[6, 0] = np.nan, np.inf, -np.inf
    x[7] = 1e20                                       # its square is not an fp32 number
    got = backend.fnn.rmsnorm_residual_q8(backend.device.upload(x), backend.device.upload(r), keep=True)
    bad = np.array([2, 4, 6, 7])
    fine = np.array([0, 1, 3, 5, 8])
    assert np.isnan(got.y8.scale.numpy()[bad]).all() and np.isnan(got.h8.scale.numpy()[bad]).all() and np.isnan(got.rstd.numpy()[bad]).all()
    assert np.all(got.y8.q.numpy()[bad] == 0) and np.all(got.y8.numpy()[0] == 0)
    y = R.rmsnorm(x[fine], r[fine], None, EPS)[2]
    assert np.all(np.abs(got.y8.numpy()[fine] - y) <= np.abs(y).max(-1, keepdims=True) * (0.51 / 127))
    assert np.array_equal(got.h.numpy(), x + r, equal_nan=True)
    w8 = backend.fnn.quantize_rows(rng.standard_normal((40, 200)).astype(np.float32))
    for act in (None, "gelu", "silu", "relu"):
        out = backend.fnn.linear_q8(got.y8, w8, act=act).numpy()
        assert np.isnan(out[bad]).all() and np.isfinite(out[fine]).all() and np.all(out[0] == 0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("features", WIDTHS + [20000])
@pytest.mark.parametrize("rows,residual,gamma,keep", [(1, True, True, False), (1, False, False, True), (130, True, True, True)])
def test_rmsnorm_residual_q8(backend, rows, features, residual, gamma, keep, dtype):
    rng = rng_for(4, rows, features)
    xd, x = put(backend, acts(rng, rows, features), dtype)
    rd, r = put(backend, rng.standard_normal((rows, features)).astype(np.float32), dtype) if residual else (None, None)
    g = (1 + 0.3 * rng.standard_normal(features)).astype(np.float32) if gamma else None
    got = backend.fnn.rmsnorm_residual_q8(xd, rd, g, eps=EPS, keep=keep)
    h, rstd, y = R.rmsnorm(x, r, g, EPS)
    assert got.h.dtype == dtype
    assert np.all(np.abs(got.h.numpy() - h) <= np.abs(h) * (U if dtype == "f32" else B + U))
    # h is one rounding off, its square two more, the sum of F squares at most F/4 + 12 in a row (four sums side by side
    # at least), half of all that shows in rstd, which takes three more roundings
    rel = (features / 4 + 16) * U
    check_quantised(got.y8, y, rel + 4 * U)
    if keep:
        check_quantised(got.h8, h, U)
        assert np.all(np.abs(got.rstd.numpy() - rstd) <= rel * rstd)
    else:
        assert got.h8 is None and got.rstd is None


def test_norm_in_place_and_into_given_tensors(backend):
    rng = rng_for(5)
    for features in (384, 1001, 20000):
        x, r = acts(rng, 50, features), acts(rng, 50, features)
        xb, rb = R.bf16(x), R.bf16(r * np.exp2(rng.integers(-20, 20, r.shape)).astype(np.float32))
        xd = backend.device.upload(xb, "bf16")
        got = backend.fnn.rmsnorm_residual_q8(xd, backend.device.upload(rb, "bf16"), out=(None, xd, None, None)).h
        assert got is xd and np.array_equal(xd.numpy(), R.bf16(xb + rb))
        want = backend.fnn.rmsnorm_residual_q8(backend.device.upload(x), backend.device.upload(r), keep=True)
        for which in (0, 1):
            xd, rd = backend.device.upload(x), backend.device.upload(r)
            y8, h8 = Rows8.empty(backend.device, x.shape), Rows8.empty(backend.device, x.shape)
            rstd = backend.device.empty((50,))
            got = backend.fnn.rmsnorm_residual_q8(xd, rd, keep=True, out=(y8, (xd, rd)[which], h8, rstd))
            assert got.h is (xd, rd)[which] and got.y8 is y8 and got.h8 is h8 and got.rstd is rstd
            for a, w in zip((got.h, y8.q, y8.scale, h8.q, h8.scale, rstd),
                            (want.h, want.y8.q, want.y8.scale, want.h8.q, want.h8.scale, want.rstd)):
                assert np.array_equal(a.numpy(), w.numpy())


def linear_case(b, M, N, K, act, bias, dtype, seed=0, junk=None, extra=0):
    rng = rng_for(6, M, N, K, seed)
    xq, xs = R.quantize(acts(rng, M, K))
    wq, ws = R.quantize((rng.standard_normal((N, K)) * K ** -0.5).astype(np.float32))
    bb = (0.1 * rng.standard_normal(N)).astype(np.float32) if bias else None
    x8, w8 = put_rows8(b, xq, xs, junk=junk, extra=extra), put_rows8(b, wq, ws, junk=junk, extra=extra)
    got = b.fnn.linear_q8(x8, w8, bb, act=act, dtype=dtype)
    pre = R.linear(xq, xs, wq, ws, bb, None)
    want = R.act(pre, act)
    # the integer sum rounds once, two scales and the bias three times; GELU and SiLU have slope below 1.13 and take a few
    # roundings of their own; then the result's type
    size = np.abs(pre) + (0 if bb is None else 2 * np.abs(bb))
    tol = 6 * U * size * (1.2 if act in ("gelu", "silu") else 1) + (64 * U * np.abs(pre) if act in ("gelu", "silu") else 0)
    tol += (B if dtype == "bf16" else U) * np.abs(want) + 1e-40
    err = np.abs(got.numpy().astype(np.float64) - want)
    assert got.dtype == dtype and np.all(err <= tol), (err / tol).max()
    return got, want


SHAPES = [(1, 1, 1), (1, 4096, 4096), (1, 1000, 17), (2, 33, 100), (3, 129, 384), (8, 256, 1024), (9, 64, 1111), (16, 512, 2048), (17, 300, 528),
          (31, 1536, 384), (32, 48, 4097), (33, 1001, 130), (64, 2048, 2048), (100, 130, 16), (128, 128, 128), (129, 255, 257),
          (255, 511, 640), (256, 256, 128), (257, 1153, 1111), (300, 8, 3000), (512, 1024, 4096), (1000, 384, 1536), (1025, 768, 768),
          (2048, 2048, 512), (4097, 520, 100), (5000, 40, 64)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_q8(backend, M, N, K):
    i = SHAPES.index((M, N, K))
    linear_case(backend, M, N, K, ("gelu", "silu", "relu", None)[i % 4], i % 3 > 0, "f32")
    linear_case(backend, M, N, K, (None, "gelu", "silu", "relu")[i % 4], i % 3 == 0, "bf16")


@pytest.mark.parametrize("M", [1, 5, 40, 300, 1500])
def test_linear_q8_ignores_what_lies_between_the_rows(backend, M):
    a, _ = linear_case(backend, M, 200, 90, None, True, "f32", junk=rng_for(7), extra=32)
    b, _ = linear_case(backend, M, 200, 90, None, True, "f32")
    assert np.array_equal(a.numpy(), b.numpy())


@pytest.mark.parametrize("M", [1, 20, 200, 2000])
def test_linear_q8_sums_are_exact_at_the_extremes(backend, M):
    """All factors at the ends of the 8-bit range, up to the longest row: the 32-bit sums do not wrap."""
    for K, qx, qw in ((131071, 127, 127), (131071, -128, -128), (131071, -128, 127), (1000, 127, -127)):
        xq, wq = np.full((M, K), qx, np.int8), np.full((70, K), qw, np.int8)
        one = np.float32(1)
        got = backend.fnn.linear_q8(put_rows8(backend, xq, np.full(M, one)), put_rows8(backend, wq, np.full(70, one))).numpy()
        assert np.all(got == np.float32(K * qx * qw))


def test_linear_q8_from_arrays_and_shapes(backend):
    rng = rng_for(8)
    x, w, b = acts(rng, 6, 96).reshape(2, 3, 96), rng.standard_normal((50, 96)).astype(np.float32), rng.standard_normal(50).astype(np.float32)
    got = backend.fnn.linear_q8(x, w, b, act="relu")
    assert isinstance(got, np.ndarray) and got.shape == (2, 3, 50)
    (xq, xs), (wq, ws) = R.quantize(x.reshape(6, 96)), R.quantize(w)
    want = R.linear(xq, xs, wq, ws, b, "relu").reshape(2, 3, 50)
    assert np.all(np.abs(got - want) <= 2 * xs.max() * np.abs(w).max() + 1e-5)       # a tie may fall the other way: one step
    w[0] = 0                                                                          # arrays are not cached
    assert np.allclose(backend.fnn.linear_q8(x, w, b)[..., 0], b[0])
    full = x.reshape(6, 96) @ w.T + b
    assert np.linalg.norm(backend.fnn.linear_q8(x, w, b).reshape(6, 50) - full) < 0.02 * np.linalg.norm(full)


def test_linear_q8_writes_its_rows_only(backend):
    """The result's neighbours in memory stay as they were, whatever the tile."""
    rng = rng_for(9)
    for M, N, K in ((1, 100, 64), (7, 65, 64), (40, 130, 200), (130, 257, 64), (1030, 260, 130)):
        for dtype, item in (("f32", 4), ("bf16", 2)):
            xq, xs = R.quantize(acts(rng, M, K))
            wq, ws = R.quantize(acts(rng, N, K))
            guard = 4096
            buf = backend.device.upload(np.full(M * N + 2 * guard, 7.0, np.float32), dtype)
            view = DeviceTensor(backend.device, buf.ptr + guard * item, (M, N), dtype, owned=False)
            backend.fnn.linear_q8(put_rows8(backend, xq, xs), put_rows8(backend, wq, ws), out=view)
            flat = buf.numpy()
            assert np.all(flat[:guard] == 7) and np.all(flat[guard + M * N:] == 7)
            want = R.linear(xq, xs, wq, ws, None, None).reshape(-1)
            assert np.all(np.abs(flat[guard: guard + M * N] - want) <= (6 * U + B) * np.abs(want) + 1e-6)


def backward_case(b, M, N, K, dtype, seed=0, junk=None):
    rng = rng_for(10, M, N, K, seed)
    xq, xs = R.quantize(acts(rng, M, K))
    wd, w = put(b, (rng.standard_normal((N, K)) * K ** -0.5).astype(np.float32), "bf16")
    gd, g = put(b, (0.01 * rng.standard_normal((M, N))).astype(np.float32), "bf16")
    gx, gw, gb = b.fnn.linear_backward_q8(gd, put_rows8(b, xq, xs, junk=junk), wd, dtype=dtype)
    x = xq * xs[:, None].astype(np.float64)
    wx, ww, wb = R.linear_backward(g, x, w)
    ax, aw, ab = R.linear_backward(np.abs(g), np.abs(x), np.abs(w))
    out = B if dtype == "bf16" else U
    for got, want, mag, n, extra in ((gx, wx, ax, N, 0), (gw, ww, aw, M, B + U), (gb, wb, ab, M, 0)):
        tol = (2 * U * n + extra) * mag + (out if got is not gb else U) * np.abs(want) + 1e-30
        err = np.abs(got.numpy().astype(np.float64) - want)
        assert np.all(err <= tol), (err / tol).max()
        # and as a whole. Two roundings to bf16 can meet in a weight gradient: x (1 + d) and the result (1 + e) with
        # |d|, |e| <= B, so one product alone (M = 1) is up to (1 + B)^2 - 1 = 2 B + B^2 off; of many products the d
        # are independent and their sum keeps that share of the norm
        whole = (B if extra else 0) + (B if out == B and got is not gb else 0)
        assert np.linalg.norm(err) <= 1e-30 + np.linalg.norm(want) * (1e-5 + whole + B * B), np.linalg.norm(err) / np.linalg.norm(want)
    return gx, gw, gb


BWD_SHAPES = [(1, 1, 1), (1, 100, 64), (2, 8, 8), (7, 33, 65), (64, 128, 256), (100, 40, 17), (128, 384, 384), (130, 257, 100), (300, 1000, 136),
              (500, 1536, 384), (777, 1001, 515), (1024, 256, 1024), (2500, 16, 700), (3000, 384, 130), (4096, 640, 512), (9000, 72, 40)]


@pytest.mark.parametrize("M,N,K", BWD_SHAPES)
def test_linear_backward_q8(backend, M, N, K):
    backward_case(backend, M, N, K, "bf16")
    a = backward_case(backend, M, N, K, "f32")
    b = backward_case(backend, M, N, K, "f32", junk=rng_for(11))
    for s, t in zip(a, b):                                            # the same bits again, whatever lies past the features
        assert np.array_equal(s.numpy(), t.numpy())


@pytest.mark.parametrize("M,N,K", [(19968, 32, 1925), (5000, 40, 1001), (6000, 300, 77), (4100, 9, 2000)])
def test_linear_backward_whose_products_are_stored_differently(backend, M, N, K):
    """One product split along k (its parts leave by TMA), the other with rows of C off 16-byte boundaries (its lanes store),
    by the same warps of one launch: the same bits every time, and right."""
    a = backward_case(backend, M, N, K, "bf16")
    for _ in range(5):
        for s, t in zip(a, backward_case(backend, M, N, K, "bf16")):
            assert np.array_equal(s.numpy(), t.numpy())


def test_linear_backward_from_arrays(backend):
    rng = rng_for(12)
    x, w, g = acts(rng, 20, 48).reshape(4, 5, 48), rng.standard_normal((30, 48)).astype(np.float32), rng.standard_normal((4, 5, 30)).astype(np.float32)
    x8 = backend.fnn.quantize_rows(x)
    gx, gw, gb = backend.fnn.linear_backward_q8(g, x8, w, dtype="f32")
    wx, ww, wb = R.linear_backward(R.bf16(g).reshape(20, 30), x8.numpy().reshape(20, 48), R.bf16(w))
    assert gx.shape == (4, 5, 48) and gw.shape == (30, 48) and gb.shape == (30,)
    for a, b in ((gx.reshape(20, 48), wx), (gw, ww), (gb, wb)):
        assert np.linalg.norm(a - b) < 4e-3 * np.linalg.norm(b)


def norm_backward_case(b, rows, features, dtype, gamma=True, residual=True):
    rng = rng_for(13, rows, features)
    hq, hs = R.quantize(acts(rng, rows, features))
    h = hq * hs[:, None].astype(np.float64)
    rstd = (1 / np.sqrt((h * h).mean(-1) + EPS)).astype(np.float32)
    gm = (1 + 0.3 * rng.standard_normal(features)).astype(np.float32) if gamma else None
    god, go = put(b, (0.01 * rng.standard_normal((rows, features))).astype(np.float32), dtype)
    grd, gr = put(b, (0.01 * rng.standard_normal((rows, features))).astype(np.float32), dtype) if residual else (None, None)
    gh, gg = b.fnn.rmsnorm_backward_q8(god, put_rows8(b, hq, hs, junk=rng_for(14)), rstd, gm, grd)
    wh, wg = R.rmsnorm_backward(go, h, rstd, gm, gr)
    r = rstd[:, None].astype(np.float64)
    n, g = np.abs(h) * r, np.abs(go * (1.0 if gm is None else gm.astype(np.float64)))
    # every factor is two or three roundings off, the row's sum F of them; then five roundings of parts that are at most
    # this large, and the result's type
    part = r * (g + n * (g * n).mean(-1, keepdims=True)) + (0 if gr is None else np.abs(gr))
    tol = part * (8 * U) + r * n * (g * n).mean(-1, keepdims=True) * (2 * features + 8) * U + (B if dtype == "bf16" else U) * np.abs(wh)
    assert gh.dtype == dtype and np.all(np.abs(gh.numpy() - wh) <= tol)
    assert np.all(np.abs(gg.numpy() - wg) <= (2 * rows + 8) * U * (np.abs(go) * n).sum(0) + 1e-30)
    return gh, gg


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("features", WIDTHS + [20000])
@pytest.mark.parametrize("rows", [1, 3, 700])
def test_rmsnorm_backward_q8(backend, rows, features, dtype):
    a = norm_backward_case(backend, rows, features, dtype)
    b = norm_backward_case(backend, rows, features, dtype)
    assert all(np.array_equal(s.numpy(), t.numpy()) for s, t in zip(a, b))
    if rows == 3:
        norm_backward_case(backend, rows, features, dtype, gamma=False, residual=False)


@pytest.mark.parametrize("features,dtype", [(11001, "f32"), (16384, "f32"), (16001, "f32"), (12000, "f32"), (16383, "bf16"), (16384, "bf16")])
def test_rows_that_fill_shared_memory(backend, features, dtype):
    """More rows than the GPU holds at once, few or one of them in each block's shared memory."""
    norm_backward_case(backend, 450, features, dtype)
    test_rmsnorm_residual_q8(backend, 450, features, True, True, True, dtype)
    test_quantize_and_read_back(backend, 450, features, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_rows_on_every_distance_from_a_boundary(backend, dtype):
    """Row lengths of every remainder: rows start on every distance from a 16-byte boundary that there is."""
    for features in range(1, 34):
        norm_backward_case(backend, 900, features, dtype)
        test_rmsnorm_residual_q8(backend, 900, features, True, True, True, dtype)
        test_quantize_and_read_back(backend, 900, features, dtype)


def test_norm_backward_against_differences(backend):
    """The kernel's gradient of sum(w * rmsnorm(h) gamma) against central differences in 64 bits."""
    rng = rng_for(15)
    rows, features = 4, 33
    x, w, gm = acts(rng, rows, features), rng.standard_normal((rows, features)).astype(np.float32), (1 + rng.random(features)).astype(np.float32)
    h8 = backend.fnn.quantize_rows(x)
    h = h8.numpy().astype(np.float64)
    rstd = R.rmsnorm(h, None, gm, EPS)[1]
    gh, gg = backend.fnn.rmsnorm_backward_q8(w, h8, rstd.astype(np.float32), gm)
    f = lambda hh, g: (w * R.rmsnorm(hh, None, g, EPS)[2]).sum()  # noqa: E731
    for i, j in ((0, 0), (1, 32), (3, 17)):
        e = np.zeros_like(h)
        e[i, j] = 1e-4
        assert abs((f(h + e, gm) - f(h - e, gm)) / 2e-4 - gh[i, j]) < 1e-4
        d = np.zeros(features)
        d[j] = 1e-4
        assert abs((f(h, gm + d) - f(h, gm - d)) / 2e-4 - gg[j]) < 1e-4


def test_norm_backward_in_place(backend):
    rng = rng_for(16)
    for features in (384, 1001, 20000):
        hq, hs = R.quantize(acts(rng, 300, features))
        h8, rstd = put_rows8(backend, hq, hs), np.ones(300, np.float32)
        go, gr = (rng.standard_normal((300, features)).astype(np.float32) for _ in range(2))
        want, wg = backend.fnn.rmsnorm_backward_q8(backend.device.upload(go), h8, rstd, None, backend.device.upload(gr))
        for which in (0, 1):
            god, grd = backend.device.upload(go), backend.device.upload(gr)
            gh, gg = backend.fnn.rmsnorm_backward_q8(god, h8, rstd, None, grd, out=((god, grd)[which], None))
            assert np.array_equal(gh.numpy(), want.numpy()) and np.array_equal(gg.numpy(), wg.numpy())


def shifted(b, x, dtype, by):
    """(x on the device, ``by`` elements past a 16-byte boundary with 7s around it, and a check that those are still there)."""
    item = 2 if dtype == "bf16" else 4
    n = int(np.prod(x.shape))
    flat = np.full(n + 64, 7.0, np.float32)
    flat[32 + by: 32 + by + n] = np.asarray(x, np.float32).reshape(-1)
    buf = b.device.upload(flat, dtype)
    view = DeviceTensor(b.device, buf.ptr + (32 + by) * item, x.shape, dtype, owned=False)
    view._owned = buf

    def untouched():
        got = buf.numpy()
        return np.all(got[: 32 + by] == 7) and np.all(got[32 + by + n:] == 7)

    return view, untouched


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,features", [(1, 8), (3, 100), (40, 384), (150, 1001), (5, 17000)])
@pytest.mark.parametrize("by", [0, 1, 3])
def test_tensors_on_any_boundary_and_what_lies_around_them(backend, rows, features, dtype, by):
    """Views that start off a 16-byte boundary give what aligned tensors give; nothing outside an output is written."""
    b, f, rng = backend, backend.fnn, rng_for(22, rows, features)
    x, r = (R.bf16(t) if dtype == "bf16" else t for t in (acts(rng, rows, features), acts(rng, rows, features)))
    gm = (1 + 0.1 * rng.standard_normal(features)).astype(np.float32)
    zeros = np.zeros((rows, features), np.float32)
    xd, rd, gd = shifted(b, x, dtype, by)[0], shifted(b, r, dtype, by)[0], shifted(b, gm, "f32", by)[0]
    h, h_ok = shifted(b, zeros, dtype, by)
    got = f.rmsnorm_residual_q8(xd, rd, gd, keep=True, out=(None, h, None, None))
    want = f.rmsnorm_residual_q8(b.device.upload(x, dtype), b.device.upload(r, dtype), gm, keep=True)
    assert h_ok() and np.array_equal(h.numpy(), want.h.numpy())
    for a, w in ((got.y8, want.y8), (got.h8, want.h8)):
        # the sums may be taken in another order: half a step, and the scales to the roundings of the sum
        assert np.allclose(a.scale.numpy(), w.scale.numpy(), rtol=(features / 4 + 16) * U, atol=0)
        assert np.mean(a.q.numpy() != w.q.numpy()) < 1e-3 and np.abs(a.q.numpy().astype(int) - w.q.numpy()).max() <= 1
    q8 = f.quantize_rows(xd)
    assert np.array_equal(q8.scale.numpy(), R.quantize(x)[1]) and np.array_equal(q8.q.numpy(), f.quantize_rows(b.device.upload(x, dtype)).q.numpy())
    y, y_ok = shifted(b, zeros, dtype, by)
    f.dequantize_rows(q8, out=y)
    assert y_ok() and np.array_equal(y.numpy(), f.dequantize_rows(q8, dtype).numpy())
    go, gh_ok = shifted(b, x, dtype, by)
    gg, gg_ok = shifted(b, gm, "f32", by)
    f.rmsnorm_backward_q8(go, want.h8, want.rstd, gd, rd, out=(go, gg))
    wh, wg = f.rmsnorm_backward_q8(b.device.upload(x, dtype), want.h8, want.rstd, gm, b.device.upload(r, dtype))
    assert gh_ok() and gg_ok()
    # both sides have these roundings (see norm_backward_case)
    n = np.abs(want.h8.numpy().astype(np.float64)) * want.rstd.numpy()[:, None]
    g = np.abs(x * gm)
    part = want.rstd.numpy()[:, None] * (g + n * (g * n).mean(-1, keepdims=True)) + np.abs(r)
    tol = 2 * (part * (2 * features + 16) * U + (B if dtype == "bf16" else U) * np.abs(wh.numpy()))
    assert np.all(np.abs(go.numpy() - wh.numpy()) <= tol)
    assert np.all(np.abs(gg.numpy() - wg.numpy()) <= 2 * (2 * rows + 8) * U * (np.abs(x) * n).sum(0) + 1e-30)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (7, 5, 3), (70, 37, 41), (70, 40, 41), (70, 37, 48), (530, 263, 130), (600, 1026, 77)])
@pytest.mark.parametrize("by", [0, 1, 2, 3, 5, 7])
def test_gradients_whose_rows_are_copied(backend, M, N, K, by):
    """grad_out and weights that TMA cannot read, amid NaN that belongs to others; every choice of results gives the same."""
    b, lib, d = backend, backend.device.lib, backend.device
    rng = rng_for(29, M, N, K)
    xq, xs = R.quantize(acts(rng, M, K))
    g, w = R.bf16((0.01 * rng.standard_normal((M, N))).astype(np.float32)), R.bf16(rng.standard_normal((N, K)).astype(np.float32))
    x8 = put_rows8(b, xq, xs)

    def among_nans(x):
        flat = np.full(x.size + 64, np.nan, np.float32)
        flat[32 + by: 32 + by + x.size] = x.reshape(-1)
        buf = d.upload(flat, "bf16")
        return buf, DeviceTensor(d, buf.ptr + (32 + by) * 2, x.shape, "bf16", owned=False)

    gbuf, gd = among_nans(g)
    wbuf, wd = among_nans(w)
    want = b.fnn.linear_backward_q8(d.upload(g, "bf16"), x8, d.upload(w, "bf16"), dtype="f32")
    wants = R.linear_backward(g, xq * xs[:, None].astype(np.float64), w)
    for choice in range(1, 8):
        outs = [d.upload(np.full(t.shape, 7.0, np.float32)) for t in wants]
        d.check(lib.grilly_linear_backward_q8(d.ctx, gd.ptr, x8.q.ptr, x8.scale.ptr, wd.ptr if choice & 1 else None,
                                              *(o.ptr if choice >> i & 1 else None for i, o in enumerate(outs)), M, N, K, x8.ld, 0))
        for i, (o, t, e) in enumerate(zip(outs, want, wants)):
            if not choice >> i & 1:
                assert np.all(o.numpy() == 7)
                continue
            assert np.array_equal(o.numpy(), t.numpy())
            assert np.linalg.norm(o.numpy() - e) <= 4e-3 * np.linalg.norm(e)


@pytest.mark.parametrize("by", [1, 4])
def test_products_on_any_boundary(backend, by):
    """Scales, bias, gradients, weights and results that start off a 16-byte boundary; results keep to themselves."""
    b, f = backend, backend.fnn
    for M, N, K in ((5, 100, 64), (70, 264, 128), (300, 520, 1300)):
        rng = rng_for(23, M, N, K)
        xq, xs = R.quantize(acts(rng, M, K))
        wq, ws = R.quantize(acts(rng, N, K))
        bias = rng.standard_normal(N).astype(np.float32)
        x8, w8 = put_rows8(b, xq, xs), put_rows8(b, wq, ws)
        xv, wv = Rows8(x8.q, shifted(b, xs, "f32", by)[0], (M, K)), Rows8(w8.q, shifted(b, ws, "f32", by)[0], (N, K))
        for dtype in ("f32", "bf16"):
            y, ok = shifted(b, np.zeros((M, N), np.float32), dtype, by)
            f.linear_q8(xv, wv, shifted(b, bias, "f32", by)[0], act="silu", out=y)
            assert ok() and np.array_equal(y.numpy(), f.linear_q8(x8, w8, bias, act="silu", dtype=dtype).numpy())
            g, w = R.bf16(rng.standard_normal((M, N)).astype(np.float32)), R.bf16(rng.standard_normal((N, K)).astype(np.float32))
            gx, gx_ok = shifted(b, np.zeros((M, K), np.float32), dtype, by)
            gw, gw_ok = shifted(b, np.zeros((N, K), np.float32), dtype, by)
            gb, gb_ok = shifted(b, bias, "f32", by)
            f.linear_backward_q8(shifted(b, g, "bf16", by)[0], xv, shifted(b, w, "bf16", by)[0], out=(gx, gw, gb))
            want = f.linear_backward_q8(b.device.upload(g, "bf16"), x8, b.device.upload(w, "bf16"), dtype=dtype)
            assert gx_ok() and gw_ok() and gb_ok()
            assert np.array_equal(gx.numpy(), want[0].numpy()) and np.array_equal(gw.numpy(), want[1].numpy())
            assert np.all(np.abs(gb.numpy() - want[2].numpy()) <= 4 * M * U * np.abs(g.astype(np.float64)).sum(0))


def test_backward_outputs_by_themselves(backend):
    """The library computes the gradients that it is asked for, each the same as with the others."""
    d, lib = backend.device, backend.device.lib
    rng = rng_for(24)
    M, N, K = 300, 72, 200
    xq, xs = R.quantize(acts(rng, M, K))
    x8 = put_rows8(backend, xq, xs)
    g, w = d.upload(rng.standard_normal((M, N)).astype(np.float32), "bf16"), d.upload(rng.standard_normal((N, K)).astype(np.float32), "bf16")
    all3 = [t.numpy() for t in backend.fnn.linear_backward_q8(g, x8, w, dtype="f32")]
    for which in range(3):
        outs = [d.empty(s) if i == which else None for i, s in enumerate(((M, K), (N, K), (N,)))]
        p = [None if t is None else t.ptr for t in outs]
        d.check(lib.grilly_linear_backward_q8(d.ctx, g.ptr, x8.q.ptr, x8.scale.ptr, w.ptr if which == 0 else None, *p, M, N, K, x8.ld, 0))
        assert np.array_equal(outs[which].numpy(), all3[which])
    hs = backend.fnn.rmsnorm_backward_q8(backend.fnn.dequantize_rows(x8), x8, np.ones(M, np.float32))[0].numpy()
    gh = d.empty((M, K))
    go = backend.fnn.dequantize_rows(x8)
    one = d.upload(np.ones(M, np.float32))
    d.check(lib.grilly_rmsnorm_backward_q8(d.ctx, go.ptr, x8.q.ptr, x8.scale.ptr, one.ptr, None, None, gh.ptr, None, M, K, x8.ld, 0))
    assert np.array_equal(gh.numpy(), hs)


@pytest.mark.parametrize("features,outs", [(384, 200), (1001, 96), (4096, 264)])
def test_a_row_gives_the_same_bits_in_every_batch(backend, features, outs):
    """Norm, quantisation and product of a row do not depend on how many rows there are, whatever kernel they take."""
    f, rng = backend.fnn, rng_for(25, features)
    x, r = R.bf16(acts(rng, 700, features)), R.bf16(acts(rng, 700, features))
    w8 = f.quantize_rows((rng.standard_normal((outs, features)) * 0.05).astype(np.float32))
    put2 = lambda t, n: backend.device.upload(t[:n], "bf16")  # noqa: E731
    results = []
    for n in (700, 257, 33, 20, 3, 1):
        got = f.rmsnorm_residual_q8(put2(x, n), put2(r, n), keep=True)
        y = f.linear_q8(got.y8, w8, act="gelu")
        results.append([t.numpy()[:1] for t in (got.y8.q, got.y8.scale, got.h8.q, got.h8.scale, got.rstd, got.h, y, f.quantize_rows(put2(x, n)).q)])
    for one in results[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(results[0], one))


def test_rows_further_apart_than_they_need_be(backend):
    """8-bit rows with room between them are written and read like dense ones, and one row without leading dimensions is a row."""
    f, d, rng = backend.fnn, backend.device, rng_for(26)
    for rows, features in ((5, 33), (70, 384), (40, 1001)):
        x = acts(rng, rows, features)
        far = lambda: Rows8(d.empty((rows, (features + 15) // 16 * 16 + 48), "i8"), d.empty((rows,)), (rows, features))  # noqa: E731
        xd, w = d.upload(x), d.upload(rng.standard_normal((40, features)).astype(np.float32), "bf16")
        y8, h8 = far(), far()
        got = f.rmsnorm_residual_q8(xd, xd, keep=True, out=(y8, None, h8, None))
        want = f.rmsnorm_residual_q8(xd, xd, keep=True)
        q8, p8 = f.quantize_rows(xd, out=far()), f.quantize_rows(xd)
        for a, b in ((y8, want.y8), (h8, want.h8), (q8, p8)):
            assert np.array_equal(a.q.numpy()[:, :features], b.q.numpy()[:, :features]) and np.all(a.q.numpy()[:, features:] == 0)
            assert np.array_equal(a.scale.numpy(), b.scale.numpy()) and np.array_equal(f.dequantize_rows(a).numpy(), f.dequantize_rows(b).numpy())
        go = d.upload(rng.standard_normal((rows, features)).astype(np.float32))
        for a, b in zip(f.rmsnorm_backward_q8(go, h8, got.rstd), f.rmsnorm_backward_q8(go, want.h8, want.rstd)):
            assert np.array_equal(a.numpy(), b.numpy())
        g = d.upload(rng.standard_normal((rows, 40)).astype(np.float32), "bf16")
        for a, b in zip(f.linear_backward_q8(g, y8, w), f.linear_backward_q8(g, want.y8, w)):
            assert np.array_equal(a.numpy(), b.numpy())
        w8 = f.quantize_rows(w)
        assert np.array_equal(f.linear_q8(y8, w8).numpy(), f.linear_q8(want.y8, w8).numpy())
        one = f.rmsnorm_residual_q8(x[0], x[0], keep=True)
        assert one.y8.shape == (features,) and one.h.shape == (features,) and one.rstd.shape == (1,)
        assert np.array_equal(one.y8.q.numpy()[0], want.y8.q.numpy()[0])
        line = f.linear_q8(one.y8, w8)
        assert line.shape == (40,) and np.array_equal(line.numpy(), f.linear_q8(want.y8, w8).numpy()[0])
        gx, gw, gb = f.linear_backward_q8(rng.standard_normal(40).astype(np.float32), one.y8, w)
        assert gx.shape == (features,) and gw.shape == (40, features) and gb.shape == (40,)
        gh, gg = f.rmsnorm_backward_q8(gx, one.h8, one.rstd)
        assert gh.shape == (features,) and gg.shape == (features,)


def test_no_rows(backend):
    d, f = backend.device, backend.fnn
    e8, w = Rows8.empty(d, (0, 64)), np.ones((8, 64), np.float32)
    r8 = f.quantize_rows(d.empty((0, 64)))
    assert r8.rows == 0 and f.dequantize_rows(r8).numpy().shape == (0, 64)
    got = f.rmsnorm_residual_q8(d.empty((0, 64)), d.empty((0, 64)), keep=True)
    assert got.y8.rows == 0 and got.rstd.shape == (0,)
    assert f.linear_q8(e8, f.quantize_rows(w)).numpy().shape == (0, 8)
    gx, gw, gb = f.linear_backward_q8(d.empty((0, 8), "bf16"), e8, d.upload(w, "bf16"))
    assert gx.shape == (0, 64) and np.all(gw.numpy() == 0) and np.all(gb.numpy() == 0)
    gh, gg = f.rmsnorm_backward_q8(d.empty((0, 64)), e8, d.empty((0,)))
    assert gh.shape == (0, 64) and np.all(gg.numpy() == 0)


def test_library_refuses_bad_geometry(backend):
    """The C entry points check what a C caller hands them, before anything is launched."""
    d, lib = backend.device, backend.device.lib
    q, s, x = d.empty((4, 64), "i8"), d.empty((4,)), d.empty((4, 64))
    before = d.launch_count()
    bad = [lib.grilly_quantize_rows(d.ctx, x.ptr, q.ptr, s.ptr, 4, 64, 72, 0), lib.grilly_quantize_rows(d.ctx, x.ptr, q.ptr, s.ptr, 4, 64, 48, 0),
           lib.grilly_quantize_rows(d.ctx, x.ptr, q.ptr, s.ptr, -1, 64, 64, 0), lib.grilly_quantize_rows(d.ctx, x.ptr, q.ptr, s.ptr, 4, 0, 64, 0),
           lib.grilly_quantize_rows(d.ctx, None, q.ptr, s.ptr, 4, 64, 64, 0), lib.grilly_quantize_rows(d.ctx, x.ptr, q.ptr + 1, s.ptr, 3, 32, 32, 0),
           lib.grilly_dequantize_rows(d.ctx, q.ptr, None, x.ptr, 4, 64, 64, 0),
           lib.grilly_rmsnorm_residual_q8(d.ctx, x.ptr, None, None, None, q.ptr, s.ptr, None, None, None, 4, 64, 64, 0.0, 0),
           lib.grilly_rmsnorm_residual_q8(d.ctx, x.ptr, None, None, None, q.ptr, s.ptr, q.ptr, None, None, 4, 64, 64, 1e-5, 0),
           lib.grilly_linear_q8(d.ctx, q.ptr, s.ptr, q.ptr, s.ptr, None, x.ptr, 4, 4, 64, 64, 64, 9, 0),
           lib.grilly_linear_q8(d.ctx, q.ptr, s.ptr, q.ptr, s.ptr, None, x.ptr, 4, 0, 64, 64, 64, 0, 0),
           lib.grilly_linear_q8(d.ctx, q.ptr, s.ptr, q.ptr, s.ptr, None, None, 4, 4, 64, 64, 64, 0, 0),
           lib.grilly_linear_backward_q8(d.ctx, None, q.ptr, s.ptr, x.ptr, x.ptr, None, None, 4, 4, 64, 64, 0),
           lib.grilly_linear_backward_q8(d.ctx, x.ptr, q.ptr, s.ptr, None, x.ptr, None, None, 4, 4, 64, 64, 0),
           lib.grilly_rmsnorm_backward_q8(d.ctx, x.ptr, q.ptr, s.ptr, None, None, None, x.ptr, None, 4, 64, 64, 0)]
    # results over operands or over each other
    w, big = d.empty((4, 64), "bf16"), d.empty((8, 64))
    bad += [lib.grilly_quantize_rows(d.ctx, x.ptr, x.ptr, s.ptr, 4, 64, 64, 0), lib.grilly_dequantize_rows(d.ctx, q.ptr, s.ptr, q.ptr, 4, 64, 64, 0),
            lib.grilly_dequantize_rows(d.ctx, q.ptr, x.ptr + 512, x.ptr, 4, 64, 64, 0),
            lib.grilly_rmsnorm_residual_q8(d.ctx, x.ptr, None, None, None, q.ptr, s.ptr, q.ptr, x.ptr, None, 4, 64, 64, 1e-5, 0),
            lib.grilly_rmsnorm_residual_q8(d.ctx, x.ptr, None, None, None, q.ptr, s.ptr, None, None, s.ptr, 4, 64, 64, 1e-5, 0),
            lib.grilly_rmsnorm_residual_q8(d.ctx, big.ptr, None, None, big.ptr + 256, q.ptr, s.ptr, None, None, None, 4, 64, 64, 1e-5, 0),
            lib.grilly_linear_q8(d.ctx, q.ptr, s.ptr, q.ptr, s.ptr, None, q.ptr, 4, 4, 64, 64, 64, 0, 0),
            lib.grilly_linear_q8(d.ctx, q.ptr, s.ptr, q.ptr, s.ptr, x.ptr + 32, x.ptr, 4, 4, 64, 64, 64, 0, 0),
            lib.grilly_linear_backward_q8(d.ctx, w.ptr, q.ptr, s.ptr, x.ptr, w.ptr, None, None, 4, 64, 64, 64, 1),
            lib.grilly_linear_backward_q8(d.ctx, big.ptr, q.ptr, s.ptr, w.ptr, None, w.ptr, None, 4, 4, 64, 64, 1),
            lib.grilly_linear_backward_q8(d.ctx, w.ptr, q.ptr, s.ptr, x.ptr, big.ptr, big.ptr, None, 4, 4, 64, 64, 0),
            lib.grilly_rmsnorm_backward_q8(d.ctx, x.ptr, q.ptr, s.ptr, s.ptr, w.ptr, None, x.ptr, w.ptr, 4, 64, 64, 0),
            lib.grilly_rmsnorm_backward_q8(d.ctx, big.ptr, q.ptr, s.ptr, s.ptr, None, None, big.ptr + 256, None, 4, 64, 64, 0)]
    assert bad == [L.ERR_INVALID_ARG] * len(bad)
    many = [lib.grilly_quantize_rows(d.ctx, x.ptr, q.ptr, s.ptr, 1, (1 << 30) + 1, (1 << 30) + 16, 0),
            lib.grilly_quantize_rows(d.ctx, x.ptr, q.ptr, s.ptr, 1, 64, 1 << 32, 0), lib.grilly_quantize_rows(d.ctx, x.ptr, q.ptr, s.ptr, 1 << 55, 64, 64, 0),
            lib.grilly_linear_q8(d.ctx, q.ptr, s.ptr, q.ptr, s.ptr, None, x.ptr, 1, (1 << 30) + 1, 64, 64, 64, 0, 0)]
    assert many == [L.ERR_UNSUPPORTED] * len(many)
    assert lib.grilly_linear_q8(d.ctx, q.ptr, s.ptr, q.ptr, s.ptr, None, x.ptr, 1, 1, 131072, 131072, 131072, 0, 0) == L.ERR_UNSUPPORTED
    assert d.launch_count() == before


def test_offsets_past_32_bits(backend):
    """More than 2^31 elements: the last rows of a tensor are where they should be."""
    d, f = backend.device, backend.fnn
    rows, features = (1 << 31) // 4096 + 70, 4096
    x = d.empty((rows, features), "bf16")
    d.check(d.lib.grilly_memset(d.ctx, x.ptr, 0, x.nbytes))
    tail = acts(rng_for(17), 64, features)
    td, t = put(backend, tail, "bf16")
    d.check(d.lib.grilly_copy_2d(d.ctx, x.ptr + (rows - 64) * features * 2, features * 2, td.ptr, features * 2, features * 2, 64))
    got = f.rmsnorm_residual_q8(x, None, keep=True, out=(None, x, None, None))
    last = lambda r8: Rows8(DeviceTensor(d, r8.q.ptr + (rows - 64) * r8.ld, (64, r8.ld), "i8", owned=False),  # noqa: E731
                            DeviceTensor(d, r8.scale.ptr + (rows - 64) * 4, (64,), "f32", owned=False), (64, features))
    want = f.rmsnorm_residual_q8(td, None, keep=True)
    for a, w in ((got.y8, want.y8), (got.h8, want.h8)):
        assert np.array_equal(last(a).q.numpy(), w.q.numpy()) and np.array_equal(last(a).scale.numpy(), w.scale.numpy())
    y = f.dequantize_rows(got.h8, out=x)
    assert np.array_equal(DeviceTensor(d, y.ptr + (rows - 64) * features * 2, (64, features), "bf16", owned=False).numpy(),
                          f.dequantize_rows(want.h8, "bf16").numpy())
    gh, _ = f.rmsnorm_backward_q8(x, got.h8, got.rstd, out=(x, None))
    wh, _ = f.rmsnorm_backward_q8(f.dequantize_rows(want.h8, "bf16"), want.h8, want.rstd)
    assert np.array_equal(DeviceTensor(d, gh.ptr + (rows - 64) * features * 2, (64, features), "bf16", owned=False).numpy(), wh.numpy())
    w8 = f.quantize_rows(acts(rng_for(18), 24, features))
    out = f.linear_q8(got.y8, w8, dtype="bf16")
    tail_out = DeviceTensor(d, out.ptr + (rows - 64) * 24 * 2, (64, 24), "bf16", owned=False).numpy()
    assert np.array_equal(tail_out, f.linear_q8(last(got.y8), w8, dtype="bf16").numpy())


@pytest.mark.parametrize("values", [1 << 31, 1 << 32])
def test_offsets_past_32_bits_in_odd_rows(backend, values):
    """The same where rows start anywhere, and with more elements than 32 bits count."""
    d, f = backend.device, backend.fnn
    features = 4097
    rows = values // features // 8 * 8 + 72
    x = d.empty((rows, features), "bf16")
    d.check(d.lib.grilly_memset(d.ctx, x.ptr, 0, x.nbytes))
    td, _ = put(backend, acts(rng_for(30), 64, features), "bf16")
    at = (rows - 64) * features * 2
    d.check(d.lib.grilly_copy_2d(d.ctx, x.ptr + at, td.nbytes, td.ptr, td.nbytes, td.nbytes, 1))
    tail = lambda t: DeviceTensor(d, t.ptr + at, (64, features), "bf16", owned=False).numpy()  # noqa: E731
    got, want = f.rmsnorm_residual_q8(x, x, keep=True, out=(None, x, None, None)), f.rmsnorm_residual_q8(td, td, keep=True)
    assert np.array_equal(tail(x), want.h.numpy())
    for a, w in ((got.y8, want.y8), (got.h8, want.h8), (f.quantize_rows(x), f.quantize_rows(want.h))):
        end = DeviceTensor(d, a.q.ptr + (rows - 64) * a.ld, (64, a.ld), "i8", owned=False)
        assert np.array_equal(end.numpy(), w.q.numpy())
    gh, _ = f.rmsnorm_backward_q8(x, got.h8, got.rstd, None, x, out=(x, None))
    assert np.array_equal(tail(gh), f.rmsnorm_backward_q8(want.h, want.h8, want.rstd, None, want.h)[0].numpy())
    f.dequantize_rows(got.h8, out=x)
    assert np.array_equal(tail(x), f.dequantize_rows(want.h8, "bf16").numpy())


def test_gradients_past_32_bits_in_odd_rows(backend):
    """grad_out with more than 2^31 elements that TMA cannot read; all but the last rows are zero."""
    d, f = backend.device, backend.fnn
    rng = rng_for(31)
    N, K, last = 1077, 40, 600
    rows = (1 << 31) // N // 8 * 8 + last
    xq, xs = R.quantize(acts(rng, last, K))
    x8, end8 = Rows8.empty(d, (rows, K)), put_rows8(backend, xq, xs)
    go = d.empty((rows, N), "bf16")
    for t in (x8.q, x8.scale, go):
        d.check(d.lib.grilly_memset(d.ctx, t.ptr, 0, t.nbytes))
    ge, g = put(backend, (0.01 * rng.standard_normal((last, N))).astype(np.float32), "bf16")
    wd, w = put(backend, rng.standard_normal((N, K)).astype(np.float32), "bf16")
    for to, end in ((go.ptr + (rows - last) * N * 2, ge), (x8.q.ptr + (rows - last) * x8.ld, end8.q), (x8.scale.ptr + (rows - last) * 4, end8.scale)):
        d.check(d.lib.grilly_copy_2d(d.ctx, to, end.nbytes, end.ptr, end.nbytes, end.nbytes, 1))
    gx, gw, gb = f.linear_backward_q8(go, x8, wd, dtype="f32")
    wants = R.linear_backward(g, xq * xs[:, None].astype(np.float64), w)
    end = DeviceTensor(d, gx.ptr + (rows - last) * K * 4, (last, K), "f32", owned=False)
    for t, e in zip((end, gw, gb), wants):
        assert np.linalg.norm(t.numpy() - e) <= 4e-3 * np.linalg.norm(e)


def layer(b, x, r, gm, w8, wd, bias, target):
    """One training step's part: norm into 8 bits, product in 8 bits, gradient of sum(y * target) back to x."""
    f = b.fnn
    n = f.rmsnorm_residual_q8(x, r, gm, keep=True)
    y = f.linear_q8(n.y8, w8, bias, dtype="bf16")
    gy, gw, gb = f.linear_backward_q8(target, n.y8, wd)
    gh, gg = f.rmsnorm_backward_q8(gy, n.h8, n.rstd, gm)
    return n, y, gw, gb, gh, gg


@pytest.mark.parametrize("rows,features,outs", [(1, 384, 1536), (130, 512, 264), (2100, 384, 1536)])
def test_a_layer_forward_and_backward(backend_bf16, rows, features, outs):
    """Norm, product and both backward passes in a row stay within the quantisation's own noise of the exact layer."""
    b, rng = backend_bf16, rng_for(19, rows)
    xd, x = put(b, acts(rng, rows, features), "bf16")
    rd, r = put(b, rng.standard_normal((rows, features)).astype(np.float32), "bf16")
    gm = (1 + 0.2 * rng.standard_normal(features)).astype(np.float32)
    wd, w = put(b, (rng.standard_normal((outs, features)) * features ** -0.5).astype(np.float32), "bf16")
    bias = (0.1 * rng.standard_normal(outs)).astype(np.float32)
    td, t = put(b, rng.standard_normal((rows, outs)).astype(np.float32), "bf16")
    n, y, gw, gb, gh, gg = layer(b, xd, rd, gm, b.fnn.quantize_rows(wd), wd, bias, td)
    h, rstd, yn = R.rmsnorm(x, r, gm, EPS)
    gy, ww, wb = R.linear_backward(t, yn, w)
    wh, wg = R.rmsnorm_backward(gy, h, rstd, gm, None)
    rel = lambda a, want: np.linalg.norm(a.numpy() - want) / np.linalg.norm(want)  # noqa: E731
    # a step is amax / 127 with amax about 8 to 30 rms here, so each 8-bit operand is off by 30 / 127 / sqrt(12) = 7 % of
    # its rms at the very most
    assert rel(y, yn @ w.T + bias) < 0.14 and rel(gw, ww) < 0.07 and rel(gb, wb) < 1e-5 and rel(gh, wh) < 0.07 and rel(gg, wg) < 0.07
    again = layer(b, xd, rd, gm, b.fnn.quantize_rows(wd), wd, bias, td)
    for a, c in zip((y, gw, gb, gh, gg), again[1:]):
        assert np.array_equal(a.numpy(), c.numpy())


def test_captured_and_replayed(lib):
    """The layer in two CUDA graphs that are replayed at once on two streams of torch's, with inputs that change in between."""
    import torch

    import grilly_b200

    b = grilly_b200.Compute(precision="bf16")
    try:
        d, f, rng = b.device, b.fnn, rng_for(20)
        stream, other = torch.cuda.Stream(), torch.cuda.Stream()
        d.set_stream(stream.cuda_stream)
        rows, features, outs = 2100, 384, 264
        names = {torch.bfloat16: "bf16", torch.float32: "f32", torch.int8: "i8"}
        view = lambda t: DeviceTensor(d, t.data_ptr(), t.shape, names[t.dtype], owned=False)  # noqa: E731
        new = lambda *s, dtype=torch.bfloat16: torch.empty(s, dtype=dtype, device="cuda")  # noqa: E731
        wt = torch.tensor(rng.standard_normal((outs, features)), dtype=torch.bfloat16, device="cuda")
        gm = torch.tensor(1 + 0.2 * rng.standard_normal(features), dtype=torch.float32, device="cuda")
        torch.cuda.synchronize()
        w8 = f.quantize_rows(view(wt))

        def tensors():
            r8 = lambda: (new(rows, features, dtype=torch.int8), new(rows, dtype=torch.float32))  # noqa: E731
            t = {"x": new(rows, features), "go": new(rows, outs), "h": new(rows, features), "y8": r8(), "h8": r8(), "rstd": new(rows, dtype=torch.float32),
                 "y": new(rows, outs), "gx": new(rows, features), "gw": new(outs, features), "gb": new(outs, dtype=torch.float32),
                 "gh": new(rows, features), "gg": new(features, dtype=torch.float32)}
            return t

        def step(t):
            y8, h8 = (Rows8(view(q), view(s), (rows, features)) for q, s in (t["y8"], t["h8"]))
            f.rmsnorm_residual_q8(view(t["x"]), view(t["x"]), view(gm), keep=True, out=(y8, view(t["h"]), h8, view(t["rstd"])))
            f.linear_q8(y8, w8, out=view(t["y"]))
            f.linear_backward_q8(view(t["go"]), y8, view(wt), out=(view(t["gx"]), view(t["gw"]), view(t["gb"])))
            f.rmsnorm_backward_q8(view(t["gx"]), h8, view(t["rstd"]), view(gm), view(t["h"]), out=(view(t["gh"]), view(t["gg"])))

        outputs = ("h", "y", "gx", "gw", "gb", "gh", "gg")
        sets, graphs = [tensors(), tensors()], []
        with torch.cuda.stream(stream):
            for t in sets:
                t["x"].normal_()
                t["go"].normal_()
                step(t)                                               # the first call of each kernel is not captured
            stream.synchronize()
            for t in sets:
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=stream):
                    step(t)
                graphs.append(g)
            for _ in range(3):
                for t in sets:
                    t["x"].normal_()
                    t["go"].normal_()
                stream.synchronize()
                graphs[0].replay()
                with torch.cuda.stream(other):                        # at the same time as the first
                    graphs[1].replay()
                stream.synchronize()
                other.synchronize()
                got = [{k: t[k].clone() for k in outputs} for t in sets]
                for t in sets:
                    for k in outputs:
                        t[k].zero_()
                    step(t)
                stream.synchronize()
                for t, seen in zip(sets, got):
                    assert all(torch.equal(t[k], seen[k]) for k in outputs)
        del graphs
        d.sync()
    finally:
        b.cleanup()


def test_two_contexts_at_the_same_time(lib):
    """Two threads with a context (and stream) each: no scratch is shared."""
    import threading

    import grilly_b200

    def work(seed, out):
        b = grilly_b200.Compute(precision="bf16")
        try:
            rng = rng_for(21, seed)
            xd, _ = put(b, acts(rng, 1500, 512), "bf16")
            wd, _ = put(b, (rng.standard_normal((512, 512)) * 0.05).astype(np.float32), "bf16")
            td, _ = put(b, rng.standard_normal((1500, 512)).astype(np.float32), "bf16")
            w8 = b.fnn.quantize_rows(wd)
            runs = []
            for _ in range(6):
                n, y, gw, gb, gh, gg = layer(b, xd, xd, None, w8, wd, None, td)
                runs.append([t.numpy() for t in (y, gw, gb, gh, gg)])
            out[seed] = runs
        finally:
            b.cleanup()

    out = {}
    threads = [threading.Thread(target=work, args=(s, out)) for s in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(out) == [0, 1]
    for runs in out.values():
        for r in runs[1:]:
            assert all(np.array_equal(a, c) for a, c in zip(runs[0], r))


def test_library_refuses_tensors_off_their_own_boundary(backend):
    """An fp32 tensor off a 4-byte boundary, a bf16 one off a 2-byte boundary: refused by every entry point, nothing launched."""
    d, lib = backend.device, backend.device.lib
    q, q2, s, s2, s3 = d.empty((4, 64), "i8"), d.empty((4, 64), "i8"), d.empty((8,)), d.empty((8,)), d.empty((8,))
    x, y, z, g, w = (d.empty((8, 64)) for _ in range(5))
    before = d.launch_count()

    def quantize(a=0, b=0, flags=0):
        return lib.grilly_quantize_rows(d.ctx, x.ptr + a, q.ptr, s.ptr + b, 4, 64, 64, flags)

    def dequantize(a=0, b=0, flags=0):
        return lib.grilly_dequantize_rows(d.ctx, q.ptr, s.ptr + a, x.ptr + b, 4, 64, 64, flags)

    def norm(by=(0,) * 7, flags=0):
        return lib.grilly_rmsnorm_residual_q8(d.ctx, x.ptr + by[0], y.ptr + by[1], g.ptr + by[2], z.ptr + by[3], q.ptr, s.ptr + by[4],
                                              q2.ptr, s2.ptr + by[5], s3.ptr + by[6], 4, 64, 64, 1e-5, flags)

    def linear(by=(0,) * 4, flags=0):
        return lib.grilly_linear_q8(d.ctx, q.ptr, s.ptr + by[0], q2.ptr, s2.ptr + by[1], s3.ptr + by[2], x.ptr + by[3], 4, 4, 64, 64, 64, 0, flags)

    def linear_backward(by=(0,) * 6, flags=0):
        return lib.grilly_linear_backward_q8(d.ctx, x.ptr + by[0], q.ptr, s.ptr + by[1], w.ptr + by[2], y.ptr + by[3], z.ptr + by[4], s3.ptr + by[5],
                                             4, 4, 64, 64, flags)

    def norm_backward(by=(0,) * 7, flags=0):
        return lib.grilly_rmsnorm_backward_q8(d.ctx, x.ptr + by[0], q.ptr, s.ptr + by[1], s2.ptr + by[2], g.ptr + by[3], y.ptr + by[4],
                                              z.ptr + by[5], w.ptr + by[6], 4, 64, 64, flags)

    bad = [quantize(1), quantize(2), quantize(0, 2), quantize(1, 0, L.FLAG_IN_BF16), dequantize(1), dequantize(0, 2), dequantize(0, 3, L.FLAG_OUT_BF16)]
    for call, n in ((norm, 7), (linear, 4), (linear_backward, 6), (norm_backward, 7)):
        for i in range(n):
            for flags in (0, L.FLAG_IN_BF16 | L.FLAG_OUT_BF16):
                bad += [call(tuple(by if j == i else 0 for j in range(n)), flags) for by in (1, 3)]
    bad += [norm((2, 0, 0, 0, 0, 0, 0)), norm((0, 0, 0, 2, 0, 0, 0)), linear((0, 0, 0, 2)), linear_backward((0, 0, 0, 2, 0, 0)),
            norm_backward((2, 0, 0, 0, 0, 0, 0)), norm_backward((0, 0, 0, 0, 0, 2, 0))]
    assert bad == [L.ERR_INVALID_ARG] * len(bad) and d.launch_count() == before
    # bf16 tensors on any 2-byte boundary are taken
    both = L.FLAG_IN_BF16 | L.FLAG_OUT_BF16
    for t in (x, y, z, g, w, s, s2, s3, q, q2):
        d.check(lib.grilly_memset(d.ctx, t.ptr, 0, t.nbytes))
    assert [quantize(2, 0, both), dequantize(0, 2, both), norm((2, 6, 0, 2, 0, 0, 0), both), linear((0, 0, 0, 2), both),
            linear_backward((2, 0, 2, 2, 2, 0), both), norm_backward((2, 0, 0, 0, 2, 2, 0), both)] == [L.OK] * 6
    d.sync()
