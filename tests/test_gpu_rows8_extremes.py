"""The 8-bit row operators at the ends of fp32's range and at the borders between kernels, against the formulas in 64 bits.

Tolerances are those of the ordinary sizes (U is half a step of fp32): a value beyond fp32's range on the way to a result that
is inside it is no reason for a larger one."""
import numpy as np
import pytest

from grilly_b200 import DeviceTensor, Rows8
from oracle import rows8 as R

from test_gpu_rows8 import EPS, U, acts, check_quantised, linear_case, put, rng_for

pytestmark = pytest.mark.gpu

# teams of 16 to 512 threads, odd rows, a block per row
FEATURES = [16, 384, 1001, 2048, 4096, 9000, 16001, 20000]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("features", FEATURES)
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_a_gamma_that_is_not_finite_leaves_the_checkpoint_alone(backend, features, dtype, value):
    """h, its 8-bit rows and rstd do not depend on gamma; every row of y has a column that is not finite."""
    b, f = backend, backend.fnn
    rng = rng_for(40, features)
    xd, x = put(b, acts(rng, 37, features), dtype)
    rd, r = put(b, rng.standard_normal((37, features)).astype(np.float32), dtype)
    gamma = np.ones(features, np.float32)
    want = f.rmsnorm_residual_q8(xd, rd, gamma, keep=True)
    gamma[rng.integers(features)] = value
    got = f.rmsnorm_residual_q8(xd, rd, gamma, keep=True)
    for a, w in ((got.h, want.h), (got.h8.q, want.h8.q), (got.h8.scale, want.h8.scale), (got.rstd, want.rstd)):
        assert np.array_equal(a.numpy(), w.numpy())
    assert np.isfinite(want.rstd.numpy()).all()
    assert np.isnan(got.y8.scale.numpy()).all() and np.all(got.y8.q.numpy() == 0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("features", FEATURES)
def test_a_norm_that_overflows_has_no_bytes(backend, features, dtype):
    """y = h rstd gamma above fp32's range although h gamma is inside it: scale NaN, q = 0, the row's checkpoint as ever."""
    b, f = backend, backend.fnn
    x = acts(rng_for(41, features), 20, features)
    x[:, 3] = 2 * np.abs(x).max(-1)          # the row's largest: its normalised value is above 1
    x *= 0.01 / np.abs(x).max(-1, keepdims=True)
    xd, x = put(b, x, dtype)
    gamma = np.ones(features, np.float32)
    gamma[3] = 3.4e38
    got = f.rmsnorm_residual_q8(xd, None, gamma, eps=1e-12, keep=True)
    h, rstd, y = R.rmsnorm(x, None, gamma, 1e-12)
    assert np.all(y[:, 3] > 3.5e38) and np.abs(h * gamma).max() < 1e37
    assert np.isnan(got.y8.scale.numpy()).all() and np.all(got.y8.q.numpy() == 0)
    check_quantised(got.h8, h, U)
    assert np.all(np.abs(got.rstd.numpy() - rstd) <= (features / 4 + 16) * U * rstd)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("features", FEATURES)
@pytest.mark.parametrize("size,scale,eps", [(1e4, 1e36, EPS), (1e-25, 1e-20, 1e-30), (1e-30, 1e-15, 1e-34)])
def test_products_with_gamma_outside_the_range_of_fp32(backend, features, dtype, size, scale, eps):
    """h gamma overflows, or is a number of a few bits or 0, while y = h rstd gamma is an ordinary number. Every second row
    is an ordinary one."""
    b, f = backend, backend.fnn
    rng = rng_for(42, features)
    rows = 41
    x = acts(rng, rows, features)
    x[::2] *= np.float32(size)
    xd, x = put(b, x, dtype)
    gamma = (scale * (1 + 0.3 * rng.standard_normal(features))).astype(np.float32)
    got = f.rmsnorm_residual_q8(xd, None, gamma, eps=eps, keep=True)
    h, rstd, y = R.rmsnorm(x, None, gamma, float(np.float32(eps)))
    assert np.abs(y).max() < 3e38
    # the tolerances of test_rmsnorm_residual_q8
    rel = (features / 4 + 16) * U
    check_quantised(got.y8, y, rel + 4 * U)
    check_quantised(got.h8, h, U)
    assert np.all(np.abs(got.rstd.numpy() - rstd) <= rel * rstd)


@pytest.mark.parametrize("features", FEATURES)
@pytest.mark.parametrize("eps", [1e-38, 1e-40, 4e-45])
def test_a_zero_row_with_the_smallest_eps(backend, features, eps):
    """rstd = 1 / sqrt(eps) where eps is below the smallest normal number; gamma of zeros gives zeros."""
    got = backend.fnn.rmsnorm_residual_q8(backend.device.upload(np.zeros((3, features), np.float32)), eps=eps, keep=True)
    want = 1 / np.sqrt(float(np.float32(eps)))
    # the inverse root to 2 ulp, improved by a step whose own roundings are below an ulp
    assert np.all(np.abs(got.rstd.numpy() - want) <= 4 * U * want)
    assert np.all(got.y8.scale.numpy() == R.TINY) and np.all(got.y8.q.numpy() == 0)
    x = backend.device.upload(acts(rng_for(43), 3, features))
    y8 = backend.fnn.rmsnorm_residual_q8(x, None, np.zeros(features, np.float32), eps=eps).y8
    assert np.all(y8.scale.numpy() == R.TINY) and np.all(y8.q.numpy() == 0)


@pytest.mark.parametrize("N,K", [(6144, 4096), (6160, 4096), (6144, 4112), (4096, 8192), (100, 4112), (2048, 16400), (2064, 16400)])
@pytest.mark.parametrize("M", [16, 17, 32, 33])
def test_linear_q8_where_one_kernel_gives_way_to_the_other(backend, M, N, K):
    """Few tokens under large weights, on both sides of the rule that chooses the kernel: right, and a token has the same bits."""
    got, _ = linear_case(backend, M, N, K, "silu", True, "f32", seed=1)
    b, f = backend, backend.fnn
    rng = rng_for(6, M, N, K, 1)            # the operands of linear_case
    xq, xs = R.quantize(acts(rng, M, K))
    wq, ws = R.quantize((rng.standard_normal((N, K)) * K ** -0.5).astype(np.float32))
    bias = (0.1 * rng.standard_normal(N)).astype(np.float32)
    def rows8(q, s):
        buf = np.zeros((len(q), (K + 15) // 16 * 16), np.int8)
        buf[:, :K] = q
        return Rows8(b.device.upload(buf, "i8"), b.device.upload(np.asarray(s, np.float32)), (len(q), K))
    one = f.linear_q8(rows8(xq[M - 1:], xs[M - 1:]), rows8(wq, ws), bias, act="silu").numpy()
    assert np.array_equal(got.numpy()[M - 1:], one)


@pytest.mark.parametrize("M", [1, 20, 40, 200, 2000])
def test_linear_q8_of_the_largest_rows_that_stay_in_range(backend, M):
    """|x| = 2^104 in every one of 131071 columns: the sum times the row's scale is just inside fp32's range."""
    K, N = 131071, 70
    xs, ws = np.full(M, np.float32(2.0 ** 104 / 127)), np.full(N, np.float32(1e-30))
    def rows8(n, s):
        return Rows8(backend.device.upload(np.full((n, K + 1), 127, np.int8), "i8"), backend.device.upload(s), (n, K))
    got = backend.fnn.linear_q8(rows8(M, xs), rows8(N, ws)).numpy()
    want = K * 127.0 * 127.0 * float(xs[0]) * float(ws[0])
    assert np.all(np.abs(got - want) <= 4 * U * want)     # the sum, two products and the result round once each


def test_the_longest_row(backend):
    """2^30 features, the most there may be: the row's ends are where they should be, the zeros between them are zeros."""
    d, f, rng = backend.device, backend.fnn, rng_for(44)
    F = 1 << 30
    x = d.empty((1, F), "bf16")
    d.check(d.lib.grilly_memset(d.ctx, x.ptr, 0, x.nbytes))
    ends = R.bf16(rng.standard_normal((1, 128)).astype(np.float32))
    for at, part in ((0, ends[:, :64]), ((F - 64) * 2, ends[:, 64:])):
        t = d.upload(part, "bf16")
        d.check(d.lib.grilly_copy_2d(d.ctx, x.ptr + at, t.nbytes, t.ptr, t.nbytes, t.nbytes, 1))
    q, s = R.quantize(ends)

    def view(t, first, n):
        item = {"i8": 1, "bf16": 2}[t.dtype]
        return DeviceTensor(d, t.ptr + first * item, (n,), t.dtype, owned=False).numpy()

    def check(r8):
        assert np.array_equal(view(r8.q, 0, 64), q[0, :64]) and np.array_equal(view(r8.q, F - 64, 64), q[0, 64:])
        assert not view(r8.q, 64, 4096).any() and not view(r8.q, F - 4160, 4096).any()

    r8 = f.quantize_rows(x)
    check(r8)
    assert np.array_equal(r8.scale.numpy(), s)
    got = f.rmsnorm_residual_q8(x, eps=1e-12, keep=True, out=(None, x, None, None))
    check(got.y8)
    check(got.h8)
    rstd = R.rmsnorm(ends, None, None, 0.0)[1] * np.sqrt(F / 128)       # eps is 8e-6 of the mean square
    assert abs(got.rstd.numpy()[0] - rstd[0]) <= (128 * U + 1e-5) * rstd[0]
    back = f.dequantize_rows(r8, out=x)
    assert np.array_equal(view(back, F - 64, 64), R.bf16((q[0, 64:] * s[0].astype(np.float64)).astype(np.float32)))


@pytest.mark.parametrize("features", [384, 1001, 4096, 17000])
def test_next_to_ties(backend, features):
    """fp32 values a few roundings away from ties: the nearest integer but for what is closer to a tie than half a step of the
    fp32 quotient (2^-18 at 64 to 127), and the documented distance from x."""
    rng = rng_for(45, features)
    a = rng.uniform(1, 2, (64, 1)) * 2.0 ** rng.integers(-60, 60, (64, 1))
    x = a * (rng.integers(-127, 127, (64, features)) + 0.5 + rng.uniform(-1, 1, (64, features)) * 2.0 ** rng.uniform(-26, -12, (64, features))) / 127
    x[:, 5] = a[:, 0]
    x = x.astype(np.float32)
    a = np.abs(x).max(-1, keepdims=True).astype(np.float64)
    steps = 127 * x.astype(np.float64) / a
    xd = backend.device.upload(x)
    in_range = (x.astype(np.float64) ** 2).sum(-1) < 3e38          # the others are infinite rows to the norm
    for r8, rows in ((backend.fnn.quantize_rows(xd), slice(None)), (backend.fnn.rmsnorm_residual_q8(xd, keep=True).h8, in_range)):
        q, s = r8.q.numpy()[rows, :features].astype(np.float64), r8.scale.numpy()[rows, None].astype(np.float64)
        assert np.all(np.abs(q - steps[rows]) <= 0.5 + 2.0 ** -18)
        clear = np.abs(steps[rows] - np.floor(steps[rows]) - 0.5) > 2.0 ** -18
        assert clear.mean() > 0.3 and np.array_equal(q[clear], np.rint(steps[rows][clear]))
        assert np.all(np.abs(q * s - x[rows]) <= (0.5 + 2.0 ** -16) * s)
