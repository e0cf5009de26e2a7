"""The 8-bit row operators at the ends of fp32's range, against the formulas in 64 bits.

Tolerances are those of the ordinary sizes (U is half a step of fp32): a value beyond fp32's range on the way to a result that
is inside it is no reason for a larger one."""
import numpy as np
import pytest

from test_gpu_rows8 import acts, put, rng_for

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
