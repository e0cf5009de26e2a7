"""The 8-bit row operators without a GPU: what their Python entry points refuse before anything reaches the library, and
the oracle's own formulas (its gradients against differences)."""
import ctypes as C

import numpy as np
import pytest

from grilly_b200 import _lib as L
from grilly_b200.device import DeviceTensor
from grilly_b200.rows8 import Rows8, Rows8Ops
from oracle import rows8 as R


class FakeLib:
    """Counts what reaches the library; every call reports success."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


class FakeDevice:
    def __init__(self):
        self.lib, self.next = FakeLib(), 4096

    def empty(self, shape, dtype="f32"):
        self.next += 1 << 20
        return DeviceTensor(self, self.next, shape, dtype, owned=False)

    def upload(self, arr, dtype="f32", round_tf32=False):
        return self.empty(np.shape(arr), dtype)

    def check(self, rc):
        assert rc == 0


class FakeFNN(Rows8Ops):
    def __init__(self):
        self.dev = FakeDevice()
        self.lib, self.ctx = self.dev.lib, 1


@pytest.fixture
def fnn():
    return FakeFNN()


def rows8(f, *shape):
    return Rows8.empty(f.dev, shape)


def test_rows8_geometry(fnn):
    d = fnn.dev
    r = Rows8.empty(d, (2, 3, 33))
    assert (r.rows, r.features, r.ld, r.q.shape) == (6, 33, 48, (6, 48)) and r.nbytes == 6 * 48 + 24
    for q, s, shape in ((d.empty((6, 33), "i8"), d.empty((6,)), (6, 33)),       # pitch not a multiple of 16
                        (d.empty((6, 32), "i8"), d.empty((6,)), (6, 33)),       # pitch below the features
                        (d.empty((5, 48), "i8"), d.empty((6,)), (6, 33)),       # too few rows
                        (d.empty((6, 48), "i8"), d.empty((5,)), (6, 33)),       # too few scales
                        (d.empty((6, 48), "f32"), d.empty((6,)), (6, 33)),      # not bytes
                        (d.empty((6, 48), "i8"), d.empty((6,), "bf16"), (6, 33)),
                        (d.empty((6, 48), "i8"), FakeDevice().empty((6,)), (6, 33)),
                        (d.empty((6, 48), "i8"), d.empty((6,)), (6, 0))):
        with pytest.raises(ValueError):
            Rows8(q, s, shape)
    with pytest.raises(ValueError):
        Rows8.empty(d, (4, 0))


def refusals():
    f32, other = (lambda f, *s: f.dev.empty(s)), (lambda f, *s: FakeDevice().empty(s))
    b16 = lambda f, *s: f.dev.empty(s, "bf16")  # noqa: E731
    i32 = lambda f, *s: f.dev.empty(s, "i32")  # noqa: E731
    return {
        "quantize int": lambda f: f.quantize_rows(i32(f, 4, 8)),
        "quantize scalar": lambda f: f.quantize_rows(np.float32(3)),
        "quantize no features": lambda f: f.quantize_rows(np.zeros((3, 0), np.float32)),
        "quantize foreign": lambda f: f.quantize_rows(other(f, 4, 8)),
        "quantize out shape": lambda f: f.quantize_rows(f32(f, 4, 8), out=rows8(f, 4, 9)),
        "quantize out foreign": lambda f: f.quantize_rows(f32(f, 4, 8), out=Rows8.empty(FakeDevice(), (4, 8))),
        "quantize out float": lambda f: f.quantize_rows(f32(f, 4, 8), out=f32(f, 4, 8)),
        "dequantize float": lambda f: f.dequantize_rows(f32(f, 4, 8)),
        "dequantize dtype": lambda f: f.dequantize_rows(rows8(f, 4, 8), dtype="f16"),
        "dequantize out type": lambda f: f.dequantize_rows(rows8(f, 4, 8), out=i32(f, 4, 8)),
        "dequantize out shape": lambda f: f.dequantize_rows(rows8(f, 4, 8), out=f32(f, 8, 4)),
        "norm residual shape": lambda f: f.rmsnorm_residual_q8(f32(f, 4, 8), f32(f, 4, 9)),
        "norm residual type": lambda f: f.rmsnorm_residual_q8(f32(f, 4, 8), b16(f, 4, 8)),
        "norm gamma size": lambda f: f.rmsnorm_residual_q8(f32(f, 4, 8), gamma=np.ones(7, np.float32)),
        "norm gamma type": lambda f: f.rmsnorm_residual_q8(f32(f, 4, 8), gamma=b16(f, 8)),
        "norm eps zero": lambda f: f.rmsnorm_residual_q8(f32(f, 4, 8), eps=0.0),
        "norm eps nan": lambda f: f.rmsnorm_residual_q8(f32(f, 4, 8), eps=float("nan")),
        "norm eps inf": lambda f: f.rmsnorm_residual_q8(f32(f, 4, 8), eps=float("inf")),
        "norm out without keep": lambda f: f.rmsnorm_residual_q8(f32(f, 4, 8), out=(None, None, rows8(f, 4, 8), None)),
        "norm out h type": lambda f: f.rmsnorm_residual_q8(f32(f, 4, 8), out=(None, b16(f, 4, 8), None, None)),
        "norm out pitches": lambda f: f.rmsnorm_residual_q8(f32(f, 4, 8), keep=True, out=(
            None, None, Rows8(f.dev.empty((4, 32), "i8"), f32(f, 4), (4, 8)), None)),
        "norm foreign residual": lambda f: f.rmsnorm_residual_q8(f32(f, 4, 8), other(f, 4, 8)),
        "linear features": lambda f: f.linear_q8(rows8(f, 4, 8), rows8(f, 5, 9)),
        "linear weights 3-D": lambda f: f.linear_q8(rows8(f, 4, 8), rows8(f, 5, 2, 8)),
        "linear no outputs": lambda f: f.linear_q8(rows8(f, 4, 8), rows8(f, 0, 8)),
        "linear act": lambda f: f.linear_q8(rows8(f, 4, 8), rows8(f, 5, 8), act="tanh"),
        "linear dtype": lambda f: f.linear_q8(rows8(f, 4, 8), rows8(f, 5, 8), dtype="i8"),
        "linear bias": lambda f: f.linear_q8(rows8(f, 4, 8), rows8(f, 5, 8), bias=np.ones(4, np.float32)),
        "linear too wide": lambda f: f.linear_q8(rows8(f, 1, 131072), rows8(f, 1, 131072)),
        "linear out shape": lambda f: f.linear_q8(rows8(f, 4, 8), rows8(f, 5, 8), out=f32(f, 5, 4)),
        "linear foreign weights": lambda f: f.linear_q8(rows8(f, 4, 8), Rows8.empty(FakeDevice(), (5, 8))),
        "linear_backward float rows": lambda f: f.linear_backward_q8(b16(f, 4, 5), f32(f, 4, 8), b16(f, 5, 8)),
        "linear_backward grad shape": lambda f: f.linear_backward_q8(b16(f, 4, 6), rows8(f, 4, 8), b16(f, 5, 8)),
        "linear_backward grad rows": lambda f: f.linear_backward_q8(b16(f, 3, 5), rows8(f, 4, 8), b16(f, 5, 8)),
        "linear_backward grad type": lambda f: f.linear_backward_q8(f32(f, 4, 5), rows8(f, 4, 8), b16(f, 5, 8)),
        "linear_backward weights": lambda f: f.linear_backward_q8(b16(f, 4, 5), rows8(f, 4, 8), b16(f, 5, 7)),
        "linear_backward out types": lambda f: f.linear_backward_q8(b16(f, 4, 5), rows8(f, 4, 8), b16(f, 5, 8), out=(
            f32(f, 4, 8), b16(f, 5, 8), None)),
        "linear_backward out i32": lambda f: f.linear_backward_q8(b16(f, 4, 5), rows8(f, 4, 8), b16(f, 5, 8), out=(
            i32(f, 4, 8), None, None)),
        "linear_backward out bias": lambda f: f.linear_backward_q8(b16(f, 4, 5), rows8(f, 4, 8), b16(f, 5, 8), out=(
            None, None, b16(f, 5))),
        "norm_backward shape": lambda f: f.rmsnorm_backward_q8(f32(f, 4, 9), rows8(f, 4, 8), f32(f, 4)),
        "norm_backward rstd": lambda f: f.rmsnorm_backward_q8(f32(f, 4, 8), rows8(f, 4, 8), f32(f, 5)),
        "norm_backward no rstd": lambda f: f.rmsnorm_backward_q8(f32(f, 4, 8), rows8(f, 4, 8), None),
        "norm_backward rstd type": lambda f: f.rmsnorm_backward_q8(f32(f, 4, 8), rows8(f, 4, 8), b16(f, 4)),
        "norm_backward types": lambda f: f.rmsnorm_backward_q8(f32(f, 4, 8), rows8(f, 4, 8), f32(f, 4), grad_residual=b16(f, 4, 8)),
        "norm_backward gamma": lambda f: f.rmsnorm_backward_q8(f32(f, 4, 8), rows8(f, 4, 8), f32(f, 4), gamma=f32(f, 9)),
        "norm_backward out": lambda f: f.rmsnorm_backward_q8(f32(f, 4, 8), rows8(f, 4, 8), f32(f, 4), out=(b16(f, 4, 8), None)),
    }


@pytest.mark.parametrize("name", sorted(refusals()))
def test_refused_before_the_library_is_reached(fnn, name):
    with pytest.raises((ValueError, TypeError)):
        refusals()[name](fnn)
    assert not fnn.lib.calls


def test_accepted_calls_hand_over_the_geometry(fnn):
    fnn.linear_q8(rows8(fnn, 2, 3, 33), rows8(fnn, 7, 33), act="gelu", dtype="bf16")
    name, a = fnn.lib.calls[-1]
    assert name == "grilly_linear_q8" and a[7:] == (6, 7, 33, 48, 48, L.ACT_GELU, L.FLAG_OUT_BF16)
    x = fnn.dev.empty((4, 8), "bf16")
    got = fnn.rmsnorm_residual_q8(x, x, keep=True, out=(None, x, None, None))     # h in place of x
    name, a = fnn.lib.calls[-1]
    assert got.h is x and a[4] == x.ptr and a[-1] == L.FLAG_IN_BF16 and got.h8.rows == 4 and got.rstd.shape == (4,)


def test_null_context_is_an_error_code(lib):
    n = (None,) * 12
    assert lib.grilly_quantize_rows(*n[:4], 1, 1, 16, 0) == L.ERR_INVALID_ARG
    assert lib.grilly_dequantize_rows(*n[:4], 1, 1, 16, 0) == L.ERR_INVALID_ARG
    assert lib.grilly_rmsnorm_residual_q8(*n[:10], 1, 1, 16, C.c_float(1e-5), 0) == L.ERR_INVALID_ARG
    assert lib.grilly_linear_q8(*n[:7], 1, 1, 1, 16, 16, 0, 0) == L.ERR_INVALID_ARG
    assert lib.grilly_linear_backward_q8(*n[:8], 1, 1, 1, 16, 0) == L.ERR_INVALID_ARG
    assert lib.grilly_rmsnorm_backward_q8(*n[:9], 1, 1, 16, 0) == L.ERR_INVALID_ARG


def test_oracle_quantises_to_half_a_step():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((50, 37)) * np.exp(rng.uniform(-30, 30, (50, 1)))).astype(np.float32)
    x[3], x[4] = 0, 1e-44
    q, s = R.quantize(x)
    assert np.abs(q).max() == 127 and np.all(q[3] == 0)
    assert np.all(np.abs(q * s[:, None].astype(np.float64) - x) <= 0.5000001 * s[:, None].astype(np.float64))
    x[5, 2], x[6, 1] = np.nan, -np.inf
    q, s = R.quantize(x)
    assert np.isnan(s[[5, 6]]).all() and np.all(q[[5, 6]] == 0) and np.isfinite(s[7:]).all()


def test_oracle_gradients_against_differences():
    rng = np.random.default_rng(1)
    h, go, gamma = rng.standard_normal((3, 7)), rng.standard_normal((3, 7)), rng.standard_normal(7)
    eps, d = 1e-5, 1e-6
    rstd = R.rmsnorm(h, None, gamma, eps)[1]
    gh, gg = R.rmsnorm_backward(go, h, rstd, gamma, None)
    loss = lambda hh, gm: (go * R.rmsnorm(hh, None, gm, eps)[2]).sum()  # noqa: E731
    for i in range(3):
        for j in range(7):
            e = np.zeros_like(h)
            e[i, j] = d
            assert abs((loss(h + e, gamma) - loss(h - e, gamma)) / (2 * d) - gh[i, j]) < 1e-4   # eps in rstd: h^2 >> eps
    for j in range(7):
        e = np.zeros(7)
        e[j] = d
        assert abs((loss(h, gamma + e) - loss(h, gamma - e)) / (2 * d) - gg[j]) < 1e-6


def test_waits_for_the_other_cta_acquire_at_cluster_scope():
    """In the kernels of CTA pairs, a barrier on which threads of the other CTA arrive is waited for by mbar_wait_cluster."""
    import re
    from pathlib import Path

    import grilly_b200

    found = 0
    for path in sorted((Path(grilly_b200.__file__).parent / "csrc").glob("*.cu*")):
        text = path.read_text()
        remote = dict(re.findall(r"const uint32_t (\w+) = map_to_cta\(&(\w+)\[", text))
        for address in re.findall(r"mbar_arrive(?:_release)?_cluster\((\w+) [+]", text):
            barrier = remote[address]
            waits = re.findall(r"\b(mbar_wait\w*)\(&" + barrier + r"\[", text)
            assert waits and set(waits) == {"mbar_wait_cluster"}, (path.name, barrier, waits)
            found += 1
    assert found >= 3


def test_half_a_step_and_the_rounding_of_the_scale():
    """|q scale - x| <= (1/2 + 2^-17) scale: x is at most half a step from q max / 127, and the scale at most 2^-24 of itself
    from max / 127, up to 127 times. Half a step alone is not a bound."""
    rng = np.random.default_rng(2)
    x = R.bf16((rng.standard_normal((300, 4000)) * np.exp(rng.uniform(-3, 3, (300, 1)))).astype(np.float32))
    # next to a tie at 126.5 steps, on the side that the rounded scale is worse for
    a = np.abs(x).max(-1).astype(np.float64)
    x[:, 0] = np.float32(a * 126.5 / 127)
    x[:, 1] = np.float32(a)
    q, s = R.quantize(x)
    steps = np.abs(q * s[:, None].astype(np.float64) - x) / s[:, None].astype(np.float64)
    assert 0.5 < steps.max() <= 0.5 + 2.0 ** -17
