"""The gated linear's activations against 64 bits, at the accuracy that include/lux3d_fused.h states for them, in every kernel.

The gate's sums are its biases: x is zero, so every product is. `up` is one the same way, so y is the activation itself and
the rounding to y's type."""
import math

import pytest

torch = pytest.importorskip("torch")

import mxfp4_reference as ref  # noqa: E402
from test_gpu_mxfp4 import ACTS, DT, dev, ops, weight  # noqa: E402,F401

pytestmark = pytest.mark.gpu

# x's type, in 4 bits, m, k, n: few rows of every way in, and each tile of test_gpu_mxfp4_tiles.py that gated calls take, some
# with rows past the last one
SIZES = [("bf16", False, 1, 32, 4001), ("f32", False, 16, 160, 4001), ("bf16", True, 5, 32, 4001), ("f16", False, 40, 32, 4001),
         ("f32", False, 773, 32, 1219), ("f32", False, 587, 1120, 589), ("bf16", False, 321, 96, 5662), ("f16", False, 484, 1152, 456),
         ("bf16", False, 452, 3840, 391), ("f16", False, 1156, 160, 1748), ("bf16", False, 2959, 32, 3815),
         ("bf16", False, 1032, 96, 7700), ("bf16", True, 835, 288, 1167), ("bf16", True, 1228, 288, 1491), ("bf16", True, 2817, 544, 5389)]


def grid(dev, n):
    """n gates: both tails of every activation, densely around zero, powers of two, the ends of f32."""
    ends = [0.0, -0.0, 1e-30, -1e-30, 2.0 ** -140, -2.0 ** -140, 5.5, -5.5, 37.5, -37.5, 300.0, -300.0, 1e6, -1e6, 3e38, -3e38]
    mid = (n - len(ends)) // 2
    v = torch.cat([torch.tensor(ends, dtype=torch.float64), torch.linspace(-110, 40, mid, dtype=torch.float64),
                   torch.linspace(-7, 7, n - len(ends) - mid, dtype=torch.float64)])
    return v.float().to(dev)


def exact(v, act):
    """The activation of v, and v times its slope."""
    v = v.double()
    if act == "gelu_erf":
        # not torch's ndtr, which loses the tail: 14% off at -8.14
        sig, grow = 0.5 * torch.special.erfc(-v * math.sqrt(0.5)), torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    else:
        c = 2 * math.sqrt(2 / math.pi)
        z, dz = (v, torch.ones_like(v)) if act == "silu" else (c * (v + 0.044715 * v ** 3), c * (1 + 3 * 0.044715 * v * v))
        sig = torch.sigmoid(z)
        grow = sig * torch.sigmoid(-z) * dz
    far = v.abs() > 1e5  # v * v * 0
    return v * sig, torch.where(far, v * sig, v * (sig + v * torch.where(far, 0.0, grow)))


def activated(ops, dev, dt, fp4, m, k, n, act, out, gate_bias):
    w = weight(dev, n, k)
    x = torch.zeros((m, k), dtype=DT[dt], device=dev)
    return ops.mxfp4_linear_gated(x, w, w, act, gate_bias=gate_bias, up_bias=torch.ones(n, device=dev), fp4=fp4, out_dtype=DT[out])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dt,fp4,m,k,n", SIZES)
def test_f32_results(ops, dev, dt, fp4, m, k, n, act):
    """12 u of the activation of a value within 4 u of v. In front: exp2 and the reciprocal within 1 ulp (2 u each), erfc's form
    2 u by its fit, its t and polynomial 2 u each, the roundings of the factor, of 1 - q or 1 + exp2 and of the product.
    Exponent: tanh GELU's v^2, its polynomial's two steps and the product with v 3.5 u, erf GELU's v^2, sum and product less,
    SiLU's one product 1.2 u. Subnormal results and sigmoids may be lost."""
    v = grid(dev, n)
    y = activated(ops, dev, dt, fp4, m, k, n, act, "f32", v)
    want, slope = exact(v, act)
    over = (y.double() - want).abs() - (12 * ref.U * want.abs() + 4 * ref.U * slope.abs() + v.double().abs() * 2.0 ** -126 + 2.0 ** -149)
    worst = int(over.max(0).values.argmax())
    assert torch.isfinite(y).all() and float(over.max()) <= 0, (act, float(v[worst]), float(y[0, worst]), float(want[worst]))


@pytest.mark.parametrize("out", ["bf16", "f16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dt,fp4,m,k,n", SIZES)
def test_2_byte_results(ops, dev, dt, fp4, m, k, n, act, out):
    """Half a step of the type on top of what the header states: 2e-5 of the value; erf GELU below -5.5 2.4e-8; nothing of
    results under |v| 2^-126."""
    v = grid(dev, n)
    v = torch.where(v.abs() < 60000, v, torch.full_like(v, 2.0))
    y = activated(ops, dev, dt, fp4, m, k, n, act, out, v)
    want = exact(v, act)[0]
    bound = 2e-5 * want.abs() + v.double().abs() * 2.0 ** -126
    if act == "gelu_erf":
        bound = bound + torch.where(v < -5.5, 2.4e-8, 0.0)
    ref.check(y, want.expand(m, n), bound.expand(m, n), f"{act} {dt} {m} x {k} -> {n} {out}")


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dt,fp4,m,k,n", SIZES[2:6])
def test_infinities(ops, dev, dt, fp4, m, k, n, act, out):
    """+inf stays, NaN stays, and -inf times the sigmoid's zero is NaN, as in v * sigmoid(v)."""
    v = torch.zeros(n, device=dev)
    v[1], v[2], v[3] = float("inf"), float("-inf"), float("nan")
    y = activated(ops, dev, dt, fp4, m, k, n, act, out, v).float()
    assert bool((y[:, 1] == float("inf")).all()) and torch.isnan(y[:, 2:4]).all() and not y[:, 4:].any() and not y[:, 0].any()
