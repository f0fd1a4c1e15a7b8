"""The linears on 4-bit weights where rows lie so far apart that the kernel of many rows cannot address them: the few-rows kernel
takes them, 32-bit offsets in none of its parts."""
import pytest

torch = pytest.importorskip("torch")

import mxfp4_reference as ref  # noqa: E402
from test_gpu_mxfp4 import DT, dev, ops, rnd, tokens, weight  # noqa: E402,F401

pytestmark = pytest.mark.gpu

# How x enters, gated, m, k, n, elements between rows of x and of y: sizes that the kernel of many rows takes when rows lie
# close (test_mxfp4_far_rows_cpu.py), and cannot address here
FAR = [("2byte", False, 100, 512, 4096, 2 ** 22 + 64, None), ("2byte", False, 100, 512, 4096, None, 2 ** 21 + 8),
       ("2byte", True, 100, 512, 4096, 2 ** 22 + 64, None), ("f32", False, 100, 512, 4096, 2 ** 21 + 64, None),
       ("f32", True, 100, 512, 4096, None, 2 ** 21 + 8), ("fp4", False, 100, 512, 4096, None, 2 ** 21 + 8),
       ("fp4", True, 100, 512, 4096, None, 2 ** 21 + 8)]


def rows_apart(dev, m, cols, apart, dt):
    if apart is None:
        return torch.empty((m, cols), dtype=dt, device=dev)
    return torch.empty((m - 1) * apart + cols, dtype=dt, device=dev).as_strided((m, cols), (apart, 1))


@pytest.mark.parametrize("kind,gated,m,k,n,x_apart,y_apart", FAR)
def test_rows_far_apart(ops, dev, kind, gated, m, k, n, x_apart, y_apart):
    from lux3d_fused import _lib
    dt = "f32" if kind == "f32" else "bf16"
    x = rows_apart(dev, m, k, x_apart, DT[dt])
    x.copy_(tokens(dev, m, k, dt))
    y = rows_apart(dev, m, n, y_apart, DT[dt])
    w, v, bias = weight(dev, n, k), weight(dev, n, k, 1), rnd(dev, n, std=0.3)
    x4 = ops.mxfp4_quantize(x) if kind == "fp4" else (None, None)
    xd = ref.dense(*x4) if kind == "fp4" else x.double()
    e = 2 * ref.U if kind == "f32" else 0.0
    d, plain = ops._d, None if kind == "fp4" else x
    if gated:
        _lib.call("lux3d_mxfp4_linear_gated", d(plain), d(x4[0]), d(x4[1]), d(v[0]), d(v[1]), None, d(w[0]), d(w[1]), d(bias), 2,
                  int(kind == "fp4"), d(y), ops._stream(x))
        want = ref.gated(ref.product(xd, ref.dense(*v), None, e), ref.product(xd, ref.dense(*w), bias, e), "silu")
    else:
        if kind == "fp4":
            _lib.call("lux3d_mxfp4_linear_fp4", None, d(x4[0]), d(x4[1]), d(w[0]), d(w[1]), d(bias), d(y), ops._stream(x))
        else:
            _lib.call("lux3d_mxfp4_linear", d(x), d(w[0]), d(w[1]), d(bias), d(y), ops._stream(x))
        want = ref.product(xd, ref.dense(*w), bias, e)
    ref.check(y, *want, f"{kind} {m} x {k} -> {n}, rows {x_apart} and {y_apart} apart")
