"""The linears on 4-bit weights with f32 x near the ends of f32, where its three bf16 terms end."""
import pytest

torch = pytest.importorskip("torch")

import mxfp4_reference as ref  # noqa: E402
from test_gpu_mxfp4 import dev, ops, tokens, weight  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [4, 40, 515])
def test_f32_at_its_ends(ops, dev, m):
    """Exact up to 2^128 (1 - 2^-9), the last value that bf16 does not round to infinity; NaN above, in its own row; below
    about 2^-110 off by less than 2^-126 a value."""
    k, n = 256, 600
    w = weight(dev, n, k)
    x = tokens(dev, m, k, "f32")
    last = torch.tensor(0x7F7F7FFF, dtype=torch.int32).view(torch.float32).item()
    x[0] *= 2.0 ** -112
    x[1, 7] = last
    dense = ref.dense(*w)
    y = ops.mxfp4_linear(x, *w)
    want, bound = ref.product(x, dense, None, 2 * ref.U)
    bound[0] += k * 2.0 ** -126 * float(dense.abs().max())
    fits = want.abs() + bound < 3.4e38
    assert torch.isfinite(y[fits]).all()
    ref.check(y[fits], want[fits], bound[fits], "ends")
    for v in (torch.tensor(0x7F7F8000, dtype=torch.int32).view(torch.float32).item(), 3.4028234e38, float("inf"), float("nan")):
        x[2, 9] = v
        z = ops.mxfp4_linear(x, *w)
        keep = torch.arange(m, device=dev) != 2
        assert torch.isnan(z[2]).all() and torch.equal(z[keep], y[keep])
