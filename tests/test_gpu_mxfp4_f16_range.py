"""The linears on 4-bit weights at the ends of f16: x in f16 takes weights as f16 holds them."""
import pytest

torch = pytest.importorskip("torch")

import mxfp4_reference as ref  # noqa: E402
from test_gpu_mxfp4 import dev, ops, tokens  # noqa: E402,F401

pytestmark = pytest.mark.gpu

ROWS = [4, 40, 515]  # few rows in one tile and two, tiles


@pytest.mark.parametrize("m", ROWS)
def test_f16_takes_weights_as_f16_holds_them(ops, dev, m):
    """Block scales 2^-40 to 2^13: subnormal weights are rounded, small ones vanish, large ones are exact."""
    k, n = 512, 600
    g = torch.Generator().manual_seed(m)
    codes = torch.randint(0, 16, (n, k), generator=g).to(torch.uint8).to(dev)
    s = torch.randint(127 - 40, 127 + 14, (n, k // 32), generator=g).to(dev)
    s[:200] = torch.randint(127 - 28, 127 - 20, (200, k // 32), generator=g).to(dev)
    w = ref.pack(codes, s)
    x = tokens(dev, m, k, "f16")
    held = ref.dense(*w).to(torch.float32).to(torch.float16)
    assert torch.isfinite(held).all() and not torch.equal(held[:200].double(), ref.dense(*w)[:200])
    y = ops.mxfp4_linear(x, *w, out_dtype=torch.float32)
    ref.check(y, *ref.product(x, held, None), "f16")
    for arith, wide in (("plain", x.bfloat16()), ("fp4", x)):  # exact in the others
        linear = ops.mxfp4_linear_fp4 if arith == "fp4" else ops.mxfp4_linear
        xd = ref.values(*ref.quantize(x)) if arith == "fp4" else wide.double()
        ref.check(linear(wide, *w, out_dtype=torch.float32), *ref.product(xd, ref.dense(*w), None), arith)


@pytest.mark.parametrize("m", ROWS)
def test_f16_weights_past_its_range_are_infinite(ops, dev, m):
    """Block scale 2^14: 3 * 2^14 is held, 4 and 6 * 2^14 are infinite, in their own columns; bf16 holds them all."""
    k, n = 96, 600
    codes = torch.randint(0, 4, (n, k), generator=torch.Generator().manual_seed(1)).to(torch.uint8).to(dev)
    codes[100, 40], codes[101, 40], codes[102, 40], codes[103, 40] = 5, 6, 7, 15
    s = torch.full((n, k // 32), 120, device=dev)
    s[100:104, 1] = 127 + 14
    w = ref.pack(codes, s)
    x = tokens(dev, m, k, "f16").abs() + 0.5  # every product with them has their sign
    x = x.clamp(max=2.0)
    y = ops.mxfp4_linear(x, *w, out_dtype=torch.float32)
    inf = float("inf")
    for col, want in ((101, inf), (102, inf), (103, -inf)):
        assert bool((y[:, col] == want).all())
    keep = torch.ones(n, dtype=torch.bool, device=dev)
    keep[101:104] = False
    ref.check(y[:, keep], *ref.product(x, ref.dense(*w)[keep], None), "the columns beside")
    assert torch.equal(torch.isinf(ops.mxfp4_dequantize(*w, torch.float16)), torch.isinf(ref.dense(*w).half()))
    ref.check(ops.mxfp4_linear(x.bfloat16(), *w, out_dtype=torch.float32), *ref.product(x.bfloat16(), ref.dense(*w), None), "bf16")
    gate = ref.pack(torch.zeros_like(codes), s)
    y = ops.mxfp4_linear_gated(x, gate, w, "silu", gate_bias=torch.ones(n, device=dev), out_dtype=torch.float32)
    assert bool((y[:, 101:103] == inf).all() and (y[:, 103] == -inf).all()) and torch.isfinite(y[:, keep]).all()
