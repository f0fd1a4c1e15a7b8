"""A gated feed-forward block on 4-bit weights whose result has a type of its own."""
import math

import pytest

torch = pytest.importorskip("torch")

from test_gpu_mxfp4 import DT, dev, ops, rnd, tokens, weight  # noqa: E402,F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [6, 300])
@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
def test_feed_forward_result_has_its_own_type(ops, dev, m, fp4, out):
    """Hidden values keep x's type: here past f16's largest, where the result is not."""
    c, h = 256, 512
    gate, up = (ops.Mxfp4MatMul(*weight(dev, h, c, seed=i)) for i in (1, 2))
    down = ops.Mxfp4MatMul.from_dense(rnd(dev, c, h, seed=3, std=1e-2 / math.sqrt(h)))
    x = tokens(dev, m, c, "bf16").clamp(-4, 4)
    big = torch.full((h,), 300.0, device=dev)
    mlp = ops.Mxfp4GatedMlp(gate, up, down, "silu", gate_bias=big, up_bias=big, fp4=fp4)
    pairs = [x] + ([ops.mxfp4_quantize(x)] if fp4 else [])
    for given in pairs:
        hidden = ops.mxfp4_linear_gated(given, (gate.q, gate.scales), (up.q, up.scales), "silu", gate_bias=big, up_bias=big, fp4=fp4)
        assert hidden.dtype == torch.bfloat16 and float(hidden.abs().max()) > 65504
        z = mlp.forward(given, out_dtype=DT[out])
        assert z.dtype == DT[out] and torch.isfinite(z).all()
        assert torch.equal(z, down.forward(hidden, None, DT[out], fp4))
    assert mlp.forward(x).dtype == torch.bfloat16
