"""Every form of the few-rows kernel of the linears on 4-bit weights: test_mxfp4_few_rows_cpu.py holds its choice to FEW."""
import pytest

torch = pytest.importorskip("torch")

import mxfp4_reference as ref  # noqa: E402,F401
from test_gpu_mxfp4 import dev, ops, rnd, run_gated, run_linear, tokens, weight  # noqa: E402,F401

pytestmark = pytest.mark.gpu

# tiles of 16 rows of x, weight tiles, wavefronts of a workgroup; x's way in: 2-byte values as they are, or f32 / 4 bits; gated;
# m, k, n. From 6144 of k on one weight tile takes 16 wavefronts.
FEW = [(1, 1, 16, two, gated, m, k, n) for two in (True, False) for gated in (False, True)
       for m, k, n in ((1, 6144, 130), (5, 8192, 2048), (16, 6176, 77), (13, 6272, 1), (16, 8192, 2048))]
FEW += [(1, 1, 8, two, gated, m, k, n) for two in (True, False) for gated in (False, True)
        for m, k, n in ((1, 6112, 130), (16, 6112, 77))]
FEW += [(1, 2, 8, two, gated, m, k, n) for two, gated, m, k, n in ((True, False, 16, 6176, 8200), (False, False, 7, 544, 8199),
                                                                   (True, True, 16, 6144, 16385), (False, True, 9, 1056, 16390))]
FEW += [(1, 4, 8, two, False, m, k, n) for two, m, k, n in ((True, 16, 1024, 24577), (False, 11, 6144, 16385))]
FEW += [(2, 1, 8, two, gated, m, k, n) for two in (True, False) for gated in (False, True) for m, k, n in ((17, 6176, 77), (33, 160, 130))]


@pytest.mark.parametrize("mt,nt,nw,two,gated,m,k,n", FEW)
def test_few_rows(ops, dev, mt, nt, nw, two, gated, m, k, n):
    for dt, arith in (("bf16", "plain"), ("f16", "plain")) if two else (("f32", "plain"), ("bf16", "fp4"), ("f16", "fp4"), ("f32", "fp4")):
        out = "f32" if m % 2 else "same"
        if gated:
            run_gated(ops, dev, m, k, n, dt, arith, "gelu_erf", out, use_bias=m != 5)
        else:
            run_linear(ops, dev, m, k, n, dt, arith, out, use_bias=m != 5)


@pytest.mark.parametrize("m,k,n", [(1, 6144, 130), (5, 8192, 2048), (16, 6176, 77), (16, 6176, 8200), (11, 6144, 16385)])
def test_packed_x_is_the_quantized_x(ops, dev, m, k, n):
    x, w, v, bias = tokens(dev, m, k, "bf16"), weight(dev, n, k), weight(dev, n, k, 1), rnd(dev, n)
    pair = ops.mxfp4_quantize(x)
    assert torch.equal(ops.mxfp4_linear_fp4(pair, *w, bias=bias), ops.mxfp4_linear_fp4(x, *w, bias=bias))
    assert torch.equal(ops.mxfp4_linear_gated(pair, v, w, fp4=True), ops.mxfp4_linear_gated(x, v, w, fp4=True))


@pytest.mark.parametrize("arith", ["plain", "fp4"])
def test_a_row_that_is_not_finite_stays_alone(ops, dev, arith):
    m, k, n = 9, 6176, 77
    x, w, bias, y = run_linear(ops, dev, m, k, n, "bf16", arith)
    x[3, 6170] = float("nan")
    z = (ops.mxfp4_linear_fp4 if arith == "fp4" else ops.mxfp4_linear)(x, *w, bias=bias)
    keep = torch.arange(m, device=dev) != 3
    assert torch.isnan(z[3]).all() and torch.equal(z[keep], y[keep])
