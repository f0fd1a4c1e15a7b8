"""What the Python entries of the linears on 4-bit weights pass on and refuse, without a GPU."""
import pytest

torch = pytest.importorskip("torch")

from lux3d_fused import _lib, ops  # noqa: E402,F401


def packed(n, k):
    return torch.zeros((n, k // 2), dtype=torch.uint8), torch.zeros(((k + 127) // 128, n, 4), dtype=torch.uint8)


@pytest.mark.parametrize("out", [None, torch.float16, torch.float32])
@pytest.mark.parametrize("fp4", [False, True])
def test_feed_forward_types(monkeypatch, fp4, out):
    """The result's type is the down-projection's alone; the hidden values have x's."""
    seen = {}

    def gated(x, gate, up, act="silu", *, gate_bias=None, up_bias=None, fp4=False, out_dtype=None):
        seen["hidden"] = out_dtype
        return x

    def linear(x, q, scales, bias=None, out_dtype=None):
        seen["result"] = out_dtype
        return x

    monkeypatch.setattr(ops, "mxfp4_linear_gated", gated)
    monkeypatch.setattr(ops, "mxfp4_linear", linear)
    monkeypatch.setattr(ops, "mxfp4_linear_fp4", linear)
    w = ops.Mxfp4MatMul(*packed(64, 64))
    ops.Mxfp4GatedMlp(w, w, w, fp4=fp4).forward(torch.zeros((2, 64), dtype=torch.bfloat16), out_dtype=out)
    assert seen == {"hidden": None, "result": out}


def test_a_pair_where_x_is_taken_as_it_is():
    """A packed x belongs to the forms that take x in 4 bits."""
    w = packed(64, 64)
    x = packed(4, 64)
    for call in (lambda: ops.mxfp4_linear(x, *w), lambda: ops.mxfp4_linear_gated(x, w, w),
                 lambda: ops.mxfp4_linear_gated(list(x), w, w, fp4=False), lambda: ops.Mxfp4MatMul(*w).forward(x),
                 lambda: ops.Mxfp4GatedMlp(*[ops.Mxfp4MatMul(*w)] * 3).forward(x)):
        with pytest.raises(_lib.Lux3dError, match="x must be a tensor") as e:
            call()
        assert e.value.code == _lib.ERR_VALUE
    for call in (lambda: ops.mxfp4_linear_fp4((x[0],), *w), lambda: ops.mxfp4_linear_gated((*x, x[0]), w, w, fp4=True),
                 lambda: ops.mxfp4_linear_fp4((None, x[1]), *w)):
        with pytest.raises(_lib.Lux3dError, match="pair") as e:
            call()
        assert e.value.code == _lib.ERR_VALUE


@pytest.mark.parametrize("exponents,code", [
    (torch.zeros(8, dtype=torch.uint8), _lib.ERR_SHAPE), (torch.zeros((2, 3, 4), dtype=torch.uint8), _lib.ERR_SHAPE),
    (torch.zeros((4, 8), dtype=torch.int32), _lib.ERR_DTYPE), (torch.zeros((4, 8)), _lib.ERR_DTYPE)])
def test_scales_of_another_form(exponents, code):
    with pytest.raises(_lib.Lux3dError, match="u8 \\[rows, k / 32\\]") as e:
        ops.mxfp4_scales(exponents)
    assert e.value.code == code
