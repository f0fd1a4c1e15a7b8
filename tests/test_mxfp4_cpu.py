"""The lux3d_mxfp4_* entries refuse invalid arguments on the host, before any HIP call (the descriptors point at fake
addresses that are never dereferenced: every call here must fail validation), and the 64-bit reference of their GPU tests
agrees with the format's definition."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import mxfp4_reference as ref  # noqa: E402
from lux3d_fused import _lib, ops  # noqa: E402

FAKE = 0x100000


def T(shape, dtype=_lib.BF16, strides=None, data=FAKE):
    if strides is None:
        strides, acc = [], 1
        for n in reversed(shape):
            strides.insert(0, acc)
            acc *= n
    return ctypes.pointer(_lib.descriptor(data, dtype, shape, strides))


def U8(*shape, **kw):
    return T(list(shape), _lib.U8, **kw)


QUANT = dict(x=T([10, 160]), q=U8(10, 80), scales=U8(2, 10, 4), stream=None)
PACKED = [
    (dict(q=None), _lib.ERR_NULL, "`q`"),
    (dict(scales=None), _lib.ERR_NULL, "`scales`"),
    (dict(q=T([10, 80], _lib.I8)), _lib.ERR_DTYPE, "u8"),
    (dict(scales=T([2, 10, 4], _lib.F32)), _lib.ERR_DTYPE, "u8"),
    (dict(q=U8(800)), _lib.ERR_SHAPE, "rows, k / 2"),
    (dict(q=U8(10, 0)), _lib.ERR_SHAPE, "multiple of 32"),
    (dict(q=U8(10, 72)), _lib.ERR_SHAPE, "multiple of 32"),
    (dict(scales=U8(10, 5)), _lib.ERR_SHAPE, "[2, 10, 4]"),
    (dict(scales=U8(1, 10, 4)), _lib.ERR_SHAPE, "[2, 10, 4]"),
    (dict(scales=U8(2, 11, 4)), _lib.ERR_SHAPE, "[2, 10, 4]"),
    (dict(q=U8(10, 80, strides=[96, 1])), _lib.ERR_LAYOUT, "contiguous"),
    (dict(scales=U8(2, 10, 4, strides=[4, 8, 1])), _lib.ERR_LAYOUT, "contiguous"),
    (dict(q=U8(10, 80, data=FAKE + 8)), _lib.ERR_LAYOUT, "aligned"),
    (dict(scales=U8(2, 10, 4, data=FAKE + 2)), _lib.ERR_LAYOUT, "aligned"),
    (dict(q=U8(11, 80), scales=U8(2, 11, 4)), _lib.ERR_SHAPE, "10, 160"),
    (dict(q=U8(10, 96), scales=U8(2, 10, 4)), _lib.ERR_SHAPE, "10, 160"),
]


@pytest.mark.parametrize("change,code,text", PACKED + [
    (dict(x=None), _lib.ERR_NULL, "`x`"),
    (dict(x=T([10, 160], _lib.I32)), _lib.ERR_DTYPE, "f32/bf16/f16"),
    (dict(x=T([10, 150])), _lib.ERR_SHAPE, "multiple of 32"),
    (dict(x=T([10, 0])), _lib.ERR_SHAPE, "multiple of 32"),
    (dict(x=T([10, 160], strides=[320, 2])), _lib.ERR_LAYOUT, "innermost"),
    (dict(x=T([10, 160], strides=[164, 1])), _lib.ERR_LAYOUT, "aligned"),
    (dict(x=T([10, 160], data=FAKE + 2)), _lib.ERR_LAYOUT, "aligned"),
    (dict(x=T([10, 160], strides=[80, 1])), _lib.ERR_LAYOUT, "overlap"),
])
def test_quantize_refusals(change, code, text):
    rc, msg = _lib.call_status("lux3d_mxfp4_quantize", *{**QUANT, **change}.values())
    assert rc == code and text in msg, (rc, msg)


@pytest.mark.parametrize("change,code,text", PACKED[:-2] + [
    (dict(y=T([11, 160])), _lib.ERR_SHAPE, "y must be [10, 160]"),
    (dict(y=T([10, 192])), _lib.ERR_SHAPE, "y must be [10, 160]"),
    (dict(y=None), _lib.ERR_NULL, "`y`"),
    (dict(y=T([10, 160], _lib.U8)), _lib.ERR_DTYPE, "f32/bf16/f16"),
    (dict(y=T([10, 160], data=FAKE + 4)), _lib.ERR_LAYOUT, "aligned"),
])
def test_dequantize_refusals(change, code, text):
    good = dict(q=QUANT["q"], scales=QUANT["scales"], y=T([10, 160]), stream=None)
    rc, msg = _lib.call_status("lux3d_mxfp4_dequantize", *{**good, **change}.values())
    assert rc == code and text in msg, (rc, msg)


LINEAR = dict(x=T([10, 160]), w=U8(40, 80), w_scales=U8(2, 40, 4), bias=None, y=T([10, 40]), stream=None)
LINEAR4 = dict(x=T([30, 160]), xq=U8(30, 80), xs=U8(2, 30, 4), w=U8(40, 80), w_scales=U8(2, 40, 4), bias=None, y=T([30, 40]),
               stream=None)
GATED = dict(x=T([30, 160]), xq=U8(30, 80), xs=U8(2, 30, 4), gate=U8(40, 80), gate_scales=U8(2, 40, 4), gate_bias=None,
             up=U8(40, 80), up_scales=U8(2, 40, 4), up_bias=None, act=2, fp4=1, y=T([30, 40]), stream=None)


@pytest.mark.parametrize("change,code,text", [
    (dict(x=None), _lib.ERR_NULL, "`x`"),
    (dict(w=None), _lib.ERR_NULL, "`w`"),
    (dict(y=None), _lib.ERR_NULL, "`y`"),
    (dict(x=T([10, 160], _lib.I8)), _lib.ERR_DTYPE, "f32/bf16/f16"),
    (dict(x=T([10, 192])), _lib.ERR_SHAPE, "192 features, the weight 160"),
    (dict(x=T([10, 160], data=FAKE + 8)), _lib.ERR_LAYOUT, "aligned"),
    (dict(y=T([10, 41])), _lib.ERR_SHAPE, "y must be [10, 40]"),
    (dict(y=T([11, 40])), _lib.ERR_SHAPE, "y must be [10, 40]"),
    (dict(y=T([10, 40], _lib.U8)), _lib.ERR_DTYPE, "f32/bf16/f16"),
    (dict(w_scales=U8(40, 2, 4)), _lib.ERR_SHAPE, "[2, 40, 4]"),
    (dict(bias=T([40])), _lib.ERR_SHAPE, "f32 [40]"),
    (dict(bias=T([39], _lib.F32)), _lib.ERR_SHAPE, "f32 [40]"),
])
def test_linear_refusals(change, code, text):
    rc, msg = _lib.call_status("lux3d_mxfp4_linear", *{**LINEAR, **change}.values())
    assert rc == code and text in msg, (rc, msg)


SHARED = [
    (dict(xq=None), _lib.ERR_NULL, "`xq`"),
    (dict(xs=None), _lib.ERR_NULL, "`xs`"),
    (dict(x=None, xq=None, xs=None), _lib.ERR_NULL, "`xq`"),
    (dict(xq=U8(29, 80), xs=U8(2, 29, 4)), _lib.ERR_SHAPE, "30, 160"),
    (dict(x=T([10, 160]), y=T([10, 40]), xs=None), _lib.ERR_NULL, "`xs`"),
    (dict(x=T([30, 192]), xq=U8(30, 96), xs=U8(2, 30, 4)), _lib.ERR_SHAPE, "192 features"),
    (dict(x=None, xq=U8(30, 96), xs=U8(2, 30, 4)), _lib.ERR_SHAPE, "192 features"),
    (dict(x=None, y=T([31, 40])), _lib.ERR_SHAPE, "y must be [30, 40]"),
]


@pytest.mark.parametrize("change,code,text", SHARED + [
    (dict(w_scales=None), _lib.ERR_NULL, "`w_scales`"),
    (dict(bias=T([39], _lib.F32)), _lib.ERR_SHAPE, "f32 [40]"),
])
def test_linear_fp4_refusals(change, code, text):
    rc, msg = _lib.call_status("lux3d_mxfp4_linear_fp4", *{**LINEAR4, **change}.values())
    assert rc == code and text in msg, (rc, msg)


@pytest.mark.parametrize("change,code,text", SHARED + [
    (dict(act=3), _lib.ERR_VALUE, "activation 3"),
    (dict(act=-1), _lib.ERR_VALUE, "activation -1"),
    (dict(fp4=2), _lib.ERR_VALUE, "fp4"),
    (dict(fp4=0), _lib.ERR_VALUE, "fp4 1"),
    (dict(fp4=0, x=None, xq=None, xs=None), _lib.ERR_NULL, "`x`"),
    (dict(gate=None), _lib.ERR_NULL, "`gate`"),
    (dict(up_scales=None), _lib.ERR_NULL, "`up_scales`"),
    (dict(gate=U8(41, 80), gate_scales=U8(2, 41, 4)), _lib.ERR_SHAPE, "`up` [40, 160]"),
    (dict(up=U8(40, 96)), _lib.ERR_SHAPE, "`up` [40, 192]"),
    (dict(gate_bias=T([41], _lib.F32)), _lib.ERR_SHAPE, "gate_bias"),
    (dict(up_bias=T([40], _lib.F16)), _lib.ERR_SHAPE, "up_bias"),
])
def test_gated_refusals(change, code, text):
    rc, msg = _lib.call_status("lux3d_mxfp4_linear_gated", *{**GATED, **change}.values())
    assert rc == code and text in msg, (rc, msg)


def test_python_refusals():
    x = torch.zeros(4, 64)
    q, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1, 4, 4, dtype=torch.uint8)
    for call in (lambda: ops.mxfp4_quantize(x), lambda: ops.mxfp4_dequantize(q, s), lambda: ops.mxfp4_linear(x, q, s),
                 lambda: ops.mxfp4_linear_fp4(x, q, s), lambda: ops.mxfp4_linear_fp4((q, s), q, s),
                 lambda: ops.mxfp4_linear_gated(x, (q, s), (q, s))):
        with pytest.raises(_lib.Lux3dError, match="must be on a GPU"):
            call()
    with pytest.raises(_lib.Lux3dError, match="act must be one of"):
        ops.mxfp4_linear_gated(x, (q, s), (q, s), "relu")


def test_grouped_scales():
    e = torch.arange(1, 19, dtype=torch.uint8).view(2, 9)
    g = ops.mxfp4_scales(e)
    assert g.shape == (3, 2, 4) and g.is_contiguous()
    assert g[0].tolist() == [[1, 2, 3, 4], [10, 11, 12, 13]] and g[2].tolist() == [[9, 0, 0, 0], [18, 0, 0, 0]]


def test_reference_by_hand():
    row = torch.zeros(1, 64)
    row[0, :12] = torch.tensor([7.9, 0.25, -0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.1, -6.0])
    row[0, 32] = 2.0 ** -149
    codes, s = ref.quantize(row)
    assert s.tolist() == [[127, 0]]
    assert codes[0, :12].tolist() == [7, 0, 8, 1, 2, 2, 4, 4, 6, 6, 7, 15] and int(codes[0, 32]) == 0
    q, scales = ref.pack(codes, s)
    assert q[0, 0] == 7 and q[0, 1] == 8 | (1 << 4) and scales.tolist() == [[[127, 0, 0, 0]]]
    back, e = ref.unpack(q, scales)
    assert torch.equal(back, codes) and torch.equal(e, s.int())
    assert ref.values(codes, s)[0, :3].tolist() == [6.0, 0.0, 0.0]
