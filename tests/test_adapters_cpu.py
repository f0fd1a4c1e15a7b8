"""lux3d_q8_0_linear_adapters refuses invalid arguments on the host, before any HIP call (the descriptors point at fake
addresses that are never dereferenced: every call here must fail validation)."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from lux3d_fused import _lib, ops  # noqa: E402

FAKE = 0x100000


def T(shape, dtype=_lib.BF16, strides=None, data=FAKE):
    if strides is None:
        strides, acc = [], 1
        for n in reversed(shape):
            strides.insert(0, acc)
            acc *= n
    return ctypes.pointer(_lib.descriptor(data, dtype, shape, strides))


GOOD = dict(x=T([10, 64]), qs=T([40, 64], _lib.I8), scales=T([40, 2], _lib.F32), bias=None, a=T([3, 8, 64]), b=T([3, 40, 8]),
            alphas=None, adapter_ids=T([2], _lib.I32), seg_offsets=None, t=T([10, 16]), bad_ids=None, y=T([10, 40]),
            stream=None)


@pytest.mark.parametrize("change,code,text", [
    (dict(x=None), _lib.ERR_NULL, "`x`"),
    (dict(a=None), _lib.ERR_NULL, "`a`"),
    (dict(b=None), _lib.ERR_NULL, "`b`"),
    (dict(t=None), _lib.ERR_NULL, "`t`"),
    (dict(adapter_ids=None), _lib.ERR_NULL, "`adapter_ids`"),
    (dict(x=T([10, 64], _lib.F16)), _lib.ERR_DTYPE, "bf16 or f32"),
    (dict(qs=T([40, 32], _lib.I8)), _lib.ERR_SHAPE, "features"),
    (dict(scales=T([40, 3], _lib.F32)), _lib.ERR_SHAPE, "scales"),
    (dict(y=T([10, 41])), _lib.ERR_SHAPE, "y must be"),
    (dict(a=T([3, 8, 64], _lib.F32)), _lib.ERR_DTYPE, "x's dtype"),
    (dict(b=T([3, 40, 8], _lib.F16)), _lib.ERR_DTYPE, "x's dtype"),
    (dict(t=T([10, 16], _lib.F32)), _lib.ERR_DTYPE, "x's dtype"),
    (dict(a=T([3, 8, 32])), _lib.ERR_SHAPE, "`a`"),
    (dict(a=T([8, 64])), _lib.ERR_SHAPE, "`a`"),
    (dict(a=T([0, 8, 64]), b=T([0, 40, 8])), _lib.ERR_SHAPE, "`a`"),
    (dict(a=T([3, 0, 64]), b=T([3, 40, 0])), _lib.ERR_SHAPE, "`a`"),
    (dict(a=T([1, 1025, 64]), b=T([1, 40, 1025])), _lib.ERR_SHAPE, "rank 1025"),
    (dict(b=T([3, 40, 9])), _lib.ERR_SHAPE, "`b`"),
    (dict(b=T([3, 40, 8], strides=[640, 16, 1])), _lib.ERR_LAYOUT, "contiguous"),
    (dict(a=T([3, 8, 64], data=FAKE + 2)), _lib.ERR_LAYOUT, "aligned"),
    (dict(t=T([10, 16], data=FAKE + 2)), _lib.ERR_LAYOUT, "aligned"),
    (dict(t=T([10, 8])), _lib.ERR_SHAPE, "`t`"),
    (dict(adapter_ids=T([2], _lib.I64)), _lib.ERR_DTYPE, "adapter_ids"),
    (dict(adapter_ids=T([0], _lib.I32)), _lib.ERR_SHAPE, "adapter_ids"),
    (dict(adapter_ids=T([3], _lib.I32)), _lib.ERR_SHAPE, "equal segments"),
    (dict(seg_offsets=T([2], _lib.I64)), _lib.ERR_SHAPE, "seg_offsets"),
    (dict(seg_offsets=T([3], _lib.I32)), _lib.ERR_DTYPE, "seg_offsets"),
    (dict(alphas=T([2], _lib.F32)), _lib.ERR_SHAPE, "alphas"),
    (dict(alphas=T([3])), _lib.ERR_DTYPE, "alphas"),
    (dict(bad_ids=T([2], _lib.I32)), _lib.ERR_SHAPE, "bad_ids"),
])
def test_refusals(change, code, text):
    rc, msg = _lib.call_status("lux3d_q8_0_linear_adapters", *{**GOOD, **change}.values())
    assert rc == code and text in msg, (rc, msg)


def test_python_refusals():
    x = torch.zeros(4, 64)
    with pytest.raises(_lib.Lux3dError, match="must be on a GPU"):
        ops.q8_0_linear_adapters(x, x, x, x, x, x)
