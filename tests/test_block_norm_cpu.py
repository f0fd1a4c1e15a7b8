"""lux3d_norm_gated_residual_norm refuses invalid arguments on the host, before any HIP call. The descriptors point at
fake addresses that are never dereferenced: every call here must fail validation."""
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


OUT, Y = T([8, 64], data=2 * FAKE), T([8, 64], data=3 * FAKE)
GOOD = dict(x=T([8, 64]), h=T([8, 64], data=4 * FAKE), post_w=None, post_b=None, ls_gamma=None, seg_offsets=None, gate=None,
            gate_base=None, pre_w=None, pre_b=None, shift=None, shift_base=None, scale=None, scale_base=None, rms=0,
            eps=1e-6, x_out=OUT, y=Y, stream=None)


@pytest.mark.parametrize("change,code,text", [
    (dict(x=None), _lib.ERR_NULL, "`x`"),
    (dict(h=None), _lib.ERR_NULL, "`h`"),
    (dict(x_out=None), _lib.ERR_NULL, "`x_out`"),
    (dict(h=T([8, 32])), _lib.ERR_SHAPE, "`h`"),
    (dict(h=T([8, 64], _lib.F32)), _lib.ERR_DTYPE, "`h`"),
    (dict(x=T([8, 64], _lib.I32)), _lib.ERR_DTYPE, "`x`"),
    (dict(x=T([8, 64], strides=[64, 2])), _lib.ERR_LAYOUT, "unit innermost"),
    (dict(x=T([2, 4, 64], strides=[999, 64, 1])), _lib.ERR_LAYOUT, "uniform row stride"),
    (dict(y=T([8, 64])), _lib.ERR_LAYOUT, "alias"),
    (dict(y=OUT), _lib.ERR_LAYOUT, "alias"),
    (dict(y=T([9, 64], data=3 * FAKE)), _lib.ERR_SHAPE, "`y`"),
    (dict(y=None, pre_w=T([64], _lib.F32)), _lib.ERR_NULL, "`y` is NULL"),
    (dict(y=None, shift=T([1, 64], _lib.F32)), _lib.ERR_NULL, "`y` is NULL"),
    (dict(post_w=T([63], _lib.F32)), _lib.ERR_SHAPE, "post_w"),
    (dict(post_b=T([64], _lib.I32)), _lib.ERR_DTYPE, "post_b"),
    (dict(ls_gamma=T([64], _lib.F32, strides=[2])), _lib.ERR_LAYOUT, "ls_gamma"),
    (dict(gate=T([3, 64], _lib.F32)), _lib.ERR_SHAPE, "equal segments"),
    (dict(gate=T([2, 64], _lib.F32), scale=T([4, 64], _lib.F32)), _lib.ERR_SHAPE, "segment counts"),
    (dict(gate=T([0, 64], _lib.F32)), _lib.ERR_SHAPE, "no segment"),
    (dict(gate_base=T([64], _lib.F32)), _lib.ERR_NULL, "gate_base"),
    (dict(gate=T([2, 64], _lib.F32), seg_offsets=T([3], _lib.I32)), _lib.ERR_DTYPE, "seg_offsets"),
    (dict(gate=T([2, 64], _lib.F32), seg_offsets=T([4], _lib.I64)), _lib.ERR_SHAPE, "segments"),
    (dict(rms=2), _lib.ERR_VALUE, "rms"),
    (dict(eps=-1.0), _lib.ERR_VALUE, "eps"),
    (dict(eps=float("nan")), _lib.ERR_VALUE, "eps"),
    (dict(x=T([8, 0]), h=T([8, 0]), x_out=T([8, 0]), y=T([8, 0])), _lib.ERR_SHAPE, "empty rows"),
])
def test_refusals(change, code, text):
    args = {**GOOD, **change}
    rc, msg = _lib.call_status("lux3d_norm_gated_residual_norm", *args.values())
    assert rc == code and text in msg, (rc, msg)


def test_python_refuses_host_tensors_and_unknown_norms():
    x = torch.zeros(4, 64)
    with pytest.raises(_lib.Lux3dError, match="must be on a GPU"):
        ops.norm_gated_residual_norm(x, x)
    with pytest.raises(_lib.Lux3dError, match="'layer' or 'rms'"):
        ops.norm_gated_residual_norm(x, x, norm="batch")
