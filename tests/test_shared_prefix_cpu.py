"""lux3d_sdpa_shared_prefix refuses invalid arguments on the host, before any HIP call (the descriptors point at fake
addresses that are never dereferenced: every call here must fail validation), and its workspace size."""
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


def size(*a):
    return _lib.LIB.lux3d_sdpa_shared_prefix_workspace(*a)


GOOD = dict(q=T([4, 8, 1, 64]), prefix_k=T([2, 500, 64]), prefix_v=T([2, 500, 64]), k=T([4, 2, 70, 64]), v=T([4, 2, 70, 64]),
            lens=T([4], _lib.I32), causal=1, scale=0.125, workspace=T([1 << 22], _lib.F32), out=T([4, 8, 1, 64]), stream=None)


@pytest.mark.parametrize("change,code,text", [
    (dict(q=None), _lib.ERR_NULL, "`q`"),
    (dict(prefix_k=None), _lib.ERR_NULL, "`prefix_k`"),
    (dict(v=None), _lib.ERR_NULL, "`v`"),
    (dict(out=None), _lib.ERR_NULL, "`out`"),
    (dict(q=T([4, 8, 64])), _lib.ERR_SHAPE, "rank 4"),
    (dict(prefix_k=T([1, 2, 500, 64])), _lib.ERR_SHAPE, "rank 3"),
    (dict(q=T([4, 8, 1, 64], _lib.I32)), _lib.ERR_DTYPE, "`q`"),
    (dict(k=T([4, 2, 70, 64], _lib.F16)), _lib.ERR_DTYPE, "`k`"),
    (dict(out=T([4, 8, 1, 64], _lib.F32)), _lib.ERR_DTYPE, "`out`"),
    (dict(q=T([4, 7, 1, 64]), out=T([4, 7, 1, 64])), _lib.ERR_SHAPE, "multiple"),
    (dict(prefix_k=T([0, 500, 64]), prefix_v=T([0, 500, 64])), _lib.ERR_SHAPE, "multiple"),
    (dict(prefix_v=T([2, 499, 64])), _lib.ERR_SHAPE, "prefix_k and prefix_v"),
    (dict(prefix_k=T([2, 500, 128])), _lib.ERR_SHAPE, "prefix_k and prefix_v"),
    (dict(k=T([3, 2, 70, 64])), _lib.ERR_SHAPE, "k and v"),
    (dict(v=T([4, 2, 71, 64])), _lib.ERR_SHAPE, "k and v"),
    (dict(out=T([4, 8, 2, 64])), _lib.ERR_SHAPE, "shape of q"),
    (dict(k=T([4, 2, 70, 64], strides=[8960, 4480, 64, 2])), _lib.ERR_LAYOUT, "`k`"),
    (dict(lens=T([4], _lib.I64)), _lib.ERR_DTYPE, "`lens`"),
    (dict(lens=T([3], _lib.I32)), _lib.ERR_SHAPE, "`lens`"),
    (dict(lens=T([4], _lib.I32, strides=[2])), _lib.ERR_SHAPE, "`lens`"),
    (dict(causal=2), _lib.ERR_VALUE, "causal"),
    (dict(scale=0.0), _lib.ERR_VALUE, "scale"),
    (dict(scale=float("inf")), _lib.ERR_VALUE, "scale"),
    (dict(workspace=None), _lib.ERR_NULL, "`workspace`"),
    (dict(workspace=T([1 << 22], _lib.BF16)), _lib.ERR_LAYOUT, "`workspace`"),
    (dict(workspace=T([1 << 22], _lib.F32, data=FAKE + 4)), _lib.ERR_LAYOUT, "`workspace`"),
    (dict(workspace=T([64], _lib.F32)), _lib.ERR_SHAPE, "are needed"),
    (dict(q=T([4, 8, 1, 600]), prefix_k=T([2, 500, 600]), prefix_v=T([2, 500, 600]), k=T([4, 2, 70, 600]),
          v=T([4, 2, 70, 600]), out=T([4, 8, 1, 600])), _lib.ERR_SHAPE, "1..512"),
])
def test_refusals(change, code, text):
    rc, msg = _lib.call_status("lux3d_sdpa_shared_prefix", *{**GOOD, **change}.values())
    assert rc == code and text in msg, (rc, msg)


def test_python_refusals():
    x = torch.zeros(1, 2, 3, 64)
    with pytest.raises(_lib.Lux3dError, match="must be on a GPU"):
        ops.sdpa_shared_prefix(x, x[0], x[0], x, x, 0.1)


def test_workspace_size():
    """Whole parts of (D + 2) values a row; none where one workgroup sees all of a row's keys, or for an empty call."""
    assert size(64, 32, 8, 1, 16384, 1000, 128) % (64 * 32 * 130) == 0 < size(64, 32, 8, 1, 16384, 1000, 128)
    assert size(8, 16, 16, 2000, 10000, 2000, 64) == 0
    for bad in ((0, 8, 2, 1, 10, 10, 64), (4, 7, 2, 1, 10, 10, 64), (4, 8, 2, 1, -1, 10, 64), (4, 8, 0, 1, 10, 10, 64)):
        assert size(*bad) == 0
