"""How much workspace lux3d_sdpa_shared_prefix asks for: what the plan of the call's own type needs, none for head dims that
leave no partial results, and enough for each type without one."""
import random

import pytest

pytest.importorskip("torch")

from lux3d_fused import _lib  # noqa: E402

FLOATS = (_lib.F32, _lib.BF16, _lib.F16)


def size(dtype, *a):
    return _lib.LIB.lux3d_sdpa_shared_prefix_workspace_dtype(dtype, *a)


def any_type(*a):
    return _lib.LIB.lux3d_sdpa_shared_prefix_workspace(*a)


def test_two_byte_types_do_not_pay_for_f32():
    for a in ((3, 32, 8, 1171, 2540, 1295, 128),):
        assert size(_lib.BF16, *a) == size(_lib.F16, *a) == 0 < size(_lib.F32, *a) == any_type(*a), a
    a = (5, 32, 8, 221, 6645, 366, 128)
    assert 0 < 2 * size(_lib.BF16, *a) < any_type(*a)


@pytest.mark.parametrize("d", [1, 32, 63, 65, 80, 96, 127, 129, 256, 512])
def test_no_workspace_where_no_part_is_left(d):
    a = (64, 32, 8, 1, 16384, 1000, d)
    assert [size(t, *a) for t in FLOATS] == [0, 0, 0] and any_type(*a) == 0


def test_a_size_for_every_type_suffices():
    r = random.Random(3)
    for _ in range(2000):
        g, hkv = r.choice([1, 2, 4, 8]), r.choice([1, 2, 4, 8, 16])
        a = (r.randint(1, 128), g * hkv, hkv, int(2 ** r.uniform(0, 12)), r.choice([0, int(2 ** r.uniform(0, 17))]),
             r.choice([0, int(2 ** r.uniform(0, 13))]), r.choice([64, 128]))
        each = [size(t, *a) for t in FLOATS]
        assert each[1] == each[2] and any_type(*a) == max(each), a


def test_nothing_for_calls_that_are_none():
    for bad in ((0, 8, 2, 1, 10, 10, 64), (4, 7, 2, 1, 10, 10, 64), (4, 8, 2, 1, -1, 10, 64), (4, 8, 0, 1, 10, 10, 64)):
        assert size(_lib.BF16, *bad) == 0
    assert size(_lib.I32, 64, 32, 8, 1, 16384, 1000, 128) == size(-1, 64, 32, 8, 1, 16384, 1000, 128) == 0
