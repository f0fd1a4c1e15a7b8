"""The sizes of the GPU tests on the few-rows linear's bits take that kernel, with each count of wavefronts."""
import pytest

pytest.importorskip("torch")

import test_gpu_q8_few_rows_bits as bits  # noqa: E402
from test_q8_tiles_cpu import choice  # noqa: E402, F401 (fixture)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sizes_take_the_few_rows_kernel(choice, dtype):  # noqa: F811
    kinds = set()
    for m, k, n in bits.SIZES:
        tile = choice(dtype, m, n, k)
        assert tile[1] == 16 and tile[0] == (16 if m <= 16 else 64), (m, k, n, tile)
        groups = -(-n // 16) * -(-m // tile[0])
        kinds.add((tile[0], 4 if groups * 4 >= 2048 or k <= 512 else 8 if groups * 8 >= 2048 or k <= 1024 else 16))
    assert kinds == {(r, w) for r in (16, 64) for w in (4, 8, 16)}
    assert choice(dtype, 61, 48, 64)[0] == choice(dtype, 61, 48, 448)[0] == 64
    m, k, n = bits.FAR
    assert choice("f32", m, n, k) == (64, 16, 1) and m > 65535 * 32
