"""The few-rows Q8_0 linear keeps its bits: against tests/golden/q8_few_rows.npz, outputs of the kernel that loaded its
operands as the matrix instructions hold them at every size (inputs from CPU generators), and from one form to the other,
with row tiles past a grid's y, against 64 bits."""
import os

import pytest

np = pytest.importorskip("numpy")
torch = pytest.importorskip("torch")

from test_gpu_q8_few_rows import TDT, _weights  # noqa: E402

pytestmark = pytest.mark.gpu
GOLDEN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden", "q8_few_rows.npz")

# rows, k, columns: one row tile with 4, 8 and 16 wavefronts, below and from k 512 on; more rows with each of the three
SIZES = [(1, 64, 40), (16, 448, 33), (7, 512, 48), (16, 960, 35), (5, 1536, 48), (16, 4160, 16), (1, 640, 8200),
         (64, 448, 16), (40, 512, 33), (33, 1024, 48), (130, 2112, 31), (61, 8192, 16)]


def linear(m, k, n, xdt, dev):
    from lux3d_fused import ops
    qs, scales = _weights(n, k, m + 3 * k + 7 * n, dev)
    x = torch.randn((m, k), generator=torch.Generator(device="cpu").manual_seed(m + k)).to(dev).to(TDT[xdt])
    bias = torch.randn(n, generator=torch.Generator(device="cpu").manual_seed(n)).to(dev)
    return ops.q8_0_linear(x, qs, scales, bias, torch.float32)


@pytest.mark.parametrize("xdt", ["bf16", "f32"])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_bits_are_kept(m, k, n, xdt):
    y = linear(m, k, n, xdt, torch.device("cuda:0")).cpu().numpy()
    with np.load(GOLDEN) as z:
        want = z[f"{m}x{k}x{n}_{xdt}"]
    assert np.array_equal(y.view(np.uint32), want)


@pytest.mark.parametrize("xdt", ["bf16", "f32"])
@pytest.mark.parametrize("k", [64, 192, 448])
def test_one_tile_and_more_rows_agree(k, xdt):
    """Below k 512 up to 16 rows load their operands directly and more go through LDS: the same sums in the same order."""
    from lux3d_fused import ops
    dev = torch.device("cuda:0")
    qs, scales = _weights(48, k, k, dev)
    x = torch.randn((61, k), generator=torch.Generator(device="cpu").manual_seed(k)).to(dev).to(TDT[xdt])
    whole = ops.q8_0_linear(x, qs, scales, None, torch.float32)
    for m0, m1 in ((0, 16), (16, 29), (45, 61), (60, 61)):
        assert torch.equal(ops.q8_0_linear(x[m0:m1], qs, scales, None, torch.float32), whole[m0:m1])


# more than 65535 row tiles of 32, f32 (the dispatch takes other kernels for so many bf16 rows)
FAR = (65535 * 32 + 33, 512, 9)


def test_row_tiles_past_the_grids_y():
    from lux3d_fused import ops
    dev = torch.device("cuda:0")
    m, k, n = FAR
    print(f"[case] q8 few rows {m} x {k} -> {n}", flush=True)
    qs, scales = _weights(n, k, 5, dev)
    x = torch.randn((m, k), generator=torch.Generator(device=dev).manual_seed(1), device=dev)
    y = ops.q8_0_linear(x, qs, scales, None, torch.float32)
    w = (qs.double().reshape(n, -1, 32) * scales.double()[:, :, None]).reshape(n, k).t().contiguous()
    for a in range(0, m, 1 << 19):
        xd = x[a:a + (1 << 19)].double()
        want, mag = xd @ w, xd.abs() @ w.abs()
        # an f32 sum's last place per MFMA, block and wavefront, and the store
        bound = (k / 32 + 40) * 2.0 ** -23 * mag + 2.0 ** -24 * want.abs()
        assert bool(((y[a:a + (1 << 19)].double() - want).abs() <= bound).all()), a
