"""lux3d_sdpa_shared_prefix where partial results are merged, against the formula in 64 bits: each form of the merge (many
parts a row, some, few parts of many rows) in each type and head dim, with parts that saw no key, and the prefix alone at
the sizes of several samples that attend to one image's tokens. Tolerances: those of test_gpu_shared_prefix.py, whose sums
over N keys take up to 64 further additions; a merge adds at most 64 parts."""
import pytest

torch = pytest.importorskip("torch")

import test_gpu_shared_prefix as base  # noqa: E402
from test_gpu_shared_prefix import dev, ops  # noqa: E402, F401 (fixtures)

pytestmark = pytest.mark.gpu

# batch, heads, key heads, queries, prefix, own keys; lengths of the own keys (None: all)
MANY = [(8, 16, 4, 1, 14094, 12, None), (5, 4, 2, 1, 9000, 3000, [3000, 0, 1, 300, 2999]), (1, 8, 1, 1, 7000, 3000, [0]),
        (1, 8, 1, 1, 7000, 3000, [2500])]
SOME = [(1, 4, 2, 1, 5000, 100, [7]), (3, 2, 1, 2, 100, 6000, [6000, 0, 577])]
FEW = [(2, 8, 4, 600, 700, 640, [640, 601]), (3, 8, 8, 200, 1029, 260, [260, 200, 3]), (300, 16, 8, 1, 900, 40, None),
       (40, 16, 4, 7, 700, 300, [(37 * i) % 301 for i in range(40)])]
# the prefix alone
ALONE = [(2, 12, 12, 4096, 1029, 0, None), (1, 3, 3, 2500, 1374, 0, None), (3, 16, 16, 130, 1374, 0, None)]


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("case", MANY + SOME + FEW + ALONE, ids=lambda c: "-".join(map(str, c[:6])))
def test_merged(ops, dev, case, d, dt):  # noqa: F811
    b, h, hkv, n, p, ls, lens = case
    for causal in (False, True) if ls else (False,):
        base.run(ops, dev, b, h, hkv, n, p, ls, d, dt, causal=causal, lens=lens)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("case", MANY[1:2] + SOME[1:] + FEW[:1], ids=lambda c: "-".join(map(str, c[:6])))
def test_merged_without_a_prefix(ops, dev, case, dt):  # noqa: F811
    """Rows that see no key at all are zero, whatever the workspace held; nothing is written past it."""
    from lux3d_fused import _lib
    b, h, hkv, n, p, ls, lens = case
    t, ln, out = base.run(ops, dev, b, h, hkv, n, 0, ls, 64, dt, causal=True, lens=lens)
    for i, m in enumerate(lens):
        assert not out[i, :, :max(n - m, 0)].any()
    size = _lib.LIB.lux3d_sdpa_shared_prefix_workspace(b, h, hkv, n, 0, ls, 64)
    assert size > 0
    ws = torch.full((size + 64,), float("nan"), device=dev)
    ws[size:] = 7.0
    got = torch.full_like(out, float("nan"))
    _lib.call("lux3d_sdpa_shared_prefix", *map(ops._d, t), ops._d(ln), 1, 0.125, ops._d(ws[:size]), ops._d(got), ops._stream(got))
    torch.cuda.synchronize()
    assert torch.equal(got, out) and bool((ws[size:] == 7).all())


@pytest.mark.parametrize("case", MANY[:2] + FEW[:2], ids=lambda c: "-".join(map(str, c[:6])))
def test_merged_in_a_graph(ops, dev, case):  # noqa: F811
    b, h, hkv, n, p, ls, lens = case
    t = base.make(dev, b, h, hkv, n, p, ls, 64, "bf16")
    ln = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    eager = ops.sdpa_shared_prefix(*t, 0.125, lens=ln, causal=True)
    base.check(eager, base.reference(*t, 0.125, lens, True), "eager")
    out = torch.empty_like(eager)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        ops.sdpa_shared_prefix(*t, 0.125, lens=ln, causal=True, out=out)
    for _ in range(4):
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        gr.replay()
        ops.sdpa_shared_prefix(*t, 0.125, lens=ln, causal=True)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
