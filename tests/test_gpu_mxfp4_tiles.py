"""The linears on 4-bit weights through every tile of theirs, at the smallest sizes that take it with whole and with cut
stages of k; what a call with rows past its last tile, with wide weights or with many tiles a workgroup can get wrong."""
import pytest

torch = pytest.importorskip("torch")

import mxfp4_reference as ref  # noqa: E402
from test_gpu_mxfp4 import DT, as_products_see, call, dev, ops, rnd, run_gated, run_linear, same_as_defined, tokens, weight  # noqa: E402,F401

pytestmark = pytest.mark.gpu

# how x enters, gated, tile rows, columns, groups that share k, few rows past the last tile apart, m, k, n: the choice of
# csrc/mxfp4_tiles.hpp, which test_mxfp4_tiles_cpu.py holds to this list
TILES = [
    ("fp4", False, 64, 64, 1, False, 456, 32, 562),
    ("fp4", False, 64, 64, 1, False, 455, 128, 561),
    ("fp4", False, 64, 64, 2, False, 455, 2784, 433),
    ("fp4", False, 64, 64, 2, False, 452, 2816, 435),
    ("fp4", False, 64, 128, 1, False, 1345, 32, 965),
    ("fp4", False, 64, 128, 1, False, 1217, 128, 1089),
    ("fp4", False, 128, 128, 1, False, 2305, 288, 1567),
    ("fp4", False, 128, 128, 1, False, 1987, 384, 1847),
    ("fp4", False, 128, 128, 1, True, 2569, 960, 3125),
    ("fp4", False, 128, 128, 1, True, 4102, 896, 2025),
    ("fp4", False, 256, 256, 1, False, 2492, 544, 4154),
    ("fp4", False, 256, 256, 1, False, 3400, 512, 2949),
    ("fp4", False, 256, 256, 1, True, 4612, 608, 3420),
    ("fp4", False, 256, 256, 1, True, 3329, 512, 4663),
    ("fp4", True, 64, 128, 1, False, 549, 32, 567),
    ("fp4", True, 64, 128, 1, False, 645, 128, 481),
    ("fp4", True, 128, 128, 1, False, 1239, 288, 1473),
    ("fp4", True, 128, 128, 1, False, 1418, 384, 1282),
    ("fp4", True, 128, 128, 1, True, 3587, 2976, 560),
    ("fp4", True, 128, 128, 1, True, 2945, 1792, 2776),
    ("fp4", True, 256, 256, 1, False, 1966, 544, 2633),
    ("fp4", True, 256, 256, 1, False, 1734, 512, 2891),
    ("fp4", True, 256, 256, 1, True, 1293, 576, 5695),
    ("fp4", True, 256, 256, 1, True, 2064, 512, 3731),
    ("2byte", False, 64, 64, 1, False, 514, 32, 468),
    ("2byte", False, 64, 64, 1, False, 513, 128, 577),
    ("2byte", False, 64, 64, 2, False, 614, 480, 533),
    ("2byte", False, 64, 64, 2, False, 577, 512, 561),
    ("2byte", False, 64, 64, 4, False, 376, 3552, 472),
    ("2byte", False, 64, 64, 4, False, 322, 3584, 482),
    ("2byte", False, 64, 128, 1, False, 1615, 32, 1217),
    ("2byte", False, 64, 128, 1, False, 1166, 128, 1665),
    ("2byte", False, 64, 128, 1, True, 2510, 992, 1558),
    ("2byte", False, 64, 128, 1, True, 1601, 896, 2512),
    ("2byte", False, 64, 128, 2, False, 779, 992, 1267),
    ("2byte", False, 64, 128, 2, False, 1092, 1024, 925),
    ("2byte", False, 64, 128, 2, True, 1159, 1632, 1709),
    ("2byte", False, 64, 128, 2, True, 1474, 1024, 1359),
    ("2byte", False, 64, 128, 4, False, 864, 3744, 1185),
    ("2byte", False, 64, 128, 4, False, 907, 3840, 1127),
    ("2byte", False, 64, 128, 4, True, 1098, 4000, 1899),
    ("2byte", False, 64, 128, 4, True, 1164, 4096, 1685),
    ("2byte", False, 128, 128, 1, False, 2191, 160, 1683),
    ("2byte", False, 128, 128, 1, False, 1799, 256, 1923),
    ("2byte", False, 128, 128, 1, True, 2955, 576, 1361),
    ("2byte", False, 128, 128, 1, True, 1668, 640, 2347),
    ("2byte", False, 128, 256, 1, False, 5833, 32, 3853),
    ("2byte", False, 128, 256, 1, False, 3083, 128, 4886),
    ("2byte", False, 128, 256, 1, True, 4225, 160, 5809),
    ("2byte", False, 128, 256, 1, True, 6150, 128, 4085),
    ("2byte", False, 256, 256, 1, False, 3845, 32, 3471),
    ("2byte", False, 256, 256, 1, False, 3588, 128, 3371),
    ("2byte", False, 256, 256, 1, True, 5391, 160, 2819),
    ("2byte", False, 256, 256, 1, True, 4109, 128, 3972),
    ("2byte", True, 64, 128, 1, False, 551, 32, 437),
    ("2byte", True, 64, 128, 1, False, 577, 128, 515),
    ("2byte", True, 64, 128, 1, True, 4677, 992, 391),
    ("2byte", True, 64, 128, 1, True, 1483, 1024, 1379),
    ("2byte", True, 64, 128, 2, False, 569, 1120, 405),
    ("2byte", True, 64, 128, 2, False, 365, 1152, 596),
    ("2byte", True, 64, 128, 2, True, 1031, 1824, 967),
    ("2byte", True, 64, 128, 2, True, 972, 1792, 1042),
    ("2byte", True, 64, 128, 4, False, 458, 3808, 389),
    ("2byte", True, 64, 128, 4, False, 455, 3840, 413),
    ("2byte", True, 64, 128, 4, True, 582, 3744, 1684),
    ("2byte", True, 64, 128, 4, True, 1097, 3840, 921),
    ("2byte", True, 128, 128, 1, False, 1634, 160, 1154),
    ("2byte", True, 128, 128, 1, False, 1415, 256, 1222),
    ("2byte", True, 128, 128, 1, True, 901, 672, 2199),
    ("2byte", True, 128, 128, 1, True, 2305, 640, 843),
    ("2byte", True, 128, 256, 1, False, 4172, 32, 2691),
    ("2byte", True, 128, 256, 1, False, 2319, 128, 3207),
    ("2byte", True, 128, 256, 1, True, 4492, 32, 5398),
    ("2byte", True, 128, 256, 1, True, 3843, 128, 4301),
    ("2byte", True, 256, 256, 1, False, 2692, 32, 2500),
    ("2byte", True, 256, 256, 1, False, 2754, 128, 2191),
    ("2byte", True, 256, 256, 1, True, 2051, 96, 4001),
    ("2byte", True, 256, 256, 1, True, 3592, 128, 2265),
    ("f32", False, 64, 64, 4, False, 582, 96, 716),
    ("f32", False, 64, 64, 4, False, 706, 128, 578),
    ("f32", False, 64, 128, 2, False, 515, 32, 745),
    ("f32", False, 64, 128, 2, False, 771, 128, 1217),
    ("f32", False, 64, 128, 2, True, 1476, 224, 1303),
    ("f32", False, 64, 128, 2, True, 1601, 256, 1210),
    ("f32", False, 64, 128, 4, False, 844, 1120, 1177),
    ("f32", False, 64, 128, 4, False, 1102, 1152, 904),
    ("f32", False, 64, 128, 4, True, 1154, 1120, 1787),
    ("f32", False, 64, 128, 4, True, 1795, 1152, 1032),
    ("f32", True, 64, 128, 2, False, 483, 32, 561),
    ("f32", True, 64, 128, 2, False, 584, 128, 595),
    ("f32", True, 64, 128, 2, True, 972, 416, 1033),
    ("f32", True, 64, 128, 2, True, 577, 384, 1745),
    ("f32", True, 64, 128, 4, False, 478, 1120, 731),
    ("f32", True, 64, 128, 4, False, 591, 1152, 548),
    ("f32", True, 64, 128, 4, True, 1607, 1120, 581),
    ("f32", True, 64, 128, 4, True, 769, 1152, 1229),
]
# workgroups that stay for a second and third tile: more 256 x 256 tiles than CUs
STAY = [(False, 8656, 512, 2308), (False, 8657, 1056, 2309), (False, 4111, 640, 8237), (True, 5121, 544, 2001), (True, 5121, 512, 2000)]
# weight tiles a workgroup of few rows: tiles, 2-byte x as it is, gated, n, k
WIDE = [(1, True, False, 8191, 512), (2, True, False, 8199, 544), (2, False, False, 8192, 512), (2, True, False, 16401, 1024),
        (4, False, False, 16390, 1056), (4, True, False, 24583, 1024), (1, False, True, 16383, 1024), (2, False, True, 16391, 1024),
        (2, True, True, 16391, 1120), (1, True, True, 16391, 992), (2, True, False, 24583, 992)]
ACTS = {"64": "silu", "128": "gelu_erf", "256": "gelu_tanh"}


@pytest.mark.parametrize("kind,gated,rows,cols,groups,split,m,k,n", TILES)
def test_tile(ops, dev, kind, gated, rows, cols, groups, split, m, k, n):
    arith = "fp4" if kind == "fp4" else "plain"
    for dt in {"fp4": ["bf16"], "2byte": ["bf16", "f16"], "f32": ["f32"]}[kind]:
        for out, bias in (("same", True), ("f32" if dt != "f32" else "f16", False)):
            if gated:
                run_gated(ops, dev, m, k, n, dt, arith, ACTS[str(rows)], out, use_bias=bias)
            else:
                run_linear(ops, dev, m, k, n, dt, arith, out, use_bias=bias)


@pytest.mark.parametrize("gated,m,k,n", STAY)
def test_workgroups_that_stay(ops, dev, gated, m, k, n):
    for out, bias in (("same", True), ("f32", False)):
        if gated:
            run_gated(ops, dev, m, k, n, "bf16", "fp4", "gelu_tanh", out, use_bias=bias)
        else:
            run_linear(ops, dev, m, k, n, "bf16", "fp4", out, use_bias=bias)


@pytest.mark.parametrize("m", [1, 5, 16])
@pytest.mark.parametrize("tiles,plain_2byte,gated,n,k", WIDE)
def test_wide_weights(ops, dev, m, tiles, plain_2byte, gated, n, k):
    for dt, arith in (("bf16", "plain"), ("f16", "plain")) if plain_2byte else (("f32", "plain"), ("bf16", "fp4"), ("f32", "fp4")):
        if gated:
            run_gated(ops, dev, m, k, n, dt, arith, "silu")
        else:
            run_linear(ops, dev, m, k, n, dt, arith)


@pytest.mark.parametrize("m", [16, 13])
def test_packed_few_rows_of_wide_weights(ops, dev, m):
    """A packed x gives the bits of the x that it was quantized from."""
    x, w = tokens(dev, m, 1056, "bf16"), weight(dev, 16391, 1056)
    assert torch.equal(ops.mxfp4_linear_fp4(ops.mxfp4_quantize(x), *w), ops.mxfp4_linear_fp4(x, *w))


@pytest.mark.parametrize("dt,m,k,n", [("bf16", 4677, 992, 391), ("f32", 1476, 224, 1303), ("bf16", 4097, 1024, 464)])
def test_rows_past_the_last_tile_in_views(ops, dev, dt, m, k, n):
    """A slice of wider rows in, a slice of a wider tensor out: what lies beside and behind stays."""
    from lux3d_fused import _lib
    wide = tokens(dev, m, k + 64, dt)
    x, w, bias = wide[:, 32:32 + k], weight(dev, n, k), rnd(dev, n)
    want = ops.mxfp4_linear(x.contiguous(), *w, bias=bias)
    for left, width in ((8, n + 24), (3, n + 7)):
        big = torch.full((m + 2, width), 5.0, dtype=DT[dt], device=dev)
        y = big[1:m + 1, left:left + n]
        _lib.call("lux3d_mxfp4_linear", ops._d(x), ops._d(w[0]), ops._d(w[1]), ops._d(bias), ops._d(y), ops._stream(x))
        assert torch.equal(y, want)
        big[1:m + 1, left:left + n] = 5.0
        assert bool((big == 5.0).all())


@pytest.mark.parametrize("gated,m,k,n", [(False, 2569, 960, 3125), (False, 4612, 608, 3420), (True, 2064, 512, 3731)])
def test_packed_rows_past_the_last_tile(ops, dev, gated, m, k, n):
    x, w, v = tokens(dev, m, k, "bf16"), weight(dev, n, k), weight(dev, n, k, 1)
    pair = ops.mxfp4_quantize(x)
    if gated:
        assert torch.equal(ops.mxfp4_linear_gated(pair, v, w, fp4=True), ops.mxfp4_linear_gated(x, v, w, fp4=True))
    else:
        assert torch.equal(ops.mxfp4_linear_fp4(pair, *w), ops.mxfp4_linear_fp4(x, *w))


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,k", [(8200, 64), (3001, 1632), (8191, 512), (20000, 32)])
def test_quantize_many_rows(ops, dev, m, k, dt):
    x = tokens(dev, m, k, dt)
    q, s = ops.mxfp4_quantize(x)
    same_as_defined(q, s, x, f"{m} x {k} {dt}")
    for out in DT.values():
        assert torch.equal(ops.mxfp4_dequantize(q, s, out), ref.dense(q, s).to(torch.float32).to(out))


def test_two_calls_at_once(ops, dev):
    """Calls on two streams that run beside each other, each with its own x and workspaces, share the weight."""
    m, k, n = 8657, 512, 2309
    w, v = weight(dev, n, k), weight(dev, n, k, 1)
    xs = [tokens(dev, m, k, "bf16", seed=s) for s in (1, 2)]
    fns = [lambda x: ops.mxfp4_linear_fp4(x, *w), lambda x: ops.mxfp4_linear_gated(x, v, w, "gelu_erf", fp4=True),
           lambda x: ops.mxfp4_linear(x, *w), lambda x: ops.mxfp4_linear(x[:7], *w)]
    want = [[f(x) for f in fns] for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(3):
        got = [[], []]
        for f in fns:
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    got[i].append(f(xs[i]))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for i in range(2) for a, b in zip(got[i], want[i]))


def test_workgroups_that_stay_in_a_graph(ops, dev):
    m, k, n = 8657, 544, 2309
    x, w = tokens(dev, m, k, "bf16"), weight(dev, n, k)
    other = tokens(dev, m, k, "bf16", seed=3)
    want, want_other = ops.mxfp4_linear_fp4(x, *w), ops.mxfp4_linear_fp4(other, *w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.mxfp4_linear_fp4(x, *w)
    for source, expect in ((None, want), (other, want_other), (None, want_other)):
        if source is not None:
            x.copy_(source)
        y.zero_()
        g.replay()
        ops.mxfp4_linear_fp4(other, *w)
        torch.cuda.synchronize()
        assert torch.equal(y, expect)
