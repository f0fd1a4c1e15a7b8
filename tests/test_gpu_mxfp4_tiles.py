"""The linears on 4-bit weights through every tile of theirs, at the smallest sizes that take it with whole and with cut
stages of k; what a call with rows past its last tile, with wide weights or with many tiles a workgroup can get wrong."""
import pytest

torch = pytest.importorskip("torch")

import mxfp4_reference as ref  # noqa: E402
from test_gpu_mxfp4 import DT, dev, ops, rnd, run_gated, run_linear, same_as_defined, tokens, weight  # noqa: E402,F401

pytestmark = pytest.mark.gpu

# how x enters, gated, tile rows, columns, groups that share k, few rows past the last tile apart, m, k, n: the choice of
# csrc/mxfp4_tiles.hpp, which test_mxfp4_tiles_cpu.py holds to this list
TILES = [
    ("fp4", False, 64, 64, 1, False, 517, 32, 501),
    ("fp4", False, 64, 64, 1, False, 449, 128, 562),
    ("fp4", False, 64, 64, 1, True, 1418, 736, 1409),
    ("fp4", False, 64, 64, 1, True, 833, 640, 2449),
    ("fp4", False, 64, 64, 2, False, 522, 2720, 399),
    ("fp4", False, 64, 64, 2, False, 396, 2816, 506),
    ("fp4", False, 64, 64, 2, True, 16388, 3616, 31),
    ("fp4", False, 64, 64, 2, True, 8195, 5120, 79),
    ("fp4", False, 64, 128, 1, False, 973, 32, 1347),
    ("fp4", False, 64, 128, 1, False, 1345, 128, 964),
    ("fp4", False, 64, 128, 1, True, 514, 32, 7596),
    ("fp4", False, 64, 128, 1, True, 577, 128, 6907),
    ("fp4", False, 128, 128, 1, False, 2323, 288, 1537),
    ("fp4", False, 128, 128, 1, False, 2004, 384, 1827),
    ("fp4", False, 128, 128, 1, True, 1936, 288, 2120),
    ("fp4", False, 128, 128, 1, True, 1665, 384, 2381),
    ("fp4", False, 256, 256, 1, False, 2891, 544, 3495),
    ("fp4", False, 256, 256, 1, False, 2891, 512, 3458),
    ("fp4", False, 256, 256, 1, True, 5902, 576, 2724),
    ("fp4", False, 256, 256, 1, True, 3085, 512, 4922),
    ("fp4", True, 64, 128, 1, False, 563, 32, 565),
    ("fp4", True, 64, 128, 1, False, 547, 128, 575),
    ("fp4", True, 64, 128, 1, True, 835, 288, 1167),
    ("fp4", True, 64, 128, 1, True, 1224, 384, 784),
    ("fp4", True, 128, 128, 1, False, 1228, 288, 1491),
    ("fp4", True, 128, 128, 1, False, 1414, 384, 1289),
    ("fp4", True, 128, 128, 1, True, 1800, 288, 1115),
    ("fp4", True, 128, 128, 1, True, 1161, 384, 1675),
    ("fp4", True, 256, 256, 1, False, 1922, 544, 2650),
    ("fp4", True, 256, 256, 1, False, 2055, 512, 2439),
    ("fp4", True, 256, 256, 1, True, 1545, 544, 4978),
    ("fp4", True, 256, 256, 1, True, 2562, 512, 2948),
    ("2byte", False, 64, 64, 1, False, 457, 32, 531),
    ("2byte", False, 64, 64, 1, False, 450, 128, 644),
    ("2byte", False, 64, 64, 1, True, 1415, 224, 1467),
    ("2byte", False, 64, 64, 1, True, 1671, 256, 1159),
    ("2byte", False, 64, 64, 2, False, 518, 480, 663),
    ("2byte", False, 64, 64, 2, False, 609, 512, 545),
    ("2byte", False, 64, 64, 2, True, 16390, 3264, 17),
    ("2byte", False, 64, 64, 2, True, 16385, 2560, 22),
    ("2byte", False, 64, 64, 4, False, 392, 3520, 439),
    ("2byte", False, 64, 64, 4, False, 452, 3584, 367),
    ("2byte", False, 64, 64, 4, True, 16400, 3840, 33),
    ("2byte", False, 64, 128, 1, False, 1672, 32, 1155),
    ("2byte", False, 64, 128, 1, False, 1154, 128, 1675),
    ("2byte", False, 64, 128, 1, True, 1537, 96, 2607),
    ("2byte", False, 64, 128, 1, True, 1543, 128, 2563),
    ("2byte", False, 64, 128, 2, False, 908, 992, 1145),
    ("2byte", False, 64, 128, 2, False, 1175, 1024, 839),
    ("2byte", False, 64, 128, 4, False, 1155, 3776, 845),
    ("2byte", False, 64, 128, 4, False, 1221, 3840, 794),
    ("2byte", False, 64, 128, 4, True, 1219, 5312, 1659),
    ("2byte", False, 64, 128, 4, True, 1604, 4992, 1186),
    ("2byte", False, 128, 128, 1, False, 2575, 160, 1411),
    ("2byte", False, 128, 128, 1, False, 2250, 256, 1540),
    ("2byte", False, 128, 128, 1, True, 1537, 160, 2563),
    ("2byte", False, 128, 128, 1, True, 2057, 256, 1965),
    ("2byte", False, 128, 256, 1, False, 4884, 32, 4611),
    ("2byte", False, 128, 256, 1, False, 4889, 128, 3111),
    ("2byte", False, 128, 256, 1, True, 5126, 32, 4757),
    ("2byte", False, 128, 256, 1, True, 2954, 128, 5528),
    ("2byte", False, 256, 256, 1, False, 3595, 32, 3730),
    ("2byte", False, 256, 256, 1, False, 3337, 128, 3587),
    ("2byte", False, 256, 256, 1, True, 3076, 96, 5258),
    ("2byte", False, 256, 256, 1, True, 3592, 128, 4526),
    ("2byte", True, 64, 128, 1, False, 513, 32, 465),
    ("2byte", True, 64, 128, 1, False, 483, 128, 611),
    ("2byte", True, 64, 128, 1, True, 321, 96, 5662),
    ("2byte", True, 64, 128, 1, True, 321, 128, 5584),
    ("2byte", True, 64, 128, 2, False, 527, 1120, 437),
    ("2byte", True, 64, 128, 2, False, 484, 1152, 456),
    ("2byte", True, 64, 128, 4, False, 528, 3744, 356),
    ("2byte", True, 64, 128, 4, False, 452, 3840, 391),
    ("2byte", True, 128, 128, 1, False, 1927, 160, 965),
    ("2byte", True, 128, 128, 1, False, 1417, 256, 1221),
    ("2byte", True, 128, 128, 1, True, 1156, 160, 1748),
    ("2byte", True, 128, 128, 1, True, 1155, 256, 1683),
    ("2byte", True, 128, 256, 1, False, 2959, 32, 3815),
    ("2byte", True, 128, 256, 1, False, 2338, 128, 3210),
    ("2byte", True, 128, 256, 1, True, 4236, 32, 2905),
    ("2byte", True, 128, 256, 1, True, 2694, 128, 3036),
    ("2byte", True, 256, 256, 1, False, 2453, 32, 2769),
    ("2byte", True, 256, 256, 1, False, 2758, 128, 2193),
    ("2byte", True, 256, 256, 1, True, 1032, 96, 7700),
    ("2byte", True, 256, 256, 1, True, 2576, 128, 3163),
    ("f32", False, 64, 64, 4, False, 713, 96, 585),
    ("f32", False, 64, 64, 4, False, 549, 128, 739),
    ("f32", False, 64, 64, 4, True, 16386, 992, 20),
    ("f32", False, 64, 64, 4, True, 16400, 1024, 54),
    ("f32", False, 64, 128, 2, False, 581, 32, 659),
    ("f32", False, 64, 128, 2, False, 1219, 128, 773),
    ("f32", False, 64, 128, 2, True, 1802, 32, 1033),
    ("f32", False, 64, 128, 2, True, 1611, 128, 1163),
    ("f32", False, 64, 128, 4, False, 974, 1120, 1051),
    ("f32", False, 64, 128, 4, False, 1155, 1152, 839),
    ("f32", False, 64, 128, 4, True, 2306, 4704, 783),
    ("f32", False, 64, 128, 4, True, 1793, 4096, 1045),
    ("f32", True, 64, 128, 2, False, 513, 32, 533),
    ("f32", True, 64, 128, 2, False, 613, 128, 561),
    ("f32", True, 64, 128, 2, True, 773, 32, 1219),
    ("f32", True, 64, 128, 2, True, 777, 128, 1223),
    ("f32", True, 64, 128, 4, False, 587, 1120, 589),
    ("f32", True, 64, 128, 4, False, 527, 1152, 609),
    ("2byte", True, 64, 128, 4, True, 16392, 8192, 1),
    ("f32", True, 64, 128, 4, True, 16392, 8192, 17),
]
# workgroups that stay for a second and third tile: more 256 x 256 tiles than CUs, twice with rows past the last one
STAY = [(False, 8656, 512, 2309), (False, 9985, 1056, 3079), (False, 4123, 640, 8238), (True, 2817, 544, 5389), (True, 3808, 512, 2694)]
# weight tiles a workgroup of few rows: tiles, 2-byte x as it is, gated, n, k
WIDE = [(1, True, False, 8191, 512), (2, True, False, 8199, 544), (2, False, False, 8192, 512), (2, True, False, 16401, 1024),
        (4, False, False, 16390, 1056), (4, True, False, 24583, 1024), (1, False, True, 16383, 1024), (2, False, True, 16391, 1024),
        (2, True, True, 16391, 1120), (1, True, True, 16391, 992), (2, True, False, 24583, 992)]
# rows past the last tile: x as it is, and packed
PLAIN_REST = [("bf16", 1537, 96, 2607), ("bf16", 16390, 3264, 17), ("bf16", 5126, 32, 4757),
              ("bf16", 3076, 96, 5258), ("f32", 1802, 32, 1033), ("f32", 2306, 4704, 783)]
PACKED_REST = [(False, 1418, 736, 1409), (False, 833, 640, 2449), (False, 16388, 3616, 31), (False, 8195, 5120, 79),
               (False, 514, 32, 7596), (False, 577, 128, 6907), (False, 1936, 288, 2120), (False, 1665, 384, 2381),
               (False, 5902, 576, 2724), (False, 3085, 512, 4922), (True, 835, 288, 1167), (True, 1224, 384, 784),
               (True, 1800, 288, 1115), (True, 1161, 384, 1675), (True, 1545, 544, 4978), (True, 2562, 512, 2948)]
ACTS = {"64": "silu", "128": "gelu_erf", "256": "gelu_tanh"}


@pytest.mark.parametrize("kind,gated,rows,cols,groups,split,m,k,n", TILES)
def test_tile(ops, dev, kind, gated, rows, cols, groups, split, m, k, n):
    arith = "fp4" if kind == "fp4" else "plain"
    for dt in {"fp4": ["bf16"], "2byte": ["bf16", "f16"], "f32": ["f32"]}[kind]:
        for out, bias in (("same", True),
              ("f32" if dt != "f32" else "f16", False)):
            if gated:
                run_gated(ops, dev, m, k, n, dt, arith, ACTS[str(rows)], out, use_bias=bias)
            else:
                run_linear(ops, dev, m, k, n, dt, arith, out, use_bias=bias)


@pytest.mark.parametrize("gated,m,k,n", STAY)
def test_workgroups_that_stay(ops, dev, gated, m, k, n):
    for out, bias in (("same", True),
              ("f32", False)):
        if gated:
            run_gated(ops, dev, m, k, n, "bf16", "fp4", "gelu_tanh", out, use_bias=bias)
        else:
            run_linear(ops, dev, m, k, n, "bf16", "fp4", out, use_bias=bias)


@pytest.mark.parametrize("m", [1, 5, 16])
@pytest.mark.parametrize("tiles,plain_2byte,gated,n,k", WIDE)
def test_wide_weights(ops, dev, m, tiles, plain_2byte, gated, n, k):
    for dt, arith in (("bf16", "plain"), ("f16", "plain")) if plain_2byte else (("f32", "plain"), ("bf16", "fp4"),
              ("f32", "fp4")):
        if gated:
            run_gated(ops, dev, m, k, n, dt, arith, "silu")
        else:
            run_linear(ops, dev, m, k, n, dt, arith)


@pytest.mark.parametrize("m", [16, 13])
def test_packed_few_rows_of_wide_weights(ops, dev, m):
    """A packed x gives the bits of the x that it was quantized from."""
    x, w = tokens(dev, m, 1056, "bf16"), weight(dev, 16391, 1056)
    assert torch.equal(ops.mxfp4_linear_fp4(ops.mxfp4_quantize(x), *w), ops.mxfp4_linear_fp4(x, *w))


@pytest.mark.parametrize("dt,m,k,n", PLAIN_REST)
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


@pytest.mark.parametrize("gated,m,k,n", PACKED_REST)
def test_packed_rows_past_the_last_tile(ops, dev, gated, m, k, n):
    x, w, v = tokens(dev, m, k, "bf16"), weight(dev, n, k), weight(dev, n, k, 1)
    pair = ops.mxfp4_quantize(x)
    if gated:
        assert torch.equal(ops.mxfp4_linear_gated(pair, v, w, fp4=True), ops.mxfp4_linear_gated(x, v, w, fp4=True))
    else:
        assert torch.equal(ops.mxfp4_linear_fp4(pair, *w), ops.mxfp4_linear_fp4(x, *w))


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,k", [(8200, 64), (3001, 1632), (8191, 512), (70000, 32), (33001, 128), (17003, 160), (16390, 256),
                                 (900, 96), (901, 224), (5001, 288)])
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
