"""Microscaled 4-bit quantisation and the linears on it against their definitions in 64 bits (tests/mxfp4_reference.py has
the formulas and the bounds' derivation). Quantisation is held to equality."""
import math

import pytest

torch = pytest.importorskip("torch")

import mxfp4_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu

DT = ref.DT
ACTS = ["silu", "gelu_erf", "gelu_tanh"]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def ops(dev):
    from lux3d_fused import ops as _ops
    return _ops


def rnd(dev, *shape, seed=0, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed + sum(s * (7 ** i) for i, s in enumerate(shape)))
    return torch.randn(shape, generator=g, device=dev) * std


def tokens(dev, m, k, dt, seed=0):
    """Rows of different size, a few channels far larger than the others, one row of zeros."""
    x = rnd(dev, m, k, seed=seed) * torch.exp(rnd(dev, m, 1, seed=seed + 1, std=0.7))
    x[:, ::37] *= 9.0
    if m > 2:
        x[m // 2] = 0
    return x.to(DT[dt])


def weight(dev, n, k, seed=0):
    codes, s = ref.quantize(rnd(dev, n, k, seed=seed, std=1.0 / math.sqrt(k)))
    return ref.pack(codes, s)


# ---- quantisation ---------------------------------------------------------------

def same_as_defined(q, scales, x, what):
    codes, s = ref.quantize(x.reshape(-1, x.shape[-1]))
    got_codes, got_s = ref.unpack(q, scales)
    assert torch.equal(got_s.cpu(), s.int().cpu()), f"{what}: exponents"
    fine = (s != 255).repeat_interleave(32, 1)
    assert torch.equal(got_codes[fine], codes[fine]), f"{what}: codes"
    pad = scales.permute(1, 0, 2).reshape(scales.shape[1], -1)[:, x.shape[-1] // 32:]
    assert int(pad.sum()) == 0, f"{what}: bytes past the last block"


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,k", [(1, 32), (2, 64), (3, 96), (31, 128), (32, 160), (33, 512), (65, 544), (7, 2048), (1000, 1056)])
def test_quantize(ops, dev, m, k, dt):
    x = tokens(dev, m, k, dt)
    q, s = ops.mxfp4_quantize(x)
    assert q.shape == (m, k // 2) and s.shape == ((k + 127) // 128, m, 4)
    same_as_defined(q, s, x, f"{m} x {k} {dt}")
    for out in DT.values():
        y = ops.mxfp4_dequantize(q, s, out)
        assert torch.equal(y, ref.dense(q, s).to(torch.float32).to(out))


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_quantize_ties_and_borders(ops, dev, dt):
    """Every half-way value, its neighbours, powers of two and the values that saturate, under every exponent of the type."""
    base = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.75, 6.0, 4.0, 2.0, 1.0, 0.5, 0.0, 0.125], dtype=torch.float64)
    fi = torch.finfo(DT[dt])
    row = torch.cat([base, -base * (1 + fi.eps), base.new_tensor([4.0]), base[1:] * (1 - fi.eps / 2), -base.flip(0)])
    lo, hi = (-24, 13) if dt == "f16" else (-140, 125)
    x = (row * ref.power(torch.arange(lo, hi))[:, None]).to(DT[dt])
    q, s = ops.mxfp4_quantize(x.to(dev))
    same_as_defined(q.cpu(), s.cpu(), x, dt)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_quantize_blocks_that_are_not_finite(ops, dev, dt):
    x = tokens(dev, 40, 160, dt)
    x[3, 33], x[4, 0], x[5, 159] = float("inf"), float("nan"), float("-inf")
    q, s = ops.mxfp4_quantize(x)
    same_as_defined(q, s, x, dt)
    y = ops.mxfp4_dequantize(q, s, torch.float32)
    bad = torch.zeros(40, 5, dtype=torch.bool, device=dev)
    bad[3, 1] = bad[4, 0] = bad[5, 4] = True
    assert torch.equal(torch.isnan(y), bad.repeat_interleave(32, 1))


def test_quantize_views(ops, dev):
    from lux3d_fused import _lib
    with pytest.raises(_lib.Lux3dError, match="aligned"):    # 1400 bytes a row
        ops.mxfp4_quantize(tokens(dev, 60, 700, "bf16")[:, 8:8 + 640])
    wide = tokens(dev, 60, 704, "bf16")
    x = wide[:, 8:8 + 640].reshape(3, 20, 640)
    q, s = ops.mxfp4_quantize(wide[:, 8:8 + 640])
    q3, s3 = ops.mxfp4_quantize(x)
    assert q3.shape == (3, 20, 320) and torch.equal(q3.view(60, 320), q) and torch.equal(s3, s)
    same_as_defined(q, s, x, "a column slice")
    every = wide[::3, 8:648]
    same_as_defined(*ops.mxfp4_quantize(every), every, "every third row")
    assert ops.mxfp4_dequantize(q3, s3, torch.bfloat16).shape == (3, 20, 640)


def test_dequantize_any_byte(ops, dev):
    """Every code under every exponent byte, 255 among them."""
    codes = torch.arange(32, device=dev, dtype=torch.uint8).remainder(16).expand(256, 32)
    s = torch.arange(256, device=dev)[:, None]
    q, scales = ref.pack(codes, s)
    want = ref.values(codes, s)
    for dt in DT.values():
        y = ops.mxfp4_dequantize(q, scales, dt)
        assert torch.equal(torch.isnan(y), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(y, nan=7.0), torch.nan_to_num(want.to(torch.float32).to(dt), nan=7.0))


def test_scales_of_a_checkpoint(ops, dev):
    for blocks in (1, 3, 4, 9):
        e = torch.randint(0, 255, (11, blocks), device=dev).to(torch.uint8)
        assert torch.equal(ops.mxfp4_scales(e), ref.pack(torch.zeros(11, 32 * blocks, dtype=torch.uint8, device=dev), e)[1])


# ---- the linears ----------------------------------------------------------------

def as_products_see(x, arith):
    """x as it enters the products, in f64, and the error of its entry."""
    if arith == "fp4":
        return ref.values(*ref.quantize(x)), 0.0
    return x.double(), 2 * ref.U if x.dtype == torch.float32 else 0.0


def call(ops, x, w, bias, arith, out=None):
    return (ops.mxfp4_linear_fp4 if arith == "fp4" else ops.mxfp4_linear)(x, *w, bias=bias, out_dtype=out)


def run_linear(ops, dev, m, k, n, dt, arith, out="same", seed=0, use_bias=True):
    print(f"[case] {arith} {dt} {m} x {k} -> {n} out {out}", flush=True)
    x, w = tokens(dev, m, k, dt, seed), weight(dev, n, k, seed)
    bias = rnd(dev, n, seed=seed, std=0.3) if use_bias else None
    y = call(ops, x, w, bias, arith, None if out == "same" else DT[out])
    torch.cuda.synchronize()
    assert y.shape == (m, n) and y.dtype == (DT[dt] if out == "same" else DT[out])
    xd, e = as_products_see(x, arith)
    ref.check(y, *ref.product(xd, ref.dense(*w), bias, e), f"{arith} {dt} {m} x {k} -> {n}")
    return x, w, bias, y


def run_gated(ops, dev, m, k, n, dt, arith, act, out="same", seed=0, use_bias=True):
    print(f"[case] gated {act} {arith} {dt} {m} x {k} -> {n} out {out}", flush=True)
    x, gate, up = tokens(dev, m, k, dt, seed), weight(dev, n, k, seed + 1), weight(dev, n, k, seed + 2)
    bg, bu = (rnd(dev, n, seed=seed, std=0.3), rnd(dev, n, seed=seed + 9, std=0.3)) if use_bias else (None, None)
    y = ops.mxfp4_linear_gated(x, gate, up, act, gate_bias=bg, up_bias=bu, fp4=arith == "fp4",
                               out_dtype=None if out == "same" else DT[out])
    torch.cuda.synchronize()
    assert y.shape == (m, n) and y.dtype == (DT[dt] if out == "same" else DT[out])
    xd, e = as_products_see(x, arith)
    ref.check(y, *ref.gated(ref.product(xd, ref.dense(*gate), bg, e), ref.product(xd, ref.dense(*up), bu, e), act),
              f"gated {act} {arith} {dt} {m} x {k} -> {n}")
    return x, gate, up, bg, bu, y


@pytest.mark.parametrize("arith", ["plain", "fp4"])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m", [1, 2, 7, 15, 16, 17, 31, 32, 33, 47, 64, 65, 127, 128, 129, 257, 515])
@pytest.mark.parametrize("k,n", [(32, 7), (160, 130), (1024, 257), (2080, 64)])
def test_linear(ops, dev, m, k, n, dt, arith):
    run_linear(ops, dev, m, k, n, dt, arith)


@pytest.mark.parametrize("arith", ["plain", "fp4"])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m,k,n", [(1, 32, 1), (2, 2048, 512), (16, 96, 33), (17, 224, 40), (40, 1120, 300), (130, 64, 129),
                                   (300, 1024, 1000), (513, 352, 260)])
def test_gated(ops, dev, m, k, n, dt, arith):
    for act in ACTS:
        run_gated(ops, dev, m, k, n, dt, arith, act)


# sizes around the borders between kernels and tiles
@pytest.mark.parametrize("arith", ["plain", "fp4"])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("m,k,n", [(255, 128, 255), (256, 256, 256), (257, 384, 513), (1029, 1024, 1024), (2049, 512, 1536),
                                   (4100, 256, 2050), (3000, 96, 4097), (8200, 64, 1030)])
def test_larger(ops, dev, m, k, n, dt, arith):
    run_linear(ops, dev, m, k, n, dt, arith)
    run_gated(ops, dev, m, k, n, dt, arith, "silu")


@pytest.mark.parametrize("arith", ["plain", "fp4"])
@pytest.mark.parametrize("m", [3, 16, 50, 300])
def test_output_types_and_no_bias(ops, dev, m, arith):
    for dt in DT:
        for out in DT:
            run_linear(ops, dev, m, 256, 72, dt, arith, out, use_bias=False)
            run_gated(ops, dev, m, 256, 72, dt, arith, "gelu_erf", out, use_bias=False)


def test_every_k_up_to_a_few_groups(ops, dev):
    for k in range(32, 673, 32):
        for m in (5, 33, 140):
            for arith in ("plain", "fp4"):
                run_linear(ops, dev, m, k, 70, "bf16", arith)


def test_activations_far_out(ops, dev):
    """The activation over its whole range, by a product that passes x through: tails to either side and zero."""
    k = 32
    codes = torch.zeros((64, k), dtype=torch.uint8, device=dev)
    codes[:, 0] = 2                                                     # one
    one = ref.pack(codes, torch.full((64, 1), 127, device=dev))
    x = torch.zeros((4001, k), device=dev)
    x[:, 0] = torch.linspace(-40, 40, 4001, device=dev)
    ones = torch.ones(64, device=dev)
    zero = ref.pack(torch.zeros_like(codes), torch.full((64, 1), 127, device=dev))
    for act in ACTS:
        y = ops.mxfp4_linear_gated(x, one, zero, act, up_bias=ones)
        want, bound = ref.activation(x[:, :1].double().expand(-1, 64), act)
        ref.check(y, want, bound, act)
        assert float(ops.mxfp4_linear_gated(torch.zeros_like(x[:20]), one, zero, act, up_bias=ones).abs().max()) == 0
    for v, want in ((float("inf"), float("inf")), (float("nan"), float("nan"))):
        x[:, 0] = 0
        bias = torch.full((64,), v, device=dev)
        for act in ACTS:
            y = ops.mxfp4_linear_gated(x[:20], one, zero, act, gate_bias=bias, up_bias=ones)
            assert bool((y == want).all()) or (math.isnan(want) and bool(torch.isnan(y).all()))


@pytest.mark.parametrize("m", [9, 40, 300])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_packed_x_is_the_quantized_x(ops, dev, m, dt):
    """One quantization for several projections gives the bits that each one's own gives."""
    x, w, bias, y = run_linear(ops, dev, m, 544, 200, dt, "fp4")
    pair = ops.mxfp4_quantize(x)
    assert torch.equal(ops.mxfp4_linear_fp4(pair, *w, bias=bias, out_dtype=DT[dt]), y)
    x, gate, up, bg, bu, y = run_gated(ops, dev, m, 544, 200, dt, "fp4", "silu")
    pair = ops.mxfp4_quantize(x)
    assert torch.equal(ops.mxfp4_linear_gated(pair, gate, up, "silu", gate_bias=bg, up_bias=bu, fp4=True, out_dtype=DT[dt]), y)
    assert ops.mxfp4_linear_fp4(pair, *w).dtype == torch.bfloat16


@pytest.mark.parametrize("m", [8, 90, 700])
@pytest.mark.parametrize("arith", ["plain", "fp4"])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_a_row_that_is_not_finite_stays_alone(ops, dev, m, dt, arith):
    x, w, bias, y = run_linear(ops, dev, m, 288, 150, dt, arith)
    rows = [1, m // 2, m - 1]
    x[rows[0], 5], x[rows[1], 280], x[rows[2], 100] = float("nan"), float("inf"), float("nan")
    z = call(ops, x, w, bias, arith)
    keep = torch.ones(m, dtype=torch.bool, device=dev)
    keep[rows] = False
    assert torch.equal(z[keep], y[keep]) and not torch.isfinite(z[~keep]).any()


@pytest.mark.parametrize("m", [8, 90, 700])
@pytest.mark.parametrize("arith", ["plain", "fp4"])
def test_weight_blocks_of_nan_and_bytes_past_the_row(ops, dev, m, arith):
    """A weight block of NaN reaches its own column alone; scale bytes past a row's last block are not scales."""
    x, w, bias, y = run_linear(ops, dev, m, 160, 150, "bf16", arith)
    x = torch.where(x == 0, torch.ones_like(x), x)
    y = call(ops, x, w, bias, arith)
    q, s = w[0].clone(), w[1].clone()
    s[1, :, 1:] = 255
    assert torch.equal(call(ops, x, (q, s), bias, arith), y)
    s[0, 77, 2] = 255
    z = call(ops, x, (q, s), bias, arith)
    keep = torch.arange(150, device=dev) != 77
    assert torch.isnan(z[:, 77]).all() and torch.equal(z[:, keep], y[:, keep])
    if arith == "fp4":
        pq, ps = ops.mxfp4_quantize(x)
        ps[1, :, 1:] = 255
        assert torch.equal(ops.mxfp4_linear_fp4((pq, ps), *w, bias=bias), y)


@pytest.mark.parametrize("m", [4, 40, 300])
@pytest.mark.parametrize("arith", ["plain", "fp4"])
def test_scales_over_the_whole_range(ops, dev, m, arith):
    """Exponents far apart within a row and at the format's ends, weights and x so that no product leaves f32."""
    k, n = 256, 96
    codes = torch.randint(0, 16, (n, k), generator=torch.Generator().manual_seed(m)).to(torch.uint8).to(dev)
    s = torch.randint(60, 180, (n, k // 32), generator=torch.Generator().manual_seed(m + 1)).to(dev)
    s[:5], s[5:9] = 3, 200
    w = ref.pack(codes, s)
    x = tokens(dev, m, k, "bf16") * 2.0 ** 20
    y = call(ops, x, w, None, arith, torch.float32)
    xd, e = as_products_see(x, arith)
    ref.check(y, *ref.product(xd, ref.dense(*w), None, e), "wide scales")


@pytest.mark.parametrize("m", [5, 40, 300])
def test_strides_and_what_lies_beside_y(ops, dev, m):
    """x as a slice of wider rows, batches, y as a slice: its rows' neighbours stay as they were, aligned or not."""
    from lux3d_fused import _lib
    w = weight(dev, 77, 256)
    for linear in (ops.mxfp4_linear, ops.mxfp4_linear_fp4):
        with pytest.raises(_lib.Lux3dError, match="aligned"):  # 1400 bytes a row
            linear(tokens(dev, m, 700, "bf16")[:, 16:16 + 256], *w)
    wide = tokens(dev, m, 704, "bf16")
    x = wide[:, 16:16 + 256]
    want = ops.mxfp4_linear(x.contiguous(), *w)
    assert torch.equal(ops.mxfp4_linear(x, *w), want)
    assert torch.equal(ops.mxfp4_linear_fp4(x, *w), ops.mxfp4_linear_fp4(x.contiguous(), *w))
    for dt in DT.values():
        whole = ops.mxfp4_linear(x, *w, out_dtype=dt)
        for left, width in ((0, 96), (8, 96), (3, 83)):
            big = torch.full((m + 2, width), 5.0, dtype=dt, device=dev)
            y = big[1:m + 1, left:left + 77]
            _lib.call("lux3d_mxfp4_linear", ops._d(x), ops._d(w[0]), ops._d(w[1]), None, ops._d(y), ops._stream(x))
            assert torch.equal(y, whole)
            big[1:m + 1, left:left + 77] = 5.0
            assert bool((big == 5.0).all())


def test_batches(ops, dev):
    x, w = tokens(dev, 60, 128, "bf16"), weight(dev, 40, 128)
    y = ops.mxfp4_linear(x.view(3, 4, 5, 128), *w)
    assert y.shape == (3, 4, 5, 40) and torch.equal(y.view(60, 40), ops.mxfp4_linear(x, *w))
    y = ops.mxfp4_linear_fp4(x.view(3, 20, 128), *w)
    assert y.shape == (3, 20, 40) and torch.equal(y.view(60, 40), ops.mxfp4_linear_fp4(x, *w))
    pair = ops.mxfp4_quantize(x.view(3, 20, 128))
    assert torch.equal(ops.mxfp4_linear_fp4(pair, *w), y)
    assert ops.mxfp4_linear(x[0], *w).shape == (40,)


def test_empty(ops, dev):
    x, w = tokens(dev, 4, 128, "bf16"), weight(dev, 40, 128)
    q, s = ops.mxfp4_quantize(x[:0])
    assert q.shape == (0, 64) and s.shape == (1, 0, 4) and ops.mxfp4_dequantize(q, s).shape == (0, 128)
    assert ops.mxfp4_linear(x[:0], *w).shape == (0, 40)
    assert ops.mxfp4_linear_fp4(x[:0], *w).shape == (0, 40)
    assert ops.mxfp4_linear_fp4((q, s), *w).shape == (0, 40)
    assert ops.mxfp4_linear_gated(x[:0], w, w).shape == (0, 40)
    none = (w[0][:0].contiguous(), w[1][:, :0].contiguous())
    assert ops.mxfp4_linear(x, *none).shape == (4, 0)
    torch.cuda.synchronize()


@pytest.mark.parametrize("m", [6, 40, 700])
@pytest.mark.parametrize("arith", ["plain", "fp4"])
def test_same_bits_on_any_stream_and_in_graphs(ops, dev, m, arith):
    """Two captured calls and eager ones between their replays, each with workspaces of its own."""
    k, n = 512, 384
    w, v = weight(dev, n, k, 1), weight(dev, n, k, 2)
    xs = [tokens(dev, m, k, "bf16", seed=s) for s in (1, 2)]
    fn = lambda x: (call(ops, x, w, None, arith), ops.mxfp4_linear_gated(x, w, v, "gelu_erf", fp4=arith == "fp4"))  # noqa: E731
    eager = [fn(x) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = fn(xs[1])
    again = fn(xs[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, eager[1])) and all(torch.equal(a, b) for a, b in zip(again, eager[0]))
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(fn(x))
        graphs.append(g)
    for _ in range(4):
        for pair in outs:
            for o in pair:
                o.fill_(float("nan"))
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        fn(xs[0])
        torch.cuda.synchronize()
        for pair, want in zip(outs, eager):
            assert all(torch.equal(a, b) for a, b in zip(pair, want))
    xs[0].copy_(xs[1])                                       # a replay reads x as it is then
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], eager[1]))


def test_offsets_past_32_bits(ops, dev):
    """A weight and an x of more than 2^31 bytes: their last rows."""
    k, n, m = 65536, 66000, 40
    x = tokens(dev, m, k, "bf16")
    q = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=dev)
    s = torch.randint(110, 122, (k // 128, n, 4), dtype=torch.uint8, device=dev)
    part = (q[-200:].contiguous(), s[:, -200:].contiguous())
    for arith in ("plain", "fp4"):
        for rows in (3, m):
            xd, e = as_products_see(x[:rows], arith)
            ref.check(call(ops, x[:rows], (q, s), None, arith)[:, -200:], *ref.product(xd, ref.dense(*part), None, e), arith)
    del q, s
    m, k = 40000, 65536
    w = weight(dev, 48, k)
    x = torch.randn((m, k), device=dev, dtype=torch.bfloat16)
    for arith in ("plain", "fp4"):
        y = call(ops, x, w, None, arith)
        xd, e = as_products_see(x[-64:], arith)
        ref.check(y[-64:], *ref.product(xd, ref.dense(*w), None, e), arith)


@pytest.mark.parametrize("m", [2, 300])
@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("act", ["gelu_erf", "silu"])
def test_feed_forward_block(ops, dev, m, fp4, act):
    """The operators as a transformer block runs them: AdaLN modulate, the gated feed-forward on packed weights, the gated
    residual. Each step is held to its definition on what the step before gave."""
    c, h, seg = 512, 1088, 2
    arith = "fp4" if fp4 else "plain"
    dense = [rnd(dev, h, c, seed=1, std=c ** -0.5), rnd(dev, h, c, seed=2, std=c ** -0.5), rnd(dev, c, h, seed=3, std=h ** -0.5)]
    gate, up, down = (ops.Mxfp4MatMul.from_dense(w) for w in dense)
    for w, d in zip((gate, up, down), dense):
        assert torch.equal(w.dequantize(torch.float32).double(), ref.values(*ref.quantize(d)))
    bias = rnd(dev, c, seed=4, std=0.2)
    x = tokens(dev, m, c, "bf16").view(seg, m // seg, c)
    mod = rnd(dev, seg, 6 * c, seed=5, std=0.3)
    shift, scale, gate_mlp = mod.chunk(6, dim=-1)[3:]
    n = ops.adaln_modulate(x, shift, scale)
    mlp = ops.Mxfp4GatedMlp(gate, up, down, act, down_bias=bias, fp4=fp4)
    z = mlp.forward(n)
    out = ops.gated_residual(x, z, gate_mlp)
    hidden = ops.mxfp4_linear_gated(n, (gate.q, gate.scales), (up.q, up.scales), act, fp4=fp4)
    xd, e = as_products_see(n.reshape(m, c), arith)
    ref.check(hidden, *ref.gated(ref.product(xd, ref.dense(gate.q, gate.scales), None, e),
                                 ref.product(xd, ref.dense(up.q, up.scales), None, e), act), "hidden")
    hd, e = as_products_see(hidden.reshape(m, h), arith)
    ref.check(z, *ref.product(hd, ref.dense(down.q, down.scales), bias, e), "down")
    want = x.double() + z.double() * gate_mlp.double()[:, None]
    ref.check(out, want.reshape(m, c), (4 * ref.U * (x.double().abs() + (z.double() * gate_mlp.double()[:, None]).abs())).reshape(m, c), "residual")
