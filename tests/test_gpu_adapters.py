"""lux3d_q8_0_linear_adapters against the formula in 64 bits.

Tolerances, with u = 2^-24 and e = eps / 2 of a type (half a rounding step): a sum of K products is formed in f32, at most
16 of them between two roundings' worth of chain, so it is off by at most (K / 16 + 64) u of its terms' magnitudes (the f32
linear's products are each within 2 u of exact as well); t = alpha x A^T is rounded once to x's type, by e |t| (f32: u); the
second product sums rank terms more; the store adds e |y| of its type. Weights count as x's type holds them.
"""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def ops(dev):
    from lux3d_fused import ops as _ops
    return _ops


def make(dev, m, k, n, r, na, dt, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + m * 7 + k + n * 3 + r)
    rnd = lambda shape, std=1.0, t=torch.float32: (torch.randn(shape, generator=g, device=dev) * std).to(t)  # noqa: E731
    qs = torch.randint(-127, 128, (n, k), generator=g, device=dev, dtype=torch.int32).to(torch.int8)
    scales = ((torch.rand((n, k // 32), generator=g, device=dev) * 0.02 + 0.004) / math.sqrt(k)).half().float()
    return dict(x=rnd((m, k), t=DT[dt]), qs=qs, scales=scales, bias=rnd(n, 0.5), a=rnd((na, r, k), 1 / math.sqrt(k), DT[dt]),
                b=rnd((na, n, r), 1 / math.sqrt(r), DT[dt]), alphas=rnd(na, 0.5) + 1.0)


def segment_of_rows(offs, rows, nseg):
    if offs is None:
        return torch.arange(rows) // max(1, rows // nseg)
    return (torch.searchsorted(offs.cpu(), torch.arange(rows), right=True) - 1).clamp(0, nseg - 1)


def reference(c, ids, offs, rows_shape_dt, use_bias=True, use_alpha=True):
    """(y, bound without the store)"""
    x = c["x"].reshape(-1, c["x"].shape[-1])
    m, k = x.shape
    n, r, na = c["qs"].shape[0], c["a"].shape[1], c["a"].shape[0]
    f32 = x.dtype == torch.float32
    e = U if f32 else torch.finfo(x.dtype).eps / 2
    w = (c["qs"].double() * c["scales"].double().repeat_interleave(32, 1)).to(x.dtype).double()
    xd = x.double()
    step = lambda terms: (terms / 16 + 64) * U  # noqa: E731
    mm = lambda p, q: torch.mm(p, q.t().contiguous())  # noqa: E731
    y, err = mm(xd, w), mm(xd.abs(), w.abs()) * (step(k) + 2 * U)
    if use_bias:
        y, err = y + c["bias"].double(), err + U * c["bias"].double().abs()
    which = ids.cpu().long()[segment_of_rows(offs, m, ids.numel())]
    for j in range(na):
        rows = (which == j).nonzero().flatten().to(x.device)
        if not rows.numel():
            continue
        a, b = c["a"][j].double(), c["b"][j].double()
        al = c["alphas"][j].double() if use_alpha else torch.ones((), dtype=torch.float64, device=x.device)
        t = al * mm(xd[rows], a)
        t_err = al.abs() * mm(xd[rows].abs(), a.abs()) * (step(k) + U) + (e + U) * t.abs()
        y[rows] += mm(t, b)
        err[rows] += mm(t_err, b.abs()) + mm(t.abs() + t_err, b.abs()) * (step(r) + r * U + 2 * U)
    return y, err + 2 * U * y.abs()


def check(got, ref, what):
    want, bound = ref
    fi = torch.finfo(got.dtype)
    bound = bound + fi.eps / 2 * (want.abs() + bound) + fi.smallest_normal * fi.eps
    got = got.reshape(want.shape)
    assert torch.isfinite(got).all(), what
    over = (got.double() - want).abs() - bound
    assert float(over.max()) <= 0, f"{what}: worst error {float((got.double() - want).abs().max()):.3g}, {int((over > 0).sum())} values past the bound"


def run(ops, dev, m, k, n, r, dt, cuts, ids, na=3, out="same", seed=0, **kw):
    c = make(dev, m, k, n, r, na, dt, seed)
    ids = torch.tensor(ids, dtype=torch.int32, device=dev)
    offs = None if cuts is None else torch.tensor(cuts, dtype=torch.int64, device=dev)
    out_dt = DT[dt] if out == "same" else DT[out]
    print(f"[case] rows {m} k {k} n {n} rank {r} {dt} -> {out} cuts {cuts} ids {ids.tolist()}", flush=True)
    y = ops.q8_0_linear_adapters(c["x"], c["qs"], c["scales"], c["a"], c["b"], ids, alphas=c["alphas"], seg_offsets=offs,
                                 bias=c["bias"], out_dtype=out_dt, **kw)
    torch.cuda.synchronize()
    assert y.dtype == out_dt and y.shape == (m, n)
    check(y, reference(c, ids, offs, None), "y")
    return c, ids, offs, y


def cuts_of(m, s):
    """s ragged segments of m rows, some of them empty."""
    c = sorted(int(m * f) for f in (0.0, 0.03, 0.03, 0.2, 0.31, 0.7, 0.93)[:s])
    return c + [m]


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 130, 257, 1029])
@pytest.mark.parametrize("k,n,r", [(64, 40, 16), (1024, 1536, 8), (512, 1000, 17)])
def test_rows(ops, dev, m, k, n, r, dt):
    run(ops, dev, m, k, n, r, dt, cuts_of(m, 7), [0, 2, 1, -1, 2, 1, 0])


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("r", [1, 2, 3, 4, 8, 12, 16, 24, 32, 33, 64, 65, 100, 130])
@pytest.mark.parametrize("m", [5, 300])
def test_ranks(ops, dev, m, r, dt):
    run(ops, dev, m, 256, 200, r, dt, cuts_of(m, 5), [1, 0, 2, 2, 0])


@pytest.mark.parametrize("m,k,n", [(1, 32, 8), (7, 96, 33), (200, 96, 130), (20, 1056, 64)])
def test_odd_blocks_of_k(ops, dev, m, k, n):
    run(ops, dev, m, k, n, 16, "bf16", cuts_of(m, 4), [0, 1, 2, -1])


# each GEMM tile: few rows, 32 / 64 / 128 / 160 x 128, 128 and 256 x 256
@pytest.mark.parametrize("m,k,n,dt", [(40, 1024, 4096, "bf16"), (256, 1024, 1024, "bf16"), (600, 512, 2048, "bf16"),
                                      (1300, 256, 4096, "bf16"), (4096, 256, 4096, "bf16"), (5000, 128, 8192, "bf16"),
                                      (3100, 128, 1024, "f32"), (512, 256, 1024, "f32"), (4096, 64, 4096, "f32")])
@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
def test_tiles_and_output_types(ops, dev, m, k, n, dt, out):
    run(ops, dev, m, k, n, 32, dt, cuts_of(m, 7), [0, 2, 1, -1, 2, 1, 0], out=out)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_a_request_a_row(ops, dev, dt):
    """Every row an adapter of its own, more segments than a wavefront has lanes."""
    for m in (12, 70, 200):
        run(ops, dev, m, 256, 384, 16, dt, list(range(m + 1)), [(5 * i) % 9 - 1 for i in range(m)], na=8)


def test_rows_before_and_past_the_offsets(ops, dev):
    for m in (30, 400):
        run(ops, dev, m, 128, 160, 8, "bf16", [4, 9, 17], [1, 2])


def test_ids_that_are_no_adapter(ops, dev):
    bad = torch.full((1,), 77, dtype=torch.int32, device=dev)
    for m in (9, 300):
        run(ops, dev, m, 128, 160, 8, "bf16", cuts_of(m, 6), [3, -1, -2, 0, 1 << 30, 2], bad_ids=bad)
        assert int(bad) == 3
        run(ops, dev, m, 128, 160, 8, "bf16", cuts_of(m, 3), [2, -1, 0], bad_ids=bad)
        assert int(bad) == 0


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("m", [9, 300])
def test_no_adapter_is_the_linear(ops, dev, m, dt):
    c, ids, offs, y = run(ops, dev, m, 256, 160, 8, dt, cuts_of(m, 3), [-1, -1, -1])
    assert torch.equal(y, ops.q8_0_linear(c["x"], c["qs"], c["scales"], c["bias"], out_dtype=DT[dt]))


@pytest.mark.parametrize("m", [9, 300])
def test_neighbours_do_not_leak(ops, dev, m):
    """A request's rows do not depend on what the others hold: NaN and infinities in their rows and adapters."""
    cuts = [0, m // 3, 2 * m // 3, m]
    c, ids, offs, y = run(ops, dev, m, 256, 160, 12, "bf16", cuts, [0, 1, -1])
    c["x"][cuts[1]:cuts[2]] = float("nan")
    c["a"][1], c["b"][1], c["alphas"][1] = float("inf"), float("nan"), float("nan")
    c["a"][2], c["b"][2] = float("nan"), float("nan")
    z = ops.q8_0_linear_adapters(c["x"], c["qs"], c["scales"], c["a"], c["b"], ids, alphas=c["alphas"], seg_offsets=offs,
                                 bias=c["bias"])
    keep = list(range(cuts[1])) + list(range(cuts[2], m))
    assert torch.equal(z[keep], y[keep]) and torch.isnan(z[cuts[1]:cuts[2]]).all()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,nseg", [(40, 160, 65), (40, 160, 66), (1500, 256, 256), (1500, 256, 257), (1500, 256, 1500), (3000, 1000, 900), (8200, 160, 700)])
def test_many_segments(ops, dev, m, n, nseg, dt):
    """Past 64 and past 256 segments, many of them empty."""
    g = torch.Generator().manual_seed(nseg)
    cuts = [0] + sorted(torch.randint(0, m + 1, (nseg - 1,), generator=g).tolist()) + [m]
    run(ops, dev, m, 192, n, 20, dt, cuts, (torch.randint(0, 4, (nseg,), generator=g) - 1).tolist())


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("m,k,n", [(9, 512, 160), (30, 512, 160), (60, 64, 200), (61, 1024, 1536), (300, 512, 1000), (700, 512, 4096),
                                   (2500, 512, 2048)])
def test_an_adapter_that_is_not_finite_stays_with_its_rows(ops, dev, m, k, n, dt):
    """Segments of a few rows, several in every tile of rows; every other one's adapter becomes NaN."""
    cuts, at = [0], 0
    while at < m:
        at = min(m, at + (1, 3, 7, 2, 20)[len(cuts) % 5])
        cuts.append(at)
    ids = [(0, 1, 2, -1)[i % 4] for i in range(len(cuts) - 1)]
    c, ids_t, offs, y = run(ops, dev, m, k, n, 20, dt, cuts, ids)
    c["a"][1], c["b"][1] = float("nan"), float("inf")
    z = ops.q8_0_linear_adapters(c["x"], c["qs"], c["scales"], c["a"], c["b"], ids_t, alphas=c["alphas"], seg_offsets=offs,
                                 bias=c["bias"], out_dtype=DT[dt])
    hit = (torch.tensor(ids)[segment_of_rows(offs, m, len(ids))] == 1).to(dev)
    assert torch.equal(z[~hit], y[~hit]) and torch.isnan(z[hit]).all()


def test_batches_strided_rows_and_defaults(ops, dev):
    c = make(dev, 6 * 50, 256, 160, 8, 3, "bf16")
    ids = torch.tensor([2, 0, -1], dtype=torch.int32, device=dev)
    x3 = c["x"].view(3, 100, 256)
    y = ops.QMatMul(c["qs"], c["scales"]).forward_adapters(x3, c["a"], c["b"], ids)
    assert y.shape == (3, 100, 160)
    check(y, reference(c, ids, None, None, use_bias=False, use_alpha=False), "equal segments")
    wide = torch.randn(300, 800, device=dev).to(torch.bfloat16)
    c["x"] = wide[:, 64:320]
    y = ops.q8_0_linear_adapters(c["x"], c["qs"], c["scales"], c["a"], c["b"], ids, alphas=c["alphas"])
    check(y, reference(c, ids, None, None, use_bias=False), "strided rows")
    # b that is not 16-byte aligned
    store = torch.randn(3 * 160 * 8 + 1, device=dev).to(torch.bfloat16)
    c["b"] = store[1:].view(3, 160, 8)
    for rows in (6, 300):
        d = dict(c, x=c["x"][:rows])
        y = ops.q8_0_linear_adapters(d["x"], c["qs"], c["scales"], c["a"], c["b"], ids)
        check(y, reference(d, ids, None, None, use_bias=False, use_alpha=False), "unaligned b")


def test_empty(ops, dev):
    c = make(dev, 4, 64, 32, 4, 2, "bf16")
    ids = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    y = ops.q8_0_linear_adapters(c["x"][:0], c["qs"], c["scales"], c["a"], c["b"], ids)
    torch.cuda.synchronize()
    assert y.shape == (0, 32)


@pytest.mark.parametrize("m", [12, 700])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_same_bits_every_time_on_any_stream_and_in_graphs(ops, dev, m, dt):
    one, two = (make(dev, m, 512, 384, 16, 3, dt, seed=s) for s in (1, 2))
    ids = torch.tensor([2, 0, -1, 1], dtype=torch.int32, device=dev)
    offs = torch.tensor(cuts_of(m, 4), dtype=torch.int64, device=dev)
    call = lambda c: ops.q8_0_linear_adapters(c["x"], c["qs"], c["scales"], c["a"], c["b"], ids, alphas=c["alphas"],  # noqa: E731
                                              seg_offsets=offs, bias=c["bias"], out_dtype=DT[dt])
    eager = [call(one), call(two)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call(two)
    again = call(one)
    torch.cuda.synchronize()
    assert torch.equal(other, eager[1]) and torch.equal(again, eager[0])
    graphs, outs = [], []
    for c in (one, two):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(call(c))
        graphs.append(gr)
    for _ in range(4):
        for o in outs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        for gr in graphs:
            gr.replay()
        call(one)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager[0]) and torch.equal(outs[1], eager[1])
    ids.copy_(torch.tensor([0, 1, 2, -1]))      # a replay reads the ids as they are then
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], call(one))
