"""lux3d_norm_gated_residual_norm against the formula in 64 bits.

Tolerances. The kernel sums a row in f32: at most 40 rounded additions on any path (32 of a lane's own values, 6 of the
wavefront's tree, 2 of the workgroup's), 64 with the few operations that follow, so a mean is off by at most 64 u mean|v|
and a normalised value n by 64 u (|n| + rstd mean|v|), u = 2^-24; the generic kernel's lanes sum width / 256 values. The
products and sums that follow add 8 u of their magnitudes, and the store half a step of the type (eps / 2). y is held to
the norm of the x_out that the call itself returned, as the operator defines it.
"""
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


def norm64(v, kind, eps):
    """The normalised rows and the bound of their f32 error (without the store)."""
    v = v.double()
    steps = 64 + v.shape[-1] // 256
    c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    rstd = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    n = c * rstd
    return n, steps * U * (n.abs() + rstd * v.abs().mean(-1, keepdim=True))


def affine(n, err, w, b):
    w = torch.ones((), dtype=torch.float64, device=n.device) if w is None else w.double()
    b = torch.zeros((), dtype=torch.float64, device=n.device) if b is None else b.double()
    return n * w + b, err * w.abs() + 8 * U * ((n * w).abs() + b.abs())


def segment_of_rows(offs, rows):
    if offs is None:
        return torch.zeros(rows, dtype=torch.long)
    o = offs.cpu()
    # the last segment that starts at or before the row; rows past the last offset are the last segment's
    seg = torch.searchsorted(o, torch.arange(rows), right=True) - 1
    return seg.clamp(0, o.numel() - 2)


def check(got, want, err, what):
    t = got.dtype
    bound = err + torch.finfo(t).eps / 2 * want.abs() * (1 + 2 * U) + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    bad = (got.double() - want).abs() - bound
    assert torch.isfinite(got).all(), what
    assert float(bad.max()) <= 0, f"{what}: off by {float((got.double() - want).abs().max()):.3g}, {int((bad > 0).sum())} values past the bound"


def run_case(ops, dev, rows, width, dt, kind, *, offs=None, parts=("post", "gamma", "gate", "pre", "mod"), base=False,
             bias=True, in_place=False, param=torch.float32, x=None, h=None, seed=0, eps=1e-6):
    g = torch.Generator(device=dev).manual_seed(seed + rows * 31 + width)
    rnd = lambda shape, mean=0.0, std=1.0, t=param: (torch.randn(shape, generator=g, device=dev) * std + mean).to(t)  # noqa: E731
    x = rnd((rows, width), t=DT[dt]) if x is None else x
    h = rnd((rows, width), 0.5, 3.0, DT[dt]) if h is None else h
    nseg = 1 if offs is None else offs.numel() - 1
    kw = {}
    if "post" in parts:
        kw.update(post_weight=rnd(width, 1.0, 0.1))
        if bias:
            kw.update(post_bias=rnd(width, 0.0, 0.2))
    if "gamma" in parts:
        kw.update(ls_gamma=rnd(width, 0.4, 0.1))
    if "pre" in parts:
        kw.update(pre_weight=rnd(width, 1.0, 0.1))
        if bias:
            kw.update(pre_bias=rnd(width, 0.0, 0.2))
    vec = rnd((nseg, 6 * width), 0.0, 0.3).chunk(6, -1)
    bases = rnd((6 * width,), 0.0, 0.3).chunk(6, -1)
    if "gate" in parts:
        kw.update(gate=vec[2], gate_base=bases[2] if base else None)
    if "mod" in parts:
        kw.update(shift=vec[3], scale=vec[4], shift_base=bases[3] if base else None, scale_base=bases[4] if base else None)
    x0, h0 = x.clone(), h.clone()
    print(f"[case] rows {rows} width {width} {dt} {kind} parts {parts} seg {nseg}", flush=True)
    xo, y = ops.norm_gated_residual_norm(x, h, norm=kind, eps=eps, seg_offsets=offs, x_out=x if in_place else None, **kw)
    torch.cuda.synchronize()
    assert torch.equal(h, h0) and (in_place or torch.equal(x, x0))
    if rows == 0:
        return
    seg = segment_of_rows(offs, rows).to(dev)
    piece = lambda name: (kw[name].double() + (kw[name + "_base"].double() if kw.get(name + "_base") is not None else 0.0))[seg]  # noqa: E731
    n, err = affine(*norm64(h0, kind, eps), kw.get("post_weight"), kw.get("post_bias"))
    factor = kw["ls_gamma"].double() if "gamma" in parts else torch.ones((), dtype=torch.float64, device=dev)
    if "gate" in parts:
        factor = factor * piece("gate")
        err = err + 2 * U * n.abs()    # gate + base is rounded
        if base:
            err = err + U * (kw["gate"].double().abs()[seg] + kw["gate_base"].double().abs()) * n.abs() / factor.abs().clamp_min(1e-30) * (
                kw["ls_gamma"].double().abs() if "gamma" in parts else 1.0)
    want = x0.double() + n * factor
    check(xo, want, err * factor.abs() + 2 * U * want.abs(), "x_out")
    n, err = affine(*norm64(xo, kind, eps), kw.get("pre_weight"), kw.get("pre_bias"))
    if "mod" in parts:
        sc, sh = piece("scale") + 1.0, piece("shift")
        mag = 3 * U * (kw["scale"].double().abs()[seg] + 1.0 + (kw["scale_base"].double().abs() if base else 0.0))
        err = err * sc.abs() + mag * n.abs() + 4 * U * ((n * sc).abs() + sh.abs())
        # pre_bias (scale + 1) and pre_weight (scale + 1) are formed before n is known
        w, b = kw.get("pre_weight"), kw.get("pre_bias")
        n0 = norm64(xo, kind, eps)[0]
        err = err + 4 * U * sc.abs() * ((n0 * (1.0 if w is None else w.double())).abs() + (0.0 if b is None else b.double().abs()))
        err = err + 4 * U * (kw["shift"].double().abs()[seg] + (kw["shift_base"].double().abs() if base else 0.0))
        n = n * sc + sh
    check(y, n, err, "y")


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("width", [1, 2, 7, 8, 64, 100, 512, 520, 1000, 1024, 1536, 2048, 2056, 4096, 8192, 8200])
def test_widths(ops, dev, width, dt, kind):
    offs = torch.tensor([0, 2, 2, 5], device=dev)
    # one value a row: LayerNorm's variance is 0 and 1 / sqrt(eps) amplifies nothing but zeros
    run_case(ops, dev, 5, width, dt, kind, offs=offs)


@pytest.mark.parametrize("rows", [1, 2, 63, 2047, 2048, 2049, 4100])
@pytest.mark.parametrize("dt,width,kind", [("bf16", 1536, "rms"), ("f32", 1024, "layer"), ("f16", 2048, "layer"),
                                           ("bf16", 1000, "layer"), ("f32", 520, "rms")])
def test_rows_in_ragged_segments(ops, dev, rows, dt, width, kind):
    cut = lambda f: int(rows * f)  # noqa: E731
    offs = torch.tensor([0, cut(0.1), cut(0.1), cut(0.35), cut(0.9), rows], device=dev)
    run_case(ops, dev, rows, width, dt, kind, offs=offs, base=True)


@pytest.mark.parametrize("parts", [(), ("post",), ("gamma",), ("gate",), ("pre",), ("mod",), ("post", "pre"),
                                   ("gamma", "gate", "mod")])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_absent_parameters(ops, dev, parts, kind):
    run_case(ops, dev, 300, 1024, "bf16", kind, parts=parts)
    run_case(ops, dev, 2500, 1024, "bf16", kind, parts=parts, bias=False)
    run_case(ops, dev, 9, 33, "f32", kind, parts=parts)


@pytest.mark.parametrize("param", [torch.bfloat16, torch.float16])
def test_parameters_of_other_types(ops, dev, param):
    offs = torch.tensor([0, 700, 2300], device=dev)
    run_case(ops, dev, 2300, 1536, "bf16", "rms", offs=offs, param=param, base=True)
    run_case(ops, dev, 40, 1536, "f32", "layer", param=param)


@pytest.mark.parametrize("rows", [50, 3000])
def test_in_place_strided_and_unaligned_rows(ops, dev, rows):
    run_case(ops, dev, rows, 1024, "bf16", "layer", in_place=True)
    wide = torch.randn(rows, 3000, device=dev).to(torch.bfloat16)
    run_case(ops, dev, rows, 1024, "bf16", "rms", x=wide[:, 8:1032], h=wide[:, 1200:2224])     # aligned, strided
    run_case(ops, dev, rows, 1024, "bf16", "rms", x=wide[:, 3:1027], h=wide[:, 1201:2225])     # unaligned
    run_case(ops, dev, rows, 1000, "bf16", "layer", x=wide[:, 1:1001], h=wide[:, 1111:2111], in_place=True)


def test_dense_segments_of_a_batch(ops, dev):
    """[B, L, C] rows with [B, C] pieces and no offsets: equal segments."""
    b, n, c = 3, 700, 1024
    g = torch.Generator(device=dev).manual_seed(4)
    x, h = (torch.randn((b, n, c), generator=g, device=dev).to(torch.bfloat16) for _ in range(2))
    p = torch.randn((b, 6 * c), generator=g, device=dev).chunk(6, -1)
    offs = torch.arange(b + 1, device=dev) * n
    a = ops.norm_gated_residual_norm(x, h, gate=p[2], shift=p[3], scale=p[4], norm="layer")
    c2 = ops.norm_gated_residual_norm(x, h, gate=p[2], shift=p[3], scale=p[4], norm="layer", seg_offsets=offs)
    assert torch.equal(a[0], c2[0]) and torch.equal(a[1], c2[1])


def test_rows_before_and_past_the_offsets(ops, dev):
    run_case(ops, dev, 2600, 1024, "bf16", "rms", offs=torch.tensor([5, 1000, 2000], device=dev))
    run_case(ops, dev, 60, 1024, "bf16", "rms", offs=torch.tensor([5, 10, 20], device=dev))


def test_last_block_without_next_norm(ops, dev):
    g = torch.Generator(device=dev).manual_seed(5)
    for rows, c in ((40, 1024), (3000, 1024), (30, 77)):
        x, h = (torch.randn((rows, c), generator=g, device=dev).to(torch.bfloat16) for _ in range(2))
        full = ops.norm_gated_residual_norm(x, h, norm="rms")
        xo, y = ops.norm_gated_residual_norm(x, h, norm="rms", next_norm=False)
        assert y is None and torch.equal(xo, full[0])


@pytest.mark.parametrize("rows", [20, 3000])
def test_a_row_that_is_not_finite_stays_alone(ops, dev, rows):
    g = torch.Generator(device=dev).manual_seed(6)
    x, h = (torch.randn((rows, 1024), generator=g, device=dev).to(torch.bfloat16) for _ in range(2))
    clean = ops.norm_gated_residual_norm(x, h, norm="layer")
    h[7, 3] = float("inf")
    x[11, 5] = float("nan")
    xo, y = ops.norm_gated_residual_norm(x, h, norm="layer")
    keep = [r for r in range(rows) if r not in (7, 11)]
    assert torch.equal(xo[keep], clean[0][keep]) and torch.equal(y[keep], clean[1][keep])
    assert torch.isnan(xo[7]).any() and torch.isnan(y[7]).all() and torch.isnan(y[11]).all()
    assert torch.isnan(xo[11]).sum() == 1


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_long_jobs(ops, dev, kind):
    """Enough rows for three workgroups a CU, in segments that end inside a workgroup's run."""
    offs = torch.tensor([0, 7, 16001, 16002, 33001], device=dev)
    run_case(ops, dev, 33001, 512, "bf16", kind, offs=offs, base=True)


def test_empty_rows(ops, dev):
    run_case(ops, dev, 0, 1024, "bf16", "rms")


@pytest.mark.parametrize("rows", [64, 5000])
def test_graph_replays_and_another_stream(ops, dev, rows):
    from lux3d_fused import _lib
    g = torch.Generator(device=dev).manual_seed(7)
    x, h = (torch.randn((rows, 1536), generator=g, device=dev).to(torch.bfloat16) for _ in range(2))
    p = torch.randn((2, 6 * 1536), generator=g, device=dev).chunk(6, -1)
    offs = torch.tensor([0, rows // 3, rows], device=dev)
    xo, y = torch.empty_like(x), torch.empty_like(x)

    def run():
        s = torch.cuda.current_stream().cuda_stream
        d = ops.desc
        _lib.call("lux3d_norm_gated_residual_norm", d(x), d(h), None, None, None, d(offs), d(p[2]), None, None, None,
                  d(p[3]), None, d(p[4]), None, 1, 1e-6, d(xo), d(y), s)
    run()
    torch.cuda.synchronize()
    eager = xo.clone(), y.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    xo.zero_(), y.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    assert torch.equal(xo, eager[0]) and torch.equal(y, eager[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _ in range(4):
        xo.fill_(float("nan")), y.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(xo, eager[0]) and torch.equal(y, eager[1])
