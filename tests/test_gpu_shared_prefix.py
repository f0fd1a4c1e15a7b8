"""lux3d_sdpa_shared_prefix against the formula in 64 bits.

Tolerances, with u = 2^-24, e = eps / 2 of the type (half a rounding step), A = sum p |v| / sum p (the magnitude that an
output sums) and N keys:
- a score sums D products in f32: off by at most (D + 4) u scale sum |q| |k|, and a probability by that much relatively,
  with 4 u of exp2 on top; numerator and denominator each carry it: 2 A (delta + 4 u).
- 2-byte types round each probability by e relatively (the denominator sums the rounded ones): 2 A e. An f16 probability
  below 2^-14 is off by 2^-25 at most, beside a sum of at least 1: N 2^-25 max |v| more.
- sums over N keys in f32, 16 at a time: at most (N / 8 + 64) u A.
- the store: e |out|.
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


def reference(q, pk, pv, k, v, scale, lens, causal):
    """(out, bound without the store) in f64; keys that a query does not see are never touched."""
    b, h, n, d = q.shape
    g = h // pk.shape[0]
    dt = q.dtype
    e = torch.finfo(dt).eps / 2 if dt != torch.float32 else 0.0
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for bi in range(b):
        length = min(max(int(lens[bi]), 0), k.shape[2]) if lens is not None else k.shape[2]
        for hi in range(h):
            keys = torch.cat([pk[hi // g], k[bi, hi // g, :length]]).double()
            vals = torch.cat([pv[hi // g], v[bi, hi // g, :length]]).double()
            if keys.shape[0] == 0:
                continue
            qq = q[bi, hi].double()
            s = torch.mm(qq, keys.t().contiguous()) * scale
            if causal:
                own = length - n + torch.arange(n, device=q.device) + 1
                hidden = torch.arange(length, device=q.device)[None, :] >= own[:, None]
                s[:, pk.shape[1]:].masked_fill_(hidden, float("-inf"))
            mag = torch.mm(qq.abs(), keys.abs().t().contiguous()) * scale
            mag = mag.masked_fill(torch.isinf(s), 0.0).amax(-1, keepdim=True)
            top = s.amax(-1, keepdim=True)
            none = torch.isinf(top)
            p = torch.exp(s - torch.where(none, torch.zeros_like(top), top))
            total = p.sum(-1, keepdim=True)
            total = torch.where(none, torch.ones_like(total), total)
            out[bi, hi] = torch.mm(p, vals) / total
            a = torch.mm(p, vals.abs()) / total
            nk = keys.shape[0]
            bound[bi, hi] = a * (2 * ((d + 4) * U * mag + 4 * U) + 2 * e + (nk / 8 + 64) * U)
            if dt == torch.float16:
                bound[bi, hi] += nk * 2.0 ** -25 * vals.abs().max()
    return out, bound


def check(got, ref, what):
    want, bound = ref
    fi = torch.finfo(got.dtype)
    bound = bound + fi.eps / 2 * want.abs() + fi.smallest_normal * fi.eps
    assert torch.isfinite(got).all(), what
    over = (got.double() - want).abs() - bound
    assert float(over.max()) <= 0, f"{what}: worst error {float((got.double() - want).abs().max()):.3g}, {int((over > 0).sum())} values past the bound"


def make(dev, b, h, hkv, n, p, ls, d, dt, layout="heads", seed=0, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed + 17 * n + p)
    rnd = lambda *shape: (torch.randn(shape, generator=g, device=dev) * std).to(DT[dt])  # noqa: E731
    if layout == "heads":  # each head's tokens together
        return rnd(b, h, n, d), rnd(hkv, p, d), rnd(hkv, p, d), rnd(b, hkv, ls, d), rnd(b, hkv, ls, d)
    if layout == "tokens":  # each token's heads together
        kv = rnd(b, ls, 2, hkv, d)
        pre = rnd(p, 2, hkv, d)
        return (rnd(b, n, h, d).transpose(1, 2), pre[:, 0].transpose(0, 1), pre[:, 1].transpose(0, 1),
                kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2))
    assert layout == "odd"  # rows of d + 3: no row but the first is 16-byte aligned
    return (rnd(b, h, n, d + 3)[..., 1:d + 1], rnd(hkv, p, d + 3)[..., 2:d + 2], rnd(hkv, p, d + 3)[..., :d],
            rnd(b, hkv, ls, d + 3)[..., 3:], rnd(b, hkv, ls, d + 3)[..., 1:d + 1])


def run(ops, dev, b, h, hkv, n, p, ls, d, dt, causal=False, lens=None, layout="heads", std=1.0, seed=0):
    t = make(dev, b, h, hkv, n, p, ls, d, dt, layout, seed, std)
    ln = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    scale = 1.0 / math.sqrt(d)
    print(f"[case] B {b} H {h}/{hkv} Lq {n} P {p} Ls {ls} D {d} {dt} causal {causal} lens {lens} {layout}", flush=True)
    out = ops.sdpa_shared_prefix(*t, scale, lens=ln, causal=causal)
    torch.cuda.synchronize()
    assert out.shape == t[0].shape and out.dtype == t[0].dtype
    check(out, reference(*t, scale, lens, causal), "out")
    return t, ln, out


# one token to a few, one sequence to many: the rows of all sequences share the prefix's tiles
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("b,h,hkv,n,d", [(1, 4, 4, 1, 64), (5, 4, 4, 1, 64), (9, 8, 2, 1, 128), (70, 2, 2, 1, 128),
                                         (3, 6, 2, 5, 64), (2, 8, 1, 8, 128), (130, 1, 1, 1, 64), (4, 2, 1, 33, 128)])
@pytest.mark.parametrize("p,ls", [(1, 1), (63, 65), (64, 64), (300, 130), (1029, 40)])
def test_few_queries(ops, dev, b, h, hkv, n, d, p, ls, dt):
    ls = max(ls, n)
    lens = [n + (7 * i + 3) % (ls - n + 1) for i in range(b)]
    run(ops, dev, b, h, hkv, n, p, ls, d, dt, causal=True, lens=lens)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b,h,hkv,n,p,ls,d", [(2, 4, 4, 128, 128, 128, 64), (2, 4, 2, 129, 65, 200, 128),
                                              (3, 2, 2, 257, 700, 257, 64), (1, 6, 3, 333, 401, 707, 128),
                                              (2, 3, 1, 100, 1, 100, 64), (1, 2, 2, 64, 2000, 64, 128),
                                              (1, 1, 1, 65, 5000, 300, 64)])
def test_many_queries(ops, dev, b, h, hkv, n, p, ls, d, causal, dt):
    lens = [ls - (11 * i) % (ls - n + 1) for i in range(b)]
    run(ops, dev, b, h, hkv, n, p, ls, d, dt, causal=causal, lens=lens)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 3, 150])
def test_no_prefix_and_no_own_keys(ops, dev, n, dt):
    run(ops, dev, 3, 4, 2, n, 0, 200, 64, dt, causal=True, lens=[200, 151, 170])
    run(ops, dev, 3, 4, 2, n, 77, 0, 64, dt)
    run(ops, dev, 3, 4, 2, n, 77, 200, 64, dt, causal=True, lens=[0, 200, 0])
    _, _, out = run(ops, dev, 3, 4, 2, n, 0, 0, 64, dt)
    assert not out.any()
    _, _, out = run(ops, dev, 3, 4, 2, n, 0, 200, 64, dt, lens=[0, 5, 0])
    assert not out[0].any() and not out[2].any() and out[1].any()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
def test_lengths_shorter_than_the_queries(ops, dev, d, dt):
    """Causal with fewer own keys than queries: the first queries see none of them; without a prefix they are zero."""
    for n in (4, 40, 200):
        run(ops, dev, 3, 2, 2, n, 70, 200, d, dt, causal=True, lens=[n - 1, 1, n // 2])
        _, _, out = run(ops, dev, 3, 2, 2, n, 0, 200, d, dt, causal=True, lens=[n - 1, 1, n // 2])
        assert not out[1, :, :n - 1].any() and out[1, :, n - 1].any()


@pytest.mark.parametrize("lens", [[-5, 400, 50], [64, 128, 65]])
def test_lengths_are_clamped(ops, dev, lens):
    run(ops, dev, 3, 4, 4, 1, 30, 130, 64, "bf16", lens=lens)
    run(ops, dev, 3, 4, 4, 140, 30, 130, 64, "bf16", lens=lens)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("layout", ["tokens", "odd"])
@pytest.mark.parametrize("n", [1, 200])
def test_layouts(ops, dev, layout, n, dt):
    run(ops, dev, 3, 4, 2, n, 130, 260, 128, dt, causal=True, lens=[260, 201, 230], layout=layout)


@pytest.mark.parametrize("d", [1, 33, 80, 256, 512])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_head_dims(ops, dev, d, dt):
    run(ops, dev, 2, 4, 2, 3, 90, 70, d, dt, causal=True, lens=[70, 9])


@pytest.mark.parametrize("std", [1e-3, 8.0])
def test_flat_and_peaked_scores(ops, dev, std):
    run(ops, dev, 3, 4, 2, 1, 700, 200, 64, "bf16", lens=[200, 3, 90], std=std)
    run(ops, dev, 2, 2, 2, 150, 700, 200, 128, "bf16", causal=True, std=std)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n,causal", [(1, True), (5, True), (200, False), (200, True)])
def test_what_lies_past_a_sequence_is_not_read(ops, dev, n, causal, dt):
    lens = [260, 200, 233]
    t, ln, clean = run(ops, dev, 3, 4, 2, n, 130, 300, 64, dt, causal=causal, lens=lens)
    for bad in (float("nan"), float("inf"), torch.finfo(DT[dt]).min):
        for x in t[3:]:
            for b, m in enumerate(lens):
                x[b, :, m:] = bad
        out = ops.sdpa_shared_prefix(*t, 0.125, lens=ln, causal=causal)
        assert torch.equal(out, clean)


def test_caches_past_32_bit_offsets(ops, dev):
    """Sequences and key heads more than 2^31 elements apart."""
    b, hkv, ls, d = 2, 2, 100, 64
    far = (1 << 31) + 4096
    store = torch.empty(far + (1 << 21), dtype=torch.bfloat16, device=dev)
    k = torch.as_strided(store, (b, hkv, ls, d), (far, 8192, d, 1))
    g = torch.Generator(device=dev).manual_seed(3)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev).to(torch.bfloat16)  # noqa: E731
    k.copy_(rnd(b, hkv, ls, d))
    pk = torch.as_strided(store, (hkv, 50, d), (far - 64 * 4096, d, 1), 1 << 20)
    pk.copy_(rnd(hkv, 50, d))
    for n in (1, 130):
        q = rnd(b, 4, n, d)
        out = ops.sdpa_shared_prefix(q, pk, pk, k, k, 0.125)
        check(out, reference(q, pk, pk, k, k, 0.125, None, False), f"far, Lq {n}")


def test_repeated_prefix_rows(ops, dev):
    """A prefix whose rows are one row (stride 0), and rows that overlap."""
    g = torch.Generator(device=dev).manual_seed(5)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev).to(torch.bfloat16)  # noqa: E731
    q, k, v = rnd(2, 2, 3, 64), rnd(2, 2, 70, 64), rnd(2, 2, 70, 64)
    for pk in (rnd(2, 1, 64).expand(2, 90, 64), torch.as_strided(rnd(9000), (2, 90, 64), (4096, 8, 1)), rnd(2, 1, 64)):
        out = ops.sdpa_shared_prefix(q, pk, pk, k, v, 0.125)
        check(out, reference(q, pk, pk, k, v, 0.125, None, False), "repeated rows")


@pytest.mark.parametrize("n", [1, 150])
def test_out_view_and_neighbours(ops, dev, n):
    """`out` as the [B, L, H, D] buffer that the caller uses next; what lies around it stays."""
    t = make(dev, 2, 4, 2, n, 100, 200, 64, "bf16")
    buf = torch.full((2, n + 2, 4, 70), 7.0, dtype=torch.bfloat16, device=dev)
    out = buf[:, 1:n + 1, :, :64].transpose(1, 2)
    got = ops.sdpa_shared_prefix(*t, 0.125, causal=True, out=out)
    check(got, reference(*t, 0.125, None, True), "out view")
    assert (buf[:, 0] == 7).all() and (buf[:, -1] == 7).all() and (buf[..., 64:] == 7).all()


@pytest.mark.parametrize("shape", [(0, 4, 2, 3, 10, 10, 64), (2, 0, 2, 3, 10, 10, 64), (2, 4, 2, 0, 10, 10, 64)])
def test_empty(ops, dev, shape):
    t = make(dev, *shape, "bf16")
    out = ops.sdpa_shared_prefix(*t, 0.125)
    torch.cuda.synchronize()
    assert out.shape == t[0].shape


@pytest.mark.parametrize("n", [1, 150])
def test_same_bits_every_time_on_any_stream_and_in_graphs(ops, dev, n):
    a = make(dev, 6, 8, 2, n, 900, 300, 128, "bf16", seed=1)
    b = make(dev, 6, 8, 2, n, 900, 300, 128, "bf16", seed=2)
    lens = torch.tensor([300, 200, 250, 290, 160, 170], dtype=torch.int32, device=dev)
    call = lambda t, out=None: ops.sdpa_shared_prefix(*t, 0.1, lens=lens, causal=True, out=out)  # noqa: E731
    eager = [call(a), call(b)]
    assert torch.equal(call(a), eager[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call(b)
    again = call(a)     # both streams at once
    torch.cuda.synchronize()
    assert torch.equal(other, eager[1]) and torch.equal(again, eager[0])
    outs = [torch.empty_like(eager[0]) for _ in range(2)]
    graphs = []
    for t, o in zip((a, b), outs):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            call(t, o)
        graphs.append(gr)
    for _ in range(4):
        for o in outs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        for gr in graphs:
            gr.replay()
        call(a)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager[0]) and torch.equal(outs[1], eager[1])
    lens.sub_(7)        # a replay reads the lengths as they are then
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], call(a))
