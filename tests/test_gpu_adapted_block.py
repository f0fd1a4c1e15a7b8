"""The operators of one served block together: norms around a residual sum, the fused projection with each request's adapter,
new keys into the caches, attention behind the shared prefix, the output projection with its adapters, and the norms again.

Each operator's result is held to its formula in 64 bits on the inputs that it got, by the bounds derived in the operators'
own tests; the block as a whole to itself: on another stream and in replayed graphs."""
import math

import pytest

torch = pytest.importorskip("torch")

import test_gpu_adapters as adapters  # noqa: E402
import test_gpu_block_norm as norms  # noqa: E402
import test_gpu_shared_prefix as prefix  # noqa: E402

pytestmark = pytest.mark.gpu

B, H, HKV, D, P, LS, RANK, NA = 3, 4, 2, 64, 130, 96, 12, 2
C = H * D
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def ops(dev):
    from lux3d_fused import ops as _ops
    return _ops


class Block:
    def __init__(self, dev, n, dt):
        g = torch.Generator(device=dev).manual_seed(n)
        rnd = lambda shape, t=DT[dt], mean=0.0: (torch.randn(shape, generator=g, device=dev) + mean).to(t)  # noqa: E731
        self.n, self.dt, rows = n, DT[dt], B * n
        self.x, self.h = rnd((rows, C)), rnd((rows, C))
        self.post, self.pre = rnd((2, C), torch.float32, 1.0), rnd((2, C), torch.float32, 1.0)
        self.proj = [adapters.make(dev, rows, C, (H + 2 * HKV) * D, RANK, NA, dt, seed=1),
                     adapters.make(dev, rows, C, C, RANK, NA, dt, seed=2)]
        self.ids = torch.tensor([1, -1, 0], dtype=torch.int32, device=dev)
        self.pk, self.pv = rnd((HKV, P, D)), rnd((HKV, P, D))
        self.lens = torch.tensor([n, n + 17, LS], dtype=torch.int32, device=dev)  # with the new tokens
        # what is behind a sequence's last key is not read
        self.cache = [torch.full((B, HKV, LS, D), float("nan"), dtype=self.dt, device=dev) for _ in range(2)]
        for c in self.cache:
            for i, length in enumerate(self.lens.tolist()):
                c[i, :, :length - n] = rnd((HKV, length - n, D))
        self.seq = torch.arange(B, device=dev)[:, None].expand(B, n)

    def linear(self, ops, i, x):
        c = self.proj[i]
        return ops.q8_0_linear_adapters(x, c["qs"], c["scales"], c["a"], c["b"], self.ids, alphas=c["alphas"],
                                        bias=c["bias"], out_dtype=self.dt)

    def run(self, ops):
        """x1, y1, the projections, the attention, h1, x2, y2"""
        x1, y1 = ops.norm_gated_residual_norm(self.x, self.h, post_weight=self.post[0], pre_weight=self.pre[0])
        qkv = self.linear(ops, 0, y1)
        heads = qkv.view(B, self.n, H + 2 * HKV, D)
        at = (self.lens.long() - self.n)[:, None] + torch.arange(self.n, device=self.x.device)
        for c, new in zip(self.cache, heads[:, :, H:].split(HKV, 2)):
            c.transpose(1, 2).index_put_((self.seq, at), new)
        out = torch.empty((B, self.n, H, D), dtype=self.dt, device=self.x.device)
        ops.sdpa_shared_prefix(heads[:, :, :H].transpose(1, 2), self.pk, self.pv, *self.cache, 1.0 / math.sqrt(D),
                               lens=self.lens, causal=True, out=out.transpose(1, 2))
        h1 = self.linear(ops, 1, out.view(B * self.n, C))
        x2, y2 = ops.norm_gated_residual_norm(x1, h1, post_weight=self.post[1], pre_weight=self.pre[1])
        return x1, y1, qkv, out, h1, x2, y2


def check_norm(x, h, post, pre, xo, y):
    n, err = norms.affine(*norms.norm64(h, "rms", 1e-6), post, None)
    want = x.double() + n
    norms.check(xo, want, err + 2 * norms.U * want.abs(), "x_out")
    norms.check(y, *norms.affine(*norms.norm64(xo, "rms", 1e-6), pre, None), "y")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 7, 40])
def test_each_operator_in_the_block(ops, dev, n, dt):
    print(f"[case] block n {n} {dt}", flush=True)
    b = Block(dev, n, dt)
    x1, y1, qkv, out, h1, x2, y2 = b.run(ops)
    torch.cuda.synchronize()
    check_norm(b.x, b.h, b.post[0], b.pre[0], x1, y1)
    adapters.check(qkv, adapters.reference({**b.proj[0], "x": y1}, b.ids, None, None), "projection")
    q = qkv.view(B, n, H + 2 * HKV, D)[:, :, :H].transpose(1, 2)
    prefix.check(out.transpose(1, 2), prefix.reference(q, b.pk, b.pv, *b.cache, 1.0 / math.sqrt(D), b.lens.tolist(), True),
                 "attention")
    adapters.check(h1, adapters.reference({**b.proj[1], "x": out.view(B * n, C)}, b.ids, None, None), "output projection")
    check_norm(x1, h1, b.post[1], b.pre[1], x2, y2)


@pytest.mark.parametrize("n", [1, 40])
def test_block_on_another_stream_and_in_graphs(ops, dev, n):
    print(f"[case] block in graphs n {n}", flush=True)
    one, two = Block(dev, n, "bf16"), Block(dev, n, "bf16")
    two.x.mul_(-0.5)
    eager = [one.run(ops), two.run(ops)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = two.run(ops)
    again = one.run(ops)
    torch.cuda.synchronize()
    for a, b in zip(again + other, eager[0] + eager[1]):
        assert torch.equal(a, b)
    graphs, outs = [], []
    for b in (one, two):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(b.run(ops))
        graphs.append(gr)
    for _ in range(4):
        for o in outs[0] + outs[1]:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        for gr in graphs:
            gr.replay()
        one.run(ops)
        torch.cuda.synchronize()
        for got, want in zip(outs[0] + outs[1], eager[0] + eager[1]):
            assert torch.equal(got, want)
