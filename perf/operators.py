"""Operators of a transformer block that serves several requests at once, as measured cases.

A case is a dict of plain values; "kind" names the operator:
  prefix    softmax attention of a batch whose sequences share one long prefix of keys: the prefix's keys and values are
            stored once for all, each sequence adds keys and values of its own
  adapters  Q8_0 linear with a low-rank adapter of each request's own beside the shared weight
  norm      norm after a block, its gate and residual scale, the residual sum and the norm before the next block
`own` chooses between the operators in elementary torch operations (32-bit, rounded once) and the framework's entry
points (`lux3d_fused.ops`). `exact` is the definition in 64 bits.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_OPS = []


def _ops():
    if not _OPS:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "candle-3d_amd"))
        from lux3d_fused import ops
        _OPS.append(ops)
    return _OPS[0]


def listed():
    return [
        # eight samples of one image, one new token each, on the image encoder's 1029 tokens: the smallest call of a step
        {"name": "prefix_token_short", "kind": "prefix", "batch": 8, "heads": 16, "kv_heads": 16, "dim": 64,
         "queries": 1, "prefix": 1029, "own": 64, "causal": True, "dtype": "bf16"},
        # 64 sequences decoding behind a long shared context, four query heads to a key head
        {"name": "prefix_token_long", "kind": "prefix", "batch": 64, "heads": 32, "kv_heads": 8, "dim": 128,
         "queries": 1, "prefix": 16384, "own": 1000, "causal": True, "dtype": "bf16"},
        # VGGT with eight frames kept: four new frames of 1374 tokens attend to the kept ones and each to itself
        {"name": "prefix_frames", "kind": "prefix", "batch": 4, "heads": 16, "kv_heads": 16, "dim": 64,
         "queries": 1374, "prefix": 10992, "own": 1374, "causal": False, "dtype": "bf16"},
        # three prompts of ragged length fed in chunks behind a shared one, odd sizes
        {"name": "prefix_chunk", "kind": "prefix", "batch": 3, "heads": 12, "kv_heads": 4, "dim": 128,
         "queries": 333, "prefix": 4001, "own": 707, "causal": True, "dtype": "f16"},
        # DINOv3 tokens of two views behind those of a reference view, in the encoder's f32
        {"name": "prefix_dinov3", "kind": "prefix", "batch": 2, "heads": 16, "kv_heads": 16, "dim": 64,
         "queries": 1029, "prefix": 1029, "own": 1029, "causal": False, "dtype": "f32"},
        # TRELLIS.2 AdaLN linear: one modulation vector per request, each request with an adapter of its own
        {"name": "adapters_adaln", "kind": "adapters", "rows": 12, "segments": 12, "adapters": 12, "k": 1536, "n": 9216,
         "rank": 16, "dtype": "bf16"},
        # TripoSG feed-forward up-projection over four requests of ragged length, one of them without an adapter
        {"name": "adapters_triposg", "kind": "adapters", "rows": 4096, "segments": 4, "adapters": 3, "k": 2048,
         "n": 8192, "rank": 64, "dtype": "bf16"},
        # DINOv3 MLP down-projection of three images in f32, short requests
        {"name": "adapters_dinov3", "kind": "adapters", "rows": 3087, "segments": 3, "adapters": 2, "k": 4096,
         "n": 1024, "rank": 32, "dtype": "f32"},
        # TRELLIS.2 SLAT output projection over many small requests, an odd rank
        {"name": "adapters_slat", "kind": "adapters", "rows": 9001, "segments": 24, "adapters": 16, "k": 1536,
         "n": 1536, "rank": 12, "dtype": "bf16"},
        # DINOv3 ViT-L block in f32: LayerNorm on both sides, LayerScale, no modulation
        {"name": "norm_dinov3", "kind": "norm", "rows": 1029, "width": 1024, "segments": 1, "norm": "layer",
         "modulated": False, "dtype": "f32"},
        # TRELLIS.2 SLAT block on a ragged batch, RMS norms, gate and modulation per request
        {"name": "norm_slat", "kind": "norm", "rows": 64000, "width": 1536, "segments": 2, "norm": "rms",
         "modulated": True, "dtype": "bf16"},
        # TripoSG block on both halves of the guidance pair
        {"name": "norm_triposg", "kind": "norm", "rows": 4098, "width": 2048, "segments": 2, "norm": "layer",
         "modulated": True, "dtype": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(["prefix", "prefix", "adapters", "adapters", "norm"])
    if kind == "prefix":
        heads, kv_heads, dim = rng.choice([(16, 16, 64), (16, 4, 64), (12, 12, 128), (12, 4, 128), (32, 8, 128), (8, 1, 64)])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        if rng.random() < 0.5:  # decoding: one token, or a few drafted ones
            queries, batch = rng.choice([1, 1, 1, rng.randint(2, 8)]), _log(rng, 1, 64)
            prefix, mine = _log(rng, 64, 24000), _log(rng, queries, 1500)
            return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "queries": queries,
                    "prefix": prefix, "own": max(queries, mine), "causal": True, "dtype": dtype}
        queries, batch = _log(rng, 9, 1400), rng.randint(1, 6)
        return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "queries": queries,
                "prefix": _log(rng, 64, 11000), "own": queries + rng.choice([0, rng.randint(1, 600)]),
                "causal": rng.random() < 0.5, "dtype": dtype}
    if kind == "adapters":
        k, n = rng.choice([(1024, 4096), (4096, 1024), (2048, 8192), (8192, 2048), (1536, 9216), (1536, 1536)])
        rows = rng.randint(1, 40) if rng.random() < 0.35 else _log(rng, 41, 9000)
        segments = rng.randint(1, min(rows, 32))
        return {"kind": kind, "rows": rows, "segments": segments, "adapters": rng.randint(1, min(16, segments)), "k": k,
                "n": n, "rank": rng.choice([4, 8, 16, 24, 32, 64, rng.randint(1, 64)]),
                "dtype": rng.choice(["bf16", "bf16", "f32"])}
    rows = _log(rng, 1, 60000)
    return {"kind": kind, "rows": rows, "width": rng.choice([1024, 1536, 2048, 1000, rng.randint(65, 2050)]),
            "segments": rng.randint(1, min(rows, 6)), "norm": rng.choice(["layer", "rms"]),
            "modulated": rng.random() < 0.6, "dtype": rng.choice(["bf16", "f16", "f32"])}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50, 8 * w["flops"] / 50 if case["dtype"] == "f32" else 0)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= most:
            return case


# ---- inputs -------------------------------------------------------------------

def _lens(case):
    """Own keys of each sequence: from the queries' own (the longest first) up to all that the buffers hold."""
    lo, span = min(case["queries"], case["own"]), case["own"] - min(case["queries"], case["own"])
    return [case["own"] - span * (b * 37 % 64) // 64 if case["causal"] else case["own"] for b in range(case["batch"])]


def _offsets(rows, segments):
    """Ragged cuts of `rows` into `segments`, every segment with a row at least."""
    cuts = [round(rows * (s / segments) ** 1.3) for s in range(segments + 1)]
    for s in range(1, segments + 1):
        cuts[s] = max(cuts[s], cuts[s - 1] + 1)
    cuts[segments] = rows
    for s in range(segments - 1, 0, -1):
        cuts[s] = min(cuts[s], cuts[s + 1] - 1)
    return cuts


class _Inputs:
    """Seeded tensors on the GPU, drawn in a fixed order."""

    def __init__(self, seed):
        self.dev = torch.device("cuda")
        self.g = torch.Generator(device=self.dev).manual_seed(int(seed) * 7919 + 29)
        self.host = torch.Generator().manual_seed(int(seed) * 104729 + 3)

    def normal(self, shape, dtype=torch.float32, mean=0.0, std=1.0):
        t = torch.randn(shape, generator=self.g, device=self.dev, dtype=torch.float32)
        return t.mul_(std).add_(mean).to(dtype)

    def shuffled(self, values, dtype):
        p = torch.randperm(len(values), generator=self.host)
        return torch.tensor(values, dtype=dtype)[p].to(self.dev)


def prepare(case, seed):
    i = _Inputs(seed)
    s = {"case": case}
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "prefix":
        b, h, hk, d, n = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["queries"]
        # q as the heads' view of a projection [B, L, H, D]; the caches with a key head's tokens together
        s.update(q=i.normal((b, n, h, d), dt).transpose(1, 2), prefix_k=i.normal((hk, case["prefix"], d), dt),
                 prefix_v=i.normal((hk, case["prefix"], d), dt), k=i.normal((b, hk, case["own"], d), dt),
                 v=i.normal((b, hk, case["own"], d), dt), lens=i.shuffled(_lens(case), torch.int32))
    elif case["kind"] == "adapters":
        m, k, n, r, na = case["rows"], case["k"], case["n"], case["rank"], case["adapters"]
        # the repacked weight (int8 and one scale per 32 values, an f16 value), of standard deviation about 1 / sqrt(k)
        qs = torch.randint(-127, 128, (n, k), generator=i.g, device=i.dev, dtype=torch.int32).to(torch.int8)
        d = torch.rand((n, k // 32), generator=i.g, device=i.dev) * 0.02 + 0.004
        scales = (d / math.sqrt(k)).to(torch.float16).to(torch.float32)
        # every adapter is some request's; one request has none where there are more requests than adapters
        ids = [j if j < na else -1 if j == na else j % na for j in range(case["segments"])]
        s.update(x=i.normal((m, k), dt), qs=qs, scales=scales, bias=i.normal(n, std=0.5),
                 a=i.normal((na, r, k), dt, std=1.0 / math.sqrt(k)), b=i.normal((na, n, r), dt, std=1.0 / math.sqrt(r)),
                 alpha=i.normal(na, mean=1.0, std=0.2),
                 ids=i.shuffled(ids, torch.int32),
                 offs=torch.tensor(_offsets(m, case["segments"]), dtype=torch.int64, device=i.dev))
    else:
        m, c, n = case["rows"], case["width"], case["segments"]
        s.update(x=i.normal((m, c), dt), h=i.normal((m, c), dt, std=3.0), post_w=i.normal(c, mean=1.0, std=0.1),
                 gamma=i.normal(c, mean=0.3, std=0.05), pre_w=i.normal(c, mean=1.0, std=0.1),
                 post_b=i.normal(c, std=0.1) if case["norm"] == "layer" else None,
                 pre_b=i.normal(c, std=0.1) if case["norm"] == "layer" else None,
                 offs=torch.tensor(_offsets(m, n), dtype=torch.int64, device=i.dev),
                 t_emb=i.normal((n, 6 * c), std=0.3) if case["modulated"] else None)
    return s


def _modulation(s):
    """gate, shift and scale of the block's modulation vector, as views of it."""
    if s["t_emb"] is None:
        return None, None, None
    p = s["t_emb"].chunk(6, dim=-1)
    return p[2], p[3], p[4]


# ---- one pass -----------------------------------------------------------------

def _plain_prefix(s):
    case = s["case"]
    b, h, hk, d, n = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["queries"]
    g, scale, mine = h // hk, 1.0 / math.sqrt(d), case["own"]
    q = s["q"].float().reshape(b, hk, g * n, d)
    k, v = s["k"].float(), s["v"].float()
    pk, pv = s["prefix_k"].float(), s["prefix_v"].float()
    # the prefix once for all sequences: the rows of a key head together
    rows = q.transpose(0, 1).reshape(hk, b * g * n, d)
    sp = torch.matmul(rows, pk.transpose(1, 2).contiguous()).view(hk, b, g * n, -1).transpose(0, 1) * scale
    so = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    j = torch.arange(mine, device=q.device)
    last = s["lens"].long()[:, None, None] - 1
    if case["causal"]:
        last = last - (n - 1) + torch.arange(n, device=q.device)[None, :, None]
    seen = (j <= last).expand(b, n, mine)[:, None].expand(b, g, n, mine).reshape(b, 1, g * n, mine)
    so = so.masked_fill(~seen, float("-inf"))
    top = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    sp, so = torch.exp(sp - top), torch.exp(so - top)
    total = sp.sum(-1, keepdim=True) + so.sum(-1, keepdim=True)
    out = torch.matmul(sp.transpose(0, 1).reshape(hk, b * g * n, -1), pv).view(hk, b, g * n, d).transpose(0, 1)
    out = (out + torch.matmul(so, v)) / torch.where(total == 0, torch.ones_like(total), total)
    return out.reshape(b, h, n, d).to(s["q"].dtype)


def _segment_of_rows(offs, rows):
    return torch.bucketize(torch.arange(rows, device=offs.device), offs[1:-1].contiguous(), right=True)


def _plain_adapters(s):
    case = s["case"]
    m, k, n, r, na = case["rows"], case["k"], case["n"], case["rank"], case["adapters"]
    x = s["x"].float()
    # weights dequantised to x's type, as the framework's linear does
    w = (s["qs"].float().view(n, k // 32, 32) * s["scales"][:, :, None]).view(n, k).to(s["x"].dtype).float()
    y = torch.matmul(x, w.t()) + s["bias"]
    which = s["ids"].long()[_segment_of_rows(s["offs"], m)]
    mine = (which[:, None] == torch.arange(na, device=x.device)).float() * s["alpha"]
    t = torch.matmul(x, s["a"].float().view(na * r, k).t()).view(m, na, r) * mine[:, :, None]
    y = y + torch.matmul(t.view(m, na * r), s["b"].float().permute(0, 2, 1).reshape(na * r, n))
    return y.to(s["x"].dtype)


def _plain_norm(x, kind, w, b, eps):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    return x if b is None else x + b


def _plain_block(s):
    case = s["case"]
    gate, shift, scale = _modulation(s)
    n = _plain_norm(s["h"].float(), case["norm"], s["post_w"], s["post_b"], 1e-6) * s["gamma"]
    if gate is not None:
        seg = _segment_of_rows(s["offs"], case["rows"])
        n = n * gate[seg]
    x = (s["x"].float() + n).to(s["x"].dtype)
    # the next norm reads the residual stream as it is stored
    y = _plain_norm(x.float(), case["norm"], s["pre_w"], s["pre_b"], 1e-6)
    if gate is not None:
        y = y * (scale[seg] + 1.0) + shift[seg]
    return x, y.to(x.dtype)


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return _plain_prefix(s) if kind == "prefix" else _plain_adapters(s) if kind == "adapters" else _plain_block(s)
    ops = _ops()
    if kind == "prefix":
        return ops.sdpa_shared_prefix(s["q"], s["prefix_k"], s["prefix_v"], s["k"], s["v"], 1.0 / math.sqrt(case["dim"]),
                                      lens=s["lens"], causal=case["causal"])
    if kind == "adapters":
        return ops.q8_0_linear_adapters(s["x"], s["qs"], s["scales"], s["a"], s["b"], s["ids"], alphas=s["alpha"],
                                        seg_offsets=s["offs"], bias=s["bias"], out_dtype=DTYPES[case["dtype"]])
    gate, shift, scale = _modulation(s)
    return ops.norm_gated_residual_norm(s["x"], s["h"], post_weight=s["post_w"], post_bias=s["post_b"],
                                        ls_gamma=s["gamma"], gate=gate, pre_weight=s["pre_w"], pre_bias=s["pre_b"],
                                        shift=shift, scale=scale, seg_offsets=s["offs"], norm=case["norm"], eps=1e-6)


# ---- what a pass cannot do without --------------------------------------------

def work(case):
    e = BYTES[case["dtype"]]
    if case["kind"] == "prefix":
        b, h, hk, d, n = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["queries"]
        lens = _lens(case)
        # query i of a causal sequence sees its last n - 1 - i keys less
        pairs = b * n * case["prefix"] + sum(n * m - (n * (n - 1) // 2 if case["causal"] else 0) for m in lens)
        return {"bytes": (2 * b * h * n * d + 2 * hk * case["prefix"] * d + 2 * hk * sum(lens) * d) * e + 4 * b,
                "flops": 4 * h * d * pairs}
    if case["kind"] == "adapters":
        m, k, n, r, na = case["rows"], case["k"], case["n"], case["rank"], case["adapters"]
        return {"bytes": m * k * e + n * k + n * k // 32 * 4 + n * 4 + na * r * (k + n) * e + m * n * e,
                "flops": 2 * m * k * n + 2 * m * r * (k + n)}
    m, c = case["rows"], case["width"]
    return {"bytes": 4 * m * c * e + (5 if case["norm"] == "layer" else 3) * c * 4
            + (3 * case["segments"] * c * 4 if case["modulated"] else 0), "flops": 0}


# ---- the definition in 64 bits --------------------------------------------------

def _exact_prefix(s):
    case = s["case"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    g, n, scale = case["heads"] // case["kv_heads"], case["queries"], 1.0 / math.sqrt(case["dim"])
    pk, pv = s["prefix_k"].double(), s["prefix_v"].double()
    for b, length in enumerate(s["lens"].tolist()):
        for h in range(case["heads"]):
            kv = h // g
            keys = torch.cat([pk[kv], s["k"][b, kv, :length].double()])
            values = torch.cat([pv[kv], s["v"][b, kv, :length].double()])
            score = torch.mm(s["q"][b, h].double(), keys.t().contiguous()) * scale
            if case["causal"]:
                hidden = torch.ones((n, n), dtype=torch.bool, device=score.device).triu(1)
                score[:, score.shape[1] - n:].masked_fill_(hidden, float("-inf"))
            out[b, h] = torch.softmax(score, -1) @ values
    return out


def _exact_adapters(s):
    case = s["case"]
    x = s["x"].double()
    w = s["qs"].double() * s["scales"].double().repeat_interleave(32, 1)
    y = x @ w.to(s["x"].dtype).double().t().contiguous() + s["bias"].double()
    offs = s["offs"].tolist()
    for j, which in enumerate(s["ids"].tolist()):
        if which >= 0:
            part = x[offs[j]:offs[j + 1]] @ s["a"][which].double().t().contiguous()
            y[offs[j]:offs[j + 1]] += s["alpha"][which].double() * (part @ s["b"][which].double().t().contiguous())
    return y


def _exact_norm(s):
    case, eps = s["case"], 1e-6

    def norm(t, w, b):
        t = t - t.mean(-1, keepdim=True) if case["norm"] == "layer" else t
        t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps) * w.double()
        return t if b is None else t + b.double()

    p = None if s["t_emb"] is None else s["t_emb"].double()
    c, offs, xs, ys = case["width"], s["offs"].tolist(), [], []
    for j in range(case["segments"]):
        rows = slice(offs[j], offs[j + 1])
        n = norm(s["h"][rows].double(), s["post_w"], s["post_b"]) * s["gamma"].double()
        n = n if p is None else n * p[j, 2 * c:3 * c]
        x = s["x"][rows].double() + n
        y = norm(x.to(s["x"].dtype).double(), s["pre_w"], s["pre_b"])
        xs.append(x)
        ys.append(y if p is None else y * (p[j, 4 * c:5 * c] + 1) + p[j, 3 * c:4 * c])
    return torch.cat(xs), torch.cat(ys)


def exact(case, seed):
    s = prepare(case, seed)
    return {"prefix": _exact_prefix, "adapters": _exact_adapters, "norm": _exact_norm}[case["kind"]](s)
