"""Linear layers on microscaled 4-bit weights, as measured cases.

A case is a dict of plain values; "kind" names the operator:
  round    quantisation to microscaled 4-bit values (e2m1, one power of two per 32 values) and back
  linear   x W^T + bias, W in 4 bits; "arith" says whether x enters as it is ("plain") or in 4 bits too ("fp4")
  gated    act(x Wg^T + bg) * (x Wu^T + bu), the first half of a gated feed-forward block, in either arithmetic
`own` chooses between the operators in elementary torch operations (32-bit, rounded once) and the framework's entry
points (`lux3d_fused.ops`). `exact` is the definition in 64 bits.

A packed matrix [rows, k]: bytes [rows, k / 2], the value of even k in the low four bits; scales [ceil(k / 128), rows, 4],
byte j of group g the exponent (bias 127) of the row's block 4 g + j.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
_OPS = []


def _ops():
    if not _OPS:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "candle-3d_amd"))
        from lux3d_fused import ops
        _OPS.append(ops)
    return _OPS[0]


def listed():
    return [
        # tokens of both halves of the guidance pair of TripoSG, as a layer receives them
        {"name": "round_tokens", "kind": "round", "rows": 4098, "k": 2048, "dtype": "bf16"},
        # a feed-forward weight of an f32 checkpoint on its way to 4 bits
        {"name": "round_weight", "kind": "round", "rows": 8192, "k": 2048, "dtype": "f32"},
        # TRELLIS.2 AdaLN linear: one modulation vector per request
        {"name": "linear_adaln", "kind": "linear", "arith": "plain", "rows": 2, "k": 1536, "n": 9216, "dtype": "bf16"},
        # TripoSG feed-forward down-projection
        {"name": "linear_triposg", "kind": "linear", "arith": "plain", "rows": 4098, "k": 8192, "n": 2048, "dtype": "bf16"},
        # DINOv3 MLP up-projection of one image, in the encoder's f32
        {"name": "linear_dinov3", "kind": "linear", "arith": "plain", "rows": 1029, "k": 1024, "n": 4096, "dtype": "f32"},
        # the TripoSG timestep embedding's projection for both halves of the guidance pair
        {"name": "fp4_token", "kind": "linear", "arith": "fp4", "rows": 2, "k": 2048, "n": 8192, "dtype": "bf16"},
        # TRELLIS.2 SLAT output projection of a ragged batch, an odd number of voxels
        {"name": "fp4_slat", "kind": "linear", "arith": "fp4", "rows": 9001, "k": 1536, "n": 1536, "dtype": "bf16"},
        # TripoSG feed-forward up-projection of four requests
        {"name": "fp4_triposg", "kind": "linear", "arith": "fp4", "rows": 16392, "k": 2048, "n": 8192, "dtype": "bf16"},
        # gated feed-forward of one conditioning vector
        {"name": "gated_token", "kind": "gated", "arith": "plain", "rows": 1, "k": 1024, "n": 4096, "act": "silu",
         "dtype": "bf16"},
        # gated feed-forward of the image encoder's tokens, f16
        {"name": "gated_dinov3", "kind": "gated", "arith": "plain", "rows": 1029, "k": 1024, "n": 4096, "act": "silu",
         "dtype": "f16"},
        # gated feed-forward on both halves of the guidance pair, 4-bit products
        {"name": "gated_triposg", "kind": "gated", "arith": "fp4", "rows": 4098, "k": 2048, "n": 8192, "act": "gelu_erf",
         "dtype": "bf16"},
        # odd sizes: hidden width no multiple of a tile, k no multiple of 128
        {"name": "gated_odd", "kind": "gated", "arith": "fp4", "rows": 777, "k": 1120, "n": 3001, "act": "gelu_tanh",
         "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(["round", "linear", "linear", "linear", "gated", "gated"])
    if kind == "round":
        return {"kind": kind, "rows": _log(rng, 1, 30000), "k": 32 * _log(rng, 2, 256), "dtype": rng.choice(["bf16", "f16", "f32"])}
    k, n = rng.choice([(1024, 4096), (4096, 1024), (2048, 8192), (8192, 2048), (1536, 9216), (1536, 1536), (2048, 2048),
                       (32 * _log(rng, 2, 256), _log(rng, 8, 9000))])
    rows = rng.randint(1, 64) if rng.random() < 0.35 else _log(rng, 65, 16000)
    case = {"kind": kind, "arith": rng.choice(["plain", "fp4"]), "rows": rows, "k": k, "n": n,
            "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if kind == "gated":
        case["act"] = rng.choice(["silu", "gelu_erf", "gelu_tanh"])
    return case


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= most:
            return case


# ---- the format, in elementary 32-bit operations --------------------------------

def _power(e):
    """2^e for whole e in -127 .. 127, from its bits: a power function may be off in its last place."""
    bits = torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22))
    return bits.to(torch.int32).view(torch.float32)


def _codes(x):
    """x [rows, k] f32 -> values on the 4-bit grid [rows, k / 32, 32], and the exponents (bias 127) [rows, k / 32]."""
    b = x.reshape(x.shape[0], -1, 32)
    top = b.abs().amax(-1)
    e = ((top.view(torch.int32) >> 23) - 2).clamp(min=0)
    v = b * _power(127 - e)[:, :, None]
    m = v.abs()
    # steps of 1/2 below 2, 1 below 4, 2 above; ties to even; 6 is the largest value
    r = torch.where(m < 2, torch.round(m * 2) / 2, torch.where(m < 4, torch.round(m), torch.round(m / 2) * 2)).clamp(max=6)
    return torch.copysign(r, v), e


def _rounded(x):
    v, e = _codes(x)
    return (v * _power(e - 127)[:, :, None]).reshape(x.shape)


def _pack(w):
    """w [n, k] f32 -> the packed bytes and the scales by groups of four blocks."""
    v, e = _codes(w)
    n, k = w.shape
    m = v.abs()
    code = torch.where(m < 2, m * 2, torch.where(m < 4, m + 2, m / 2 + 4)).to(torch.uint8) + torch.signbit(v).to(torch.uint8) * 8
    code = code.reshape(n, k // 2, 2)
    groups = (k + 127) // 128
    s = torch.zeros((n, groups * 4), dtype=torch.uint8, device=w.device)
    s[:, :k // 32] = e.to(torch.uint8)
    return code[:, :, 0] | (code[:, :, 1] << 4), s.view(n, groups, 4).permute(1, 0, 2).contiguous()


def _unpack(q, s):
    n, k = q.shape[0], q.shape[1] * 2
    code = torch.stack([q & 15, q >> 4], -1).reshape(n, k).long()
    table = torch.tensor(VALUES + [-v for v in VALUES], device=q.device)
    e = s.permute(1, 0, 2).reshape(n, -1)[:, :k // 32].to(torch.int32) - 127
    return (table[code].view(n, k // 32, 32) * _power(e)[:, :, None]).view(n, k)


# ---- inputs -------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 31)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda") * std

    rows, k = case["rows"], case["k"]
    x = normal(rows, k)
    # channels far larger than the others, as activations have them, and tokens of different size
    x *= torch.where(torch.rand(k, generator=g, device="cuda") < 0.01, 12.0, 1.0)
    x *= torch.exp(normal(rows, 1, std=0.5))
    s = {"case": case, "x": x.to(DTYPES[case["dtype"]])}
    if case["kind"] == "round":
        return s
    for name in ("up", "gate") if case["kind"] == "gated" else ("up",):
        s[name] = _pack(normal(case["n"], k, std=1.0 / math.sqrt(k)))
        s[name + "_bias"] = normal(case["n"], std=0.2)
    return s


# ---- one pass -----------------------------------------------------------------

def _plain_act(v, act):
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu_erf":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))


def _plain(s):
    case, x = s["case"], s["x"].float()
    if case["kind"] == "round":
        return _rounded(x).to(s["x"].dtype)
    if case["arith"] == "fp4":
        x = _rounded(x)
    y = torch.matmul(x, _unpack(*s["up"]).t()) + s["up_bias"]
    if case["kind"] == "gated":
        y = _plain_act(torch.matmul(x, _unpack(*s["gate"]).t()) + s["gate_bias"], case["act"]) * y
    return y.to(s["x"].dtype)


def run(s):
    if not own:
        return _plain(s)
    ops, case = _ops(), s["case"]
    if case["kind"] == "round":
        q, scales = ops.mxfp4_quantize(s["x"])
        return ops.mxfp4_dequantize(q, scales, s["x"].dtype)
    if case["kind"] == "gated":
        return ops.mxfp4_linear_gated(s["x"], s["gate"], s["up"], case["act"], gate_bias=s["gate_bias"],
                                      up_bias=s["up_bias"], fp4=case["arith"] == "fp4")
    linear = ops.mxfp4_linear_fp4 if case["arith"] == "fp4" else ops.mxfp4_linear
    return linear(s["x"], *s["up"], bias=s["up_bias"])


# ---- what a pass cannot do without --------------------------------------------

def work(case):
    m, k, e = case["rows"], case["k"], BYTES[case["dtype"]]
    if case["kind"] == "round":
        return {"bytes": 2 * m * k * e, "flops": 0}
    n, mats = case["n"], 2 if case["kind"] == "gated" else 1
    return {"bytes": m * k * e + mats * (n * k // 2 + n * k // 32 + 4 * n) + m * n * e, "flops": 2 * m * k * n * mats}


# ---- the definition in 64 bits --------------------------------------------------

def _exact_power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_rounded(x):
    """Each value of a block of 32 goes to the nearest of the block's fifteen, by the midpoints between them."""
    b = x.reshape(x.shape[0], -1, 32)
    _, e = torch.frexp(b.abs().amax(-1, keepdim=True))  # amax = m 2^e, 1/2 <= m < 1
    unit = _exact_power((e - 3).clamp(min=-127))
    t = b.abs() / unit
    out = torch.zeros_like(t)
    for j in range(7):
        mid = (VALUES[j] + VALUES[j + 1]) / 2
        # a tie goes to the neighbour whose last bit is 0: the one of even place
        past = t >= mid if j % 2 else t > mid
        out = torch.where(past, torch.full_like(t, VALUES[j + 1]), out)
    return (torch.sign(b) * out * unit).reshape(x.shape)


def _exact_weight(packed):
    q, s = packed
    n, k = q.shape[0], 2 * q.shape[1]
    w = torch.empty((n, k), dtype=torch.float64, device=q.device)
    for half in range(2):
        code = (q >> (4 * half)) & 15
        sign, exponent, mantissa = 1.0 - 2.0 * (code >> 3).double(), ((code >> 1) & 3).long(), (code & 1).double()
        w[:, half::2] = sign * torch.where(exponent == 0, 0.5 * mantissa, _exact_power(exponent - 1) * (1 + 0.5 * mantissa))
    for b in range(k // 32):
        w[:, 32 * b:32 * b + 32] *= _exact_power(s[b // 4, :, b % 4].long() - 127)[:, None]
    return w


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["kind"] == "round" or case["arith"] == "fp4":
        x = _exact_rounded(x)
    if case["kind"] == "round":
        return x
    up = torch.addmm(s["up_bias"].double(), x, _exact_weight(s["up"]).t())
    if case["kind"] == "linear":
        return up
    v = torch.addmm(s["gate_bias"].double(), x, _exact_weight(s["gate"]).t())
    if case["act"] == "silu":
        return v * torch.sigmoid(v) * up
    if case["act"] == "gelu_erf":
        return v * torch.special.ndtr(v) * up
    return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)) * up
