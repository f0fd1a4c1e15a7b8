"""The microscaled 4-bit format and its linears in 64 bits, for the tests."""
import math

import torch

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24
VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)

# the erf GELU's polynomial as the kernels hold it, for the bound of its evaluation
ERF_P = (2.30221868, 0.10480535, 6.56670745e-05, 0.000170996558, 1.36602803e-05, 6.01039289e-07, 1.58674034e-08,
         2.34277681e-10, 1.48678726e-12)


def power(e):
    """2^e exactly, whole e in -1022 .. 1023."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantize(x):
    """x [rows, k] -> (codes u8 [rows, k], exponents [rows, k / 32]) by the definition: the nearest value, ties to even."""
    b = x.double().reshape(x.shape[0], -1, 32)
    top = b.abs().amax(-1)
    _, e = torch.frexp(torch.where(torch.isfinite(top), top, torch.ones_like(top)))
    s = torch.where(top == 0, torch.zeros_like(e), (e - 3 + 127).clamp(min=0))
    s = torch.where(torch.isfinite(b).all(-1), s, torch.full_like(s, 255))
    t = b.abs() / power(s - 127)[:, :, None]
    code = torch.zeros_like(t, dtype=torch.uint8)
    for j in range(7):
        mid = (VALUES[j] + VALUES[j + 1]).item() / 2
        code += ((t >= mid) if j % 2 else (t > mid)).to(torch.uint8)  # a tie goes to the even code
    return (code + 8 * torch.signbit(b).to(torch.uint8)).reshape(x.shape), s


def values(codes, s):
    """Codes [rows, k] and exponents [rows, k / 32] -> f64."""
    table = torch.cat([VALUES, -VALUES]).to(codes.device)
    v = table[codes.long()].reshape(codes.shape[0], -1, 32)
    scale = torch.where(s == 255, torch.full_like(s, 0, dtype=torch.float64) * math.nan, power(s.long() - 127))
    return (v * scale[:, :, None]).reshape(codes.shape)


def pack(codes, s):
    c = codes.reshape(codes.shape[0], -1, 2)
    rows, blocks = s.shape
    g = (blocks + 3) // 4
    e = torch.zeros((rows, 4 * g), dtype=torch.uint8, device=s.device)
    e[:, :blocks] = s.to(torch.uint8)
    return c[:, :, 0] | (c[:, :, 1] << 4), e.view(rows, g, 4).permute(1, 0, 2).contiguous()


def unpack(q, scales):
    """(codes, exponents) of packed storage."""
    rows = scales.shape[1]
    q = q.reshape(rows, -1)
    codes = torch.stack([q & 15, q >> 4], -1).reshape(rows, -1)
    return codes, scales.permute(1, 0, 2).reshape(rows, -1)[:, :codes.shape[1] // 32].int()


def dense(q, scales):
    return values(*unpack(q, scales))


def product(x, w, bias, e_x=0.0):
    """(x W^T + bias, a bound on the error of its f32 sum). A sum of K products is formed in f32 from pieces of 16 products
    at least, so it is off by at most (K / 16 + 64) u of its terms' magnitudes, the bias among them (tiles: the sum starts
    at it, and it passes every one of the K / 16 + 64 additions); f32 x enters as three bf16 terms, each product within 2 u."""
    xd, wd = x.double(), w.double()
    y = torch.mm(xd, wd.t().contiguous())
    err = torch.mm(xd.abs(), wd.abs().t().contiguous()) * ((x.shape[1] / 16 + 64) * U + e_x)
    if bias is not None:
        y, err = y + bias.double(), err + (x.shape[1] / 16 + 64) * U * bias.double().abs()
    return y, err + U * y.abs()


def activation(v, act):
    """(act(v), a bound on its evaluation): the polynomial of degree 8 in f32 by Horner's rule (18 u of its terms'
    magnitudes), times v, enters exp2; 1 + exp2, its reciprocal and the product take 8 u; erf's fit 1.7e-7. From 2^126 on
    the reciprocal of 1 + exp2 is subnormal and comes out as 0, which takes |v| 2^-126 at most (tanh GELU below -10)."""
    t = v * v
    if act == "silu":
        sig, terms, fit = torch.sigmoid(v), torch.full_like(v, 1.4427), 0.0
    elif act == "gelu_tanh":
        sig, terms, fit = torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)), 2.3023 + 0.10295 * t, 0.0
    else:
        sig = torch.special.ndtr(v)
        tt = t.clamp(max=30.25)
        terms, fit = sum(c * tt ** i for i, c in enumerate(ERF_P)), 1.7e-7
    y = v * sig
    return y, fit + v.abs() * 2.0 ** -126 + y.abs() * ((1 - sig) * v.abs() * math.log(2) * 18 * U * terms + 8 * U)


def gated(gate, up, act):
    """act(g) * u from two (value, bound) pairs. No activation here is steeper than 1.13."""
    (g, eg), (u, eu) = gate, up
    a, ea = activation(g, act)
    ea = ea + 1.13 * eg
    y = a * u
    return y, ea * u.abs() + a.abs() * eu + ea * eu + U * y.abs()


def check(got, want, bound, what):
    """got against want within bound and one rounding to got's type."""
    fi = torch.finfo(got.dtype)
    got = got.reshape(want.shape).double()
    bound = bound + fi.eps / 2 * (want.abs() + bound) + fi.smallest_normal * fi.eps
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - bound
    assert float(over.max()) <= 0, (f"{what}: worst error {float((got - want).abs().max()):.3g}, "
                                    f"{int((over > 0).sum())} of {over.numel()} values past the bound")
