"""The window-cache operators in 64 bits, row by row, and how far a kernel's
result may be from them.

Bounds count roundings. u(T) = finfo(T).eps / 2 is the most a rounding to T
moves a value, relative to it; F = 2^-24 is that of fp32.

Attention: o = sum_j p_j v_j / sum_j p_j.
  * a logit is a sum of D products: off by at most (D + 4) F scale sum|q k| (any
    order of summation), and its distance to the maximum is rounded before the
    exponential: 2 F |logit - max| more; the fast exponential adds 2^-21.
    A weight is therefore off by w = 2 max_j(logit error) + 2^-20 relative.
  * kernels that multiply weights and values as 16-bit operands round each weight
    once: u(T), or in fp16 2^-32 of the largest weight where that is more (they
    are held at least 2^7 times larger, and fp16 steps by 2^-24 at its low end).
    4-bit caches fold a group's scale into the weight first and round to bf16: u(bf16).
  * a 4-bit row enters as scale * code and lowest apart: its |k| and |v| above are
    15 scale + |lowest|, an upper bound of both parts.
  * sums of n terms in up to n / 8 + 64 steps a chain: (n / 8 + 64) F.
  * the result is rounded to T.
  |got - o| <= u(T) |o| + (1 + u(T)) (2 w + u(P) + 2 (n / 8 + 64) F) sum p |v| / sum p + tiny(T) (+ n 2^-32 max|v|)
"""
from __future__ import annotations

import math

import torch

F = 2.0 ** -24
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def attention(q, k, v, see, scale, dtype, sizes=None):
    """q [H, n, D], k and v [H, m, D] in float64, see [n, m] (or [H, n, m]):
    the result and its bound. A row that sees nothing is 0, exactly. ``sizes``:
    the bounds on |k| and |v| of 4-bit rows."""
    k_size, v_size = sizes or (k.abs(), v.abs())
    see = see.expand(q.shape[0], -1, -1)
    seen_any = see.any(-1, keepdim=True)
    logits = torch.where(see, q @ k.transpose(1, 2) * scale, -math.inf)
    top = torch.where(seen_any, logits.amax(-1, keepdim=True), 0.0)
    p = torch.where(see, torch.exp(logits - top), 0.0)
    total = torch.where(seen_any, p.sum(-1, keepdim=True), 1.0)
    # a masked value never counts, whatever it is: 0 * inf is left out by hand
    finite = torch.isfinite(v).all(-1)
    clean = torch.where(finite[..., None], v, 0.0)
    clean_size = torch.where(finite[..., None], v_size, 0.0)
    out, size = p @ clean / total, p @ clean_size / total
    spread = torch.where(see, (logits - top).abs(), 0.0).amax(-1, keepdim=True)
    products = torch.where(see, q.abs() @ k_size.transpose(1, 2) * abs(scale), 0.0).amax(-1, keepdim=True)
    w = 2 * ((q.shape[-1] + 4) * F * products + 2 * F * spread) + 2.0 ** -20
    n = see.sum(-1, keepdim=True)
    u, up = unit(dtype), unit(torch.bfloat16 if sizes else dtype)
    bound = u * out.abs() + (1 + u) * (2 * w + up + 2 * (n / 8 + 64) * F) * size + TINY[dtype]
    if dtype == torch.float16 and not sizes:
        bound = bound + n * 2.0 ** -32 * clean_size.amax()
    return out, torch.where(seen_any, bound, 0.0)


def check(got, want, bound, what=""):
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: {int((~torch.isfinite(got)).sum())} values are not finite"
    off = (got - want).abs()
    worst = (off - bound).max().item()
    assert worst <= 0, f"{what}: {int((off > bound).sum())} of {off.numel()} values past their bound, the worst by {worst:.3g}"


def rotated(x, positions, frequencies, gain, epsilon, dtype):
    """Norm and rotation of x [n, H, D] at int64 positions [n]: result and bound.

    The mean square is a sum of up to 8 terms a lane and log2(lanes) <= 5 more
    steps: 13 F, half of it after the root; root, quotient and two products add
    4 F: a normed value is off by 11 F relative at most. An angle's fraction of a
    turn is rounded to fp32 (2 pi F / 2 radians) and sincospi is good to 2 F;
    products and sum add 2 F more: at most 24 F (|a| + |b|) for a pair (a, b)."""
    x = x.double()
    if gain is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + epsilon) * gain.double()
    out, slack = x.clone(), 24 * F * x.abs()
    r = frequencies.shape[0]
    angle = positions[:, None, None].double() * frequencies
    a, b = x[..., 0:2 * r:2], x[..., 1:2 * r:2]
    out[..., 0:2 * r:2] = a * angle.cos() - b * angle.sin()
    out[..., 1:2 * r:2] = a * angle.sin() + b * angle.cos()
    slack[..., 0:2 * r:2] = slack[..., 1:2 * r:2] = 24 * F * (a.abs() + b.abs())
    return out, slack + unit(dtype) * (out.abs() + slack) + TINY[dtype]


def slots_of(position, newest, sinks, window):
    """The slot of each position (a list), None where it does not stay."""
    return [p if p < sinks else sinks + (p - sinks) % window if p > newest - window else None for p in position]


def quantise(x):
    """[..., D] fp32 -> (codes [..., D] uint8, scale, lowest [..., D / 32] bf16), the stored definition."""
    x = x.float().unflatten(-1, (-1, 32))
    low, high = x.amin(-1), x.amax(-1)
    scale, lowest = ((high - low) * torch.tensor(1 / 15, dtype=torch.float32, device=x.device)).bfloat16(), low.bfloat16()
    s = scale.float()[..., None]
    codes = torch.where(s > 0, torch.round((x - lowest.float()[..., None]) / s).clamp(0, 15), torch.zeros_like(x))
    return codes.to(torch.uint8).flatten(-2), scale, lowest


def pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def unpack(packed, scales):
    """What 4-bit rows stand for, in float64."""
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).unflatten(-1, (-1, 32)).double()
    return (codes * scales[..., 0:1].double() + scales[..., 1:2].double()).flatten(-2)
