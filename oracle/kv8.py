"""The 8-bit KV cache and the attention over it, restated in 64 bits (test infrastructure only).

A cache is a function of the bf16 keys and values written so far, whatever calls wrote
them: ``Cache`` holds those, ``expected`` gives the codes, scales and tails that a
sequence of n positions must have, ``values`` what the cache then stands for, ``attend``
softmax attention over it with an elementwise bound on what the kernels may be off by.
"""
from __future__ import annotations

import math

import torch

BLOCK = 64
TOP = {torch.int8: 127, torch.float8_e4m3fn: 448}
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}   # half a step, relative to the value
FP16 = 2.0 ** -11


def round_e4m3(y: torch.Tensor) -> torch.Tensor:
    """float64 to the nearest e4m3 value, ties to even: steps of 2^(e - 3), e >= -6."""
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(y / step) * step


def quantise(x: torch.Tensor, dtype: torch.dtype):
    """Blocks [..., 64, D] of bf16 values -> (codes as float64 values, fp32 scales).  x * top / amax in
    float64 is within 2^-52 of the quotient of two integers of at most 15 and 8 bits, which is either a
    tie (then a multiple of 2^-10 below 2^9, which the division gives exactly) or at least 2^-17 off one."""
    top, v = TOP[dtype], x.double()
    amax = v.abs().amax((-1, -2))
    ok = torch.isfinite(v).all(-1).all(-1)
    safe = torch.where(ok & (amax > 0), amax, torch.ones_like(amax))
    y = torch.where(ok[..., None, None], v, torch.zeros_like(v)) * top / safe[..., None, None]
    y = torch.round(y) if dtype == torch.int8 else round_e4m3(y)
    scale = torch.clamp(amax.float() / top, min=2.0 ** -126)
    return y, torch.where(ok, scale, torch.full_like(scale, float("nan")))


def values(k: torch.Tensor, v: torch.Tensor, n: int, dtype: torch.dtype):
    """What the cache holds of keys and values [KVH, >= n, D] (bf16) after n positions, float64 [KVH, n, D]."""
    out = []
    for x in (k, v):
        y = x[:, :n].double().clone()
        for i in range(0, n // BLOCK * BLOCK, BLOCK):
            code, scale = quantise(x[:, i:i + BLOCK], dtype)
            y[:, i:i + BLOCK] = code * scale.double()[:, None, None]
        out.append(y)
    return out


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """bf16 [n, heads, D] at the angle rows [n, D/2]: fp32 products and sums, each rounded by itself."""
    x1, x2 = x.float().chunk(2, dim=-1)
    c, s = cos[:, None], sin[:, None]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1).to(torch.bfloat16)


def attend(q: torch.Tensor, p: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, window: int = 0,
           sinks: int = 0):
    """q [T, H, D] (bf16) at positions p [T] (negative: outside) over float64 keys and values [KVH, n, D]
    -> (out float64 [T, H, D], bound [T, H, D]).

    The bound: a score is a sum of D products in fp32 and two more roundings, off by at most
    (D + 2) 2^-24 sum |q k| scale; a query element below 2^-31 of its row's largest is rounded to steps
    of 2^-38 of that (fp16 of the scaled row), 2^-39 max |q| |k| each.  The difference to the maximum, the
    exponential (one unit in the last place), the base change and the logarithm in the exponent add
    2^-19 + 2^-22 |s - max|.  A probability's relative error d enters numerator and denominator.

    P is rounded once for the product, to fp16 (2^-11; the pair of bf16 over the open block leaves 2^-16),
    and the denominator may be the sum of the rounded ones.  sum w_i (1 + r_i) v_i / sum w_i (1 + r_i) is then
    off by at most sum w_i |r_i| (|v_i| + |out|).

    fp16 has steps of 2^-24 below 2^-14.  What is rounded is P g with g >= 2^3, P relative to a reference
    that is at or below the row's maximum: half a step is 2^-25 / g <= 2^-28 in units in which the
    denominator is at least 1, so a seen position's value enters wrong by at most 2^-28 |v| and the
    denominator by 2^-28.

    Sums over n positions and split states add (n + 64) 2^-24 of the magnitudes, the output is rounded to
    bf16 once.  Sums are held in units of at least 2^-32, so that fp32's smallest step, 2^-149, is 2^-117.

    Only values that a row sees are in its bound, but they have to be numbers throughout."""
    T, H, D = q.shape
    KVH, n, _ = k.shape
    at = torch.arange(n)
    seen = (at <= p[:, None])
    if window:
        seen = seen & ((at > p[:, None] - window) | (at < sinks))
    out = torch.zeros((T, H, D), dtype=torch.float64)
    bound = torch.zeros_like(out)
    rows = seen.any(1)
    G = H // KVH
    for h in range(H):
        kk, vv = k[h // G], v[h // G]
        qq = q[:, h].double()
        s = (qq @ kk.T * scale).masked_fill(~seen, float("-inf"))
        mag = (qq.abs() @ kk.abs().T * abs(scale)).masked_fill(~seen, 0.0)
        m = s.amax(1, keepdim=True)
        m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
        e = torch.exp(s - m)
        gap = torch.where(seen, (s - m).abs(), torch.zeros_like(s))
        flushed = 2.0 ** -39 * qq.abs().amax(1, keepdim=True) * kk.abs().sum(1) * abs(scale)
        d = (D + 2) * 2.0 ** -24 * mag + flushed.masked_fill(~seen, 0.0) + 2.0 ** -19 + 2.0 ** -22 * gap
        d = d + d.masked_fill(~seen, 0.0).amax(1, keepdim=True)            # the maximum is off as well
        l = e.sum(1, keepdim=True)
        w = torch.where(rows[:, None], e / torch.where(l > 0, l, torch.ones_like(l)), torch.zeros_like(e))
        out[:, h] = w @ vv
        spread = (w * d) @ vv.abs() + (w * d).sum(1, keepdim=True) * (w @ vv.abs())
        mean, o = w @ vv.abs(), out[:, h].abs()
        small = 2.0 ** -28 * (seen.double() @ vv.abs() + seen.sum(1, keepdim=True) * o)
        bound[:, h] = 1.01 * (spread + small + FP16 * (mean + o) + HALF[torch.bfloat16] * o) + (
            (n + 64) * 2.0 ** -24 * mean + n * 2.0 ** -116)
    return out, bound
