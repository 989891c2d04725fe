"""The 8-bit cache, rotary positions and attention over the cache, in 64 bits from their definitions."""
from __future__ import annotations

import math

import torch

BLOCK = 32


def codes(block: torch.Tensor) -> torch.Tensor:
    """round_half_even(127 x / max|x|) of a block of FP16 or BF16 numbers, exactly: a quotient that is on a tie is so in 64 bits
    too, and one that is not is further from it than 64-bit division errs (both operands have at most eleven bits)."""
    wide = block.double()
    top = wide.abs().amax()
    return torch.round(wide * 127.0 / top) if top > 0 else torch.zeros_like(wide)


def held(x: torch.Tensor, length: int) -> torch.Tensor:
    """[tokens, heads, d] as the cache gives them back (64 bits, not yet rounded to the cache's type), zeros behind ``length``."""
    out = torch.zeros_like(x, dtype=torch.float64)
    out[:length] = x[:length].double()
    for begin in range(0, length // BLOCK * BLOCK, BLOCK):
        for head in range(x.shape[1]):
            block = x[begin:begin + BLOCK, head]
            top = block.float().abs().amax()
            if not torch.isfinite(block.float()).all():
                out[begin:begin + BLOCK, head] = torch.nan
            else:
                scale = (top / 127.0).double()             # FP32, as it is stored
                out[begin:begin + BLOCK, head] = codes(block) * scale
    return out


def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, scale: float, interleaved: bool) -> torch.Tensor:
    """[..., heads, d] turned, in 64 bits."""
    turned = 2 * inv_freq.numel()
    angle = positions.double()[..., None, None] * inv_freq.double()
    c, s = angle.cos() * scale, angle.sin() * scale
    out = x.double().clone()
    if interleaved:
        a, b = x.double()[..., 0:turned:2], x.double()[..., 1:turned:2]
        out[..., 0:turned:2], out[..., 1:turned:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x.double()[..., :turned // 2], x.double()[..., turned // 2:turned]
        out[..., :turned // 2], out[..., turned // 2:turned] = a * c - b * s, b * c + a * s
    return out


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, length: int, count: int, softmax_scale: float):
    """One sequence: q [tokens, q_heads, d], k and v [length, kv_heads, d] in 64 bits.  Returns the output and, for the bound on a
    kernel's error, sum p |v| / sum p."""
    tokens, q_heads, d = q.shape
    group = q_heads // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    weight = torch.zeros_like(out)
    last = length - count + torch.arange(count, device=q.device)                  # position of each query
    hidden = torch.arange(length, device=q.device)[None, :] > last[:, None]
    some = (last >= 0)[:, None, None]
    for head in range(k.shape[1] if length > 0 and count > 0 else 0):
        rows = q[:count, head * group:(head + 1) * group].double()
        scores = torch.einsum("ihd,td->iht", rows, k[:, head]) * softmax_scale
        p = torch.softmax(scores.masked_fill(hidden[:, None, :] & some, -math.inf), -1)
        out[:count, head * group:(head + 1) * group] = torch.where(some, p @ v[:, head], 0.0)
        weight[:count, head * group:(head + 1) * group] = torch.where(some, p @ v[:, head].abs(), 0.0)
    return out, weight


def attention_bound(out: torch.Tensor, weight: torch.Tensor, dtype: torch.dtype, top: float) -> torch.Tensor:
    """How far a kernel may be off: a probability is rounded to FP16, off by half a step, 2^-11 of itself, and where the sum is of the
    rounded ones it is off by as much (sum p_i (1 + e_i) v_i / sum p_i (1 + e_i) with |e_i| <= 2^-11 differs from sum p_i v_i by
    sum p_i e_i (v_i - out) to first order, at most 2^-11 of sum p |v| and 2^-11 of |out|); scores are FP32 sums of exact products
    and their exponentials good to some 2^-18 of themselves (scores below 100: 100 * 2^-24 from each of a handful of roundings), for
    which there is 2^-13; the result is rounded once to its type; and probabilities far below the largest are held in steps of 2^-35
    of it (``top`` is the largest |v| times the number of tokens)."""
    return weight * (2.0 ** -11 + 2.0 ** -13) + out.abs() * (2.0 ** -11 + torch.finfo(dtype).eps / 2) + top * 2.0 ** -34
