"""Float64 restatement of the 4-bit K/V cache and the attention over it, for
tests: the quantiser, the page blocks' byte layout, and softmax attention
written row by row from the definitions in include/ltxb.h. No counterpart in
the reference (it keeps no K/V between calls)."""

from __future__ import annotations

import math

import torch

PAGE, HD = 64, 128


def bf16(x: torch.Tensor) -> torch.Tensor:
    """float64 -> nearest bf16 value (ties to even), as float64, without a detour through float32."""
    m, e = torch.frexp(x)
    # bf16: 8 significant bits, smallest exponent that of 2^-133
    step = torch.ldexp(torch.ones_like(x), torch.clamp(e - 8, min=-133))
    return torch.where(torch.isfinite(x), torch.round(x / step) * step, x)


def quantise(x: torch.Tensor, group: int):
    """codes [..., 128] int64, scale and zero [..., 128 / group] float64 of bf16-valued x [..., 128]."""
    g = x.double().reshape(*x.shape[:-1], HD // group, group)
    zero = g.amin(-1)
    rng = g.amax(-1) - zero
    scale = bf16(rng / 15)
    s, z = scale[..., None], zero[..., None]
    d = g - z
    b = d - g
    off = (g - (d - b)) + (-z - b)  # g - z = d + off: a difference beyond 53 bits leaves a remainder,
    q = torch.where(s > 0, d / s, torch.zeros_like(g))
    code = torch.round(q).clamp(0, 15)
    rest = d - s * code             # which decides what only rounding made a tie
    code = code + ((s > 0) & (rest == s / 2) & (off > 0)) - (1.0 * ((s > 0) & (rest == -s / 2) & (off < 0)))
    bad = ~torch.isfinite(rng.float())
    scale = torch.where(bad, torch.full_like(scale, math.nan), scale)
    code = torch.where(bad[..., None], torch.zeros_like(code), code)
    return code.to(torch.int64).reshape(x.shape), scale, zero


def values(code, scale, zero):
    group = HD // scale.shape[-1]
    return zero.repeat_interleave(group, -1) + scale.repeat_interleave(group, -1) * code.double()


def held(x: torch.Tensor, group: int) -> torch.Tensor:
    """What the cache holds for x, in float64."""
    return values(*quantise(x, group))


def nibble(block: bytes, at: int, n: int) -> int:
    return (block[at + n // 2] >> (4 * (n % 2))) & 15


def k_code(block: bytes, t: int, d: int) -> int:
    return nibble(block, 64 * t, ((d // 8) % 4) * 32 + (d // 32) * 8 + d % 8)


def v_code(block: bytes, t: int, d: int) -> int:
    return nibble(block, 4096 + 512 * (t // 8) + 64 * ((d // 4) % 8) + 16 * ((t % 8) // 2) + 8 * (t % 2),
                  (d // 32) * 4 + d % 4)


def attention(q, k, v, causal: bool, scale: float | None = None, gate=None) -> torch.Tensor:
    """One sequence: q [n, H, 128], k / v [len, Hkv, 128] (float64 values), the
    rows being the last n tokens; rows that see nothing are zero."""
    n, H, _ = q.shape
    length, hk, _ = k.shape
    scale = 1.0 / math.sqrt(HD) if scale is None else scale
    out = torch.zeros(n, H, HD, dtype=torch.float64)
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    for h in range(H):
        kh, vh = k[:, h // (H // hk)], v[:, h // (H // hk)]
        s = q[:, h] @ kh.T * scale
        for i in range(n):
            seen = min(length, length - n + i + 1) if causal else length
            if seen > 0:
                p = torch.softmax(s[i, :seen], 0)
                out[i, h] = p @ vh[:seen]
    return out if gate is None else out * gate.double().cpu()[:, :, None]
