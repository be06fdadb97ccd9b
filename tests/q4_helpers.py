"""The 4-bit cache's format restated value by value in 64 bits, and dense caches
with the values that it holds."""
from __future__ import annotations

import math

import torch

ORDER = [0, 2, 4, 6, 1, 3, 5, 7]  # the channels of a 32-bit word, lowest first


def least_scale(dtype):
    return 2.0 ** -120 if dtype == torch.bfloat16 else 2.0 ** -21


def quantise(x, dtype):
    """Codes (int64), zero points and scales (float64) of x [..., d]."""
    x = x.double().unflatten(-1, (-1, 32))
    lo, hi = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
    # (32 bits, of halves that stay within them)
    t = ((hi / 2 - lo / 2).float() / torch.full_like(hi, 7.5, dtype=torch.float32)).double()
    m, e = torch.frexp(t)
    s = torch.ldexp(torch.ceil(m * 16) / 16, e)
    s = torch.where(t > 0, s.clamp(min=least_scale(dtype)), 0.0)
    by = torch.where(s > 0, s, 1.0)
    z = torch.round(-lo / by)
    n = torch.round(x / by[..., None])
    n = torch.where((n * by[..., None]).abs() > torch.finfo(dtype).max, n - n.sign(), n)
    c = (n + z[..., None]).clamp(0, 15)
    odd = ~x.isfinite().all(-1)
    z, s = torch.where(odd, 0.0, z), torch.where(odd, float("nan"), s)
    c = torch.where(odd[..., None], 0.0, c)
    return c.long(), z.long(), s


def values(x, dtype):
    """What a cache holds for x [..., d], in 64 bits."""
    c, z, s = quantise(x, dtype)
    return ((c - z[..., None]) * s[..., None]).flatten(-2)


def pack(k, v, dtype, into=None, at=None):
    """A cache [n_pages, hkv, page / 16, 18 d] of dense k and v [n_pages, hkv, page,
    d]; with `into` and `at` (a mask [n_pages, page]) only those tokens of it."""
    P, H, page, d = k.shape
    cache = torch.zeros(P, H, page // 16, 18 * d, dtype=torch.uint8, device=k.device)
    halves = []
    for x in (k, v):
        c, z, s = quantise(x, dtype)
        c = c.flatten(-2).view(P, H, page // 16, 16, d // 8, 8)[..., ORDER]
        b = (c[..., 0::2] | c[..., 1::2] << 4).flatten(-3).to(torch.uint8)  # [.., 16 * d / 2]
        bits = s.to(torch.bfloat16).view(torch.int16).int() & 0xFFF0 | z.int()
        bits = bits.view(P, H, page // 16, 4, 4, d // 32).permute(0, 1, 2, 5, 4, 3).flatten(3)
        p = torch.stack([bits & 255, bits >> 8 & 255], -1).flatten(3).to(torch.uint8)
        halves.append((b, p))
    new = torch.cat([halves[0][0], halves[1][0], halves[0][1], halves[1][1]], -1)
    if into is None:
        return cache.copy_(new)
    mine = token_bytes(at, H, d)
    into[mine] = new[mine]
    return into


def token_bytes(at, H, d):
    """The bytes [n_pages, H, page / 16, 18 d] of a cache that belong to the tokens
    of the mask at [n_pages, page]."""
    P, page = at.shape
    tok = torch.arange(16, device=at.device)
    codes = tok.repeat_interleave(d // 2)
    # scales: [d / 32, token % 4, token / 4] of two bytes
    i = torch.arange(16, device=at.device)
    scales = (i // 4 + 4 * (i % 4)).repeat(d // 32).repeat_interleave(2)
    owner = torch.cat([codes, codes, scales, scales])
    return at.view(P, 1, page // 16, 16)[..., owner].expand(P, H, page // 16, 18 * d)


def token_values(cache, page_index, head, token, d):
    """The key and the value [d] at one place, byte by byte (for small checks)."""
    b = cache[page_index, head, token // 16].tolist()
    t, out = token % 16, []
    for side in range(2):
        x = []
        for ch in range(d):
            nib = ORDER.index(ch % 8)
            byte = b[side * 8 * d + t * (d // 2) + ch // 8 * 4 + nib // 2]
            at = 16 * d + side * d + 2 * (ch // 32 * 16 + t % 4 * 4 + t // 4)
            bits = b[at] | b[at + 1] << 8
            e = bits >> 7 & 255
            s = math.nan if e == 255 else 0.0 if e == 0 else (1 + (bits >> 4 & 7) / 8) * 2.0 ** (e - 127)
            x.append(((byte >> nib % 2 * 4 & 15) - (bits & 15)) * s)
        out.append(x)
    return out


def turned(x, positions, inv_freq, weight, eps, scaling=1.0):
    """The heads' norm and the rotation of x [n, heads, d] in 64 bits, and the size
    of the terms that make each element up."""
    x = x.double()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    if inv_freq is None:
        return x, x.abs()
    a = (positions.double()[:, None] * inv_freq.double())[:, None]
    c, s = a.cos() * scaling, a.sin() * scaling
    lo, hi = x.chunk(2, -1)
    size = torch.cat([(lo * c).abs() + (hi * s).abs(), (hi * c).abs() + (lo * s).abs()], -1)
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1), size
