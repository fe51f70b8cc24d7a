"""The serving operators in 64 bits, by their definitions, on torch tensors of any device."""
import math

import torch


def padded(dim):
    return -(-dim // 64) * 64


def e4m3_values(codes):
    """Value of every e4m3 byte, from its fields."""
    b = codes.long()
    e, m = b >> 3 & 15, (b & 7).double()
    v = torch.where(e > 0, (8 + m) * torch.exp2((e - 10).double()), m * 2.0 ** -9)
    v = torch.where((b & 127) == 127, torch.nan, v)
    return torch.where(b > 127, -v, v)


def blocks(pool, page, dim):
    """Views of the codes: keys [pages, kv heads, page, padded], values [pages, kv heads, padded, page]."""
    dp = padded(dim)
    return pool[..., :page * dp].unflatten(-1, (page, dp)), pool[..., page * dp:].unflatten(-1, (dp, page))


def sequence_kv(pool, scales, table, length, page, dim):
    """Keys and values [length, kv heads, dim] of one sequence (a row of the page table) in float64."""
    k, v = blocks(pool, page, dim)
    pos = torch.arange(length, device=pool.device)
    pages, off = table.long()[pos // page], pos % page
    s = scales.double()[pages]  # [length, kv heads, 2]
    keys = e4m3_values(k[pages, :, off, :dim]) * s[..., 0, None]
    values = e4m3_values(v[pages, :, :dim, off]) * s[..., 1, None]
    return keys, values


def attention(q, keys, values, positions, scale, window=0, keep=0, missing=None):
    """q [rows, heads, dim] float64; `missing`: truth values of tokens that lie on no page."""
    rows, heads, dim = q.shape
    length, kvh = keys.shape[:2]
    key = torch.arange(length, device=q.device)
    pos = positions[:, None]
    seen = key <= pos
    if window:
        seen &= (key > pos - window) | (key < keep)
    if missing is not None:
        seen &= ~missing
    out = torch.zeros_like(q)
    for h in range(heads):
        g = h * kvh // heads
        s = (q[:, h] @ keys[:, g].t() * scale).masked_fill(~seen, -math.inf)
        m = s.amax(-1, keepdim=True) if length else torch.full((rows, 1), -math.inf, dtype=q.dtype, device=q.device)
        p = torch.exp(s - torch.where(m > -math.inf, m, 0.0))
        p = torch.where(seen, p, 0.0)  # what is not seen may be anything
        total = p.sum(-1, keepdim=True)
        v = torch.where(seen.any(0)[:, None], values[:, g], 0.0)
        out[:, h] = torch.where(total == 0, 0.0, p @ v / torch.where(total == 0, 1.0, total))
    return out


def rotate(x, positions, dims, base):
    out, half = x.clone(), dims // 2
    for i in range(half):
        t = positions.double() * base ** (-2.0 * i / dims)
        c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
        out[..., i] = x[..., i] * c - x[..., i + half] * s
        out[..., i + half] = x[..., i + half] * c + x[..., i] * s
    return out


def block_scale(amax):
    """Smallest power of two >= 2^-100 that keeps amax within 448."""
    fraction, e = math.frexp(float(amax) / 448)
    return max(2.0 ** -100, 2.0 ** (e if fraction > 0.5 else e - 1)) if amax > 0 else 2.0 ** -100


def q4_codes(packed, n, k):
    """Codes 0..15 [n, k] out of the tiles."""
    row, col = torch.arange(n, device=packed.device)[:, None], torch.arange(k, device=packed.device)
    field = col % 8 // 2 + col % 2 * 4
    byte = (row % 8 * 4 + col % 64 // 16) * 16 + row % 16 // 8 * 8 + col % 16 // 8 * 4 + field // 2
    return packed[row // 16, col // 64, byte].long() >> 4 * (field % 2) & 15


def q4_weights(packed, scales, n, k, group):
    col = torch.arange(k, device=packed.device)
    return (q4_codes(packed, n, k) - 8).double() * scales.double()[col // group][:, :n].t()
