"""Plain restatement of the paged cache's operators on the CPU, for tests: 4-bit quantisation in
fp32 as documented, attention in 64 bits."""

import math

import torch


def rotate(x, positions, table):
    """x bf16 [L, heads, d], positions [L] -> fp32, products and sums rounded one by one."""
    rotary = table.shape[1]
    half = rotary // 2
    x = x.float()
    c, s = table[positions, None, :half], table[positions, None, half:]
    a, b = x[..., :half], x[..., half:rotary]
    return torch.cat((a * c - b * s, b * c + a * s, x[..., rotary:]), -1)


def _codes(x, scale):
    n = torch.where(scale > 0, torch.round(x / scale), torch.zeros_like(x))
    return torch.nan_to_num(n, nan=0.0).clamp(-7, 7)


def int4_keys(x):
    """fp32 [..., d] -> the fp32 values that the 4-bit keys stand for."""
    g = x.unflatten(-1, (-1, 32))
    s = (g.abs().amax(-1, keepdim=True) / 7).to(torch.bfloat16).float()
    return (_codes(g, s) * s).flatten(-2)


def int4_values(x):
    g = x.unflatten(-1, (-1, 32))
    size = g.abs().amax(-1, keepdim=True) / 7
    top = size.amax(-2, keepdim=True)
    bits = (top.view(torch.int32) >> 23) & 255
    e = (bits - 127).clamp(-60, 126)
    up, down = ((e + 127) << 23).view(torch.float32), ((127 - e) << 23).view(torch.float32)
    s = (size * down).to(torch.float16).float() * up
    return (_codes(g, s) * s).flatten(-2)


def attention(q, k, v, position0, scale):
    """q [n, H, d], k / v [T, Hkv, d] -> (out [n, H, d], lse [n, H], weighted mean of |v|, largest weighted |v| of
    one token [n, H]) in 64 bits; row i sees 0 .. position0 + i of the T tokens."""
    n, heads, d = q.shape
    group = heads // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(group, 1), v.double().repeat_interleave(group, 1)
    s = torch.einsum("nhd,thd->nht", q, k) * scale
    seen = torch.arange(k.shape[0])[None] <= position0 + torch.arange(n)[:, None]
    s = s.masked_fill(~seen[:, None], -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None])
    most = (p * v.abs().amax(-1).t()).amax(-1)
    return torch.einsum("nht,thd->nhd", p, v), lse, torch.einsum("nht,thd->nhd", p, v.abs()), most
