"""Definitions in 64 bits of the 8-bit KV cache and of the 8-bit integer projection (plain torch on any device).

A cache is a dict with ``fmt`` ("int8" | "e4m3"), ``block``, ``k``, ``v`` (codes as float64 numbers ``[B,KVH,rows,d]``) and
``ks``, ``vs`` (float64 scales ``[B,KVH,blocks]``)."""
import math

import torch

TOP = {"int8": 127.0, "e4m3": 448.0}


def nearest(y, fmt):
    """Nearest number of the format (ties to even); the caller keeps |y| within the format's range."""
    if fmt == "int8":
        return torch.round(y)
    mag = y.abs().clamp(min=2.0 ** -12)
    step = torch.exp2(torch.floor(torch.log2(mag)).clamp(min=-6.0) - 3.0)
    return torch.round(y / step) * step


def half_step(y, fmt):
    """Largest distance of a nearest number from y."""
    if fmt == "int8":
        return torch.full_like(y, 0.5)
    return torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -12))).clamp(min=-6.0) - 4.0)


def quantise(x, block, fmt):
    """x float64 ``[..., n, d]`` -> (codes, scales ``[..., ceil(n / block)]``)."""
    n, d = x.shape[-2:]
    nb = -(-n // block)
    codes, scales = torch.zeros_like(x), torch.zeros(*x.shape[:-2], nb, dtype=torch.float64, device=x.device)
    for j in range(nb):
        rows = x[..., j * block:(j + 1) * block, :]
        a = rows.abs().amax((-1, -2))
        scales[..., j] = a / TOP[fmt]
        live = (a > 0) & torch.isfinite(a)
        y = rows * TOP[fmt] / torch.where(live, a, torch.ones_like(a))[..., None, None]
        codes[..., j * block:(j + 1) * block, :] = torch.where(live[..., None, None], nearest(y, fmt), torch.zeros_like(y))
    return codes, scales


def values(codes, scales, block):
    n = codes.shape[-2]
    return codes * scales.repeat_interleave(block, -1)[..., :n, None]


def append(codes, scales, new, pos, block, fmt):
    """One (sequence, head): codes ``[rows, d]``, scales ``[blocks]``, new ``[d]``.  Returns what the rounding acts on as
    well: (codes, scales, unrounded codes of the block's rows up to pos)."""
    codes, scales = codes.clone(), scales.clone()
    j, first = pos // block, pos // block * block
    s0 = scales[j].item() if pos % block else 0.0
    want = new.abs().max().item() / TOP[fmt]
    s1 = max(s0, want)
    raw = codes[first:pos + 1].clone()
    if want > s0:
        raw[:-1] = raw[:-1] * (s0 / s1)
    raw[-1] = new / s1 if s1 > 0 else torch.zeros_like(new)
    codes[first:pos + 1] = nearest(raw, fmt)
    scales[j] = s1
    return codes, scales, raw


def attention(q, k, v, rows, scale=None):
    """One sequence: q ``[H,d]``, k, v ``[KVH,n,d]``, the positions ``rows``.  Returns (out ``[H,d]``, sum of weight x |v|
    ``[H,d]``, logits ``[H,len(rows)]``, sum of |q||k| x scale, the largest)."""
    H, d = q.shape
    G = H // k.shape[0]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    if len(rows) == 0:
        z = torch.zeros_like(q)
        return z, z, torch.zeros(H, 0, dtype=q.dtype, device=q.device), 0.0
    kk, vv = k[:, rows].repeat_interleave(G, 0), v[:, rows].repeat_interleave(G, 0)
    logits = torch.einsum("hd,hnd->hn", q, kk) * scale
    size = (torch.einsum("hd,hnd->hn", q.abs(), kk.abs()) * scale).max().item()
    p = torch.softmax(logits, 1)
    return torch.einsum("hn,hnd->hd", p, vv), torch.einsum("hn,hnd->hd", p, vv.abs()), logits, size


def linear(x8, sx, w8, sw, residual=None):
    y = (x8.double() @ w8.double().t()) * sx.double()[:, None] * sw.double()[None]
    return y if residual is None else y + residual.double()
