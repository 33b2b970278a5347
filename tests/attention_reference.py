"""The attention half of a decoder layer in 64 bits on the CPU, straight from the formulas (torch for indexing and products)."""
from __future__ import annotations

import math

import numpy as np
import torch


def rms(x, weight, eps):
    x = x.double()
    return x if weight is None else x * weight.double() / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)


def rotate(x, positions, inv_freq, interleaved, amplitude):
    """x [rows][heads][dim] (64 bits)."""
    n = inv_freq.numel()
    y = x.clone()
    for i in range(n):
        t = positions.double() * inv_freq[i]
        c, s = (amplitude * t.cos())[:, None], (amplitude * t.sin())[:, None]
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def quantise(x):
    """[..., dim] -> (codes 0..15 in dimension order, FP16 scales [..., dim / 32]), from 64 bits."""
    g = x.double().unflatten(-1, (-1, 32))
    scales = torch.from_numpy((g.abs().amax(-1).numpy() / 7).astype(np.float16))
    s = scales.double()[..., None]
    codes = torch.where(s > 0, torch.round(g / s).clamp(-7, 7), 0.0).flatten(-2).to(torch.int64) + 8
    return codes, scales


def dequantise(codes, scales):
    return (codes.double() - 8) * scales.double().repeat_interleave(32, -1)


def word_order(dim):
    """Dimension held by nibble n of a stored row, n = 0 .. dim - 1."""
    groups = dim // 32
    return torch.tensor([32 * (w % groups) + 8 * (w // groups) + i for w in range(dim // 8) for i in range(8)])


def store(pool, page, head, slot, page_size, k, v):
    """Writes one token's K and V values (64 bits, [dim]) into a CPU pool, quantised."""
    dim = k.numel()
    block = pool[page, head]
    at = 0
    for x in (k, v):
        codes, scales = quantise(x)
        nibbles = codes[word_order(dim)]
        block[at + slot * dim // 2:at + (slot + 1) * dim // 2] = (nibbles[0::2] | nibbles[1::2] << 4).to(torch.uint8)
        at += page_size * dim // 2
        block[at + slot * dim // 16:at + (slot + 1) * dim // 16] = scales.view(torch.uint8)
        at += page_size * dim // 16


def fetch(pool, page, page_size, dim):
    """K and V values of all slots of a page, [kv_heads][page_size][dim] in 64 bits."""
    out, at = [], 0
    for _ in range(2):
        codes = pool[page, :, at:at + page_size * dim // 2].reshape(-1, page_size, dim // 2)
        at += page_size * dim // 2
        scales = pool[page, :, at:at + page_size * dim // 16].contiguous().view(torch.float16).reshape(-1, page_size, dim // 32)
        at += page_size * dim // 16
        nibbles = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).to(torch.int64)
        values = torch.empty_like(nibbles)
        values[..., word_order(dim)] = nibbles
        out.append(dequantise(values, scales))
    return out


def tokens(pool, table_row, context, page_size, dim):
    """K and V of a sequence, [context][kv_heads][dim]."""
    if not context:
        z = torch.zeros((0, pool.shape[1], dim), dtype=torch.float64)
        return z, z
    got = [fetch(pool, int(p), page_size, dim) for p in table_row[:-(-context // page_size)]]
    return tuple(torch.cat([g[i] for g in got], 1).transpose(0, 1)[:context] for i in range(2))


def attention(q, k, v, first, scale, window):
    """One sequence: q [rows][heads][dim] at positions first, first + 1, ...; returns (out, bound) where bound is what an element may be off
    through the kernels' arithmetic: weights p are FP16 (twice rounded where V's scale is multiplied in, 2 * 2^-11), K and V values may
    be FP16 (2^-11 each, K's through the score: scale * sum |q k| * 2^-11), sums are 32 bits (well below these).  A relative error
    d_t of the weights moves sum(p v) / sum(p) by at most 2 max(d) sum(p |v|)."""
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for r in range(rows):
        at = first + r
        low = max(0, at - window + 1) if window else 0
        if at < 0:
            continue
        ks, vs = (x[low:at + 1].repeat_interleave(group, 1) for x in (k, v))
        x = q[r].double()
        score = scale * (ks * x).sum(-1)
        size = abs(scale) * (ks.abs() * x.abs()).sum(-1).amax(0)
        p = torch.softmax(score, 0)[..., None]
        out[r] = (p * vs).sum(0)
        bound[r] = (2 * (2 * 2 ** -11 + 2 ** -11 + 2 ** -11 * size)[:, None]) * (p * vs.abs()).sum(0)
    return out, bound


def yarn_like(n, factor):
    f = 10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)
    return f / factor, 1 + 0.1 * math.log(factor)


def fill(pool, table_row, page_size, k, v):
    """Writes a whole sequence, k and v [tokens][kv_heads][dim] in 64 bits, into a CPU pool, quantised."""
    count, dim = k.shape[0], k.shape[2]
    t = torch.arange(count)
    page, slot = table_row[t // page_size].long(), t % page_size
    at = 0
    for x in (k, v):
        codes, scales = quantise(x)
        nibbles = codes[..., word_order(dim)]
        for data, width in (((nibbles[..., 0::2] | nibbles[..., 1::2] << 4).to(torch.uint8), dim // 2), (scales.contiguous().view(torch.uint8), dim // 16)):
            part = pool[:, :, at:at + page_size * width].unflatten(-1, (page_size, width))
            part[page, :, slot] = data
            at += page_size * width


def marked(rows, context, dim):
    """A sequence that tells which 32 tokens were attended to: V is 7 in dimension (t / 32) % dim and zero elsewhere, and the score of token t
    (for a query that is 1 in dimension 0 and zero elsewhere, scale ln 2) is t / 1024 % 3 in the exponent of two.  Returns k, v [context][dim] and
    the output [rows][dim]; all weights are powers of two and all products exact."""
    t = torch.arange(context)
    k, v = torch.zeros((context, dim), dtype=torch.float64), torch.zeros((context, dim), dtype=torch.float64)
    k[:, 0], k[:, 1] = (t // 1024 % 3).double(), 7.0  # the group's scale is one
    v[t, t // 32 % dim] = 7.0
    weight = (t <= torch.arange(context - rows, context)[:, None]) * 2.0 ** k[:, 0]
    return k, v, weight @ v / weight.sum(1, keepdim=True)
