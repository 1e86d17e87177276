"""Rotary positions, the paged cache and its attention restated in 64 bits on the CPU, element by element from their definitions."""
from __future__ import annotations

import math

import torch


def inv_freq(pairs, base=10000.0):
    return torch.tensor([base ** (-i / pairs) for i in range(pairs)], dtype=torch.float64)


def rotary(x, positions, freq, sections, interleaved):
    """x [tokens, heads, d]; positions [axes, tokens].  Returns (result, |x| + |y| of each pair at its two places: the scale of
    a rounding of the turn)."""
    x = x.double()
    out, size = x.clone(), torch.zeros_like(x)
    pairs = freq.shape[0]
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    for i in range(pairs):
        a = positions[axis[i]].double() * freq[i]
        re, im = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
        out[..., re], out[..., im] = x[..., re] * c - x[..., im] * s, x[..., re] * s + x[..., im] * c
        size[..., re] = size[..., im] = x[..., re].abs() + x[..., im].abs()
    return out, size


def rotary_tolerance(want, size, dtype):
    """One rounding at the store: half a step relative to the value.  Before it, in 32 bits (half a step is 2^-24): the fraction
    of a turn is at most 1/2, so its rounding moves the angle by at most pi 2^-24; sine and cosine are good to 2 steps (2^-22
    each); two products and a sum round once each.  All of it times |x| + |y|: below (3.2 + 8 + 3) 2^-24."""
    return want.abs() * (torch.finfo(dtype).eps / 2) * (1 + 2.0 ** -10) + size * 16 * 2.0 ** -24 + 1e-30 + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def attention(q, k_cache, v_cache, page_table, q_start, kv_len, scale, window, sinks):
    """Returns (out, sum_j w_j |v_j|, the largest scale * sum_d |q_d k_d|), the first two [tokens, heads, d] (NaN rows: nobody's)."""
    q, kc, vc = q.double(), k_cache.double(), v_cache.double()
    tokens, heads, d = q.shape
    pages, page, kv_heads, _ = kc.shape
    out = torch.full((tokens, heads, d), float("nan"), dtype=torch.float64)
    size = torch.zeros_like(out)
    largest = 0.0
    for b in range(page_table.shape[0]):
        begin, end, length = int(q_start[b]), int(q_start[b + 1]), int(kv_len[b])
        length = max(0, min(length, page_table.shape[1] * page))
        n = end - begin
        for i in range(n):
            pos = length - n + i
            keys = [j for j in range(0, pos + 1) if window == 0 or pos - j < window or j < sinks]
            t = begin + i
            if not keys:
                out[t] = 0.0
                continue
            at = torch.tensor(keys)
            pg = page_table[b].long()[at // page]
            good = (pg >= 0) & (pg < pages)
            kk = torch.where(good[:, None, None], kc[pg.clamp(0, pages - 1), at % page], torch.zeros((), dtype=torch.float64))   # [keys, kv_heads, d]
            vv = torch.where(good[:, None, None], vc[pg.clamp(0, pages - 1), at % page], torch.zeros((), dtype=torch.float64))
            for h in range(heads):
                g = h // (heads // kv_heads)
                s = kk[:, g] @ q[t, h] * scale
                largest = max(largest, float((kk[:, g].abs() @ q[t, h].abs()).max()) * abs(scale))
                w = torch.softmax(s, 0)
                out[t, h] = w @ vv[:, g]
                size[t, h] = w @ vv[:, g].abs()
    return out, size, largest


def attention_tolerance(want, size, largest, dtype):
    """One rounding of the result at the store, one of each weight to the tensors' type before the second product: half a step
    (u) each, relative to the value and to the weighted sum of |v|.  A score is a sum of d products in 32 bits whose steps
    (2^-23, the tensor core cuts off) add up to at most d 2^-23 of sum |q k|; a score that is off by x scales its weight by
    e^x, in the sum of weights as well: twice that.  A quarter of a chunk's exponentials are polynomials whose relative error
    is at most 2^-13.7 (bf16; f32 has none of them) or 2^-18.5 (f16), again in the sum as well: 2^-12.7 and 2^-17.5; the
    hardware's exponential and the sums of weights add 2^-18 for up to some thousand keys.  The weights are taken
    relative to a maximum that may lag by 2^8, which costs no accuracy."""
    u = torch.finfo(dtype).eps / 2
    d = want.shape[-1]
    return want.abs() * u * (1 + 2.0 ** -7) + size * (u + 2 * largest * d * 2.0 ** -23 + (2.0 ** -12.7 if dtype == torch.bfloat16 else 2.0 ** -17.5) + 2.0 ** -18) + 1e-30 + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def make_batch(new, lens, page, kv_heads, d, dtype, seed=0, heads_first=False, spare=2, width=None, fill=None):
    """A pool with random pages for each sequence: (k_cache, v_cache, page_table, q_start, kv_len) on the CPU.  `fill`: what the
    slots hold that no token was written to (default: random leftovers)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    k = torch.randn(pages, page, kv_heads, d, generator=g).to(dtype)
    v = torch.randn(pages, page, kv_heads, d, generator=g).to(dtype)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    width = max(need + [1]) if width is None else width
    table = torch.full((len(new), width), -1, dtype=torch.int32)
    at = 0
    written = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        for j in range(lens[b]):
            written[order[at + j // page], j % page] = True
        at += n
    if fill is not None:
        k[~written], v[~written] = fill, fill
    if heads_first:
        k, v = (t.permute(0, 2, 1, 3).contiguous().transpose(1, 2) for t in (k, v))
    q_start = torch.tensor([0] + list(new)).cumsum(0).to(torch.int32)
    return k, v, table, q_start, torch.tensor(lens, dtype=torch.int32)


def to_device(t, device):
    """A copy with the same strides."""
    out = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=device)
    out.copy_(t)
    return out


def scale_of(d):
    return 1.0 / math.sqrt(d)
