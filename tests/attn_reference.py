"""Plain attention over a paged cache in 64 bits, with the error that the
kernels' roundings can make of it (shared by the attention tests)."""
from __future__ import annotations

import math

import torch


def make_batch(new, total, page, extra_pages=0, seed=0, slack_rows=0, device="cuda"):
    """q_start, seq_lens, page_table (entries in a random order, -1 behind the
    last) and the number of pages, for `new` new tokens of `total`."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-t // page) for t in total]
    pool = sum(pages) + 1 + extra_pages
    order = torch.randperm(pool, generator=g).to(torch.int32)
    table = torch.full((len(new), max(max(pages), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    starts = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32)
    lens = torch.tensor(total, dtype=torch.int32)
    return starts.to(device), lens.to(device), table.to(device), pool


def gather(cache, table_row, tokens, layout):
    """[tokens, heads, dim] in 64 bits of one sequence."""
    c = cache if layout == "NHD" else cache.transpose(1, 2)
    bits = c.view(torch.uint8) if c.dtype == torch.float8_e4m3fn else c
    page = c.shape[1]
    need = -(-tokens // page)
    x = bits[table_row[:need].long()].flatten(0, 1)[:tokens]
    return (x.view(c.dtype) if bits is not c else x).double()


def attention(q, k_cache, v_cache, new, total, table, layout="NHD", k_scale=None, v_scale=None, scale=None, window=0):
    """(out, lse, bound): out [rows, heads, dim] float64 with zeros where a row
    sees nothing; bound is what out may be off by.

    With w the softmax weights, A = sum w |v|, u the half step of the type
    that holds the probabilities and r that of out:
      probabilities rounded once:  u A, and at most 2^-25 each below fp16's
                                   normal range (the largest is 1): 2^-25 sum |v| / l
      a score's error e (dot of n products in fp32, scale, 2^x to 2^-18) moves
      a weight by at most 2 e:     2 e A
      sums of weights and of products over the tokens in fp32: tokens 2^-24 A
      the result rounded:          r |out|
    """
    rows, heads, d = q.shape
    kv_heads = k_cache.shape[2 if layout == "NHD" else 1]
    group = heads // kv_heads
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(rows, heads, d, dtype=torch.float64, device=q.device)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    e4m3 = k_cache.dtype == torch.float8_e4m3fn
    u = (torch.finfo(torch.float16 if e4m3 else q.dtype).eps) / 2
    r = torch.finfo(q.dtype).eps / 2
    at = 0
    for b, (n, t) in enumerate(zip(new, total)):
        own = slice(at, at + n)
        at += n
        if n == 0 or t == 0:
            continue
        k, v = gather(k_cache, table[b], t, layout), gather(v_cache, table[b], t, layout)
        if e4m3:
            k = k * (1 if k_scale is None else k_scale.double()[:, None])
            v = v * (1 if v_scale is None else v_scale.double()[:, None])
        pos = torch.arange(t - n, t, device=q.device)[:, None]
        j = torch.arange(t, device=q.device)[None]
        sees = j <= pos
        if window:
            sees &= j > pos - window
        any_ = sees.any(1)
        for h in range(heads):
            qq, kk, vv = q[own, h].double(), k[:, h // group], v[:, h // group]
            s = (qq @ kk.T * scale).masked_fill(~sees, -math.inf)
            lse[own, h] = torch.logsumexp(s, 1)
            w = torch.softmax(s, 1).masked_fill(~sees, 0)
            w[~any_] = 0
            vv = vv.masked_fill(~sees.any(0)[:, None], 0)
            o = w @ vv
            out[own, h] = o
            mag = (qq.abs() @ kk.abs().T * scale).masked_fill(~sees, 0).amax(1, keepdim=True)
            e = (d + 4) * 2.0 ** -24 * mag + 2.0 ** -18
            a = w @ vv.abs()
            ell = torch.exp(lse[own, h] - s.amax(1))[:, None].nan_to_num(1.0).clamp(min=1.0)
            small = 2.0 ** -25 * (sees.double() @ vv.abs()) / ell if u < 2.0 ** -9 else 0
            bound[own, h] = u * a + small + 2 * e * a + t * 2.0 ** -24 * a + r * o.abs() + 2.0 ** -24
    return out, lse, bound
