"""Attention of the batches that a server forms: many short prompts, one long
sequence ahead of short ones, prompts and decode rows in one call.

Bounds are attn_reference.attention's.  The rows of q differ in range by powers
of two, as the heads of a model do."""
from __future__ import annotations

import pytest
import torch

from attn_reference import attention, make_batch

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
PAIRS = [("fp16", "fp16"), ("bf16", "bf16"), ("fp16", "e4m3"), ("bf16", "e4m3")]


def check(b2g, new, total, hq, hkv, d, page, dtype, cache, window=0, calls=10, seed=5):
    starts, lens, table, pool = make_batch(new, total, page, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    k, v = (torch.randn(pool, page, hkv, d, device="cuda", generator=g).to(TYPES[cache]) for _ in range(2))
    ks = vs = None
    if cache == "e4m3":
        ks, vs = (0.5 + torch.rand(hkv, device="cuda", generator=g) for _ in range(2))
    kv = b2g.PagedCache(k, v, k_scale=ks, v_scale=vs)
    q = torch.randn(sum(new), hq, d, device="cuda", generator=g)
    turn = torch.arange(sum(new), device="cuda")[:, None] // 16 + torch.arange(hq, device="cuda")
    q = (q * 2.0 ** (turn % 7 - 3)[..., None]).to(TYPES[dtype])
    op = b2g.AttnOp(hq, hkv, d, len(new), dtype=dtype, cache_dtype=cache)
    ws, lse = op.workspace(), torch.empty(sum(new), hq, device="cuda")
    first = op.enqueue(q, kv, starts, lens, table, max_q=max(new), window=window, lse=lse, workspace=ws)
    torch.cuda.synchronize()
    assert b2g.device_error() == 0
    want, want_lse, bound = attention(q, k, v, new, total, table, "NHD", ks, vs, None, window)
    err = (first.double() - want).abs()
    assert bool((err <= bound).all()), f"largest error / bound {float((err / bound).max()):.3g}"
    # A score's error (d products in fp32, the scale, 2^x to 2^-18), that of a sum of weights, and one rounding.
    size = q.double().abs().sum(2) * float((k.float().abs().amax() * (1 if ks is None else ks.max()))) * d ** -0.5
    off = (lse.double() - want_lse).abs()
    assert bool((off <= (d + 4) * 2.0 ** -24 * size + 2.0 ** -18 + max(total) * 2.0 ** -24 + 2.0 ** -23 * want_lse.abs()).all())
    for _ in range(calls - 1):
        again = op.enqueue(q, kv, starts, lens, table, max_q=max(new), window=window, workspace=ws)
        assert torch.equal(again, first)
    assert b2g.device_error() == 0


@pytest.mark.parametrize("dtype,cache", PAIRS)
@pytest.mark.parametrize("d", [128, 64])
def test_many_short_prompts(b2g, cuda, dtype, cache, d):
    """More items of one unit than blocks: a block takes several."""
    new = [20 + (i * 37) % 109 for i in range(64)]
    check(b2g, new, new, 32, 8, d, 16, dtype, cache)


@pytest.mark.parametrize("dtype,cache", PAIRS)
def test_short_prompts_behind_a_long_sequence(b2g, cuda, dtype, cache):
    """Split items first, then ones of a single unit."""
    new = [200] + [1 + (i * 53) % 128 for i in range(100)]
    check(b2g, new, [20000] + new[1:], 8, 4, 128, 64, dtype, cache)


@pytest.mark.parametrize("dtype,cache", PAIRS)
def test_prompts_among_decode_rows(b2g, cuda, dtype, cache):
    new = [1 if i % 3 else 70 + i for i in range(60)]
    total = [n + (i * 211) % 900 for i, n in enumerate(new)]
    check(b2g, new, total, 24, 8, 128, 16, dtype, cache)


@pytest.mark.parametrize("dtype,cache", PAIRS)
def test_windows_that_leave_one_unit(b2g, cuda, dtype, cache):
    new = [90 + (i * 17) % 60 for i in range(40)]
    check(b2g, new, [n + (i * 97) % 700 for i, n in enumerate(new)], 16, 8, 64, 32, dtype, cache, window=33)
