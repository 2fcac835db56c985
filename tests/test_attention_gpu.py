"""Attention over a paged cache against plain attention in 64 bits.

The bound on each output is derived in attn_reference.attention before any
run; the log-sums are held to the same score error plus one fp32 rounding."""
from __future__ import annotations

import math

import pytest
import torch

from attn_reference import attention, make_batch

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


def make_cache(b2g, pool, page, hkv, d, cache, layout="NHD", seed=0, fill=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (pool, page, hkv, d) if layout == "NHD" else (pool, hkv, page, d)
    k = torch.randn(shape, device="cuda", generator=g).to(TYPES[cache])
    v = torch.randn(shape, device="cuda", generator=g).to(TYPES[cache])
    ks = vs = None
    if cache == "e4m3":
        ks = 0.5 + torch.rand(hkv, device="cuda", generator=g)
        vs = 0.5 + torch.rand(hkv, device="cuda", generator=g)
    return b2g.PagedCache(k, v, layout, k_scale=ks, v_scale=vs)


def rand_q(rows, hq, d, dtype, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(rows, hq, d, device="cuda", generator=g).to(TYPES[dtype])


def poison(cache, table, total, layout):
    """NaN in every slot that no sequence's length covers."""
    used = torch.zeros(cache.k.shape[0], cache.page_size, dtype=torch.bool, device="cuda")
    for b, t in enumerate(total):
        for i in range(-(-t // cache.page_size)):
            n = min(cache.page_size, t - i * cache.page_size)
            used[int(table[b, i]), :n] = True
    for x in (cache.k, cache.v):
        y = x if layout == "NHD" else x.transpose(1, 2)
        if x.dtype == torch.float8_e4m3fn:
            y.view(torch.uint8)[~used] = 0x7F
        else:
            y[~used] = math.nan


def check(b2g, new, total, hq, hkv, d, page, dtype="fp16", cache="fp16", layout="NHD", window=0, seed=0, max_q="known",
          scale=None, slack=0, q=None):
    starts, lens, table, pool = make_batch(new, total, page, seed=seed)
    kv = make_cache(b2g, pool, page, hkv, d, cache, layout, seed)
    poison(kv, table, total, layout)
    rows = sum(new) + slack
    q = rand_q(rows, hq, d, dtype, seed + 1) if q is None else q
    op = b2g.AttnOp(hq, hkv, d, max_batch=len(new), dtype=dtype, cache_dtype=cache)
    out = torch.full((rows, hq, d), 7.0, dtype=q.dtype, device="cuda")
    lse = torch.full((rows, hq), 7.0, device="cuda")
    ws = op.workspace()
    for _ in range(2):  # the second call finds the workspace as the first one left it
        got = op.enqueue(q, kv, starts, lens, table, max_q=max(max(new), 1) if max_q == "known" else max_q, out=out,
                         lse=lse, window=window, scale=scale, workspace=ws)
        torch.cuda.synchronize()
    assert got is out and b2g.device_error() == 0
    want, want_lse, bound = attention(q[:sum(new)], kv.k, kv.v, new, total, table, layout, kv.k_scale, kv.v_scale, scale,
                                      window)
    n = sum(new)
    err = (out[:n].double() - want).abs()
    assert bool((err <= bound).all()), f"largest error / bound {float((err / bound).max()):.3g}"
    seen = want_lse > -math.inf
    assert bool((lse[:n][~seen] == -math.inf).all())
    off = (lse[:n].double() - want_lse)[seen].abs()
    assert bool((off <= 2.0 ** -16 + 2.0 ** -22 * want_lse[seen].abs()).all())
    assert bool((out[n:] == 7.0).all()) and bool((lse[n:] == 7.0).all())
    return out


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("dtype,cache", [("fp16", "fp16"), ("bf16", "bf16"), ("fp16", "e4m3"), ("bf16", "e4m3")])
def test_decode_types(b2g, cuda, dtype, cache, d):
    check(b2g, [1, 1, 1, 1], [1, 63, 200, 777], 8, 2, d, 16, dtype, cache)


@pytest.mark.parametrize("group", [1, 2, 3, 4, 7, 8, 16, 32])
def test_groups(b2g, cuda, group):
    check(b2g, [1, 2], [130, 65], 2 * group, 2, 128, 16)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 17, 64, 128, 1000])
def test_page_sizes(b2g, cuda, page):
    check(b2g, [1, 3, 1], [5, 300, 129], 4, 2, 128, page)


@pytest.mark.parametrize("cache", ["fp16", "e4m3"])
def test_heads_before_tokens(b2g, cuda, cache):
    check(b2g, [1, 2, 30], [90, 300, 129], 6, 2, 128, 32, "fp16", cache, layout="HND")


@pytest.mark.parametrize("window", [1, 2, 16, 100, 4096])
def test_window(b2g, cuda, window):
    check(b2g, [1, 4, 2, 40], [1, 500, 129, 300], 4, 2, 128, 16, window=window)


@pytest.mark.parametrize("max_q", ["known", None, 1])
def test_ragged_chunks(b2g, cuda, max_q):
    check(b2g, [5, 1, 0, 17, 33, 3], [5, 700, 40, 17, 400, 64], 6, 2, 128, 16, max_q=max_q, slack=3)


@pytest.mark.parametrize("dtype,cache,d", [("fp16", "fp16", 128), ("bf16", "bf16", 128), ("fp16", "e4m3", 128),
                                           ("bf16", "e4m3", 64), ("fp16", "fp16", 64)])
@pytest.mark.parametrize("n", [100, 128, 257, 700])
def test_prompt_chunks(b2g, cuda, dtype, cache, d, n):
    check(b2g, [n, n // 3], [n, n + 333], 8, 2, d, 16, dtype, cache)


def test_prompt_window(b2g, cuda):
    check(b2g, [300, 200], [300, 900], 8, 2, 128, 64, "bf16", "bf16", window=150)


def test_rows_that_see_nothing(b2g, cuda):
    """More new rows than the length counts: the first ones lie before the
    sequence's start; a length of zero leaves every row empty."""
    check(b2g, [4, 3, 40], [2, 0, 10], 4, 2, 128, 16)
    check(b2g, [200], [100], 4, 2, 128, 16)


def test_many_sequences(b2g, cuda):
    new = [1 + i % 2 for i in range(300)]
    total = [n + (i * 37) % 200 for i, n in enumerate(new)]
    check(b2g, new, total, 4, 2, 64, 16)


def test_long_context_split_over_blocks(b2g, cuda):
    check(b2g, [1], [40001], 8, 1, 128, 64)
    check(b2g, [2, 1], [30000, 3], 8, 2, 128, 64, "bf16", "e4m3")


def test_long_context_chunk(b2g, cuda):
    check(b2g, [130], [20000], 4, 1, 128, 64, "bf16", "bf16")


def test_large_scores(b2g, cuda):
    """Scores in the thousands: the running maximum moves often, weights are
    close to one and zero."""
    g = torch.Generator(device="cuda").manual_seed(9)
    q = (torch.randn(3, 4, 128, device="cuda", generator=g) * 100).half()
    check(b2g, [1, 2], [500, 300], 4, 2, 128, 16, q=q)


def test_bf16_rows_out_of_fp16_range_over_8bit_cache(b2g, cuda):
    g = torch.Generator(device="cuda").manual_seed(9)
    q = (torch.randn(3, 4, 128, device="cuda", generator=g) * 1e6).bfloat16()
    check(b2g, [1, 2], [50, 30], 4, 2, 128, 16, "bf16", "e4m3", q=q, scale=1e-6)
    q = (torch.randn(40, 4, 128, device="cuda", generator=g) * 1e-8).bfloat16()
    check(b2g, [40], [130], 4, 2, 128, 16, "bf16", "e4m3", q=q, scale=1e7)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("cache", ["fp16", "e4m3"])
def test_offsets_beyond_32_bits(b2g, cuda, new, cache):
    """Two pages 34 GB apart: beyond 2^32 elements, and 2^31 pieces of 16 bytes."""
    d, page, total = 128, 16, 24
    size = 1 if cache == "e4m3" else 2
    gap = (34 << 30) // size  # elements
    buf = torch.empty(gap * size + (1 << 20), dtype=torch.uint8, device="cuda").view(TYPES[cache])
    shape, strides = (2, page, 2, d), (gap, 4 * d, d, 1)
    k, v = buf.as_strided(shape, strides), buf.as_strided(shape, strides, 2 * d)
    kv = b2g.PagedCache(k, v)
    starts, lens, table = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, total], [total], [[1, 0]]))
    x = torch.randn(total, 2, 2, d, device="cuda").half()
    b2g.kv_append(x[:, 0], x[:, 1], kv, starts, lens, table)
    q = rand_q(new, 4, d, "fp16")  # 40 new rows: the first 16 lie before the start
    starts = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    op = b2g.AttnOp(4, 2, d, 1, cache_dtype=cache)
    out = op.enqueue(q, kv, starts, lens, table, max_q=new)
    torch.cuda.synchronize()
    assert b2g.device_error() == 0
    small = [torch.stack([c[0], c[1]]).contiguous() for c in (k.view(torch.uint8) if size == 1 else k,
                                                             v.view(torch.uint8) if size == 1 else v)]
    small = [c.view(TYPES[cache]) for c in small]
    want, _, bound = attention(q, *small, [new], [total], table)
    assert bool(((out.double() - want).abs() <= bound).all())
    del buf, k, v, kv
    torch.cuda.empty_cache()


def test_strided_q_and_out(b2g, cuda):
    """q and out inside wider rows, as a fused projection leaves them."""
    hq, hkv, d, n = 4, 2, 128, 5
    starts, lens, table, pool = make_batch([n, 1], [n + 20, 9], 16)
    kv = make_cache(b2g, pool, 16, hkv, d, "fp16")
    wide = torch.randn(n + 1, hq + 2 * hkv, d, device="cuda").half()
    q = wide[:, :hq]
    res = torch.zeros(n + 1, 2 * hq, d, device="cuda", dtype=torch.float16)
    op = b2g.AttnOp(hq, hkv, d, 2)
    op.enqueue(q, kv, starts, lens, table, out=res[:, hq:])
    want, _, bound = attention(q, kv.k, kv.v, [n, 1], [n + 20, 9], table)
    assert bool(((res[:, hq:].double() - want).abs() <= bound).all())
    assert bool((res[:, :hq] == 0).all())


@pytest.mark.parametrize("new", [1, 60])
def test_bad_pages_are_not_read(b2g, cuda, new):
    """A table entry outside the cache: its tokens are not seen, the error word is set."""
    starts, lens, table, pool = make_batch([new], [100], 16)
    kv = make_cache(b2g, pool, 16, 2, 128, "fp16")
    q = rand_q(new, 4, 128, "fp16")
    op = b2g.AttnOp(4, 2, 128, 1)
    for bad in (-1, pool, 2 ** 31 - 1):
        broken = table.clone()
        broken[0, 1] = bad  # tokens 16..31
        out = op.enqueue(q, kv, starts, lens, broken, max_q=new)
        torch.cuda.synchronize()
        assert b2g.device_error() == 6
        k, v = (x[table[0].long()].flatten(0, 1)[:100].double() for x in (kv.k, kv.v))
        pos = torch.arange(100 - new, 100, device="cuda")[:, None]
        j = torch.arange(100, device="cuda")[None]
        hidden = (j > pos) | ((j >= 16) & (j < 32))
        for h in range(4):
            s = (q[:, h].double() @ k[:, h // 2].T * 128 ** -0.5).masked_fill(hidden, -math.inf)
            want = torch.softmax(s, 1) @ v[:, h // 2]
            assert float((out[:, h].double() - want).abs().max()) <= 2e-2
    assert b2g.device_error() == 0


def test_length_past_the_table(b2g, cuda):
    starts, lens, table, pool = make_batch([1], [32], 16)
    kv = make_cache(b2g, pool, 16, 2, 128, "fp16")
    q = rand_q(1, 4, 128, "fp16")
    op = b2g.AttnOp(4, 2, 128, 1)
    out = op.enqueue(q, kv, starts, lens + 100, table)
    torch.cuda.synchronize()
    assert b2g.device_error() == 6
    assert bool(out.isfinite().all())


@pytest.mark.parametrize("new", [1, 50])
def test_captured_and_replayed_with_other_lengths(b2g, cuda, new):
    total = [300, 40 + new]
    starts, lens, table, pool = make_batch([new, new], total, 16)
    kv = make_cache(b2g, pool, 16, 2, 128, "bf16")
    q = rand_q(2 * new, 8, 128, "bf16")
    op = b2g.AttnOp(8, 2, 128, 2, dtype="bf16")
    ws = op.workspace()
    out = torch.empty_like(q)
    op.enqueue(q, kv, starts, lens, table, max_q=new, out=out, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        op.enqueue(q, kv, starts, lens, table, max_q=new, out=out, workspace=ws)
    for a, b in ((300, 40 + new), (new, new), (123, 31 + new)):
        a = max(a, new)
        lens.copy_(torch.tensor([a, b], dtype=torch.int32))
        out.fill_(0)
        g.replay()
        torch.cuda.synchronize()
        want, _, bound = attention(q, kv.k, kv.v, [new, new], [a, b], table)
        assert bool(((out.double() - want).abs() <= bound).all())
    assert b2g.device_error() == 0


def test_two_streams_with_a_workspace_each(b2g, cuda):
    starts, lens, table, pool = make_batch([1] * 4, [900, 20, 300, 64], 16)
    kv = make_cache(b2g, pool, 16, 2, 128, "fp16")
    op = b2g.AttnOp(8, 2, 128, 4)
    q = rand_q(4, 8, 128, "fp16")
    want = op.enqueue(q, kv, starts, lens, table, max_q=1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(20):
        outs.append(op.enqueue(q, kv, starts, lens, table, max_q=1, stream=streams[i % 2]))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)


def test_same_call_same_bits(b2g, cuda):
    """Parts are joined in one order: repeated calls agree to the last bit."""
    starts, lens, table, pool = make_batch([1, 1, 90], [20000, 5, 700], 64)
    kv = make_cache(b2g, pool, 64, 2, 128, "fp16")
    q = rand_q(92, 8, 128, "fp16")
    op = b2g.AttnOp(8, 2, 128, 3)
    ws = op.workspace()
    for max_q in (1, 90):
        first = op.enqueue(q, kv, starts, lens, table, max_q=max_q, workspace=ws)
        for _ in range(5):
            assert torch.equal(op.enqueue(q, kv, starts, lens, table, max_q=max_q, workspace=ws), first)


def test_refusals(b2g, cuda):
    starts, lens, table, pool = make_batch([1], [32], 16)
    kv = make_cache(b2g, pool, 16, 2, 128, "fp16")
    q = rand_q(1, 4, 128, "fp16")
    op = b2g.AttnOp(4, 2, 128, 1)
    with pytest.raises(ValueError):
        op.enqueue(q.bfloat16(), kv, starts, lens, table)
    with pytest.raises(ValueError):
        op.enqueue(q, kv, starts.long(), lens, table)
    with pytest.raises(ValueError):
        op.enqueue(q, kv, starts, lens, table.cpu())
    with pytest.raises(ValueError):
        op.enqueue(q, kv, starts, lens, table, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(b2g.B2GError):
        op.enqueue(q, kv, starts, lens, table, window=-1)
    with pytest.raises(b2g.B2GError):
        op.enqueue(q, make_cache(b2g, pool, 16, 2, 128, "e4m3"), starts, lens, table)
    with pytest.raises(b2g.B2GError):
        b2g.AttnOp(4, 2, 128, 1).enqueue(torch.cat([q, q]), kv, torch.cat([starts, starts[:1] + 2]),
                                         torch.cat([lens, lens]), torch.cat([table, table]))
