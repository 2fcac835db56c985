"""The operators as they are used together: prompts of several sequences
through AttentionBlock (normalised rows, 8-bit products, append with rotation,
attention, residual), then decode steps through a captured graph of the block
and the MLP stack, against the same layer in 64 bits.

The reference quantises its rows as the library does.  What differs is the
16-bit rounding between the operators (2^-11 relative each): in units of a
code (up to 127) that moves a value by at most 0.06, on average by 0.01, so
about one code in a hundred falls to its neighbour, an error of 0.1 codes rms
against codes of about 40 rms: 2.5e-3 of a product, two products, the E4M3
stack at its own 5e-3: 1.5e-2 of an update's norm bounds their sum."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HIDDEN, HQ, HKV, D, PAGE, INTER = 512, 8, 2, 64, 16, 1024
TOL = 1.5e-2


def quantised(v):
    s = v.abs().amax(1, keepdim=True).clamp(min=1e-12) / 127
    return torch.round(v / s) * s


def norm(h, gamma):
    return h * torch.rsqrt(h.square().mean(1, keepdim=True) + 1e-5) * gamma


def rotate(x, pos, freq):
    a = pos.double()[:, None] * freq.double()
    c, s = a.cos()[:, None], a.sin()[:, None]
    lo, hi = x[..., :D // 2], x[..., D // 2:]
    return torch.cat((lo * c - hi * s, hi * c + lo * s), -1)


def layer(h, new, seqs, wqkv, wo, gamma, freq):
    """h + attention block in 64 bits; seqs: each sequence's (k, v), extended."""
    x = quantised(norm(h, gamma)) @ wqkv.T
    x = x.view(-1, HQ + 2 * HKV, D)
    out = torch.zeros(h.shape[0], HQ, D, dtype=torch.float64, device=h.device)
    at = 0
    for b, n in enumerate(new):
        own = slice(at, at + n)
        at += n
        before = seqs[b][0].shape[0]
        pos = torch.arange(before, before + n, device=h.device)
        q, k, v = x[own].split((HQ, HKV, HKV), 1)
        q, k = rotate(q, pos, freq), rotate(k, pos, freq)
        seqs[b] = (torch.cat((seqs[b][0], k)), torch.cat((seqs[b][1], v)))
        kk, vv = (t.repeat_interleave(HQ // HKV, 1) for t in seqs[b])
        s = torch.einsum("nhd,jhd->hnj", q, kk) / math.sqrt(D)
        j = torch.arange(kk.shape[0], device=h.device)
        s = s.masked_fill(j[None] > pos[:, None], -math.inf)
        out[own] = torch.einsum("hnj,jhd->nhd", torch.softmax(s, -1), vv)
    return h + quantised(out.flatten(1)) @ wo.T



@pytest.mark.parametrize("cache", ["fp16", "fp8_e4m3"])
def test_prompts_then_decode_steps(b2g, cuda, cache):
    g = torch.Generator(device="cuda").manual_seed(3)

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).half()

    wqkv = b2g.quantize_i8_weights(rand((HQ + 2 * HKV) * D, HIDDEN, scale=HIDDEN ** -0.5), "NK")
    wo = b2g.quantize_i8_weights(rand(HQ * D, HIDDEN, scale=(HQ * D) ** -0.5), "KN")
    gamma = (1 + rand(HIDDEN, scale=0.1))
    freq = (10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) * 2 / D)).float().cuda()
    dq = [w[0].double() * w[1].double()[:, None] for w in (wqkv, wo)]
    block = b2g.AttentionBlock(HIDDEN, HQ, HKV, D, max_rows=128, max_batch=3, wqkv=wqkv, wo=wo, inv_freq=freq,
                               gamma=gamma, cache_dtype=cache)
    pool = 24
    kc, vc = (torch.full((pool, PAGE, HKV, D), math.nan, device="cuda", dtype=torch.float16) for _ in range(2))
    if cache == "fp8_e4m3":
        kc, vc = (torch.full((pool, PAGE, HKV, D), 0x7F, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
                  for _ in range(2))
    paged = b2g.PagedCache(kc, vc)
    table = torch.randperm(pool, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(3, 8).cuda()
    ws = block.workspace()
    # 8-bit keys and values: half a step of 2^-4 each, averaged over the tokens
    tol = TOL if cache == "fp16" else 6e-2

    new = [37, 5, 70]
    h = rand(sum(new), HIDDEN)
    seqs = [(torch.zeros(0, HKV, D, dtype=torch.float64, device="cuda"),) * 2 for _ in new]
    base = h.double()
    want = layer(base, new, seqs, *dq, gamma.double(), freq)
    starts = torch.tensor([0, 37, 42, 112], dtype=torch.int32, device="cuda")
    lens = torch.tensor(new, dtype=torch.int32, device="cuda")
    out = block.enqueue(h, paged, starts, lens, table, ws, max_q=70)
    torch.cuda.synchronize()
    assert out is h and b2g.device_error() == 0
    assert float((h.double() - want).norm() / (want - base).norm()) <= tol

    stack = b2g.Stack(HIDDEN, INTER, 1, max_m=8)
    mlp = []
    packed = []
    for K, N in ((HIDDEN, INTER), (HIDDEN, INTER), (INTER, HIDDEN)):
        q, s = b2g.quantize_e4m3(rand(K, N, scale=K ** -0.5), "channel_fp32")
        packed.append((q, s))
        mlp.append(q.view(torch.float8_e4m3fn).double() * s.double())
    stack.set_layer(0, stack.gate_up.prepack(packed[0][0], packed[1][0]), torch.cat([packed[0][1], packed[1][1]]),
                    stack.down.prepack(packed[2][0]), packed[2][1])
    act, sws = torch.empty(3, INTER, dtype=torch.float16, device="cuda"), stack.workspace("cuda")
    h = torch.zeros(3, HIDDEN, dtype=torch.float16, device="cuda")
    one = torch.arange(4, dtype=torch.int32, device="cuda")

    def step():
        block.enqueue(h, paged, one, lens, table, ws, max_q=1)
        stack.enqueue(h, act, sws)

    graph = None
    for i in range(4):
        x = rand(3, HIDDEN)
        h.copy_(x)
        lens += 1
        base = x.double()
        mid = layer(base, [1, 1, 1], seqs, *dq, gamma.double(), freq)
        n = norm(mid, torch.ones((), dtype=torch.float64, device="cuda"))
        gate, up = n @ mlp[0], n @ mlp[1]
        want = mid + (gate * torch.sigmoid(gate) * up) @ mlp[2]
        if i < 2:
            step()
        else:  # the same buffers, other lengths: a captured step
            if graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    step()
                h.copy_(x)
            graph.replay()
        torch.cuda.synchronize()
        assert b2g.device_error() == 0
        assert float((h.double() - want).norm() / (want - base).norm()) <= tol


@pytest.mark.parametrize("cache", ["bf16", "fp8_e4m3"])
def test_prompts_and_decode_rows_in_one_call(b2g, cuda, cache):
    """bf16, calls that hold prompts, decode rows or both, a sequence without a row
    among them.  Roundings between the operators are 2^-8 where fp16's are 2^-11: a
    value moves by half a code at most and 0.08 on average, so eight codes in a
    hundred fall to their neighbour, 0.28 codes rms of about 40: 7e-3 a product,
    with the 2^-8 of q, k, v and of the probabilities under 4e-2 of an update; h
    itself is rounded once.  8-bit keys and values: 6e-2 as above, sqrt of the
    squares' sum."""
    g = torch.Generator(device="cuda").manual_seed(8)

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).bfloat16()

    wqkv = b2g.quantize_i8_weights(rand((HQ + 2 * HKV) * D, HIDDEN, scale=HIDDEN ** -0.5), "NK")
    wo = b2g.quantize_i8_weights(rand(HQ * D, HIDDEN, scale=(HQ * D) ** -0.5), "KN")
    gamma = 1 + rand(HIDDEN, scale=0.1)
    freq = (10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) * 2 / D)).float().cuda()
    dq = [w[0].double() * w[1].double()[:, None] for w in (wqkv, wo)]
    block = b2g.AttentionBlock(HIDDEN, HQ, HKV, D, max_rows=256, max_batch=4, wqkv=wqkv, wo=wo, inv_freq=freq,
                               gamma=gamma, dtype="bf16", cache_dtype=cache)
    pool = 64
    kind = torch.bfloat16 if cache == "bf16" else torch.float8_e4m3fn
    paged = b2g.PagedCache(*(torch.zeros(pool, PAGE, HKV, D, device="cuda").to(kind) for _ in range(2)))
    table = torch.randperm(pool, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(4, 16).cuda()
    ws = block.workspace()
    tol = 4e-2 if cache == "bf16" else 7.2e-2
    seqs = [(torch.zeros(0, HKV, D, dtype=torch.float64, device="cuda"),) * 2 for _ in range(4)]
    for new in ([90, 3, 40, 0], [1, 60, 1, 20], [1, 1, 0, 100], [1, 1, 1, 1]):
        h = rand(sum(new) + 2, HIDDEN)  # two rows behind the last sequence
        base = h[:sum(new)].double()
        want = layer(base, new, seqs, *dq, gamma.double(), freq)
        starts = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
        lens = torch.tensor([k.shape[0] for k, _ in seqs], dtype=torch.int32, device="cuda")
        block.enqueue(h, paged, starts, lens, table, ws, max_q=max(new))
        torch.cuda.synchronize()
        assert b2g.device_error() == 0
        off = h[:sum(new)].double() - want
        assert float(off.norm()) <= tol * float((want - base).norm()) + 2.0 ** -8 * float(want.norm())


def test_out_over_q(b2g, cuda):
    """AttnOp's out may be q itself, split items among them."""
    from attn_reference import attention, make_batch
    for new, total in (([1, 1], [9000, 5]), ([150, 3], [3000, 30])):
        starts, lens, table, pool = make_batch(new, total, 64)
        kv = b2g.PagedCache(*(torch.randn(pool, 64, 2, 128, device="cuda").half() for _ in range(2)))
        q = torch.randn(sum(new), 8, 128, device="cuda").half()
        want, _, bound = attention(q, kv.k, kv.v, new, total, table)
        op = b2g.AttnOp(8, 2, 128, 2)
        out = op.enqueue(q, kv, starts, lens, table, max_q=max(new), out=q)
        assert out is q and bool(((q.double() - want).abs() <= bound).all())
