"""kv_append against its definition in 64 bits.

A rotated value is two products and a sum in fp32 of a cosine and sine that
are right to 2^-22 (the angle is reduced in 64 bits): off by at most
2^-20 (|a| + |b|) before it is rounded once to its type."""
from __future__ import annotations

import math

import pytest
import torch

from attn_reference import make_batch

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


def inv_freq(n):
    return (10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))).float().cuda()


def rotated(x, pos, freq, interleaved):
    """(values, sum of magnitudes) in 64 bits."""
    n = freq.shape[0]
    y, mag = x.double().clone(), x.double().abs().clone()
    a = pos.double()[:, None] * freq.double()
    c, s = a.cos()[:, None], a.sin()[:, None]
    i = torch.arange(n, device=x.device)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    u, v = x.double()[..., lo], x.double()[..., hi]
    y[..., lo], y[..., hi] = u * c - v * s, v * c + u * s
    mag[..., lo] = mag[..., hi] = u.abs() + v.abs()
    return y, mag


def near(got, want, mag, t):
    """Within the rounding of t; E4M3 saturates at 448, its smallest step is 2^-9."""
    g = got.double()
    if t == torch.float8_e4m3fn:
        want = want.clamp(-448, 448)
        return bool(((g - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 + 2.0 ** -19 * mag).all())
    return bool(((g - want).abs() <= torch.finfo(t).eps / 2 * want.abs() + 2.0 ** -20 * mag + 2.0 ** -25).all())


def check(b2g, new, total, hq, hkv, d, page, dtype, cache="same", n_freq=None, interleaved=False, layout="NHD",
          with_q=True, in_place=False, slack=0, far=0):
    cache = dtype if cache == "same" else cache
    t, tc = TYPES[dtype], TYPES[cache]
    starts, lens, table, pool = make_batch(new, [x + 0 for x in total], page, extra_pages=2)
    rows = sum(new) + slack
    g = torch.Generator(device="cuda").manual_seed(11)
    shape = (pool, page, hkv, d) if layout == "NHD" else (pool, hkv, page, d)
    kc = torch.randn(shape, device="cuda", generator=g).to(tc)
    vc = torch.randn(shape, device="cuda", generator=g).to(tc)
    before = [x.view(torch.uint8).clone() for x in (kc, vc)]
    ks = vs = None
    if cache == "e4m3":
        ks, vs = (0.01 + torch.rand(hkv, device="cuda", generator=g) for _ in range(2))
    kv = b2g.PagedCache(kc, vc, layout, k_scale=ks, v_scale=vs)
    qkv = torch.randn(rows, hq + 2 * hkv, d, device="cuda", generator=g).to(t)  # as one projection leaves them
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    q0, k0 = q.clone(), k.clone()
    freq = inv_freq(d // 2 if n_freq is None else n_freq)
    q_out = None if in_place or not with_q else torch.full((rows, hq, d), 7.0, dtype=t, device="cuda")
    out = b2g.kv_append(k, v, kv, starts, lens, table, q=q if with_q else None, q_out=q_out, inv_freq=freq,
                        interleaved=interleaved)
    torch.cuda.synchronize()
    assert b2g.device_error() == 0
    n = sum(new)
    pos = torch.cat([torch.arange(a - b, a) for a, b in zip(total, new)]).cuda()
    seq = torch.cat([torch.full((b,), i) for i, b in enumerate(new)]).long().cuda()
    keep = pos >= 0
    wq, mq = rotated(q0[:n], pos, freq, interleaved)
    if with_q:
        assert near(out[:n], wq, mq, t)
        assert torch.equal(out[n:], q0[n:] if in_place else torch.full_like(out[n:], 7.0))
    wk, mk = rotated(k0[:n], pos, freq, interleaved)
    wv = v[:n].double()
    if cache == "e4m3":
        wk, mk, wv = wk / ks.double()[:, None], mk / ks.double()[:, None], wv / vs.double()[:, None]
    page_id, slot = table[seq[keep], pos[keep] // page].long(), pos[keep] % page
    touched = torch.zeros(pool, page, dtype=torch.bool, device="cuda")
    touched[page_id, slot] = True
    for x, old, want, mag in ((kc, before[0], wk, mk), (vc, before[1], wv, wv.abs())):
        y = x.view(torch.uint8).view(*shape[:3], -1)
        y, o = (a if layout == "NHD" else a.transpose(1, 2) for a in (y, old.view(y.shape)))
        assert torch.equal(y[~touched], o[~touched])  # every other row as it was
        assert near(y[page_id, slot].contiguous().view(tc), want[keep], mag[keep], tc)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype,cache", [("fp16", "same"), ("bf16", "same"), ("fp16", "e4m3"), ("bf16", "e4m3")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_types_and_styles(b2g, cuda, d, dtype, cache, interleaved):
    check(b2g, [1, 5, 0, 40], [1, 70, 9, 300], 6, 2, d, 16, dtype, cache, interleaved=interleaved, slack=3)


@pytest.mark.parametrize("page", [1, 7, 16, 128, 1000])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_pages_and_layouts(b2g, cuda, page, layout):
    check(b2g, [3, 1, 20], [3, 500, 100], 4, 1, 128, page, "bf16", layout=layout)


@pytest.mark.parametrize("n_freq", [0, 8, 16, 48])
@pytest.mark.parametrize("interleaved", [False, True])
def test_partly_rotated_heads(b2g, cuda, n_freq, interleaved):
    check(b2g, [4], [90], 3, 3, 128, 16, "fp16", n_freq=n_freq, interleaved=interleaved)


def test_without_q_and_in_place(b2g, cuda):
    check(b2g, [4, 2], [90, 2], 4, 2, 128, 16, "fp16", with_q=False)
    check(b2g, [4, 2], [90, 2], 4, 2, 128, 16, "fp16", in_place=True, slack=2)


def test_one_head_and_many(b2g, cuda):
    check(b2g, [3], [8], 1, 1, 64, 16, "fp16")
    check(b2g, [3], [8], 64, 16, 128, 16, "bf16")


def test_many_sequences(b2g, cuda):
    check(b2g, [1] * 1100, [1 + i % 90 for i in range(1100)], 2, 1, 64, 16, "fp16")
    check(b2g, [i % 4 for i in range(200)], [4 + i % 90 for i in range(200)], 2, 1, 64, 16, "fp16")


def test_rows_before_the_start(b2g, cuda):
    """More new rows than the length counts: q is rotated, nothing is cached for them."""
    check(b2g, [5, 3], [2, 0], 2, 1, 64, 16, "fp16")


def test_far_positions(b2g, cuda):
    """Position 10^6: an angle in 32 bits would be off by 0.03."""
    total = 1000000
    table = torch.full((1, total // 16 + 1), -1, dtype=torch.int32, device="cuda")
    table[0, (total - 1) // 16] = 0
    k = torch.randn(1, 1, 128, device="cuda").half()
    cache = b2g.PagedCache(torch.zeros(1, 16, 1, 128, device="cuda", dtype=torch.float16),
                           torch.zeros(1, 16, 1, 128, device="cuda", dtype=torch.float16))
    b2g.kv_append(k, k, cache, torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                  torch.tensor([total], dtype=torch.int32, device="cuda"), table, inv_freq=inv_freq(64))
    want, mag = rotated(k, torch.tensor([total - 1], device="cuda"), inv_freq(64), False)
    assert near(cache.k[0, (total - 1) % 16], want[0], mag[0], torch.float16)


def test_bad_pages_are_not_written(b2g, cuda):
    kc, vc = (torch.zeros(4, 16, 2, 64, device="cuda", dtype=torch.float16) for _ in range(2))
    cache = b2g.PagedCache(kc, vc)
    k = torch.ones(20, 2, 64, device="cuda", dtype=torch.float16)
    starts = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    lens = torch.tensor([20], dtype=torch.int32, device="cuda")
    for bad in (-1, 4, 2 ** 31 - 1):
        kc.zero_()
        table = torch.tensor([[bad, 2]], dtype=torch.int32, device="cuda")
        b2g.kv_append(k, k, cache, starts, lens, table)
        torch.cuda.synchronize()
        assert b2g.device_error() == 6
        assert bool((kc[2, :4] == 1).all()) and int(kc.sum()) == 4 * 2 * 64
    b2g.kv_append(k, k, cache, starts, lens + 100, torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert b2g.device_error() == 6  # past the table


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_8bit_codes_are_the_rounded_quotients(b2g, cuda, dtype):
    """Codes of value / scale, divided in fp32 and rounded once: ties
    (which a product by 1 / scale leaves on either side), neighbours of ties,
    saturation, and scales whose reciprocal fp32 does not hold."""
    t, d = TYPES[dtype], 64
    scales = [m / 64 for m in range(33, 64, 2)] + [m / 7 for m in range(1, 9)] + [1e-39, 2e-38, 1e-30, 1e30, 3e38, 1.0]
    ties = [m * 2.0 ** e for m in range(17, 32, 2) for e in range(-11, 5)] + [m * 2.0 ** -10 for m in range(1, 16, 2)]
    s = torch.tensor(scales, dtype=torch.float32)
    v = (torch.tensor(ties, dtype=torch.float64)[:, None] * s.double()).float().to(t)  # exact on a tie or next to it
    g = torch.Generator().manual_seed(4)
    v = torch.cat([v, -v, torch.randn(300, len(scales), generator=g).to(t), torch.zeros(4, len(scales)).to(t)])
    v = v.nan_to_num(posinf=1.0, neginf=-1.0)
    rows = -(-v.shape[0] // d)
    x = torch.zeros(rows * d, len(scales), dtype=t)
    x[:v.shape[0]] = v
    x = x.view(rows, d, len(scales)).transpose(1, 2).contiguous()  # [rows, heads, dim], a scale a head
    want = (x.float() / s[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).float()
    kc, vc = (torch.zeros(-(-rows // 16), 16, len(scales), d, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
              for _ in range(2))
    cache = b2g.PagedCache(kc, vc, k_scale=s.cuda(), v_scale=s.cuda())
    args = (torch.tensor(a, dtype=torch.int32, device="cuda") for a in ([0, rows], [rows], [list(range(kc.shape[0]))]))
    b2g.kv_append(x.cuda(), x.cuda(), cache, *args)
    torch.cuda.synchronize()
    for c in (kc, vc):
        got = c.float().flatten(0, 1)[:rows].cpu()
        assert torch.equal(got, want), f"{int((got != want).sum())} of {want.numel()} codes differ"


def test_refusals(b2g, cuda):
    kc, vc = (torch.zeros(4, 16, 2, 64, device="cuda", dtype=torch.float16) for _ in range(2))
    cache = b2g.PagedCache(kc, vc)
    k = torch.ones(1, 2, 64, device="cuda", dtype=torch.float16)
    args = (cache, *(torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1], [1], [[0]])))
    b2g.kv_append(k, k, *args)
    with pytest.raises(ValueError):
        b2g.kv_append(k, k[:, :1], *args)
    with pytest.raises(ValueError):
        b2g.kv_append(k, k, *args, q_out=k)
    with pytest.raises(ValueError):
        b2g.kv_append(k, k, *args, inv_freq=inv_freq(8).double())
    with pytest.raises(b2g.B2GError):  # not a multiple of 8
        b2g.kv_append(k, k, *args, inv_freq=inv_freq(12))
    with pytest.raises(b2g.B2GError):  # more than a head has
        b2g.kv_append(k, k, *args, inv_freq=inv_freq(40))
    with pytest.raises(b2g.B2GError):  # the cache's type
        b2g.kv_append(k.bfloat16(), k.bfloat16(), *args)
    with pytest.raises(ValueError):
        b2g.PagedCache(kc, vc.bfloat16())
    with pytest.raises(b2g.B2GError):  # rows off 16 bytes
        odd = torch.ones(2 * 64 + 1, device="cuda", dtype=torch.float16)[1:].view(1, 2, 64)
        b2g.kv_append(odd, odd, *args)
