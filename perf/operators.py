"""What the framework's attention and 8-bit integer operators are measured on.

Three operators: the 8-bit integer matrix product with a scale for each token
and channel (``I8Op``), given either 8-bit codes or 16-bit rows that it
quantises (and normalises) on the way; the append to a paged key/value cache
with the position rotation (``kv_append``); the attention of new tokens over
that cache (``AttnOp``).  With ``own`` false ``run`` computes them with
elementary torch operations in 32 bits (angles in 64), with ``own`` true
through the package.
"""
import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


def _package():
    if "b2g" in sys.modules:
        return sys.modules["b2g"]
    path = Path.cwd() / "llama-3.2-3b-instruct-gemm-optimization_b200" / "__init__.py"
    spec = importlib.util.spec_from_file_location("b2g", path, submodule_search_locations=[str(path.parent)])
    mod = importlib.util.module_from_spec(spec)
    sys.modules["b2g"] = mod
    spec.loader.exec_module(mod)
    return mod


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _mat(name, m, n, k, dtype, fuse, given="codes"):
    """`given`: 8-bit codes with their scales, or 16-bit "rows", or 16-bit rows
    that are normalised first ("rms")."""
    return {"name": name, "op": "matmul", "m": m, "n": n, "k": k, "dtype": dtype, "fuse": fuse, "given": given}


def _cache(name, op, batch, new, context, ragged, hq, hkv, d, page, dtype, cache, **more):
    """`new`: the most new tokens of a sequence, `context`: the most tokens a
    sequence has after them; `ragged`: lengths differ between sequences."""
    return dict({"name": name, "op": op, "batch": batch, "new": new, "context": context, "ragged": ragged, "hq": hq,
                 "hkv": hkv, "d": d, "page": page, "dtype": dtype, "cache": cache}, **more)


def listed():
    return [
        # one token through an output projection, onto the residual stream
        _mat("matmul 1 token, residual", 1, 4096, 8192, "fp16", "residual"),
        # a batch of decoding sequences through gate||up
        _mat("matmul 64 tokens, gate||up", 64, 8192, 4096, "fp16", "gate_up"),
        # a decode step's 16-bit rows through the down projection
        _mat("linear 8 rows, residual", 8, 4096, 8192, "fp16", "residual", "rows"),
        # a ragged prompt's hidden states, normalised, through the query, key and value projection
        _mat("linear 517 rows, rms", 517, 6144, 4096, "bf16", "none", "rms"),
        # a large prompt chunk
        _mat("matmul 4096 tokens", 4096, 8192, 8192, "bf16", "none"),
        # a decode step of many sequences
        _cache("append decode, 64 sequences", "append", 64, 1, 2048, True, 32, 8, 128, 16, "fp16", "fp16", interleaved=False),
        # prompt chunks into an 8-bit cache
        _cache("append prompts, 8-bit cache", "append", 5, 4000, 6000, True, 32, 8, 128, 64, "bf16", "e4m3", interleaved=True),
        # one sequence decoding: latency
        _cache("attention decode, 1 sequence", "attention", 1, 1, 4001, False, 24, 8, 128, 16, "fp16", "fp16", window=0),
        # many sequences decoding: bandwidth
        _cache("attention decode, 64 sequences", "attention", 64, 1, 8192, True, 32, 8, 128, 16, "bf16", "bf16", window=0),
        # two long contexts in an 8-bit cache, a few drafted tokens each
        _cache("attention long, 8-bit cache", "attention", 2, 4, 131072, False, 32, 8, 128, 64, "fp16", "e4m3", window=0),
        # chunks of prompts behind earlier tokens
        _cache("attention prompt chunks", "attention", 3, 2048, 6000, True, 32, 8, 128, 64, "bf16", "bf16", window=0),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["matmul", "matmul", "append", "attention", "attention"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "matmul":
        m, n, k = _spread(rng, 1, 4096), _spread(rng, 128, 8192), _spread(rng, 128, 8192)
        fuse, given = rng.choice(["none", "residual", "gate_up"]), rng.choice(["codes", "rows", "rms"])
        return _mat("", m // 2 + 1 if fuse == "gate_up" else m, n, k if given == "codes" else (k + 7) // 8 * 8, dtype, fuse, given)
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4])
    d, page = rng.choice([64, 128]), rng.choice([8, 16, 32, 64, 128, 17])
    cache = rng.choice([dtype, "e4m3"])
    if op == "append":
        batch = _spread(rng, 1, 64)
        new = _spread(rng, 1, max(1, 12000 // batch))
        return _cache("", op, batch, new, new + _spread(rng, 1, 2048), True, hq, hkv, d, page, dtype, cache,
                      interleaved=rng.random() < 0.5)
    window = rng.choice([0, 0, 0, 100, 1024])
    if rng.random() < 0.5:  # decode
        batch = _spread(rng, 1, 64)
        new, context = rng.choice([1, 1, 2, 4]), _spread(rng, 16, 300000 // batch if batch > 4 else 100000)
    else:  # prompt chunks
        batch = _spread(rng, 1, 6)
        new = _spread(rng, 16, 2048)
        context = new + _spread(rng, 1, 3500)
    return _cache("", op, batch, new, max(new, context), True, hq, hkv, d, page, dtype, cache, window=window)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 1009 + 17)


def _padded_codes(g, rows, cols):
    """Random 8-bit codes, rows 16-byte aligned as quantize_i8_rows leaves them."""
    ld = -(-cols // 16) * 16
    return torch.randint(-127, 128, (rows, ld), dtype=torch.int8, device=DEV, generator=g)[:, :cols]


def _lengths(case):
    """(new tokens, tokens after them) of each sequence: host lists that go by
    the case alone, so that its outputs have one shape."""
    r = random.Random(case["batch"] * 1000003 + case["new"] * 1009 + case["context"])
    new, total = [], []
    for b in range(case["batch"]):
        n, t = case["new"], case["context"]
        if case["ragged"] and b:
            n = r.randint(max(1, n // 4), n)
            t = r.randint(max(n, t // 4), t)
        new.append(n)
        total.append(t)
    return new, total


def _inv_freq(d):
    # Llama's base
    return (500000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)).float()


def prepare(case, seed):
    g = _generator(seed)
    st = {"case": case}
    if case["op"] == "matmul":
        t = TYPES[case["dtype"]]
        m, n, k = case["m"], case["n"], case["k"]
        planes = 2 if case["fuse"] == "gate_up" else 1
        if case["given"] == "codes":
            st["xq"] = _padded_codes(g, m, k)
            st["sx"] = (0.5 + torch.rand(m, device=DEV, generator=g)) / 73
        else:
            st["x"] = torch.randn(m, k, device=DEV, generator=g).to(t)
            st["gamma"] = (1 + 0.1 * torch.randn(k, device=DEV, generator=g)).to(t) if case["given"] == "rms" else None
        st["wq"] = _padded_codes(g, planes * n, k)
        # scales that leave outputs of order one
        st["sw"] = (0.5 + torch.rand(planes * n, device=DEV, generator=g)) / 73 / math.sqrt(k)
        st["residual"] = torch.randn(m, n, device=DEV, generator=g).to(t) if case["fuse"] == "residual" else None
        if own:
            b2g = _package()
            fuse = {"none": b2g.FUSE_NONE, "residual": b2g.FUSE_RESIDUAL_ADD, "gate_up": b2g.FUSE_GATE_UP_SILU}[case["fuse"]]
            fuse |= b2g.FUSE_RMSNORM_INPUT if case["given"] == "rms" else 0
            st["handle"] = b2g.I8Op(k, n, max_m=m, fuse=fuse, dtype=case["dtype"])
            st["workspace"] = st["handle"].workspace(DEV)
        return st
    t, tc = TYPES[case["dtype"]], TYPES[case["cache"]]
    new, total = _lengths(case)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    pages = [-(-n // page) for n in total]
    most = max(pages)
    pool = sum(pages) + 3
    order = torch.randperm(pool, device=DEV, generator=g).to(torch.int32)
    table = torch.full((len(total), most), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    st["table"], st["max_q"] = table, max(new)
    st["q_start"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    st["lens"] = torch.tensor(total, dtype=torch.int32, device=DEV)
    rows = starts[-1]
    st["k_cache"] = torch.randn(pool, page, hkv, d, device=DEV, generator=g).to(tc)
    st["v_cache"] = torch.randn(pool, page, hkv, d, device=DEV, generator=g).to(tc)
    st["k_scale"] = st["v_scale"] = None
    if case["cache"] == "e4m3":
        st["k_scale"] = 0.5 + torch.rand(hkv, device=DEV, generator=g)
        st["v_scale"] = 0.5 + torch.rand(hkv, device=DEV, generator=g)
    st["q"] = torch.randn(rows, hq, d, device=DEV, generator=g).to(t)
    if case["op"] == "append":
        st["k"] = torch.randn(rows, hkv, d, device=DEV, generator=g).to(t)
        st["v"] = torch.randn(rows, hkv, d, device=DEV, generator=g).to(t)
        st["q_out"] = torch.empty_like(st["q"])
        st["inv_freq"] = _inv_freq(d).to(DEV)
    if own:
        b2g = _package()
        st["b2g"] = b2g
        st["cache"] = b2g.PagedCache(st["k_cache"], st["v_cache"], k_scale=st["k_scale"], v_scale=st["v_scale"])
        if case["op"] == "attention":
            st["handle"] = b2g.AttnOp(hq, hkv, d, max_batch=case["batch"], dtype=case["dtype"], cache_dtype=case["cache"])
            st["workspace"] = st["handle"].workspace(DEV)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
EPS = 1e-5


def _run_matmul(st):
    case, wq, sw = st["case"], st["wq"], st["sw"]
    if own and case["given"] == "codes":
        return st["handle"].enqueue_codes(st["xq"], st["sx"], wq, sw, residual=st["residual"], workspace=st["workspace"])
    if own:
        return st["handle"].enqueue(st["x"], wq, sw, residual=st["residual"], gamma=st["gamma"], rms_eps=EPS,
                                    workspace=st["workspace"])
    if case["given"] == "codes":
        xq, sx = st["xq"].float(), st["sx"]
    else:
        x = st["x"].float()
        if st["gamma"] is not None:
            x = x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS) * st["gamma"].float()
        sx = x.abs().amax(1).clamp(min=1e-12) / 127
        xq = torch.round(x / sx[:, None])
    # blocks of 1024 products of at most 127 * 127 sum to less than 2^24: exact
    # in 32 bits; the blocks' sums are added in 64
    k = xq.shape[1]
    pad = -k % 1024
    a = torch.nn.functional.pad(xq, (0, pad)).view(xq.shape[0], -1, 1024).transpose(0, 1)
    b = torch.nn.functional.pad(wq.float(), (0, pad)).view(wq.shape[0], -1, 1024).permute(1, 2, 0)
    y = (torch.bmm(a, b).sum(0, dtype=torch.float64) * sx[:, None] * sw[None]).float()
    if case["fuse"] == "gate_up":
        gate, up = y.chunk(2, dim=1)
        y = gate / (1 + torch.exp(-gate)) * up
    if case["fuse"] == "residual":
        y = y + st["residual"].float()
    return y.to(TYPES[case["dtype"]])


def _positions(st, rows):
    """(sequence, position) of each row of new tokens."""
    at = torch.arange(rows, device=DEV)
    b = torch.searchsorted(st["q_start"], at.to(torch.int32), right=True) - 1
    end = st["q_start"][1:][b]
    return b, (st["lens"][b] - end).long() + at


def _rotate(x, pos, inv_freq, interleaved):
    angle = pos.double()[:, None] * inv_freq.double()[None]
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = x.float()
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def _into_cache(st, cache, x, scale, page, slot):
    if scale is not None:
        x = (x / scale[:, None]).clamp(-448, 448)
        # an index_put of 8-bit floats: their bytes
        cache.view(torch.uint8)[page, slot] = x.to(cache.dtype).view(torch.uint8)
    else:
        cache[page, slot] = x.to(cache.dtype)


def _run_append(st):
    case = st["case"]
    if own:
        st["b2g"].kv_append(st["k"], st["v"], st["cache"], st["q_start"], st["lens"], st["table"], q=st["q"],
                            q_out=st["q_out"], inv_freq=st["inv_freq"], interleaved=case["interleaved"])
        return st["k_cache"], st["v_cache"], st["q_out"]
    b, pos = _positions(st, st["q"].shape[0])
    page, slot = st["table"][b, pos // case["page"]].long(), pos % case["page"]
    _into_cache(st, st["k_cache"], _rotate(st["k"], pos, st["inv_freq"], case["interleaved"]), st["k_scale"], page, slot)
    _into_cache(st, st["v_cache"], st["v"].float(), st["v_scale"], page, slot)
    st["q_out"].copy_(_rotate(st["q"], pos, st["inv_freq"], case["interleaved"]))
    return st["k_cache"], st["v_cache"], st["q_out"]


def _run_attention(st):
    case, q = st["case"], st["q"]
    if own:
        return st["handle"].enqueue(q, st["cache"], st["q_start"], st["lens"], st["table"], max_q=st["max_q"],
                                    window=case["window"], workspace=st["workspace"])
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    batch, rows, n = case["batch"], q.shape[0], st["max_q"]
    table = st["table"].clamp(min=0).long()
    bits = torch.uint8 if case["cache"] == "e4m3" else st["k_cache"].dtype
    k = st["k_cache"].view(bits)[table].view(st["k_cache"].dtype).float().view(batch, -1, hkv, d)
    v = st["v_cache"].view(bits)[table].view(st["v_cache"].dtype).float().view(batch, -1, hkv, d)
    if st["k_scale"] is not None:
        k, v = k * st["k_scale"][:, None], v * st["v_scale"][:, None]
    b, pos = _positions(st, rows)
    i = torch.arange(rows, device=DEV) - st["q_start"][b]
    padded = torch.zeros(batch, n, hkv, hq // hkv, d, device=DEV)
    padded[b, i] = q.float().view(rows, hkv, hq // hkv, d)
    where = torch.full((batch, n), -1, device=DEV)
    where[b, i] = pos
    j = torch.arange(k.shape[1], device=DEV)
    seen = j <= where[..., None]
    if case["window"]:
        seen &= j > where[..., None] - case["window"]
    s = torch.matmul(padded.permute(0, 2, 3, 1, 4).reshape(batch, hkv, -1, d), k.permute(0, 2, 3, 1)) / math.sqrt(d)
    s = s.view(batch, hkv, -1, n, k.shape[1]).masked_fill_(~seen[:, None, None], -math.inf)
    s -= s.amax(-1, keepdim=True).clamp(min=-1e30)
    s.exp_()
    total = s.sum(-1, keepdim=True)
    out = torch.matmul(s.view(batch, hkv, -1, k.shape[1]), v.permute(0, 2, 1, 3)).view(batch, hkv, -1, n, d)
    out = out / total.clamp(min=1e-30)
    return out.permute(0, 3, 1, 2, 4)[b, i].reshape(rows, hq, d).to(q.dtype)


def run(state):
    return {"matmul": _run_matmul, "append": _run_append, "attention": _run_attention}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _seen(n, t, window):
    """(cached tokens that some new token sees, pairs of new and cached tokens)."""
    first = t - n
    if not window:
        return t, n * first + n * (n + 1) // 2
    pairs = sum(min(first + i + 1, window) for i in range(n))
    return min(t, n + window - 1), pairs


def work(case):
    if case["op"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        planes = 2 if case["fuse"] == "gate_up" else 1
        moved = m * k * (1 if case["given"] == "codes" else 2) + planes * n * k + 4 * (m + planes * n) + 2 * m * n * (2 if case["fuse"] == "residual" else 1)
        return {"bytes": moved, "flops": 2 * m * n * k * planes}
    new, total = _lengths(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    size = 1 if case["cache"] == "e4m3" else 2
    rows = sum(new)
    if case["op"] == "append":
        return {"bytes": rows * d * (2 * hq * 2 + 2 * hkv * (2 + size)) + 16 * case["batch"], "flops": rows * d * 3 * (hq + hkv)}
    seen = [_seen(n, t, case["window"]) for n, t in zip(new, total)]
    cached, pairs = sum(s[0] for s in seen), sum(s[1] for s in seen)
    return {"bytes": cached * hkv * d * 2 * size + rows * hq * d * 4, "flops": 4 * d * hq * pairs}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "matmul":
        n = case["n"]
        w = st["wq"].double() * st["sw"].double()[:, None]
        if case["given"] == "codes":
            x = st["xq"].double() * st["sx"].double()[:, None]
        else:
            x = st["x"].double()
            if case["given"] == "rms":
                x = x / (x.pow(2).sum(1, keepdim=True) / case["k"] + EPS).sqrt() * st["gamma"].double()
            step = x.abs().max(1, keepdim=True).values / 127
            x = torch.round(x / step) * step
        y = x @ w.T
        if case["fuse"] == "gate_up":
            return y[:, :n] * torch.sigmoid(y[:, :n]) * y[:, n:]
        return y if case["fuse"] == "none" else y + st["residual"].double()
    new, total = _lengths(case)
    page, d, group = case["page"], case["d"], case["hq"] // case["hkv"]
    kc, vc, table = st["k_cache"].double(), st["v_cache"].double(), st["table"].long()
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    row = 0
    for b, (n, t) in enumerate(zip(new, total)):
        own_rows = slice(row, row + n)
        row += n
        if case["op"] == "append":
            pos = torch.arange(t - n, t, device=DEV)
            turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                               pos[:, None, None].double() * st["inv_freq"].double())

            def turned(x):
                x = x[own_rows].double()
                if case["interleaved"]:
                    z = torch.view_as_complex(x.reshape(*x.shape[:2], -1, 2).contiguous()) * turn
                    return torch.view_as_real(z).reshape(x.shape)
                z = torch.complex(x[..., :d // 2], x[..., d // 2:]) * turn
                return torch.cat((z.real, z.imag), -1)

            k, v = turned(st["k"]), st["v"][own_rows].double()
            if case["cache"] == "e4m3":
                k = (k / st["k_scale"].double()[:, None]).clamp(-448, 448)
                v = (v / st["v_scale"].double()[:, None]).clamp(-448, 448)
            kc[table[b, pos // page], pos % page] = k
            vc[table[b, pos // page], pos % page] = v
            out[own_rows] = turned(st["q"])
            continue
        used = table[b, :-(-t // page)]
        k, v = kc[used].flatten(0, 1)[:t], vc[used].flatten(0, 1)[:t]
        if case["cache"] == "e4m3":
            k, v = k * st["k_scale"].double()[:, None], v * st["v_scale"].double()[:, None]
        pos = torch.arange(t - n, t, device=DEV)[:, None]
        j = torch.arange(t, device=DEV)[None]
        hidden = (j > pos) | (j <= pos - case["window"]) if case["window"] else j > pos
        for h in range(case["hq"]):
            s = (st["q"][own_rows, h].double() @ k[:, h // group].T) / math.sqrt(d)
            out[own_rows, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v[:, h // group]
    return (kc, vc, out) if case["op"] == "append" else out
