"""Refusals of the 8-bit product, the cache append and the attention, without
a GPU: an op created on a machine without one answers sizes and checks
arguments (every check comes before any CUDA call of an enqueue)."""
from __future__ import annotations

import ctypes

import pytest

OK, INVALID, UNSUPPORTED, CUDA = 0, 1, 2, 3
A = 1 << 20  # an aligned address that nothing reads


def pack(fields, values):
    s = fields()
    for k, v in values.items():
        assert any(k == n for n, _ in fields._fields_), k
        setattr(s, k, v)
    return bytes(s)


I8 = dict(m=4, x=0, ldx=0, gamma=0, rms_eps=1e-5, x_codes=A, ld_codes=64, x_scales=A, w_codes=A, ldw=64, w_scales=A,
          residual=0, ldr=0, y=A, ldy=32, workspace=A)
ROWS = dict(m=4, k=64, dtype=0, rmsnorm=0, x=A, ldx=64, gamma=0, rms_eps=1e-5, codes=A, ld_codes=64, scales=A)
CACHE = dict(k=A, v=A, k_scale=0, v_scale=0, stride_page=16 * 256, stride_token=256, stride_head=128, num_pages=8,
             page_size=16, kv_heads=2, head_dim=128, dtype=0)
BATCH = dict(batch=2, rows=5, max_q=3, max_pages=4, page_table_stride=4, q_start=A, seq_lens=A, page_table=A)
APPEND = dict(dtype=0, q_heads=4, n_freq=64, interleaved=0, inv_freq=A, k=A, stride_k=256, stride_k_head=128, v=A,
              stride_v=256, stride_v_head=128, q=A, stride_q=512, stride_q_head=128, q_out=A, stride_qo=512,
              stride_qo_head=128)
ATTN = dict(q=A, stride_q=512, stride_q_head=128, out=A, stride_o=512, stride_o_head=128, lse=0, scale=0.1, window=0,
            workspace=A)


@pytest.fixture(scope="module")
def no_gpu():
    import torch
    if torch.cuda.is_available():
        pytest.skip("the valid calls here name addresses that a GPU would read")


@pytest.mark.parametrize("f,want", [
    (dict(), OK), (dict(in_features=0), INVALID), (dict(out_features=-1), INVALID), (dict(max_m=0), INVALID),
    (dict(dtype=1), INVALID), (dict(dtype=7), INVALID), (dict(fuse=8), INVALID), (dict(fuse=5), UNSUPPORTED),
    (dict(in_features=131072), UNSUPPORTED), (dict(in_features=131071), OK), (dict(max_m=1 << 21), UNSUPPORTED),
    (dict(fuse=3, dtype=2), OK)])
def test_i8_fields(b2g, no_gpu, f, want):
    h = ctypes.c_void_p()
    v = dict(dict(in_features=64, out_features=32, max_m=4, dtype=0, fuse=0), **f)
    assert b2g.lib().b2g_i8_create(ctypes.byref(b2g.I8Fields(**v)), ctypes.byref(h)) == want
    assert (h.value is not None) == (want == OK)
    b2g.lib().b2g_i8_destroy(h)


@pytest.mark.parametrize("fuse,change", [
    (0, dict(m=0)), (0, dict(m=5)), (0, dict(x=A, ldx=64)), (0, dict(x_codes=0)), (0, dict(x_codes=A + 8)),
    (0, dict(ld_codes=63)), (0, dict(ld_codes=72)), (0, dict(x_scales=0)), (0, dict(x_scales=A + 2)),
    (0, dict(w_codes=0)), (0, dict(w_codes=A + 4)), (0, dict(ldw=48)), (0, dict(ldw=65)), (0, dict(w_scales=0)),
    (0, dict(y=0)), (0, dict(y=A + 1)), (0, dict(ldy=31)), (0, dict(residual=A, ldr=32)), (4, dict()),
    (4, dict(residual=A, ldr=31)), (0, dict(workspace=0)), (0, dict(workspace=A + 16)), (0, dict(gamma=A)),
    (2, dict()), (2, dict(x_codes=0, x_scales=0, x=A, ldx=60)), (2, dict(x_codes=0, x_scales=0, x=A + 8, ldx=64)),
    (0, dict(x_codes=0, x_scales=0, x=A, ldx=64, gamma=A)), (0, dict(x_codes=0, x=A, ldx=64))])
def test_i8_arguments(b2g, no_gpu, fuse, change):
    op = b2g.I8Op(64, 32, 4, fuse)
    good = dict(I8, **(dict(residual=A, ldr=32) if fuse & 4 else {}))
    if fuse & 2:
        good.update(x_codes=0, x_scales=0, x=A, ldx=64)
    call = lambda v: b2g.lib().b2g_i8_enqueue(op.h, pack(b2g.I8Args, v), None)  # noqa: E731
    assert call(good) == CUDA  # nothing to refuse but the missing device
    if change or fuse == 2:
        assert call(dict(I8, **change) if not change or fuse & 6 else dict(good, **change)) == INVALID
    else:
        assert call(dict(I8)) == INVALID
    assert b2g.lib().b2g_i8_enqueue(None, pack(b2g.I8Args, good), None) == INVALID
    assert b2g.lib().b2g_i8_enqueue(op.h, None, None) == INVALID


def test_i8_sizes(b2g, no_gpu):
    small, large = b2g.I8Op(64, 32, 4), b2g.I8Op(8192, 8192, 4096)
    assert 0 < small.workspace_bytes() < large.workspace_bytes() and small.workspace_bytes() % 256 == 0
    assert b2g.lib().b2g_i8_workspace_size(None, None) == INVALID
    assert b2g.lib().b2g_i8_workspace_init(small.h, ctypes.c_void_p(A + 8), None) == INVALID
    assert b2g.lib().b2g_i8_destroy(None) == OK


@pytest.mark.parametrize("change", [
    dict(m=0), dict(k=0), dict(dtype=1), dict(x=0), dict(x=A + 8), dict(ldx=63), dict(ldx=68), dict(codes=0),
    dict(ld_codes=63), dict(ld_codes=72), dict(scales=0), dict(scales=A + 1), dict(gamma=A),
    dict(gamma=A + 8, rmsnorm=1)])
def test_rows_arguments(b2g, no_gpu, change):
    assert b2g.lib().b2g_i8_quantize_rows(pack(b2g.I8RowsArgs, dict(ROWS, **change)), None) == INVALID
    assert b2g.lib().b2g_i8_quantize_rows(pack(b2g.I8RowsArgs, ROWS), None) == CUDA


def test_weights_arguments(b2g, no_gpu):
    f = b2g.lib().b2g_i8_quantize_weights
    good = [A, 64, 32, 0, 0, A, 64, A, None]
    assert f(*good) == CUDA
    for i, v in ((0, None), (0, A + 1), (1, 0), (2, 0), (3, 2), (4, 1), (5, None), (5, A + 8), (6, 48), (6, 72), (7, None)):
        bad = list(good)
        bad[i] = v
        assert f(*bad) == INVALID, (i, v)


BAD_CACHE = [(dict(k=0), INVALID), (dict(v=A + 8), INVALID), (dict(dtype=2), INVALID), (dict(dtype=5), INVALID),
             (dict(num_pages=0), INVALID), (dict(page_size=0), INVALID), (dict(kv_heads=0), INVALID),
             (dict(head_dim=96), UNSUPPORTED), (dict(stride_page=4), INVALID), (dict(stride_token=-256), INVALID),
             (dict(stride_token=64), INVALID), (dict(stride_head=64), INVALID), (dict(stride_head=132), INVALID),
             (dict(k_scale=A), INVALID), (dict(dtype=1, k_scale=A + 2), INVALID)]
BAD_BATCH = [(dict(batch=0), INVALID), (dict(rows=0), INVALID), (dict(max_q=0), INVALID), (dict(max_pages=0), INVALID),
             (dict(page_table_stride=3), INVALID), (dict(q_start=0), INVALID), (dict(seq_lens=0), INVALID),
             (dict(page_table=A + 2), INVALID)]


@pytest.mark.parametrize("args,cache,batch,want",
                         [(a, {}, {}, INVALID) for a in (
                             dict(dtype=1), dict(k=0), dict(k=A + 8), dict(stride_k=252), dict(stride_k=64),
                             dict(stride_k_head=64), dict(v=0), dict(stride_v_head=130), dict(q=0), dict(q_out=0),
                             dict(q_heads=0), dict(q_heads=-1), dict(stride_q=100), dict(stride_qo_head=4),
                             dict(n_freq=-8), dict(n_freq=4), dict(n_freq=72), dict(inv_freq=0), dict(inv_freq=A + 2))]
                         + [({}, c, {}, w) for c, w in BAD_CACHE] + [({}, {}, b, w) for b, w in BAD_BATCH]
                         + [(dict(q=0, q_out=0, q_heads=0), {}, {}, CUDA), (dict(n_freq=0, inv_freq=0), {}, {}, CUDA),
                            ({}, dict(dtype=1), {}, CUDA)])
def test_append_arguments(b2g, no_gpu, args, cache, batch, want):
    call = lambda a, c, b: b2g.lib().b2g_kv_append(  # noqa: E731
        pack(b2g.KvAppendArgs, dict(APPEND, **a)), pack(b2g.KvCache, dict(CACHE, **c)), pack(b2g.KvBatch, dict(BATCH, **b)),
        None)
    assert call({}, {}, {}) == CUDA
    assert call(args, cache, batch) == want
    assert b2g.lib().b2g_kv_append(None, pack(b2g.KvCache, CACHE), pack(b2g.KvBatch, BATCH), None) == INVALID
    assert b2g.lib().b2g_kv_append(pack(b2g.KvAppendArgs, APPEND), None, pack(b2g.KvBatch, BATCH), None) == INVALID
    assert b2g.lib().b2g_kv_append(pack(b2g.KvAppendArgs, APPEND), pack(b2g.KvCache, CACHE), None, None) == INVALID


@pytest.mark.parametrize("f,want", [
    (dict(), OK), (dict(q_heads=0), INVALID), (dict(kv_heads=0), INVALID), (dict(q_heads=5), INVALID),
    (dict(max_batch=0), INVALID), (dict(dtype=1), INVALID), (dict(cache_dtype=2), INVALID), (dict(cache_dtype=1), OK),
    (dict(head_dim=96), UNSUPPORTED), (dict(q_heads=66), UNSUPPORTED), (dict(q_heads=64), OK)])
def test_attn_fields(b2g, no_gpu, f, want):
    h = ctypes.c_void_p()
    v = dict(dict(q_heads=4, kv_heads=2, head_dim=128, max_batch=2, dtype=0, cache_dtype=0), **f)
    assert b2g.lib().b2g_attn_create(ctypes.byref(b2g.AttnFields(**v)), ctypes.byref(h)) == want
    assert (h.value is not None) == (want == OK)
    b2g.lib().b2g_attn_destroy(h)


@pytest.mark.parametrize("args,cache,batch,want",
                         [(a, {}, {}, INVALID) for a in (
                             dict(q=0), dict(q=A + 8), dict(stride_q=4), dict(stride_q=252), dict(stride_q_head=64),
                             dict(out=0), dict(stride_o=64), dict(lse=A + 2), dict(scale=0.0), dict(scale=-1.0),
                             dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(workspace=0),
                             dict(workspace=A + 64))]
                         + [({}, c, {}, w) for c, w in BAD_CACHE] + [({}, {}, b, w) for b, w in BAD_BATCH]
                         + [({}, dict(kv_heads=1), {}, INVALID), ({}, dict(head_dim=64), {}, INVALID),
                            ({}, dict(dtype=1), {}, INVALID), ({}, {}, dict(batch=3), INVALID),
                            ({}, {}, dict(rows=1 << 30), UNSUPPORTED), ({}, dict(num_pages=1 << 24), {}, UNSUPPORTED),
                            (dict(window=2 ** 31 - 1), {}, {}, CUDA), (dict(window=5), {}, {}, CUDA)])
def test_attn_arguments(b2g, no_gpu, args, cache, batch, want):
    op = b2g.AttnOp(4, 2, 128, max_batch=2)
    call = lambda a, c, b: b2g.lib().b2g_attn_enqueue(  # noqa: E731
        op.h, pack(b2g.AttnArgs, dict(ATTN, **a)), pack(b2g.KvCache, dict(CACHE, **c)), pack(b2g.KvBatch, dict(BATCH, **b)),
        None)
    assert call({}, {}, {}) == CUDA
    assert call(args, cache, batch) == want
    assert op.workspace_bytes() > 0
    assert b2g.lib().b2g_attn_enqueue(None, pack(b2g.AttnArgs, ATTN), pack(b2g.KvCache, CACHE), pack(b2g.KvBatch, BATCH),
                                      None) == INVALID


def test_tensors_off_the_gpu_are_refused(b2g, no_gpu):
    import torch
    x = torch.zeros(4, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        b2g.quantize_i8_rows(x)
    with pytest.raises(ValueError):
        b2g.I8Op(64, 32, 4).enqueue(x, torch.zeros(32, 64, dtype=torch.int8), torch.zeros(32))
    with pytest.raises(ValueError):
        b2g.PagedCache(torch.zeros(2, 16, 2, 64), torch.zeros(2, 16, 2, 64))


def test_packed_structures_have_the_c_layout(b2g):
    """The byte strings that the calls pass are the structures' own layout."""
    for fields, packer in ((b2g.I8Args, b2g._pack_i8), (b2g.KvBatch, b2g._pack_batch), (b2g.AttnArgs, b2g._pack_attn),
                           (b2g.KvCache, b2g._pack_cache), (b2g.KvAppendArgs, b2g._pack_append),
                           (b2g.I8RowsArgs, b2g._pack_rows)):
        values = [i + 1.5 if t is ctypes.c_float else i + 1 for i, (_, t) in enumerate(fields._fields_)]
        assert fields.from_buffer_copy(packer(*values)) is not None
        got = fields.from_buffer_copy(packer(*values))
        assert [getattr(got, n) for n, _ in fields._fields_] == values
