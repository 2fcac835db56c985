// serve_api.cpp -- the C ABI of the 8-bit integer product and of the
// attention over a paged cache: argument checks, sizes and launches.
#include <new>

#include "serve.h"

using namespace b2g;

struct b2g_i8_op {
  b2g_i8_fields f;
  int planes, device, num_sms;
  size_t off_codes, off_scales, off_partials, bytes;  // workspace: counters, codes, scales, split tiles' sums
  long long ld_codes;
};

struct b2g_attn {
  b2g_attn_fields f;
  int device, num_sms;
  size_t off_parts, bytes;  // workspace: counters, parts of split items
};

namespace {

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
bool is_act(int32_t t) { return t == B2G_DTYPE_FP16 || t == B2G_DTYPE_BF16; }
b2g_status cuda_status(cudaError_t e) { return e == cudaSuccess ? B2G_OK : B2G_ERR_CUDA; }
cudaStream_t cu(b2g_stream_t s) { return reinterpret_cast<cudaStream_t>(s); }
size_t up(size_t n, size_t to) { return (n + to - 1) / to * to; }

// Rows of a matrix whose row starts are 16-byte aligned.
bool rows16(const void* p, int64_t ld, int64_t cols, int bytes) {
  return p && aligned(p, 16) && ld >= cols && ld * bytes % 16 == 0;
}

b2g_status current_device(int* dev) { return cudaGetDevice(dev) == cudaSuccess ? B2G_OK : B2G_ERR_CUDA; }

// The device an op is made for.  On a machine without one (build-time sizing)
// the op has a B200's SM count: it answers sizes and checks arguments, and
// its enqueue returns B2G_ERR_CUDA.
b2g_status op_device(int* dev, int* sms) {
  const cudaError_t e = cudaGetDevice(dev);
  if (e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver) {
    *dev = -1;
    *sms = 148;
    return B2G_OK;
  }
  if (e != cudaSuccess) return B2G_ERR_CUDA;
  return cuda_status(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, *dev));
}

b2g_status check_cache(const b2g_kv_cache* c, int32_t act) {
  if (!c || !c->k || !c->v) return B2G_ERR_INVALID;
  if (c->dtype != act && c->dtype != B2G_DTYPE_FP8_E4M3) return B2G_ERR_INVALID;
  if (c->num_pages < 1 || c->page_size < 1 || c->kv_heads < 1) return B2G_ERR_INVALID;
  if (c->head_dim != 64 && c->head_dim != 128) return B2G_ERR_UNSUPPORTED;
  const int bytes = c->dtype == B2G_DTYPE_FP8_E4M3 ? 1 : 2;
  if (!aligned(c->k, 16) || !aligned(c->v, 16)) return B2G_ERR_INVALID;
  for (int64_t st : {c->stride_page, c->stride_token, c->stride_head})
    if (st < 0 || st * bytes % 16 != 0) return B2G_ERR_INVALID;
  // Elements of different tokens or heads must not overlap.
  if (c->page_size > 1 && c->stride_token < c->head_dim) return B2G_ERR_INVALID;
  if (c->kv_heads > 1 && c->stride_head < c->head_dim) return B2G_ERR_INVALID;
  if (c->num_pages > 1 && c->stride_page < c->head_dim) return B2G_ERR_INVALID;
  if (c->dtype != B2G_DTYPE_FP8_E4M3 && (c->k_scale || c->v_scale)) return B2G_ERR_INVALID;
  if (!aligned(c->k_scale, 4) || !aligned(c->v_scale, 4)) return B2G_ERR_INVALID;
  // The attention counts 16-byte pieces of the cache in 32 bits.
  const unsigned __int128 span = (unsigned __int128)(c->num_pages - 1) * c->stride_page +
                                 (unsigned __int128)(c->page_size - 1) * c->stride_token +
                                 (unsigned __int128)(c->kv_heads - 1) * c->stride_head + c->head_dim;
  if (span * bytes > (unsigned __int128)1 << 36) return B2G_ERR_UNSUPPORTED;
  return B2G_OK;
}

b2g_status check_batch(const b2g_kv_batch* b) {
  if (!b || !b->q_start || !b->seq_lens || !b->page_table) return B2G_ERR_INVALID;
  if (b->batch < 1 || b->rows < 1 || b->max_q < 1 || b->max_pages < 1) return B2G_ERR_INVALID;
  if (b->page_table_stride < b->max_pages) return B2G_ERR_INVALID;
  if (!aligned(b->q_start, 4) || !aligned(b->seq_lens, 4) || !aligned(b->page_table, 4)) return B2G_ERR_INVALID;
  return B2G_OK;
}

bool heads16(const void* p, int64_t stride_row, int64_t stride_head, int heads, int dim, int rows) {
  if (!p || !aligned(p, 16) || stride_row % 8 || stride_head % 8) return false;
  if (heads > 1 && stride_head < dim) return false;
  return rows == 1 || stride_row >= dim;
}

}  // namespace

extern "C" {

// ---------------------------------------------------------------------------
// 8-bit integer product
// ---------------------------------------------------------------------------
b2g_status b2g_i8_quantize_rows(const b2g_i8_rows_args* a, b2g_stream_t stream) {
  if (!a || a->m < 1 || a->k < 1 || !is_act(a->dtype)) return B2G_ERR_INVALID;
  if (!rows16(a->x, a->ldx, a->k, 2) || !rows16(a->codes, a->ld_codes, a->k, 1)) return B2G_ERR_INVALID;
  if (!a->scales || !aligned(a->scales, 4)) return B2G_ERR_INVALID;
  if (a->gamma && (!a->rmsnorm || !aligned(a->gamma, 16))) return B2G_ERR_INVALID;
  I8RowsParams p = {};
  p.x = a->x;
  p.ldx = a->ldx;
  p.gamma = a->gamma;
  p.eps = a->rms_eps;
  p.codes = static_cast<int8_t*>(a->codes);
  p.ldc = a->ld_codes;
  p.scales = a->scales;
  p.m = a->m;
  p.k = a->k;
  p.bf16 = a->dtype == B2G_DTYPE_BF16;
  p.rmsnorm = a->rmsnorm != 0;
  return cuda_status(launch_i8_quantize_rows(p, cu(stream)));
}

b2g_status b2g_i8_quantize_weights(const void* w16, int32_t K, int32_t N, int32_t layout, int32_t dtype, void* codes,
                                   int64_t ld_codes, float* scales, b2g_stream_t stream) {
  if (!w16 || K < 1 || N < 1 || !is_act(dtype) || !scales) return B2G_ERR_INVALID;
  if (layout != B2G_LAYOUT_KN && layout != B2G_LAYOUT_NK) return B2G_ERR_INVALID;
  if (!aligned(w16, 2) || !aligned(scales, 4) || !rows16(codes, ld_codes, K, 1)) return B2G_ERR_INVALID;
  return cuda_status(launch_i8_quantize_weights(w16, K, N, layout, dtype == B2G_DTYPE_BF16,
                                                static_cast<int8_t*>(codes), ld_codes, scales, cu(stream)));
}

b2g_status b2g_i8_create(const b2g_i8_fields* f, b2g_i8_op** out) {
  if (out) *out = nullptr;
  if (!f || !out) return B2G_ERR_INVALID;
  if (f->in_features < 1 || f->out_features < 1 || f->max_m < 1 || !is_act(f->dtype)) return B2G_ERR_INVALID;
  if (f->fuse & ~(B2G_FUSE_GATE_UP_SILU | B2G_FUSE_RMSNORM_INPUT | B2G_FUSE_RESIDUAL_ADD)) return B2G_ERR_INVALID;
  if ((f->fuse & B2G_FUSE_GATE_UP_SILU) && (f->fuse & B2G_FUSE_RESIDUAL_ADD)) return B2G_ERR_UNSUPPORTED;
  if (f->in_features > B2G_I8_MAX_K) return B2G_ERR_UNSUPPORTED;
  if (f->out_features > (1 << 24) || f->max_m > (1 << 20)) return B2G_ERR_UNSUPPORTED;
  int dev = -1, sms = 0;
  const b2g_status st = op_device(&dev, &sms);
  if (st != B2G_OK) return st;
  b2g_i8_op* op = new (std::nothrow) b2g_i8_op();
  if (!op) return B2G_ERR_OOM;
  op->f = *f;
  op->planes = (f->fuse & B2G_FUSE_GATE_UP_SILU) ? 2 : 1;
  op->device = dev;
  op->num_sms = sms;
  op->ld_codes = (long long)up(f->in_features, 16);
  op->off_codes = up((size_t)sms * 4, 256);
  op->off_scales = op->off_codes + up((size_t)op->ld_codes * f->max_m, 256);
  op->off_partials = op->off_scales + up((size_t)f->max_m * 4, 256);
  op->bytes = op->off_partials + i8_partial_bytes(f->max_m, op->planes, sms);
  *out = op;
  return B2G_OK;
}

b2g_status b2g_i8_destroy(b2g_i8_op* op) {
  delete op;
  return B2G_OK;
}

b2g_status b2g_i8_workspace_size(const b2g_i8_op* op, size_t* bytes) {
  if (!op || !bytes) return B2G_ERR_INVALID;
  *bytes = op->bytes;
  return B2G_OK;
}

b2g_status b2g_i8_workspace_init(const b2g_i8_op* op, void* ws, b2g_stream_t stream) {
  if (!op || !ws || !aligned(ws, 256)) return B2G_ERR_INVALID;
  return cuda_status(cudaMemsetAsync(ws, 0, op->bytes, cu(stream)));
}

b2g_status b2g_i8_enqueue(const b2g_i8_op* op, const b2g_i8_args* a, b2g_stream_t stream) {
  if (!op || !a) return B2G_ERR_INVALID;
  const int K = op->f.in_features, N = op->f.out_features;
  const bool norm = (op->f.fuse & B2G_FUSE_RMSNORM_INPUT) != 0, resid = (op->f.fuse & B2G_FUSE_RESIDUAL_ADD) != 0;
  if (a->m < 1 || a->m > op->f.max_m) return B2G_ERR_INVALID;
  if ((a->x != nullptr) == (a->x_codes != nullptr)) return B2G_ERR_INVALID;
  if (a->x) {
    if (!rows16(a->x, a->ldx, K, 2) || a->x_scales) return B2G_ERR_INVALID;
    if (a->gamma && (!norm || !aligned(a->gamma, 16))) return B2G_ERR_INVALID;
  } else {
    if (norm || a->gamma) return B2G_ERR_INVALID;
    if (!rows16(a->x_codes, a->ld_codes, K, 1) || !a->x_scales || !aligned(a->x_scales, 4)) return B2G_ERR_INVALID;
  }
  if (!rows16(a->w_codes, a->ldw, K, 1) || !a->w_scales || !aligned(a->w_scales, 4)) return B2G_ERR_INVALID;
  if (!a->y || !aligned(a->y, 2) || a->ldy < N) return B2G_ERR_INVALID;
  if (resid != (a->residual != nullptr) || (resid && (!aligned(a->residual, 2) || a->ldr < N))) return B2G_ERR_INVALID;
  if (!a->workspace || !aligned(a->workspace, 256)) return B2G_ERR_INVALID;
  int dev = -1;
  b2g_status st = current_device(&dev);
  if (st != B2G_OK) return st;
  if (dev != op->device) return B2G_ERR_INVALID;
  int* error = registered_error_word(dev);
  if (!error) return B2G_ERR_CUDA;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  I8Params p = {};
  if (a->x) {
    b2g_i8_rows_args r = {};
    r.m = a->m;
    r.k = K;
    r.dtype = op->f.dtype;
    r.rmsnorm = norm;
    r.x = a->x;
    r.ldx = a->ldx;
    r.gamma = a->gamma;
    r.rms_eps = a->rms_eps;
    r.codes = ws + op->off_codes;
    r.ld_codes = op->ld_codes;
    r.scales = reinterpret_cast<float*>(ws + op->off_scales);
    st = b2g_i8_quantize_rows(&r, stream);
    if (st != B2G_OK) return st;
    p.x = static_cast<const int8_t*>(r.codes);
    p.ldx = r.ld_codes;
    p.sx = r.scales;
  } else {
    p.x = static_cast<const int8_t*>(a->x_codes);
    p.ldx = a->ld_codes;
    p.sx = a->x_scales;
  }
  p.w = static_cast<const int8_t*>(a->w_codes);
  p.ldw = a->ldw;
  p.sw = a->w_scales;
  p.residual = a->residual;
  p.ldr = a->ldr;
  p.y = a->y;
  p.ldy = a->ldy;
  p.m = a->m;
  p.n = N;
  p.k = K;
  p.planes = op->planes;
  p.bf16 = op->f.dtype == B2G_DTYPE_BF16;
  return cuda_status(launch_i8_product(p, op->num_sms, reinterpret_cast<int*>(ws),
                                       reinterpret_cast<int*>(ws + op->off_partials), error, a->x != nullptr,
                                       cu(stream)));
}

// ---------------------------------------------------------------------------
// Paged cache
// ---------------------------------------------------------------------------
b2g_status b2g_kv_append(const b2g_kv_append_args* a, const b2g_kv_cache* c, const b2g_kv_batch* b,
                         b2g_stream_t stream) {
  if (!a || !is_act(a->dtype)) return B2G_ERR_INVALID;
  b2g_status st = check_cache(c, a->dtype);
  if (st == B2G_OK) st = check_batch(b);
  if (st != B2G_OK) return st;
  const int dim = c->head_dim;
  if (!heads16(a->k, a->stride_k, a->stride_k_head, c->kv_heads, dim, b->rows)) return B2G_ERR_INVALID;
  if (!heads16(a->v, a->stride_v, a->stride_v_head, c->kv_heads, dim, b->rows)) return B2G_ERR_INVALID;
  if (a->q_heads < 0 || (a->q_heads > 0) != (a->q != nullptr) || (a->q != nullptr) != (a->q_out != nullptr))
    return B2G_ERR_INVALID;
  if (a->q && (!heads16(a->q, a->stride_q, a->stride_q_head, a->q_heads, dim, b->rows) ||
               !heads16(a->q_out, a->stride_qo, a->stride_qo_head, a->q_heads, dim, b->rows)))
    return B2G_ERR_INVALID;
  if (a->n_freq < 0 || a->n_freq % 8 || 2 * a->n_freq > dim) return B2G_ERR_INVALID;
  if (a->n_freq && (!a->inv_freq || !aligned(a->inv_freq, 4))) return B2G_ERR_INVALID;
  int dev = -1;
  st = current_device(&dev);
  if (st != B2G_OK) return st;
  int sms = 0;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return B2G_ERR_CUDA;
  KvAppendParams p = {*a, *c, *b, registered_error_word(dev)};
  if (!p.a.inv_freq) p.a.n_freq = 0;
  if (!p.error) return B2G_ERR_CUDA;
  return cuda_status(launch_kv_append(p, sms, cu(stream)));
}

b2g_status b2g_attn_create(const b2g_attn_fields* f, b2g_attn** out) {
  if (out) *out = nullptr;
  if (!f || !out) return B2G_ERR_INVALID;
  if (f->q_heads < 1 || f->kv_heads < 1 || f->q_heads % f->kv_heads || f->max_batch < 1) return B2G_ERR_INVALID;
  if (!is_act(f->dtype) || (f->cache_dtype != f->dtype && f->cache_dtype != B2G_DTYPE_FP8_E4M3))
    return B2G_ERR_INVALID;
  if (f->head_dim != 64 && f->head_dim != 128) return B2G_ERR_UNSUPPORTED;
  if (f->q_heads / f->kv_heads > 32 || f->q_heads > 65535) return B2G_ERR_UNSUPPORTED;
  int dev = -1, sms = 0;
  const b2g_status st = op_device(&dev, &sms);
  if (st != B2G_OK) return st;
  b2g_attn* op = new (std::nothrow) b2g_attn();
  if (!op) return B2G_ERR_OOM;
  op->f = *f;
  op->device = dev;
  op->num_sms = sms;
  op->off_parts = attn_counter_bytes(sms);
  op->bytes = op->off_parts + attn_part_bytes(sms, f->head_dim);
  *out = op;
  return B2G_OK;
}

b2g_status b2g_attn_destroy(b2g_attn* op) {
  delete op;
  return B2G_OK;
}

b2g_status b2g_attn_workspace_size(const b2g_attn* op, size_t* bytes) {
  if (!op || !bytes) return B2G_ERR_INVALID;
  *bytes = op->bytes;
  return B2G_OK;
}

b2g_status b2g_attn_workspace_init(const b2g_attn* op, void* ws, b2g_stream_t stream) {
  if (!op || !ws || !aligned(ws, 256)) return B2G_ERR_INVALID;
  return cuda_status(cudaMemsetAsync(ws, 0, op->off_parts, cu(stream)));
}

b2g_status b2g_attn_enqueue(const b2g_attn* op, const b2g_attn_args* a, const b2g_kv_cache* c, const b2g_kv_batch* b,
                            b2g_stream_t stream) {
  if (!op || !a) return B2G_ERR_INVALID;
  b2g_status st = check_cache(c, op->f.dtype);
  if (st == B2G_OK) st = check_batch(b);
  if (st != B2G_OK) return st;
  if (c->dtype != op->f.cache_dtype || c->kv_heads != op->f.kv_heads || c->head_dim != op->f.head_dim)
    return B2G_ERR_INVALID;
  if (b->batch > op->f.max_batch) return B2G_ERR_INVALID;
  // Rows are counted per k/v head in 32 bits.
  if ((int64_t)b->rows * (op->f.q_heads / op->f.kv_heads) > (1 << 30)) return B2G_ERR_UNSUPPORTED;
  const int dim = op->f.head_dim, heads = op->f.q_heads;
  if (!heads16(a->q, a->stride_q, a->stride_q_head, heads, dim, b->rows)) return B2G_ERR_INVALID;
  if (!heads16(a->out, a->stride_o, a->stride_o_head, heads, dim, b->rows)) return B2G_ERR_INVALID;
  if (!aligned(a->lse, 4) || a->window < 0 || !(a->scale > 0) || a->scale > 1e30f) return B2G_ERR_INVALID;
  if (!a->workspace || !aligned(a->workspace, 256)) return B2G_ERR_INVALID;
  int dev = -1;
  st = current_device(&dev);
  if (st != B2G_OK) return st;
  if (dev != op->device) return B2G_ERR_INVALID;
  AttnParams p = {};
  p.a = *a;
  if (p.a.window > (1 << 30)) p.a.window = 1 << 30;  // more than a cache holds
  p.c = *c;
  p.b = *b;
  p.q_heads = heads;
  p.group = heads / op->f.kv_heads;
  p.bf16 = op->f.dtype == B2G_DTYPE_BF16;
  p.error = registered_error_word(dev);
  if (!p.error) return B2G_ERR_CUDA;
  p.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (c->page_size == 1 << i) p.page_shift = i;
  p.counters = static_cast<int*>(a->workspace);
  p.parts = static_cast<uint8_t*>(a->workspace) + op->off_parts;
  return cuda_status(launch_attention(p, op->num_sms, cu(stream)));
}

}  // extern "C"
