// serve.h -- internal interface between the host API (serve_api.cpp) and the
// kernels of the 8-bit integer product (i8.cu), the cache append
// (kv_append.cu) and the attention over the cache (attention.cu).
#pragma once
#include <atomic>
#include <cstddef>
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

#include "../../include/b200gemv.h"

namespace b2g {

// api.cpp: this device's error word, registered so that b2g_device_error
// finds it (NULL: no such device, or a CUDA error).
int* registered_error_word(int dev);

// Lets a kernel use `bytes` of dynamic shared memory on the current device,
// once per device (`done` has a bit for each).
inline cudaError_t allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>* done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done->load(std::memory_order_acquire) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done->fetch_or(bit, std::memory_order_release);
  return e;
}

// cuTensorMapEncodeTiled through the runtime's driver entry point.
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiledFn encode_tiled_fn() {
  static const EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}

// ---------------------------------------------------------------------------
// i8.cu
// ---------------------------------------------------------------------------
struct I8RowsParams {
  const void* x;
  long long ldx;
  const void* gamma;
  float eps;
  int8_t* codes;
  long long ldc;
  float* scales;
  int m, k, bf16, rmsnorm;
};
cudaError_t launch_i8_quantize_rows(const I8RowsParams& p, cudaStream_t stream);
cudaError_t launch_i8_quantize_weights(const void* w, int K, int N, int layout, int bf16, int8_t* codes,
                                       long long ldc, float* scales, cudaStream_t stream);

struct I8Params {
  const int8_t* x;  // [m, ldx] codes
  long long ldx;
  const float* sx;
  const int8_t* w;  // [planes * n, ldw] codes
  long long ldw;
  const float* sw;
  const void* residual;
  long long ldr;
  void* y;
  long long ldy;
  int m, n, k, planes, bf16;
};
// Bytes of the split tiles' partial sums for calls of up to max_m rows.
size_t i8_partial_bytes(int max_m, int planes, int num_sms);
// counters: [num_sms] zeros, left zero.  after_quantiser: the launch before
// this one in the stream is the quantiser of p.x (the weights may be read
// before it ends).
cudaError_t launch_i8_product(const I8Params& p, int num_sms, int* counters, int* partials, int* error,
                              bool after_quantiser, cudaStream_t stream);

// ---------------------------------------------------------------------------
// kv_append.cu, attention.cu
// ---------------------------------------------------------------------------
struct KvAppendParams {
  b2g_kv_append_args a;
  b2g_kv_cache c;
  b2g_kv_batch b;
  int* error;
};
cudaError_t launch_kv_append(const KvAppendParams& p, int num_sms, cudaStream_t stream);

struct AttnParams {
  b2g_attn_args a;
  b2g_kv_cache c;
  b2g_kv_batch b;
  int q_heads, group, bf16;
  int least_units;  // units of work a block at least
  int page_shift;   // log2 of the page size, -1: no power of two
  int* error;
  int* counters;  // [blocks] zeros, left zero
  void* parts;    // [blocks][2] parts of split items
};
// Blocks an SM at most, and counters and parts of an item that a block can share
// (the tiles kernel: two tiles an item).
constexpr int kAttnBlocks = 2, kAttnTiles = 2;
// Bytes of counters and of parts for any call on a device of num_sms SMs.
size_t attn_counter_bytes(int num_sms);
size_t attn_part_bytes(int num_sms, int head_dim);
cudaError_t launch_attention(const AttnParams& p, int num_sms, cudaStream_t stream);

}  // namespace b2g
