// serve.cuh -- device helpers shared by the kernels of i8.cu, kv_append.cu and
// attention.cu: the 16-bit activation types and the batch's lookups.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "device.cuh"
#include "serve.h"

namespace b2g {

// Launches a kernel that may start before the one ahead of it in the stream
// has ended (programmatic dependent launch): its blocks set themselves up and
// wait (griddepcontrol.wait, in every block) before they touch global memory.
template <typename P>
cudaError_t launch_after(void (*kernel)(P), dim3 grid, dim3 block, int smem, int cluster, cudaStream_t stream,
                         const P& params) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, kernel, params);
}

// Thread-block clusters: a barrier over all their threads, and a peer's
// shared memory.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_map(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ int ld_cluster(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

constexpr int kErrBadPage = 6;  // a page table entry outside the cache, or a token past the table

template <typename T>
struct Act;
template <>
struct Act<__half> {
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
};
template <>
struct Act<__nv_bfloat16> {
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
};

// One sequence's rows and cached length, clamped to what the buffers hold.
struct SeqSpan {
  int first, n;  // its rows are first .. first + n - 1
  int ctx;       // position of its row 0 (negative: more rows than the length counts)
};
__device__ __forceinline__ SeqSpan seq_span(const b2g_kv_batch& b, int s) {
  SeqSpan r;
  const int lo = min(max(b.q_start[s], 0), b.rows);
  const int hi = min(max(b.q_start[s + 1], lo), b.rows);
  r.first = lo;
  r.n = hi - lo;
  r.ctx = max(b.seq_lens[s], 0) - r.n;
  return r;
}

// The sequence whose rows hold row t: the last one that starts at or before
// t.  All 32 lanes search together, 32 probes a step.
__device__ __forceinline__ int find_sequence(const b2g_kv_batch& b, int t, int lane) {
  int lo = 0, n = b.batch;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lane * step;
    const bool in = at < n && b.q_start[lo + at] <= t;
    const int last = max(__popc(__ballot_sync(0xffffffffu, in)) - 1, 0) * step;
    lo += last;
    n = min(step, n - last);
  }
  return lo;
}

// The page of token position pos of sequence s, or -1 (with the error word
// set) where the table or the cache does not have it.
__device__ __forceinline__ int page_of(const b2g_kv_batch& b, const b2g_kv_cache& c, int s, int page_index,
                                       int* error) {
  int page = -1;
  if (page_index < b.max_pages) page = b.page_table[(long long)s * b.page_table_stride + page_index];
  if (page < 0 || page >= c.num_pages) {
    *error = kErrBadPage;
    return -1;
  }
  return page;
}

}  // namespace b2g
