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
constexpr int kErrAlignment = 7;  // shared memory not placed as a kernel needs it

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

// 16 bytes of activations, widened.
template <typename T>
__device__ __forceinline__ void unpack8(uint4 v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = Act<T>::unpack(w[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}

// One sequence's rows and cached length, clamped to what the buffers hold.
struct SeqSpan {
  int first, n;  // its rows are first .. first + n - 1
  int ctx;       // position of its row 0 (negative: more rows than the length counts)
};
__host__ __device__ __forceinline__ SeqSpan seq_span(const b2g_kv_batch& b, int s) {
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
__host__ __device__ __forceinline__ int page_of(const b2g_kv_batch& b, const b2g_kv_cache& c, int s, int page_index,
                                       int* error) {
  int page = -1;
  if (page_index < b.max_pages) page = b.page_table[(long long)s * b.page_table_stride + page_index];
  if (page < 0 || page >= c.num_pages) {
    *error = kErrBadPage;
    return -1;
  }
  return page;
}

// a * b / c; short work's products fit 32 bits, whose division is a fraction
// of the 64-bit one's time.
__host__ __device__ __forceinline__ long long mul_div(long long a, int b, long long c) {
  const unsigned long long n = (unsigned long long)a * b;
  if ((n | (unsigned long long)c) >> 32 == 0) return (unsigned)n / (unsigned)c;
  return (long long)(n / (unsigned long long)c);
}
// ---------------------------------------------------------------------------
// The attention kernels' work list.  An item is (sequence, tile of rows, k/v
// head): the rows of a k/v head are its new tokens times its group of q
// heads, row r being token r / group and head r % group of the group.  An
// item's visible cached tokens are cut into units of UNIT tokens; the units
// of all items in order are dealt to the blocks in equal consecutive ranges,
// so that long contexts, many short ones and ragged mixtures all fill the
// GPU, from lengths that only the device knows.  A range's first and last
// item may be shared with other blocks.
// ---------------------------------------------------------------------------
struct AttnItem {
  SeqSpan s;
  int b, tile, h;
  int lo, hi;      // visible cached tokens [lo, hi)
  int u_lo, u_hi;  // units [u_lo, u_hi), at least one
};

template <int ROWS, int UNIT>
struct AttnWork {
  const AttnParams& p;
  int cap;  // tokens that the page table has entries for
  __host__ __device__ __forceinline__ explicit AttnWork(const AttnParams& p_) : p(p_) {
    cap = (int)min((long long)p_.b.max_pages * p_.c.page_size, 0x7fffffffLL - UNIT);
  }
  __host__ __device__ __forceinline__ int tiles(const SeqSpan& s) const { return (s.n * p.group + ROWS - 1) / ROWS; }
  __host__ __device__ __forceinline__ void range(AttnItem& it) const {
    const int first = it.tile * ROWS / p.group;
    const int last = min(it.s.n - 1, (it.tile * ROWS + ROWS - 1) / p.group);
    if (it.s.ctx + last >= cap) *p.error = kErrBadPage;
    it.hi = max(min(it.s.ctx + last + 1, cap), 0);
    it.lo = p.a.window > 0 ? min(max(it.s.ctx + first - p.a.window + 1, 0), it.hi) : 0;
    it.u_lo = it.lo / UNIT;
    it.u_hi = max((it.hi + UNIT - 1) / UNIT, it.u_lo + 1);
  }
  // Units of a sequence's items; *longer is set if they are more than four on
  // average.
  __host__ __device__ __forceinline__ long long units(int b, bool* longer = nullptr) const {
    AttnItem it;
    it.s = seq_span(p.b, b);
    long long n = 0;
    const int nt = tiles(it.s);
    for (it.tile = 0; it.tile < nt; ++it.tile) {
      range(it);
      n += it.u_hi - it.u_lo;
    }
    if (longer) *longer |= n > 4LL * nt;
    return n * p.c.kv_heads;
  }
  // The item that holds unit `at` of sequence b; `at` becomes the unit's
  // offset in the item.
  __host__ __device__ __forceinline__ AttnItem find(int b, long long& at) const {
    AttnItem it;
    it.b = b;
    it.s = seq_span(p.b, b);
    for (it.tile = 0;; ++it.tile) {
      range(it);
      const long long n = (long long)(it.u_hi - it.u_lo) * p.c.kv_heads;
      if (at < n) break;
      at -= n;
    }
    it.h = (int)mul_div(at, 1, it.u_hi - it.u_lo);
    at -= (long long)it.h * (it.u_hi - it.u_lo);
    return it;
  }
  // The next item in order (false: none left).
  __host__ __device__ __forceinline__ bool next(AttnItem& it) const {
    if (++it.h < p.c.kv_heads) return true;
    it.h = 0;
    if (++it.tile < tiles(it.s)) {
      range(it);
      return true;
    }
    it.tile = 0;
    while (++it.b < p.b.batch) {
      it.s = seq_span(p.b, it.b);
      if (it.s.n > 0) {
        range(it);
        return true;
      }
    }
    return false;
  }
};

// A block's place in the work list.
struct AttnShare {
  long long total, begin, end;  // units
  int blocks;                   // that share the list; others have none
  int b;                        // the sequence of unit `begin`,
  long long at;                 // and the unit's offset in it
};

// The unit that block c's range begins with.
__host__ __device__ __forceinline__ long long attn_begin(const AttnShare& s, int c) { return mul_div(s.total, c, s.blocks); }

// Sums the list (all threads; sh: a word a warp, two at least) and finds the block's
// range.  At least `least` units a block, so that short work is not cut finer
// than the joining of its pieces is worth; BY_LENGTH: one, where no sequence's
// items are longer than four units (a block that takes several short items has
// them one after the other).
template <bool BY_LENGTH, typename Work>
__device__ __forceinline__ AttnShare attn_share(const Work& w, int least, long long* sh) {
  const int threads = blockDim.x, batch = w.p.b.batch;
  const int per = (batch + threads - 1) / threads;
  const int b0 = min((int)threadIdx.x * per, batch), b1 = min(b0 + per, batch);
  long long sum = 0;
  bool longer = false;
  for (int b = b0; b < b1; ++b) sum += w.units(b, BY_LENGTH ? &longer : nullptr);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long incl = sum;
#pragma unroll
  for (int off = 1; off < 32; off *= 2) {
    const long long o = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += o;
  }
  if (lane == 31) sh[warp] = incl;
  if (!BY_LENGTH)
    __syncthreads();
  else if (!__syncthreads_or(longer))
    least = 1;
  long long before = 0, total = 0;
  for (int i = 0; i < threads / 32; ++i) {
    if (i < warp) before += sh[i];
    total += sh[i];
  }
  __syncthreads();
  AttnShare r;
  r.total = total;
  r.blocks = (int)max(1LL, min((long long)gridDim.x, (total + least - 1) / least));
  r.begin = attn_begin(r, blockIdx.x);
  r.end = attn_begin(r, blockIdx.x + 1);
  if ((int)blockIdx.x >= r.blocks) r.begin = r.end = total;
  // The thread whose sequences hold `begin` tells the others.
  const long long from = before + incl - sum;
  if (r.begin >= from && r.begin < from + sum) {
    long long at = r.begin - from;
    int b = b0;
    for (long long n; at >= (n = w.units(b)); ++b) at -= n;
    sh[0] = b;
    sh[1] = at;
  }
  __syncthreads();
  r.b = (int)sh[0];
  r.at = sh[1];
  __syncthreads();
  return r;
}
// The block that has unit u.
__host__ __device__ __forceinline__ int attn_owner(const AttnShare& s, long long u) {
  const unsigned long long n = (unsigned long long)(u + 1) * s.blocks - 1;
  if ((n | (unsigned long long)s.total) >> 32 == 0) return (int)((unsigned)n / (unsigned)s.total);
  return (int)(n / (unsigned long long)s.total);
}

}  // namespace b2g
