// kv_append.cu -- new tokens' keys and values into a paged cache, with the
// position rotation of k and q on the way.  Bound by memory: 14,000 rows into an
// 8-bit cache 69 us, 0.78 of a copy's rate; a decode step of 64 rows 3.2 us, its
// launch.
#include <algorithm>

#include "serve.cuh"

namespace b2g {
namespace {

// sin and cos of pos * freq.  The product and its reduction to a fraction of
// a turn are in 64 bits: at position 10^5 a 32-bit angle is off by up to 4e-3.
__device__ __forceinline__ float2 sin_cos(int pos, float freq) {
  const double turns = (double)pos * (double)freq * 0.15915494309189533577;  // 1 / (2 pi)
  const float frac = (float)(turns - rint(turns));
  float s, c;
  sincospif(2.0f * frac, &s, &c);
  return make_float2(s, c);
}

__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}

// Codes of eight values divided by s, each the fp32 quotient rounded.  Apart from
// the product with 1 / s, so that its code (64 copies of a division) stays out of
// the row loop's: 73 us with it there.
__device__ __noinline__ uint2 e4m3_divided(float4 a, float4 b, float s) {
  return make_uint2(e4m3_pair(a.x / s, a.y / s) | e4m3_pair(a.z / s, a.w / s) << 16,
                    e4m3_pair(b.x / s, b.y / s) | e4m3_pair(b.z / s, b.w / s) << 16);
}
// The same.  `below` and `above` are 1 / s less and plus 2^-21 of it: a product with
// 1 / s is off from the quotient by less than that (half a step, 2^-24, each for
// 1 / s, the product, `below` itself and the quotient), so the quotient lies between
// the two products, and where their codes agree it has the same.  Where not (one
// value in 50,000, and values on a tie, which a product alone leaves on either side)
// it is divided.  14,000 rows into an 8-bit cache: 69 us; 65 with the product alone,
// 86 with divisions only.
__device__ __forceinline__ uint2 e4m3_quotients(const float* v, float s, float below, float above) {
  uint32_t lo[2], hi[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float* x = v + 4 * j;
    lo[j] = e4m3_pair(x[0] * below, x[1] * below) | e4m3_pair(x[2] * below, x[3] * below) << 16;
    hi[j] = e4m3_pair(x[0] * above, x[1] * above) | e4m3_pair(x[2] * above, x[3] * above) << 16;
  }
  if (lo[0] == hi[0] && lo[1] == hi[1]) return make_uint2(lo[0], lo[1]);
  return e4m3_divided(make_float4(v[0], v[1], v[2], v[3]), make_float4(v[4], v[5], v[6], v[7]), s);
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float* f) {
  return make_uint4(Act<T>::pack(f[0], f[1]), Act<T>::pack(f[2], f[3]), Act<T>::pack(f[4], f[5]),
                    Act<T>::pack(f[6], f[7]));
}

// A block takes `rows` rows, a thread the same two 8-element chunks of a q, k
// or v head in each of them, so what they are gets worked out once (by row and
// chunk in turn the divisions took as long as the memory traffic).  The rows'
// chunks are asked for before the rows' places and angles are worked out,
// which take a chain of dependent reads.
constexpr int kMostThreads = 384, kMaxRows = 4;

template <typename T, bool FP8>
__global__ void __launch_bounds__(kMostThreads, 2) kv_append_kernel(const KvAppendParams p, int rows) {
  __shared__ __align__(16) float2 rot[kMaxRows][64];
  __shared__ long long slot_sh[kMaxRows];
  __shared__ bool in_sh[kMaxRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row0 = blockIdx.x * rows, n_rows = min(rows, p.b.rows - row0);
  const int n_freq = p.a.n_freq;
  const int per_head = p.c.head_dim / 16;
  const int n_q = p.a.q_heads * per_head, n_k = p.c.kv_heads * per_head, per_row = n_q + 2 * n_k;
  pdl_wait();
  pdl_launch_dependents();
  for (int item = threadIdx.x; item < per_row || item == (int)threadIdx.x; item += blockDim.x) {
    const bool mine = item < per_row;
    const int kind = item < n_q ? 0 : item < n_q + n_k ? 1 : 2;
    const int local = item - (kind == 0 ? 0 : kind == 1 ? n_q : n_q + n_k);
    const int head = local / per_head, at = local - head * per_head;
    // Two 8-element chunks half a head apart, so that a warp's accesses are
    // whole lines (16 elements a thread in one run leave every 32-byte sector to
    // two instructions: 90 us for 14,000 rows of 48 heads, 66 so).  Halves that are shorter
    // than that pair over n_freq, and what is behind them is in runs of 16.
    const bool halves_style = kind != 2 && !p.a.interleaved && n_freq > 0;
    const bool halves = halves_style && at * 8 < n_freq;
    const int e0 = halves_style && !halves ? 16 * at : 8 * at;
    const int e1 = halves ? e0 + n_freq : halves_style ? e0 + 8 : e0 + p.c.head_dim / 2;
    const bool pairs = kind != 2 && p.a.interleaved;
    const bool pairs0 = pairs && e0 < 2 * n_freq, pairs1 = pairs && e1 < 2 * n_freq;
    const T* src = static_cast<const T*>(kind == 0 ? p.a.q : kind == 1 ? p.a.k : p.a.v);
    const long long step = kind == 0 ? p.a.stride_q : kind == 1 ? p.a.stride_k : p.a.stride_v;
    src += row0 * step + head * (kind == 0 ? p.a.stride_q_head : kind == 1 ? p.a.stride_k_head : p.a.stride_v_head);
    uint4 lo[kMaxRows], hi[kMaxRows];
#pragma unroll
    for (int u = 0; u < kMaxRows; ++u)
      if (mine && u < n_rows) {
        lo[u] = *reinterpret_cast<const uint4*>(src + u * step + e0);
        hi[u] = *reinterpret_cast<const uint4*>(src + u * step + e1);
      }
    if (item == (int)threadIdx.x) {  // the first time round: every thread is here
      if (warp < n_rows) {
        const int t = row0 + warp;
        const int s = find_sequence(p.b, t, lane);
        const SeqSpan q = seq_span(p.b, s);
        const bool in = t >= q.first && t < q.first + q.n;  // else a row behind the last sequence
        const int pos = q.ctx + (t - q.first);
        for (int i = lane; in && i < n_freq; i += 32) rot[warp][i] = sin_cos(pos, p.a.inv_freq[i]);
        long long slot = -1;
        if (in && pos >= 0) {
          const int page_index = pos / p.c.page_size;
          const int page = page_of(p.b, p.c, s, page_index, p.error);
          if (page >= 0)
            slot = page * p.c.stride_page + (long long)(pos - page_index * p.c.page_size) * p.c.stride_token;
        }
        if (lane == 0) {
          slot_sh[warp] = slot;
          in_sh[warp] = in;
        }
      }
      __syncthreads();
    }
    float by = 1.0f, below = 1.0f, above = 1.0f;  // no scale: the value itself
    if constexpr (FP8) {
      const float* scale = kind == 1 ? p.c.k_scale : p.c.v_scale;
      if (mine && kind != 0 && scale) {
        by = scale[head];
        const float inv = 1.0f / by;
        // 1 / s far out in fp32's range: codes that never agree.
        const bool normal = inv >= 0x1p-120f && inv <= 0x1p120f;
        below = normal ? inv * (1.0f - 0x1p-21f) : 0.0f;
        above = normal ? inv * (1.0f + 0x1p-21f) : INFINITY;
      }
    }
#pragma unroll
    for (int u = 0; u < kMaxRows; ++u) {
      if (!mine || u >= n_rows) continue;
      const long long slot = slot_sh[u];
      if (!in_sh[u] || (kind != 0 && slot < 0)) continue;
      float a[8], b[8];
      unpack8<T>(lo[u], a);
      unpack8<T>(hi[u], b);
      if (halves) {
        const float4* r4 = reinterpret_cast<const float4*>(rot[u] + e0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 r = r4[j];  // sine and cosine of two frequencies
          float x = a[2 * j], y = b[2 * j];
          a[2 * j] = x * r.y - y * r.x;
          b[2 * j] = y * r.y + x * r.x;
          x = a[2 * j + 1], y = b[2 * j + 1];
          a[2 * j + 1] = x * r.w - y * r.z;
          b[2 * j + 1] = y * r.w + x * r.z;
        }
      }
      auto turn_pairs = [&](float (&v)[8], int e) {
        const float4* r4 = reinterpret_cast<const float4*>(rot[u] + e / 2);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float4 r = r4[j];
          float x = v[4 * j], y = v[4 * j + 1];
          v[4 * j] = x * r.y - y * r.x;
          v[4 * j + 1] = y * r.y + x * r.x;
          x = v[4 * j + 2], y = v[4 * j + 3];
          v[4 * j + 2] = x * r.w - y * r.z;
          v[4 * j + 3] = y * r.w + x * r.z;
        }
      };
      if (pairs0) turn_pairs(a, e0);
      if (pairs1) turn_pairs(b, e1);
      if (kind == 0) {
        T* dst = static_cast<T*>(p.a.q_out) + (row0 + u) * p.a.stride_qo + head * p.a.stride_qo_head;
        *reinterpret_cast<uint4*>(dst + e0) = pack8<T>(a);
        *reinterpret_cast<uint4*>(dst + e1) = pack8<T>(b);
        continue;
      }
      const long long to = slot + head * p.c.stride_head;
      void* cache = kind == 1 ? p.c.k : p.c.v;
      if constexpr (FP8) {
        uint8_t* dst = static_cast<uint8_t*>(cache) + to;
        *reinterpret_cast<uint2*>(dst + e0) = e4m3_quotients(a, by, below, above);
        *reinterpret_cast<uint2*>(dst + e1) = e4m3_quotients(b, by, below, above);
      } else {
        T* dst = static_cast<T*>(cache) + to;
        *reinterpret_cast<uint4*>(dst + e0) = pack8<T>(a);
        *reinterpret_cast<uint4*>(dst + e1) = pack8<T>(b);
      }
    }
  }
}

template <typename T, bool FP8>
cudaError_t launch(const KvAppendParams& p, int num_sms, cudaStream_t stream) {
  // Rows a block: one while the rows are few (latency), else as many as keep
  // four blocks an SM.
  const int rows = std::min(kMaxRows, std::max(1, p.b.rows / (4 * num_sms)));
  const int per_row = (p.a.q_heads + 2 * p.c.kv_heads) * p.c.head_dim / 16;
  const int threads = std::min(kMostThreads, std::max(32 * kMaxRows, (per_row + 31) / 32 * 32));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.b.rows + rows - 1) / rows);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv_append_kernel<T, FP8>, p, rows);
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendParams& p, int num_sms, cudaStream_t stream) {
  const bool fp8 = p.c.dtype == B2G_DTYPE_FP8_E4M3;
  if (p.a.dtype == B2G_DTYPE_BF16)
    return fp8 ? launch<__nv_bfloat16, true>(p, num_sms, stream) : launch<__nv_bfloat16, false>(p, num_sms, stream);
  return fp8 ? launch<__half, true>(p, num_sms, stream) : launch<__half, false>(p, num_sms, stream);
}

}  // namespace b2g
