// kv_append.cu -- new tokens' keys and values into a paged cache, with the
// position rotation of k and q on the way.
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

// One thread's piece of a head: 16 elements in two 16-byte chunks.
template <typename T>
__device__ __forceinline__ void unpack8(uint4 v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = Act<T>::unpack(w[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float* f) {
  return make_uint4(Act<T>::pack(f[0], f[1]), Act<T>::pack(f[2], f[3]), Act<T>::pack(f[4], f[5]),
                    Act<T>::pack(f[6], f[7]));
}

// One block per row: its 16-element pieces (q heads, then k heads, then v
// heads) over the threads.  Piece i of a rotated head uses the frequencies
// 8i .. 8i + 7: the halves style pairs elements 8i.. with n_freq + 8i.., the
// interleaved style the elements 16i .. 16i + 15 among themselves.
template <typename T, bool FP8>
__global__ void __launch_bounds__(256) kv_append_kernel(const KvAppendParams p) {
  __shared__ float2 rot[128];
  const int t = blockIdx.x;
  const int lane = threadIdx.x & 31;
  const int s = find_sequence(p.b, t, lane);
  const SeqSpan q = seq_span(p.b, s);
  if (t < q.first || t >= q.first + q.n) return;  // a row behind the last sequence
  const int pos = q.ctx + (t - q.first);
  const int n_freq = p.a.n_freq;
  if ((int)threadIdx.x < n_freq) rot[threadIdx.x] = sin_cos(pos, p.a.inv_freq[threadIdx.x]);
  long long slot = -1;
  if (pos >= 0) {
    const int page_index = pos / p.c.page_size;
    const int page = page_of(p.b, p.c, s, page_index, p.error);
    if (page >= 0)
      slot = page * p.c.stride_page + (long long)(pos - page_index * p.c.page_size) * p.c.stride_token;
  }
  __syncthreads();
  const int per_head = p.c.head_dim / 16;
  const int n_q = p.a.q_heads * per_head, n_k = p.c.kv_heads * per_head;
  for (int i = threadIdx.x; i < n_q + 2 * n_k; i += blockDim.x) {
    const int kind = i < n_q ? 0 : i < n_q + n_k ? 1 : 2;
    const int local = kind == 0 ? i : kind == 1 ? i - n_q : i - n_q - n_k;
    const int head = local / per_head, piece = local - head * per_head;
    if (kind != 0 && slot < 0) continue;
    const bool turned = kind != 2 && piece * 8 < n_freq;
    // Elements of the two chunks: the pair partner is n_freq away, or the
    // next chunk; pieces behind the rotated part are plain neighbours.
    const bool halves = turned && !p.a.interleaved;
    const int e0 = halves ? 8 * piece : 16 * piece, e1 = halves ? e0 + n_freq : e0 + 8;
    const T* src = kind == 0   ? static_cast<const T*>(p.a.q) + t * p.a.stride_q + head * p.a.stride_q_head
                   : kind == 1 ? static_cast<const T*>(p.a.k) + t * p.a.stride_k + head * p.a.stride_k_head
                               : static_cast<const T*>(p.a.v) + t * p.a.stride_v + head * p.a.stride_v_head;
    float a[8], b[8];
    unpack8<T>(*reinterpret_cast<const uint4*>(src + e0), a);
    unpack8<T>(*reinterpret_cast<const uint4*>(src + e1), b);
    if (turned) {
      const float2* r = rot + 8 * piece;
      if (halves) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = a[j], y = b[j];
          a[j] = x * r[j].y - y * r[j].x;
          b[j] = y * r[j].y + x * r[j].x;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x = a[2 * j], y = a[2 * j + 1];
          a[2 * j] = x * r[j].y - y * r[j].x;
          a[2 * j + 1] = y * r[j].y + x * r[j].x;
          x = b[2 * j], y = b[2 * j + 1];
          b[2 * j] = x * r[4 + j].y - y * r[4 + j].x;
          b[2 * j + 1] = y * r[4 + j].y + x * r[4 + j].x;
        }
      }
    }
    if (kind == 0) {
      T* dst = static_cast<T*>(p.a.q_out) + t * p.a.stride_qo + head * p.a.stride_qo_head;
      *reinterpret_cast<uint4*>(dst + e0) = pack8<T>(a);
      *reinterpret_cast<uint4*>(dst + e1) = pack8<T>(b);
      continue;
    }
    const long long at = slot + head * p.c.stride_head;
    void* base = kind == 1 ? p.c.k : p.c.v;
    if constexpr (FP8) {
      const float* scale = kind == 1 ? p.c.k_scale : p.c.v_scale;
      const float sc = scale ? scale[head] : 1.0f;
      uint8_t* dst = static_cast<uint8_t*>(base) + at;
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        w[j] = e4m3_pair(a[4 * j] / sc, a[4 * j + 1] / sc) | e4m3_pair(a[4 * j + 2] / sc, a[4 * j + 3] / sc) << 16;
        w[2 + j] = e4m3_pair(b[4 * j] / sc, b[4 * j + 1] / sc) | e4m3_pair(b[4 * j + 2] / sc, b[4 * j + 3] / sc) << 16;
      }
      *reinterpret_cast<uint2*>(dst + e0) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(dst + e1) = make_uint2(w[2], w[3]);
    } else {
      T* dst = static_cast<T*>(base) + at;
      *reinterpret_cast<uint4*>(dst + e0) = pack8<T>(a);
      *reinterpret_cast<uint4*>(dst + e1) = pack8<T>(b);
    }
  }
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendParams& p, cudaStream_t stream) {
  const bool fp8 = p.c.dtype == B2G_DTYPE_FP8_E4M3;
  const dim3 grid(p.b.rows), block(256);
  if (p.a.dtype == B2G_DTYPE_BF16) {
    if (fp8) kv_append_kernel<__nv_bfloat16, true><<<grid, block, 0, stream>>>(p);
    else kv_append_kernel<__nv_bfloat16, false><<<grid, block, 0, stream>>>(p);
  } else {
    if (fp8) kv_append_kernel<__half, true><<<grid, block, 0, stream>>>(p);
    else kv_append_kernel<__half, false><<<grid, block, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace b2g
