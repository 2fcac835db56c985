// attention.cu -- attention of new tokens over a paged key/value cache.
#include "serve.cuh"

namespace b2g {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// One block of four warps per (row, head); a lane holds D / 32 elements, a
// warp takes every fourth cached token with a running maximum and sum.
template <typename T, bool FP8, int D>
__global__ void __launch_bounds__(128) attention_kernel(const AttnParams p) {
  constexpr int E = D / 32;
  __shared__ float sh_m[4], sh_l[4], sh_o[4][D];
  const int t = blockIdx.x, h = blockIdx.y, kvh = h / p.group;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int s = find_sequence(p.b, t, lane);
  const SeqSpan span = seq_span(p.b, s);
  if (t < span.first || t >= span.first + span.n) return;
  const int pos = span.ctx + (t - span.first);
  const T* q = static_cast<const T*>(p.a.q) + t * p.a.stride_q + h * p.a.stride_q_head;
  const float ks = (FP8 && p.c.k_scale) ? p.c.k_scale[kvh] : 1.0f;
  const float vs = (FP8 && p.c.v_scale) ? p.c.v_scale[kvh] : 1.0f;
  float qf[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qf[e] = Act<T>::to_float(q[lane * E + e]);
    o[e] = 0.f;
  }
  const float scale = p.a.scale * ks * kLog2e;
  float m = -INFINITY, l = 0.f;
  const int lo = p.a.window > 0 ? max(pos - p.a.window + 1, 0) : 0;
  for (int j = lo + warp; j <= pos; j += 4) {
    const int pi = j / p.c.page_size;
    const int page = page_of(p.b, p.c, s, pi, p.error);
    if (page < 0) continue;
    const long long at = page * p.c.stride_page + (long long)(j - pi * p.c.page_size) * p.c.stride_token +
                         kvh * p.c.stride_head + lane * E;
    float k[E], v[E], dot = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (FP8) {
        k[e] = __half2float(__ushort_as_half((unsigned short)e4m3x2_to_f16x2(static_cast<const uint8_t*>(p.c.k)[at + e])));
        v[e] = __half2float(__ushort_as_half((unsigned short)e4m3x2_to_f16x2(static_cast<const uint8_t*>(p.c.v)[at + e])));
      } else {
        k[e] = Act<T>::to_float(static_cast<const T*>(p.c.k)[at + e]);
        v[e] = Act<T>::to_float(static_cast<const T*>(p.c.v)[at + e]);
      }
      dot += qf[e] * k[e];
    }
    for (int off = 16; off; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    dot *= scale;
    const float mn = fmaxf(m, dot);
    const float a = exp2f(m - mn), w = exp2f(dot - mn);
    l = l * a + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * a + w * v[e];
    m = mn;
  }
  if (lane == 0) {
    sh_m[warp] = m;
    sh_l[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) sh_o[warp][lane * E + e] = o[e];
  __syncthreads();
  if (warp) return;
  const float mm = fmaxf(fmaxf(sh_m[0], sh_m[1]), fmaxf(sh_m[2], sh_m[3]));
  float ll = 0.f, oo[E];
#pragma unroll
  for (int e = 0; e < E; ++e) oo[e] = 0.f;
  for (int w = 0; w < 4; ++w) {
    const float a = sh_m[w] == -INFINITY ? 0.f : exp2f(sh_m[w] - mm);
    ll += sh_l[w] * a;
#pragma unroll
    for (int e = 0; e < E; ++e) oo[e] += sh_o[w][lane * E + e] * a;
  }
  T* out = static_cast<T*>(p.a.out) + t * p.a.stride_o + h * p.a.stride_o_head;
  const float inv = ll > 0.f ? vs / ll : 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) out[lane * E + e] = Act<T>::from_float(oo[e] * inv);
  if (p.a.lse && lane == 0)
    p.a.lse[(long long)t * p.q_heads + h] = ll > 0.f ? (mm + log2f(ll)) / kLog2e : -INFINITY;
}

template <typename T, bool FP8>
cudaError_t launch_typed(const AttnParams& p, cudaStream_t stream) {
  const dim3 grid(p.b.rows, p.q_heads);
  if (p.c.head_dim == 128) attention_kernel<T, FP8, 128><<<grid, 128, 0, stream>>>(p);
  else attention_kernel<T, FP8, 64><<<grid, 128, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attention(const AttnParams& p, cudaStream_t stream) {
  const bool fp8 = p.c.dtype == B2G_DTYPE_FP8_E4M3;
  if (p.bf16) return fp8 ? launch_typed<__nv_bfloat16, true>(p, stream) : launch_typed<__nv_bfloat16, false>(p, stream);
  return fp8 ? launch_typed<__half, true>(p, stream) : launch_typed<__half, false>(p, stream);
}

}  // namespace b2g
