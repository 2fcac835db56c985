// i8.cu -- matrix product in 8-bit integers with a scale for each row of x
// and each output channel, and the quantisers that make its operands.
#include "serve.cuh"

namespace b2g {
namespace {

// v / s rounded to the nearest integer, ties to even (a row that is not
// finite has s = NaN and zero codes).
__device__ __forceinline__ int code_of(float v, float s) { return s == s ? __float2int_rn(v / s) : 0; }
__device__ __forceinline__ float scale_of(float amax) {
  return amax <= 3.4028235e38f ? fmaxf(amax, 1e-12f) / 127.0f : __uint_as_float(0x7fffffffu);
}
// Maximum that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) { return a > b || a != a ? a : b; }

template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const I8RowsParams p) {
  __shared__ float red[8];
  const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* gamma = static_cast<const T*>(p.gamma);
  float r = 1.0f;
  if (p.rmsnorm) {
    float ss = 0.f;
    for (int i = threadIdx.x; i < p.k; i += 256) {
      const float v = Act<T>::to_float(x[i]);
      ss += v * v;
    }
    for (int off = 16; off; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    if (lane == 0) red[warp] = ss;
    __syncthreads();
    ss = 0.f;
    for (int w = 0; w < 8; ++w) ss += red[w];
    r = rsqrtf(ss / (float)p.k + p.eps);
    __syncthreads();
  }
  float a = 0.f;
  for (int i = threadIdx.x; i < p.k; i += 256) {
    float v = Act<T>::to_float(x[i]) * r;
    if (gamma) v *= Act<T>::to_float(gamma[i]);
    a = max_nan(a, fabsf(v));
  }
  for (int off = 16; off; off >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, off));
  if (lane == 0) red[warp] = a;
  __syncthreads();
  for (int w = 0; w < 8; ++w) a = max_nan(a, red[w]);
  const float s = scale_of(a);
  for (int i = threadIdx.x; i < p.k; i += 256) {
    float v = Act<T>::to_float(x[i]) * r;
    if (gamma) v *= Act<T>::to_float(gamma[i]);
    p.codes[row * p.ldc + i] = (int8_t)code_of(v, s);
  }
  if (threadIdx.x == 0) p.scales[row] = s;
}

// One-off: 32 output channels a block, both passes over K.
template <typename T>
__global__ void __launch_bounds__(1024) quantize_weights_kernel(const T* __restrict__ w, int K, int N, int layout,
                                                                int8_t* __restrict__ codes, long long ldc,
                                                                float* __restrict__ scales) {
  __shared__ float tile[32][33];
  __shared__ float sc[32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int n0 = blockIdx.x * 32;
  float a = 0.f;
  // KN: lanes over channels; NK: lanes over k, a warp per channel.
  if (layout == B2G_LAYOUT_KN) {
    if (n0 + tx < N)
      for (int k = ty; k < K; k += 32) a = max_nan(a, fabsf(Act<T>::to_float(w[(long long)k * N + n0 + tx])));
    tile[ty][tx] = a;
  } else {
    if (n0 + ty < N)
      for (int k = tx; k < K; k += 32) a = max_nan(a, fabsf(Act<T>::to_float(w[(long long)(n0 + ty) * K + k])));
    tile[tx][ty] = a;
  }
  __syncthreads();
  if (ty == 0) {
    for (int i = 0; i < 32; ++i) a = max_nan(a, tile[i][tx]);
    sc[tx] = scale_of(a);
    if (n0 + tx < N) scales[n0 + tx] = sc[tx];
  }
  __syncthreads();
  for (int k0 = 0; k0 < K; k0 += 32) {
    if (layout == B2G_LAYOUT_KN) {
      if (k0 + ty < K && n0 + tx < N) tile[ty][tx] = Act<T>::to_float(w[(long long)(k0 + ty) * N + n0 + tx]);
      __syncthreads();
      if (n0 + ty < N && k0 + tx < K) codes[(n0 + ty) * ldc + k0 + tx] = (int8_t)code_of(tile[tx][ty], sc[ty]);
      __syncthreads();
    } else if (n0 + ty < N && k0 + tx < K) {
      codes[(n0 + ty) * ldc + k0 + tx] =
          (int8_t)code_of(Act<T>::to_float(w[(long long)(n0 + ty) * K + k0 + tx]), sc[ty]);
    }
  }
}

// acc -> y of one element.
template <typename T>
__device__ __forceinline__ void finish(const I8Params& p, int i, int j, int acc, int acc_up) {
  float v = (float)acc * p.sx[i] * p.sw[j];
  if (p.planes == 2) {
    const float u = (float)acc_up * p.sx[i] * p.sw[p.n + j];
    v = v / (1.0f + __expf(-v)) * u;
  }
  if (p.residual) v += Act<T>::to_float(static_cast<const T*>(p.residual)[i * p.ldr + j]);
  static_cast<T*>(p.y)[i * p.ldy + j] = Act<T>::from_float(v);
}

// 32 x 32 outputs a block, 32 k a step.
template <typename T>
__global__ void __launch_bounds__(256) product_kernel(const I8Params p) {
  __shared__ int xs[32][9], ws[2][32][9];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int i0 = blockIdx.y * 32, j0 = blockIdx.x * 32;
  int acc[2][4] = {};
  for (int k0 = 0; k0 < p.k; k0 += 32) {
    const int r = threadIdx.x >> 3, c = threadIdx.x & 7;
    auto load = [&](const int8_t* row, bool in) {
      const int k = k0 + 4 * c;
      if (!in || k >= p.k) return 0;
      unsigned v = *reinterpret_cast<const unsigned*>(row + k);
      if (p.k - k < 4) v &= (1u << (8 * (p.k - k))) - 1;
      return (int)v;
    };
    xs[r][c] = load(p.x + (i0 + r) * p.ldx, i0 + r < p.m);
    for (int pl = 0; pl < p.planes; ++pl)
      ws[pl][r][c] = load(p.w + ((long long)pl * p.n + j0 + r) * p.ldw, j0 + r < p.n);
    __syncthreads();
    for (int c2 = 0; c2 < 8; ++c2)
      for (int u = 0; u < 4; ++u)
        for (int pl = 0; pl < p.planes; ++pl) acc[pl][u] = __dp4a(xs[ty + 8 * u][c2], ws[pl][tx][c2], acc[pl][u]);
    __syncthreads();
  }
  for (int u = 0; u < 4; ++u)
    if (i0 + ty + 8 * u < p.m && j0 + tx < p.n) finish<T>(p, i0 + ty + 8 * u, j0 + tx, acc[0][u], acc[1][u]);
}

}  // namespace

cudaError_t launch_i8_quantize_rows(const I8RowsParams& p, cudaStream_t stream) {
  if (p.bf16) quantize_rows_kernel<__nv_bfloat16><<<p.m, 256, 0, stream>>>(p);
  else quantize_rows_kernel<__half><<<p.m, 256, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_i8_quantize_weights(const void* w, int K, int N, int layout, int bf16, int8_t* codes,
                                       long long ldc, float* scales, cudaStream_t stream) {
  const int grid = (N + 31) / 32;
  if (bf16)
    quantize_weights_kernel<<<grid, 1024, 0, stream>>>(static_cast<const __nv_bfloat16*>(w), K, N, layout, codes,
                                                       ldc, scales);
  else
    quantize_weights_kernel<<<grid, 1024, 0, stream>>>(static_cast<const __half*>(w), K, N, layout, codes, ldc,
                                                       scales);
  return cudaGetLastError();
}

cudaError_t launch_i8_product(const I8Params& p, cudaStream_t stream) {
  const dim3 grid((p.n + 31) / 32, (p.m + 31) / 32);
  if (p.bf16) product_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(p);
  else product_kernel<__half><<<grid, 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace b2g
