// i8.cu -- matrix product in 8-bit integers with a scale for each row of x
// and each output channel, and the quantisers that make its operands.
#include "serve.cuh"
#include "tc.cuh"

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
  pdl_launch_dependents();
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

// ---------------------------------------------------------------------------
// The product.  D[channel, token] = sum_k w[channel, k] x[token, k]: a tile is
// 128 channels (A: M = 128) by bn tokens (B: N = bn, 32..256), so that a
// decode step's few tokens waste no more than a narrow N, and both planes of
// gate||up land in the same thread (lane = channel).
//
// One persistent CTA per SM.  Warp 0 streams 128-byte k blocks of both
// operands through a ring of stages (TMA, 128-byte swizzle, zeros outside the
// matrices), warp 1 issues tcgen05.mma.kind::i8 into one of two accumulators
// in tensor memory, warps 2..5 drain the other one.  Work is cut as whole
// tiles where they fill the SMs, else as equal ranges of k blocks ("units"):
// a range's tiles at its two ends are shared with other CTAs, which leave
// their int32 sums in the workspace; the last to arrive adds them (integer
// sums: the order does not matter) and finishes the tile.
// ---------------------------------------------------------------------------
constexpr int kI8Threads = 192;
constexpr int kI8MaxStages = 12;
constexpr int kKBlock = 128;
constexpr int kChTile = 128;
constexpr int kI8SmemBytes = 200 * 1024 + 1024;  // ring and its alignment

struct I8Tc {
  CUtensorMap mw, mx;
  I8Params p;
  int bn, stages, kb, tok_tiles, tiles, whole;
  int tmem_cols;
  long long units;
  long long slot_ints;  // int32 words of one partial
  int* counters;        // [grid], zero between launches
  int* partials;        // [grid][2][slot_ints]
  int* error;
};

// The pieces of this CTA's work: k blocks [k0, k1) of a tile.
struct I8Seg {
  long long u, end;  // units (split) or tiles (whole)
  int tile, k0, k1;
  __device__ __forceinline__ void begin(const I8Tc& t) {
    const int c = blockIdx.x, g = gridDim.x;
    u = t.whole ? c : c * t.units / g;
    end = t.whole ? t.tiles : (c + 1) * t.units / g;
  }
  __device__ __forceinline__ bool next(const I8Tc& t) {
    if (u >= end) return false;
    if (t.whole) {
      tile = (int)u;
      k0 = 0;
      k1 = t.kb;
      u += gridDim.x;
    } else {
      tile = (int)(u / t.kb);
      k0 = (int)(u - (long long)tile * t.kb);
      k1 = (int)min((long long)t.kb, k0 + (end - u));
      u += k1 - k0;
    }
    return true;
  }
};

__device__ __forceinline__ int i8_owner(const I8Tc& t, long long u) {
  return (int)(((u + 1) * gridDim.x - 1) / t.units);
}

template <typename T, int PLANES>
__global__ void __launch_bounds__(kI8Threads, 1) i8_product_kernel(const __grid_constant__ I8Tc t) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[kI8MaxStages], empty[kI8MaxStages], acc_full[2], acc_empty[2], drain;
  __shared__ uint32_t tmem_base_sh;
  __shared__ int last_sh;
  uint8_t* ring = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stage_bytes = PLANES * kChTile * kKBlock + t.bn * kKBlock;
  if (threadIdx.x == 0) {
    for (int i = 0; i < t.stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 128);
    }
    mbar_init(&drain, 1);
    fence_mbarrier_init();
  }
  if (warp == 1) tmem_alloc(&tmem_base_sh, t.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&t.mw);
      tma_prefetch_desc(&t.mx);
      auto load_w = [&](int stage, const I8Seg& s, int k) {
        uint8_t* dst = ring + stage * stage_bytes;
#pragma unroll
        for (int pl = 0; pl < PLANES; ++pl)
          tma_load_2d(dst + pl * kChTile * kKBlock, &t.mw, k * kKBlock, pl * t.p.n + s.tile / t.tok_tiles * kChTile,
                      &full[stage]);
      };
      auto load_x = [&](int stage, const I8Seg& s, int k) {
        tma_load_2d(ring + stage * stage_bytes + PLANES * kChTile * kKBlock, &t.mx, k * kKBlock,
                    s.tile % t.tok_tiles * t.bn, &full[stage]);
      };
      // The first stages' weights do not depend on the launch before this one.
      I8Seg s;
      s.begin(t);
      int issued = 0;
      while (issued < t.stages && s.next(t))
        for (int k = s.k0; k < s.k1 && issued < t.stages; ++k, ++issued) {
          mbar_arrive_expect_tx(&full[issued], stage_bytes);
          load_w(issued, s, k);
        }
      pdl_wait();
      s.begin(t);
      int i = 0;  // k blocks so far
      bool ok = true;
      while (ok && s.next(t))
        for (int k = s.k0; k < s.k1; ++k, ++i) {
          const int stage = i % t.stages;
          if (i >= issued) {
            if (!mbar_wait_bounded(&empty[stage], (i / t.stages - 1) & 1)) {
              *t.error = kErrEmptyWait;
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&full[stage], stage_bytes);
            load_w(stage, s, k);
          }
          load_x(stage, s, k);
        }
      // After an error the copies in flight land before this CTA's memory goes.
      if (!ok)
        for (int j = max(0, i - t.stages); j < i; ++j) mbar_wait_bounded(&full[j % t.stages], (j / t.stages) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = tc_idesc(2, 1, 1, 0, t.bn);  // s32 = s8 * s8
      const uint32_t ring_addr = smem_addr(ring);
      I8Seg s;
      s.begin(t);
      int i = 0, n = 0;
      bool ok = true;
      while (ok && s.next(t)) {
        const int buf = n & 1;
        if (!mbar_wait_bounded(&acc_empty[buf], ((n >> 1) & 1) ^ 1)) {
          *t.error = kErrEmptyWait;
          ok = false;
          break;
        }
        tc_fence_after();
        for (int k = s.k0; k < s.k1; ++k, ++i) {
          const int stage = i % t.stages;
          if (!mbar_wait_bounded(&full[stage], (i / t.stages) & 1)) {
            *t.error = kErrFullWait;
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = ring_addr + stage * stage_bytes;
          const uint64_t db = smem_desc_sw128(a0 + PLANES * kChTile * kKBlock, 16, 1024);
#pragma unroll
          for (int pl = 0; pl < PLANES; ++pl) {
            const uint64_t da = smem_desc_sw128(a0 + pl * kChTile * kKBlock, 16, 1024);
            const uint32_t d = tmem + (buf * PLANES + pl) * t.bn;
#pragma unroll
            for (int j = 0; j < 4; ++j)  // 32 k an instruction: 2 units of 16 bytes
              mma_i8_ss(d, da + 2 * j, db + 2 * j, idesc, k > s.k0 || j > 0);
          }
          tc_commit(&empty[stage]);
        }
        if (ok) tc_commit(&acc_full[buf]);
        ++n;
      }
      if (!ok) {
        tc_commit(&drain);
        mbar_wait_bounded(&drain, 0);
      }
    }
  } else {
    pdl_wait();
    const int quad = warp & 3, et = threadIdx.x - 64;
    const int ch = quad * 32 + lane;  // channel in the tile
    const uint32_t lane_addr = tmem + ((uint32_t)(quad * 32) << 16);
    const I8Params& p = t.p;
    I8Seg s;
    s.begin(t);
    int n = 0;
    while (s.next(t)) {
      const int buf = n & 1;
      const int tok0 = s.tile % t.tok_tiles * t.bn, j = s.tile / t.tok_tiles * kChTile + ch;
      const int cols = min(t.bn, p.m - tok0);
      const bool split = s.k0 != 0 || s.k1 != t.kb;
      float sw[PLANES];
#pragma unroll
      for (int pl = 0; pl < PLANES; ++pl) sw[pl] = j < p.n ? p.sw[pl * p.n + j] : 0.f;
      if (!mbar_wait_bounded(&acc_full[buf], (n >> 1) & 1)) {
        *t.error = kErrFullWait;
        break;
      }
      tc_fence_after();
      int c_first = 0, c_last = 0;
      bool finish = true;
      if (split) {
        c_first = i8_owner(t, (long long)s.tile * t.kb);
        c_last = i8_owner(t, (long long)(s.tile + 1) * t.kb - 1);
        int* mine = t.partials + ((long long)blockIdx.x * 2 + (n > 0)) * t.slot_ints;
        for (int c0 = 0; c0 < cols; c0 += 32) {
#pragma unroll
          for (int pl = 0; pl < PLANES; ++pl) {
            uint32_t r[32];
            tmem_ld32(lane_addr + (buf * PLANES + pl) * t.bn + c0, r);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (c0 + c < cols) __stcg(mine + (pl * t.bn + c0 + c) * kChTile + ch, (int)r[c]);
          }
        }
        __threadfence();
        named_sync(1, 128);
        if (et == 0) {
          const int seen = atom_add_acq_rel_gpu(t.counters + c_first, 1);
          last_sh = seen == c_last - c_first;
          if (last_sh) t.counters[c_first] = 0;
        }
        named_sync(1, 128);
        finish = last_sh != 0;
        __threadfence();
      }
      if (finish) {
        for (int c0 = 0; c0 < cols; c0 += 32) {
          uint32_t r[PLANES][32];
#pragma unroll
          for (int pl = 0; pl < PLANES; ++pl) tmem_ld32(lane_addr + (buf * PLANES + pl) * t.bn + c0, r[pl]);
          tmem_wait_ld();
          if (split) {
            for (int c = c_first; c <= c_last; ++c) {
              if (c == (int)blockIdx.x) continue;
              // Its first range unless it began before this tile.
              const int which = c * t.units / gridDim.x / t.kb != s.tile;
              const int* from = t.partials + ((long long)c * 2 + which) * t.slot_ints;
#pragma unroll
              for (int pl = 0; pl < PLANES; ++pl)
#pragma unroll
                for (int cc = 0; cc < 32; ++cc)
                  if (c0 + cc < cols) r[pl][cc] += __ldcg(from + (pl * t.bn + c0 + cc) * kChTile + ch);
            }
          }
          if (j < p.n) {
#pragma unroll
            for (int cc = 0; cc < 32; ++cc) {
              if (c0 + cc >= cols) break;
              const int i = tok0 + c0 + cc;
              const float sx = p.sx[i];
              float v = (float)(int)r[0][cc] * sw[0] * sx;
              if constexpr (PLANES == 2) {
                const float u = (float)(int)r[1][cc] * sw[1] * sx;
                v = v / (1.0f + __expf(-v)) * u;
              }
              if (p.residual) v += Act<T>::to_float(static_cast<const T*>(p.residual)[i * p.ldr + j]);
              static_cast<T*>(p.y)[i * p.ldy + j] = Act<T>::from_float(v);
            }
          }
        }
      }
      tc_fence_before();
      mbar_arrive(&acc_empty[buf]);
      ++n;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, t.tmem_cols);
}

// cuTensorMapEncodeTiled through the runtime's driver entry point.
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled_fn() {
  static EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}

// Rows of bytes, 128 columns by box_rows a load, zeros outside.
bool encode_rows(CUtensorMap* map, const void* base, long long rows, long long cols, long long ld, int box_rows) {
  const EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {kKBlock, (cuuint32_t)box_rows};
  const cuuint32_t step[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, step,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int up32(int n) { return (n + 31) / 32 * 32; }
// Tokens of a tile for m rows: the fewest tiles of at most 256 / planes
// columns, evened out.
int i8_bn(int m, int planes) {
  const int most = 256 / planes;
  const int tiles = (m + most - 1) / most;
  return up32((m + tiles - 1) / tiles);
}

template <typename T, int PLANES>
cudaError_t launch_product(const I8Tc& t, int grid, int smem, bool pdl, cudaStream_t stream) {
  cudaError_t e = cudaFuncSetAttribute(i8_product_kernel<T, PLANES>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kI8SmemBytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kI8Threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, i8_product_kernel<T, PLANES>, t);
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

size_t i8_partial_bytes(int max_m, int planes, int num_sms) {
  const int most = 256 / planes;
  const int bn = max_m <= most ? up32(max_m) : most;
  return (size_t)num_sms * 2 * planes * bn * kChTile * 4;
}

cudaError_t launch_i8_product(const I8Params& p, int num_sms, int* counters, int* partials, int* error, bool pdl,
                              cudaStream_t stream) {
  I8Tc t;
  t.p = p;
  t.bn = i8_bn(p.m, p.planes);
  const int stage_bytes = (p.planes * kChTile + t.bn) * kKBlock;
  t.stages = kI8SmemBytes / stage_bytes;
  if (t.stages > kI8MaxStages) t.stages = kI8MaxStages;
  while (t.stages * stage_bytes + 1024 > kI8SmemBytes) --t.stages;
  t.kb = (p.k + kKBlock - 1) / kKBlock;
  t.tok_tiles = (p.m + t.bn - 1) / t.bn;
  t.tiles = t.tok_tiles * ((p.n + kChTile - 1) / kChTile);
  t.units = (long long)t.tiles * t.kb;
  t.tmem_cols = 32;
  while (t.tmem_cols < 2 * p.planes * t.bn) t.tmem_cols *= 2;
  t.slot_ints = (long long)p.planes * t.bn * kChTile;
  t.counters = counters;
  t.partials = partials;
  t.error = error;
  // Whole tiles where the last wave leaves at most a tenth of the SMs' time idle.
  const int waves = (t.tiles + num_sms - 1) / num_sms;
  t.whole = t.tiles * 10LL >= (long long)waves * num_sms * 9;
  const int grid = t.whole ? (t.tiles < num_sms ? t.tiles : num_sms) : (int)(t.units < num_sms ? t.units : num_sms);
  if (!encode_rows(&t.mw, p.w, (long long)p.planes * p.n, p.k, p.ldw, kChTile) ||
      !encode_rows(&t.mx, p.x, p.m, p.k, p.ldx, t.bn))
    return cudaErrorInvalidValue;
  const int smem = t.stages * stage_bytes + 1024;
  if (p.bf16)
    return p.planes == 2 ? launch_product<__nv_bfloat16, 2>(t, grid, smem, pdl, stream)
                         : launch_product<__nv_bfloat16, 1>(t, grid, smem, pdl, stream);
  return p.planes == 2 ? launch_product<__half, 2>(t, grid, smem, pdl, stream)
                       : launch_product<__half, 1>(t, grid, smem, pdl, stream);
}

}  // namespace b2g
