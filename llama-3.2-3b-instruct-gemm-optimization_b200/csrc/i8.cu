// i8.cu -- matrix product in 8-bit integers with a scale for each row of x
// and each output channel, and the quantisers that make its operands.
#include <atomic>

#include <algorithm>

#include "serve.cuh"
#include "tc.cuh"

namespace b2g {
namespace {

// v / s rounded to the nearest integer, ties to even.  Adding 1.5 * 2^23 to a
// quotient leaves its integer in the low bits.
__device__ __forceinline__ uint32_t code_of(float v, float s) {
  return __float_as_uint(v / s + 12582912.0f) & 0xff;
}
// Eight of them, a byte each.  v * (1 / s) is off by at most 2^-22 of it, less
// than 2^-15: where every product is further than that from a tie its integer
// is the quotient's, else (one value in 16,000) the quotients are taken.
__device__ __forceinline__ uint2 codes_of(const float (&v)[8], float s, float inv) {
  uint32_t w[2] = {0, 0};
  float off = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float q = v[e] * inv, r = q + 12582912.0f;
    off = fmaxf(off, fabsf(q - (r - 12582912.0f)));
    w[e / 4] |= (__float_as_uint(r) & 0xff) << (8 * (e % 4));
  }
  if (off > 0.5f - 0x1p-15f) {
    w[0] = w[1] = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e / 4] |= code_of(v[e], s) << (8 * (e % 4));
  }
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ float scale_of(float amax) {
  return amax <= 3.4028235e38f ? fmaxf(amax, 1e-12f) / 127.0f : __uint_as_float(0x7fffffffu);
}
// Maximum of absolute values that keeps a NaN: as integers the patterns of
// |v| are in order, infinity above the finite ones and NaNs on top.
__device__ __forceinline__ float max_abs(float a, float v) {
  return __uint_as_float(max(__float_as_uint(a), __float_as_uint(v) & 0x7fffffffu));
}

// Elements 8c .. 8c + 7 of a row of k, as they are (zeros behind its end).
template <typename T>
__device__ __forceinline__ uint4 load8(const T* row, int c, int k) {
  if (8 * c + 8 <= k) return *reinterpret_cast<const uint4*>(row + 8 * c);
  uint32_t w[4] = {0, 0, 0, 0};
  const uint16_t* h = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (8 * c + i < k) w[i / 2] |= (uint32_t)h[8 * c + i] << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// One block a row.  A thread keeps up to 32 elements (four 16-byte loads) as
// they come, so a row of up to 32 x threads elements is read once (a longer
// one again for each pass) and six blocks an SM fit; each pass widens and
// normalises them again, to the same bits.  4096 rows of 8192 with RMSNorm:
// 30.5 us, 3.3 TB/s (conversions and the sums' barriers; 2.4 us for 8 rows, its launch).
template <typename T, bool RMS>
__global__ void __launch_bounds__(512) quantize_rows_kernel(const I8RowsParams p) {
  constexpr int NC = 4;
  __shared__ float red[2][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* gamma = static_cast<const T*>(p.gamma);
  const int chunks = (p.k + 7) / 8, per_pass = NC * blockDim.x;
  const bool resident = chunks <= per_pass;
  pdl_wait();
  pdl_launch_dependents();  // behind the wait: the launch after this one may read weights at once
  uint4 raw[NC];
  auto load = [&](int base) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = base + i * blockDim.x + threadIdx.x;
      raw[i] = c < chunks ? load8(x, c, p.k) : make_uint4(0, 0, 0, 0);
    }
  };
  float r = 1.0f;
  // Chunk i of the pass at `base`, normalised.
  auto values = [&](int base, int i, float (&v)[8]) {
    unpack8<T>(raw[i], v);
    if constexpr (RMS) {
      const int c = base + i * blockDim.x + threadIdx.x;
      if (gamma && c < chunks) {
        float g[8];
        unpack8<T>(load8(gamma, c, p.k), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = v[e] * r * g[e];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= r;
      }
    }
  };
  load(0);
  if constexpr (RMS) {
    float ss = 0.f;
    for (int base = 0; base < chunks; base += per_pass) {
      if (base) load(base);
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        float v[8];
        unpack8<T>(raw[i], v);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += v[e] * v[e];
      }
    }
    for (int off = 16; off; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    if (lane == 0) red[0][warp] = ss;
    __syncthreads();
    ss = lane < warps ? red[0][lane] : 0.f;
    for (int off = 16; off; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    r = rsqrtf(ss / (float)p.k + p.eps);
    if (!resident) load(0);
  }
  float a = 0.f;
  for (int base = 0; base < chunks; base += per_pass) {
    if (base) load(base);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      float v[8];
      values(base, i, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) a = max_abs(a, v[e]);
    }
  }
  for (int off = 16; off; off >>= 1) a = max_abs(a, __shfl_xor_sync(0xffffffffu, a, off));
  if (lane == 0) red[1][warp] = a;
  __syncthreads();
  a = lane < warps ? red[1][lane] : 0.f;
  for (int off = 16; off; off >>= 1) a = max_abs(a, __shfl_xor_sync(0xffffffffu, a, off));
  const float s = scale_of(a);
  const bool finite = s == s;
  const float inv = 1.0f / s;
  int8_t* codes = p.codes + row * p.ldc;
  for (int base = 0; base < chunks; base += per_pass) {
    if (!resident) load(base);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = base + i * blockDim.x + threadIdx.x;
      if (c >= chunks) continue;
      float v[8];
      values(base, i, v);
      const uint2 w = finite ? codes_of(v, s, inv) : make_uint2(0, 0);
      if (8 * c + 8 <= p.k) {
        *reinterpret_cast<uint2*>(codes + 8 * c) = w;
      } else {
        for (int e = 0; 8 * c + e < p.k; ++e) codes[8 * c + e] = (int8_t)((e < 4 ? w.x : w.y) >> (8 * (e % 4)));
      }
    }
  }
  if (threadIdx.x == 0) p.scales[row] = s;
}

// The code of a weight; a channel that is not finite (s NaN) has zero codes.
__device__ __forceinline__ int8_t channel_code(float v, float s) {
  return s == s ? (int8_t)code_of(v, s) : (int8_t)0;
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
      for (int k = ty; k < K; k += 32) a = max_abs(a, Act<T>::to_float(w[(long long)k * N + n0 + tx]));
    tile[ty][tx] = a;
  } else {
    if (n0 + ty < N)
      for (int k = tx; k < K; k += 32) a = max_abs(a, Act<T>::to_float(w[(long long)(n0 + ty) * K + k]));
    tile[tx][ty] = a;
  }
  __syncthreads();
  if (ty == 0) {
    a = 0.f;
    for (int i = 0; i < 32; ++i) a = max_abs(a, tile[i][tx]);
    const float s = scale_of(a);
    sc[tx] = s;
    if (n0 + tx < N) scales[n0 + tx] = s;
  }
  __syncthreads();
  for (int k0 = 0; k0 < K; k0 += 32) {
    if (layout == B2G_LAYOUT_KN) {
      if (k0 + ty < K && n0 + tx < N) tile[ty][tx] = Act<T>::to_float(w[(long long)(k0 + ty) * N + n0 + tx]);
      __syncthreads();
      if (n0 + ty < N && k0 + tx < K) codes[(n0 + ty) * ldc + k0 + tx] = channel_code(tile[tx][ty], sc[ty]);
      __syncthreads();
    } else if (n0 + ty < N && k0 + tx < K) {
      codes[(n0 + ty) * ldc + k0 + tx] = channel_code(Act<T>::to_float(w[(long long)(n0 + ty) * K + k0 + tx]), sc[ty]);
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
// in tensor memory, warps 2..5 drain the other one.
// Many tokens take a deep tile instead: 2 x 128 channels by up to 256 tokens,
// which moves two thirds of the bytes a product from L2 (what bounds the narrow
// one: 240 clocks an MMA of 128 x 256 where the tensor cores need 128), but
// fills tensor memory with one accumulator, drained by eight warps between
// tiles.  4096 x 8192 x 8192: 192 us in a loop (2.9 POP/s, 0.86 of the rate that
// the bf16 peak implies), 247 in narrow tiles.
// Work is cut in one of three ways (i8_plan).  Whole tiles, in turn.  A
// cluster of 2, 4 or 8 CTAs a tile, where that many fit: each takes a part of K
// and leaves its int32 sums in its shared memory, and each finishes a part of
// the columns from everybody's (one token by 8192 x 4096: 13 us, 18.6 through
// global memory).  For a long K and very few tiles equal ranges of k blocks
// ("units"; 30 x 300 x 8000: 7.9 us, clusters of eight 10.9): a range's tiles at
// its two ends are shared with other CTAs, which all add their int32 sums into
// the workspace (integers: the order does not matter); the last to arrive
// finishes the tile and leaves zeros behind.
// ---------------------------------------------------------------------------
constexpr int kI8MaxStages = 12;
constexpr int kKBlock = 128;
constexpr int kChTile = 128;
constexpr int kI8SmemBytes = 200 * 1024 + 1024;  // ring and its alignment

struct I8Tc {
  CUtensorMap mw, mx;
  I8Params p;
  int bn, stages, kb, tok_tiles, tiles, whole;
  int cluster;          // CTAs a tile (1: none)
  int acc_cols;         // tensor-memory columns of an accumulator
  int tmem_cols, after_quantiser;
  long long units;
  long long slot_ints;  // int32 words of one partial
  int* counters;        // [grid], zero between launches
  int* partials;        // [grid][slot_ints] sums of the split tile whose first k block a CTA has; zero between launches
  int* error;
};

// The pieces of this CTA's work: k blocks [k0, k1) of a tile.
struct I8Seg {
  long long u, end;  // units (split) or tiles (whole)
  int tile, k0, k1;
  __device__ __forceinline__ void begin(const I8Tc& t) {
    const int c = blockIdx.x, g = gridDim.x;
    if (t.cluster > 1) {
      u = c;
      end = c + 1;
      return;
    }
    u = t.whole ? c : c * t.units / g;
    end = t.whole ? t.tiles : (c + 1) * t.units / g;
  }
  __device__ __forceinline__ bool next(const I8Tc& t) {
    if (u >= end) return false;
    if (t.cluster > 1) {
      const int rank = (int)u % t.cluster;
      tile = (int)u / t.cluster;
      k0 = rank * t.kb / t.cluster;
      k1 = (rank + 1) * t.kb / t.cluster;
      ++u;
    } else if (t.whole) {
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

// The scaled sum, or SiLU(gate) * up.
template <bool GATE>
__device__ __forceinline__ float i8_value(int acc, int acc_up, float sw, float sw_up, float sx) {
  const float v = (float)acc * sw * sx;
  if constexpr (!GATE) return v;
  // v / (1 + exp(-v)), for v < 0 as v exp(v) / (1 + exp(v)): the divisor is at most
  // 2 (past 2^126 the fast division gives 0).  Off by (|v| + 8) 2^-22 of the value at
  // most: the exponential's argument is rounded, the rest is a few ulp.  (The division
  // rounded to nearest made a gate||up product of 2048 x 8192 x 4096 1.4 times slower.)
  const float e = __expf(-fabsf(v));
  return __fdividef(v < 0.0f ? v * e : v, 1.0f + e) * ((float)acc_up * sw_up * sx);
}

// PLANES 128-row weight tiles a stage: gate and up (GATE), or two channel tiles.
template <typename T, int PLANES, bool GATE, bool DEEP>
__global__ void __launch_bounds__(DEEP ? 320 : 192, 1) i8_product_kernel(const __grid_constant__ I8Tc t) {
  constexpr int kEpi = DEEP ? 256 : 128;  // epilogue threads
  constexpr int kBufs = DEEP ? 1 : 2;     // accumulators
  constexpr int kChannels = GATE ? kChTile : PLANES * kChTile;  // of a tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[kI8MaxStages], empty[kI8MaxStages], acc_full[2], acc_empty[2], drain;
  __shared__ uint32_t tmem_base_sh;
  __shared__ int last_sh, gave_up_sh;
  __shared__ __align__(16) float sx_sh[2][256];
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
      mbar_init(&acc_empty[i], kEpi);
    }
    mbar_init(&drain, 1);
    fence_mbarrier_init();
    gave_up_sh = 0;
  }
  int sent = 0;  // thread 0: k blocks asked for
  auto give_up = [&](int code) {
    *t.error = code;
    gave_up_sh = 1;
  };
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
          tma_load_2d(dst + pl * kChTile * kKBlock, &t.mw, k * kKBlock,
                      pl * (GATE ? t.p.n : kChTile) + s.tile / t.tok_tiles * kChannels, &full[stage]);
      };
      auto load_x = [&](int stage, const I8Seg& s, int k) {
        tma_load_2d(ring + stage * stage_bytes + PLANES * kChTile * kKBlock, &t.mx, k * kKBlock,
                    s.tile % t.tok_tiles * t.bn, &full[stage]);
      };
      // Behind the quantiser the first stages' weights are asked for at once:
      // it does not write them, and what came before it is complete.
      if (!t.after_quantiser) pdl_wait();
      I8Seg s;
      s.begin(t);
      int issued = 0;
      while (t.after_quantiser && issued < t.stages && s.next(t))
        for (int k = s.k0; k < s.k1 && issued < t.stages; ++k, ++issued) {
          mbar_arrive_expect_tx(&full[issued], stage_bytes);
          load_w(issued, s, k);
        }
      if (t.after_quantiser) pdl_wait();
      s.begin(t);
      int i = 0;  // k blocks so far
      bool ok = true;
      while (ok && s.next(t))
        for (int k = s.k0; k < s.k1; ++k, ++i) {
          const int stage = i % t.stages;
          if (i >= issued) {
            if (i >= t.stages && !mbar_wait_spin(&empty[stage], (i / t.stages - 1) & 1)) {
              give_up(kErrEmptyWait);
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&full[stage], stage_bytes);
            load_w(stage, s, k);
          }
          load_x(stage, s, k);
        }
      sent = i;
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
        const int buf = n % kBufs;
        if (!mbar_wait_spin(&acc_empty[buf], ((n / kBufs) & 1) ^ 1)) {
          give_up(kErrEmptyWait);
          ok = false;
          break;
        }
        tc_fence_after();
        for (int k = s.k0; k < s.k1; ++k, ++i) {
          const int stage = i % t.stages;
          if (!mbar_wait_spin(&full[stage], (i / t.stages) & 1)) {
            give_up(kErrFullWait);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = ring_addr + stage * stage_bytes;
          const uint64_t db = smem_desc_sw128(a0 + PLANES * kChTile * kKBlock, 16, 1024);
#pragma unroll
          for (int pl = 0; pl < PLANES; ++pl) {
            const uint64_t da = smem_desc_sw128(a0 + pl * kChTile * kKBlock, 16, 1024);
            const uint32_t d = tmem + (buf * PLANES + pl) * t.acc_cols;
#pragma unroll
            for (int j = 0; j < 4; ++j)  // 32 k an instruction: 2 units of 16 bytes
              mma_i8_ss(d, da + 2 * j, db + 2 * j, idesc, k > s.k0 || j > 0);
          }
          tc_commit(&empty[stage]);
        }
        if (ok) tc_commit(&acc_full[buf]);
        ++n;
      }
    }
  } else {
    pdl_wait();
    pdl_launch_dependents();  // behind the wait: what came before this launch is complete
    const int quad = warp & 3, et = threadIdx.x - 64;
    const int ch = quad * 32 + lane;  // channel in the tile
    const uint32_t lane_addr = tmem + ((uint32_t)(quad * 32) << 16);
    const I8Params& p = t.p;
    I8Seg s;
    s.begin(t);
    int n = 0;
    // After a wait that has run out its thread goes through the remaining pieces
    // without waiting, so that barriers and warp-wide instructions still meet.
    bool ok = true;
    while (s.next(t)) {
      const int buf = n % kBufs;
      const int tok0 = s.tile % t.tok_tiles * t.bn, j = s.tile / t.tok_tiles * kChannels + ch;
      const int cols = min(t.bn, p.m - tok0);
      const bool split = t.cluster == 1 && (s.k0 != 0 || s.k1 != t.kb);
      float sw[PLANES];
#pragma unroll
      for (int pl = 0; pl < PLANES; ++pl) {
        const int c = j + (GATE ? 0 : pl * kChTile);
        sw[pl] = c < p.n ? p.sw[(GATE ? pl * p.n : 0) + c] : 0.f;
      }
      // Everything the epilogue reads from global memory is asked for before
      // the accumulator is waited for (residual rows: a chunk ahead).
      float* sx = sx_sh[n & 1];
      for (int c = et; c < cols; c += kEpi) sx[c] = p.sx[tok0 + c];
      // 32 columns at a time (two groups of warps take them in turn), with
      // pointers that advance: a 64-bit product an address was half of the
      // epilogue (256 columns: 5 us, 10 before).
      const int first = DEEP ? 32 * (et >> 7) : 0;
      constexpr int kStepCols = 32 * (kEpi / 128), kOuts = GATE ? 1 : PLANES;
      T res[kOuts][32];
      auto load_residual = [&](int c0) {
        if (!p.residual) return;
#pragma unroll
        for (int o = 0; o < kOuts; ++o) {
          const T* col = static_cast<const T*>(p.residual) + (tok0 + min(c0, cols - 1)) * p.ldr +
                         min(j + o * kChTile, p.n - 1);
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            res[o][c] = *col;
            col += c0 + c < cols - 1 ? p.ldr : 0;
          }
        }
      };
      if (t.cluster == 1) load_residual(first);
      named_sync(1, kEpi);
      if (ok && !mbar_wait_spin(&acc_full[buf], (n / kBufs) & 1)) {
        give_up(kErrFullWait);
        ok = false;
      }
      __syncwarp();
      tc_fence_after();
      // Columns go 32 at a time; those behind the last row are read (scratch or
      // a clamped row) and not stored, so that no load waits on a branch.
      bool finish = true;
      int* sums = nullptr;
      if (!DEEP && t.cluster > 1) {
        // The ring is free: every MMA that read it is done.  [plane][column][channel].
        int* mine = reinterpret_cast<int*>(ring);
        for (int c0 = 0; c0 < cols; c0 += 32) {
#pragma unroll
          for (int pl = 0; pl < PLANES; ++pl) {
            uint32_t r[32];
            tmem_ld32(lane_addr + (buf * PLANES + pl) * t.acc_cols + c0, r);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c) mine[(pl * t.bn + c0 + c) * kChTile + ch] = (int)r[c];
          }
        }
        break;  // the only segment; the rest is behind the cluster's barrier
      }
      if (!DEEP && split) {
        const int c_first = i8_owner(t, (long long)s.tile * t.kb);
        const int c_last = i8_owner(t, (long long)(s.tile + 1) * t.kb - 1);
        sums = t.partials + c_first * t.slot_ints + ch;
        for (int c0 = 0; c0 < cols; c0 += 32) {
#pragma unroll
          for (int pl = 0; pl < PLANES; ++pl) {
            uint32_t r[32];
            tmem_ld32(lane_addr + (buf * PLANES + pl) * t.acc_cols + c0, r);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (c0 + c < cols) atomicAdd(sums + (pl * t.bn + c0 + c) * kChTile, (int)r[c]);
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
        for (int c0 = first; c0 < cols; c0 += kStepCols) {
          uint32_t r[PLANES][32];
          const int rows = cols - c0;  // of this chunk, if less than 32
          if (!DEEP && split) {
#pragma unroll
            for (int pl = 0; pl < PLANES; ++pl)
#pragma unroll
              for (int c = 0; c < 32; ++c) r[pl][c] = __ldcg(sums + (pl * t.bn + c0 + c) * kChTile);
#pragma unroll
            for (int pl = 0; pl < PLANES; ++pl)
#pragma unroll
              for (int c = 0; c < 32; ++c) __stcg(sums + (pl * t.bn + c0 + c) * kChTile, 0);
          } else {
#pragma unroll
            for (int pl = 0; pl < PLANES; ++pl) tmem_ld32(lane_addr + (buf * PLANES + pl) * t.acc_cols + c0, r[pl]);
            tmem_wait_ld();
          }
          T out[kOuts][32];
#pragma unroll
          for (int o = 0; o < kOuts; ++o)
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              float v = i8_value<GATE>((int)r[o][c], (int)r[PLANES - 1][c], sw[o], sw[PLANES - 1], sx[c0 + c]);
              if (p.residual) v += Act<T>::to_float(res[o][c]);
              out[o][c] = Act<T>::from_float(v);
            }
          // Loaded before the stores: residual and y may be one buffer, but a
          // chunk's rows are its own.
          load_residual(c0 + kStepCols);
#pragma unroll
          for (int o = 0; o < kOuts; ++o) {
            if (j + o * kChTile >= p.n) continue;
            T* to = static_cast<T*>(p.y) + (tok0 + c0) * p.ldy + j + o * kChTile;
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              if (c < rows) *to = out[o][c];
              to += p.ldy;
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
  if (!DEEP && t.cluster > 1) {
    // This CTA's columns of the tile, from all the cluster's sums.  What comes
    // from global memory is asked for before the barrier.
    const I8Params& p = t.p;
    const int rank = blockIdx.x % t.cluster, tile = blockIdx.x / t.cluster;
    const int ch = (warp & 3) * 32 + lane, j = tile / t.tok_tiles * kChTile + ch;
    const int tok0 = tile % t.tok_tiles * t.bn, cols = min(t.bn, p.m - tok0);
    const int c_begin = rank * cols / t.cluster, c_end = (rank + 1) * cols / t.cluster;
    const bool mine = warp >= 2 && j < p.n;
    constexpr int C = 16;  // columns at a time
    float sw[PLANES];
    T res[C];
    auto load_residual = [&](int c0) {
      if (!mine || !p.residual) return;
      const T* col = static_cast<const T*>(p.residual) + (long long)(tok0 + max(min(c0, c_end - 1), 0)) * p.ldr + j;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        res[c] = *col;
        col += c0 + c < c_end - 1 ? p.ldr : 0;
      }
    };
#pragma unroll
    for (int pl = 0; pl < PLANES; ++pl) sw[pl] = mine ? p.sw[pl * p.n + j] : 0.f;
    load_residual(c_begin);
    cluster_sync();
    if (warp >= 2) {
      const uint32_t sums = smem_addr(ring) + ch * 4;
      for (int c0 = c_begin; c0 < c_end; c0 += C) {
        const int n = min(C, c_end - c0);
        int acc[PLANES][C] = {};
        for (int peer = 0; peer < t.cluster; ++peer) {
          const uint32_t from = cluster_map(sums, peer);
#pragma unroll
          for (int pl = 0; pl < PLANES; ++pl)
#pragma unroll
            for (int c = 0; c < C; ++c)
              acc[pl][c] += ld_cluster(from + (pl * t.bn + c0 + min(c, n - 1)) * kChTile * 4);
        }
        T out[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
          float v = i8_value<GATE>(acc[0][c], acc[PLANES - 1][c], sw[0], sw[PLANES - 1], sx_sh[0][c0 + min(c, n - 1)]);
          if (p.residual) v += Act<T>::to_float(res[c]);
          out[c] = Act<T>::from_float(v);
        }
        load_residual(c0 + C);
        if (mine) {
          T* to = static_cast<T*>(p.y) + (long long)(tok0 + c0) * p.ldy + j;
#pragma unroll
          for (int c = 0; c < C; ++c) {
            if (c < n) *to = out[c];
            to += p.ldy;
          }
        }
      }
    }
    __syncwarp();
    cluster_sync();  // peers may still be reading this CTA's sums
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (gave_up_sh) {
    // Nobody may have waited for what is on its way: copies and products end
    // before shared and tensor memory go.
    bool ok = true;
    if (threadIdx.x == 0)
      for (int i = max(0, sent - t.stages); i < sent; ++i)
        ok = ok && mbar_wait_spin(&full[i % t.stages], (i / t.stages) & 1);
    if (threadIdx.x == 32) {
      tc_commit(&drain);
      ok = mbar_wait_spin(&drain, 0);
    }
    if (!ok) *t.error = kErrDrainWait;
    __syncwarp();
  }
  if (warp == 1) tmem_dealloc(tmem, t.tmem_cols);
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
template <typename T, int PLANES, bool GATE, bool DEEP>
cudaError_t launch_product(const I8Tc& t, int grid, int smem, cudaStream_t stream) {
  static std::atomic<uint64_t> allowed{0};  // devices whose limit is set
  const auto kernel = i8_product_kernel<T, PLANES, GATE, DEEP>;
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kernel), kI8SmemBytes, &allowed);
  if (e != cudaSuccess) return e;
  return launch_after(kernel, dim3(grid), dim3(DEEP ? 320 : 192), smem, t.cluster, stream, t);
}

template <typename T>
cudaError_t launch_typed(const I8Tc& t, bool deep, int grid, int smem, cudaStream_t stream) {
  if (t.p.planes == 2)
    return deep ? launch_product<T, 2, true, true>(t, grid, smem, stream)
                : launch_product<T, 2, true, false>(t, grid, smem, stream);
  return deep ? launch_product<T, 2, false, true>(t, grid, smem, stream)
              : launch_product<T, 1, false, false>(t, grid, smem, stream);
}

int div_up(long long a, long long b) { return (int)((a + b - 1) / b); }

// How a product is cut: columns of a tile, one of the ways above.
struct I8Plan {
  int bn = 0, cluster = 1;
  bool deep = false, whole = true;
};

// The cut with the least estimated time.  The terms, in ns, were fitted to 90
// products of 1..8000 tokens, each timed under every cut (the choice is 1.1% off
// the best of them on average; choosing by how full the last wave is was 34% off):
// a k block takes 400 a plane (540 a deep one), or what L2 delivers to all CTAs at
// 14.5 bytes a ns; an epilogue 20 a column (26 next to the next tile's loads, 24 deep).
I8Plan i8_plan(int m, int n, int k, int planes, int num_sms) {
  const int kb = div_up(k, kKBlock), ch = div_up(n, kChTile);
  // Clusters of 4 and 8 that the GPCs of 148 SMs hold: 33 and 15.
  const int fit[9] = {0, 0, num_sms / 2, 0, num_sms * 9 / 40, 0, 0, 0, (num_sms + 2) / 10};
  I8Plan best;
  double least = 1e30;
  const auto take = [&](double ns, int bn, int cluster, bool deep, bool whole) {
    if (ns >= least) return;
    least = ns;
    best.bn = bn, best.cluster = cluster, best.deep = deep, best.whole = whole;
  };
  const auto block_ns = [&](double alone, int ctas, int rows) {
    return std::max(alone, std::min(ctas, num_sms) * (rows * (double)kKBlock) / 14500);
  };
  // Tiles of a quarter of the most columns at least: smaller ones never won.
  const int most = std::min(up32(m), 256 / planes);
  for (int bn = most; bn >= std::max(32, most / 4); bn -= 32) {
    const int tiles = div_up(m, bn) * ch, rows = planes * kChTile + bn;
    const double loop = kb * block_ns(400 * planes, tiles, rows), tail = 20.0 * bn;
    take(loop + tail + (div_up(tiles, num_sms) - 1) * std::max(loop, 26.0 * bn), bn, 1, false, true);
    for (int c = 2; c <= 8 && c <= kb; c *= 2)
      if (tiles <= fit[c])
        take(div_up(kb, c) * block_ns(400 * planes, tiles * c, rows) + (c == 2 ? 700 : c == 4 ? 1800 : 4100) +
                 28.0 * bn * planes, bn, c, false, true);
    if (bn == most) {  // shared ranges: atomics for each valid column, and two waits
      const long long units = (long long)tiles * kb;
      take(3300 + div_up(units, std::min<long long>(units, num_sms)) * 1050.0 * planes +
               63.0 * std::min(bn, m) * planes, bn, 1, false, false);
    }
  }
  const int deep_most = std::min(up32(m), 256), deep_ch = planes == 2 ? ch : div_up(n, 2 * kChTile);
  for (int bn = deep_most; bn >= std::max(32, deep_most / 2); bn -= 16) {
    const int tiles = div_up(m, bn) * deep_ch;
    take(div_up(tiles, num_sms) * (kb * block_ns(540, tiles, 2 * kChTile + bn) + 24.0 * bn), bn, 1, true, true);
  }
  return best;
}

}  // namespace

cudaError_t launch_i8_quantize_rows(const I8RowsParams& p, cudaStream_t stream) {
  // Four 16-byte loads a thread, 64 to 512 threads.
  const int threads = std::min(512, std::max(64, (p.k + 1023) / 1024 * 32));
  void (*kernel)(I8RowsParams) =
      p.bf16 ? (p.rmsnorm ? quantize_rows_kernel<__nv_bfloat16, true> : quantize_rows_kernel<__nv_bfloat16, false>)
             : (p.rmsnorm ? quantize_rows_kernel<__half, true> : quantize_rows_kernel<__half, false>);
  return launch_after(kernel, dim3(p.m), dim3(threads), 0, 1, stream, p);
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
  return (size_t)num_sms * planes * bn * kChTile * 4;
}

cudaError_t launch_i8_product(const I8Params& p, int num_sms, int* counters, int* partials, int* error,
                              bool after_quantiser, cudaStream_t stream) {
  const I8Plan plan = i8_plan(p.m, p.n, p.k, p.planes, num_sms);
  const bool deep = plan.deep;
  I8Tc t;
  t.p = p;
  t.bn = plan.bn;
  t.tok_tiles = div_up(p.m, t.bn);
  t.tiles = t.tok_tiles * div_up(p.n, deep && p.planes == 1 ? 2 * kChTile : kChTile);
  const int stage_tiles = deep ? 2 : p.planes;
  const int stage_bytes = (stage_tiles * kChTile + t.bn) * kKBlock;
  t.stages = std::min(kI8MaxStages, (kI8SmemBytes - 1024) / stage_bytes);
  // Narrow tiles of one plane leave room for a second CTA, the next launch's: it
  // sets itself up while this one runs (12.9 us a product of 1 x 8192 x 4096
  // instead of 14.1), and 100 KB in flight still hide the latency.  Two planes
  // need the bytes (gate||up of 8 x 8192 x 4096: 16.3 us, 19.9 with 74 KB).
  if (t.bn <= 64 && stage_tiles == 1) t.stages = std::min(t.stages, 100 * 1024 / stage_bytes);
  t.kb = div_up(p.k, kKBlock);
  t.units = (long long)t.tiles * t.kb;
  t.acc_cols = deep ? 256 : t.bn;
  t.tmem_cols = 32;
  while (t.tmem_cols < (deep ? 1 : 2) * stage_tiles * t.acc_cols) t.tmem_cols *= 2;
  t.slot_ints = (long long)p.planes * t.bn * kChTile;
  t.counters = counters;
  t.partials = partials;
  t.error = error;
  t.whole = plan.whole;
  t.cluster = plan.cluster;
  const int grid = t.cluster > 1 ? t.tiles * t.cluster
                                 : (int)std::min<long long>(t.whole ? t.tiles : t.units, num_sms);
  t.after_quantiser = after_quantiser;
  if (!encode_rows(&t.mw, p.w, (long long)p.planes * p.n, p.k, p.ldw, kChTile) ||
      !encode_rows(&t.mx, p.x, p.m, p.k, p.ldx, t.bn))
    return cudaErrorInvalidValue;
  const int smem = t.stages * stage_bytes + 1024;
  return p.bf16 ? launch_typed<__nv_bfloat16>(t, deep, grid, smem, stream)
                : launch_typed<__half>(t, deep, grid, smem, stream);
}

}  // namespace b2g
