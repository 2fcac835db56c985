// attn_rows.cuh -- attention of few rows a k/v head (decode steps, drafts):
// bound by reading the cache once.
//
// A block of four warps walks its share of the work list in units of 64
// cached tokens, 16 a warp.  Each warp streams its own tokens' keys and
// values through its own ring of shared memory with 16-byte asynchronous
// copies (page by page, nothing shared, so no barrier in the loop), and keeps
// its own running maximum, sum and output for the 16 rows of the tile in
// m16n8k16 fragments.  At the end of an item the warps' parts are joined in
// shared memory, and the blocks' parts of a split item by the last block to
// arrive, always in the same order.
// 64 sequences of up to 8192 tokens, 32 heads on 8, bf16: 209 us, 0.94 of a
// copy's rate.  Two of 131072 over an 8-bit cache, 4 tokens each: 130 us, 0.63
// (two warps a scheduler wait out the latencies of copy, widen, multiply: 0.42 of
// the issue slots, 0.47 of the memory's time).
#pragma once
#include <type_traits>

#include "serve.cuh"

namespace b2g {

constexpr float kLog2e = 1.4426950408889634f;

// 2^x to 2^-22 of its value; 0 for -infinity and below 2^-126.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool BF16>
__device__ __forceinline__ void mma_act(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    mma_16816(d, a[0], a[1], a[2], a[3], b0, b1);
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 16 bytes global -> shared, zeros where !in (src is not read then).
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// T: the activations' type.  With an 8-bit cache the products run in fp16
// (every E4M3 value is one): bf16 rows of q are brought into its range by a
// power of two each.
template <typename T, bool FP8, int D>
struct RowsKernel {
  static constexpr int kRows = 16, kUnit = 64, kWarps = 4;
  static constexpr bool kBf16 = !FP8 && sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value;
  static constexpr int kRowBytes = D * (FP8 ? 1 : 2);
  static constexpr int kTileBytes = 16 * kRowBytes;       // 16 tokens of keys or values
  static constexpr int kStageBytes = 2 * kTileBytes;      // of one warp
  static constexpr int kBlocks = kAttnBlocks;             // an SM
  static constexpr int kStages = 49152 / kBlocks / kStageBytes;  // 48 KB of a warp's place in flight
  static constexpr int kNT = D / 8;                       // output tiles of 8 columns
  static constexpr int kSmem = kWarps * kStages * kStageBytes + kNT * 32 * 16;
  static constexpr int kPartFloats = 16 * D + 32;         // a part: [row][column], then maxima and sums of 16 rows

  using Work = AttnWork<kRows, kUnit>;

  // 16-byte chunk of a token's row inside its tile.  Sixteen or eight chunks
  // a row: eight consecutive tokens' same chunk lie in different banks.
  static __device__ __forceinline__ uint32_t chunk_at(int token, int c) {
    if constexpr (kRowBytes == 64) return token * 64 + ((c ^ ((token >> 1) & 3)) * 16);
    if constexpr (FP8) return token * kRowBytes + ((c ^ (((token & 1) << 2) | ((token >> 1) & 3))) * 16);
    return token * kRowBytes + ((c ^ (token & 7)) * 16);
  }

  // Column of element e (0, 1) of output tile j for lane quarter q.
  static __device__ __forceinline__ int column(int j, int q, int e) {
    if constexpr (FP8) return 16 * (j / 2) + 4 * q + 2 * e + (j & 1);
    return 8 * j + 2 * q + e;
  }

  static __device__ void run(const AttnParams& p);
};

template <typename T, bool FP8, int D>
__device__ void RowsKernel<T, FP8, D>::run(const AttnParams& p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ long long sh[8];
  __shared__ float sh_ml[2][16], sh_red[8][16];
  __shared__ int sh_last;
  __shared__ uint32_t seen_sh[kWarps][kStages];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const uint32_t ring = smem_addr(smem) + warp * kStages * kStageBytes;
  float* join = reinterpret_cast<float*>(smem + kWarps * kStages * kStageBytes);
  pdl_wait();
  pdl_launch_dependents();
  const Work w(p);
  const AttnShare share = attn_share<false>(w, p.least_units, sh);
  if (share.begin >= share.end) return;

  // The stream of units: where the copies are, ahead of the products.
  long long at0 = share.at;
  AttnItem pi = w.find(share.b, at0);
  int pu = pi.u_lo + (int)at0;
  long long left = share.end - share.begin;  // units not yet asked for
  // Lanes 0..15 (and 16..31 again): a token's row in the cache in units of 16
  // bytes (a cache spans less than 2^32 of them), and whether it is there.
  uint32_t row_at = 0;
  bool row_in = false;
  const int shift = p.page_shift;
  constexpr int kPer16 = FP8 ? 16 : 8;  // elements
  const uint32_t step_token = (uint32_t)(p.c.stride_token / kPer16), step_head = (uint32_t)(p.c.stride_head / kPer16),
                 step_page = (uint32_t)(p.c.stride_page / kPer16);
  auto look_up = [&]() {
    if (left <= 0) return;
    const int j = pu * kUnit + warp * 16 + (lane & 15);
    row_in = false;
    if (j >= pi.lo && j < pi.hi) {
      const int pg = shift >= 0 ? j >> shift : j / p.c.page_size;
      const int page = page_of(p.b, p.c, pi.b, pg, p.error);
      row_in = page >= 0;
      if (row_in) row_at = page * step_page + (j - pg * p.c.page_size) * step_token + pi.h * step_head;
    }
  };
  const uint8_t* kb = static_cast<const uint8_t*>(p.c.k);
  const uint8_t* vb = static_cast<const uint8_t*>(p.c.v);
  // Copies the next unit's tokens; seen_sh: bit t says that token t is there.
  auto copy = [&](int to) {
    if (left > 0) {
      constexpr int kChunks = kRowBytes / 16, kPerPass = 32 / kChunks;  // tokens a pass of the lanes
      const int c = lane % kChunks;
      const uint32_t dst = ring + to * kStageBytes;
      const uint32_t mask = __ballot_sync(0xffffffffu, row_in) & 0xffff;
      if (lane == 0) seen_sh[warp][to] = mask;
#pragma unroll
      for (int i = 0; i < 16 / kPerPass; ++i) {
        const int t = i * kPerPass + lane / kChunks;
        const bool in = mask >> t & 1;
        const uint32_t row = __shfl_sync(0xffffffffu, row_at, t);  // every lane takes part
        const unsigned long long off = in ? (unsigned long long)(row + c) * 16 : 0;
        cp_async16_or_zero(dst + chunk_at(t, c), kb + off, in);
        cp_async16_or_zero(dst + kTileBytes + chunk_at(t, c), vb + off, in);
      }
      --left;
      if (++pu == pi.u_hi && left > 0) {
        w.next(pi);
        pu = pi.u_lo;
      }
    }
    cp_async_commit();
  };
  look_up();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    copy(i);
    look_up();
  }

  // The products.
  at0 = share.at;
  AttnItem it = w.find(share.b, at0);
  long long pos = share.begin;  // units done
  int stage = 0;
  for (;;) {
    const int u0 = it.u_lo + (int)at0;
    const long long item_begin = pos - at0;
    const int units = (int)min((long long)(it.u_hi - u0), share.end - pos);
    const bool split = units != it.u_hi - it.u_lo;
    // q as A fragments, scaled into fp16's range where the cache is 8-bit.
    const int rows = it.s.n * p.group;
    uint32_t qf[D / 16][4];
    float q_mul[2];
    int row_pos[2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int r = it.tile * kRows + g + 8 * hf;
      const int i = r / p.group;
      const bool in = r < rows;
      row_pos[hf] = in ? it.s.ctx + i : -1;
      const T* src = static_cast<const T*>(p.a.q) + (long long)(it.s.first + i) * p.a.stride_q +
                     (it.h * p.group + r - i * p.group) * p.a.stride_q_head;
      float amax = 0.f;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          // Elements of k slots 2q, 2q + 1 (half 0) and 8 + 2q, 9 + 2q (half 1).
          // 8-bit: D / 4 consecutive elements a lane in two runs (see below).
          const int d = FP8 ? (D == 128 ? (s / 4) * 64 + q4 * 16 + (s % 4) * 4 + 2 * half
                                        : q4 * 16 + s * 4 + 2 * half)
                            : 16 * s + 8 * half + 2 * q4;
          uint32_t v = in ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
          qf[s][half * 2 + hf] = v;
          if constexpr (FP8 && std::is_same<T, __nv_bfloat16>::value) {
            const float2 f = Act<T>::unpack(v);
            amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
      }
      q_mul[hf] = 1.0f;
      if constexpr (FP8 && std::is_same<T, __nv_bfloat16>::value) {
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int e = (int)(__float_as_uint(amax) >> 23);  // amax = 2^(e - 127) * 1.x
        float up = 1.0f;
        if (e > 0 && e < 255) {
          up = __uint_as_float((uint32_t)min(max(127 + 13 - (e - 127), 1), 253) << 23);
          q_mul[hf] = 1.0f / up;
        }
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float2 f = Act<T>::unpack(qf[s][half * 2 + hf]);
            qf[s][half * 2 + hf] = Act<__half>::pack(f.x * up, f.y * up);
          }
      }
    }
    const float ks = FP8 && p.c.k_scale ? p.c.k_scale[it.h] : 1.0f;
    const float scale[2] = {p.a.scale * kLog2e * ks * q_mul[0], p.a.scale * kLog2e * ks * q_mul[1]};
    const int low[2] = {p.a.window > 0 ? row_pos[0] - p.a.window : -1, p.a.window > 0 ? row_pos[1] - p.a.window : -1};

    // Positions of the tile's first and last row: tokens between need no mask.
    const int first_pos = it.s.ctx + it.tile * kRows / p.group;
    const int last_low =
        p.a.window > 0 ? it.s.ctx + (min(it.tile * kRows + kRows, rows) - 1) / p.group - p.a.window : -1;

    float o[kNT][4];
#pragma unroll
    for (int j = 0; j < kNT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int n = 0; n < units; ++n) {
      // The stage that was read last is free: ask for the next unit.
      copy(stage == 0 ? kStages - 1 : stage - 1);
      look_up();
      cp_async_wait<kStages - 1>();
      __syncwarp();
      const uint32_t here = seen_sh[warp][stage];
      const uint32_t kt = ring + stage * kStageBytes, vt = kt + kTileBytes;
      stage = stage == kStages - 1 ? 0 : stage + 1;
      if (here != 0) {
        // Even and odd k steps in sums of their own: chains of half the length.
        float s[2][4] = {}, s_odd[2][4] = {};
        if constexpr (!FP8) {
          // Matrices: tokens 0-7 / 8-15 by d halves of a k16 step.
          const int t = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
#pragma unroll
          for (int ss = 0; ss < D / 16; ++ss) {
            uint32_t b[4];
            ldsm4(b, kt + chunk_at(t, 2 * ss + half));
            mma_act<kBf16>(ss & 1 ? s_odd[0] : s[0], qf[ss], b[0], b[1]);
            mma_act<kBf16>(ss & 1 ? s_odd[1] : s[1], qf[ss], b[2], b[3]);
          }
        } else {
          // A product over d may take d in any order: lane quarter q takes the
          // 16 bytes q (and 4 + q) of a token, four k16 steps of 2 + 2.
#pragma unroll
          for (int hf = 0; hf < D / 64; ++hf) {
            const uint4 v0 = lds128_at(kt + chunk_at(g, hf * 4 + q4)), v1 = lds128_at(kt + chunk_at(8 + g, hf * 4 + q4));
            const uint32_t w0[4] = {v0.x, v0.y, v0.z, v0.w}, w1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t b0, b1;
              e4m3x4_to_f16x2x2(w0[i], b0, b1);
              mma_act<false>(i & 1 ? s_odd[0] : s[0], qf[hf * 4 + i], b0, b1);
              e4m3x4_to_f16x2x2(w1[i], b0, b1);
              mma_act<false>(i & 1 ? s_odd[1] : s[1], qf[hf * 4 + i], b0, b1);
            }
          }
        }
        // Scores of rows g, g + 8 and tokens 8 nt + 2q, + 1.
        const int j0 = (u0 + n) * kUnit + warp * 16;
        float mx[2];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] = (s[nt][e] + s_odd[nt][e]) * scale[e >> 1];
        if (here != 0xffff || j0 + 15 > first_pos || j0 <= last_low) {
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int t = nt * 8 + 2 * q4 + (e & 1), j = j0 + t, hf = e >> 1;
              if (!(j <= row_pos[hf] && j > low[hf] && (here >> t & 1))) s[nt][e] = -INFINITY;
            }
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          mx[hf] = fmaxf(fmaxf(s[0][2 * hf], s[0][2 * hf + 1]), fmaxf(s[1][2 * hf], s[1][2 * hf + 1]));
        float al[2];
        bool same = true;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 1));
          mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 2));
          const float mn = fmaxf(m[hf], mx[hf]);
          const float base = mn == -INFINITY ? 0.f : mn;
          al[hf] = exp2_fast(m[hf] - base);
          same = same && m[hf] == mn;
          m[hf] = mn;
          mx[hf] = base;
        }
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][e] = exp2_fast(s[nt][e] - mx[e >> 1]);
        if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) l[hf] *= al[hf];
#pragma unroll
          for (int j = 0; j < kNT; ++j) {
            o[j][0] *= al[0];
            o[j][1] *= al[0];
            o[j][2] *= al[1];
            o[j][3] *= al[1];
          }
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          l[hf] += (s[0][2 * hf] + s[0][2 * hf + 1]) + (s[1][2 * hf] + s[1][2 * hf + 1]);
        using P = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
        const uint32_t pf[4] = {Act<P>::pack(s[0][0], s[0][1]), Act<P>::pack(s[0][2], s[0][3]),
                                Act<P>::pack(s[1][0], s[1][1]), Act<P>::pack(s[1][2], s[1][3])};
        // Values: matrices of tokens 0-7 / 8-15 by 16-byte chunks, transposed.
        const int t = lane & 15, half = lane >> 4;
#pragma unroll
        for (int c = 0; c < kRowBytes / 16; c += 2) {
          uint32_t b[4];
          ldsm4_t(b, vt + chunk_at(t, c + half));
          if constexpr (!FP8) {
            mma_act<kBf16>(o[c], pf, b[0], b[1]);
            mma_act<kBf16>(o[c + 1], pf, b[2], b[3]);
          } else {
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
              // Bytes: token 2q (d 2n, 2n + 1), token 2q + 1 (the same d).
              uint32_t e0, o0, e1, o1;
              e4m3x4_to_f16x2x2(__byte_perm(b[2 * cc], 0, 0x3120), e0, o0);
              e4m3x4_to_f16x2x2(__byte_perm(b[2 * cc + 1], 0, 0x3120), e1, o1);
              mma_act<false>(o[2 * (c + cc)], pf, e0, e1);
              mma_act<false>(o[2 * (c + cc) + 1], pf, o0, o1);
            }
          }
        }
      }
      __syncwarp();
    }
    pos += units;

    // The warps' parts, into warp 0's.
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
      l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
    }
    float4* jo = reinterpret_cast<float4*>(join);
    for (int from = 1; from < kWarps; ++from) {
      if (warp == from) {
#pragma unroll
        for (int j = 0; j < kNT; ++j) jo[j * 32 + lane] = make_float4(o[j][0], o[j][1], o[j][2], o[j][3]);
        if (q4 == 0) {
          sh_ml[0][g] = m[0];
          sh_ml[0][g + 8] = m[1];
          sh_ml[1][g] = l[0];
          sh_ml[1][g + 8] = l[1];
        }
      }
      __syncthreads();
      if (warp == 0) {
        float a[2], b[2];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const float mo = sh_ml[0][g + 8 * hf];
          const float mn = fmaxf(m[hf], mo), base = mn == -INFINITY ? 0.f : mn;
          a[hf] = exp2_fast(m[hf] - base);
          b[hf] = exp2_fast(mo - base);
          l[hf] = l[hf] * a[hf] + sh_ml[1][g + 8 * hf] * b[hf];
          m[hf] = mn;
        }
#pragma unroll
        for (int j = 0; j < kNT; ++j) {
          const float4 v = jo[j * 32 + lane];
          o[j][0] = o[j][0] * a[0] + v.x * b[0];
          o[j][1] = o[j][1] * a[0] + v.y * b[0];
          o[j][2] = o[j][2] * a[1] + v.z * b[1];
          o[j][3] = o[j][3] * a[1] + v.w * b[1];
        }
      }
      __syncthreads();
    }
    const float vs = FP8 && p.c.v_scale ? p.c.v_scale[it.h] : 1.0f;
    const int valid = min(rows - it.tile * kRows, kRows);  // rows of the tile
    // Two (or, 8-bit: four, tiles j and j + 1 interleave) consecutive columns
    // of row g + 8 hf at a time.
    auto pieces = [&](int hf, auto take) {
#pragma unroll
      for (int j = 0; j < kNT; j += FP8 ? 2 : 1) {
        if constexpr (FP8)
          take(column(j, q4, 0), o[j][2 * hf], o[j + 1][2 * hf], o[j][2 * hf + 1], o[j + 1][2 * hf + 1]);
        else
          take(column(j, q4, 0), o[j][2 * hf], o[j][2 * hf + 1], 0.f, 0.f);
      }
    };
    auto place = [&](int r, long long* t, int* h) {  // token and head of row r of the tile
      const int rr = it.tile * kRows + r, i = rr / p.group;
      *t = it.s.first + i;
      *h = it.h * p.group + rr - i * p.group;
    };
    auto write_lse = [&](long long t, int h, float mm, float ll) {
      if (p.a.lse) p.a.lse[t * p.q_heads + h] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) / kLog2e;
    };
    if (!split) {
      if (warp == 0) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int r = g + 8 * hf;
          if (r >= valid) continue;
          long long t;
          int h;
          place(r, &t, &h);
          const float inv = l[hf] == 0.f ? 0.f : vs / l[hf];
          T* out = static_cast<T*>(p.a.out) + t * p.a.stride_o + h * p.a.stride_o_head;
          pieces(hf, [&](int col, float a, float b, float c, float d) {
            if constexpr (FP8)
              *reinterpret_cast<uint2*>(out + col) =
                  make_uint2(Act<T>::pack(a * inv, b * inv), Act<T>::pack(c * inv, d * inv));
            else
              *reinterpret_cast<uint32_t*>(out + col) = Act<T>::pack(a * inv, b * inv);
          });
          if (q4 == 0) write_lse(t, h, m[hf], l[hf]);
        }
      }
    } else {
      // This block's part, and the join by the last block to arrive.
      float* parts = static_cast<float*>(p.parts);
      const int c_first = attn_owner(share, item_begin);
      const int c_last = attn_owner(share, item_begin + (it.u_hi - it.u_lo) - 1);
      // A block's first segment is its part 0; only the item's first block can
      // have begun before it.
      const int first_part = attn_begin(share, c_first) < item_begin;
      auto part = [&](int c) { return parts + (c * 2 + (c == c_first ? first_part : 0)) * (long long)kPartFloats; };
      if (warp == 0) {
        float* mine = part(blockIdx.x);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int r = g + 8 * hf;
          if (r >= valid) continue;
          pieces(hf, [&](int col, float a, float b, float c, float d) {
            if constexpr (FP8)
              __stcg(reinterpret_cast<float4*>(mine + r * D + col), make_float4(a, b, c, d));
            else
              __stcg(reinterpret_cast<float2*>(mine + r * D + col), make_float2(a, b));
          });
          if (q4 == 0) {
            __stcg(mine + 16 * D + r, m[hf]);
            __stcg(mine + 16 * D + 16 + r, l[hf]);
          }
        }
        __threadfence();
        __syncwarp();
        if (lane == 0) {
          const int n = atom_add_acq_rel_gpu(p.counters + c_first, 1);
          sh_last = n == c_last - c_first;
          if (sh_last) p.counters[c_first] = 0;
        }
      }
      __syncthreads();
      if (sh_last) {
        __threadfence();
        // The parts' weights, 32 parts at a time, in the join buffer: [part][row].
        constexpr int kChunk = 32;
        static_assert(kChunk * 16 * 4 <= kNT * 32 * 16, "join buffer");
        const int r = threadIdx.x & 15, lead = threadIdx.x >> 4;  // eight parts at once
        // The first chunk's maxima and sums are kept; more than 32 parts are rare.
        float mc[kChunk / 8], lc[kChunk / 8], mm = -INFINITY;
        auto load_ml = [&](int c0) {
#pragma unroll
          for (int i = 0; i < kChunk / 8; ++i) {
            const int c = c0 + lead + 8 * i;
            mc[i] = -INFINITY;
            lc[i] = 0.f;
            if (c > c_last || r >= valid) continue;
            mc[i] = __ldcg(part(c) + 16 * D + r);
            lc[i] = __ldcg(part(c) + 16 * D + 16 + r);
          }
        };
        for (int c = c_first + kChunk + lead; c <= c_last; c += 8)
          if (r < valid) mm = fmaxf(mm, __ldcg(part(c) + 16 * D + r));
        load_ml(c_first);
#pragma unroll
        for (int i = 0; i < kChunk / 8; ++i) mm = fmaxf(mm, mc[i]);
        sh_red[lead][r] = mm;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) mm = fmaxf(mm, sh_red[i][r]);
        const float base = mm == -INFINITY ? 0.f : mm;
        constexpr int kVec = D / 4, kMine = 16 * kVec / 128;  // four columns a thread, kMine times
        float4 acc[kMine];
#pragma unroll
        for (int i = 0; i < kMine; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        float ll = 0.f;
        for (int c0 = c_first; c0 <= c_last; c0 += kChunk) {
          const int n = min(kChunk, c_last + 1 - c0);
          if (c0 > c_first) load_ml(c0);
#pragma unroll
          for (int i = 0; i < kChunk / 8; ++i) {
            const float a = exp2_fast(mc[i] - base);
            ll += lc[i] * a;
            join[(lead + 8 * i) * 16 + r] = a;
          }
          __syncthreads();
#pragma unroll 8
          for (int c = 0; c < n; ++c) {
            const float4* po = reinterpret_cast<const float4*>(part(c0 + c));
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
              const int at = threadIdx.x + 128 * i, row = at / kVec;
              if (row >= valid) continue;
              const float a = join[c * 16 + row];
              const float4 v = __ldcg(po + at);
              acc[i].x += v.x * a;
              acc[i].y += v.y * a;
              acc[i].z += v.z * a;
              acc[i].w += v.w * a;
            }
          }
          __syncthreads();
        }
        __syncthreads();
        sh_red[lead][r] = ll;
        __syncthreads();
        if (lead == 0) {
          ll = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) ll += sh_red[i][r];
          sh_ml[0][r] = ll;
          if (r < valid) {
            long long t;
            int h;
            place(r, &t, &h);
            write_lse(t, h, mm, ll);
          }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const int at = threadIdx.x + 128 * i, row = at / kVec;
          if (row >= valid) continue;
          long long t;
          int h;
          place(row, &t, &h);
          const float inv = sh_ml[0][row] == 0.f ? 0.f : vs / sh_ml[0][row];
          T* out = static_cast<T*>(p.a.out) + t * p.a.stride_o + h * p.a.stride_o_head + (at - row * kVec) * 4;
          *reinterpret_cast<uint2*>(out) = make_uint2(Act<T>::pack(acc[i].x * inv, acc[i].y * inv),
                                                      Act<T>::pack(acc[i].z * inv, acc[i].w * inv));
        }
      }
      __syncthreads();
    }
    if (pos >= share.end) break;
    w.next(it);
    at0 = 0;
  }
  cp_async_wait<0>();
}

template <typename T, bool FP8, int D>
__global__ void __launch_bounds__(128, RowsKernel<T, FP8, D>::kBlocks) attn_rows_kernel(const __grid_constant__ AttnParams p) {
  RowsKernel<T, FP8, D>::run(p);
}

}  // namespace b2g
