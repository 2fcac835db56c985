// attn_tiles.cuh -- attention of many rows a k/v head (prompt chunks): bound
// by the tensor cores and by the exponentials.
//
// A persistent block an SM walks its share of the work list in units of 128
// cached tokens by 256 rows (two tiles of 128, one tcgen05 M each):
//   warps 0-3, 4-7   softmax of tile 0 and 1: a thread owns a row.  S comes
//                    from tensor memory, P goes back over it in 16 bits.  The
//                    running maximum is only moved (and O rescaled in tensor
//                    memory) once it has grown by 2^8, so P stays in fp16's
//                    range and most units touch O not at all.
//   warps 8-11       keys and values, page by page, into a ring of 128-token
//                    stages (16-byte asynchronous copies in the 128-byte
//                    swizzle; an 8-bit cache is widened to fp16 on the way),
//                    and the rows of q.
//   warp 12          issues S = Q K^T and O += P V.  While one tile's softmax
//                    runs, the tensor cores work on the other tile.
// Tensor memory: S0, S1 (128 columns each), O0, O1 (D columns each).  A tile's
// S(j + 1) is issued behind its O += P(j) V(j) and one commit covers both, so
// the softmax warps that see S(j + 1) may touch O.
// Every wait is bounded; after one has run out its thread goes through the
// remaining steps without waiting, so that barriers still meet.
#pragma once
#include "attn_rows.cuh"
#include "tc.cuh"

namespace b2g {

template <int N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <typename T, bool FP8, int D>
struct TilesKernel {
  static constexpr int kRows = 256, kTile = 128, kUnit = 128, kThreads = 512;
  static constexpr bool kBf16 = !FP8 && std::is_same<T, __nv_bfloat16>::value;  // the products' type
  static constexpr bool kScaleQ = FP8 && std::is_same<T, __nv_bfloat16>::value;  // bf16 q into fp16's range
  static constexpr int kPanels = D / 64;             // 128-byte panels of a row
  static constexpr int kPanelBytes = kTile * 128;
  static constexpr int kTileBytes = kPanels * kPanelBytes;  // 128 tokens or rows, 16-bit
  static constexpr int kStages = 4;
  static constexpr int kStagingBytes = FP8 ? kTile * D : 0;  // an 8-bit tile
  static constexpr int kOffRing = 2 * kTileBytes, kOffStaging = kOffRing + kStages * kTileBytes;
  static constexpr int kSmem = kOffStaging + 2 * kStagingBytes;
  static constexpr int kPartFloats = kTile * D + 2 * kTile;  // of a tile: [D / 4][row][4], maxima, sums
  using Work = AttnWork<kRows, kUnit>;
  using P16 = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;

  struct Shared {
    uint64_t kv_full[kStages], kv_empty[kStages], q_full, q_empty, s_full[2], p_full[2], o_full[2], drain;
    long long share[kThreads / 32];
    long long row_at[2][kTile];  // the unit's tokens' rows in the cache, -1: none
    uint32_t there[8][4];        // bit t: token t of unit (u mod 8) is there
    uint8_t q_exp[kRows];        // kScaleQ: exponent of the row's power of two
    uint32_t tmem;
    int last[2];
  };
  static_assert(sizeof(Shared) <= 3072, "static shared memory");

  // Byte of 16-byte chunk c (of D / 8) of row r in a 16-bit tile.
  static __device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    return (c >> 3) * kPanelBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
  }

  static __device__ void load(const AttnParams& p, Shared& s, uint32_t smem, const AttnShare& share);
  static __device__ void multiply(const AttnParams& p, Shared& s, uint32_t smem, const AttnShare& share);
  static __device__ void softmax(const AttnParams& p, Shared& s, const AttnShare& share, int tile);
};

// The segments (parts of items) of a share, in order.
template <typename Work>
struct AttnWalk {
  const Work& w;
  const AttnShare& share;
  AttnItem it;
  long long pos;
  int u0, units;     // this segment's units
  long long origin;  // the item's first unit in the list
  bool fresh = true;
  __device__ __forceinline__ AttnWalk(const Work& w_, const AttnShare& s_) : w(w_), share(s_), pos(s_.begin) {}
  __device__ __forceinline__ bool next() {
    if (!fresh) pos += units;
    if (pos >= share.end) return false;
    long long at = 0;
    if (fresh) {
      at = share.at;
      it = w.find(share.b, at);
    } else {
      w.next(it);
    }
    fresh = false;
    u0 = it.u_lo + (int)at;
    origin = pos - at;
    units = (int)min((long long)(it.u_hi - u0), share.end - pos);
    return true;
  }
  __device__ __forceinline__ bool split() const { return units != it.u_hi - it.u_lo; }
  __device__ __forceinline__ int rows() const { return it.s.n * w.p.group - it.tile * 256; }  // from the item's first on
};

// ---------------------------------------------------------------------------
// Loads
// ---------------------------------------------------------------------------
template <typename T, bool FP8, int D>
__device__ void TilesKernel<T, FP8, D>::load(const AttnParams& p, Shared& s, uint32_t smem, const AttnShare& share) {
  const int tid = threadIdx.x & 127, lane = tid & 31, warp = tid >> 5;
  const Work w(p);
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (ok && !mbar_wait_bounded(bar, parity)) {
      *p.error = kErrEmptyWait;
      ok = false;
    }
  };
  // Copies are announced two groups behind, once they have landed.
  uint64_t* pending[2] = {nullptr, nullptr};
  auto announce = [&](uint64_t* bar) {
    if (bar) {
      fence_proxy_async_shared();
      mbar_arrive(bar);
    }
  };
  auto commit = [&](uint64_t* bar) {
    cp_async_commit();
    cp_async_wait<2>();
    announce(pending[0]);
    pending[0] = pending[1];
    pending[1] = bar;
  };
  auto flush = [&]() {
    cp_async_wait<0>();
    announce(pending[0]);
    announce(pending[1]);
    pending[0] = pending[1] = nullptr;
  };

  // A thread looks up token tid of a unit.
  auto look_up = [&](const AttnItem& it, int unit) -> long long {
    const int j = unit * kUnit + tid;
    if (j < it.lo || j >= it.hi) return -1;
    const int pg = j / p.c.page_size;
    const int page = page_of(p.b, p.c, it.b, pg, p.error);
    if (page < 0) return -1;
    return page * p.c.stride_page + (long long)(j - pg * p.c.page_size) * p.c.stride_token + it.h * p.c.stride_head;
  };
  auto note = [&](int n, long long at) {  // unit n of this block
    s.row_at[n & 1][tid] = at;
    const uint32_t mask = __ballot_sync(0xffffffffu, at >= 0);
    if (lane == 0) s.there[n & 7][warp] = mask;
  };

  constexpr int kChunks = D * (FP8 ? 1 : 2) / 16;  // of a cached row
  constexpr int kPasses = kTile * kChunks / 128;   // 16-byte copies a thread
  const int c = tid % kChunks, t0 = tid / kChunks;
  auto copy_tile = [&](int n, const void* cache, uint32_t dst, bool staged) {
    const uint8_t* base = static_cast<const uint8_t*>(cache) + c * 16;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int t = t0 + i * (128 / kChunks);
      const long long at = s.row_at[n & 1][t];
      const bool in = at >= 0;
      cp_async16_or_zero(dst + (staged ? (i * 128 + tid) * 16 : chunk_at(t, c)),
                         base + (in ? at * (FP8 ? 1 : 2) : 0), in);
    }
  };

  int tiles = 0;  // ring tiles asked for (16-bit) or filled (8-bit)
  int n_q = 0;    // q loads
  auto load_q = [&](const AttnWalk<Work>& k) {
    if (n_q > 0) wait(&s.q_empty, (n_q - 1) & 1);
    ++n_q;
    const int rows = k.rows();
    for (int i = 0; i < 2; ++i) {
      const int r = i * 128 + tid, abs_r = k.it.tile * kRows + r;
      const bool in = r < rows;
      const int tok = abs_r / p.group;
      const T* src = static_cast<const T*>(p.a.q);
      if (in)
        src += (long long)(k.it.s.first + tok) * p.a.stride_q + (k.it.h * p.group + abs_r - tok * p.group) * p.a.stride_q_head;
      const uint32_t dst = smem + i * kTileBytes;
      if constexpr (!kScaleQ) {
#pragma unroll
        for (int ch = 0; ch < D / 8; ++ch) cp_async16_or_zero(dst + chunk_at(tid, ch), src + (in ? ch * 8 : 0), in);
      } else {
        uint32_t top = 0;
        for (int ch = 0; in && ch < D / 8; ++ch) {
          const uint4 v = *reinterpret_cast<const uint4*>(src + ch * 8);
          for (uint32_t x : {v.x, v.y, v.z, v.w}) top = max(top, max(x & 0x7fff, x >> 16 & 0x7fff));
        }
        const int e = (int)(top >> 7);  // bf16 exponent of the largest
        const int ue = e > 0 && e < 255 ? min(max(127 + 13 - (e - 127), 1), 253) : 127;
        s.q_exp[r] = (uint8_t)ue;
        const float by = __uint_as_float((uint32_t)ue << 23);
        for (int ch = 0; ch < D / 8; ++ch) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (in) v = *reinterpret_cast<const uint4*>(src + ch * 8);
          uint32_t o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float2 f = Act<T>::unpack(o[x]);
            o[x] = Act<__half>::pack(f.x * by, f.y * by);
          }
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst + chunk_at(tid, ch)), "r"(o[0]), "r"(o[1]),
                       "r"(o[2]), "r"(o[3])
                       : "memory");
        }
      }
    }
  };

  if constexpr (!FP8) {
    AttnWalk<Work> k(w, share);
    bool more = k.next();
    if (more) note(0, look_up(k.it, k.u0));
    for (int n = 1; more; ++n) {  // the unit whose rows are looked up next
      const int units = k.units;
      for (int j = 0; j < units; ++j, ++n) {
        named_sync(3, 128);  // the unit's rows are known; the one before is done with its
        for (int kv = 0; kv < 2; ++kv, ++tiles) {
          const int st = tiles % kStages;
          if (tiles >= kStages) wait(&s.kv_empty[st], (tiles / kStages - 1) & 1);
          copy_tile(n - 1, kv == 0 ? p.c.k : p.c.v, smem + kOffRing + st * kTileBytes, false);
          commit(&s.kv_full[st]);
          if (j == 0 && kv == 0) {
            load_q(k);
            commit(&s.q_full);
          }
        }
        if (j + 1 < units) note(n, look_up(k.it, k.u0 + j + 1));
      }
      --n;
      more = k.next();
      if (more) note(n, look_up(k.it, k.u0));
    }
    flush();
  } else {
    // 8-bit: copies run two tiles ahead into private staging slots (a thread
    // widens what it has copied itself).
    uint32_t slot[2] = {smem + kOffStaging, smem + kOffStaging + kStagingBytes};
    AttnWalk<Work> ahead(w, share), k(w, share);
    int an = 0, aj = 0, akv = 0;  // the next tile to copy: unit an, its values if akv
    bool amore = ahead.next();
    if (amore) note(0, look_up(ahead.it, ahead.u0));
    auto copy_next = [&](int to) {
      if (amore) {
        if (akv == 0) named_sync(3, 128);
        copy_tile(an, akv == 0 ? p.c.k : p.c.v, slot[to], true);
        if (akv == 1) {
          ++an;
          if (++aj == ahead.units) {
            amore = ahead.next();
            aj = 0;
          }
          if (amore) note(an, look_up(ahead.it, ahead.u0 + aj));
        }
        akv ^= 1;
      }
      cp_async_commit();
    };
    copy_next(0);
    copy_next(1);
    while (k.next()) {
      for (int j = 0; j < k.units; ++j)
        for (int kv = 0; kv < 2; ++kv, ++tiles) {
          const int st = tiles % kStages, sl = tiles & 1;
          cp_async_wait<1>();
          uint4 v[kPasses];
#pragma unroll
          for (int i = 0; i < kPasses; ++i) v[i] = lds128_at(slot[sl] + (i * 128 + tid) * 16);
          if (tiles >= kStages) wait(&s.kv_empty[st], (tiles / kStages - 1) & 1);
          const uint32_t dst = smem + kOffRing + st * kTileBytes;
#pragma unroll
          for (int i = 0; i < kPasses; ++i) {
            const int t = t0 + i * (128 / kChunks);
            const uint32_t wd[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
            uint32_t o[8];
#pragma unroll
            for (int x = 0; x < 4; ++x) e4m3x4_to_f16x2x2(wd[x], o[2 * x], o[2 * x + 1]);
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst + chunk_at(t, 2 * c)), "r"(o[0]), "r"(o[1]),
                         "r"(o[2]), "r"(o[3])
                         : "memory");
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst + chunk_at(t, 2 * c + 1)), "r"(o[4]),
                         "r"(o[5]), "r"(o[6]), "r"(o[7])
                         : "memory");
          }
          copy_next(sl);  // the slot's bytes are in the ring
          announce(&s.kv_full[st]);
          if (j == 0 && kv == 0) {
            load_q(k);
            cp_async_commit();
            cp_async_wait<0>();
            announce(&s.q_full);
          }
        }
    }
    cp_async_wait<0>();
  }
}

// ---------------------------------------------------------------------------
// Products
// ---------------------------------------------------------------------------
template <typename T, bool FP8, int D>
__device__ void TilesKernel<T, FP8, D>::multiply(const AttnParams& p, Shared& s, uint32_t smem, const AttnShare& share) {
  constexpr int kFmt = kBf16 ? 1 : 0;
  constexpr uint32_t kQk = tc_idesc(1, kFmt, kFmt, 0, kUnit), kPv = tc_idesc(1, kFmt, kFmt, 1, D);
  const Work w(p);
  AttnWalk<Work> k(w, share);
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (ok && !mbar_wait_bounded(bar, parity)) {
      *p.error = kErrFullWait;
      ok = false;
    }
    tc_fence_after();
  };
  const uint32_t tm = s.tmem;
  auto wait_tile = [&](int i) { wait(&s.kv_full[i % kStages], (i / kStages) & 1); };
  auto qk = [&](int t, int i) {  // S_t = Q_t (ring tile i)^T
    if (!ok) return;
    const uint64_t a = smem_desc_sw128(smem + t * kTileBytes, 16, 1024);
    const uint64_t b = smem_desc_sw128(smem + kOffRing + (i % kStages) * kTileBytes, 16, 1024);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const uint32_t off = ((ks >> 2) * kPanelBytes + (ks & 3) * 32) >> 4;
      mma_f16_ss(tm + t * kUnit, a + off, b + off, kQk, ks > 0);
    }
  };
  auto pv = [&](int t, int i, bool first) {  // O_t (+)= P_t (ring tile i)
    if (!ok) return;
    const uint64_t b = smem_desc_sw128(smem + kOffRing + (i % kStages) * kTileBytes, kPanelBytes, 1024);
#pragma unroll
    for (int ks = 0; ks < kUnit / 16; ++ks)
      mma_f16_ts(tm + 2 * kUnit + t * D, tm + t * kUnit + ks * 8, b + ((ks * 2048) >> 4), kPv, !first || ks > 0);
  };
  int i = 0, segs = 0;        // ring tiles so far, segments
  uint32_t p_par[2] = {0, 0};
  while (k.next()) {
    const int nt = k.rows() > kTile ? 2 : 1;
    wait(&s.q_full, segs & 1);
    wait_tile(i);
    for (int t = 0; t < nt; ++t) {
      qk(t, i);
      tc_commit(&s.s_full[t]);
    }
    tc_commit(&s.kv_empty[i % kStages]);
    if (k.units == 1) tc_commit(&s.q_empty);
    for (int j = 0; j < k.units; ++j, i += 2) {
      const bool last = j + 1 == k.units;
      wait_tile(i + 1);
      for (int t = 0; t < nt; ++t) {
        wait(&s.p_full[t], p_par[t]);
        p_par[t] ^= 1;
        pv(t, i + 1, j == 0);
        if (last) {
          tc_commit(&s.o_full[t]);
        } else {
          if (t == 0) wait_tile(i + 2);
          qk(t, i + 2);
          tc_commit(&s.s_full[t]);
        }
      }
      tc_commit(&s.kv_empty[(i + 1) % kStages]);
      if (!last) tc_commit(&s.kv_empty[(i + 2) % kStages]);
      if (j + 2 == k.units) tc_commit(&s.q_empty);
    }
    ++segs;
  }
  if (!ok) {
    tc_commit(&s.drain);
    mbar_wait_bounded(&s.drain, 0);
  }
}

// ---------------------------------------------------------------------------
// Softmax, results, and the join of split items
// ---------------------------------------------------------------------------
template <typename T, bool FP8, int D>
__device__ void TilesKernel<T, FP8, D>::softmax(const AttnParams& p, Shared& s, const AttnShare& share, int tile) {
  const int tid = threadIdx.x & 127, warp = tid >> 5;
  const uint32_t lane_at = (uint32_t)(warp * 32) << 16;
  const uint32_t tm_s = s.tmem + lane_at + tile * kUnit, tm_o = s.tmem + lane_at + 2 * kUnit + tile * D;
  const Work w(p);
  AttnWalk<Work> k(w, share);
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (ok && !mbar_wait_bounded(bar, parity)) {
      *p.error = kErrFullWait;
      ok = false;
    }
    __syncwarp();
    tc_fence_after();
  };
  uint32_t s_par = 0, o_par = 0;
  int n = 0;  // units of this block so far
  while (k.next()) {
    const int rows = k.rows();
    if (tile * kTile >= rows) {
      n += k.units;
      continue;
    }
    const int r = tile * kTile + tid, abs_r = k.it.tile * kRows + r;
    const bool in = r < rows;
    const int tok = abs_r / p.group;
    const int row_pos = in ? k.it.s.ctx + tok : -1;
    const int low = p.a.window > 0 ? row_pos - p.a.window : -1;
    // Positions of the tile's first and last row: units between need no mask.
    const int first_pos = k.it.s.ctx + (k.it.tile * kRows + tile * kTile) / p.group;
    const int last_low =
        p.a.window > 0 ? k.it.s.ctx + (k.it.tile * kRows + min(tile * kTile + kTile, rows) - 1) / p.group - p.a.window : -1;
    float scale = p.a.scale * kLog2e * (FP8 && p.c.k_scale ? p.c.k_scale[k.it.h] : 1.0f);
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j < k.units; ++j, ++n) {
      const int j0 = (k.u0 + j) * kUnit;
      wait(&s.s_full[tile], s_par);
      s_par ^= 1;
      if constexpr (kScaleQ) {
        if (j == 0) scale *= 1.0f / __uint_as_float((uint32_t)s.q_exp[r] << 23);
      }
      uint32_t x[4][32];
#pragma unroll
      for (int i = 0; i < 4; ++i) tmem_ld32(tm_s + 32 * i, x[i]);
      const uint32_t* there = s.there[n & 7];
      const uint32_t all = there[0] & there[1] & there[2] & there[3];
      tmem_wait_ld();
      if (all != 0xffffffffu || j0 + kUnit - 1 > first_pos || j0 <= last_low) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int below = row_pos - (j0 + 32 * i) + 1, hidden = low - (j0 + 32 * i) + 1;
          uint32_t mask = there[i];
          mask &= below >= 32 ? 0xffffffffu : below <= 0 ? 0u : (1u << below) - 1;
          mask &= hidden >= 32 ? 0u : hidden <= 0 ? 0xffffffffu : ~((1u << hidden) - 1);
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (!(mask >> c & 1)) x[i][c] = 0xff800000u;
        }
      }
      float mx[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mx[i] = __uint_as_float(x[i][0]);
#pragma unroll
        for (int c = 1; c < 32; ++c) mx[i] = fmaxf(mx[i], __uint_as_float(x[i][c]));
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
      if (j == 0) {
        m = top;
      } else {
        const bool grown = top > m + 8.0f;
        if (__any_sync(0xffffffffu, grown)) {
          const float by = grown ? exp2_fast(m - top) : 1.0f;
          if (grown) m = top;
          l *= by;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            uint32_t o[32];
            tmem_ld32(tm_o + 32 * i, o);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * by);
            tmem_st32(tm_o + 32 * i, o);
          }
        }
      }
      const float neg = m == -INFINITY ? 0.f : -m;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < 64; c += 2) {
          const float a = exp2_fast(fmaf(__uint_as_float(x[2 * i + c / 32][c % 32]), scale, neg));
          const float b = exp2_fast(fmaf(__uint_as_float(x[2 * i + c / 32][c % 32 + 1]), scale, neg));
          sum[c & 2] += a;
          sum[(c & 2) + 1] += b;
          pk[c / 2] = Act<P16>::pack(a, b);
        }
        tmem_st32(tm_s + 32 * i, pk);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&s.p_full[tile]);
    }
    wait(&s.o_full[tile], o_par);
    o_par ^= 1;

    const float vs = FP8 && p.c.v_scale ? p.c.v_scale[k.it.h] : 1.0f;
    const long long t = k.it.s.first + tok;
    const int h = k.it.h * p.group + abs_r - tok * p.group;
    T* out = static_cast<T*>(p.a.out) + t * p.a.stride_o + h * p.a.stride_o_head;
    auto write32 = [&](int c0, const float* v, float inv) {  // columns c0 .. c0 + 31
#pragma unroll
      for (int c = 0; c < 32; c += 8)
        *reinterpret_cast<uint4*>(out + c0 + c) =
            make_uint4(Act<T>::pack(v[c] * inv, v[c + 1] * inv), Act<T>::pack(v[c + 2] * inv, v[c + 3] * inv),
                       Act<T>::pack(v[c + 4] * inv, v[c + 5] * inv), Act<T>::pack(v[c + 6] * inv, v[c + 7] * inv));
    };
    auto write_lse = [&](float mm, float ll) {
      if (p.a.lse) p.a.lse[t * p.q_heads + h] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) / kLog2e;
    };
    if (!k.split()) {
      const float inv = l == 0.f ? 0.f : vs / l;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        uint32_t o[32];
        tmem_ld32(tm_o + 32 * i, o);
        tmem_wait_ld();
        float f[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) f[c] = l == 0.f ? 0.f : __uint_as_float(o[c]);
        if (in) write32(32 * i, f, inv);
      }
      if (in) write_lse(m, l);
    } else {
      float* parts = static_cast<float*>(p.parts);
      const int c_first = attn_owner(share, k.origin);
      const int c_last = attn_owner(share, k.origin + (k.it.u_hi - k.it.u_lo) - 1);
      auto part = [&](int c) {  // its first segment unless it began before this item
        const bool first = (long long)c * share.total / share.blocks >= k.origin;
        return parts + (((long long)c * 2 + (first ? 0 : 1)) * 2 + tile) * kPartFloats;
      };
      float* mine = part(blockIdx.x);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        uint32_t o[32];
        tmem_ld32(tm_o + 32 * i, o);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 32; c += 4)
          __stcg(reinterpret_cast<float4*>(mine) + (8 * i + c / 4) * kTile + tid,
                 make_float4(__uint_as_float(o[c]), __uint_as_float(o[c + 1]), __uint_as_float(o[c + 2]),
                             __uint_as_float(o[c + 3])));
      }
      __stcg(mine + kTile * D + tid, m);
      __stcg(mine + kTile * D + kTile + tid, l);
      __threadfence();
      named_sync(1 + tile, 128);
      if (tid == 0) {
        int* counter = p.counters + 2 * c_first + tile;
        s.last[tile] = atom_add_acq_rel_gpu(counter, 1) == c_last - c_first;
        if (s.last[tile]) *counter = 0;
      }
      named_sync(1 + tile, 128);
      if (s.last[tile]) {
        __threadfence();
        float mm = -INFINITY, ll = 0.f;
#pragma unroll 4
        for (int c = c_first; c <= c_last; ++c) mm = fmaxf(mm, __ldcg(part(c) + kTile * D + tid));
        const float base = mm == -INFINITY ? 0.f : mm;
#pragma unroll 4
        for (int c = c_first; c <= c_last; ++c)
          ll += __ldcg(part(c) + kTile * D + kTile + tid) * exp2_fast(__ldcg(part(c) + kTile * D + tid) - base);
        const float inv = ll == 0.f ? 0.f : vs / ll;
        for (int i = 0; i < D / 32; ++i) {
          float f[32] = {};
#pragma unroll 2
          for (int c = c_first; c <= c_last; ++c) {
            const float a = exp2_fast(__ldcg(part(c) + kTile * D + tid) - base);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const float4 v = __ldcg(reinterpret_cast<const float4*>(part(c)) + (8 * i + x) * kTile + tid);
              f[4 * x] += v.x * a;
              f[4 * x + 1] += v.y * a;
              f[4 * x + 2] += v.z * a;
              f[4 * x + 3] += v.w * a;
            }
          }
          if (in) write32(32 * i, f, inv);
        }
        if (in) write_lse(mm, ll);
      }
    }
    tc_fence_before();  // this tile's O is read: the next P lets it be overwritten
  }
}

template <typename T, bool FP8, int D>
__global__ void __launch_bounds__(512, 1) attn_tiles_kernel(const __grid_constant__ AttnParams p) {
  using K = TilesKernel<T, FP8, D>;
  extern __shared__ __align__(1024) uint8_t dyn[];
  __shared__ typename K::Shared s;
  const int warp = threadIdx.x >> 5;
  const uint32_t smem = smem_addr(dyn);
  if (smem & 1023) {  // the swizzle needs it; the array's alignment gives it
    *p.error = kErrAlignment;
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < K::kStages; ++i) {
      mbar_init(&s.kv_full[i], 128);
      mbar_init(&s.kv_empty[i], 1);
    }
    mbar_init(&s.q_full, 128);
    mbar_init(&s.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.p_full[i], 128);
      mbar_init(&s.o_full[i], 1);
    }
    mbar_init(&s.drain, 1);
    fence_mbarrier_init();
  }
  if (warp == 12) tmem_alloc(&s.tmem, 512);
  tc_fence_before();
  pdl_wait();
  pdl_launch_dependents();
  const typename K::Work w(p);
  const AttnShare share = attn_share(w, p.least_units, s.share);  // synchronises the block
  tc_fence_after();
  // 512 threads of 128 registers: 2 x 128 x 192 + 2 x 128 x 64 is the same sum.
  if (warp < 8) {
    reg_inc<192>();
    K::softmax(p, s, share, warp >> 2);
  } else if (warp < 12) {
    reg_dec<64>();
    K::load(p, s, smem, share);
  } else {
    reg_dec<64>();
    if (threadIdx.x == 12 * 32) K::multiply(p, s, smem, share);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(s.tmem, 512);
}

}  // namespace b2g
