// attn_tiles.cuh -- attention of many rows a k/v head (prompt chunks): bound
// by the tensor cores and by the exponentials.
//
// A persistent block an SM walks its share of the work list in units of 128
// cached tokens by 256 rows (two tiles of 128, one tcgen05 M each):
//   warps 0-3, 4-7   softmax of tile 0 and 1: a thread owns a row.  64 columns
//                    of S come from tensor memory into registers, P goes back
//                    over them in 16 bits.  The running maximum is only moved
//                    (and O rescaled in tensor memory) once it has grown by
//                    2^8, so P stays in fp16's range and most steps touch O
//                    not at all.
//   warps 8-11       keys and values, page by page, into a ring of 128-token
//                    stages (16-byte asynchronous copies in the 128-byte
//                    swizzle; an 8-bit cache is widened to fp16 on the way),
//                    and the rows of q.
//   warps 12, 13     issue S = Q K^T and O += P V of tile 0 and 1 in steps of 64
//                    tokens.  (Two of them: a wait of theirs stands ~250 clocks
//                    in line behind the softmax warps' exponentials, and one
//                    warp's waits are the other's products.)
// Tensor memory: S0, S1 (two buffers of 64 columns each), O0, O1 (D columns
// each).  With two buffers the scores of step u + 1 are there when a tile's
// softmax gets to them, so neither side waits for the other's latency (with
// one buffer of 128 columns a unit took 4650 clocks, 1800 of them from a P to
// the next S).  A tile's S(u + 2) is issued behind its O += P(u) V(u) into the
// same buffer and one commit covers both.  An item's last two O += P V have a
// barrier of their own: the next item's S is issued without a word from the
// softmax warps, and on s_full its phase could end before a warp that stood
// still had seen theirs.
// Three chunks of up to 2048 tokens at up to 6000, 32 heads on 8, bf16: 395 us in
// a short run, 0.89 PFLOP/s (442 in a long one at the power limit); over an 8-bit
// cache 467.  The softmax warps take 2000 clocks for 64 columns of both tiles, of
// which the exponentials are 1024.  Of issue slots 40% are used, of the tensor
// pipe's time 40%, of the special-function unit's 45%; registers are spilled, but
// outside the loop (230 spill loads of a scheduler's warps in a launch).
// Every wait is bounded.  After one has run out a products' warp is done; a thread
// of the others goes through the remaining steps without waiting, so that their
// barriers still meet (the loads without issuing or announcing anything, which a
// barrier's later phase would count).  The block ends behind the copies and
// products that it has issued.
#pragma once
#include "attn_rows.cuh"
#include "tc.cuh"

namespace b2g {

// Maximum of three; a NaN stays one.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Two floats in one register pair, one instruction for both.
__device__ __forceinline__ uint64_t pair2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// The cache as tensors of (dim, row of a page, head, page) for whole units of
// pages that a unit is cut into evenly (box_rows rows a load, 0: not so).
struct AttnTma {
  CUtensorMap k, v;
  int box_rows;
};
struct AttnTilesParams {
  AttnParams p;
  AttnTma tma;
};

template <typename T, bool FP8, int D>
struct TilesKernel {
  static constexpr int kRows = 256, kTile = 128, kUnit = 128, kStep = 64, kThreads = 512;
  static constexpr bool kBf16 = !FP8 && std::is_same<T, __nv_bfloat16>::value;  // the products' type
  static constexpr bool kScaleQ = FP8 && std::is_same<T, __nv_bfloat16>::value;  // bf16 q into fp16's range
  static constexpr int kPanels = D / 64;             // 128-byte panels of a row
  static constexpr int kPanelBytes = kTile * 128;
  static constexpr int kTileBytes = kPanels * kPanelBytes;  // 128 tokens or rows, 16-bit
  static constexpr int kStages = FP8 ? 4 : 5;
  static constexpr int kStagingBytes = FP8 ? kTile * D : 0;  // an 8-bit tile
  static constexpr int kOffRing = 2 * kTileBytes, kOffStaging = kOffRing + kStages * kTileBytes;
  static constexpr int kSmem = kOffStaging + 2 * kStagingBytes;
  static constexpr int kPartFloats = kTile * D + 2 * kTile;  // of a tile: [D / 4][row][4], maxima, sums
  using Work = AttnWork<kRows, kUnit>;
  using P16 = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;

  struct Shared {
    uint64_t kv_full[kStages], kv_empty[kStages], q_full, q_empty, s_full[2][2], p_full[2][2], o_full[2][2],
        drain[2];
    long long share[kThreads / 32];
    long long row_at[2][kTile];  // the unit's tokens' rows in the cache, -1: none
    uint32_t there[8][4];        // bit t: token t of unit (u mod 8) is there
    // kScaleQ: exponent of the row's power of two, by the segment's parity.  The
    // next segment's q may be loaded as soon as this one's last Q K^T is done, and
    // the softmax warps may still be writing the one before.  Of that one they have
    // read theirs: its products waited for their P.
    uint8_t q_exp[2][kRows];
    uint32_t tmem;
    int last[2];
  };
  static_assert(sizeof(Shared) <= 3 * 1024, "static shared memory");

  // Byte of 16-byte chunk c (of D / 8) of row r in a 16-bit tile.
  static __device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    return (c >> 3) * kPanelBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
  }

  static __device__ void load(const AttnTma& tma, const AttnParams& p, Shared& s, uint32_t smem, const AttnShare& share);
  static __device__ void multiply(const AttnParams& p, Shared& s, uint32_t smem, const AttnShare& share, int t);
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
__device__ void TilesKernel<T, FP8, D>::load(const AttnTma& tma, const AttnParams& p, Shared& s, uint32_t smem, const AttnShare& share) {
  const int tid = threadIdx.x & 127, lane = tid & 31, warp = tid >> 5;
  const Work w(p);
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (ok && !mbar_wait_spin(bar, parity)) {
      *p.error = kErrEmptyWait;
      ok = false;
    }
  };
  // Copies are announced once they have landed: two groups behind, or all of
  // them before the thread blocks for a free stage.
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
    if (n_q > 0 && !mbar_test(&s.q_empty, (n_q - 1) & 1)) {
      flush();
      wait(&s.q_empty, (n_q - 1) & 1);
    }
    ++n_q;
    if (!ok) return;
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
        s.q_exp[~n_q & 1][r] = (uint8_t)ue;  // n_q counts this one already
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
          sts128_at(dst + chunk_at(tid, ch), make_uint4(o[0], o[1], o[2], o[3]));
        }
      }
    }
  };

  if constexpr (!FP8) {
    AttnWalk<Work> k(w, share);
    bool more = k.next();
    // Warp 0's lanes each load one box of whole units.
    const int boxes = tma.box_rows ? kUnit / tma.box_rows : 0;
    const int box = lane / kPanels, panel = lane % kPanels;
    int box_page[2] = {0, 0}, box_row[2] = {0, 0};
    auto look_up_box = [&](int n, int unit) {
      if (warp != 0 || box >= boxes) return;
      const int j = unit * kUnit + box * tma.box_rows;
      const int pg = j / p.c.page_size;
      const int page = pg < p.b.max_pages ? p.b.page_table[(long long)k.it.b * p.b.page_table_stride + pg] : 0;
      const int row = j - pg * p.c.page_size;
      if (n & 1) {
        box_page[1] = page;
        box_row[1] = row;
      } else {
        box_page[0] = page;
        box_row[0] = row;
      }
    };
    auto prepare = [&](int n, int unit) {
      look_up_box(n, unit);
      note(n, look_up(k.it, unit));
    };
    int sent = 0;  // tiles before a wait ran out
    if (more) prepare(0, k.u0);
    for (int n = 1; more; ++n) {  // the unit whose rows are looked up next
      const int units = k.units;
      for (int j = 0; j < units; ++j, ++n) {
        named_sync(3, 128);  // the unit's rows are known; the one before is done with its
        const uint32_t* there = s.there[(n - 1) & 7];
        const bool whole = boxes && (there[0] & there[1] & there[2] & there[3]) == 0xffffffffu;
        for (int kv = 0; kv < 2; ++kv) {
          const int st = tiles % kStages;
          if (tiles >= kStages) {
            const uint32_t parity = (tiles / kStages - 1) & 1;
            if (!mbar_test(&s.kv_empty[st], parity)) {
              flush();
              wait(&s.kv_empty[st], parity);
            }
          }
          if (ok) sent = tiles + 1;
          ++tiles;
          uint64_t* full = &s.kv_full[st];
          const uint32_t dst = smem + kOffRing + st * kTileBytes;
          if (whole) {
            if (ok) {
              if (tid == 0) mbar_arrive_expect_tx(full, kTileBytes);
              else mbar_arrive(full);
            }
            __syncwarp();
            if (warp == 0 && box < boxes && ok)
              tma_load_4d(dst + panel * kPanelBytes + box * tma.box_rows * 128, kv == 0 ? &tma.k : &tma.v, panel * 64,
                          (n & 1) ? box_row[0] : box_row[1], k.it.h, (n & 1) ? box_page[0] : box_page[1], full);
          } else if (ok) {
            copy_tile(n - 1, kv == 0 ? p.c.k : p.c.v, dst, false);
            commit(full);
          }
          if (j == 0 && kv == 0) {
            load_q(k);
            if (ok) commit(&s.q_full);
          }
        }
        if (whole) flush();  // copies behind which none may come for long
        if (j + 1 < units) prepare(n, k.u0 + j + 1);
      }
      --n;
      more = k.next();
      if (more) prepare(n, k.u0);
    }
    flush();
    // Whoever was to use them may have given up: bulk copies land before this
    // block's memory goes.
    bool landed = true;
    for (int j = max(0, sent - kStages); j < sent; ++j)
      landed = landed && mbar_wait_spin(&s.kv_full[j % kStages], (j / kStages) & 1);
    if (!landed) *p.error = kErrDrainWait;
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
            sts128_at(dst + chunk_at(t, 2 * c), make_uint4(o[0], o[1], o[2], o[3]));
            sts128_at(dst + chunk_at(t, 2 * c + 1), make_uint4(o[4], o[5], o[6], o[7]));
          }
          copy_next(sl);  // the slot's bytes are in the ring
          if (ok) announce(&s.kv_full[st]);
          if (j == 0 && kv == 0) {
            load_q(k);
            cp_async_commit();
            cp_async_wait<0>();
            if (ok) announce(&s.q_full);
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
__device__ void TilesKernel<T, FP8, D>::multiply(const AttnParams& p, Shared& s, uint32_t smem, const AttnShare& share,
                                       int t) {
  constexpr int kFmt = kBf16 ? 1 : 0;
  constexpr uint32_t kQk = tc_idesc(1, kFmt, kFmt, 0, kStep), kPv = tc_idesc(1, kFmt, kFmt, 1, D);
  const Work w(p);
  AttnWalk<Work> k(w, share);
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    const bool ok = mbar_wait_spin(bar, parity);
    if (!ok) *p.error = kErrFullWait;
    tc_fence_after();
    return ok;
  };
  const uint32_t tm = s.tmem;
  // Places in the ring, kept by counting: this thread's own instructions are
  // on the way from one product to the next.
  struct Place {
    int st = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ Place after() const {
      Place r;
      r.st = st + 1 == kStages ? 0 : st + 1;
      r.parity = parity ^ (st + 1 == kStages);
      return r;
    }
  };
  const uint64_t q_desc = smem_desc_sw128(smem, 16, 1024), k_desc = smem_desc_sw128(smem + kOffRing, 16, 1024),
                 v_desc = smem_desc_sw128(smem + kOffRing, kPanelBytes, 1024);
  auto qk = [&](const Place& at, int half) {  // S_t[half] = Q_t (half of K)^T
    const uint64_t a = q_desc + t * (kTileBytes >> 4), b = k_desc + at.st * (kTileBytes >> 4) + half * (kStep * 128 >> 4);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const uint32_t off = ((ks >> 2) * kPanelBytes + (ks & 3) * 32) >> 4;
      mma_f16_ss(tm + t * kUnit + half * kStep, a + off, b + off, kQk, ks > 0);
    }
  };
  auto pv = [&](const Place& at, int half, bool first) {  // O_t (+)= P_t[half] (half of V)
    const uint64_t b = v_desc + at.st * (kTileBytes >> 4) + half * (kStep * 128 >> 4);
#pragma unroll
    for (int ks = 0; ks < kStep / 16; ++ks)
      mma_f16_ts(tm + 2 * kUnit + t * D, tm + t * kUnit + half * kStep + ks * 8, b + ((ks * 2048) >> 4), kPv,
                 !first || ks > 0);
  };
  auto run = [&]() {  // false: a wait ran out
    Place kp;  // of the next keys
    uint32_t q_par = 0, p_par = 0;
    while (k.next()) {
      const bool mine = t * kTile < k.rows();  // else this warp only hands the stages back
      const int units = k.units;
      auto give_back = [&](uint64_t* bar) {
        if (mine) tc_commit(bar);
        else mbar_arrive(bar);
      };
      if (!wait(&s.q_full, q_par)) return false;
      q_par ^= 1;
      if (!wait(&s.kv_full[kp.st], kp.parity)) return false;
      if (mine) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          qk(kp, half);
          tc_commit(&s.s_full[t][half]);
        }
      }
      give_back(&s.kv_empty[kp.st]);
      if (units == 1) give_back(&s.q_empty);
      for (int j = 0; j < units; ++j) {
        const bool last = j + 1 == units;
        const Place vp = kp.after();
        kp = vp.after();
        if (!wait(&s.kv_full[vp.st], vp.parity)) return false;
        if (!last && !wait(&s.kv_full[kp.st], kp.parity)) return false;
        if (mine) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (!wait(&s.p_full[t][half], p_par)) return false;
            pv(vp, half, j == 0 && half == 0);
            if (!last) qk(kp, half);
            tc_commit(last ? &s.o_full[t][half] : &s.s_full[t][half]);
          }
          p_par ^= 1;
        }
        give_back(&s.kv_empty[vp.st]);
        if (!last) give_back(&s.kv_empty[kp.st]);
        if (j + 2 == units) give_back(&s.q_empty);
      }
    }
    return true;
  };
  run();
  // The softmax warps may have given up: products end before tensor memory goes.
  tc_commit(&s.drain[t]);
  if (!mbar_wait_spin(&s.drain[t], 0)) *p.error = kErrDrainWait;
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
    if (ok && !mbar_wait_spin(bar, parity)) {
      *p.error = kErrFullWait;
      ok = false;
    }
    __syncwarp();
    tc_fence_after();
  };
  uint32_t par = 0;  // of s_full[0], s_full[1] and o_full, a bit each (a register each: 341 us against 327, D = 64)
  int n = 0;  // units of this block so far
  for (int seg = 0; k.next(); ++seg) {
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
    for (int u = 0; u < 2 * k.units; ++u) {
      const int half = u & 1;
      const int j0 = k.u0 * kUnit + u * kStep;
      const uint32_t at = tm_s + half * kStep;
      wait(&s.s_full[tile][half], par >> half & 1);
      par ^= 1 << half;
      uint32_t x[2][32];
      tmem_ld32(at, x[0]);
      tmem_ld32(at + 32, x[1]);
      if constexpr (kScaleQ) {
        if (u == 0) scale *= 1.0f / __uint_as_float((uint32_t)s.q_exp[seg & 1][r] << 23);
      }
      const uint2 there = *reinterpret_cast<const uint2*>(&s.there[(n + (u >> 1)) & 7][2 * half]);
      const bool masked = (there.x & there.y) != 0xffffffffu || j0 + kStep - 1 > first_pos || j0 <= last_low;
      tmem_wait_ld();
      if (__builtin_expect(masked, 0)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int below = row_pos - (j0 + 32 * i) + 1, hidden = low - (j0 + 32 * i) + 1;
          uint32_t mask = i ? there.y : there.x;
          mask &= below >= 32 ? 0xffffffffu : below <= 0 ? 0u : (1u << below) - 1;
          mask &= hidden >= 32 ? 0u : hidden <= 0 ? 0xffffffffu : ~((1u << hidden) - 1);
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (!(mask >> c & 1)) x[i][c] = 0xff800000u;
        }
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 64; c += 2)
        mx[c / 2 % 4] = max3(mx[c / 2 % 4], __uint_as_float(x[c / 32][c % 32]), __uint_as_float(x[c / 32][c % 32 + 1]));
      const float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]) * scale;
      if (u == 0) {
        m = top;
      } else {
        const bool grown = !(top <= m + 8.0f);  // also where top is NaN: the row becomes NaN
        if (__builtin_expect(__any_sync(0xffffffffu, grown), 0)) {
          const float by = grown ? exp2_fast(m - top) : 1.0f;
          if (grown) m = top;
          l *= by;
          // Behind the last step's products comes the other buffer's next phase,
          // or the first of the item's last two.
          if (u + 1 < 2 * k.units) wait(&s.s_full[tile][half ^ 1], par >> (half ^ 1) & 1);
          else wait(&s.o_full[tile][0], par >> 2);
#pragma unroll 1
          for (int i = 0; i < D / 16; ++i) {
            uint32_t o[16];
            tmem_ld16(tm_o + 16 * i, o);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * by);
            tmem_st16(tm_o + 16 * i, o);
          }
        }
      }
      const float neg = m == -INFINITY ? 0.f : -m;
      const uint64_t scale2 = pair2(scale, scale), neg2 = pair2(neg, neg);
      uint64_t sum[2] = {0, 0};
      uint32_t pk[32];
#pragma unroll
      for (int c = 0; c < 64; c += 2) {
        const uint64_t t2 =
            fma2(pair2(__uint_as_float(x[c / 32][c % 32]), __uint_as_float(x[c / 32][c % 32 + 1])), scale2, neg2);
        const float2 t = unpair2(t2);
        const float2 e = make_float2(exp2_fast(t.x), exp2_fast(t.y));
        sum[c / 2 & 1] = add2(sum[c / 2 & 1], pair2(e.x, e.y));
        pk[c / 2] = Act<P16>::pack(e.x, e.y);
      }
      tmem_st32(at, pk);
      const float2 both = unpair2(add2(sum[0], sum[1]));
      l += both.x + both.y;
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&s.p_full[tile][half]);
    }
    n += k.units;
    wait(&s.o_full[tile][1], par >> 2);  // all of the item's products
    par ^= 4;

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
      if (p.a.lse) p.a.lse[t * p.q_heads + h] = mm == -INFINITY ? -INFINITY : (mm + log2f(ll)) / kLog2e;
    };
    if (!k.split()) {
      const bool none = m == -INFINITY;  // nothing seen
      const float inv = none ? 0.f : vs / l;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        uint32_t o[32];
        tmem_ld32(tm_o + 32 * i, o);
        tmem_wait_ld();
        float f[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) f[c] = __uint_as_float(o[c]);
        if (in) write32(32 * i, f, inv);
      }
      if (in) write_lse(m, l);
    } else {
      float* parts = static_cast<float*>(p.parts);
      const int c_first = attn_owner(share, k.origin);
      const int c_last = attn_owner(share, k.origin + (k.it.u_hi - k.it.u_lo) - 1);
      // A block's first segment is its part 0; only the item's first block can
      // have begun before it.
      const int first_part = attn_begin(share, c_first) < k.origin;
      auto part = [&](int c) {
        return parts + ((c * 2 + (c == c_first ? first_part : 0)) * 2 + tile) * (long long)kPartFloats;
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
        const float inv = mm == -INFINITY ? 0.f : vs / ll;
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
__global__ void __launch_bounds__(512, 1) attn_tiles_kernel(const __grid_constant__ AttnTilesParams a) {
  const AttnParams& p = a.p;
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
      mbar_init(&s.kv_empty[i], 2);
    }
    mbar_init(&s.q_full, 128);
    mbar_init(&s.q_empty, 2);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s.s_full[i >> 1][i & 1], 1);
      mbar_init(&s.p_full[i >> 1][i & 1], 128);
      mbar_init(&s.o_full[i >> 1][i & 1], 1);
    }
    mbar_init(&s.drain[0], 1);
    mbar_init(&s.drain[1], 1);
    fence_mbarrier_init();
  }
  if (warp == 12) tmem_alloc(&s.tmem, 512);
  tc_fence_before();
  pdl_wait();
  pdl_launch_dependents();
  const typename K::Work w(p);
  const AttnShare share = attn_share<true>(w, p.least_units, s.share);  // synchronises the block
  tc_fence_after();
  if (warp < 8) {
    K::softmax(p, s, share, warp >> 2);
  } else if (warp < 12) {
    K::load(a.tma, p, s, smem, share);
  } else {
    if (warp < 14 && (threadIdx.x & 31) == 0) K::multiply(p, s, smem, share, warp - 12);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(s.tmem, 512);
}

}  // namespace b2g
