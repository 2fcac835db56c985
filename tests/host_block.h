// host_block.h -- runs the thread blocks of a kernel on the CPU, one block after
// the other: what the kernels' headers call (device.cuh, tc.cuh and the small
// inline-PTX helpers beside them), written for the host.
//
// Every thread of a block is a context of its own and gives up the processor
// where it meets others (mbarriers, named barriers, warp collectives).  Which
// one goes on, when a matrix product or a bulk copy that was issued takes
// place, and how long a warp stands still is drawn from a seed, so that orders
// that a GPU takes once in a million launches come up.  What is checked on the
// way: a phase of an mbarrier gets no more arrivals than it has room for, the
// lanes of a warp meet in the same collective, and no copy or product is still on
// its way when the block has ended.  Waits can be made to run out, too.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <cmath>
#include <algorithm>
#include <deque>
#include <functional>
#include <vector>
#include <ucontext.h>

#include <cuda.h>
#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#undef __shared__
#undef __launch_bounds__
#undef __grid_constant__
#undef __forceinline__
#undef __device__
#undef __host__
#undef __global__
#define __shared__ static
#define __launch_bounds__(...)
#define __grid_constant__
#define __forceinline__ inline
#define __device__
#define __host__
#define __global__

namespace emu {

struct Dim { unsigned x = 0, y = 0, z = 0; };
inline Dim threadIdx_, blockIdx_, blockDim_, gridDim_;

alignas(1024) inline uint8_t smem[256 * 1024];
inline uint32_t tmem[128][512];
inline uint32_t tmem_held = 0;

// ---------------------------------------------------------------------------
inline uint64_t rng_state = 1;
inline unsigned draw(unsigned n) {  // 0 .. n - 1
  rng_state = rng_state * 6364136223846793005ull + 1442695040888963407ull;
  return (unsigned)((rng_state >> 33) % n);
}

inline const char* failure = nullptr;  // the first thing that went wrong
inline void fail(const char* what) {
  if (!failure) failure = what;
}

// An mbarrier in its 64 bits.
struct Bar {
  int32_t tx : 24;
  uint32_t phase : 8;
  uint16_t pending, expected;
};
static_assert(sizeof(Bar) == 8, "an mbarrier's place");

struct Thread {
  ucontext_t ctx;
  bool done = false;
  // What it waits for: a phase of an mbarrier, or to be let go by others.
  Bar* bar = nullptr;
  uint32_t parity = 0;
  bool blocked = false, expired = false;
  long long asleep_until = 0;
  const char* collective = nullptr;
  uint64_t in = 0, out = 0;
  struct Copy { uint32_t dst; const void* src; bool in; };
  std::vector<std::vector<Copy>> groups;  // of 16-byte copies, committed
  std::vector<Copy> open;
  struct Op { std::function<void()> run; bool commit; };
  std::deque<Op> tensor;  // matrix products and commits, in order
};
inline std::vector<Thread> threads;
inline ucontext_t main_ctx;
inline int current = 0;
inline long long now = 0;
inline std::vector<std::function<void()>> bulk;  // bulk copies on their way
struct NamedBar { int count = 0; bool any = false; };
inline NamedBar named[16];
inline int sleepiness = 0;  // one in how many arrivals sends its warp to sleep (0: none)
inline std::function<bool(int)> expire;  // whether this wait of a thread runs out though its phase ends

inline Thread& self() { return threads[current]; }
inline void yield() { swapcontext(&self().ctx, &main_ctx); }

inline void complete(Bar* b) {
  if (b->pending == 0 && b->tx == 0) {
    b->phase ^= 1;
    b->pending = b->expected;
  }
}
inline void arrive(Bar* b) {
  if (b->pending == 0) {
    fail("more arrivals than a phase has room for");
    return;
  }
  --b->pending;
  complete(b);
}
inline bool passed(const Bar* b, uint32_t parity) { return b->phase != (parity & 1); }

// Lanes of a warp meet: each leaves a value, `join` makes everybody's result of
// all 32 when the last one comes.
inline void collective(const char* name, uint64_t value, const std::function<void(Thread*)>& join) {
  Thread& t = self();
  Thread* warp = &threads[current / 32 * 32];
  t.collective = name;
  t.in = value;
  int here = 0;
  for (int i = 0; i < 32; ++i) here += warp[i].collective && strcmp(warp[i].collective, name) == 0;
  if (here == 32) {
    join(warp);
    for (int i = 0; i < 32; ++i) warp[i].collective = nullptr, warp[i].blocked = false;
    return;
  }
  t.blocked = true;
  yield();
}
inline uint64_t exchange(const char* name, uint64_t v, int from) {
  const int lane = current % 32;
  collective(name, v, [](Thread* w) {
    for (int i = 0; i < 32; ++i) w[i].out = w[i].in;
  });
  return threads[current / 32 * 32 + (from >= 0 && from < 32 ? from : lane)].out;
}
inline uint32_t ballot(const char* name, bool v) {
  collective(name, v, [](Thread* w) {
    uint32_t m = 0;
    for (int i = 0; i < 32; ++i) m |= (uint32_t)(w[i].in & 1) << i;
    for (int i = 0; i < 32; ++i) w[i].out = m;
  });
  return (uint32_t)self().out;
}
inline bool barrier(int id, int n, bool v = false) {
  NamedBar& b = named[id];
  b.any |= v;
  if (++b.count == n) {
    for (Thread& t : threads)
      if (t.blocked && t.collective == nullptr && t.parity == 1000u + id) t.blocked = false, t.out = b.any;
    const bool any = b.any;
    b = NamedBar();
    return any;
  }
  self().parity = 1000u + id;
  self().blocked = true;
  yield();
  return self().out != 0;
}

inline void copy16(const Thread::Copy& c) {
  if (c.in) memcpy(smem + c.dst, c.src, 16);
  else memset(smem + c.dst, 0, 16);
}

// The block's threads run `body`; what is issued to the tensor cores and the
// copy engine takes place in between.
inline void run_block(int n_threads, const std::function<void()>& body) {
  static std::function<void()> fn;
  fn = body;
  threads.clear();
  threads.resize(n_threads);
  constexpr size_t kStack = 192 * 1024;
  static std::vector<std::vector<uint8_t>> stacks;
  while ((int)stacks.size() < n_threads) stacks.emplace_back(kStack);
  bulk.clear();
  for (NamedBar& b : named) b = NamedBar();
  for (uint32_t(&lane)[512] : tmem)
    for (uint32_t& v : lane) v = 0x7fc00000u;  // NaN
  memset(smem, 0xff, sizeof smem);
  blockDim_.x = n_threads;
  for (int i = 0; i < n_threads; ++i) {
    Thread& t = threads[i];
    getcontext(&t.ctx);
    t.ctx.uc_stack.ss_sp = stacks[i].data();
    t.ctx.uc_stack.ss_size = kStack;
    t.ctx.uc_link = &main_ctx;
    makecontext(&t.ctx, (void (*)())(+[] {
                  fn();
                  threads[current].done = true;
                }), 0);
  }
  std::vector<int> ready;
  for (now = 0; !failure; ++now) {
    // Hardware: the front of an issuer's queue, or any bulk copy.
    std::vector<int> issuers;
    for (int i = 0; i < n_threads; ++i)
      if (!threads[i].tensor.empty()) issuers.push_back(i);
    const unsigned units = issuers.size() + (bulk.empty() ? 0 : 1);
    ready.clear();
    bool asleep = false, live = false;
    for (int i = 0; i < n_threads; ++i) {
      Thread& t = threads[i];
      if (t.done) continue;
      live = true;
      if (t.blocked) continue;
      if (t.bar && !t.expired && !passed(t.bar, t.parity)) continue;
      if (t.asleep_until > now) {
        asleep = true;
        continue;
      }
      ready.push_back(i);
    }
    if (!live) break;
    if (units && (ready.empty() || draw(4) == 0)) {
      const unsigned pick = draw(units);
      if (pick < issuers.size()) {
        auto& q = threads[issuers[pick]].tensor;
        auto op = std::move(q.front());
        q.pop_front();
        op.run();
      } else {
        const unsigned i = draw(bulk.size());
        auto op = std::move(bulk[i]);
        bulk.erase(bulk.begin() + i);
        op();
      }
      continue;
    }
    if (ready.empty()) {
      if (asleep) {  // all others wait for the sleepers
        for (Thread& t : threads) t.asleep_until = 0;
        continue;
      }
      bool any = false;  // waits with a limit run out, all others wait for good
      for (Thread& t : threads)
        if (!t.done && !t.blocked && t.bar) t.expired = any = true;
      if (!any) fail("hang: threads wait for others that never come");
      continue;
    }
    // A warp's ready lanes go one after the other.
    const int first = ready[draw(ready.size())] / 32;
    for (int i : ready) {
      if (i / 32 != first || threads[i].asleep_until > now) continue;
      current = i;
      threadIdx_.x = i;
      swapcontext(&main_ctx, &threads[i].ctx);
    }
  }
  if (!bulk.empty()) fail("bulk copies on their way when the block ended");
  for (Thread& t : threads) {
    for (auto& op : t.tensor)
      if (!op.commit) fail("products on their way when the block ended");
    for (auto& g : t.groups)
      if (!g.empty()) fail("copies on their way when the block ended");
  }
  if (tmem_held) fail("tensor memory held when the block ended");
}

}  // namespace emu

static emu::Dim &threadIdx = emu::threadIdx_, &blockIdx = emu::blockIdx_, &blockDim = emu::blockDim_,
                &gridDim = emu::gridDim_;

// ---------------------------------------------------------------------------
// CUDA's own names
// ---------------------------------------------------------------------------
template <typename A, typename B>
constexpr typename std::common_type<A, B>::type min(A a, B b) {
  using C = typename std::common_type<A, B>::type;
  return (C)a < (C)b ? (C)a : (C)b;
}
template <typename A, typename B>
constexpr typename std::common_type<A, B>::type max(A a, B b) {
  using C = typename std::common_type<A, B>::type;
  return (C)a > (C)b ? (C)a : (C)b;
}
inline uint32_t __float_as_uint(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }
inline float __uint_as_float(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
inline uint32_t __byte_perm(uint32_t, uint32_t, uint32_t) { abort(); }
inline int __popc(uint32_t v) { return __builtin_popcount(v); }
inline float rsqrtf(float v) { return 1 / sqrtf(v); }
inline float __expf(float v) { return expf(v); }
inline float __fdividef(float a, float b) { return b > 0x1p126f && b < INFINITY ? a * 0.f : a / b; }
template <typename T> inline T __ldcg(const T* p) { return *p; }
template <typename T> inline void __stcg(T* p, T v) { *p = v; }
inline void __threadfence() {}
inline int atomicAdd(int* p, int v) { const int old = *p; *p += v; return old; }
inline void __syncthreads() { emu::barrier(0, blockDim.x); }
inline int __syncthreads_or(int v) { return emu::barrier(0, blockDim.x, v != 0); }
inline void __syncwarp(uint32_t = 0xffffffffu) { emu::collective("__syncwarp", 0, [](emu::Thread*) {}); }
template <typename T>
inline T emu_shfl(const char* name, T v, int from) {
  uint64_t u = 0;
  memcpy(&u, &v, sizeof v);
  u = emu::exchange(name, u, from);
  memcpy(&v, &u, sizeof v);
  return v;
}
template <typename T> inline T __shfl_sync(uint32_t, T v, int lane) { return emu_shfl("__shfl_sync", v, lane); }
template <typename T> inline T __shfl_xor_sync(uint32_t, T v, int m) { return emu_shfl("__shfl_xor_sync", v, (emu::current % 32) ^ m); }
template <typename T> inline T __shfl_up_sync(uint32_t, T v, int d) { return emu_shfl("__shfl_up_sync", v, emu::current % 32 - d); }
inline uint32_t __ballot_sync(uint32_t, bool v) { return emu::ballot("__ballot_sync", v); }
inline bool __any_sync(uint32_t, bool v) { return emu::ballot("__any_sync", v) != 0; }
inline bool __all_sync(uint32_t, bool v) { return emu::ballot("__all_sync", v) == 0xffffffffu; }

namespace b2g {

// ---------------------------------------------------------------------------
// device.cuh
// ---------------------------------------------------------------------------
enum : int { kErrNone = 0, kErrFullWait = 1, kErrEmptyWait = 2, kErrDrainWait = 3, kErrPeerWait = 4, kErrGridWait = 5 };

inline uint32_t smem_addr(const void* p) { return (uint32_t)(static_cast<const uint8_t*>(p) - emu::smem); }
inline emu::Bar* bar_of(uint64_t* b) { return reinterpret_cast<emu::Bar*>(b); }
inline void mbar_init(uint64_t* b, uint32_t count) { *bar_of(b) = {0, 0, (uint16_t)count, (uint16_t)count}; }
inline void fence_mbarrier_init() {}
inline void mbar_arrive(uint64_t* b) {
  emu::arrive(bar_of(b));
  // A warp may stand still behind any arrival.
  if (emu::sleepiness && emu::draw(emu::sleepiness) == 0)
    for (int i = 0; i < 32; ++i) emu::threads[emu::current / 32 * 32 + i].asleep_until = emu::now + emu::draw(4000);
  emu::yield();
}
inline void mbar_arrive_expect_tx(uint64_t* b, uint32_t bytes) {
  bar_of(b)->tx += bytes;
  emu::arrive(bar_of(b));
}
inline bool mbar_test(uint64_t* b, uint32_t parity) { return emu::passed(bar_of(b), parity); }
inline bool mbar_wait_spin(uint64_t* b, uint32_t parity) {
  emu::Thread& t = emu::self();
  if (emu::expire && emu::expire(emu::current)) return false;
  t.bar = bar_of(b);
  t.parity = parity & 1;
  t.expired = false;
  do emu::yield();
  while (!t.expired && !emu::passed(bar_of(b), parity));
  t.bar = nullptr;
  return !t.expired;
}
inline bool mbar_wait_bounded(uint64_t* b, uint32_t parity) { return mbar_wait_spin(b, parity); }
inline void pdl_wait() {}
inline void pdl_launch_dependents() {}
inline void named_sync(int id, int n) { emu::barrier(id, n); }
inline int atom_add_acq_rel_gpu(int* p, int v) { return atomicAdd(p, v); }
inline void e4m3x4_to_f16x2x2(uint32_t w, uint32_t& lo, uint32_t& hi) {
  uint32_t h[4];
  for (int i = 0; i < 4; ++i) h[i] = __half_raw(__nv_cvt_fp8_to_halfraw((uint8_t)(w >> 8 * i), __NV_E4M3)).x;
  lo = h[0] | h[1] << 16;
  hi = h[2] | h[3] << 16;
}
inline void mma_16816(float (&)[4], uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) { abort(); }
inline uint4 lds128_at(uint32_t a) { uint4 v; memcpy(&v, emu::smem + a, 16); return v; }
inline void sts128_at(uint32_t a, uint4 v) { memcpy(emu::smem + a, &v, 16); }

// ---------------------------------------------------------------------------
// tc.cuh
// ---------------------------------------------------------------------------
inline void tmem_alloc(uint32_t* out, uint32_t cols) {
  emu::collective("tmem_alloc", 0, [](emu::Thread*) {});
  emu::tmem_held = cols;
  *out = 0;
}
inline void tmem_dealloc(uint32_t, uint32_t) {
  emu::collective("tmem_dealloc", 0, [](emu::Thread*) {});
  emu::tmem_held = 0;
}
inline void tc_fence_after() {}
inline void tc_fence_before() {}
inline void tmem_wait_ld() { emu::collective("tmem_wait_ld", 0, [](emu::Thread*) {}); }
inline void tmem_wait_st() { emu::collective("tmem_wait_st", 0, [](emu::Thread*) {}); }
template <int N>
inline void tmem_load(uint32_t addr, uint32_t (&r)[N]) {
  emu::collective("tmem_ld", 0, [](emu::Thread*) {});
  const int lane = (addr >> 16) + emu::current % 32;
  if ((int)(addr >> 16) != emu::current / 32 % 4 * 32) return emu::fail("tensor memory of another warp's lanes");
  for (int i = 0; i < N; ++i) r[i] = emu::tmem[lane][(addr & 0xffff) + i];
}
template <int N>
inline void tmem_store(uint32_t addr, const uint32_t (&r)[N]) {
  emu::collective("tmem_st", 0, [](emu::Thread*) {});
  const int lane = (addr >> 16) + emu::current % 32;
  for (int i = 0; i < N; ++i) emu::tmem[lane][(addr & 0xffff) + i] = r[i];
}
inline void tmem_ld32(uint32_t a, uint32_t (&r)[32]) { tmem_load(a, r); }
inline void tmem_ld16(uint32_t a, uint32_t (&r)[16]) { tmem_load(a, r); }
inline void tmem_st32(uint32_t a, const uint32_t (&r)[32]) { tmem_store(a, r); }
inline void tmem_st16(uint32_t a, const uint32_t (&r)[16]) { tmem_store(a, r); }

inline uint64_t smem_desc_sw128(uint32_t addr, uint32_t lead_bytes, uint32_t stride_bytes) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)((lead_bytes >> 4) & 0x3FFF) << 16 |
         (uint64_t)((stride_bytes >> 4) & 0x3FFF) << 32 | 1ull << 46 | 2ull << 61;
}
constexpr uint32_t tc_idesc(int d_format, int a_format, int b_format, int b_mn_major, int n) {
  return (uint32_t)d_format << 4 | (uint32_t)a_format << 7 | (uint32_t)b_format << 10 | (uint32_t)b_mn_major << 16 |
         (uint32_t)(n >> 3) << 17 | (uint32_t)(128 >> 4) << 24;
}
// Byte `k` of row `r`, rows of 128 bytes along K; the swizzle goes by the address.
inline const uint8_t* k_major(uint64_t d, int r, int k) {
  const uint32_t a = (uint32_t)(d & 0x3FFF) * 16 + r / 8 * ((uint32_t)(d >> 32 & 0x3FFF) * 16) + r % 8 * 128 + k;
  return emu::smem + (a ^ (a >> 7 & 7) << 4);
}
// Element (k, n) of 16 bits, rows of 64 of them along N.
inline const uint8_t* mn_major(uint64_t d, int k, int n) {
  const uint32_t a = (uint32_t)(d & 0x3FFF) * 16 + k / 8 * ((uint32_t)(d >> 32 & 0x3FFF) * 16) + k % 8 * 128 +
                     n / 64 * ((uint32_t)(d >> 16 & 0x3FFF) * 16) + n % 64 * 2;
  return emu::smem + (a ^ (a >> 7 & 7) << 4);
}
inline float f16_value(uint16_t v, bool bf16) {
  if (bf16) return __uint_as_float((uint32_t)v << 16);
  __half_raw h;
  h.x = v;
  return __half2float(__half(h));
}
inline void issue(std::function<void()> f, bool commit = false) {
  emu::self().tensor.push_back({std::move(f), commit});
}
inline void f16_product(uint32_t d, const float* a, uint64_t b, uint32_t idesc, bool accumulate) {
  const int n = (idesc >> 17 & 63) * 8;
  const bool bf16 = idesc >> 10 & 7, mn = idesc >> 16 & 1;
  std::vector<float> bv(n * 16);
  for (int j = 0; j < n; ++j)
    for (int k = 0; k < 16; ++k) {
      uint16_t v;
      memcpy(&v, mn ? mn_major(b, k, j) : k_major(b, j, 2 * k), 2);
      bv[j * 16 + k] = f16_value(v, bf16);
    }
  for (int i = 0; i < 128; ++i)
    for (int j = 0; j < n; ++j) {
      float s = accumulate ? __uint_as_float(emu::tmem[i][d + j]) : 0.f;
      for (int k = 0; k < 16; ++k) s += a[i * 16 + k] * bv[j * 16 + k];
      emu::tmem[i][d + j] = __float_as_uint(s);
    }
}
inline void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  issue([=] {
    float av[128 * 16];
    for (int i = 0; i < 128; ++i)
      for (int k = 0; k < 16; ++k) {
        uint16_t v;
        memcpy(&v, k_major(a, i, 2 * k), 2);
        av[i * 16 + k] = f16_value(v, idesc >> 7 & 7);
      }
    f16_product(d, av, b, idesc, accumulate);
  });
}
inline void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  issue([=] {
    float av[128 * 16];
    for (int i = 0; i < 128; ++i)
      for (int k = 0; k < 16; ++k)
        av[i * 16 + k] = f16_value((uint16_t)(emu::tmem[i][a + k / 2] >> 16 * (k & 1)), idesc >> 7 & 7);
    f16_product(d, av, b, idesc, accumulate);
  });
}
inline void mma_i8_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  issue([=] {
    const int n = (idesc >> 17 & 63) * 8;
    std::vector<int> bv(n * 32);
    for (int j = 0; j < n; ++j)
      for (int k = 0; k < 32; ++k) bv[j * 32 + k] = (int8_t)*k_major(b, j, k);
    for (int i = 0; i < 128; ++i) {
      int av[32];
      for (int k = 0; k < 32; ++k) av[k] = (int8_t)*k_major(a, i, k);
      for (int j = 0; j < n; ++j) {
        int s = accumulate ? (int)emu::tmem[i][d + j] : 0;
        for (int k = 0; k < 32; ++k) s += av[k] * bv[j * 32 + k];
        emu::tmem[i][d + j] = (uint32_t)s;
      }
    }
  });
}
inline void tc_commit(uint64_t* b) {
  issue([=] { emu::arrive(bar_of(b)); }, true);
}
inline void fence_proxy_async_shared() {}

// A tensor map as the copies here read it.
struct HostMap {
  const uint8_t* base;
  int rank, size, dims[4], box[4];
  long long strides[4];  // bytes
};
static_assert(sizeof(HostMap) <= sizeof(CUtensorMap), "a tensor map's place");
// A box of 128-byte rows, swizzled, zeros outside.
inline void tma_load(uint32_t dst, const CUtensorMap* map, std::vector<int> at, uint64_t* bar) {
  HostMap m;
  memcpy(&m, map, sizeof m);
  if (at[0] * m.size % 16) emu::fail("a bulk copy off 16 bytes");
  emu::bulk.push_back([=] {
    const int row_bytes = m.box[0] * m.size;
    int rows = 1;
    for (int i = 1; i < m.rank; ++i) rows *= m.box[i];
    for (int r = 0; r < rows; ++r)
      for (int x = 0; x < m.box[0]; ++x) {
        bool in = at[0] + x >= 0 && at[0] + x < m.dims[0];
        long long off = (long long)(at[0] + x) * m.size;
        for (int i = 1, rest = r; i < m.rank; rest /= m.box[i], ++i) {
          const int c = at[i] + rest % m.box[i];
          in = in && c >= 0 && c < m.dims[i];
          off += c * m.strides[i];
        }
        uint32_t a = dst + r * row_bytes + x * m.size;
        a ^= (a >> 7 & 7) << 4;
        if (in) memcpy(emu::smem + a, m.base + off, m.size);
        else memset(emu::smem + a, 0, m.size);
      }
    emu::Bar* b = bar_of(bar);
    b->tx -= rows * row_bytes;
    emu::complete(b);
  });
}
inline void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  tma_load(smem_addr(dst), map, {x, y}, bar);
}
inline void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  tma_load(dst, map, {x, y, z, w}, bar);
}
inline void tma_prefetch_desc(const CUtensorMap*) {}

// ---------------------------------------------------------------------------
// serve.cuh, attn_rows.cuh, attn_tiles.cuh
// ---------------------------------------------------------------------------
inline void cluster_sync() { abort(); }  // blocks run one after the other
inline uint32_t cluster_map(uint32_t, uint32_t) { abort(); }
inline int ld_cluster(uint32_t) { abort(); }

inline float exp2_fast(float x) { return x < -126.f ? 0.f : exp2f(x); }
template <bool BF16>
inline void mma_act(float (&)[4], const uint32_t (&)[4], uint32_t, uint32_t) { abort(); }
inline void ldsm4(uint32_t (&)[4], uint32_t) { abort(); }
inline void ldsm4_t(uint32_t (&)[4], uint32_t) { abort(); }
inline void cp_async16_or_zero(uint32_t dst, const void* src, bool in) { emu::self().open.push_back({dst, src, in}); }
inline void cp_async_commit() {
  emu::Thread& t = emu::self();
  if (emu::draw(2)) {  // landed at once, or when it is waited for
    for (const auto& c : t.open) emu::copy16(c);
    t.open.clear();
  }
  t.groups.push_back(std::move(t.open));
  t.open.clear();
}
template <int N>
inline void cp_async_wait() {
  emu::Thread& t = emu::self();
  while (t.groups.size() > N) {
    for (const auto& c : t.groups.front()) emu::copy16(c);
    t.groups.erase(t.groups.begin());
  }
}
inline float max3(float a, float b, float c) {
  if (a != a || b != b || c != c) return NAN;
  return fmaxf(fmaxf(a, b), c);
}
inline uint64_t pair2(float a, float b) { return __float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32; }
inline float2 unpair2(uint64_t v) { return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))); }
inline uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  const float2 x = unpair2(a), y = unpair2(b), z = unpair2(c);
  return pair2(fmaf(x.x, y.x, z.x), fmaf(x.y, y.y, z.y));
}
inline uint64_t add2(uint64_t a, uint64_t b) {
  const float2 x = unpair2(a), y = unpair2(b);
  return pair2(x.x + y.x, x.y + y.y);
}

}  // namespace b2g
