"""The prompt attention's kernel, block by block on the CPU (host_block.h), in
orders of its warps, products and copies that are drawn: its hand-overs may not
lean on one side being quick."""
from __future__ import annotations

import subprocess

import pytest

from host_block import compile_blocks

PROGRAM = r"""
#include "attn_tiles.cuh"
using namespace b2g;

static float uniform() { return (float)emu::draw(2001) / 1000 - 1; }
template <typename T> T to16(float v);
template <> __half to16(float v) { return __float2half_rn(v); }
template <> __nv_bfloat16 to16(float v) { return __float2bfloat16_rn(v); }
static double value(__half v) { return __half2float(v); }
static double value(__nv_bfloat16 v) { return __bfloat162float(v); }
static double value(uint8_t v) { return __half2float(__half(__half_raw(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3)))); }

// first .. last: threads whose `late`th wait runs out (none: first < 0).
static int first = -1, last = -1, late = 0;

template <typename T, bool FP8, int D>
int run(std::vector<int> fresh, std::vector<int> total, int kv_heads, int group, int page, int grid, int least) {
  using K = TilesKernel<T, FP8, D>;
  using C = typename std::conditional<FP8, uint8_t, T>::type;
  const int batch = fresh.size(), heads = kv_heads * group;
  std::vector<int> start(1, 0), table;
  int max_pages = 1, pages = 0;
  for (int t : total) max_pages = std::max(max_pages, (t + page - 1) / page);
  for (int b = 0; b < batch; ++b) {
    start.push_back(start[b] + fresh[b]);
    for (int i = 0; i < max_pages; ++i) table.push_back(i * page < total[b] ? pages++ : -1);
  }
  const int rows = start[batch];
  std::vector<T> q(rows * heads * D), out(q.size(), to16<T>(7));
  std::vector<C> kc(pages * page * kv_heads * D), vc(kc.size());
  for (int r = 0; r < rows; ++r)  // rows and heads at norms that differ by powers of two
    for (int h = 0; h < heads; ++h)
      for (int d = 0; d < D; ++d)
        q[(r * heads + h) * D + d] = to16<T>(ldexpf(uniform(), (r / 16 + h) % 4));
  for (auto* c : {&kc, &vc})
    for (C& x : *c) {
      if constexpr (FP8) x = (uint8_t)(emu::draw(2) * 128 + emu::draw(0x41));
      else x = to16<T>(uniform());
    }
  AttnTilesParams a = {};
  AttnParams& p = a.p;
  int error = 0;
  std::vector<int> counters(3 * grid);
  std::vector<float> parts(grid * 4 * K::kPartFloats, NAN), lse(rows * heads, 7.f);
  p.a.q = q.data(), p.a.stride_q = heads * D, p.a.stride_q_head = D;
  p.a.out = out.data(), p.a.stride_o = heads * D, p.a.stride_o_head = D;
  p.a.lse = lse.data(), p.a.scale = 1 / sqrtf(D);
  p.c.k = kc.data(), p.c.v = vc.data();
  p.c.stride_page = page * kv_heads * D, p.c.stride_token = kv_heads * D, p.c.stride_head = D;
  p.c.num_pages = pages, p.c.page_size = page, p.c.kv_heads = kv_heads, p.c.head_dim = D;
  p.b.batch = batch, p.b.rows = rows, p.b.max_q = rows, p.b.max_pages = max_pages, p.b.page_table_stride = max_pages;
  p.b.q_start = start.data(), p.b.seq_lens = total.data(), p.b.page_table = table.data();
  p.q_heads = heads, p.group = group, p.least_units = least, p.page_shift = -1;
  p.error = &error, p.counters = counters.data(), p.parts = parts.data();
  if (!FP8 && page % 8 == 0 && 128 % page == 0) {
    a.tma.box_rows = page;
    for (int i = 0; i < 2; ++i) {
      HostMap m = {(const uint8_t*)(i ? p.c.v : p.c.k), 4, 2, {D, page, kv_heads, pages}, {64, page, 1, 1},
                   {2, p.c.stride_token * 2, D * 2, p.c.stride_page * 2}};
      memcpy(i ? &a.tma.v : &a.tma.k, &m, sizeof m);
    }
  }
  emu::gridDim_.x = grid;
  for (int c = 0; c < grid; ++c) {
    emu::blockIdx_.x = c;
    std::vector<int> waits(K::kThreads);
    emu::expire = nullptr;
    if (first >= 0) emu::expire = [&](int i) { return i >= first && i <= last && ++waits[i] == late; };
    emu::run_block(K::kThreads, [&] { attn_tiles_kernel<T, FP8, D>(a); });
    if (emu::failure) return printf("block %d: %s\n", c, emu::failure), 1;
  }
  if (first >= 0) return error ? 0 : (printf("no error is set\n"), 1);
  if (error) return printf("error word %d\n", error), 1;
  for (int c : counters)
    if (c) return printf("counters are left dirty\n"), 1;
  // Probabilities are rounded once (2^-8 or 2^-11 of each), the result again; scores and sums in fp32.
  const double u = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 0x1p-8 : 0x1p-11;
  for (int b = 0; b < batch; ++b)
    for (int i = 0; i < fresh[b]; ++i)
      for (int h = 0; h < heads; ++h) {
        const int r = start[b] + i, pos = total[b] - fresh[b] + i;
        const T* qr = &q[(r * heads + h) * D];
        std::vector<double> s(pos + 1), o(D), mag(D);
        auto at = [&](int j) {
          return ((long long)table[b * max_pages + j / page] * page + j % page) * kv_heads * D + h / group * D;
        };
        double top = -INFINITY, sum = 0;
        for (int j = 0; j <= pos; ++j) {
          for (int d = 0; d < D; ++d) s[j] += value(qr[d]) * value(kc[at(j) + d]);
          top = std::max(top, s[j] *= p.a.scale);
        }
        for (int j = 0; j <= pos; ++j) sum += s[j] = exp(s[j] - top);
        for (int j = 0; j <= pos; ++j)
          for (int d = 0; d < D; ++d) {
            const double x = s[j] / sum * value(vc[at(j) + d]);
            o[d] += x, mag[d] += fabs(x);
          }
        for (int d = 0; d < D; ++d) {
          const double got = value(out[(r * heads + h) * D + d]);
          if (!(fabs(got - o[d]) <= 1.02 * u * mag[d] + u * fabs(o[d]) + 1e-4))
            return printf("sequence %d token %d head %d element %d: %g, %g expected\n", b, i, h, d, got, o[d]), 1;
        }
        if (!(fabs(lse[r * heads + h] - (top + log(sum))) <= 1e-4)) return printf("log-sum of row %d: %g, %g expected\n", r, lse[r * heads + h], top + log(sum)), 1;
      }
  return 0;
}

int main(int argc, char** argv) {
  const int type = atoi(argv[1]), batch = atoi(argv[2]), sleepy = atoi(argv[3]);
  for (int seed = 1; seed <= atoi(argv[4]); ++seed) {
    emu::rng_state = seed;
    emu::sleepiness = sleepy;
    if (argc > 5) first = atoi(argv[5]), last = atoi(argv[6]), late = 1 + (seed - 1) % atoi(argv[7]);
    std::vector<int> fresh, total;
    int least = 1, grid = 2;
    if (batch == 0) {  // short prompts: several items of one unit a block
      fresh = {100, 23, 128, 61};
      total = fresh;
    } else {  // a long sequence ahead of short ones: an item that two blocks share, then short ones
      fresh = {140, 30, 75, 9};
      total = {400, 30, 75, 120};
      least = 4;
    }
    const int bad = type == 0   ? run<__nv_bfloat16, true, 64>(fresh, total, 2, 2, 16, grid, least)
                    : type == 1 ? run<__nv_bfloat16, false, 64>(fresh, total, 2, 2, 16, grid, least)
                    : type == 2 ? run<__half, true, 64>(fresh, total, 2, 2, 24, grid, least)
                                : run<__half, false, 128>(fresh, total, 2, 2, 24, grid, least);
    if (bad) return printf("seed %d\n", seed), 1;
  }
  puts("ok");
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    return compile_blocks(tmp_path_factory.mktemp("blocks"), PROGRAM)


TYPES = ["bf16 over e4m3", "bf16", "fp16 over e4m3", "fp16"]
BATCHES = ["short prompts", "a long one ahead"]


def run(program, types, batch, sleepiness, seeds, *expire):
    args = [TYPES.index(types), BATCHES.index(batch), sleepiness, seeds, *expire]
    out = subprocess.run([str(program), *map(str, args)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout + out.stderr


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("types", TYPES[1:])
def test_warps_in_even_turns(program, types, batch):
    run(program, types, batch, 0, 2)


def test_scales_of_rows_outlive_the_next_loads(program):
    """bf16 rows over an 8-bit cache, each in a range of its own: a block that
    takes several items of one unit keeps an item's scales until its softmax has
    read them, however far the loads and products are ahead."""
    run(program, TYPES[0], BATCHES[0], 0, 5)


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("types", TYPES)
def test_warps_that_stand_still(program, types, batch):
    """One arrival in 3000 sends its warp to sleep for up to 4000 turns: no phase
    of a barrier may pass before all who wait for it have seen it."""
    run(program, types, batch, 3000, 10)


@pytest.mark.parametrize("threads", [(0, 31), (5, 5), (128, 255), (256, 383), (256, 256), (300, 300), (384, 384), (416, 416)],
                         ids=["a softmax warp", "a softmax lane", "a tile's softmax", "the loads", "the first load lane",
                              "another load lane", "products of tile 0", "products of tile 1"])
@pytest.mark.parametrize("types", TYPES)
def test_waits_that_run_out(program, types, threads):
    """Whichever wait of these threads runs out: the block ends, with an error
    set, and no copy or product is on its way behind it."""
    run(program, types, BATCHES[1], 0, 6, *threads, 6)
