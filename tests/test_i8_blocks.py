"""The 8-bit product's kernel, block by block on the CPU (host_block.h): its
three ways to cut the work (a cluster's blocks run at the same time, so not that
one), orders of warps, products and copies that are drawn, and waits that run
out."""
from __future__ import annotations

import subprocess

import pytest

from host_block import compile_blocks

PROGRAM = r"""
#include "i8.cu"
using namespace b2g;

static int first = -1, last = -1, late = 0;  // threads whose `late`th wait runs out
static int div_up(int a, int b) { return (a + b - 1) / b; }
static void map(CUtensorMap* to, const std::vector<int8_t>& v, int rows, int k, int ld, int box) {
  HostMap m = {(const uint8_t*)v.data(), 2, 1, {k, rows}, {kKBlock, box}, {1, ld}};
  memcpy(to, &m, sizeof m);
}

template <int PLANES, bool GATE, bool DEEP>
int run(int m, int n, int k, int bn, int grid, bool whole, bool residual) {
  using T = __half;
  const int planes = GATE ? 2 : 1, ld = (k + 15) / 16 * 16, wide = DEEP && !GATE ? 2 : 1;
  std::vector<int8_t> x(m * ld), w(planes * n * ld);
  for (auto* v : {&x, &w})
    for (int8_t& c : *v) c = (int8_t)(emu::draw(255) - 127);
  std::vector<float> sx(m), sw(planes * n);
  for (auto* v : {&sx, &sw})
    for (float& s : *v) s = (1 + emu::draw(100)) / 3000.f;
  std::vector<T> y(m * n), res(m * n);
  for (T& r : res) r = __float2half_rn(emu::draw(100) / 50.f - 1);
  int error = 0;
  I8Tc t = {};
  t.p = {x.data(), ld, sx.data(), w.data(), ld, sw.data(), residual ? res.data() : nullptr, n, y.data(), n, m, n, k, planes, 0};
  t.bn = bn;
  t.tok_tiles = div_up(m, bn);
  t.tiles = t.tok_tiles * div_up(n, wide * kChTile);
  const int stage_tiles = DEEP ? 2 : planes, stage = (stage_tiles * kChTile + bn) * kKBlock;
  t.stages = std::min(3, (kI8SmemBytes - 1024) / stage);
  t.kb = div_up(k, kKBlock);
  t.whole = whole;
  t.cluster = 1;
  t.acc_cols = DEEP ? 256 : bn;
  t.tmem_cols = 512;
  t.units = (long long)t.tiles * t.kb;
  t.slot_ints = (long long)planes * bn * kChTile;
  std::vector<int> counters(grid), partials(grid * t.slot_ints);
  t.counters = counters.data(), t.partials = partials.data(), t.error = &error;
  map(&t.mw, w, planes * n, k, ld, kChTile);
  map(&t.mx, x, m, k, ld, bn);
  bool expired = false;
  emu::gridDim_.x = grid;
  for (int c = 0; c < grid; ++c) {
    emu::blockIdx_.x = c;
    std::vector<int> waits(320);
    emu::expire = nullptr;
    if (first >= 0)
      emu::expire = [&](int i) { return i >= first && i <= last && ++waits[i] == late && (expired = true); };
    emu::run_block(DEEP ? 320 : 192, [&] { i8_product_kernel<T, PLANES, GATE, DEEP>(t); });
    if (emu::failure) return printf("block %d: %s\n", c, emu::failure), 1;
  }
  if (expired) return error ? 0 : (printf("no error is set\n"), 1);
  if (error) return printf("error word %d\n", error), 1;
  for (auto* v : {&counters, &partials})
    for (int c : *v)
      if (c) return printf("the workspace is left dirty\n"), 1;
  for (int i = 0; i < m; ++i)
    for (int j = 0; j < n; ++j) {
      double v[2] = {0, 0};
      for (int pl = 0; pl < planes; ++pl) {
        for (int e = 0; e < k; ++e) v[pl] += x[i * ld + e] * w[(pl * n + j) * ld + e];
        v[pl] *= (double)sx[i] * sw[pl * n + j];
      }
      double want = GATE ? v[0] / (1 + exp(-v[0])) * v[1] : v[0];
      if (residual) want += __half2float(res[i * n + j]);
      const double got = __half2float(y[i * n + j]);
      // One rounding to fp16, and fp32's: (|g| + 8) 2^-22 for SiLU, three half steps else.
      if (!(fabs(got - want) <= (0x1p-11 + (fabs(v[0]) + 8) * 0x1p-22) * fabs(want) + 0x1p-20))
        return printf("row %d channel %d: %g, %g expected\n", i, j, got, want), 1;
    }
  return 0;
}

int main(int argc, char** argv) {
  const int cut = atoi(argv[1]);
  for (int seed = 1; seed <= atoi(argv[3]); ++seed) {
    emu::rng_state = seed;
    emu::sleepiness = atoi(argv[2]);
    if (argc > 4) first = atoi(argv[4]), last = atoi(argv[5]), late = 1 + (seed - 1) % atoi(argv[6]);
    const int bad = cut == 0   ? run<1, false, false>(90, 300, 450, 32, 2, true, true)
                    : cut == 1 ? run<2, true, false>(70, 200, 300, 32, 3, true, false)
                    : cut == 2 ? run<1, false, false>(40, 200, 900, 64, 3, false, true)
                    : cut == 3 ? run<2, true, false>(33, 150, 700, 64, 3, false, false)
                    : cut == 4 ? run<2, false, true>(150, 300, 300, 80, 2, true, true)
                               : run<2, true, true>(100, 200, 300, 64, 2, true, false);
    if (bad) return printf("seed %d\n", seed), 1;
  }
  puts("ok");
}
"""

CUTS = ["whole tiles", "whole tiles, gate||up", "shared ranges", "shared ranges, gate||up", "deep tiles",
        "deep tiles, gate||up"]


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    def change(name, text):  # the kernels without their launches
        if name != "i8.cu":
            return text
        return text[:text.index("// Rows of bytes, 128 columns by box_rows a load")] + "}\n}\n"
    return compile_blocks(tmp_path_factory.mktemp("blocks"), PROGRAM, ["i8.cu"], change)


def run(program, cut, *args):
    out = subprocess.run([str(program), str(CUTS.index(cut)), *map(str, args)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout + out.stderr


@pytest.mark.parametrize("sleepiness", [0, 200])
@pytest.mark.parametrize("cut", CUTS)
def test_products(program, cut, sleepiness):
    run(program, cut, sleepiness, 3)


@pytest.mark.parametrize("threads", [(0, 0), (32, 32), (64, 95), (64, 64), (100, 100), (64, 319)],
                         ids=["the loads", "the products", "an epilogue warp", "the first epilogue lane",
                              "another epilogue lane", "the epilogue"])
@pytest.mark.parametrize("cut", CUTS)
def test_waits_that_run_out(program, cut, threads):
    """Whichever wait of these threads runs out: the block ends, with an error
    set, and no copy or product is on its way behind it."""
    run(program, cut, 0, 6, *threads, 3)
