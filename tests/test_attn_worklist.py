"""The attention kernels' work list and page look-ups on the CPU: the functions
that the kernels run, compiled for the host.

For random batches (ragged, empty, with lengths and row ranges that are wrong)
every block's walk has to cover each unit of each (sequence, tile, head) once,
stay inside the buffers, and agree with the arithmetic by which the blocks of a
split item find one another's parts."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

from conftest import PKG_DIR, ROOT

PROGRAM = r"""
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "serve.cuh"
using namespace b2g;

static unsigned state = 1;
static int draw(int lo, int hi) {
  state = state * 1664525u + 1013904223u;
  return lo + (int)((state >> 8) % (unsigned)(hi - lo + 1));
}
#define CHECK(x) do { if (!(x)) { printf("line %d: %s (case %d)\n", __LINE__, #x, case_no); exit(1); } } while (0)

template <int ROWS, int UNIT>
void run(int case_no) {
  using Work = AttnWork<ROWS, UNIT>;
  AttnParams p = {};
  int error = 0;
  p.error = &error;
  const bool wrong = case_no % 3 == 2;
  const int batch = draw(1, 9);
  p.b.batch = batch;
  p.c.kv_heads = draw(1, 4);
  p.group = draw(1, 9);
  p.c.page_size = draw(1, 40);
  p.c.num_pages = draw(1, 50);
  p.b.max_pages = draw(1, 60);
  p.b.page_table_stride = p.b.max_pages + draw(0, 3);
  p.a.window = draw(0, 2) ? 0 : draw(1, 700);
  std::vector<int> start(batch + 1), lens(batch), table(batch * p.b.page_table_stride);
  start[0] = wrong ? draw(-5, 5) : 0;
  for (int b = 0; b < batch; ++b) {
    start[b + 1] = start[b] + (draw(0, 3) ? draw(0, 4) : draw(0, 90)) - (wrong ? draw(0, 6) : 0);
    lens[b] = draw(0, p.b.max_pages * p.c.page_size + (wrong ? 500 : 0)) - (wrong ? 3 : 0);
  }
  p.b.rows = wrong ? draw(1, 60) : std::max(1, start[batch]);
  for (int& t : table) t = wrong ? draw(-3, p.c.num_pages + 3) : draw(0, p.c.num_pages - 1);
  p.b.q_start = start.data();
  p.b.seq_lens = lens.data();
  p.b.page_table = table.data();
  Work w(p);
  AttnShare s = {};
  for (int b = 0; b < batch; ++b) {
    const SeqSpan q = seq_span(p.b, b);
    CHECK(q.first >= 0 && q.n >= 0 && q.first + q.n <= p.b.rows);
    s.total += w.units(b);
  }
  const int grid = draw(1, 40), least = draw(1, 4);
  s.blocks = (int)std::max(1LL, std::min<long long>(grid, (s.total + least - 1) / least));
  CHECK(attn_begin(s, 0) == 0 && attn_begin(s, s.blocks) == s.total);
  long long next = 0;
  int b = 0, tile = 0, h = 0, u = -1;  // what has to come next
  for (int c = 0; c < s.blocks; ++c) {
    s.begin = attn_begin(s, c);
    s.end = attn_begin(s, c + 1);
    CHECK(s.begin == next);
    if (s.begin >= s.end) continue;
    s.b = 0;
    s.at = s.begin;
    for (long long n; s.at >= (n = w.units(s.b)); ++s.b) s.at -= n;
    long long at = s.at;
    AttnItem it = w.find(s.b, at);
    for (;;) {
      while (seq_span(p.b, b).n == 0 || tile >= w.tiles(seq_span(p.b, b))) ++b, tile = 0, h = 0;
      CHECK(it.b == b && it.tile == tile && it.h == h);
      CHECK(it.lo >= 0 && it.lo <= it.hi && it.hi <= w.cap && it.u_hi > it.u_lo);
      CHECK(it.u_lo * UNIT <= it.lo || it.lo == it.hi);
      CHECK((long long)it.u_hi * UNIT >= it.hi);
      for (int j = it.lo; j < it.hi; ++j) {
        int e = 0;
        const int page = page_of(p.b, p.c, it.b, j / p.c.page_size, &e);
        CHECK(page >= -1 && page < p.c.num_pages && (page == -1) == (e == kErrBadPage));
        if (!wrong) CHECK(page >= 0);
      }
      const int u0 = it.u_lo + (int)at;
      CHECK(u0 == (u < 0 ? it.u_lo : u));
      const int units = (int)std::min<long long>(it.u_hi - u0, s.end - next);
      const long long origin = next - at;
      for (int i = 0; i < units; ++i) CHECK(attn_owner(s, next + i) == c);
      const int first = attn_owner(s, origin), last = attn_owner(s, origin + (it.u_hi - it.u_lo) - 1);
      CHECK(first <= c && c <= last);
      // A block's first segment is part 0, a later one part 1; only the item's
      // first block can have begun before it.
      CHECK((next != s.begin) == (c == first && attn_begin(s, c) < origin));
      next += units;
      u = u0 + units == it.u_hi ? -1 : u0 + units;
      if (u < 0 && ++h == p.c.kv_heads) h = 0, ++tile;
      if (next >= s.end) break;
      CHECK(w.next(it));
      at = 0;
    }
  }
  CHECK(next == s.total);
  if (!wrong) CHECK(error == 0);
}

int main() {
  for (int i = 0; i < 4000; ++i) {
    run<16, 64>(i);
    run<256, 128>(i);
  }
  int case_no = -1;
  for (int i = 0; i < 200000; ++i) {  // the 32-bit and the 64-bit division
    AttnShare s = {};
    s.total = i % 2 ? draw(1, 100000) : (long long)draw(1, 1 << 22) * draw(1, 1 << 12);
    s.blocks = (int)std::min<long long>(s.total, draw(1, 300));  // never more than units
    const int c = draw(0, s.blocks - 1);
    CHECK(attn_begin(s, c) == (long long)((__int128)s.total * c / s.blocks));
    CHECK(attn_begin(s, c) < attn_begin(s, c + 1));
    CHECK(attn_owner(s, attn_begin(s, c)) == c && attn_owner(s, attn_begin(s, c + 1) - 1) == c);
  }
  puts("ok");
}
"""


def test_worklist_and_pages(tmp_path):
    nvcc = Path("/usr/local/cuda/bin/nvcc")
    nvcc = str(nvcc) if nvcc.exists() else shutil.which("nvcc")
    if nvcc is None:
        pytest.skip("no nvcc")
    src, exe = tmp_path / "worklist.cu", tmp_path / "worklist"
    src.write_text(PROGRAM)
    subprocess.run([nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "-I", str(PKG_DIR / "csrc"),
                    "-I", str(ROOT / "include"), "-o", str(exe), str(src)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout
