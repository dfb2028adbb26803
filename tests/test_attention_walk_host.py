"""What an attention kernel makes of a plan, compiled for the host: numbers that a plan of this step holds go through unchanged, and
no number that memory can hold leads outside the call's own arrays."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "attention.cuh"
#include <cstdio>
#include <cstdlib>
#include <random>
using namespace sb200;
#define REQUIRE(x) do { if (!(x)) { printf("line %d: %s (case %d)\n", __LINE__, #x, n); return 1; } } while (0)

static std::mt19937 rng(7);
static int below(int n) { return (int)(rng() % (unsigned)n); }
static int anything() {
  switch (below(6)) {
    case 0: return below(40) - 4;
    case 1: return (int)rng();
    case 2: return INT32_MIN + below(3);
    case 3: return INT32_MAX - below(3);
    case 4: return (1 << 30) + below(5) - 2;
    default: return below(3000);
  }
}

static AttnArgs arguments() {
  AttnArgs a = {};
  const int groups[] = {1, 2, 3, 4, 7, 8, 71}, pages[] = {1, 3, 8, 16, 24, 100, 1 << 20}, windows[] = {0, 0, 1, 100, (1 << 30) - 1};
  a.group = groups[below(7)];
  a.kv_heads = 1 + below(9);
  a.page_size = pages[below(7)];
  a.by_group = FastDiv::of(a.group);
  a.by_page = FastDiv::of(a.page_size);
  a.window = windows[below(5)];
  a.num_tokens = below(8) ? 1 + below(3000) : (1 << 30) / a.group > (1 << 28) ? 1 << 28 : (1 << 30) / a.group;
  a.workers = 1 + below(256);
  a.rows_many = below(2) ? 256 : 64;
  a.rows_few = below(2) ? 16 : 4;
  a.slot_rows = a.rows_many;
  a.num_kv_indices = below(5) ? below(5000) : INT32_MAX;
  const int64_t listed = std::min(a.num_kv_indices * a.page_size, (int64_t)kAttnMaxKeys);
  a.blocks = (int)((listed + kAttnBlock - 1) / kAttnBlock);
  a.plan.tiles_cap = 1 + below(1000);
  return a;
}

int main() {
  int some = 0;
  for (int n = 0; n < 2000000; ++n) {
    const AttnArgs a = arguments();
    const int most = below(2) ? a.rows_many : a.rows_few;
    const AttnTile t = {anything(), anything(), anything(), anything(), anything(), anything(), anything(), anything()};
    // (as the walk holds them)
    const int4 cur = make_int4(below(a.plan.tiles_cap), below(a.kv_heads), below(2) ? 0 : attn_clamp(anything(), 0, kAttnMaxKeys / kAttnBlock), 0);
    const int4 end = below(2) ? make_int4(cur.x, cur.y, anything(), 0) : make_int4(anything(), anything(), anything(), 0);
    int slot = below(2 * a.workers);
    const AttnPiece p = attn_piece(a, t, cur, end, most, &slot);
    REQUIRE(p.t.nrows >= 0 && (p.t.nrows == 0 || (p.t.nrows <= p.stride && p.stride <= most)));
    REQUIRE(p.head >= 0 && p.head < a.kv_heads && p.slot >= -1 && p.slot < 2 * a.workers);
    REQUIRE(p.b0 >= 0 && p.b1 >= p.b0 && p.b1 - p.b0 <= a.blocks && p.lo >= 0 && p.lo <= kAttnMaxKeys && p.hi >= 0);
    some += p.t.nrows > 0 && p.b1 > p.b0;
    {  // the steps of a warp, as the kernels count them (in 32 bits): no more than listed keys
      const int x = (int)((unsigned)(p.t.blk_lo + p.b0) * kAttnBlock), y = (int)((unsigned)(p.t.blk_lo + p.b1) * kAttnBlock);
      const int64_t key = (std::max(p.lo, x) & ~63) + 7 * 16, stop = std::min(p.hi, y);
      REQUIRE(key <= INT32_MAX && key >= 0 && stop - key <= (int64_t)a.blocks * kAttnBlock);
    }
    for (int r : {0, p.t.nrows - 1}) {
      if (r < 0 || r >= p.t.nrows) continue;
      int token, head, pos;
      attn_row(a, p, r, &token, &head, &pos);
      REQUIRE(token >= 0 && token < a.num_tokens && head >= 0 && head < a.kv_heads * a.group);
    }
  }
  const int n = -1;
  REQUIRE(some > 1000);
  // Tiles as the plan kernel makes them: requests of q tokens, `len` keys (maybe fewer than new tokens), some pages.
  for (int n = 0; n < 200000; ++n) {
    AttnArgs a = arguments();
    if (a.num_tokens > 100000) a.num_tokens = 100000;
    const int most = below(2) ? a.rows_many : a.rows_few;
    const int q_row = below(a.num_tokens), q = 1 + below(a.num_tokens - q_row);
    const int64_t pages_before = below(3), room = std::min((int64_t)(1 + below(1 << 20)), (int64_t)kAttnMaxKeys);
    const int64_t pages = (room + a.page_size - 1) / a.page_size;
    a.num_kv_indices = pages_before + pages + below(3);
    const int64_t listed = std::min(a.num_kv_indices * a.page_size, (int64_t)kAttnMaxKeys);
    a.blocks = (int)((listed + kAttnBlock - 1) / kAttnBlock);
    const int len = below(10) ? (int)room : below((int)room + 1);
    const int tiles = (int)(((int64_t)q * a.group + most - 1) / most), row0 = below(tiles) * most;
    const int nrows = (int)std::min((int64_t)most, (int64_t)q * a.group - row0);
    const int tok0 = row0 / a.group, tok1 = (row0 + nrows - 1) / a.group, pos0 = len - q;
    const int hi = std::max(0, pos0 + tok1 + 1), lo = a.window > 0 ? std::max(0, pos0 + tok0 + 1 - a.window) : 0;
    AttnTile t = {q_row, row0, nrows, 1, pos0, (int)pages_before, lo / kAttnBlock, 0};
    t.nblk = std::max(0, (hi + kAttnBlock - 1) / kAttnBlock - t.blk_lo);
    const int head = below(a.kv_heads), b0 = t.nblk ? below(t.nblk) : 0, b1 = b0 + (t.nblk > b0 ? 1 + below(t.nblk - b0) : 0);
    const int4 cur = make_int4(3, head, b0, 0), end = b1 < t.nblk ? make_int4(3, head, b1, 0) : make_int4(4, 0, 0, 0);
    const int slot0 = below(2 * a.workers);
    int slot = slot0;
    const int had = a.num_tokens;
    if (!below(4)) a.num_tokens = 1 + below(had);  // q with fewer rows than planned
    const int rows = std::min(nrows, std::max(0, (a.num_tokens - q_row) * a.group - row0));
    const AttnPiece p = attn_piece(a, t, cur, end, most, &slot);
    const bool whole = b0 == 0 && b1 == t.nblk;
    REQUIRE(p.t.nrows == rows && p.head == head && p.slot == (whole ? -1 : slot0) && slot == slot0 + !whole);
    if (rows) {
      REQUIRE(p.stride == nrows && p.b0 == b0 && p.b1 == b1);
      REQUIRE(p.t.blk_lo == t.blk_lo && p.t.nblk == t.nblk && p.t.page_at == t.page_at && p.t.pos0 == pos0);
      const int last = (row0 + rows - 1) / a.group;
      REQUIRE(p.t.q_row == q_row && p.t.row0 == row0);
      REQUIRE(p.hi == std::max(0, pos0 + last + 1) && p.lo == lo);
    }
  }
  puts("fine");
  return 0;
}
"""


def test_pieces_of_any_plan(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    src, exe = tmp_path / "walk.cu", tmp_path / "walk"
    src.write_text(PROGRAM)
    cmd = [nvcc, "-O2", "-std=c++17", "--expt-relaxed-constexpr", "-gencode", "arch=compute_100a,code=sm_100a",
           "-I", os.path.join(ROOT, "sarathi_serve_b200", "csrc"), str(src), "-o", str(exe)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout == "fine\n", r.stdout
