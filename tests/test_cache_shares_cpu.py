"""Which tiles of the paged cache each CTA of the streaming attention takes, compiled for the host and walked as the kernel walks them: every tile of every unit once, in
order, and the parts of a shared unit where the merge looks for them. A list too long for 32 bits, or a request that has most of it, shows here and not on the device."""
import subprocess

import pytest
import torch

from torch_mlu_b200 import build

PROGRAM = r"""
#include <algorithm>
#include <cstdio>
#include <cstdint>
#include <random>
#include <vector>
#include "cache_shares.cuh"
using namespace sdpa_b200;

struct Lists {
  const int32_t *seq_lens, *cu_q;
  int batch, heads_kv, group, total_q, rows, rows_shift, tile_shift, max_len, grid, pause, first_q, max_rows;
};

static int failed = 0;
#define CHECK(ok, ...) do { if (!(ok) && failed++ < 20) { std::printf("line %d: ", __LINE__); std::printf(__VA_ARGS__); std::printf("\n"); } } while (0)

// The walk of all CTAs of a launch, or of the first, the last and some between them where `sample` is set
static void walk_launch(const char* name, const Lists& p, bool sample) {
  int64_t all_tiles = 0, all_units = 0;
  for (int b = 0; b < p.batch; ++b) {
    const Request r = request_at(p, b);
    CHECK(r.tiles >= 1 && r.units >= 0, "%s: request %d", name, b);
    CHECK(r.q0 == (p.cu_q ? p.cu_q[b] : p.first_q + b) && (p.cu_q || r.rows_q == 1), "%s: rows of request %d", name, b);
    all_tiles += static_cast<int64_t>(r.tiles) * r.units;
    all_units += r.units;
  }
  CHECK(all_tiles + p.pause * all_units <= INT32_MAX, "%s: the launch has too many requests", name);
  if (failed) return;
  const int tiles = static_cast<int>(all_tiles), units = static_cast<int>(all_units);
  int walked = 0;
  struct At { int index, unit, tile; } next = {0, 0, 0};  // the tile that the next CTA has to begin with
  { Request r = {-1, 0, 0, 0, 0, 1, 0}; int unit = 0; next_unit(p, r, unit); next = {r.index, unit, 0}; }
  struct Begun { int from, to, slot; bool open; Request r; int unit; } begun = {};
  for (int cta = 0; cta < p.grid; ++cta) {
    if (sample && cta % 37 != 0 && cta != p.grid - 1) continue;
    Share s = {};
    const int first = tiles == 0 ? -1 : deal(s, p, tiles, units, cta);
    if (first < 0) {
      CHECK(tiles <= cta, "%s: CTA %d has nothing, %d tiles", name, cta, tiles);
      continue;
    }
    int before = 0;
    bool found = false;
    for (int b = 0; b < p.batch && !found; ++b) {
      const Request r = request_at(p, b);
      const int mine = tiles_of(r) + s.pause * r.units;
      if (first < before + mine) {
        begin_in(s, r, first - before, cta);
        found = true;
      } else {
        before += mine;
      }
    }
    CHECK(found && s.places > 0 && s.unit >= 0 && s.unit < s.request.units && s.tile >= 0 && s.tile < s.request.tiles, "%s: CTA %d begins nowhere", name, cta);
    if (failed) return;
    if (sample) {
      CHECK(before + s.unit * (s.request.tiles + s.pause) + s.pause + s.tile >= first, "%s: CTA %d", name, cta);
      if (s.places < s.request.tiles - s.tile) {
        const int last = s.cta_behind(cta, s.request.tiles - s.tile - s.places - 1);
        CHECK(last > cta && last < p.grid, "%s: CTA %d ends in %d", name, cta, last);
      }
      continue;
    }
    // ---- as the arithmetic warps do
    Request r = s.request, next_r = r;
    int unit = s.unit, tile = s.tile, following = unit;
    bool first_unit = true;
    for (int places = s.places; places > 0;) {
      const int seg = std::min(places, r.tiles - tile);
      places -= seg + s.pause;
      CHECK(r.index == next.index && unit == next.unit && tile == next.tile, "%s: CTA %d begins with (%d, %d, %d), not with (%d, %d, %d)", name, cta, r.index, unit, tile, next.index,
            next.unit, next.tile);
      if (failed) return;
      if (places > 0) next_unit(p, next_r, following);
      const bool whole = seg == r.tiles;
      const int slot = first_unit ? 0 : 1;
      if (tile == 0 && !whole) {  // the unit that the merge is told of
        CHECK(!begun.open, "%s: two open units", name);
        begun = {cta, s.cta_behind(cta, r.tiles - seg - 1), slot, true, r, unit};
        CHECK(begun.to > cta && begun.to < p.grid, "%s: CTA %d to %d", name, cta, begun.to);
      } else if (!whole) {  // a part of it: each CTA's first, one CTA after the other
        CHECK(begun.open && begun.r.index == r.index && begun.unit == unit && slot == 0 && cta == begun.from + 1 && cta <= begun.to, "%s: part of CTA %d", name, cta);
        begun.from = cta;
        CHECK((tile + seg == r.tiles) == (cta == begun.to), "%s: CTA %d ends the unit", name, cta);
        if (tile + seg == r.tiles) begun.open = false;
      }
      walked += seg;
      if (tile + seg < r.tiles) {
        next = {r.index, unit, tile + seg};
      } else {
        Request after = r;
        int u = unit;
        next_unit(p, after, u);
        next = {after.index, u, 0};
      }
      tile = 0;
      first_unit = false;
      r = next_r;
      unit = following;
    }
  }
  if (!sample) CHECK(walked == tiles && !begun.open && next.index >= p.batch, "%s: %d of %d tiles", name, walked, tiles);
}

// The same of all launches of a call
static void walk(const char* name, const std::vector<int32_t>& lens, const std::vector<int32_t>& rows_q, int heads_kv, int group, int unit_rows, int tile_shift, int capacity, bool cu,
                 int sms = 148, bool sample = false) {
  std::vector<int32_t> offsets(1, 0);
  for (int r : rows_q) offsets.push_back(offsets.back() + r);
  Lists all = {lens.data(), cu ? offsets.data() : nullptr, static_cast<int>(lens.size()), heads_kv, group, offsets.back(), unit_rows,
               unit_rows == 8 ? 3 : unit_rows == 16 ? 4 : unit_rows == 32 ? 5 : 6, tile_shift, capacity, 2 * sms, unit_rows == 64 ? 0 : 2, 0,
               std::max(1, *std::max_element(rows_q.begin(), rows_q.end()))};
  const int at_once = requests_at_once(all);
  CHECK(at_once > 0, "%s: too long", name);
  for (int first = 0; first < all.batch && !failed; first += at_once) {
    Lists p = all;
    p.batch = std::min(at_once, all.batch - first);
    p.seq_lens += first;
    if (p.cu_q) p.cu_q += first;
    p.first_q = first;
    walk_launch(name, p, sample);
  }
}

int main() {
  std::mt19937 g(1);
  auto draw = [&](int lo, int hi) { return static_cast<int>(lo + g() % static_cast<unsigned>(hi - lo + 1)); };
  for (int it = 0; it < 3000 && !failed; ++it) {
    const int batch = draw(1, it % 3 ? 9 : 300), unit_rows = 8 << draw(0, 3), top = draw(1, it % 2 ? 3000 : 300), most = draw(0, unit_rows == 64 ? 200 : unit_rows), group = draw(1, 9);
    std::vector<int32_t> lens, rows;
    for (int b = 0; b < batch; ++b) {
      lens.push_back(draw(0, 9) ? draw(0, top) : draw(-1, 1));
      rows.push_back(draw(0, 7) ? draw(0, most) : 0);
    }
    walk("drawn", lens, rows, draw(1, 9), group, unit_rows, 7 + draw(0, 1), draw(0, 1) ? top : 1 << 20, true, draw(1, 160));
  }
  auto mixed = [](int decodes, int len, int rows, int long_len, std::vector<int32_t>& lens, std::vector<int32_t>& q, int at) {
    lens.assign(decodes, len);
    q.assign(decodes, 1);
    lens.insert(lens.begin() + at, long_len);
    q.insert(q.begin() + at, rows);
  };
  std::vector<int32_t> lens, q;
  // one long chunk among many requests of a token has nearly all tiles: 8192 rows behind 131072 tokens, 32 heads over 8, beside 255
  for (int at : {0, 100, 255}) {
    mixed(255, 5000, 8192, 131072, lens, q, at);
    walk("one chunk of 8192 among 255", lens, q, 8, 4, 64, 7, 131072, true);
  }
  mixed(16383, 1, 3000, 20000, lens, q, 7000);
  walk("one chunk of 3000 among 16383", lens, q, 8, 2, 64, 8, 20000, true);
  lens.assign(512, 65536);
  q.assign(512, 8192);
  walk("512 chunks of 8192", lens, q, 8, 4, 64, 7, 65536, true, 148, true);
  // more than 2^32 tiles
  lens.assign(1024, 1 << 20);
  q.assign(1024, 8192);
  walk("1024 chunks of 8192 behind a million", lens, q, 8, 4, 64, 7, 1 << 20, true, 148, true);
  lens.assign(16384, 1 << 20);
  walk("16384 decodes of a million, 128 heads", lens, std::vector<int32_t>(16384, 1), 128, 1, 8, 7, 1 << 20, false, 148, true);
  lens.assign(1, INT32_MAX);
  walk("the longest request", lens, std::vector<int32_t>(1, 1), 1, 1, 8, 7, INT32_MAX - 256, true);
  return failed != 0;
}
"""


def test_every_tile_once_and_every_part_found(tmp_path):
    try:
        nvcc = build._nvcc()
    except RuntimeError:
        pytest.skip("needs nvcc")
    src = tmp_path / "shares.cu"
    src.write_text(PROGRAM)
    subprocess.run([nvcc, "-std=c++17", "-O2", "-I", build.CSRC, str(src), "-o", str(tmp_path / "shares")], check=True)
    run = subprocess.run([str(tmp_path / "shares")], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


def test_a_request_whose_tiles_do_not_fit_is_refused(native_lib):
    """One row of 512 kv heads over a table of 2^31 tokens has 2^32 tiles of 256."""
    import ctypes
    from test_kv_cache_cpu import _cache, _set
    from torch_mlu_b200 import _cabi
    for blocks, status in ((1 << 24, _cabi.UNSUPPORTED), (1 << 20, _cabi.NO_DEVICE)):
        p = _cache()
        _set(heads_kv=512, heads_q=512, head_dim=64, block_size=128, max_seqlen_q=1, total_q=3, max_blocks=blocks, table_stride=blocks, q_row_stride=512 * 64, q_head_stride=64,
             o_row_stride=512 * 64, o_head_stride=64)(p)
        got = native_lib.sdpa_b200_cache_attention(ctypes.byref(p), 4096, 1 << 30, None)
        if status == _cabi.UNSUPPORTED:
            assert got == status and "is too long" in native_lib.sdpa_b200_last_error().decode(), native_lib.sdpa_b200_last_error()
        elif not torch.cuda.is_available():  # fits: only the device is missing
            assert got == status


def test_workspace_of_many_requests_at_a_large_bound(native_lib):
    """16-bit copies are made for as many requests at a time as fit 4 GiB, and not at all where one does not: a bound on lengths never decides whether a call can be made."""
    import ctypes
    from test_kv_cache_cpu import _cache, _set
    from torch_mlu_b200 import _cabi
    n = ctypes.c_size_t(0)
    sizes = []
    for batch, rows, bound in ((32, 2048, 8192), (32, 2048, 131072), (256, 2048, 131072), (1, 2048, 1 << 20), (1, 2048, (1 << 20) + 1), (100000, 512, 4096)):
        p = _cache()
        _set(heads_kv=8, heads_q=32, q_row_stride=4096, o_row_stride=4096, batch=batch, total_q=rows * min(batch, 32), max_seqlen_q=rows, max_seqlen_k=bound, max_blocks=1 << 14, table_stride=1 << 14)(p)
        assert native_lib.sdpa_b200_cache_attention_workspace_bytes(ctypes.byref(p), ctypes.byref(n)) == 0
        sizes.append(n.value)
        assert n.value <= (4 << 30) + (1 << 20)
        got = native_lib.sdpa_b200_cache_attention(ctypes.byref(p), 4096, n.value, None)
        assert torch.cuda.is_available() or got == _cabi.NO_DEVICE  # nothing else is in the way
    assert 32 * 8192 * 8 * 128 * 4 <= sizes[0] < sizes[1] and sizes[3] >= 4 << 30 and sizes[4] < 1 << 27


def test_sizes_whose_product_passes_64_bits(native_lib):
    """4 * 2^31 tokens * 2^24 heads * 128 is 2^64: answered as any other size, by streaming or by a refusal."""
    import ctypes
    from test_kv_cache_cpu import _cache, _set
    from torch_mlu_b200 import _cabi
    n = ctypes.c_size_t(0)
    for heads in (1 << 22, (1 << 23) - 5, 1 << 23):
        for bound in (2 ** 31 - 1, 1 << 30, 1 << 20):
            p = _cache()
            _set(heads_kv=heads, heads_q=heads, q_row_stride=heads * 128, o_row_stride=heads * 128, k_block_stride=heads * 64 * 128, v_block_stride=heads * 64 * 128,
                 max_seqlen_q=100, total_q=200, max_seqlen_k=bound, batch=2)(p)
            assert native_lib.sdpa_b200_cache_attention_workspace_bytes(ctypes.byref(p), ctypes.byref(n)) == 0 and 0 < n.value < 1 << 27
            got = native_lib.sdpa_b200_cache_attention(ctypes.byref(p), 4096, n.value, None)
            assert got in (_cabi.UNSUPPORTED, _cabi.NO_DEVICE) or torch.cuda.is_available()
