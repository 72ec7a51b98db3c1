// What each CTA of the streaming attention over the paged cache works on (cache_attention.cu): host and device, so that the arithmetic can be checked without a GPU.
//
// The list of all tiles: request by request, unit by unit, a place for each tile of a unit, behind `pause` empty ones that stand for the hand-over from unit to unit. Every CTA takes
// an equal contiguous share of the places, the first of them one longer where they do not come out even, and works on the tiles whose places are in its own. Places are counted in
// 32 bits: the lengths are data, but a launch takes no more requests than whose places fit at their longest (requests_at_once).
#pragma once

#include <cstdint>

namespace sdpa_b200 {

constexpr int kTilesToPause = 4;  // a CTA with fewer tiles than that has few hand-overs: the places are the tiles

// A request as units see it. One that is longer than its table has one token, in a block that there is none of, which all its rows see.
struct Request {
  int index, len, rows_q, q0;  // tokens in the cache, rows of q, the first of them
  int in_front;                // row i sees i + 1 + in_front tokens where causal
  int tiles, units;            // per unit; 0 units: no rows
};

template <class P>
__host__ __device__ __forceinline__ Request request_at(const P& p, int b) {
  Request r;
  r.index = b;
  const int len = p.seq_lens[b];
  const bool too_long = len > p.max_len;
  r.len = too_long ? 1 : len < 0 ? 0 : len;
  r.q0 = p.cu_q ? p.cu_q[b] : p.first_q + b;
  r.rows_q = 1;
  if (p.cu_q) r.rows_q = p.cu_q[b + 1] > r.q0 ? p.cu_q[b + 1] - r.q0 : 0;
  if (r.q0 < 0 || r.q0 + static_cast<int64_t>(r.rows_q) > p.total_q) r.rows_q = 0;  // offsets that leave q: no rows
  r.in_front = too_long ? r.len : r.len - r.rows_q;
  if (r.rows_q > p.max_rows) r.rows_q = p.max_rows;  // what the places were counted with: those behind are not walked
  r.tiles = (r.len + (1 << p.tile_shift) - 1) >> p.tile_shift;
  if (r.tiles < 1) r.tiles = 1;  // an empty request has rows to write too
  r.units = p.heads_kv * ((r.rows_q * p.group + p.rows - 1) >> p.rows_shift);
  return r;
}

// (those of others see less than their length in front of their first row)
__host__ __device__ __forceinline__ bool longer_than_table(const Request& r) { return r.in_front == r.len; }

__host__ __device__ __forceinline__ int tiles_of(const Request& r) { return r.tiles * r.units; }

// the next unit and its request, or one without units behind the last
template <class P>
__host__ __device__ __forceinline__ void next_unit(const P& p, Request& r, int& unit) {
  if (++unit < r.units) return;
  unit = 0;
  int b = r.index + 1;
  do {
    if (b >= p.batch) {
      r = {b, 0, 0, 0, 0, 1, 0};
      return;
    }
    r = request_at(p, b++);
  } while (r.units == 0);
}

// How many requests the places of a launch fit 32 bits with, whatever their lengths and offsets are; 0: not even those of one
template <class P>
inline int requests_at_once(const P& p) {
  const int64_t units = p.heads_kv * ((static_cast<int64_t>(p.max_rows) * p.group + p.rows - 1) >> p.rows_shift);
  const int64_t of_unit = (static_cast<int64_t>(p.max_len) + (1 << p.tile_shift) - 1) / (1 << p.tile_shift) + p.pause;
  const int64_t n = units > INT32_MAX ? 0 : INT32_MAX / (units * of_unit);
  return n < p.batch ? static_cast<int>(n) : p.batch;
}

struct Share {
  int places;         // from the first tile of the CTA on; 0: it has none
  Request request;    // where it begins
  int unit, tile;
  int pause;
  int each, longer;   // places of a share, how many shares have one more
  // the CTA that has the place `at` places behind the last of CTA `cta`'s share
  __host__ __device__ __forceinline__ int cta_behind(int cta, int at) const {
    const int more = longer - cta - 1 > 0 ? longer - cta - 1 : 0;
    const int in_longer = more * (each + 1);
    return cta + 1 + (at < in_longer ? at / (each + 1) : more + (at - in_longer) / each);
  }
};

// Deals the list out. Returns the CTA's first place, or -1 where it has none: those without a tile would leave no part where the merge looks for one.
template <class P>
__host__ __device__ __forceinline__ int deal(Share& s, const P& p, int tiles, int units, int cta) {
  s.pause = tiles >= kTilesToPause * p.grid ? p.pause : 0;
  const int places = tiles + s.pause * units, ctas = tiles < p.grid ? tiles : p.grid;
  if (cta >= ctas) return -1;
  s.each = places / ctas;
  s.longer = places - s.each * ctas;
  return cta * s.each + (cta < s.longer ? cta : s.longer);
}

// The share begins in request r, `at` places behind its first.
__host__ __device__ __forceinline__ void begin_in(Share& s, const Request& r, int at, int cta) {
  const int of_unit = r.tiles + s.pause;
  s.request = r;
  s.unit = at / of_unit;
  const int behind = at - s.unit * of_unit - s.pause;  // the unit's first tile; less than 0: empty places in front of it are left
  s.tile = behind > 0 ? behind : 0;
  s.places = s.each + (cta < s.longer ? 1 : 0) + (behind < 0 ? behind : 0);
}

}  // namespace sdpa_b200
