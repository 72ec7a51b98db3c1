// What the streaming attention kernels over the paged cache have in common (cache_attention.cu: 8-bit codes, cache4_attention.cu: 4-bit ones): parameters, which
// tiles a CTA takes, and what is left of units that several CTAs worked on.
#pragma once

#include "cache_common.cuh"
#include "cache_shares.cuh"

namespace sdpa_b200 {

// The unit that begins in a CTA's share and ends in a later one's: what the merge kernel needs to know. `last` < 0: there is none.
struct SharedUnit {
  int last, slot, head, row0, rows, q0;  // the CTA that ends it; where the first CTA's part is; kv head, rows [row0, row0 + rows) of the request whose tokens begin at q0
};

struct StreamParams {
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  const void* k_scale;  // fp32 of a block and head, or bf16 of a token, head and 32 elements
  const void* v_scale;
  const int32_t* block_table;
  const int32_t* seq_lens;
  const int32_t* cu_q;
  float* part_o;    // [2 per CTA][rows][head_dim], normalised
  float* part_lse;  // [2 per CTA][rows], log2 domain; -inf: no key seen, NaN: a NaN row
  SharedUnit* shared_units;  // one per CTA
  uint32_t* status;
  int64_t q_row, q_head, o_row, o_head, table_stride;
  int batch, heads_q, heads_kv, group, total_q, max_blocks, num_blocks, shift, rows, rows_shift, grid, causal, f16;
  int tile_shift;  // log2 of a tile's tokens
  int pause;       // see share_of
  int first_q, max_rows;  // the first request's row of q where there are no offsets; rows that a request may have
  int cluster, units_each;  // CTAs that share a unit, units that each request has room for: see share_in_cluster
  int max_len;  // tokens that a table's row holds
  float scale_log2;
};

// CTAs of the kernel for 4-bit codes on an SM, by the rows of a unit
__host__ __device__ constexpr int stream4_ctas_per_sm(int rows) { return rows == 8 ? 3 : 2; }
// The kernel for 4-bit codes (cache4_attention.cu), with p.grid CTAs
cudaError_t launch_stream4(const StreamParams& p, const CUtensorMap& tm_k, const CUtensorMap& tm_v, int head_dim, cudaStream_t stream, bool overlap);

namespace {

constexpr int kWarps = 4;                  // those that do the arithmetic
constexpr int kThreads = (kWarps + 2) * 32;  // and two that load: registers are dealt out as for six warps anyway
constexpr int kCtasPerSm = 2;
constexpr int kMaxSms = 160;  // workspace sizes do not ask the device: an upper bound of its SMs (148)
constexpr int kPause = 2;  // see share_of
// Sums are kept in this unit: they are up to 2^100 a token where the largest weight is that of a block of the least scale, and no less than 2^-121 where it is that of bf16's largest
constexpr float kSumUnit = 0x1p-15f;

__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void prefetch_l1(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }
// barrier over the warps that do the arithmetic
__device__ __forceinline__ void arithmetic_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory"); }

// One 8 x 8 matrix of 16-bit elements: row g, columns 2t and 2t + 1 in, row 2t and 2t + 1, column g out
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// over the eight lanes that share t = lane % 4
__device__ __forceinline__ float column_max(float x) {
#pragma unroll
  for (int d = 4; d < 32; d *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
  return x;
}
__device__ __forceinline__ float column_sum(float x) {
#pragma unroll
  for (int d = 4; d < 32; d *= 2) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}

// A CTA's share of the list of all tiles (cache_shares.cuh). The empty places in front of a unit stand for what the hand-over from unit
// to unit takes, which is about that of two tiles (not so with 64 rows, whose warps have nothing to merge and more to do per tile: 59.5 us with it, 58.8 without, 4 requests
// of 32 rows). Measured with equal shares of the tiles | of the places, one token each, us: 64 requests
// of 200 to 1800 37.9 | 33.9, 128 of 100 to 900 52.8 | 39.9, 32 of 100 to 2000 with 32 kv heads 62 | 48.5, 64 of 500 to 4000 59.3 | 55.5; 4 tokens, 16 of 300 to 9000 at
// head_dim 64 22.0 | 19.8. With pauses of one place the second took 43.9, with three the same, and 8 tokens of 32 requests 53.8 instead of 52.0.
//
// Every warp finds it for itself, so that none waits for another.
__device__ __forceinline__ Share share_of(const StreamParams& p, int cta, int lane) {
  auto add_tiles_of = [&](int b, int& tiles, int& units) {
    if (b >= p.batch) return;
    const Request r = request_at(p, b);
    units += r.units;
    tiles += tiles_of(r);
  };
  int tiles_of_first = 0, units_of_first = 0;  // of the first 32 requests
  add_tiles_of(lane, tiles_of_first, units_of_first);
  int tiles = tiles_of_first, units = units_of_first;
#pragma unroll 4
  for (int b = lane + 32; b < p.batch; b += 32) add_tiles_of(b, tiles, units);
  tiles = __reduce_add_sync(0xffffffffu, tiles);
  Share s = {};
  if (tiles == 0) return s;
  const int first = deal(s, p, tiles, tiles >= kTilesToPause * p.grid ? __reduce_add_sync(0xffffffffu, units) : 0, cta);
  if (first < 0) return s;
  int before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    int mine = tiles_of_first, mine_units = units_of_first;
    if (b0 != 0) {
      mine = mine_units = 0;
      add_tiles_of(b0 + lane, mine, mine_units);
    }
    mine += s.pause * mine_units;
    int run = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int x = __shfl_up_sync(0xffffffffu, run, d);
      if (lane >= d) run += x;
    }
    const unsigned behind = __ballot_sync(0xffffffffu, first < before + run);
    if (behind != 0) {
      const int at = __ffs(behind) - 1;
      before += __shfl_sync(0xffffffffu, run - mine, at);
      begin_in(s, request_at(p, b0 + at), first - before, cta);
      break;
    }
    before += __shfl_sync(0xffffffffu, run, 31);
  }
  return s;
}

// A row out of its merged parts: kPer of its dimensions a lane, sums of the weights 2^(lse - top) and of the parts by them
template <int kPer>
__device__ __forceinline__ void write_row(const StreamParams& p, int q0, int head, int row, int lane, const float (&acc)[kPer], float sum, float top, bool nan) {
  const int i = row / p.group, hq = head * p.group + row - i * p.group;
  const float inv = nan ? __int_as_float(0x7fffffff) : sum > 0.f ? 1.f / sum : 0.f;
  uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + (q0 + i) * p.o_row + hq * p.o_head + kPer * lane);
#pragma unroll
  for (int e = 0; e < kPer; e += 2) dst[e / 2] = p.f16 ? pack_f16x2(acc[e] * inv, acc[e + 1] * inv) : pack_bf16x2(acc[e] * inv, acc[e + 1] * inv);
  if (lane == 0) p.lse[static_cast<int64_t>(hq) * p.total_q + q0 + i] = !nan && sum > 0.f ? (top + log2f(sum)) * 0.6931471805599453f : INFINITY;
}

// Where a cluster of CTAs takes a unit: each a stretch of its tiles. Nothing is looked up but the one request.
__device__ __forceinline__ Share share_in_cluster(const StreamParams& p, int cta) {
  const int unit = cta / p.cluster, rank = cta - unit * p.cluster, b = unit / p.units_each;
  Share s = {};
  s.request = request_at(p, b);
  s.unit = unit - b * p.units_each;
  s.each = (s.request.tiles + p.cluster - 1) / p.cluster;
  s.tile = rank * s.each;
  if (s.unit < s.request.units) s.places = max(min(s.each, s.request.tiles - s.tile), 0);
  return s;
}

// Behind a cluster barrier: the CTAs' parts of the cluster's unit become its rows, dealt out to all warps of the cluster.
template <int kD, int kAllWarps>
__device__ __forceinline__ void merge_in_cluster(const StreamParams& p, const Share& share, const float* own_part, const float* own_lse, int warp, int lane) {
  const Request& r = share.request;
  const int row0 = share.unit / p.heads_kv * p.rows, head = share.unit - share.unit / p.heads_kv * p.heads_kv;
  const int rank = blockIdx.x - blockIdx.x / p.cluster * p.cluster;
  if (share.unit < r.units && share.each < r.tiles) {  // (a single CTA's unit is done)
    const int n_rows = min(p.rows, r.rows_q * p.group - row0);
    for (int rr = rank + p.cluster * warp; rr < n_rows; rr += p.cluster * kAllWarps) {
      constexpr int kPer = kD / 32;
      float v[8][kPer];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const uint32_t src = smem_u32(own_part + rr * kD + kPer * lane);
#pragma unroll
        for (int e = 0; e < kPer; ++e) v[c][e] = 0.f;
        if (c * share.each >= r.tiles) continue;  // without tiles: its part was never written
        if constexpr (kPer == 4) {
          const float4 x = cluster_ld_f32x4(src, c);
          v[c][0] = x.x, v[c][1] = x.y, v[c][2] = x.z, v[c][3] = x.w;
        } else {
          const float2 x = cluster_ld_f32x2(src, c);
          v[c][0] = x.x, v[c][1] = x.y;
        }
      }
      const float x = lane < p.cluster ? cluster_ld_f32(smem_u32(own_lse + rr), lane) : -INFINITY;
      const bool nan = __any_sync(0xffffffffu, isnan(x));
      float top = x;
#pragma unroll
      for (int d = 1; d < 8; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      top = __shfl_sync(0xffffffffu, top, 0);
      const float w = x == -INFINITY ? 0.f : exp2f(x - top);
      float sum = 0.f, acc[kPer] = {};
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float wc = __shfl_sync(0xffffffffu, w, c);
        sum += wc;
#pragma unroll
        for (int e = 0; e < kPer; ++e) acc[e] = fmaf(wc, v[c][e], acc[e]);
      }
      write_row<kPer>(p, r.q0, head, row0 + rr, lane, acc, sum, top, nan);
    }
  }
}

}  // namespace
}  // namespace sdpa_b200
