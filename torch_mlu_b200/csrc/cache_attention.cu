// Attention over the 8-bit paged cache. No counterpart in the reference, which has no paged cache.
//
//   s_ij = scale * ks[block(j), h] * <q_i, kc_j>,  out_i = sum_j softmax_j(s_i) * vs[block(j), h] * vc_j
//
// over the cached tokens j of the request, j <= i + len - rows of q where causal. Two paths:
//
// 1. Few rows per request (decode steps, drafted tokens): cache_stream_kernel, bound by the codes that come out of HBM. A unit is (request,
//    kv head, chunk of up to 64 rows (query token, query head of the group)), whose codes are read once for all its rows: S^T = K Q^T and
//    O^T = V^T W^T in mma.sync.m16n8k16, tokens and dimensions in M, 8 rows in N, so that the few rows of a decode step leave no part of an
//    instruction empty. The lengths are on the GPU; every CTA sums them up and takes an equal contiguous share of all units' tiles of 128 or
//    256 tokens and of the hand-overs between units, so that all SMs are done at the same time however long each request is. A unit that several CTAs worked on leaves fp32
//    parts in the workspace, at most two per CTA, and a second kernel merges them. Few short units are taken by a cluster of CTAs each instead.
//    Two warps of a CTA, one for K and one for V, look up blocks and scales, two groups of 32 pages ahead, and fill a ring of tiles by TMA (a
//    copy takes its warp about 100 cycles, which one warp with 16 of them per tile of 16 KB - blocks of 16 tokens, head_dim 64 - could not keep
//    up with); four do the arithmetic, as 1, 2 or 4 groups of 8 or 16 rows by 4, 2 or 1 parts of a tile's tokens.
//    Codes become f16, exactly. Q rows are brought to f16 by a power of two each (their largest element to 2^14..2^15: a bf16 element loses only
//    what is 2^-39 of the row's largest). The scale of K goes onto the fp32 scores; that of V into the exponent, so that the weights
//    w_j = 2^(s_j + log2 vs_j - m) with m their running maximum are f16 numbers of up to 2^15 which keep all 11 bits down to 2^-29 of the
//    largest, whatever scales blocks have, and the products add up in the tensor core's fp32 accumulators without a pass over them. The sum of
//    the softmax takes w_j / vs_j in fp32; from the first tile on that has a scale of V above 1 it takes 2^(s_j - m), another exponential, since w_j may then be too small
//    for 32 bits beside a key whose value is 2^100 times as large (in a loop of its own: within the one for all calls it cost 2 to 5%).
//    Measured, one token per request, head_dim 128: 64 requests of 2048 to 32768 tokens, 8 kv heads, 1.9 GB of codes: 292 to 300 us, 6.3 to 6.5 TB/s, 97 to 99% of a
//    copy's rate. What is small does not get there: about 4 us go by before the first tile is there, 2 to 3 in a unit's hand-over between warps,
//    2 to 3 in the merge, and shares are whole tiles. 64 requests of 200 to 1800: 34 us, 3.7 TB/s; one of 1000, in clusters: 6.2 us.
// 2. Many rows (chunks of prompts): the tensor cores bound it. cache_gather_kernel brings the request's codes * scales into 16-bit packed tensors
//    in the workspace (exact with the powers of two that the store kernel chooses, within the type's range), and the prefill kernel does the rest. 512 tokens behind 7680,
//    2 requests, 32 heads of 128: 134 to 139 us.
#include <algorithm>
#include <type_traits>

#include "cache_common.cuh"
#include "cache_shares.cuh"

namespace sdpa_b200 {
namespace {

constexpr int kWarps = 4;                  // those that do the arithmetic
constexpr int kThreads = (kWarps + 2) * 32;  // and two that load: registers are dealt out as for six warps anyway
constexpr int kCtasPerSm = 2;
constexpr int kMaxSms = 160;  // workspace sizes do not ask the device: an upper bound of its SMs (148)
constexpr int kPause = 2;  // see share_of
constexpr int kTilesInCluster = 8;          // that a CTA of a cluster may get: see cluster_of
constexpr int kMostClusterCtas = 256;       // clusters of eight find room for that many CTAs at once
constexpr float kLeastScale = 0x1p-100f;   // of V: a block of zeros may have a scale of 0, which has no logarithm
// Sums are kept in this unit: they are up to 2^100 a token where the largest weight is that of a block of the least scale, and no less than 2^-121 where it is that of bf16's largest
constexpr float kSumUnit = 0x1p-15f;
// Scales of V above it are far from the least one: a weight times its scale, or what such products are multiplied by when their maximum moves, may then be too small for 32 bits
// though the weight itself counts. Up to it, a key that is lost has less than 2^-26 of the largest weight.
constexpr float kFarScale = 1.f;

struct StreamParams {
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_table;
  const int32_t* seq_lens;
  const int32_t* cu_q;
  float* part_o;    // [2 per CTA][rows][head_dim], normalised
  float* part_lse;  // [2 per CTA][rows], log2 domain; -inf: no key seen, NaN: a NaN row
  struct SharedUnit* shared_units;  // one per CTA
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

// The unit that begins in a CTA's share and ends in a later one's: what the merge kernel needs to know. `last` < 0: there is none.
struct SharedUnit {
  int last, slot, head, row0, rows, q0;  // the CTA that ends it; where the first CTA's part is; kv head, rows [row0, row0 + rows) of the request whose tokens begin at q0
};

// Tokens of a tile, 32 KB of K and V, and those that a warp handles at a time: its products, maxima over lanes, exponentials and products again are one long chain, in which the
// blocks of 16 tokens run beside each other; as many as registers hold.
template <int kD>
__host__ __device__ constexpr int tile_tokens() { return kD == 64 ? 256 : 128; }
template <int kD>
__host__ __device__ constexpr int step_tokens() { return kD == 64 ? 64 : 32; }
// Tiles in a CTA's ring: what lets two CTAs share an SM's 228 KB (64 rows: Q is there too).
template <int kRowWarps, int kD>
__host__ __device__ constexpr int ring_stages() { return kD == 128 && kRowWarps == 4 ? 2 : 3; }
template <int kD>
__host__ __device__ constexpr uint32_t stage_bytes() { return 2u * tile_tokens<kD>() * kD; }
// B fragments of Q: in registers where there is room; else in shared memory, for each group of 16 rows
template <int kRowBlocks, int kD>
__host__ __device__ constexpr bool q_in_registers() { return kRowBlocks == 1 || kD == 64; }
template <int kRowBlocks, int kRowWarps, int kD>
__host__ __device__ constexpr uint32_t stream_smem_bytes() {
  return 1024 + ring_stages<kRowWarps, kD>() * (stage_bytes<kD>() + tile_tokens<kD>() + 16) + 16 + kWarps * 16 * 8 +
         (q_in_registers<kRowBlocks, kD>() ? 0 : kRowWarps * kRowBlocks * (kD / 16) * 2 * 128);
}

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

// kRowBlocks: blocks of 8 rows of a warp. kRowWarps: groups of that many rows of a unit; the warps of a group share the tile's tokens.
template <int kRowBlocks, int kRowWarps, int kD, bool kInt8, bool kCluster>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
cache_stream_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const StreamParams p) {
  constexpr int kChunks = kD / 16;                           // 16 dimensions each
  constexpr int kSt = ring_stages<kRowWarps, kD>();
  constexpr bool kQInRegisters = q_in_registers<kRowBlocks, kD>();
  constexpr uint32_t kStageBytes = stage_bytes<kD>();
  constexpr int kParts = kWarps / kRowWarps;                 // of a tile's tokens
  constexpr int kTileTokens = tile_tokens<kD>(), kStepTokens = step_tokens<kD>(), kHalves = kStepTokens / 16;
  constexpr int kSlots = kTileTokens / 16;                   // the fewest tokens with scales of their own are 16
  constexpr int kPartTokens = kTileTokens / kParts;
  constexpr int kRowsOfWarp = 8 * kRowBlocks;
  constexpr float kBias = 15.f;  // weights are kept times 2^15: the largest is 2^15, the smallest normal f16 number 2^-29 of it
  constexpr int kState = kChunks * kRowBlocks * 4 * 32;      // floats of a warp's accumulators
  static_assert(kWarps * kState * 4 <= kStageBytes || kParts == 1, "the warps' states do not fit a tile's place");
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t ring = (raw_addr + 1023u) & ~1023u;
  uint8_t* ring_ptr = smem_raw + (ring - raw_addr);
  float4* slot_scales = reinterpret_cast<float4*>(ring_ptr + kSt * kStageBytes);  // [stage][16 tokens]: of K, log2 of that of V, kSumUnit over that of V, 1 where one of V's is far
  float2* row_state = reinterpret_cast<float2*>(slot_scales + kSt * kSlots);      // [warp][row]: maximum and sum
  uint2* q_state = reinterpret_cast<uint2*>(row_state + kWarps * 16);             // [row group][block of 8 rows][chunk][lane]: B fragments
  constexpr int kQWords = kQInRegisters ? 0 : kRowWarps * kRowBlocks * kChunks * 32;
  const uint32_t full = smem_u32(q_state + kQWords), empty = full + 8 * kSt;
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(reinterpret_cast<uint64_t*>(q_state + kQWords) + 2 * kSt);

  // kCluster: this CTA's part of the unit
  float* own_part = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(abort_flag) + 4 + 15) & ~static_cast<uintptr_t>(15));  // [row][dimension]
  float* own_lse = own_part + kRowsOfWarp * kD;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (kCluster && threadIdx.x < kRowsOfWarp) own_lse[threadIdx.x] = -INFINITY;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSt; ++i) {
      mbar_init(full + 8 * i, 2);
      mbar_init(empty + 8 * i, kWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp >= kWarps && elect_one()) tma_prefetch_desc(warp == kWarps ? &tm_k : &tm_v);
  __syncthreads();
  wait_for_previous_grid();
  if (threadIdx.x == 0) launch_dependents();  // behind the wait: the merge kernel's blocks wait for this grid only
  const Share share = kCluster ? share_in_cluster(p, blockIdx.x) : share_of(p, blockIdx.x, lane);
  if (share.places > 0 && warp >= kWarps) {
    // ================================================================ the loading warps, one for K and one for V
    // Lane i has page 32 * group + i of a unit: block number (num_blocks: none in the cache, behind which the copy finds zeros; -1: no such page) and scale. Three
    // groups are under way: the one that tiles are copied from, the next with its scales, and the block numbers of the one behind.
    const bool keys = warp == kWarps;
    const CUtensorMap* map = keys ? &tm_k : &tm_v;
    const float* scales = keys ? p.k_scale : p.v_scale;
    struct Place {
      Request r;
      int unit, group, head;
    };
    auto advance = [&](Place& x) {
      if (static_cast<int64_t>((x.group + 1) * 32) << p.shift < x.r.len) {
        ++x.group;
      } else {
        x.group = 0;
        if (x.r.units > 0) next_unit(p, x.r, x.unit);
        x.head = x.unit % p.heads_kv;
      }
    };
    auto block_at = [&](const Place& x) {
      const int page = x.group * 32 + lane;
      if ((static_cast<int64_t>(page) << p.shift) >= x.r.len) return -1;
      const int id = page < p.max_blocks && !longer_than_table(x.r) ? p.block_table[x.r.index * p.table_stride + page] : -1;
      return id >= 0 && id < p.num_blocks ? id : p.num_blocks;
    };
    auto scale_at = [&](const Place& x, int id) {
      if (id >= 0 && id < p.num_blocks) return scales[static_cast<int64_t>(id) * p.heads_kv + x.head];
      return keys && id == p.num_blocks ? __int_as_float(0x7fffffff) : 0.f;  // none in the cache: the scores of those who see it are NaN
    };
    Place cur, nxt, far;
    cur.r = share.request;
    cur.unit = share.unit;
    cur.head = cur.unit % p.heads_kv;
    int tile = share.tile;
    cur.group = ((tile * kTileTokens) >> p.shift) >> 5;
    nxt = far = cur;
    int id = block_at(cur), next_id = -1, far_id = -1;
    float scale = scale_at(cur, id), next_scale = 0.f;
    auto next_group = [&]() {
      cur = nxt, id = next_id, scale = next_scale;
      nxt = far, next_id = far_id;
      next_scale = scale_at(nxt, next_id);
      advance(far);
      far_id = block_at(far);
    };
    const int pages = kTileTokens >> p.shift;  // of a tile
    bool ok = true, far_scales = false;  // a scale of V above kFarScale has been seen, in this tile or before
    int step = 0;
    bool first = true;
    for (int places = share.places; places > 0;) {
      const int page0 = (tile * kTileTokens) >> p.shift;
      if (page0 >> 5 != cur.group) next_group();  // the unit goes on in its next group
      const bool tokens = tile * kTileTokens < cur.r.len;
      const uint32_t st = step % kSt, bar = full + 8 * st;
      if (tokens) {
        const uint32_t dst = ring + st * kStageBytes + (keys ? 0u : kTileTokens * kD);
        if (ok && step >= kSt) ok = mbar_wait(empty + 8 * st, (step / kSt + 1) & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const int mine = __shfl_sync(0xffffffffu, id, ((page0 & 31) + lane) & 31);
        const int n = __popc(__ballot_sync(0xffffffffu, lane < pages && mine >= 0));
        if (elect_one()) mbar_expect_tx(bar, static_cast<uint32_t>(n << p.shift) * kD);
#pragma unroll 1
        for (int i = 0; i < n; i += 4) {  // their numbers come by four: one at a time cost a call with blocks of 16 tokens 3% more
          int blocks[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) blocks[e] = __shfl_sync(0xffffffffu, mine, (i + e) & 31);
          if (elect_one()) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (i + e < n) tma_load_4d(dst + ((i + e) << p.shift) * kD, map, bar, 0, 0, cur.head, blocks[e]);
          }
        }
      }
      if (first) {  // the first copies are under way
        advance(nxt);
        next_id = block_at(nxt);
        far = nxt;
        advance(far);
        far_id = block_at(far);
      }
      if (tokens) {
        const int src = (page0 & 31) + ((lane % kSlots) * 16 >> p.shift);
        const float own = __shfl_sync(0xffffffffu, scale, src);
        float* slot = reinterpret_cast<float*>(slot_scales + st * kSlots + lane);
        if (lane < kSlots) {
          if (keys) {
            slot[0] = fabsf(own) == INFINITY ? __int_as_float(0x7fffffff) : own;
          } else {
            const float used = own >= 0.f ? fmaxf(own, kLeastScale) : __int_as_float(0x7fffffff);
            slot[1] = log2f(used);
            slot[2] = kSumUnit / used;
            if (__any_sync((1u << kSlots) - 1, used > kFarScale)) far_scales = true;
            slot[3] = far_scales ? 1.f : 0.f;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
        ++step;
      }
      if (first) next_scale = scale_at(nxt, next_id);
      first = false;
      --places;
      if (++tile == cur.r.tiles) {
        tile = 0;
        places -= share.pause;
        next_group();
      }
    }
  }

  SharedUnit left = {-1, 0, 0, 0, 0, 0};
  if (share.places > 0 && warp < kWarps) {
    // ================================================================ the arithmetic. Fragments: a thread has rows 2t and 2t + 1 of every 8
    const int g = lane >> 2;
    const int t = lane & 3;
    const int row_group = warp / kParts, part = warp % kParts;
    const int mrow = lane & 7, mat = lane >> 3;
    auto chunk_at = [&](int row, int chunk) -> uint32_t {  // byte offset of a 16-byte chunk of a row in a swizzled tile
      if constexpr (kD == 128) return row * 128 + ((chunk ^ (row & 7)) << 4);
      return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
    };
    bool ok = true;
    int step = 0;  // tiles read
    Request r = share.request;
    int unit = share.unit, tile = share.tile;
    Request next_r = r;
    int next = unit;  // the unit behind
    bool first_unit = true;
    for (int places = share.places; places > 0;) {
      const int seg_tiles = min(places, r.tiles - tile);
      places -= seg_tiles + share.pause;
      const int row0 = unit / p.heads_kv * p.rows, head = unit - unit / p.heads_kv * p.heads_kv;
      const int n_rows = min(p.rows, r.rows_q * p.group - row0);
      const int my_row0 = row0 + kRowsOfWarp * row_group;
      // ---- this lane's row of Q as B fragments, row g of every 8: elements as f16. Thread t has dimensions 4t..4t+3 of every 16
      uint32_t qb[kRowBlocks][kQInRegisters ? kChunks : 1][2];
      uint2* my_q = q_state + row_group * kRowBlocks * kChunks * 32 + lane;
      float2 factor[kRowBlocks];  // of rows 2t, 2t + 1, with the softmax scale
      int2 limit[kRowBlocks];     // how many tokens they see
#pragma unroll
      for (int nb = 0; nb < kRowBlocks; ++nb) {
        const int row = my_row0 + 8 * nb + g, i = row / p.group;
        const bool have = row < row0 + n_rows;
        const uint16_t* src = p.q + (r.q0 + i) * p.q_row + (head * p.group + row - i * p.group) * p.q_head + 4 * t;
        uint2 w[kChunks];
#pragma unroll
        for (int k = 0; k < kChunks; ++k) w[k] = have ? *reinterpret_cast<const uint2*>(src + 16 * k) : make_uint2(0u, 0u);
        float largest = 0.f;
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
          const float2 a = p.f16 ? unpack_16x2<true>(w[k].x) : unpack_16x2<false>(w[k].x), b = p.f16 ? unpack_16x2<true>(w[k].y) : unpack_16x2<false>(w[k].y);
          largest = fmaxf(largest, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))));
        }
        largest = quad_max(largest);
        const int e = min(max(static_cast<int>(__float_as_uint(largest) >> 23) - 127, -100), 127);
        const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 - e) << 23);
        const float down = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - 14 + e) << 23);
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
          const float2 a = p.f16 ? unpack_16x2<true>(w[k].x) : unpack_16x2<false>(w[k].x), b = p.f16 ? unpack_16x2<true>(w[k].y) : unpack_16x2<false>(w[k].y);
          const uint2 packed = make_uint2(pack_f16x2(a.x * up, a.y * up), pack_f16x2(b.x * up, b.y * up));
          if constexpr (kQInRegisters) {
            qb[nb][k][0] = packed.x;
            qb[nb][k][1] = packed.y;
          } else if (part == 0) {
            my_q[(nb * kChunks + k) * 32] = packed;
          }
        }
        const int sees = p.causal ? min(r.len, i + 1 + r.in_front) : r.len;
        factor[nb] = make_float2(__shfl_sync(0xffffffffu, down, 8 * t), __shfl_sync(0xffffffffu, down, 8 * t + 4));
        limit[nb] = make_int2(__shfl_sync(0xffffffffu, sees, 8 * t), __shfl_sync(0xffffffffu, sees, 8 * t + 4));
      }
      if constexpr (!kQInRegisters) arithmetic_sync();
      if (places > 0) {  // where the next unit's rows of Q are: they come nearer while this one's tiles are worked on
        next_unit(p, next_r, next);
        const int next_row0 = next / p.heads_kv * p.rows + kRowsOfWarp * row_group;
#pragma unroll
        for (int nb = 0; nb < kRowBlocks; ++nb) {
          const int row = next_row0 + 8 * nb + g, i = row / p.group;
          if (t * 64 < kD && row < next_r.rows_q * p.group)
            prefetch_l1(p.q + (next_r.q0 + i) * p.q_row + ((next - next / p.heads_kv * p.heads_kv) * p.group + row - i * p.group) * p.q_head + 64 * t);
        }
      }
      // tokens that all of the warp's rows see, and those that any of them does
      const int last_row = min(my_row0 + kRowsOfWarp - 1, row0 + n_rows - 1);
      const int seen_by_all = p.causal ? min(r.len, my_row0 / p.group + 1 + r.in_front) : r.len;
      const int seen_by_any = my_row0 >= row0 + n_rows ? 0 : p.causal ? min(r.len, last_row / p.group + 1 + r.in_front) : r.len;

      float o[kRowBlocks][kChunks][4];  // dimensions 2g, 2g, 2g + 1, 2g + 1 of every 16, rows 2t, 2t + 1, 2t, 2t + 1
      float2 m[kRowBlocks], l[kRowBlocks];  // running maximum of score + log2 of V's scale; this thread's share of the sums, in units of kSumUnit
#pragma unroll
      for (int nb = 0; nb < kRowBlocks; ++nb) {
        m[nb] = make_float2(-INFINITY, -INFINITY);
        l[nb] = make_float2(0.f, 0.f);
#pragma unroll
        for (int ch = 0; ch < kChunks; ++ch) o[nb][ch][0] = o[nb][ch][1] = o[nb][ch][2] = o[nb][ch][3] = 0.f;
      }

      for (int i = 0; i < seg_tiles; ++i) {
        const int tile_tok = (tile + i) * kTileTokens;
        if (tile_tok >= r.len) break;  // a request without tokens
        const uint32_t st = step % kSt;
        if (ok) ok = mbar_wait(full + 8 * st, (step / kSt) & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        __syncwarp();
        // ---- S^T = K Q^T, 16 tokens at a time. The contraction runs over head_dim in the order in which ldmatrix hands out bytes
        // s: tokens g, g, g + 8, g + 8 of each half, rows 2t, 2t + 1, 2t, 2t + 1
        auto scores = [&](int c, float (&s)[kRowBlocks][kHalves][4]) {
          const uint32_t k_smem = ring + st * kStageBytes + (part * kPartTokens + c) * kD;
#pragma unroll
          for (int half = 0; half < kHalves; ++half)
#pragma unroll
            for (int nb = 0; nb < kRowBlocks; ++nb) s[nb][half][0] = s[nb][half][1] = s[nb][half][2] = s[nb][half][3] = 0.f;
#pragma unroll
          for (int ch = 0; ch < kChunks; ch += 2) {
            uint32_t q[2][kRowBlocks][2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int nb = 0; nb < kRowBlocks; ++nb) {
                if constexpr (kQInRegisters) {
                  q[e][nb][0] = qb[nb][ch + e][0];
                  q[e][nb][1] = qb[nb][ch + e][1];
                } else {
                  const uint2 w = my_q[(nb * kChunks + ch + e) * 32];
                  q[e][nb][0] = w.x;
                  q[e][nb][1] = w.y;
                }
              }
#pragma unroll
            for (int half = 0; half < kHalves; ++half) {
              uint32_t kf[4];  // tokens 0-7 and 8-15 of a chunk, the same of the next
              ldmatrix_x4(k_smem + chunk_at(half * 16 + (mat & 1) * 8 + mrow, ch + (mat >> 1)), kf);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                uint32_t a0, a1, a2, a3;
                codes_to_f16<kInt8>(kf[2 * e], a0, a2);
                codes_to_f16<kInt8>(kf[2 * e + 1], a1, a3);
#pragma unroll
                for (int nb = 0; nb < kRowBlocks; ++nb) mma_16816<true>(s[nb][half], a0, a1, a2, a3, q[e][nb][0], q[e][nb][1]);
              }
            }
          }
        };
        auto work_on = [&](int c, auto far_tag) {
          constexpr bool kFar = decltype(far_tag)::value;
          const int in_tile = part * kPartTokens + c, tok = tile_tok + in_tile;
          const uint32_t v_smem = ring + st * kStageBytes + in_tile * kD + kTileTokens * kD;
          float s[kRowBlocks][kHalves][4];
          scores(c, s);
          float4 sc[kHalves];
#pragma unroll
          for (int half = 0; half < kHalves; ++half) sc[half] = slot_scales[st * kSlots + in_tile / 16 + half];
          uint32_t pb[kRowBlocks][kHalves][2];  // weights as B fragments: tokens 2t, 2t + 1 (and 8 behind) of each half, row g
          bool moved = false;
          float2 a[kRowBlocks];
#pragma unroll
          for (int nb = 0; nb < kRowBlocks; ++nb) {
            // scores and log2 of V's scale, masked where a row ends inside the step
#pragma unroll
            for (int half = 0; half < kHalves; ++half) {
              const float ks = sc[half].x, lv = sc[half].y;
              const float fx = factor[nb].x * ks, fy = factor[nb].y * ks;
              s[nb][half][0] = fmaf(s[nb][half][0], fx, lv);
              s[nb][half][1] = fmaf(s[nb][half][1], fy, lv);
              s[nb][half][2] = fmaf(s[nb][half][2], fx, lv);
              s[nb][half][3] = fmaf(s[nb][half][3], fy, lv);
            }
            if (tok + kStepTokens > seen_by_all) {
#pragma unroll
              for (int half = 0; half < kHalves; ++half) {
                const int j = tok + half * 16 + g;
                if (j >= limit[nb].x) s[nb][half][0] = -INFINITY;
                if (j >= limit[nb].y) s[nb][half][1] = -INFINITY;
                if (j + 8 >= limit[nb].x) s[nb][half][2] = -INFINITY;
                if (j + 8 >= limit[nb].y) s[nb][half][3] = -INFINITY;
              }
            }
            float mx = s[nb][0][0], my = s[nb][0][1];
#pragma unroll
            for (int half = 0; half < kHalves; ++half) {
              mx = max3(mx, s[nb][half][0], s[nb][half][2]);
              my = max3(my, s[nb][half][1], s[nb][half][3]);
            }
            mx = fmaxf(m[nb].x, column_max(mx));
            my = fmaxf(m[nb].y, column_max(my));
            // a row that has seen no key has o = l = 0: any finite factor will do
            a[nb] = make_float2(mx == -INFINITY ? 1.f : ex2_approx(m[nb].x - mx), my == -INFINITY ? 1.f : ex2_approx(m[nb].y - my));
            if constexpr (kFar) {  // sums take the factor in two steps, and weights without the scales; numbers below 2^-126 count
              const float vx = mx == -INFINITY ? 0.f : mx, vy = my == -INFINITY ? 0.f : my;
              const float hx = exp2f(0.5f * (m[nb].x - vx)), hy = exp2f(0.5f * (m[nb].y - vy));
              l[nb].x = l[nb].x * hx * hx;
              l[nb].y = l[nb].y * hy * hy;
#pragma unroll
              for (int half = 0; half < kHalves; ++half) {
                const float lv = sc[half].y;
                l[nb].x += exp2f(s[nb][half][0] - lv - vx) + exp2f(s[nb][half][2] - lv - vx);
                l[nb].y += exp2f(s[nb][half][1] - lv - vy) + exp2f(s[nb][half][3] - lv - vy);
              }
            } else {
              l[nb].x *= a[nb].x;
              l[nb].y *= a[nb].y;
            }
            moved = moved || a[nb].x != 1.f || a[nb].y != 1.f;
            m[nb] = make_float2(mx, my);
            const float ux = mx == -INFINITY ? 0.f : mx - kBias, uy = my == -INFINITY ? 0.f : my - kBias;
#pragma unroll
            for (int half = 0; half < kHalves; ++half) {
              const float rv = sc[half].z;
              const float x0 = ex2_approx(s[nb][half][0] - ux), y0 = ex2_approx(s[nb][half][1] - uy);
              const float x1 = ex2_approx(s[nb][half][2] - ux), y1 = ex2_approx(s[nb][half][3] - uy);
              if constexpr (!kFar) {
                l[nb].x = fmaf(x0 + x1, rv, l[nb].x);
                l[nb].y = fmaf(y0 + y1, rv, l[nb].y);
              }
              pb[nb][half][0] = transpose_8x8(pack_f16x2(x0, y0));
              pb[nb][half][1] = transpose_8x8(pack_f16x2(x1, y1));
            }
          }
          if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int nb = 0; nb < kRowBlocks; ++nb)
#pragma unroll
              for (int ch = 0; ch < kChunks; ++ch) {
                o[nb][ch][0] *= a[nb].x;
                o[nb][ch][1] *= a[nb].y;
                o[nb][ch][2] *= a[nb].x;
                o[nb][ch][3] *= a[nb].y;
              }
          }
          // ---- O^T += V^T W^T, 16 tokens at a time. What stands behind the request's last token may be anything: it must not meet a weight of 0
          auto add_half = [&](int half, uint32_t keep0, uint32_t keep1) {
            uint32_t weights[kRowBlocks][2];
#pragma unroll
            for (int nb = 0; nb < kRowBlocks; ++nb)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                weights[nb][e] = pb[nb][0][e];
#pragma unroll
                for (int x = 1; x < kHalves; ++x) weights[nb][e] = half == x ? pb[nb][x][e] : weights[nb][e];
              }
#pragma unroll
            for (int ch = 0; ch < kChunks; ch += 2) {
              uint32_t vf[4];
              ldmatrix_x4_trans(v_smem + chunk_at(half * 16 + (mat & 1) * 8 + mrow, ch + (mat >> 1)), vf);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                uint32_t even0, odd0, even1, odd1;  // f16 pairs of two tokens: dimension 2g, dimension 2g + 1
                codes_to_f16_by_two<kInt8>(vf[2 * e] & keep0, even0, odd0);
                codes_to_f16_by_two<kInt8>(vf[2 * e + 1] & keep1, even1, odd1);
#pragma unroll
                for (int nb = 0; nb < kRowBlocks; ++nb) mma_16816<true>(o[nb][ch + e], even0, odd0, even1, odd1, weights[nb][0], weights[nb][1]);
              }
            }
          };
          if (tok + kStepTokens <= r.len) {
#pragma unroll
            for (int half = 0; half < kHalves; ++half) add_half(half, ~0u, ~0u);
          } else {
            auto keep = [&](int j) { return (j < r.len ? 0xffffu : 0u) | (j + 1 < r.len ? 0xffff0000u : 0u); };
#pragma unroll 1
            for (int half = 0; half < kHalves; ++half) {
              const int j = tok + half * 16 + 2 * t;
              if (tok + half * 16 < r.len) add_half(half, keep(j), keep(j + 8));
            }
          }
        };
        const int end = min(kPartTokens, seen_by_any - tile_tok - part * kPartTokens);
        if (slot_scales[st * kSlots].w == 0.f) {
#pragma unroll 1
          for (int c = 0; c < end; c += kStepTokens) work_on(c, std::false_type{});
        } else {
#pragma unroll 1
          for (int c = 0; c < end; c += kStepTokens) work_on(c, std::true_type{});
        }
        // every lane has read the tile: it may be filled again, but for the segment's last, whose place the warps hand their states over in
        if (i + 1 < seg_tiles) {
          __syncwarp();
          if (lane == 0) mbar_arrive(empty + 8 * st);
          ++step;
        }
      }
      const bool tokens = r.len > 0;
      const uint32_t st = step % kSt;
#pragma unroll
      for (int nb = 0; nb < kRowBlocks; ++nb) l[nb] = make_float2(column_sum(l[nb].x), column_sum(l[nb].y));
      // ---- the parts of a tile's tokens come together: every warp takes some of the dimensions, of all parts
      constexpr int kMine = kChunks / kParts;
      float* states = reinterpret_cast<float*>(ring_ptr + st * kStageBytes) + row_group * kParts * kState + lane;
      if (kParts > 1 && tokens) {
        arithmetic_sync();
#pragma unroll
        for (int nb = 0; nb < kRowBlocks; ++nb) {
#pragma unroll
          for (int ch = 0; ch < kChunks; ++ch)
#pragma unroll
            for (int e = 0; e < 4; ++e) states[part * kState + ((nb * kChunks + ch) * 4 + e) * 32] = o[nb][ch][e];
          if (g == 0) {
            row_state[warp * 16 + 8 * nb + 2 * t] = make_float2(m[nb].x, l[nb].x);
            row_state[warp * 16 + 8 * nb + 2 * t + 1] = make_float2(m[nb].y, l[nb].y);
          }
        }
        arithmetic_sync();
      }
      const bool whole = seg_tiles == r.tiles;
      const int slot = first_unit ? 0 : 1;
#pragma unroll
      for (int nb = 0; nb < kRowBlocks; ++nb) {
        float acc[kMine][4];
        float mm[2] = {m[nb].x, m[nb].y}, sum[2] = {l[nb].x, l[nb].y};
        if (kParts > 1 && tokens) {
          float2 others[2][kParts];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            mm[x] = -INFINITY;
            sum[x] = 0.f;
#pragma unroll
            for (int w = 0; w < kParts; ++w) {
              others[x][w] = row_state[(row_group * kParts + w) * 16 + 8 * nb + 2 * t + x];
              mm[x] = fmaxf(mm[x], others[x][w].x);
            }
          }
#pragma unroll
          for (int ch = 0; ch < kMine; ++ch) acc[ch][0] = acc[ch][1] = acc[ch][2] = acc[ch][3] = 0.f;
#pragma unroll
          for (int w = 0; w < kParts; ++w) {
            float f[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float h = others[x][w].x == -INFINITY ? 0.f : ex2_approx(0.5f * (others[x][w].x - mm[x]));
              f[x] = h * h;
              sum[x] = fmaf(others[x][w].y * h, h, sum[x]);
            }
#pragma unroll
            for (int ch = 0; ch < kMine; ++ch)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[ch][e] = fmaf(states[w * kState + ((nb * kChunks + part * kMine + ch) * 4 + e) * 32], f[e & 1], acc[ch][e]);
          }
        } else {
#pragma unroll
          for (int ch = 0; ch < kMine; ++ch)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[ch][e] = o[nb][ch][e];  // all of them, or zeros
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int row = my_row0 + 8 * nb + 2 * t + x;
          if (row >= row0 + n_rows) continue;
          const float inv = sum[x] > 0.f ? kSumUnit / sum[x] : sum[x];  // 0 stays 0, NaN stays NaN
          const float lse2 = sum[x] == 0.f ? -INFINITY : mm[x] - kBias - log2f(kSumUnit) + log2f(sum[x]);
          const int dim0 = part * kMine * 16 + 2 * g;
          if (whole) {
            const int i = row / p.group, hq = head * p.group + row - i * p.group;
            uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + (r.q0 + i) * p.o_row + hq * p.o_head + dim0);
#pragma unroll
            for (int ch = 0; ch < kMine; ++ch) {
              const float even = acc[ch][x] * inv, odd = acc[ch][2 + x] * inv;
              dst[8 * ch] = p.f16 ? pack_f16x2(even, odd) : pack_bf16x2(even, odd);
            }
            if (g == 0 && part == 0) p.lse[static_cast<int64_t>(hq) * p.total_q + r.q0 + i] = sum[x] > 0.f ? lse2 * 0.6931471805599453f : INFINITY;
          } else {
            const int64_t at = kCluster ? row - row0 : (2 * static_cast<int64_t>(blockIdx.x) + slot) * p.rows + row - row0;
            float* dst = (kCluster ? own_part : p.part_o) + at * kD + dim0;
#pragma unroll
            for (int ch = 0; ch < kMine; ++ch) *reinterpret_cast<float2*>(dst + 16 * ch) = make_float2(acc[ch][x] * inv, acc[ch][2 + x] * inv);
            if (g == 0 && part == 0) (kCluster ? own_lse : p.part_lse)[at] = lse2;
          }
        }
      }
      if (tokens) {
        fence_proxy_async_smem();  // what was handed over goes before the copy into the same place
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + 8 * st);
        ++step;
      }
      // begun here, where the share ends; ended by the CTA whose share holds its last tile
      if (tile == 0 && !whole) left = {share.cta_behind(blockIdx.x, r.tiles - seg_tiles - 1), slot, head, row0, n_rows, r.q0};
      tile = 0;
      first_unit = false;
      r = next_r;
      unit = next;
    }
  }
  if constexpr (kCluster) {
    cluster_sync();  // every CTA's part is written
    const Request& r = share.request;
    const int row0 = share.unit / p.heads_kv * p.rows, head = share.unit - share.unit / p.heads_kv * p.heads_kv;
    const int rank = blockIdx.x - blockIdx.x / p.cluster * p.cluster;
    if (share.unit < r.units && share.each < r.tiles) {  // (a single CTA's unit is done)
      const int n_rows = min(p.rows, r.rows_q * p.group - row0);
      for (int rr = rank + p.cluster * warp; rr < n_rows; rr += p.cluster * (kWarps + 2)) {
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
    cluster_sync();  // the others have read this CTA's
  } else {
    if (threadIdx.x == 0) p.shared_units[blockIdx.x] = left;
  }
  if (lane == 0) drain_after_abort(abort_flag);
  if (threadIdx.x == 0 && *abort_flag != 0) atomicExch(p.status, static_cast<uint32_t>(SDPA_B200_DEVICE_TIMEOUT));
}

// Merges the parts of the units that several CTAs worked on: block (i, j) those of the unit that CTA i began, rows 4j to 4j + 3, a warp each.
// What it takes is a chain of latencies, behind a call whose own work is a few of them: with the first eight parts asked for beside their weights instead of
// behind them 4 drafted tokens of 16 requests take 22.0 us and not 23.2, one token of 1000 8.4 and not 8.75. Sixteen took registers and were slower elsewhere.
template <int kD>
__global__ void __launch_bounds__(128) cache_merge_kernel(const StreamParams p) {
  constexpr int kPer = kD / 32, kEarly = 8;
  const int lane = threadIdx.x & 31, rr = blockIdx.y * 4 + (threadIdx.x >> 5), first = blockIdx.x;
  wait_for_previous_grid();
  launch_dependents();
  const SharedUnit u = p.shared_units[first];
  if (u.last < 0 || rr >= u.rows) return;
  auto part = [&](int c) { return (2 * static_cast<int64_t>(c) + (c == first ? u.slot : 0)) * p.rows + rr; };
  float top = -INFINITY, sum = 0.f, acc[kPer];
  bool nan = false;
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
  for (int base = first; base <= u.last; base += 32) {
    const int n = min(32, u.last - base + 1);
    const float x = lane < n ? p.part_lse[part(base + lane)] : -INFINITY;
    auto load = [&](int j, float (&v)[kPer]) {
      const float* src = p.part_o + part(base + j) * kD + kPer * lane;
      if constexpr (kPer == 4) {
        const float4 q = *reinterpret_cast<const float4*>(src);
        v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
      } else {
        const float2 q = *reinterpret_cast<const float2*>(src);
        v[0] = q.x, v[1] = q.y;
      }
    };
    float early[kEarly][kPer];  // asked for beside their weights
#pragma unroll
    for (int j = 0; j < kEarly; ++j) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) early[j][e] = 0.f;
      if (j < n) load(j, early[j]);
    }
    nan = nan || __any_sync(0xffffffffu, isnan(x));
    float mn = x;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, d));
    mn = fmaxf(mn, top);
    const float a = top == -INFINITY ? 0.f : exp2f(top - mn), w = x == -INFINITY ? 0.f : exp2f(x - mn);
    top = mn;
    float s = w;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
    sum = sum * a + s;
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] *= a;
#pragma unroll
    for (int j = 0; j < kEarly; ++j) {
      const float wj = __shfl_sync(0xffffffffu, w, j);
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] = fmaf(wj, early[j][e], acc[e]);
    }
#pragma unroll 8
    for (int j = kEarly; j < n; ++j) {
      const float wj = __shfl_sync(0xffffffffu, w, j);
      float v[kPer];
      load(j, v);
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] = fmaf(wj, v[e], acc[e]);
    }
  }
  write_row<kPer>(p, u.q0, u.head, u.row0 + rr, lane, acc, sum, top, nan);
}

// ---- many rows: the codes of all requests as packed 16-bit K and V
struct GatherParams {
  const uint8_t* cache[2];
  const float* scale[2];
  uint16_t* out[2];
  const int32_t* cu_q;
  int32_t* cu;  // offsets of queries [2 * batch + 1], then of keys
  int64_t block[2], head[2], row[2];
  const int32_t* block_table;
  const int32_t* seq_lens;
  int64_t table_stride;
  int batch, total_q, heads, max_blocks, num_blocks, shift;
  int max_k, max_len;  // tokens that a request has here at most, that a table's row holds
};

constexpr int kGatherTokens = 32;  // of a block; with 64 the call of 512 rows took 137 us, with 32 135, with 64 and stores that left gaps to be filled by the next ones 140
constexpr int64_t kMostGatheredBytes = int64_t(4) << 30;  // of the 16-bit copies in the workspace
constexpr int kKeyTile = 128;  // keys that the prefill kernel reads at a time, from a sequence's start

__host__ __device__ __forceinline__ int64_t padded_keys(int64_t n) { return (n + kKeyTile - 1) / kKeyTile * kKeyTile; }

// two elements in 16 bits, the largest number of the type where they are beyond it: a code is rounded, and the elements 65504 of f16 or 3.39e38 of bf16 come back as
// 2^16 or 2^128. NaN stays.
template <bool kF16>
__device__ __forceinline__ uint32_t pack_16x2_finite(float lo, float hi) {
  uint32_t r;
  if constexpr (kF16) asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Block (i, h, b): tokens 32i to 32i + 31 of request b, kv head h, keys and values. The prefill kernel's last tile of a sequence goes on into the rows behind it,
// where a weight of 0 would meet another request's NaN, or whatever the workspace held. So every request's rows are filled up to a whole tile with zeros, and these
// stand in the list of sequences as one of their own, without queries. A request that is longer than its table has the most tokens here that any may have, which
// are no fewer than its rows, so that each of them sees the first; all are in a block that there is none of.
template <int kD, bool kInt8, bool kF16>
__global__ void __launch_bounds__(256) cache_gather_kernel(const GatherParams p) {
  __shared__ int sums[8];
  const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
  auto len_of = [&](int given) { return given > p.max_len ? p.max_k : min(max(given, 0), p.max_k); };
  const int given = p.seq_lens[b], len = len_of(given), padded = static_cast<int>(padded_keys(len));
  const int max_blocks = given > p.max_len ? 0 : p.max_blocks;
  int before = 0;
  for (int i = tid; i < b; i += 256) before += static_cast<int>(padded_keys(len_of(p.seq_lens[i])));
#pragma unroll
  for (int d = 1; d < 32; d *= 2) before += __shfl_xor_sync(0xffffffffu, before, d);
  if ((tid & 31) == 0) sums[tid >> 5] = before;
  __syncthreads();
  before = 0;
  for (int w = 0; w < 8; ++w) before += sums[w];
  if (blockIdx.x == 0 && h == 0 && tid == 0) {
    int32_t* cu_k = p.cu + 2 * p.batch + 1;
    auto offset = [&](int i) { return min(max(p.cu_q[i], 0), p.total_q); };  // the prefill kernel writes where they say
    p.cu[2 * b] = offset(b);
    p.cu[2 * b + 1] = offset(b + 1);
    cu_k[2 * b] = before;
    cu_k[2 * b + 1] = before + len;
    if (b == p.batch - 1) {
      p.cu[2 * p.batch] = offset(p.batch);
      cu_k[2 * p.batch] = before + padded;
    }
  }
  constexpr int kLanes = kD / 8, kTimes = kGatherTokens * kLanes / 256;  // eight codes of K and of V a thread and time: the stores of a warp leave no gaps
  static_assert(kTimes >= 1, "a block has threads to spare");
  const int tok0 = blockIdx.x * kGatherTokens + tid / kLanes, at = tid % kLanes * 8;
  int id[kTimes];
#pragma unroll
  for (int i = 0; i < kTimes; ++i) {
    const int tok = tok0 + i * (256 / kLanes), page = tok >> p.shift;
    id[i] = tok < len && page < max_blocks ? p.block_table[b * p.table_stride + page] : -1;
  }
  uint2 w[kTimes][2];
  float scale[kTimes][2];
#pragma unroll
  for (int i = 0; i < kTimes; ++i) {
    const int tok = tok0 + i * (256 / kLanes), place = tok & ((1 << p.shift) - 1);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      w[i][x] = make_uint2(0u, 0u);
      // a block outside the cache: its scores are NaN, for those who see them
      scale[i][x] = tok < len && x == 0 ? __int_as_float(0x7fffffff) : 0.f;
      if (id[i] < 0 || id[i] >= p.num_blocks) continue;
      w[i][x] = *reinterpret_cast<const uint2*>(p.cache[x] + id[i] * p.block[x] + h * p.head[x] + place * p.row[x] + at);
      scale[i][x] = p.scale[x][static_cast<int64_t>(id[i]) * p.heads + h];
    }
  }
#pragma unroll
  for (int i = 0; i < kTimes; ++i) {
    const int tok = tok0 + i * (256 / kLanes);
    if (tok >= padded) break;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      uint32_t f[4], c[2] = {w[i][x].x, w[i][x].y};
      const float own = fabsf(scale[i][x]) == INFINITY || (x == 1 && scale[i][x] < 0.f) ? __int_as_float(0x7fffffff) : scale[i][x];  // as on the other path
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t lo, hi;
        codes_to_f16<kInt8>(c[e], lo, hi);
        const float2 u = unpack_16x2<true>(lo), v = unpack_16x2<true>(hi);
        f[2 * e] = pack_16x2_finite<kF16>(u.x * own, u.y * own);
        f[2 * e + 1] = pack_16x2_finite<kF16>(v.x * own, v.y * own);
      }
      *reinterpret_cast<uint4*>(p.out[x] + ((static_cast<int64_t>(before) + tok) * p.heads + h) * kD + at) = make_uint4(f[0], f[1], f[2], f[3]);
    }
  }
}

// Tokens that a table's row holds
int table_tokens(const sdpa_b200_cache_params& p) { return static_cast<int>(std::min<int64_t>(static_cast<int64_t>(p.max_blocks) * p.block_size, INT32_MAX - 256)); }

// Tokens of the longest request among the 16-bit copies, no fewer than any has rows
int most_gathered(const sdpa_b200_cache_params& p) { return std::max(p.max_seqlen_k, p.max_seqlen_q); }

// Keys and values of one request among the 16-bit copies, at its longest; one more than fits where they do not
int64_t gathered_bytes(const sdpa_b200_cache_params& p) {
  const int64_t rows = padded_keys(most_gathered(p)) * p.heads_kv, row_bytes = 4 * p.head_dim;
  return rows <= kMostGatheredBytes / row_bytes ? rows * row_bytes : kMostGatheredBytes + 1;
}

// Requests that are gathered at a time. What they hold is not known here: by the bound on lengths, which may be the table's, the copies of a large batch would take more memory than
// the cache itself. 64 requests of 512 rows behind 32768 tokens, 32/8 heads of 128, in two launches of each kernel instead of one: 16.8 instead of 16.7 ms.
int gathered_at_once(const sdpa_b200_cache_params& p) {
  const int64_t most = std::min<int64_t>(kMostGatheredBytes / gathered_bytes(p), 32767), launches = (p.batch + most - 1) / most;
  return static_cast<int>((p.batch + launches - 1) / launches);  // launches of equal size
}

// Path 1 costs its units of 64 rows, path 2 the gathering of every kv head's tokens and the prefill kernel's waves of units of up to 256 rows of a query head, all per
// token in the cache. So the length does not decide, and in units of 64 rows a token's gathering is 0.9 and a wave 95 (head_dim 64: 150). Measured, 4 requests of 5000
// tokens, us, path 1 | 2: 32/8 heads of 128, 24 rows 58 | 86, 40 79 | 88, 56 99 | 88, 96 144 | 89; 16/16, 64 60 | 106, 128 101 | 107, 160 144 | 115; 64/8, 40 123 | 148,
// 64 188 | 150; 16/4 of 64, 64 36 | 63, 128 61 | 64, 160 73 | 81. 16 requests of 1000, 32/8 of 128, 40 76 | 78, 64 95 | 79.
bool streams(const sdpa_b200_cache_params& p) {
  const int64_t group = p.heads_q / p.heads_kv, batch = p.batch;
  if (p.cu_seqlens_q == nullptr || p.max_seqlen_q * group <= 64 || gathered_bytes(p) > kMostGatheredBytes) return true;
  // requests of equal rows, or of any: half a unit each is empty then
  const double units = p.total_q == batch * p.max_seqlen_q ? static_cast<double>(batch * ((p.max_seqlen_q * group + 63) / 64)) : p.total_q * group / 64.0 + 0.5 * batch;
  const int64_t blocks = p.heads_q * std::max<int64_t>(batch, (p.total_q + 255) / 256);
  return (units - 0.9 * batch) * p.heads_kv <= (p.head_dim == 64 ? 150.0 : 95.0) * static_cast<double>((blocks + 147) / 148);
}

int check_attention(const sdpa_b200_cache_params* p) {
  int st = check_cache(p, "cache_attention");
  if (st != SDPA_B200_OK) return st;
  if (p->batch <= 0 || p->total_q <= 0 || p->heads_q <= 0 || p->max_blocks <= 0 || p->table_stride < p->max_blocks) {
    set_error("cache_attention: batch, total_q, heads_q and max_blocks must be positive, a table row must hold max_blocks (got %d, %d, %d, %d, %lld)", p->batch,
              p->total_q, p->heads_q, p->max_blocks, static_cast<long long>(p->table_stride));
    return SDPA_B200_INVALID_ARG;
  }
  if (p->heads_q % p->heads_kv != 0) {
    set_error("Number of heads in key/value must divide number of heads in query (%d vs %d)", p->heads_kv, p->heads_q);
    return SDPA_B200_INVALID_ARG;
  }
  if (p->max_seqlen_q <= 0 || p->max_seqlen_k <= 0) {
    set_error("sequence lengths must be positive (max_seqlen_q %d, max_seqlen_k %d)", p->max_seqlen_q, p->max_seqlen_k);
    return SDPA_B200_INVALID_ARG;
  }
  if (p->cu_seqlens_q == nullptr && (p->total_q != p->batch || p->max_seqlen_q != 1)) {
    set_error("cache_attention: without cu_seqlens_q there is one row of q per request (got %d rows, %d requests, max_seqlen_q %d)", p->total_q, p->batch,
              p->max_seqlen_q);
    return SDPA_B200_INVALID_ARG;
  }
  if (!(p->softmax_scale > 0.f) || !(p->softmax_scale < 3.0e38f)) {
    set_error("softmax_scale must be positive and finite (got %g)", static_cast<double>(p->softmax_scale));
    return SDPA_B200_INVALID_ARG;
  }
  if (static_cast<int64_t>(p->heads_q) * p->max_seqlen_q > INT32_MAX / 2 || static_cast<int64_t>(p->total_q) * p->heads_q > INT32_MAX) {
    set_error("cache_attention: rows of q are counted in 32 bits");
    return SDPA_B200_INVALID_ARG;
  }
  const void* tensors[2] = {p->q, p->out};
  const int64_t strides[2][2] = {{p->q_row_stride, p->q_head_stride}, {p->o_row_stride, p->o_head_stride}};
  for (int i = 0; i < 2; ++i) {
    if (tensors[i] == nullptr || (reinterpret_cast<uintptr_t>(tensors[i]) & 15u) != 0) {
      set_error("cache_attention: %s must be a 16-byte aligned device pointer", i ? "out" : "q");
      return SDPA_B200_INVALID_ARG;
    }
    if ((p->total_q > 1 && (strides[i][0] <= 0 || strides[i][0] % 8 != 0)) || (p->heads_q > 1 && (strides[i][1] <= 0 || strides[i][1] % 8 != 0))) {
      set_error("cache_attention: %s needs row and head strides that are positive multiples of 8 elements (got %lld, %lld)", i ? "out" : "q",
                static_cast<long long>(strides[i][0]), static_cast<long long>(strides[i][1]));
      return SDPA_B200_INVALID_ARG;
    }
  }
  const void* words[4] = {p->lse, p->block_table, p->seq_lens, p->cu_seqlens_q};
  for (int i = 0; i < 4; ++i) {
    if ((words[i] == nullptr && i < 3) || (reinterpret_cast<uintptr_t>(words[i]) & 3u) != 0) {
      set_error("cache_attention: lse, block_table and seq_lens must be given, and 4-byte aligned as cu_seqlens_q");
      return SDPA_B200_INVALID_ARG;
    }
  }
  if ((reinterpret_cast<uintptr_t>(p->device_status) & 3u) != 0) {
    set_error("device_status must be 4-byte aligned");
    return SDPA_B200_INVALID_ARG;
  }
  return SDPA_B200_OK;
}

int unit_rows(const sdpa_b200_cache_params& p) {
  const int64_t rows = static_cast<int64_t>(p.max_seqlen_q) * (p.heads_q / p.heads_kv);
  return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}

size_t round_256(size_t n) { return (n + 255) / 256 * 256; }

// Where the units are few and short, a cluster of 2 to 8 CTAs takes each, the tiles in equal stretches, and merges its parts through distributed shared memory: no lengths to be
// summed up in front and no second kernel behind. That leaves SMs idle where units are of many lengths, so it is for up to eight tiles a CTA of the longest. Measured, shares of
// the list | clusters, one token each, 32/8 heads of 128, us: 1 request of 1000 8.6 | 6.1, of 4000 12.0 | 8.4, of 8000 17.4 | 11.5; 4 of 600 to 5000 15.2 | 10.1, of 8000
// 21.8 | 17.9; 8 of 300 to 1000 9.6 | 7.9, of 600 to 4000 14.3 | 13.0; 16 of 100 to 500 12.2 | 7.9, of 100 to 2000 13.9 | 12.4, of 2000 21.0 | 17.9. Beyond: 1 of 32000
// 24.2 | 31.0, 16 of 600 to 8000 28.0 | 34.4, 4 tokens of 16 of 300 to 9000 at head_dim 64 19.9 | 24.0.
int cluster_of(const sdpa_b200_cache_params& c, int rows, int64_t units, int tile_shift) {
  const int64_t tiles = (static_cast<int64_t>(c.max_seqlen_k) + (1 << tile_shift) - 1) >> tile_shift;
  if (rows > 16 || tiles < 2) return 0;
  int size = 8;
  while (size > 1 && (units * size > kMostClusterCtas || size / 2 >= tiles)) size /= 2;
  return size > 1 && tiles <= kTilesInCluster * size ? size : 0;
}

// What the list of tiles and its units depend on, of all requests; no device is asked
StreamParams list_of(const sdpa_b200_cache_params& c) {
  StreamParams p = {};
  p.block_table = c.block_table;
  p.seq_lens = c.seq_lens;
  p.cu_q = c.cu_seqlens_q;
  p.table_stride = c.table_stride;
  p.batch = c.batch;
  p.heads_q = c.heads_q;
  p.heads_kv = c.heads_kv;
  p.group = c.heads_q / c.heads_kv;
  p.total_q = c.total_q;
  p.max_rows = c.max_seqlen_q;
  p.max_blocks = c.max_blocks;
  p.rows = unit_rows(c);
  p.rows_shift = p.rows == 8 ? 3 : p.rows == 16 ? 4 : p.rows == 32 ? 5 : 6;
  p.tile_shift = c.head_dim == 64 ? 8 : 7;
  p.pause = p.rows == 64 ? 0 : kPause;
  p.max_len = table_tokens(c);
  return p;
}

// Requests [first, first + count)
int launch_stream(const sdpa_b200_cache_params& c, int first, int count, char* workspace, uint32_t* status, cudaStream_t stream) {
  const int sms = sm_count();
  if (sms <= 0 || sms > kMaxSms) {
    set_error("cache_attention: cannot use a device with %d SMs", sms);
    return SDPA_B200_NO_DEVICE;
  }
  StreamParams p = list_of(c);
  p.batch = count;
  p.block_table += first * p.table_stride;
  p.seq_lens += first;
  if (p.cu_q != nullptr) p.cu_q += first;
  p.first_q = first;
  p.q = static_cast<const uint16_t*>(c.q);
  p.out = static_cast<uint16_t*>(c.out);
  p.lse = c.lse;
  p.k_scale = c.k_scale;
  p.v_scale = c.v_scale;
  p.status = status;
  p.q_row = c.q_row_stride;
  p.q_head = c.q_head_stride;
  p.o_row = c.o_row_stride;
  p.o_head = c.o_head_stride;
  p.num_blocks = c.num_blocks;
  p.shift = block_shift(c.block_size);
  p.causal = c.is_causal;
  p.f16 = c.dtype == SDPA_B200_F16;
  p.scale_log2 = c.softmax_scale * 1.4426950408889634f;
  // a CTA per tile, up to one wave
  const int64_t units = static_cast<int64_t>(count) * c.heads_kv * ((static_cast<int64_t>(c.max_seqlen_q) * p.group + p.rows - 1) / p.rows);
  const int64_t tiles = units * ((static_cast<int64_t>(c.max_seqlen_k) + (1 << p.tile_shift) - 1) >> p.tile_shift);
  p.grid = static_cast<int>(tiles < kCtasPerSm * sms ? tiles : kCtasPerSm * sms);
  // a cluster for each unit
  p.units_each = static_cast<int>(units / count);
  p.cluster = cluster_of(c, p.rows, units, p.tile_shift);
  if (p.cluster > 0) p.grid = static_cast<int>(units) * p.cluster;
  const size_t rows = static_cast<size_t>(kCtasPerSm) * kMaxSms * 2 * p.rows;
  p.part_o = reinterpret_cast<float*>(workspace + kWorkspaceHeaderBytes);
  p.part_lse = p.part_o + rows * c.head_dim;
  p.shared_units = reinterpret_cast<SharedUnit*>(p.part_lse + rows);
  CUtensorMap tm_k, tm_v;
  int st = make_cache_tensor_map(&tm_k, c.k_cache, c.head_dim, c.block_size, c.heads_kv, c.num_blocks, c.k_row_stride, c.k_head_stride, c.k_block_stride, c.block_size);
  if (st != SDPA_B200_OK) return st;
  st = make_cache_tensor_map(&tm_v, c.v_cache, c.head_dim, c.block_size, c.heads_kv, c.num_blocks, c.v_row_stride, c.v_head_stride, c.v_block_stride, c.block_size);
  if (st != SDPA_B200_OK) return st;
  cudaError_t err = cudaSuccess;
  auto launch_as = [&](auto blocks_tag, auto rows_tag, auto dim_tag, auto int8_tag, auto cluster_tag) {
    constexpr bool kInt8 = decltype(int8_tag)::value, kCluster = decltype(cluster_tag)::value;
    constexpr int kRowBlocks = decltype(blocks_tag)::value, kRowWarps = decltype(rows_tag)::value, kD = decltype(dim_tag)::value;
    constexpr uint32_t kSmem = stream_smem_bytes<kRowBlocks, kRowWarps, kD>() + (kCluster ? 32 + 8 * kRowBlocks * (kD + 1) * 4 : 0);
    static_assert(kCtasPerSm * (kSmem + 1024) <= 228 * 1024, "two CTAs do not fit an SM");
    auto kernel = cache_stream_kernel<kRowBlocks, kRowWarps, kD, kInt8, kCluster>;
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (err == cudaSuccess)
      err = launch_behind(kernel, dim3(p.grid), kThreads, kSmem, stream, c.device_status != nullptr, kCluster ? p.cluster : 1, tm_k, tm_v, p);
  };
  auto launch = [&](auto blocks_tag, auto rows_tag, auto dim_tag, auto int8_tag) {
    if constexpr (decltype(rows_tag)::value == 1) {
      if (p.cluster > 0) return launch_as(blocks_tag, rows_tag, dim_tag, int8_tag, std::true_type{});
    }
    launch_as(blocks_tag, rows_tag, dim_tag, int8_tag, std::false_type{});
  };
  auto launch_code = [&](auto blocks_tag, auto rows_tag, auto dim_tag) {
    c.code == SDPA_B200_INT8 ? launch(blocks_tag, rows_tag, dim_tag, std::true_type{}) : launch(blocks_tag, rows_tag, dim_tag, std::false_type{});
  };
  auto launch_dim = [&](auto blocks_tag, auto rows_tag) {
    c.head_dim == 64 ? launch_code(blocks_tag, rows_tag, std::integral_constant<int, 64>{}) : launch_code(blocks_tag, rows_tag, std::integral_constant<int, 128>{});
  };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  if (p.rows == 8) launch_dim(One{}, One{});
  else if (p.rows == 16) launch_dim(Two{}, One{});
  else if (p.rows == 32) launch_dim(Two{}, Two{});
  else launch_dim(Two{}, std::integral_constant<int, 4>{});
  if (err != cudaSuccess) {
    set_error("cache_attention: launch failed: %s", cudaGetErrorString(err));
    return SDPA_B200_LAUNCH_FAILED;
  }
  count_launch();
  if (p.cluster > 0 || p.grid == 1 || c.max_seqlen_k <= 1 << p.tile_shift) return SDPA_B200_OK;  // no unit is shared, or merged already
  cudaLaunchConfig_t cfg = {};  // under this grid's tail, under stream capture too: what stands in front is a kernel of this call
  cfg.gridDim = dim3(p.grid - 1, p.rows / 4);
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  err = c.head_dim == 64 ? cudaLaunchKernelEx(&cfg, cache_merge_kernel<64>, p) : cudaLaunchKernelEx(&cfg, cache_merge_kernel<128>, p);
  if (err != cudaSuccess) {
    set_error("cache_attention merge: launch failed: %s", cudaGetErrorString(err));
    return SDPA_B200_LAUNCH_FAILED;
  }
  count_launch();
  return SDPA_B200_OK;
}

// Requests [first, first + count)
int launch_gathered(const sdpa_b200_cache_params& c, int first, int count, char* workspace, uint32_t* status, cudaStream_t stream) {
  // behind the header the prefill kernel's own one, then K, V and the offsets
  sdpa_b200_params f = {};
  GatherParams g;
  char* at = workspace + 2 * kWorkspaceHeaderBytes;
  const int64_t copies = count * gathered_bytes(c);
  g.out[0] = reinterpret_cast<uint16_t*>(at);
  g.out[1] = reinterpret_cast<uint16_t*>(at + copies / 2);
  g.cu = reinterpret_cast<int32_t*>(at + copies);
  g.cu_q = c.cu_seqlens_q + first;
  g.cache[0] = static_cast<const uint8_t*>(c.k_cache);
  g.cache[1] = static_cast<const uint8_t*>(c.v_cache);
  g.scale[0] = c.k_scale;
  g.scale[1] = c.v_scale;
  g.block[0] = c.k_block_stride, g.head[0] = c.k_head_stride, g.row[0] = c.k_row_stride;
  g.block[1] = c.v_block_stride, g.head[1] = c.v_head_stride, g.row[1] = c.v_row_stride;
  g.block_table = c.block_table + first * c.table_stride;
  g.seq_lens = c.seq_lens + first;
  g.table_stride = c.table_stride;
  g.batch = count;
  g.total_q = c.total_q;
  g.heads = c.heads_kv;
  g.max_blocks = c.max_blocks;
  g.num_blocks = c.num_blocks;
  g.shift = block_shift(c.block_size);
  g.max_k = most_gathered(c);
  g.max_len = table_tokens(c);
  const dim3 grid(static_cast<unsigned>(padded_keys(g.max_k) / kGatherTokens), c.heads_kv, count);
  const bool f16 = c.dtype == SDPA_B200_F16;
  auto launch = [&](auto dim, auto int8) {
    constexpr int kD = decltype(dim)::value;
    constexpr bool kInt8 = decltype(int8)::value;
    if (f16) cache_gather_kernel<kD, kInt8, true><<<grid, 256, 0, stream>>>(g);
    else cache_gather_kernel<kD, kInt8, false><<<grid, 256, 0, stream>>>(g);
  };
  auto launch_dim = [&](auto dim) { c.code == SDPA_B200_INT8 ? launch(dim, std::true_type{}) : launch(dim, std::false_type{}); };
  c.head_dim == 64 ? launch_dim(std::integral_constant<int, 64>{}) : launch_dim(std::integral_constant<int, 128>{});
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) {
    set_error("cache_attention gather: launch failed: %s", cudaGetErrorString(err));
    return SDPA_B200_LAUNCH_FAILED;
  }
  count_launch();
  f.q = c.q;
  f.k = g.out[0];
  f.v = g.out[1];
  f.out = c.out;
  f.lse = c.lse;
  f.cu_seqlens_q = g.cu;
  f.cu_seqlens_k = g.cu + 2 * count + 1;
  f.batch = 2 * count;
  f.heads_q = c.heads_q;
  f.heads_kv = c.heads_kv;
  f.head_dim = c.head_dim;
  f.max_seqlen_q = c.max_seqlen_q;
  f.max_seqlen_k = g.max_k;
  f.total_q = c.total_q;
  f.total_k = static_cast<int32_t>(count * padded_keys(g.max_k));
  f.q_row_stride = c.q_row_stride;
  f.q_head_stride = c.q_head_stride;
  f.o_row_stride = c.o_row_stride;
  f.o_head_stride = c.o_head_stride;
  f.k_row_stride = f.v_row_stride = static_cast<int64_t>(c.heads_kv) * c.head_dim;
  f.k_head_stride = f.v_head_stride = c.head_dim;
  f.softmax_scale = c.softmax_scale;
  f.is_causal = c.is_causal;
  f.dtype = c.dtype;
  f.kernel = SDPA_B200_KERNEL_PREFILL;
  f.device_status = status;
  const int st = validate_forward_args(&f);
  if (st != SDPA_B200_OK) return st;
  return launch_fwd_prefill(f, workspace + kWorkspaceHeaderBytes, stream);
}

size_t workspace_bytes_of(const sdpa_b200_cache_params& p) {
  if (!streams(p)) {
    const size_t n = gathered_at_once(p);
    return 2 * kWorkspaceHeaderBytes + n * gathered_bytes(p) + round_256((4 * n + 2) * 4);
  }
  const size_t ctas = static_cast<size_t>(kCtasPerSm) * kMaxSms;
  return kWorkspaceHeaderBytes + round_256(ctas * 2 * unit_rows(p) * (p.head_dim + 1) * 4 + ctas * sizeof(SharedUnit));
}

}  // namespace
}  // namespace sdpa_b200

extern "C" SDPA_B200_API int sdpa_b200_cache_attention_workspace_bytes(const sdpa_b200_cache_params* p, size_t* bytes) {
  using namespace sdpa_b200;
  if (bytes == nullptr) {
    set_error("bytes is NULL");
    return SDPA_B200_INVALID_ARG;
  }
  const int st = check_attention(p);
  if (st != SDPA_B200_OK) return st;
  *bytes = workspace_bytes_of(*p);
  return SDPA_B200_OK;
}

extern "C" SDPA_B200_API int sdpa_b200_cache_attention(const sdpa_b200_cache_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace sdpa_b200;
  int st = check_attention(p);
  if (st != SDPA_B200_OK) return st;
  const size_t need = workspace_bytes_of(*p);
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0 || workspace_bytes < need) {
    set_error("cache_attention: the workspace must be a device pointer aligned to 256 bytes, of %zu bytes (got %zu)", need, workspace_bytes);
    return SDPA_B200_INVALID_ARG;
  }
  if (streams(*p) && requests_at_once(list_of(*p)) == 0) {
    set_error("cache_attention: a request of %d rows of %d heads and the %lld tokens of its table is too long", p->max_seqlen_q, p->heads_q,
              static_cast<long long>(p->max_blocks) * p->block_size);
    return SDPA_B200_UNSUPPORTED;
  }
  if (!streams(*p) && p->heads_kv > 65535) {
    set_error("cache_attention: many rows per request come with up to 65535 heads of the cache (got %d)", p->heads_kv);
    return SDPA_B200_UNSUPPORTED;
  }
  st = check_device();
  if (st != SDPA_B200_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p->device_status == nullptr && cudaMemsetAsync(workspace, 0, kWorkspaceHeaderBytes, s) != cudaSuccess) {
    set_error("clearing the workspace header failed: %s", cudaGetErrorString(cudaGetLastError()));
    return SDPA_B200_LAUNCH_FAILED;
  }
  uint32_t* status = p->device_status != nullptr ? p->device_status : static_cast<uint32_t*>(workspace);
  const bool few_rows = streams(*p);
  const int at_once = few_rows ? requests_at_once(list_of(*p)) : gathered_at_once(*p);
  for (int64_t first = 0; first < p->batch && st == SDPA_B200_OK; first += at_once) {
    const int count = static_cast<int>(std::min<int64_t>(at_once, p->batch - first));
    st = (few_rows ? launch_stream : launch_gathered)(*p, static_cast<int>(first), count, static_cast<char*>(workspace), status, s);
  }
  return st;
}
