// Attention of few rows per request over the 4-bit paged cache: the kernel behind cache_attention.cu's list of tiles. No counterpart in the reference, which has no paged cache.
//
//   s_ij = scale * sum_g ks[j, g] <q_ig, kc_jg>,  out_id = sum_j softmax_j(s_i) * vs[j, g(d)] * vc_jd
//
// over groups g of 32 dimensions, each with a bf16 scale of its own for every token and kv head; codes are whole numbers from -8 to 7. Units, shares, ring of tiles, loading warps and
// the merge are those of the 8-bit kernel (cache_attention.cu); what differs is what a byte costs: with 4.5 bits an element, twice the products and conversions per byte that
// comes out of HBM. So:
// * Codes of K become f16 with one AND-XOR each two: the low bits of a 16-bit word are the f16 subnormal u * 2^-24, u = code + 8, of the even nibbles, those of the odd
//   ones 16 times that, for which Q is divided by 16. The 8 comes off in the accumulators, which begin with -8 * 2^-24 * sum of the group's q instead of 0: u is small, so
//   that the sums lose three of fp32's bits to it.
// * The scale of K goes onto the group's fp32 sums: 4 multiply-adds for each 32 x 16 codes a warp converts, where scaling the codes would take 8.
// * Codes of V become code * 2^-9 by one multiply-add each two more: sums over tens of thousands of tokens would lose too much to an offset. (Products of the weights with -8 in every step instead, off
//   the step's products, were no faster: 8 requests of 32768 78.1 us, with the multiply-adds 77.3.)
// * The scale of V is taken apart: a power of two 2^e, above the largest of a step's tokens, goes into the exponent of the softmax weight (as the 8-bit scale does), what is left, below 1 and exact
//   in f16, onto the weights, 2 multiplications for 32 x 16 codes. A group whose scale is 2^-14 of 2^e has its products' full 11 bits only where the weight is that much above the smallest
//   normal one; where tokens are further apart than 2^10, each has an e of its own, and the sums of the softmax are formed without them, as the 8-bit kernel does for scales far apart: 64 requests of 8192 161 us instead of
//   147. Tokens of zeros, which the store gives 2^-100, have no part in that: with one, every 16th or all of them 147 to 149 (162 when any of them sent its unit that way).
// * The plain way masks scores and takes their maximum in front of the row's factor. That needs a factor that is a normal number and scores below 2^20, which Q's largest elements and the
//   step's scales of K bound; other steps multiply first and take the maximum off before anything else, so that scores of any size are right.
// * The loading warps only issue copies, codes by TMA and scales by cp.async, and wait for nothing but room. A warp of the arithmetic brings the scales of V of its own tokens into these
//   forms, a token or two a lane, beside its products with K.
// Measured, one token per request, 32/8 heads of 128: 64 requests of 2048 to 32768 tokens, 1.34 GB: 327 us (312 to 330 by box and lengths), 4.1 TB/s, 62% of a copy's rate; 8 of 32768 78; one of 1000, in clusters, 7. Without
// the arithmetic the first takes 228: it is the length of a step's chain in each warp that bounds it, with the logic pipe at 53% and the tensor pipe at 22%, no pipe alone.
#include <type_traits>

#include "cache_stream.cuh"

namespace sdpa_b200 {
namespace {

constexpr float kBias = 14.f;      // weights are kept times 2^14: times the rest of V's scale they fit f16
// Exponents e of V's scales. Between these two, weights, sums and what they are multiplied by when their maximum moves fit 32 bits for all keys that count, 2^-26 of the largest or more: they
// are as far as 2^(20 + 80 + 26) apart. What is below the least (2^-100 is the smallest scale that the store kernel chooses) has smaller rests, down to 2^-24; a token without a scale has
// that exponent, so that no other falls behind it. From the first scale above the most on, a unit's steps go the other way.
constexpr int kLeastExponent = -80;
constexpr int kMostExponent = 20;
constexpr int kZeroField = 27;  // bf16's exponent of 2^-100, which the store gives zeros: such a token takes its step's exponent, whatever that is
constexpr int kPlainExponents = 10;  // e of a step's tokens up to that far below the largest: the rests of V's scales stay normal f16 numbers, or the groups' own distance makes them less
constexpr int kPlainScores = 20;     // the plain way is for scores below 2^20, of which a weight's exponent is told to 1/16: larger ones are rounded before their maximum is taken off, so that it becomes 0
constexpr float kLeastFactor = 0x1p-126f;  // a row's factor, where it is a normal number: a masked score times 0 would be NaN
constexpr float kMostFactor = 0x1p100f;

// Loading warps: one for K and one for V, or, where an SM has three CTAs and each of them more time for a tile, one for both
template <int kRowBlocks>
__host__ __device__ constexpr int loading_warps() { return stream4_ctas_per_sm(8 * kRowBlocks) > 2 ? 1 : 2; }
template <int kRowBlocks>
__host__ __device__ constexpr int threads() { return (kWarps + loading_warps<kRowBlocks>()) * 32; }
template <int kD>
__host__ __device__ constexpr int tile_tokens() { return kD == 64 ? 256 : 128; }
template <int kD>
__host__ __device__ constexpr int step_tokens() { return kD == 64 ? 64 : 32; }
template <int kD>
__host__ __device__ constexpr uint32_t stage_bytes() { return tile_tokens<kD>() * kD; }  // codes of K and of V
template <int kD>
__host__ __device__ constexpr uint32_t scale_bytes() { return tile_tokens<kD>() * (kD / 32) * 2 * 2; }  // their scales
// What a warp keeps of a step's scales of V, for two steps in turn: e of each token, the rests by pairs of tokens
template <int kD>
__host__ __device__ constexpr uint32_t step_scale_bytes() { return step_tokens<kD>() * (4 + kD / 32 * 2); }
// B fragments of Q: in registers where there is room; else in shared memory, with their sums (8 rows, head_dim 128: 332 us so, 339 from registers that spill, 64 requests of 2048 to 32768)
template <int kRowBlocks, int kD>
__host__ __device__ constexpr bool q_in_registers() { return kD == 64; }
template <int kRowBlocks, int kRowWarps, int kD>
__host__ __device__ constexpr uint32_t q_bytes() { return q_in_registers<kRowBlocks, kD>() ? 0 : kRowWarps * kRowBlocks * (kD / 32) * (512 + 64); }
template <int kRowBlocks, int kRowWarps, int kD, bool kCluster>
__host__ __device__ constexpr uint32_t smem_bytes(int stages) {
  return 1024 + stages * (stage_bytes<kD>() + scale_bytes<kD>() + 16) + 16 + kWarps * (2 * step_scale_bytes<kD>() + 8 * 8) + q_bytes<kRowBlocks, kRowWarps, kD>() +
         (kCluster ? 32 + 8 * kRowBlocks * (kD + 1) * 4 : 0);
}
// Tiles in a CTA's ring: what lets an SM's CTAs share its 228 KB
template <int kRowBlocks, int kRowWarps, int kD, bool kCluster>
__host__ __device__ constexpr int ring_stages() {
  int n = 5;
  while (stream4_ctas_per_sm(8 * kRowBlocks) * (smem_bytes<kRowBlocks, kRowWarps, kD, kCluster>(n) + 1024) > 228 * 1024) --n;
  return n;
}

// Eight codes as f16 pairs (n, n + 4), n = 0..3: the subnormals u * 2^-24 for even n, 16 times that for odd n, u = code + 8. `eights` are 0x00080008 and 0x00800080, in registers: with
// the mask as an immediate operand a pair is one instruction then.
__device__ __forceinline__ void codes_to_subnormal(uint32_t w, const uint32_t (&eights)[2], uint32_t (&x)[4]) {
#pragma unroll
  for (int n = 0; n < 4; ++n)  // (w & mask) ^ eights
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(x[n]) : "r"(n < 2 ? w : w >> 8), "r"(n & 1 ? 0x00f000f0u : 0x000f000fu), "r"(eights[n & 1]));
}
// The same as normal numbers, code * 2^-9. `parts`: 2^15 and 2^11, minus 8 * 2^-9
__device__ __forceinline__ void codes_to_numbers(uint32_t w, const uint32_t (&eights)[2], const uint32_t (&parts)[3], uint32_t (&x)[4]) {
  codes_to_subnormal(w, eights, x);
#pragma unroll
  for (int n = 0; n < 4; ++n) asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(x[n]) : "r"(parts[n & 1]), "r"(parts[2]));
}
// D = A B + C, C elsewhere than D
__device__ __forceinline__ void mma_16816_from(float (&d)[4], const float4& c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c.x), "f"(c.y), "f"(c.z), "f"(c.w));
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ void copy_16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// This thread's arrival, when its copies so far are there
__device__ __forceinline__ void arrive_behind_copies(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ const uint4 no_scales[1] = {{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u}};

// kRowBlocks: blocks of 8 rows of a warp. kRowWarps: groups of that many rows of a unit; the warps of a group share the tile's tokens.
template <int kRowBlocks, int kRowWarps, int kD, bool kCluster>
__global__ void __launch_bounds__(threads<kRowBlocks>(), stream4_ctas_per_sm(8 * kRowBlocks))
cache4_stream_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const StreamParams p) {
  constexpr int kLoaders = loading_warps<kRowBlocks>();
  constexpr int kGroups = kD / 32;
  constexpr int kChunks = kD / 16;                           // of 16 dimensions, an MMA each
  constexpr int kRowBytes = kD / 2;
  constexpr int kSt = ring_stages<kRowBlocks, kRowWarps, kD, kCluster>();
  constexpr bool kQInRegisters = q_in_registers<kRowBlocks, kD>();
  constexpr uint32_t kStageBytes = stage_bytes<kD>();
  constexpr int kParts = kWarps / kRowWarps;                 // of a tile's tokens
  constexpr int kTileTokens = tile_tokens<kD>(), kStepTokens = step_tokens<kD>(), kHalves = kStepTokens / 16;
  constexpr int kPartTokens = kTileTokens / kParts;
  constexpr int kRowsOfWarp = 8 * kRowBlocks;
  constexpr float kUnit = 0x1p9f;                            // what accumulators lack
  constexpr int kState = kChunks * 4 * 32;                   // floats of a warp's accumulators, of 8 rows
  static_assert(kWarps * kState * 4 <= kStageBytes, "the warps' states do not fit a tile's place");
  static_assert(kSt >= 3, "too few tiles under way");
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t ring = (raw_addr + 1023u) & ~1023u;
  uint8_t* ring_ptr = smem_raw + (ring - raw_addr);
  uint16_t* tile_scales = reinterpret_cast<uint16_t*>(ring_ptr + kSt * kStageBytes);     // [stage][K, V][token][group]
  float* v_tokens = reinterpret_cast<float*>(tile_scales + kSt * 2 * kTileTokens * kGroups);  // [warp][step in turn][token]: e of its scales, where a step has several
  uint32_t* v_rests = reinterpret_cast<uint32_t*>(v_tokens + kWarps * 2 * kStepTokens);  // [warp][step in turn][pair of tokens][group]: f16 scales over 2^e
  float2* row_state = reinterpret_cast<float2*>(v_rests + kWarps * kStepTokens * kGroups);  // [warp][row of 8]: maximum and sum
  uint4* q_state = reinterpret_cast<uint4*>(row_state + kWarps * 8);                      // [row group][block of 8 rows][group][lane]: B fragments
  constexpr int kQWords = kQInRegisters ? 0 : kRowWarps * kRowBlocks * kGroups * 32;
  float4* q_sums = reinterpret_cast<float4*>(q_state + kQWords);                           // [row group][block of 8 rows][group][t]: twice those of two rows
  const uint32_t full = smem_u32(q_sums + kQWords / 8), empty = full + 8 * kSt;
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(reinterpret_cast<uint64_t*>(q_sums + kQWords / 8) + 2 * kSt);

  // kCluster: this CTA's part of the unit
  float* own_part = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(abort_flag) + 4 + 15) & ~static_cast<uintptr_t>(15));  // [row][dimension]
  float* own_lse = own_part + kRowsOfWarp * kD;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (kCluster && threadIdx.x < kRowsOfWarp) own_lse[threadIdx.x] = -INFINITY;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSt; ++i) {
      mbar_init(full + 8 * i, 32 * kLoaders);  // every lane of the loading warps, when its scales are there
      mbar_init(empty + 8 * i, kWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kWarps && elect_one()) tma_prefetch_desc(&tm_k);
  if (warp == kWarps + kLoaders - 1 && elect_one()) tma_prefetch_desc(&tm_v);
  __syncthreads();
  wait_for_previous_grid();
  if (threadIdx.x == 0) launch_dependents();  // behind the wait: the merge kernel's blocks wait for this grid only
  const Share share = kCluster ? share_in_cluster(p, blockIdx.x) : share_of(p, blockIdx.x, lane);
  if (share.places > 0 && warp >= kWarps) {
    // ================================================================ the loading warps
    // Lane i has page 32 * group + i of a unit: its block number (num_blocks: none in the cache, behind which the copy finds zeros; -1: no such page). Three groups are under
    // way: the one that tiles are copied from, the next, and the one behind.
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
    Place cur, nxt, far;
    cur.r = share.request;
    cur.unit = share.unit;
    cur.head = cur.unit % p.heads_kv;
    int tile = share.tile;
    cur.group = ((tile * kTileTokens) >> p.shift) >> 5;
    nxt = far = cur;
    int id = block_at(cur), next_id = -1, far_id = -1;
    // Scales are copied 16 bytes at a time, of one page: a lane's copies of a tile, and where they are in a page. The rest is kept in a form in which a tile costs few instructions: this
    // warp's time for a tile bounds the call where the arithmetic does not.
    constexpr int kTokensAtOnce = 8 / kGroups, kCopies = kTileTokens / kTokensAtOnce / 32;
    const int64_t block_scales = (static_cast<int64_t>(p.heads_kv) << p.shift) * kGroups;
    const bool has_k = warp == kWarps, has_v = warp == kWarps + kLoaders - 1;
    const uint16_t *k_scales[kCopies], *v_scales[kCopies];  // those of block 0, for the unit's head
    int unit_pages;
    bool some_missing;  // among the group's blocks
    auto enter = [&]() {
      unit_pages = static_cast<int>((static_cast<int64_t>(cur.r.len) + (1 << p.shift) - 1) >> p.shift);
      some_missing = __any_sync(0xffffffffu, id == p.num_blocks);
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const int tok = (lane + 32 * i) * kTokensAtOnce;
        const int64_t at = ((static_cast<int64_t>(cur.head) << p.shift) + (tok & ((1 << p.shift) - 1))) * kGroups;
        k_scales[i] = static_cast<const uint16_t*>(p.k_scale) + at;
        v_scales[i] = static_cast<const uint16_t*>(p.v_scale) + at;
      }
    };
    auto next_group = [&]() {
      cur = nxt, id = next_id;
      nxt = far, next_id = far_id;
      advance(far);
      far_id = block_at(far);
      enter();
    };
    const int pages = kTileTokens >> p.shift;  // of a tile
    const uint32_t page_bytes = static_cast<uint32_t>(kRowBytes) << p.shift;
    bool ok = true, first = true, filled = false;
    uint32_t st = 0, phase = 1;  // the ring's next place; what is waited for there once it has been round
    enter();
    for (int places = share.places; places > 0;) {
      const int page0 = (tile * kTileTokens) >> p.shift;
      if (page0 >> 5 != cur.group) next_group();  // the unit goes on in its next group
      if (tile * kTileTokens < cur.r.len) {
        const uint32_t bar = full + 8 * st, dst = ring + st * kStageBytes;
        const int n = min(pages, unit_pages - page0);
        int blocks[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) blocks[e] = __shfl_sync(0xffffffffu, id, (page0 + e) & 31);
        if (filled) {
          if (ok) ok = mbar_wait(empty + 8 * st, phase, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        if (elect_one()) {
          mbar_expect_tx(bar, (kLoaders == 1 ? 2 : 1) * n * page_bytes);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (e >= n) break;
            if (has_k) tma_load_4d(dst + e * page_bytes, &tm_k, bar, 0, 0, cur.head, blocks[e]);
            if (has_v) tma_load_4d(dst + kTileTokens * kRowBytes + e * page_bytes, &tm_v, bar, 0, 0, cur.head, blocks[e]);
          }
        }
#pragma unroll 1
        for (int i = 4; i < n; i += 4) {
#pragma unroll
          for (int e = 0; e < 4; ++e) blocks[e] = __shfl_sync(0xffffffffu, id, (page0 + i + e) & 31);
          if (elect_one()) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (i + e >= n) break;
              if (has_k) tma_load_4d(dst + (i + e) * page_bytes, &tm_k, bar, 0, 0, cur.head, blocks[e]);
              if (has_v) tma_load_4d(dst + kTileTokens * kRowBytes + (i + e) * page_bytes, &tm_v, bar, 0, 0, cur.head, blocks[e]);
            }
          }
        }
        // those of a block that is not there are NaN, those behind the last page stay what they are
        const uint32_t scale_dst = smem_u32(tile_scales) + st * (2 * kTileTokens * kGroups * 2) + 16 * lane;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const int page = ((lane + 32 * i) * kTokensAtOnce) >> p.shift, block = __shfl_sync(0xffffffffu, id, (page0 + page) & 31);
          const int64_t at = block * block_scales;
          const void *from_k = k_scales[i] + at, *from_v = v_scales[i] + at;
          if (some_missing && block == p.num_blocks) from_k = from_v = no_scales;
          if (page < n) {
            if (has_k) copy_16_async(scale_dst + 32 * 16 * i, from_k);
            if (has_v) copy_16_async(scale_dst + kTileTokens * kGroups * 2 + 32 * 16 * i, from_v);
          }
        }
        arrive_behind_copies(bar);
        if (++st == kSt) {
          st = 0;
          phase ^= 1;
          filled = true;
        }
      }
      if (first) {  // the first copies are under way
        advance(nxt);
        next_id = block_at(nxt);
        far = nxt;
        advance(far);
        far_id = block_at(far);
        first = false;
      }
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
    auto chunk_at = [&](int row, int chunk) -> uint32_t {  // byte offset of a 16-byte chunk (32 dimensions) of a row in a swizzled tile
      if constexpr (kD == 128) return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
      return row * 32 + ((chunk ^ ((row >> 2) & 1)) << 4);
    };
    bool ok = true;
    uint32_t st = 0, phase = 0;  // the ring's next place, its barrier's parity
    auto next_place = [&]() {
      if (++st == kSt) st = 0, phase ^= 1;
    };
    int turn = 0;  // of the places for a step's scales
    const uint32_t none = *abort_flag & 0x40000000u;  // 0, which the compiler does not know: so that these stay in registers
    const uint32_t eights[2] = {0x00080008u | none, 0x00800080u | none};
    const uint32_t parts[3] = {0x78007800u | none, 0x68006800u | none, 0xa400a400u | none};
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
      bool far_apart = false;
      int step_e = 0;  // of V's scales, of a step that goes the plain way
      // ---- this lane's row of Q as B fragments, row g of every 8: elements as f16. Thread t has dimensions 8t..8t+7 of every 32: pairs (n, n + 4), those of odd n over 16
      uint4 qb[kRowBlocks][kQInRegisters ? kGroups : 1];
      float4 qs[kRowBlocks][kQInRegisters ? kGroups : 1];  // of rows 2t, 2t + 1, 2t, 2t + 1: -8 times what the group's elements add up to, in the products' unit
      uint4* my_q = q_state + row_group * kRowBlocks * kGroups * 32 + lane;
      float4* my_sums = q_sums + row_group * kRowBlocks * kGroups * 4;
      float2 factor[kRowBlocks];  // of rows 2t, 2t + 1, with the softmax scale and the 2^24 that the products lack
      int2 limit[kRowBlocks];     // how many tokens they see
      float least = INFINITY, most = 0.f;  // factor of the warp's rows
#pragma unroll
      for (int nb = 0; nb < kRowBlocks; ++nb) {
        const int row = my_row0 + 8 * nb + g, i = row / p.group;
        const bool have = row < row0 + n_rows;
        const uint16_t* src = p.q + (r.q0 + i) * p.q_row + (head * p.group + row - i * p.group) * p.q_head + 8 * t;
        uint4 w[kGroups];
#pragma unroll
        for (int k = 0; k < kGroups; ++k) w[k] = have ? *reinterpret_cast<const uint4*>(src + 32 * k) : make_uint4(0u, 0u, 0u, 0u);
        auto floats = [&](const uint4& q, float (&x)[8]) {
          const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = p.f16 ? unpack_16x2<true>(words[e]) : unpack_16x2<false>(words[e]);
            x[2 * e] = f.x, x[2 * e + 1] = f.y;
          }
        };
        float largest = 0.f;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
          float x[8];
          floats(w[k], x);
#pragma unroll
          for (int e = 0; e < 8; ++e) largest = fmaxf(largest, fabsf(x[e]));
        }
        largest = quad_max(largest);
        const int e2 = min(max(static_cast<int>(__float_as_uint(largest) >> 23) - 127, -100), 127);
        const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 - e2) << 23);
        const float down = fminf(p.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - 14 + e2) << 23), 0x1.fffffep127f);
        least = fminf(least, down);
        most = fmaxf(most, down);
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
          float x[8];
          floats(w[k], x);
          const float odd = up * 0.0625f;
          const uint4 packed = make_uint4(pack_f16x2(x[0] * up, x[4] * up), pack_f16x2(x[1] * odd, x[5] * odd), pack_f16x2(x[2] * up, x[6] * up),
                                          pack_f16x2(x[3] * odd, x[7] * odd));
          const float2 a = unpack_16x2<true>(packed.x), b = unpack_16x2<true>(packed.y), c = unpack_16x2<true>(packed.z), d = unpack_16x2<true>(packed.w);
          float sum = (a.x + a.y + c.x + c.y) + 16.f * (b.x + b.y + d.x + d.y);
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          sum *= -0x1p-21f;
          const float2 sums = make_float2(__shfl_sync(0xffffffffu, sum, 8 * t), __shfl_sync(0xffffffffu, sum, 8 * t + 4));
          if constexpr (kQInRegisters) {
            qb[nb][k] = packed;
            qs[nb][k] = make_float4(sums.x, sums.y, sums.x, sums.y);
          } else if (part == 0) {
            my_q[(nb * kGroups + k) * 32] = packed;
            if (g == 0) my_sums[(nb * kGroups + k) * 4 + t] = make_float4(sums.x, sums.y, sums.x, sums.y);
          }
        }
        const int sees = p.causal ? min(r.len, i + 1 + r.in_front) : r.len;
        factor[nb] = make_float2(__shfl_sync(0xffffffffu, down, 8 * t), __shfl_sync(0xffffffffu, down, 8 * t + 4));
        limit[nb] = make_int2(__shfl_sync(0xffffffffu, sees, 8 * t), __shfl_sync(0xffffffffu, sees, 8 * t + 4));
      }
      // numbers that are not negative are ordered as integers
      least = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(least)));
      most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
      const bool huge = most > kMostFactor * 0x1p-24f;  // no room for the 2^24: the scores take it
      // Scales of K (bf16 bits) from which on the plain way is left: |score| is at most kGroups * K's scale * 2^(exponent of the largest factor, 24 more, + 1) / 2. 0: always
      const int most_field = static_cast<int>(__float_as_uint(most) >> 23) + 24;
      uint32_t k_limit = static_cast<uint32_t>(min(127 + kPlainScores + 127 - (kGroups == 4 ? 2 : 1) - most_field, 255)) << 7;
      if (huge || least * 0x1p24f < kLeastFactor) k_limit = 0u;
      if (!huge) {
#pragma unroll
        for (int nb = 0; nb < kRowBlocks; ++nb) factor[nb] = make_float2(factor[nb].x * 0x1p24f, factor[nb].y * 0x1p24f);
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

      float o[kRowBlocks][kChunks][4];  // [2c + j]: dimensions 32c + 4g + 2j, the same, the next, the next; rows 2t, 2t + 1, 2t, 2t + 1
      float2 m[kRowBlocks], l[kRowBlocks];  // running maximum of score + e; this thread's share of the sums, in units of kSumUnit
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
        if (ok) ok = mbar_wait(full + 8 * st, phase, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        __syncwarp();
        // ---- the scales of a step: a lane has one token, or two with half as many groups. Whether the step goes the plain way: V's scales are taken apart by one 2^e for all of its tokens
        auto take_scales = [&](int c) {
          const int in_tile = part * kPartTokens + c;
          constexpr int kOfLane = kStepTokens / 32, kWords = 2 / kOfLane;  // words of a token
          const uint16_t* src = tile_scales + (2 * st * kTileTokens + in_tile + kOfLane * lane) * kGroups;
          const uint2 raw_k = *reinterpret_cast<const uint2*>(src), raw_v = *reinterpret_cast<const uint2*>(src + kTileTokens * kGroups);
          uint32_t words[2] = {raw_v.x, raw_v.y}, top[kOfLane];  // top: a token's largest scale
          bool bad[kOfLane];
          int lowest = 1 << 16, highest = 0;                      // exponent fields of the lane's; lowest -1: not the plain way
#pragma unroll
          for (int x = 0; x < kOfLane; ++x) {
            const bool there = tile_tok + in_tile + kOfLane * lane + x < r.len;
            uint32_t of_k = kOfLane == 1 ? __vmaxu2(raw_k.x & 0x7fff7fffu, raw_k.y & 0x7fff7fffu) : (x ? raw_k.y : raw_k.x) & 0x7fff7fffu;
            top[x] = 0u;
#pragma unroll
            for (int e = 0; e < kWords; ++e) {
              uint32_t& w = words[kOfLane == 1 ? e : x];
              if (!there) w = 0u;
              top[x] = __vmaxu2(top[x], w & 0x7fff7fffu);
            }
            of_k = there ? max(of_k & 0xffffu, of_k >> 16) : 0u;
            top[x] = max(top[x] & 0xffffu, top[x] >> 16);
            bad[x] = max(of_k, top[x]) >= 0x7f80u;  // of K or of V: who sees the token is NaN
            const int of_token = static_cast<int>(top[x] >> 7);
            if (!bad[x]) highest = max(highest, of_token);
            if (of_token > kZeroField) lowest = min(lowest, of_token);
            if (bad[x] || of_k >= k_limit) lowest = -1;
          }
          const int field = __reduce_max_sync(0xffffffffu, highest);
          const bool plain = __all_sync(0xffffffffu, lowest >= max(field - kPlainExponents, 0)) && field <= 126 + kMostExponent && !far_apart;
          float* tokens = v_tokens + (2 * warp + turn) * kStepTokens + kOfLane * lane;
          uint32_t* rests = v_rests + (2 * warp + turn) * (kStepTokens / 2) * kGroups;
          uint32_t rest[2];
          auto rest_of = [&](uint32_t w, float down) { return pack_f16x2(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xffff0000u) * down); };
          if (plain) {
            step_e = max(field - 126, kLeastExponent);
            const float down = __uint_as_float(static_cast<uint32_t>(127 - step_e) << 23);  // 2^-e
            rest[0] = rest_of(words[0], down);
            rest[1] = rest_of(words[1], down);
          } else {
            bool is_far = false;
#pragma unroll
            for (int x = 0; x < kOfLane; ++x) {
              const int e2 = bad[x] ? 0 : min(max(static_cast<int>(top[x] >> 7) - 126, kLeastExponent), 126);
              is_far = is_far || e2 > kMostExponent;
              const float down = __uint_as_float(static_cast<uint32_t>(127 - e2) << 23);
              tokens[x] = bad[x] ? __int_as_float(0x7fffffff) : static_cast<float>(e2);
#pragma unroll
              for (int e = 0; e < kWords; ++e) rest[kOfLane == 1 ? e : x] = bad[x] ? 0u : rest_of(words[kOfLane == 1 ? e : x], down);
            }
            far_apart = __any_sync(0xffffffffu, is_far) || far_apart;
          }
          if constexpr (kOfLane == 1) {
            // lanes of a pair of tokens: the even one has groups 0 and 1 of both, the odd one 2 and 3
            const uint32_t other = __shfl_xor_sync(0xffffffffu, lane & 1 ? rest[0] : rest[1], 1);
            rest[0] = lane & 1 ? other : rest[0], rest[1] = lane & 1 ? rest[1] : other;
          }
          *reinterpret_cast<uint2*>(rests + 2 * lane) = make_uint2(__byte_perm(rest[0], rest[1], 0x5410), __byte_perm(rest[0], rest[1], 0x7632));
          __syncwarp();
          return plain;
        };
        auto work_on = [&](int c) {
          const int in_tile = part * kPartTokens + c, tok = tile_tok + in_tile;
          // ---- S^T = K Q^T, 16 tokens and 32 dimensions at a time
          // s: tokens g, g, g + 8, g + 8 of each half, rows 2t, 2t + 1, 2t, 2t + 1
          const uint32_t k_smem = ring + st * kStageBytes + in_tile * kRowBytes;
          const uint16_t* ks = tile_scales + (2 * st * kTileTokens + in_tile + g) * kGroups;
          float s[kRowBlocks][kHalves][4];
#pragma unroll
          for (int ch = 0; ch < kGroups; ch += 2) {
            uint4 q[2][kRowBlocks];
            float4 begin[2][kRowBlocks];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int nb = 0; nb < kRowBlocks; ++nb) {
                if constexpr (kQInRegisters) {
                  q[e][nb] = qb[nb][ch + e];
                  begin[e][nb] = qs[nb][ch + e];
                } else {
                  q[e][nb] = my_q[(nb * kGroups + ch + e) * 32];
                  begin[e][nb] = my_sums[(nb * kGroups + ch + e) * 4 + t];
                }
              }
#pragma unroll
            for (int half = 0; half < kHalves; ++half) {
              uint32_t kf[4];  // tokens 0-7 and 8-15 of a group, the same of the next
              ldmatrix_x4(k_smem + chunk_at(half * 16 + (mat & 1) * 8 + mrow, ch + (mat >> 1)), kf);
              const uint32_t near = *reinterpret_cast<const uint32_t*>(ks + half * 16 * kGroups + ch), behind = *reinterpret_cast<const uint32_t*>(ks + (half * 16 + 8) * kGroups + ch);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                uint32_t x[4], y[4];
                codes_to_subnormal(kf[2 * e], eights, x);
                codes_to_subnormal(kf[2 * e + 1], eights, y);
                const float kg = __uint_as_float(e ? near & 0xffff0000u : near << 16), kg8 = __uint_as_float(e ? behind & 0xffff0000u : behind << 16);
#pragma unroll
                for (int nb = 0; nb < kRowBlocks; ++nb) {
                  float a[4];
                  mma_16816_from(a, begin[e][nb], x[0], y[0], x[1], y[1], q[e][nb].x, q[e][nb].y);
                  mma_16816<true>(a, x[2], y[2], x[3], y[3], q[e][nb].z, q[e][nb].w);
                  if (ch + e == 0) {
                    s[nb][half][0] = a[0] * kg, s[nb][half][1] = a[1] * kg, s[nb][half][2] = a[2] * kg8, s[nb][half][3] = a[3] * kg8;
                  } else {
                    s[nb][half][0] = fmaf(a[0], kg, s[nb][half][0]), s[nb][half][1] = fmaf(a[1], kg, s[nb][half][1]);
                    s[nb][half][2] = fmaf(a[2], kg8, s[nb][half][2]), s[nb][half][3] = fmaf(a[3], kg8, s[nb][half][3]);
                  }
                }
              }
            }
          }
          const bool plain = take_scales(c);  // beside the products: neither waits for the other
          uint32_t pb[kRowBlocks][kHalves][2];  // weights as B fragments: tokens 2t, 2t + 1 (and 8 behind) of each half, row g
          bool moved = false;
          float2 a[kRowBlocks];
          auto weigh = [&](auto plain_tag) {
            constexpr bool kPlain = decltype(plain_tag)::value;
#pragma unroll
            for (int nb = 0; nb < kRowBlocks; ++nb) {
              // masked where a row ends inside the step; in the plain way scores as they are, else with the softmax scale and e
              [[maybe_unused]] float near[kPlain ? 1 : kHalves], behind[kPlain ? 1 : kHalves];  // e of tokens g, g + 8
              if constexpr (!kPlain) {
                const float2 by = huge ? make_float2(1.f, 1.f) : factor[nb];
                if (huge) {
#pragma unroll
                  for (int half = 0; half < kHalves; ++half)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nb][half][e] = s[nb][half][e] * 0x1p24f * (e & 1 ? factor[nb].y : factor[nb].x);
                }
#pragma unroll
                for (int half = 0; half < kHalves; ++half) {
                  near[half] = v_tokens[(2 * warp + turn) * kStepTokens + half * 16 + g];
                  behind[half] = v_tokens[(2 * warp + turn) * kStepTokens + half * 16 + 8 + g];
                  s[nb][half][0] = fmaf(s[nb][half][0], by.x, near[half]);
                  s[nb][half][1] = fmaf(s[nb][half][1], by.y, near[half]);
                  s[nb][half][2] = fmaf(s[nb][half][2], by.x, behind[half]);
                  s[nb][half][3] = fmaf(s[nb][half][3], by.y, behind[half]);
                }
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
              mx = column_max(mx);
              my = column_max(my);
              if constexpr (kPlain) {
                mx = fmaf(mx, factor[nb].x, static_cast<float>(step_e));
                my = fmaf(my, factor[nb].y, static_cast<float>(step_e));
              }
              mx = fmaxf(m[nb].x, mx);
              my = fmaxf(m[nb].y, my);
              // a row that has seen no key has o = l = 0: any finite factor will do
              const float vx = mx == -INFINITY ? 0.f : mx, vy = my == -INFINITY ? 0.f : my;
              a[nb] = make_float2(mx == -INFINITY ? 1.f : ex2_approx(m[nb].x - mx), my == -INFINITY ? 1.f : ex2_approx(m[nb].y - my));
              moved = moved || a[nb].x != 1.f || a[nb].y != 1.f;
              float2 sum = make_float2(0.f, 0.f);
#pragma unroll
              for (int half = 0; half < kHalves; ++half) {
                float2 w[2];
                if constexpr (kPlain) {
                  const float2 up = make_float2(static_cast<float>(step_e) - vx + kBias, static_cast<float>(step_e) - vy + kBias);
#pragma unroll
                  for (int e = 0; e < 2; ++e) w[e] = fma2(make_float2(s[nb][half][2 * e], s[nb][half][2 * e + 1]), factor[nb], up);
                } else {
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const float of_token = e ? behind[half] : near[half], of_v = isnan(of_token) ? 0.f : of_token;  // NaN is in the scores of those who see the token
                    const float2 below = make_float2(s[nb][half][2 * e] - vx, s[nb][half][2 * e + 1] - vy);  // 0 for the largest, however large that is
                    w[e] = make_float2(below.x + kBias, below.y + kBias);
                    sum = add2(sum, make_float2(exp2f(below.x - of_v), exp2f(below.y - of_v)));
                  }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  w[e] = make_float2(ex2_approx(w[e].x), ex2_approx(w[e].y));
                  if constexpr (kPlain) sum = add2(sum, w[e]);
                  pb[nb][half][e] = transpose_8x8(pack_f16x2(w[e].x, w[e].y));
                }
              }
              if constexpr (kPlain) {
                const float unit = kSumUnit * __uint_as_float(static_cast<uint32_t>(127 - step_e) << 23);
                l[nb] = fma2(sum, make_float2(unit, unit), mul2(l[nb], a[nb]));
              } else {  // sums take the factor in two steps, and weights without the scales; numbers below 2^-126 count
                const float hx = exp2f(0.5f * (m[nb].x - vx)), hy = exp2f(0.5f * (m[nb].y - vy));
                constexpr float kUp = 0x1p14f * kSumUnit;  // what the other sums are multiplied by
                l[nb] = make_float2(fmaf(kUp, sum.x, l[nb].x * hx * hx), fmaf(kUp, sum.y, l[nb].y * hy * hy));
              }
              m[nb] = make_float2(mx, my);
            }
          };
          if (plain) weigh(std::true_type{});
          else weigh(std::false_type{});
          if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int nb = 0; nb < kRowBlocks; ++nb)
#pragma unroll
              for (int ch = 0; ch < kChunks; ++ch) {
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                  const float2 x = mul2(make_float2(o[nb][ch][e], o[nb][ch][e + 1]), a[nb]);
                  o[nb][ch][e] = x.x, o[nb][ch][e + 1] = x.y;
                }
              }
          }
          // ---- O^T += V^T W^T, 16 tokens and 32 dimensions at a time
          const uint32_t v_smem = ring + st * kStageBytes + (kTileTokens + in_tile) * kRowBytes;
          const uint32_t* rests = v_rests + ((2 * warp + turn) * (kStepTokens / 2) + t) * kGroups;
#pragma unroll
          for (int ch = 0; ch < kGroups; ch += 2) {
#pragma unroll
            for (int half = 0; half < kHalves; ++half) {
              uint32_t vf[4];
              ldmatrix_x4_trans(v_smem + chunk_at(half * 16 + (mat & 1) * 8 + mrow, ch + (mat >> 1)), vf);
              const uint2 rest = *reinterpret_cast<const uint2*>(rests + half * 8 * kGroups + ch), rest8 = *reinterpret_cast<const uint2*>(rests + (half * 8 + 4) * kGroups + ch);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                uint32_t x[4], y[4];  // f16 pairs of two tokens: dimensions 4g to 4g + 3
                codes_to_numbers(vf[2 * e], eights, parts, x);
                codes_to_numbers(vf[2 * e + 1], eights, parts, y);
#pragma unroll
                for (int nb = 0; nb < kRowBlocks; ++nb) {
                  const uint32_t w0 = mul_f16x2(pb[nb][half][0], e ? rest.y : rest.x), w1 = mul_f16x2(pb[nb][half][1], e ? rest8.y : rest8.x);
                  mma_16816<true>(o[nb][2 * (ch + e)], x[0], x[1], y[0], y[1], w0, w1);
                  mma_16816<true>(o[nb][2 * (ch + e) + 1], x[2], x[3], y[2], y[3], w0, w1);
                }
              }
            }
          }
        };
        const int end = min(kPartTokens, seen_by_any - tile_tok - part * kPartTokens);
#pragma unroll 1
        for (int c = 0; c < end; c += kStepTokens) {
          work_on(c);
          turn ^= 1;
        }
        // every lane has read the tile: it may be filled again, but for the segment's last, whose place the warps hand their states over in
        if (i + 1 < seg_tiles) {
          __syncwarp();
          if (lane == 0) mbar_arrive(empty + 8 * st);
          next_place();
        }
      }
      const bool tokens = r.len > 0;
#pragma unroll
      for (int nb = 0; nb < kRowBlocks; ++nb) l[nb] = make_float2(column_sum(l[nb].x), column_sum(l[nb].y));
      // ---- the parts of a tile's tokens come together, 8 rows at a time: every warp takes some of the dimensions, of all parts
      constexpr int kMine = kChunks / kParts;
      float* states = reinterpret_cast<float*>(ring_ptr + st * kStageBytes) + row_group * kParts * kState + lane;
      const bool whole = seg_tiles == r.tiles;
      const int slot = first_unit ? 0 : 1;
#pragma unroll
      for (int nb = 0; nb < kRowBlocks; ++nb) {
        float acc[kMine][4];
        float mm[2] = {m[nb].x, m[nb].y}, sum[2] = {l[nb].x, l[nb].y};
        if (kParts > 1 && tokens) {
          arithmetic_sync();
#pragma unroll
          for (int ch = 0; ch < kChunks; ++ch)
#pragma unroll
            for (int e = 0; e < 4; ++e) states[part * kState + (ch * 4 + e) * 32] = o[nb][ch][e];
          if (g == 0) {
            row_state[warp * 8 + 2 * t] = make_float2(m[nb].x, l[nb].x);
            row_state[warp * 8 + 2 * t + 1] = make_float2(m[nb].y, l[nb].y);
          }
          arithmetic_sync();
          float2 others[2][kParts];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            mm[x] = -INFINITY;
            sum[x] = 0.f;
#pragma unroll
            for (int w = 0; w < kParts; ++w) {
              others[x][w] = row_state[(row_group * kParts + w) * 8 + 2 * t + x];
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
              for (int e = 0; e < 4; ++e) acc[ch][e] = fmaf(states[w * kState + ((part * kMine + ch) * 4 + e) * 32], f[e & 1], acc[ch][e]);
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
          auto dim_of = [&](int ch) { return 32 * ((part * kMine + ch) >> 1) + 4 * g + 2 * ((part * kMine + ch) & 1); };
          if (whole) {
            const int i = row / p.group, hq = head * p.group + row - i * p.group;
            uint16_t* dst = p.out + (r.q0 + i) * p.o_row + hq * p.o_head;
#pragma unroll
            for (int ch = 0; ch < kMine; ++ch) {
              const float even = acc[ch][x] * kUnit * inv, odd = acc[ch][2 + x] * kUnit * inv;
              *reinterpret_cast<uint32_t*>(dst + dim_of(ch)) = p.f16 ? pack_f16x2(even, odd) : pack_bf16x2(even, odd);
            }
            if (g == 0 && part == 0) p.lse[static_cast<int64_t>(hq) * p.total_q + r.q0 + i] = sum[x] > 0.f ? lse2 * 0.6931471805599453f : INFINITY;
          } else {
            const int64_t at = kCluster ? row - row0 : (2 * static_cast<int64_t>(blockIdx.x) + slot) * p.rows + row - row0;
            float* dst = (kCluster ? own_part : p.part_o) + at * kD;
#pragma unroll
            for (int ch = 0; ch < kMine; ++ch) *reinterpret_cast<float2*>(dst + dim_of(ch)) = make_float2(acc[ch][x] * kUnit * inv, acc[ch][2 + x] * kUnit * inv);
            if (g == 0 && part == 0) (kCluster ? own_lse : p.part_lse)[at] = lse2;
          }
        }
      }
      if (tokens) {
        fence_proxy_async_smem();  // what was handed over goes before the copy into the same place
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + 8 * st);
        next_place();
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
    merge_in_cluster<kD, kWarps + kLoaders>(p, share, own_part, own_lse, warp, lane);
    cluster_sync();  // the others have read this CTA's
  } else {
    if (threadIdx.x == 0) p.shared_units[blockIdx.x] = left;
  }
  if (lane == 0) drain_after_abort(abort_flag);
  if (threadIdx.x == 0 && *abort_flag != 0) atomicExch(p.status, static_cast<uint32_t>(SDPA_B200_DEVICE_TIMEOUT));
}

template <int kRowBlocks, int kRowWarps, int kD, bool kCluster>
cudaError_t launch_as(const StreamParams& p, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t stream, bool overlap) {
  constexpr uint32_t kSmem = smem_bytes<kRowBlocks, kRowWarps, kD, kCluster>(ring_stages<kRowBlocks, kRowWarps, kD, kCluster>());
  auto kernel = cache4_stream_kernel<kRowBlocks, kRowWarps, kD, kCluster>;
  const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (err != cudaSuccess) return err;
  return launch_behind(kernel, dim3(p.grid), threads<kRowBlocks>(), kSmem, stream, overlap, kCluster ? p.cluster : 1, tm_k, tm_v, p);
}

template <int kD>
cudaError_t launch_dim(const StreamParams& p, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t stream, bool overlap) {
  if (p.rows == 8) return (p.cluster > 0 ? launch_as<1, 1, kD, true> : launch_as<1, 1, kD, false>)(p, tm_k, tm_v, stream, overlap);
  if (p.rows == 16) return (p.cluster > 0 ? launch_as<2, 1, kD, true> : launch_as<2, 1, kD, false>)(p, tm_k, tm_v, stream, overlap);
  return (p.rows == 32 ? launch_as<2, 2, kD, false> : launch_as<2, 4, kD, false>)(p, tm_k, tm_v, stream, overlap);
}

}  // namespace

cudaError_t launch_stream4(const StreamParams& p, const CUtensorMap& tm_k, const CUtensorMap& tm_v, int head_dim, cudaStream_t stream, bool overlap) {
  return (head_dim == 64 ? launch_dim<64> : launch_dim<128>)(p, tm_k, tm_v, stream, overlap);
}

}  // namespace sdpa_b200
