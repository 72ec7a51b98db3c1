// Attention over the 8-bit paged cache. No counterpart in the reference, which has no paged cache.
//
//   s_ij = scale * ks[block(j), h] * <q_i, kc_j>,  out_i = sum_j softmax_j(s_i) * vs[block(j), h] * vc_j
//
// over the cached tokens j of the request, j <= i + len - rows of q where causal. Two paths:
//
// 1. Few rows per request (decode steps, drafted tokens): cache_stream_kernel, bound by the codes that come out of HBM. A unit is (request,
//    kv head, chunk of up to 16 rows (query token, query head of the group)): the rows ride in the M dimension of mma.sync.m16n8k16, so that codes are
//    read once for all of them. The lengths are on the GPU; every CTA sums them up and takes an equal contiguous share of all units' tiles of 128 tokens,
//    so that all SMs stream the same number of bytes however long each request is. A unit that several CTAs worked on leaves fp32 parts in the workspace,
//    at most two per CTA, and a second kernel merges them.
//    Codes become f16, exactly. Q rows are brought to f16 by a power of two each (their largest element to 2^14..2^15: a bf16 element loses
//    only what is 2^-39 of the row's largest), P is f16 in [0, 2^15], whose smaller weights keep all 11 bits down to 2^-29 of the largest; the scales of blocks
//    go onto the fp32 scores and products. Sums are fp32.
// 2. Many rows (chunks of prompts): the tensor cores bound it. cache_gather_kernel brings the request's codes * scales into 16-bit packed tensors in the
//    workspace (exact with the powers of two that the store kernel chooses), and the prefill kernel does the rest.
#include <type_traits>

#include "cache_common.cuh"

namespace sdpa_b200 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStepTokens = 32;                   // tokens a warp handles per step
constexpr int kTileTokens = kWarps * kStepTokens;  // 128
constexpr int kCtasPerSm = 2;
constexpr int kMaxSms = 160;  // workspace sizes do not ask the device: an upper bound of its SMs (148)
constexpr int kRows = 16;     // most rows of a unit

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
  int batch, heads_q, heads_kv, group, total_q, max_blocks, num_blocks, shift, rows, grid, causal, f16;
  float scale_log2;
};

// The unit that begins in a CTA's share and ends in a later one's: what the merge kernel needs to know. `last` < 0: there is none.
struct SharedUnit {
  int request, unit, last, slot;
};

// A request as units see it
struct Request {
  int index, len, rows_q, q0;  // tokens in the cache, rows of q, the first of them
  int tiles, units;            // per unit; 0 units: no rows
};

__device__ __forceinline__ Request request_at(const StreamParams& p, int b) {
  Request r;
  r.index = b;
  r.len = max(p.seq_lens[b], 0);
  r.q0 = p.cu_q ? p.cu_q[b] : b;
  r.rows_q = p.cu_q ? max(p.cu_q[b + 1] - r.q0, 0) : 1;
  if (r.q0 < 0 || r.q0 + static_cast<int64_t>(r.rows_q) > p.total_q) r.rows_q = 0;  // offsets that leave q: no rows
  r.tiles = max((r.len + kTileTokens - 1) / kTileTokens, 1);  // an empty request has rows to write too
  r.units = p.heads_kv * ((r.rows_q * p.group + p.rows - 1) / p.rows);
  return r;
}

// Stages of each warp's ring: what lets two CTAs share an SM's 228 KB.
template <bool kHi, int kD>
__host__ __device__ constexpr int ring_stages() { return (kHi ? 2 : 3) * (128 / kD); }
template <int kD>
__host__ __device__ constexpr uint32_t stage_bytes() { return 2u * kStepTokens * kD; }
template <bool kHi, int kD>
__host__ __device__ constexpr int merge_floats() { return ((kHi ? 4 : 2) * (kD / 8) + (kHi ? 4 : 2)) * 32; }
template <bool kHi, int kD>
__host__ __device__ constexpr uint32_t stream_smem_bytes() {
  constexpr int kSt = ring_stages<kHi, kD>();
  return 1024 + kWarps * kSt * stage_bytes<kD>() + (kWarps - 1) * merge_floats<kHi, kD>() * 4 + kWarps * kSt * (8 + 16) + 16;
}

// kHi: a unit has more than 8 rows, so fragment rows 8-15 are in use too.
template <bool kHi, int kD, bool kInt8>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
cache_stream_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const StreamParams p) {
  constexpr int kKSteps = kD / 16;
  constexpr int kNBlocks = kD / 8;
  constexpr int kSt = ring_stages<kHi, kD>();
  constexpr uint32_t kStageBytes = stage_bytes<kD>();
  constexpr int kMergeFloats = merge_floats<kHi, kD>();
  constexpr float kBias = 15.f;  // P is kept as 2^15 * weight: the largest is 2^15, the smallest normal one 2^-29 of it
  extern __shared__ uint8_t smem_raw[];
  __shared__ int64_t warp_tiles[kWarps];
  __shared__ int64_t start_before;
  __shared__ int start_request;
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  float* merge = reinterpret_cast<float*>(smem_raw + (base - raw_addr) + kWarps * kSt * kStageBytes);
  float4* stage_scales = reinterpret_cast<float4*>(merge + (kWarps - 1) * kMergeFloats);  // (ks, vs) of the two halves of a step
  const uint32_t bars = smem_u32(stage_scales + kWarps * kSt);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(reinterpret_cast<uint64_t*>(stage_scales + kWarps * kSt) + kWarps * kSt);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2;  // fragment row / token within a block of 8
  const int t = lane & 3;
  const uint32_t ring = base + warp * (kSt * kStageBytes);
  const uint32_t bar = bars + warp * (kSt * 8);
  float4* scales = stage_scales + warp * kSt;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kWarps * kSt; ++i) mbar_init(bars + 8 * i, 1);
    *abort_flag = 0;
    start_request = -1;
    fence_mbar_init();
  }
  if (elect_one()) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  wait_for_previous_grid();
  if (threadIdx.x == 0) launch_dependents();  // behind the wait: the merge kernel's blocks wait for this grid only
  __syncthreads();

  // ---- this CTA's share of the list of all tiles: sum over the requests, then the request that the share begins in
  auto tiles_of = [&](int b) -> int64_t {
    if (b >= p.batch) return 0;
    const Request r = request_at(p, b);
    return static_cast<int64_t>(r.tiles) * r.units;
  };
  int64_t total = 0;
  for (int b = threadIdx.x; b < p.batch; b += kThreads) total += tiles_of(b);
#pragma unroll
  for (int d = 1; d < 32; d *= 2) total += __shfl_xor_sync(0xffffffffu, total, d);
  if (lane == 0) warp_tiles[warp] = total;
  __syncthreads();
  total = warp_tiles[0] + warp_tiles[1] + warp_tiles[2] + warp_tiles[3];
  const int64_t ctas = min(total, static_cast<int64_t>(p.grid));  // those that get a tile: the others would leave no part where the merge looks for one
  const int64_t index = min(static_cast<int64_t>(blockIdx.x), ctas), end_index = min(index + 1, ctas);
  const int64_t first = ctas ? index * total / ctas : 0, last = ctas ? end_index * total / ctas : 0;
  if (first < last) {
    int64_t before = 0;
    for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
      const int64_t mine = tiles_of(b0 + threadIdx.x);
      int64_t run = mine;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int64_t x = __shfl_up_sync(0xffffffffu, run, d);
        if (lane >= d) run += x;
      }
      __syncthreads();
      if (lane == 31) warp_tiles[warp] = run;
      __syncthreads();
      int64_t at = before;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) at += warp_tiles[w];
        before += warp_tiles[w];
      }
      at += run - mine;
      if (first >= at && first < at + mine) {
        start_request = b0 + threadIdx.x;
        start_before = at;
      }
      if (first < before) break;
    }
    __syncthreads();
  }
  const int64_t n_tiles = last - first;
  SharedUnit left = {0, 0, -1, 0};
  if (n_tiles > 0 && start_request >= 0) {
    // ---- the load side of the warp's ring: its own request, unit and tile, kSt steps ahead of the arithmetic
    Request ld = request_at(p, start_request);
    int ld_unit = static_cast<int>((first - start_before) / ld.tiles);
    int ld_tile = static_cast<int>((first - start_before) % ld.tiles);
    int64_t ld_left = n_tiles;  // tiles of the share that have not been looked at
    int ld_step = 0;            // stages filled
    int group_of = -1, group_unit = -1, group_request = -1;
    int g_id = -1;  // lane i: page 32 * group_of + i of ld, its block and scales
    float g_ks = 0.f, g_vs = 0.f;
    auto next_unit = [&](Request& r, int& unit) {
      if (++unit < r.units) return;
      unit = 0;
      int b = r.index + 1;
      do r = request_at(p, b++);
      while (r.units == 0);  // more tiles are left, so there is one
    };
    // fills the next stage, if the share has a step of this warp left
    auto load_next = [&]() {
      while (ld_left > 0) {
        const int tok = ld_tile * kTileTokens + warp * kStepTokens;
        const bool have = tok < ld.len;
        if (have) {
          const int page = tok >> p.shift, grp = page >> 5;
          if (grp != group_of || ld_unit != group_unit || ld.index != group_request) {
            group_of = grp;
            group_unit = ld_unit;
            group_request = ld.index;
            const int mine = grp * 32 + lane;
            g_id = -1;
            g_ks = g_vs = 0.f;
            if ((static_cast<int64_t>(mine) << p.shift) < ld.len) {
              if (mine < p.max_blocks) g_id = p.block_table[ld.index * p.table_stride + mine];
              if (g_id >= 0 && g_id < p.num_blocks) {
                const int64_t at = static_cast<int64_t>(g_id) * p.heads_kv + ld_unit % p.heads_kv;
                g_ks = p.k_scale[at];
                g_vs = p.v_scale[at];
              } else {
                g_id = p.num_blocks;  // behind the cache: the copy brings zeros, the scale makes the scores of those who see them NaN
                g_ks = __int_as_float(0x7fffffff);
              }
            }
          }
          const bool halves = p.shift == 4;  // two blocks per step
          const int src = page & 31, src2 = halves ? (src + 1) & 31 : src;  // a step begins at an even page
          const int id0 = __shfl_sync(0xffffffffu, g_id, src), id1 = __shfl_sync(0xffffffffu, g_id, src2);
          const float4 sc = make_float4(__shfl_sync(0xffffffffu, g_ks, src), __shfl_sync(0xffffffffu, g_vs, src),
                                        __shfl_sync(0xffffffffu, g_ks, src2), __shfl_sync(0xffffffffu, g_vs, src2));
          const uint32_t st = ld_step % kSt;
          const uint32_t k_dst = ring + st * kStageBytes, v_dst = k_dst + kStepTokens * kD, full = bar + 8 * st;
          if (elect_one()) {
            scales[st] = sc;
            mbar_arrive_expect_tx(full, kStageBytes);
            const int head = ld_unit % p.heads_kv;
            if (halves) {
              const int other = id1 < 0 ? p.num_blocks : id1;  // no such page: zeros
              tma_load_4d(k_dst, &tm_k, full, 0, 0, head, id0);
              tma_load_4d(k_dst + 16 * kD, &tm_k, full, 0, 0, head, other);
              tma_load_4d(v_dst, &tm_v, full, 0, 0, head, id0);
              tma_load_4d(v_dst + 16 * kD, &tm_v, full, 0, 0, head, other);
            } else {
              const int row = tok & ((1 << p.shift) - 1);
              tma_load_4d(k_dst, &tm_k, full, 0, row, head, id0);
              tma_load_4d(v_dst, &tm_v, full, 0, row, head, id0);
            }
          }
          ++ld_step;
        }
        --ld_left;
        if (++ld_tile == ld.tiles) {
          ld_tile = 0;
          if (ld_left > 0) next_unit(ld, ld_unit);
        }
        if (have) return;
      }
    };
    for (int i = 0; i < kSt; ++i) load_next();

    const int mrow = lane & 7, mat = lane >> 3;
    auto chunk_at = [&](int row, int chunk) -> uint32_t {  // byte offset of a 16-byte chunk of a row in a swizzled stage
      if constexpr (kD == 128) return row * 128 + ((chunk ^ (row & 7)) << 4);
      return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
    };
    bool ok = true;
    int step = 0;  // stages read
    Request r = request_at(p, start_request);
    int unit = static_cast<int>((first - start_before) / r.tiles);
    int tile = static_cast<int>((first - start_before) % r.tiles);
    bool first_unit = true;
    for (int64_t done = 0; done < n_tiles;) {
      const int seg_tiles = static_cast<int>(min(n_tiles - done, static_cast<int64_t>(r.tiles - tile)));
      const int head = unit % p.heads_kv, row0 = unit / p.heads_kv * p.rows;
      const int n_rows = min(p.rows, r.rows_q * p.group - row0);
      // ---- rows g and g + 8: where they are, the tokens they see, their elements as f16
      uint32_t qa[kKSteps][4];
      float factor[2];
      int limit[2];
#pragma unroll
      for (int hi = 0; hi < 2; ++hi) {
        const int row = row0 + g + 8 * hi;
        const int i = row / p.group;
        limit[hi] = p.causal ? min(r.len, i + 1 + r.len - r.rows_q) : r.len;
        uint2 w[kKSteps];
        const bool have = (kHi || hi == 0) && g + 8 * hi < n_rows;
        const uint16_t* src = p.q + (r.q0 + i) * p.q_row + (head * p.group + row - i * p.group) * p.q_head + 4 * t;
        float largest = 0.f;
#pragma unroll
        for (int k = 0; k < kKSteps; ++k) {
          w[k] = have ? *reinterpret_cast<const uint2*>(src + 16 * k) : make_uint2(0u, 0u);
          const float2 a = p.f16 ? unpack_16x2<true>(w[k].x) : unpack_16x2<false>(w[k].x), b = p.f16 ? unpack_16x2<true>(w[k].y) : unpack_16x2<false>(w[k].y);
          largest = fmaxf(largest, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))));
        }
        largest = quad_max(largest);
        const int e = min(max(static_cast<int>(__float_as_uint(largest) >> 23) - 127, -100), 127);
        const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 - e) << 23);
        factor[hi] = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - 14 + e) << 23);
#pragma unroll
        for (int k = 0; k < kKSteps; ++k) {
          const float2 a = p.f16 ? unpack_16x2<true>(w[k].x) : unpack_16x2<false>(w[k].x), b = p.f16 ? unpack_16x2<true>(w[k].y) : unpack_16x2<false>(w[k].y);
          qa[k][hi] = pack_f16x2(a.x * up, a.y * up);
          qa[k][2 + hi] = pack_f16x2(b.x * up, b.y * up);
        }
      }
      const int seen_by_all = p.causal ? min(r.len, row0 / p.group + 1 + r.len - r.rows_q) : r.len;

      float o[kNBlocks][4];
#pragma unroll
      for (int nb = 0; nb < kNBlocks; ++nb) o[nb][0] = o[nb][1] = o[nb][2] = o[nb][3] = 0.f;
      float m[2] = {-INFINITY, -INFINITY};  // running max, log2 domain
      float l[2] = {0.f, 0.f};              // this thread's share of the running sums, times 2^kBias

      for (int i = 0; i < seg_tiles; ++i) {
        const int tok = (tile + i) * kTileTokens + warp * kStepTokens;
        if (tok >= r.len) continue;
        const uint32_t st = step % kSt;
        const uint32_t k_smem = ring + st * kStageBytes, v_smem = k_smem + kStepTokens * kD;
        if (ok) ok = mbar_wait(bar + 8 * st, (step / kSt) & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        ++step;
        __syncwarp();
        const float4 sc = scales[st];  // written by a lane of this warp

        // ---- S = Q K^T. The contraction runs over head_dim in the order in which ldmatrix hands out bytes: thread t has dimensions
        // 4t..4t+3 of every 16, of K and of Q
        float s[4][4];
#pragma unroll
        for (int blk = 0; blk < 4; ++blk) {
          s[blk][0] = s[blk][1] = s[blk][2] = s[blk][3] = 0.f;
#pragma unroll
          for (int ch = 0; ch < kKSteps; ch += 4) {
            uint32_t kf[4];
            ldmatrix_x4(k_smem + chunk_at(blk * 8 + mrow, ch + mat), kf);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t b0, b1;
              codes_to_f16<kInt8>(kf[j], b0, b1);
              mma_rows<kHi, true>(s[blk], qa[ch + j], b0, b1);
            }
          }
        }
        // ---- scores in the log2 domain (thread holds tokens tok + blk * 8 + 2t + {0, 1}), masked where a row ends inside the step
#pragma unroll
        for (int blk = 0; blk < 4; ++blk) {
          const float ks = blk < 2 ? sc.x : sc.z;
          s[blk][0] *= factor[0] * ks;
          s[blk][1] *= factor[0] * ks;
          s[blk][2] *= factor[1] * ks;
          s[blk][3] *= factor[1] * ks;
        }
        if (tok + kStepTokens > seen_by_all) {
#pragma unroll
          for (int blk = 0; blk < 4; ++blk) {
            const int j = tok + blk * 8 + 2 * t;
            if (j >= limit[0]) s[blk][0] = -INFINITY;
            if (j + 1 >= limit[0]) s[blk][1] = -INFINITY;
            if (j >= limit[1]) s[blk][2] = -INFINITY;
            if (j + 1 >= limit[1]) s[blk][3] = -INFINITY;
          }
        }
        uint32_t pa[2][4];
        float a[2] = {1.f, 1.f};
#pragma unroll
        for (int hi = 0; hi < (kHi ? 2 : 1); ++hi) {
          float top = fmaxf(s[0][2 * hi], s[0][2 * hi + 1]);
#pragma unroll
          for (int blk = 1; blk < 4; ++blk) top = max3(top, s[blk][2 * hi], s[blk][2 * hi + 1]);
          const float mn = fmaxf(m[hi], quad_max(top));
          // a row that has seen no key has o = l = 0: any finite factor will do
          a[hi] = mn == -INFINITY ? 1.f : ex2_approx(m[hi] - mn);
          m[hi] = mn;
          const float u = mn == -INFINITY ? 0.f : mn - kBias;
          float sum = 0.f;
#pragma unroll
          for (int blk = 0; blk < 4; ++blk) {
            const float x = ex2_approx(s[blk][2 * hi] - u), y = ex2_approx(s[blk][2 * hi + 1] - u);
            sum += x + y;
            pa[blk >> 1][(blk & 1) * 2 + hi] = pack_f16x2(x, y);
          }
          l[hi] = fmaf(l[hi], a[hi], sum);
        }
        if constexpr (!kHi) pa[0][1] = pa[0][3] = pa[1][1] = pa[1][3] = 0u;
        if (__any_sync(0xffffffffu, a[0] != 1.f || a[1] != 1.f)) {
#pragma unroll
          for (int nb = 0; nb < kNBlocks; ++nb) {
            o[nb][0] *= a[0];
            o[nb][1] *= a[0];
            o[nb][2] *= a[1];
            o[nb][3] *= a[1];
          }
        }
        // what stands behind the request's last token may be anything: it must not meet a weight of 0
        uint32_t keep[2][2] = {{~0u, ~0u}, {~0u, ~0u}};
        if (tok + kStepTokens > r.len) {
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = tok + half * 16 + e * 8 + 2 * t;
              keep[half][e] = (j < r.len ? 0xffffu : 0u) | (j + 1 < r.len ? 0xffff0000u : 0u);
            }
        }
        // ---- O += vs * (P V), 16 tokens at a time
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (half == 1 && tok + 16 >= r.len) break;
          const float vs = half ? sc.w : sc.y;
#pragma unroll
          for (int ch = 0; ch < kKSteps; ch += 2) {
            uint32_t vf[4];
            ldmatrix_x4_trans(v_smem + chunk_at(half * 16 + (mat & 1) * 8 + mrow, ch + (mat >> 1)), vf);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t even0, odd0, even1, odd1;  // f16 pairs of two tokens: dimension 2g, dimension 2g + 1
              codes_to_f16_by_two<kInt8>(vf[2 * e] & keep[half][0], even0, odd0);
              codes_to_f16_by_two<kInt8>(vf[2 * e + 1] & keep[half][1], even1, odd1);
              float d[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
              mma_rows<kHi, true>(d[0], pa[half], even0, even1);
              mma_rows<kHi, true>(d[1], pa[half], odd0, odd1);
#pragma unroll
              for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int y = 0; y < (kHi ? 4 : 2); ++y) o[2 * (ch + e) + x][y] = fmaf(d[x][y], vs, o[2 * (ch + e) + x][y]);
            }
          }
        }
        __syncwarp();  // the stage has been read by every lane: refill it
        if (ok) load_next();
      }

      // ---- merge the four warps: 1-3 hand their state over in fragment order, warp 0 folds it into its own
#pragma unroll
      for (int hi = 0; hi < 2; ++hi) l[hi] = quad_sum(l[hi]);
      __syncthreads();  // warp 0 has read what the previous unit left here
      constexpr int kPer = kHi ? 4 : 2, kTail = kNBlocks * kPer * 32;
      if (warp > 0) {
        float* dst = merge + (warp - 1) * kMergeFloats + lane;
#pragma unroll
        for (int nb = 0; nb < kNBlocks; ++nb)
#pragma unroll
          for (int e = 0; e < kPer; ++e) dst[(nb * kPer + e) * 32] = o[nb][e];
#pragma unroll
        for (int hi = 0; hi < (kHi ? 2 : 1); ++hi) {
          dst[kTail + 64 * hi] = m[hi];
          dst[kTail + 64 * hi + 32] = l[hi];
        }
      }
      __syncthreads();
      const bool whole = seg_tiles == r.tiles;
      const int slot = first_unit ? 0 : 1;
      if (warp == 0) {
#pragma unroll
        for (int hi = 0; hi < (kHi ? 2 : 1); ++hi) {
          float mm = m[hi];
#pragma unroll
          for (int w = 0; w < kWarps - 1; ++w) mm = fmaxf(mm, merge[w * kMergeFloats + kTail + 64 * hi + lane]);
          auto weight = [&](float x) { return x == -INFINITY ? 0.f : ex2_approx(x - mm); };
          float f = weight(m[hi]), sum = l[hi] * f;
#pragma unroll
          for (int nb = 0; nb < kNBlocks; ++nb) {
            o[nb][2 * hi] *= f;
            o[nb][2 * hi + 1] *= f;
          }
#pragma unroll
          for (int w = 0; w < kWarps - 1; ++w) {
            const float* src = merge + w * kMergeFloats + lane;
            f = weight(src[kTail + 64 * hi]);
            sum += src[kTail + 64 * hi + 32] * f;
#pragma unroll
            for (int nb = 0; nb < kNBlocks; ++nb) {
              o[nb][2 * hi] += src[(nb * kPer + 2 * hi) * 32] * f;
              o[nb][2 * hi + 1] += src[(nb * kPer + 2 * hi + 1) * 32] * f;
            }
          }
          const int rr = g + 8 * hi;
          if (rr < n_rows) {
            const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);  // NaN stays NaN
            const float lse2 = sum == 0.f ? -INFINITY : mm - kBias + log2f(sum);
            if (whole) {
              const int row = row0 + rr, i = row / p.group, hq = head * p.group + row - i * p.group;
              uint16_t* dst = p.out + (r.q0 + i) * p.o_row + hq * p.o_head + 4 * t;
#pragma unroll
              for (int ch = 0; ch < kKSteps; ++ch) {  // dimensions 4t..4t+3 of every 16: even, odd, even, odd
                const float x0 = o[2 * ch][2 * hi] * inv, x1 = o[2 * ch + 1][2 * hi] * inv, x2 = o[2 * ch][2 * hi + 1] * inv, x3 = o[2 * ch + 1][2 * hi + 1] * inv;
                *reinterpret_cast<uint2*>(dst + 16 * ch) = p.f16 ? make_uint2(pack_f16x2(x0, x1), pack_f16x2(x2, x3)) : make_uint2(pack_bf16x2(x0, x1), pack_bf16x2(x2, x3));
              }
              if (t == 0) p.lse[static_cast<int64_t>(hq) * p.total_q + r.q0 + i] = sum > 0.f ? lse2 * 0.6931471805599453f : INFINITY;
            } else {
              const int64_t at = (2 * static_cast<int64_t>(blockIdx.x) + slot) * p.rows + rr;
              float* dst = p.part_o + at * kD + 4 * t;
#pragma unroll
              for (int ch = 0; ch < kKSteps; ++ch)
                *reinterpret_cast<float4*>(dst + 16 * ch) = make_float4(o[2 * ch][2 * hi] * inv, o[2 * ch + 1][2 * hi] * inv, o[2 * ch][2 * hi + 1] * inv, o[2 * ch + 1][2 * hi + 1] * inv);
              if (t == 0) p.part_lse[at] = lse2;
            }
          }
        }
      }
      if (tile == 0 && !whole) {  // begun here, ended by the CTA whose share holds its last tile
        const int64_t end = first + done + r.tiles - 1;
        left = {r.index, unit, static_cast<int>(((end + 1) * ctas - 1) / total), slot};
      }
      done += seg_tiles;
      tile = 0;
      first_unit = false;
      if (done < n_tiles) next_unit(r, unit);
    }
  }
  if (threadIdx.x == 0) p.shared_units[blockIdx.x] = left;
  if (lane == 0) drain_after_abort(abort_flag);
  if (threadIdx.x == 0 && *abort_flag != 0) atomicExch(p.status, static_cast<uint32_t>(SDPA_B200_DEVICE_TIMEOUT));
}

// Merges the parts of the units that several CTAs worked on: block (i, j) those of the unit that CTA i began, rows 4j to 4j + 3, a warp each.
template <int kD>
__global__ void __launch_bounds__(128) cache_merge_kernel(const StreamParams p) {
  constexpr int kPer = kD / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rr = blockIdx.y * 4 + warp;
  wait_for_previous_grid();
  launch_dependents();
  const SharedUnit u = p.shared_units[blockIdx.x];
  if (u.last < 0) return;
  const Request r = request_at(p, u.request);
  const int row = u.unit / p.heads_kv * p.rows + rr;
  if (rr >= p.rows || row >= r.rows_q * p.group) return;
  auto part = [&](int c) { return (2 * static_cast<int64_t>(c) + (c == static_cast<int>(blockIdx.x) ? u.slot : 0)) * p.rows + rr; };
  float top = -INFINITY;
  bool nan = false;
  for (int c = blockIdx.x + lane; c <= u.last; c += 32) {
    const float x = p.part_lse[part(c)];
    nan = nan || isnan(x);
    top = fmaxf(top, x);
  }
#pragma unroll
  for (int d = 1; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  nan = __any_sync(0xffffffffu, nan);
  float sum = 0.f, acc[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
  if (top != -INFINITY) {
#pragma unroll 4
    for (int c = blockIdx.x; c <= u.last; ++c) {
      const int64_t at = part(c);
      const float x = p.part_lse[at], w = x == -INFINITY ? 0.f : exp2f(x - top);
      sum += w;
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] = fmaf(w, p.part_o[at * kD + e * 32 + lane], acc[e]);
    }
  }
  const int i = row / p.group, hq = u.unit % p.heads_kv * p.group + row - i * p.group;
  const float inv = nan ? __int_as_float(0x7fffffff) : sum > 0.f ? 1.f / sum : 0.f;
  uint16_t* dst = p.out + (r.q0 + i) * p.o_row + hq * p.o_head;
#pragma unroll
  for (int e = 0; e < kPer; ++e) dst[e * 32 + lane] = p.f16 ? to_16<true>(acc[e] * inv) : to_16<false>(acc[e] * inv);
  if (lane == 0) p.lse[static_cast<int64_t>(hq) * p.total_q + r.q0 + i] = !nan && sum > 0.f ? (top + log2f(sum)) * 0.6931471805599453f : INFINITY;
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
  int batch, heads, max_blocks, num_blocks, shift, max_k;
};

constexpr int kGatherTokens = 64;
constexpr int kKeyTile = 128;  // keys that the prefill kernel reads at a time, from a sequence's start

__host__ __device__ __forceinline__ int64_t padded_keys(int64_t n) { return (n + kKeyTile - 1) / kKeyTile * kKeyTile; }

// Block (i, h, b): tokens 64i to 64i + 63 of request b, kv head h, keys and values. The prefill kernel's last tile of a sequence goes on into the rows behind it,
// where a weight of 0 would meet another request's NaN, or whatever the workspace held. So every request's rows are filled up to a whole tile with zeros, and these
// stand in the list of sequences as one of their own, without queries.
template <int kD, bool kInt8, bool kF16>
__global__ void __launch_bounds__(256) cache_gather_kernel(const GatherParams p) {
  __shared__ int sums[8];
  const int b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
  auto len_of = [&](int i) { return min(max(p.seq_lens[i], 0), p.max_k); };
  int before = 0;
  for (int i = tid; i < b; i += 256) before += static_cast<int>(padded_keys(len_of(i)));
#pragma unroll
  for (int d = 1; d < 32; d *= 2) before += __shfl_xor_sync(0xffffffffu, before, d);
  if ((tid & 31) == 0) sums[tid >> 5] = before;
  __syncthreads();
  before = 0;
  for (int w = 0; w < 8; ++w) before += sums[w];
  const int len = len_of(b), padded = static_cast<int>(padded_keys(len));
  if (blockIdx.x == 0 && h == 0 && tid == 0) {
    int32_t* cu_k = p.cu + 2 * p.batch + 1;
    p.cu[2 * b] = p.cu_q[b];
    p.cu[2 * b + 1] = p.cu_q[b + 1];
    cu_k[2 * b] = before;
    cu_k[2 * b + 1] = before + len;
    if (b == p.batch - 1) {
      p.cu[2 * p.batch] = p.cu_q[p.batch];
      cu_k[2 * p.batch] = before + padded;
    }
  }
  constexpr int kLanes = kD / 16;  // 16 codes a thread
  for (int i = tid; i < kGatherTokens * kLanes; i += 256) {
    const int tok = blockIdx.x * kGatherTokens + i / kLanes, at = i % kLanes * 16;
    if (tok >= padded) break;
    const int page = tok >> p.shift, place = tok & ((1 << p.shift) - 1);
    const int id = tok < len && page < p.max_blocks ? p.block_table[b * p.table_stride + page] : -1;
    const bool bad = id < 0 || id >= p.num_blocks;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      uint4 w = make_uint4(0u, 0u, 0u, 0u);
      float scale = tok < len && x == 0 ? __int_as_float(0x7fffffff) : 0.f;  // a block outside the cache: its scores are NaN, for those who see them
      if (!bad) {
        w = *reinterpret_cast<const uint4*>(p.cache[x] + id * p.block[x] + h * p.head[x] + place * p.row[x] + at);
        scale = p.scale[x][static_cast<int64_t>(id) * p.heads + h];
      }
      uint32_t f[8], c[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t lo, hi;
        codes_to_f16<kInt8>(c[e], lo, hi);
        const float2 u = unpack_16x2<true>(lo), v = unpack_16x2<true>(hi);
        f[2 * e] = pack_16x2<kF16>(u.x * scale, u.y * scale);
        f[2 * e + 1] = pack_16x2<kF16>(v.x * scale, v.y * scale);
      }
      uint4* dst = reinterpret_cast<uint4*>(p.out[x] + ((static_cast<int64_t>(before) + tok) * p.heads + h) * kD + at);
      dst[0] = make_uint4(f[0], f[1], f[2], f[3]);
      dst[1] = make_uint4(f[4], f[5], f[6], f[7]);
    }
  }
}

// Rows that the longest request may have for path 1: above, path 2. At 32/8 heads a unit of 16 rows streams the cache in HBM's time, and each further one
// adds that of its products; the prefill kernel works on tiles of 256 rows of one query head.
constexpr int kMostStreamRows = 512;

bool streams(const sdpa_b200_cache_params& p) {
  return static_cast<int64_t>(p.max_seqlen_q) * (p.heads_q / p.heads_kv) <= kMostStreamRows || p.cu_seqlens_q == nullptr;
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
  return static_cast<int64_t>(p.max_seqlen_q) * (p.heads_q / p.heads_kv) <= 8 ? 8 : kRows;
}

size_t round_256(size_t n) { return (n + 255) / 256 * 256; }

size_t gather_bytes(const sdpa_b200_cache_params& p) {
  return static_cast<size_t>(p.batch) * padded_keys(p.max_seqlen_k) * p.heads_kv * p.head_dim * 2;
}

int launch_stream(const sdpa_b200_cache_params& c, char* workspace, uint32_t* status, cudaStream_t stream) {
  const int sms = sm_count();
  if (sms <= 0 || sms > kMaxSms) {
    set_error("cache_attention: cannot use a device with %d SMs", sms);
    return SDPA_B200_NO_DEVICE;
  }
  StreamParams p;
  p.q = static_cast<const uint16_t*>(c.q);
  p.out = static_cast<uint16_t*>(c.out);
  p.lse = c.lse;
  p.k_scale = c.k_scale;
  p.v_scale = c.v_scale;
  p.block_table = c.block_table;
  p.seq_lens = c.seq_lens;
  p.cu_q = c.cu_seqlens_q;
  p.status = status;
  p.q_row = c.q_row_stride;
  p.q_head = c.q_head_stride;
  p.o_row = c.o_row_stride;
  p.o_head = c.o_head_stride;
  p.table_stride = c.table_stride;
  p.batch = c.batch;
  p.heads_q = c.heads_q;
  p.heads_kv = c.heads_kv;
  p.group = c.heads_q / c.heads_kv;
  p.total_q = c.total_q;
  p.max_blocks = c.max_blocks;
  p.num_blocks = c.num_blocks;
  p.shift = block_shift(c.block_size);
  p.rows = unit_rows(c);
  p.causal = c.is_causal;
  p.f16 = c.dtype == SDPA_B200_F16;
  p.scale_log2 = c.softmax_scale * 1.4426950408889634f;
  // a CTA per tile, up to one wave
  const int64_t units = static_cast<int64_t>(c.batch) * c.heads_kv * ((static_cast<int64_t>(c.max_seqlen_q) * p.group + p.rows - 1) / p.rows);
  const int64_t tiles = units * ((static_cast<int64_t>(c.max_seqlen_k) + kTileTokens - 1) / kTileTokens);
  p.grid = static_cast<int>(tiles < kCtasPerSm * sms ? tiles : kCtasPerSm * sms);
  const size_t rows = static_cast<size_t>(kCtasPerSm) * kMaxSms * 2 * p.rows;
  p.part_o = reinterpret_cast<float*>(workspace + kWorkspaceHeaderBytes);
  p.part_lse = p.part_o + rows * c.head_dim;
  p.shared_units = reinterpret_cast<SharedUnit*>(p.part_lse + rows);
  CUtensorMap tm_k, tm_v;
  const int box = c.block_size < kStepTokens ? c.block_size : kStepTokens;
  int st = make_cache_tensor_map(&tm_k, c.k_cache, c.head_dim, c.block_size, c.heads_kv, c.num_blocks, c.k_row_stride, c.k_head_stride, c.k_block_stride, box);
  if (st != SDPA_B200_OK) return st;
  st = make_cache_tensor_map(&tm_v, c.v_cache, c.head_dim, c.block_size, c.heads_kv, c.num_blocks, c.v_row_stride, c.v_head_stride, c.v_block_stride, box);
  if (st != SDPA_B200_OK) return st;
  cudaError_t err = cudaSuccess;
  auto launch = [&](auto hi_tag, auto dim_tag, auto int8_tag) {
    constexpr bool kHi = decltype(hi_tag)::value, kInt8 = decltype(int8_tag)::value;
    constexpr int kD = decltype(dim_tag)::value;
    constexpr uint32_t kSmem = stream_smem_bytes<kHi, kD>();
    static_assert(kCtasPerSm * (kSmem + 1024) <= 228 * 1024, "two CTAs do not fit an SM");
    auto kernel = cache_stream_kernel<kHi, kD, kInt8>;
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (err == cudaSuccess) err = launch_behind(kernel, dim3(p.grid), kThreads, kSmem, stream, false, 1, tm_k, tm_v, p);
  };
  auto launch_code = [&](auto hi_tag, auto dim_tag) {
    c.code == SDPA_B200_INT8 ? launch(hi_tag, dim_tag, std::true_type{}) : launch(hi_tag, dim_tag, std::false_type{});
  };
  auto launch_dim = [&](auto hi_tag) {
    c.head_dim == 64 ? launch_code(hi_tag, std::integral_constant<int, 64>{}) : launch_code(hi_tag, std::integral_constant<int, 128>{});
  };
  p.rows > 8 ? launch_dim(std::true_type{}) : launch_dim(std::false_type{});
  if (err != cudaSuccess) {
    set_error("cache_attention: launch failed: %s", cudaGetErrorString(err));
    return SDPA_B200_LAUNCH_FAILED;
  }
  count_launch();
  if (p.grid == 1) return SDPA_B200_OK;  // nobody to share a unit with
  const dim3 merge_grid(p.grid - 1, (p.rows + 3) / 4);
  err = c.head_dim == 64 ? launch_behind(cache_merge_kernel<64>, merge_grid, 128, 0, stream, true, 1, p)
                         : launch_behind(cache_merge_kernel<128>, merge_grid, 128, 0, stream, true, 1, p);
  if (err != cudaSuccess) {
    set_error("cache_attention merge: launch failed: %s", cudaGetErrorString(err));
    return SDPA_B200_LAUNCH_FAILED;
  }
  count_launch();
  return SDPA_B200_OK;
}

int launch_gathered(const sdpa_b200_cache_params& c, char* workspace, uint32_t* status, cudaStream_t stream) {
  // the prefill kernel's own workspace in front, then K, V and the offsets
  sdpa_b200_params f = {};
  GatherParams g;
  char* at = workspace + kWorkspaceHeaderBytes;
  g.out[0] = reinterpret_cast<uint16_t*>(at);
  g.out[1] = reinterpret_cast<uint16_t*>(at + gather_bytes(c));
  g.cu = reinterpret_cast<int32_t*>(at + 2 * gather_bytes(c));
  g.cu_q = c.cu_seqlens_q;
  g.cache[0] = static_cast<const uint8_t*>(c.k_cache);
  g.cache[1] = static_cast<const uint8_t*>(c.v_cache);
  g.scale[0] = c.k_scale;
  g.scale[1] = c.v_scale;
  g.block[0] = c.k_block_stride, g.head[0] = c.k_head_stride, g.row[0] = c.k_row_stride;
  g.block[1] = c.v_block_stride, g.head[1] = c.v_head_stride, g.row[1] = c.v_row_stride;
  g.block_table = c.block_table;
  g.seq_lens = c.seq_lens;
  g.table_stride = c.table_stride;
  g.batch = c.batch;
  g.heads = c.heads_kv;
  g.max_blocks = c.max_blocks;
  g.num_blocks = c.num_blocks;
  g.shift = block_shift(c.block_size);
  g.max_k = c.max_seqlen_k;
  const dim3 grid(static_cast<unsigned>(padded_keys(c.max_seqlen_k) / kGatherTokens), c.heads_kv, c.batch);
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
  f.cu_seqlens_k = g.cu + 2 * c.batch + 1;
  f.batch = 2 * c.batch;
  f.heads_q = c.heads_q;
  f.heads_kv = c.heads_kv;
  f.head_dim = c.head_dim;
  f.max_seqlen_q = c.max_seqlen_q;
  f.max_seqlen_k = c.max_seqlen_k;
  f.total_q = c.total_q;
  f.total_k = static_cast<int32_t>(c.batch * padded_keys(c.max_seqlen_k));
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
  return launch_fwd_prefill(f, workspace, stream);
}

size_t workspace_bytes_of(const sdpa_b200_cache_params& p) {
  if (!streams(p)) return kWorkspaceHeaderBytes + 2 * gather_bytes(p) + round_256((4 * static_cast<size_t>(p.batch) + 2) * 4);
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
  if (!streams(*p) && (p->batch > 65535 || p->heads_kv > 65535)) {
    set_error("cache_attention: many rows per request come in batches of up to 65535, with up to 65535 heads (got %d, %d)", p->batch, p->heads_kv);
    return SDPA_B200_UNSUPPORTED;
  }
  if (!streams(*p) && p->batch * padded_keys(p->max_seqlen_k) > INT32_MAX) {
    set_error("cache_attention: batch * max_seqlen_k must be below 2^31 for long requests");
    return SDPA_B200_INVALID_ARG;
  }
  st = check_device();
  if (st != SDPA_B200_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p->device_status == nullptr && cudaMemsetAsync(workspace, 0, kWorkspaceHeaderBytes, s) != cudaSuccess) {
    set_error("clearing the workspace header failed: %s", cudaGetErrorString(cudaGetLastError()));
    return SDPA_B200_LAUNCH_FAILED;
  }
  uint32_t* status = p->device_status != nullptr ? p->device_status : static_cast<uint32_t*>(workspace);
  if (streams(*p)) return launch_stream(*p, static_cast<char*>(workspace), status, s);
  return launch_gathered(*p, static_cast<char*>(workspace), status, s);
}
