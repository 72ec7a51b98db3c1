// Keys and values of a serving step into the 8-bit paged cache. No counterpart in the reference, which has no paged cache.
//
// Per (block, head) that gets tokens: need = the smallest power of two at which the largest new element is a code, scale = max(old, need) where
// the block holds earlier tokens, code = round(x / scale). Decoding raises the scale of a block that fills up token by token; earlier tokens are then
// read, multiplied by old / scale and rounded again. With powers of two that costs e4m3 only what falls below its smallest numbers, and a
// dequantised element is exact in 16 bits within their range (the code of f16's 65504 is 65536).
//
// Bound by HBM for prompts (two bytes read and one written per element), by latency for decode steps. The tokens of one block stand next to each other,
// so a run of them is found from the slots alone: it begins where a token's block is not that of the token with a place in front. A CTA takes a window of
// tokens for one head of the keys or values; its first warp finds the runs that begin there. Runs of a few tokens (decode steps) are a warp's each; on a
// longer one all warps work, each thread with its elements in registers between the largest element and the codes, so that they are read once.
// Measured (8192 tokens of 4 prompts, 8 heads of 128, bf16 beside their queries to e4m3): 57 us with a warp for each run, which found it by itself, and
// elements looked at one by one; 21 with a warp that finds runs for the CTA and the largest element two at a time as integers; 16.5 with a path of its own for
// runs without gaps; 15.3 with all slots asked for before any is looked at; 14.2 with seven CTAs on an SM instead of six (3.5 TB/s; the few bytes spilled for it
// cost the smallest calls 0.1 to 0.2). Of the 14.2 (14.0 a call back to back, under the tail of the one in front), launch and runs are 4, and reading, codes and writing follow one another in a CTA. Rows held in
// shared memory, those of the next head asked for ahead, one or eight warps instead of four, and asking L2 for the window's rows while the runs are found were no faster.
#include "cache_common.cuh"

namespace sdpa_b200 {
namespace {

constexpr int kWarps = 4;
constexpr int kHeld = 8;         // rows that a thread keeps in registers
constexpr int kMostWindow = 64;  // tokens of a window

struct StoreSide {
  const uint16_t* in;
  uint8_t* cache;
  float* scale;
  int64_t in_row, in_head, block, head, row;
};

struct StoreParams {
  StoreSide side[2];  // keys, values
  const int32_t* slots;
  int tokens, heads, num_slots, shift;
  int window;  // tokens of a CTA: 4, or a multiple of 32 up to kMostWindow
};

template <bool kF16>
__device__ __forceinline__ void to_floats(const uint4& w, float (&x)[8]) {
  const float2 a = unpack_16x2<kF16>(w.x), b = unpack_16x2<kF16>(w.y), c = unpack_16x2<kF16>(w.z), d = unpack_16x2<kF16>(w.w);
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y, x[4] = c.x, x[5] = c.y, x[6] = d.x, x[7] = d.y;
}

// What a thread has of a run's rows: row0, row0 + step, ... of n, eight elements of each
struct Rows {
  const uint16_t* in;
  uint8_t* cache;
  float* scale;
  int64_t in_row, row;
  int row0, step, n, place;
};

// Earlier tokens of the block rounded again to a scale that has grown. `down` = 1 / new scale, a power of two.
template <bool kInt8>
__device__ __noinline__ void round_again(const Rows& w, float old, float down) {
  for (int r = w.row0; r < w.place; r += w.step) {
    const uint2 codes = *reinterpret_cast<const uint2*>(w.cache + r * w.row);
    uint32_t h[4];
    codes_to_f16<kInt8>(codes.x, h[0], h[1]);
    codes_to_f16<kInt8>(codes.y, h[2], h[3]);
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack_16x2<true>(h[e]);
      v[2 * e] = f.x * old * down;
      v[2 * e + 1] = f.y * old * down;
    }
    *reinterpret_cast<uint2*>(w.cache + r * w.row) = make_uint2(values_to_codes<kInt8>(v[0], v[1], v[2], v[3]), values_to_codes<kInt8>(v[4], v[5], v[6], v[7]));
  }
}

__device__ __forceinline__ uint32_t larger(uint32_t top, const uint4& w) {
  return __vmaxu2(__vmaxu2(top, w.x & 0x7fff7fffu), __vmaxu2(w.y & 0x7fff7fffu, __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)));
}
template <uint32_t kInf>
__device__ __forceinline__ uint32_t larger_finite(uint32_t top, const uint4& w) {
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = words[i] & 0x7fffu, hi = words[i] >> 16 & 0x7fffu;
    top = max(top, max(lo < kInf ? lo : 0u, hi < kInf ? hi : 0u));
  }
  return top;
}

// Tokens [first, first + count) of the call, one block's; `rows`: their places are place, place + 1, ..., none left out
struct Run {
  int first, count, block, place;
  bool rows;
};

template <int kD, bool kInt8, bool kF16>
__global__ void __launch_bounds__(kWarps * 32, 7) store_kernel(const StoreParams p) {
  constexpr int kLanes = kD / 8, kRows = 32 / kLanes;  // lanes per row, rows per step of a warp
  __shared__ Run runs[kMostWindow];
  __shared__ int num_runs;
  __shared__ uint32_t warp_top[2][kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / kLanes, at = lane % kLanes * 8;
  const int mask = (1 << p.shift) - 1;
  // the heads of a window stand next to each other: together they read whole tokens
  const int unit = blockIdx.x % (2 * p.heads), head = unit >> 1, own0 = static_cast<int>(blockIdx.x / (2 * p.heads)) * p.window;
  const StoreSide& x = p.side[unit & 1];
  auto block_of = [&](int t) {
    const int slot = t < p.tokens ? p.slots[t] : -1;
    return slot < 0 || slot >= p.num_slots ? -1 : slot >> p.shift;
  };

  // by one warp: the runs that begin in the window whose first token is own0. All slots that it is likely to need are asked for at once
  auto find_runs = [&](int own0) {
    auto slot_at = [&](int t) { return t >= 0 && t < p.tokens ? p.slots[t] : -1; };
    auto block_at = [&](int slot) { return slot < 0 || slot >= p.num_slots ? -1 : slot >> p.shift; };
    const int front = slot_at(own0 - 32 + lane), end = own0 + p.window;
    int slot = slot_at(own0 + lane), slot1 = slot_at(own0 + 32 + lane), slot2 = slot_at(own0 + 64 + lane);
    const int front_block = block_at(front);
    const unsigned front_placed = __ballot_sync(0xffffffffu, front_block >= 0);
    int last = own0 - 1 - __clz(front_placed);  // the nearest token with a place, and its block
    int last_block = __shfl_sync(0xffffffffu, front_block, front_placed ? 31 - __clz(front_placed) : 0);
    int last_slot = __shfl_sync(0xffffffffu, front, 31);
    int found = 0;
    bool open = false;  // the run that goes on behind the 32 tokens looked at
    Run run = {};
    for (int base = own0;; base += 32) {
      const int b = block_at(slot);
      const unsigned placed = __ballot_sync(0xffffffffu, b >= 0), in_front = (1u << lane) - 1, below = placed & in_front;
      const int from_lane = __shfl_sync(0xffffffffu, b, below ? 31 - __clz(below) : 0);
      const int slot_in_front = __shfl_up_sync(0xffffffffu, slot, 1);
      // a run begins where the nearest token with a place in front, within 32, is in another block
      const int before = below ? from_lane : base + lane - last <= 32 ? last_block : -1;
      const unsigned firsts = __ballot_sync(0xffffffffu, b >= 0 && b != before);
      const unsigned parted = __ballot_sync(0xffffffffu, slot != (lane == 0 ? last_slot : slot_in_front) + 1);
      // the open run ends with the last token in front of the next one
      if (open) {
        const unsigned more = firsts ? placed & ((firsts & -firsts) - 1) : placed;
        if (more != 0) {
          run.count = base + 32 - __clz(more) - run.first;
          run.rows = run.rows && parted << __clz(more) == 0;
        }
        if (firsts != 0) {
          if (lane == 0) runs[found - 1] = run;
          open = false;
        }
      }
      const unsigned own = base + 32 <= end ? firsts : base < end ? firsts & ((1u << (end - base)) - 1) : 0u;
      if (own != 0) {
        const unsigned behind = firsts & ~(in_front << 1 | 1u);
        const unsigned mine = placed & ~in_front & (behind ? (behind & -behind) - 1 : ~0u);
        const int n = 32 - __clz(mine) - lane;
        const unsigned inside = (n >= 32 ? ~0u : (1u << n) - 1) << lane & ~(1u << lane);  // bits lane + 1 to lane + n - 1
        const Run r = {base + lane, n, b, slot & mask, (parted & inside) == 0};
        if (own >> lane & 1) runs[found + __popc(own & in_front)] = r;
        const int l = 31 - __clz(own);
        run = {base + l, __shfl_sync(0xffffffffu, n, l), __shfl_sync(0xffffffffu, b, l), __shfl_sync(0xffffffffu, r.place, l), __shfl_sync(0xffffffffu, r.rows, l) != 0};
        open = firsts >> l == 1u;
        found += __popc(own);
      }
      if (placed != 0) {
        last = base + 31 - __clz(placed);
        last_block = __shfl_sync(0xffffffffu, b, 31 - __clz(placed));
      }
      if (base + 32 >= end && (!open || last < base)) break;  // no token behind is within 32
      last_slot = __shfl_sync(0xffffffffu, slot, 31);
      slot = slot1, slot1 = slot2;
      slot2 = slot_at(base + 96 + lane);
    }
    __syncwarp();
    if (lane == 0) {
      if (open) runs[found - 1] = run;
      num_runs = found;
    }
  };

  if (threadIdx.x == 0) launch_dependents();
  wait_for_previous_grid();
  if (warp == 0) find_runs(own0);
  __syncthreads();

  const int count = num_runs;
  int shared_runs = 0;
  for (int turn = 0; turn < count; ++turn) {
    const int t0 = runs[turn].first, n = runs[turn].count, block = runs[turn].block, place = runs[turn].place;
    const bool alone = n <= kRows * kHeld;
    if (alone && turn % kWarps != warp) continue;
    const Rows w = {x.in + t0 * x.in_row + head * x.in_head + at, x.cache + block * x.block + head * x.head + at,
                    x.scale + static_cast<int64_t>(block) * p.heads + head, x.in_row, x.row, alone ? sub : warp * kRows + sub, alone ? kRows : kWarps * kRows, n, place};
    const float old = place > 0 ? *w.scale : 0.f;
    // The largest of `top` over the run's warps. One barrier for each is enough, with words that change with every call; also: every warp has read the old scale
    auto over_warps = [&](uint32_t top) {
      top = __reduce_max_sync(0xffffffffu, __vmaxu2(top, top >> 16) & 0xffffu);
      if (alone) {
        __syncwarp();
        return top;
      }
      const int buf = shared_runs++ & 1;
      if (lane == 0) warp_top[buf][warp] = top;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kWarps; ++i) top = max(top, warp_top[buf][i]);
      return top;
    };
    auto new_scale = [&](uint32_t top, bool broken) {
      const float need = scale_for<kInt8>(unpack_16x2<kF16>(top).x);
      float now = place > 0 && (old >= need || isnan(old)) ? old : need;
      if (place > 0 && now != old && !isnan(old)) round_again<kInt8>(w, old, 1.f / now);
      if (kInt8 && broken) now = __int_as_float(0x7fffffff);
      if (lane == 0 && (alone || warp == 0)) *w.scale = now;
      return now;
    };

    // ---- 16-bit floats without their signs are ordered as integers, infinity and NaN behind all numbers: two at a time
    constexpr uint32_t kInf = kF16 ? 0x7c00u : 0x7f80u;
    uint4 held[kHeld];
    uint32_t top = 0u;
    const bool fits = runs[turn].rows && n <= kHeld * w.step;
    if (fits) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int r = w.row0 + i * w.step;
        held[i] = make_uint4(0u, 0u, 0u, 0u);
        if (r < n) held[i] = *reinterpret_cast<const uint4*>(w.in + r * w.in_row);
      }
#pragma unroll
      for (int i = 0; i < kHeld; ++i) top = larger(top, held[i]);
    } else {
      for (int r = w.row0; r < n; r += w.step)
        if (block_of(t0 + r) >= 0) top = larger(top, *reinterpret_cast<const uint4*>(w.in + r * w.in_row));
    }
    top = over_warps(top);
    const bool broken = top >= kInf;  // the same in all warps of the run
    if (broken) {  // the largest finite one
      top = 0u;
      for (int r = w.row0; r < n; r += w.step)
        if (block_of(t0 + r) >= 0) top = larger_finite<kInf>(top, *reinterpret_cast<const uint4*>(w.in + r * w.in_row));
      top = over_warps(top);
    }
    const float now = new_scale(top, broken);

    // ---- codes. All elements are within the largest code where none is infinite or NaN; with a scale that is a power of two, multiplying by the
    // reciprocal is dividing. Elsewhere each element is looked at.
    if (fits && !broken && (__float_as_uint(now) & 0x7fffffu) == 0) {
      const float inv = 1.f / now;
      uint8_t* to = w.cache + place * w.row;
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int r = w.row0 + i * w.step;
        if (r >= n) continue;
        float v[8];
        to_floats<kF16>(held[i], v);
        *reinterpret_cast<uint2*>(to + r * w.row) =
            make_uint2(values_to_codes_within<kInt8>(v[0], v[1], v[2], v[3], inv), values_to_codes_within<kInt8>(v[4], v[5], v[6], v[7], inv));
      }
    } else {
      for (int r = w.row0; r < n; r += w.step) {
        const int slot = p.slots[t0 + r];
        // the same slot again with the next token: the later stays
        if (block_of(t0 + r) < 0 || (r + 1 < n && p.slots[t0 + r + 1] == slot)) continue;
        float v[8];
        to_floats<kF16>(*reinterpret_cast<const uint4*>(w.in + r * w.in_row), v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __fdiv_rn(v[e], now);
        *reinterpret_cast<uint2*>(w.cache + (slot & mask) * w.row) = make_uint2(values_to_codes<kInt8>(v[0], v[1], v[2], v[3]), values_to_codes<kInt8>(v[4], v[5], v[6], v[7]));
      }
    }
  }
}

int check_input(const char* name, const void* ptr, int64_t row, int64_t head, int tokens, int heads) {
  if (ptr == nullptr || (reinterpret_cast<uintptr_t>(ptr) & 15u) != 0) {
    set_error("cache_store: %s must be a 16-byte aligned device pointer", name);
    return SDPA_B200_INVALID_ARG;
  }
  if ((tokens > 1 && (row < 0 || row % 8 != 0)) || (heads > 1 && (head < 0 || head % 8 != 0))) {
    set_error("cache_store: %s needs token and head strides that are multiples of 8 elements (got %lld, %lld)", name, static_cast<long long>(row),
              static_cast<long long>(head));
    return SDPA_B200_INVALID_ARG;
  }
  return SDPA_B200_OK;
}

}  // namespace
}  // namespace sdpa_b200

extern "C" SDPA_B200_API int sdpa_b200_cache_store(const sdpa_b200_cache_params* p, void* stream) {
  using namespace sdpa_b200;
  int st = check_cache(p, "cache_store");
  if (st != SDPA_B200_OK) return st;
  if (p->num_tokens <= 0) {
    set_error("cache_store: num_tokens must be positive (got %d)", p->num_tokens);
    return SDPA_B200_INVALID_ARG;
  }
  if (p->slots == nullptr || (reinterpret_cast<uintptr_t>(p->slots) & 3u) != 0) {
    set_error("cache_store: slots must be a 4-byte aligned device pointer");
    return SDPA_B200_INVALID_ARG;
  }
  if (p->heads_kv > 32767) {
    set_error("cache_store: at most 32767 heads (got %d)", p->heads_kv);
    return SDPA_B200_UNSUPPORTED;
  }
  st = check_input("key", p->key, p->key_row_stride, p->key_head_stride, p->num_tokens, p->heads_kv);
  if (st == SDPA_B200_OK) st = check_input("value", p->value, p->value_row_stride, p->value_head_stride, p->num_tokens, p->heads_kv);
  if (st != SDPA_B200_OK) return st;
  if (p->code == SDPA_B200_INT4 && static_cast<int64_t>(p->num_tokens) * p->heads_kv > INT32_MAX / 2) {  // rows are counted in 32 bits there
    set_error("cache_store: too many tokens (%d) for %d heads", p->num_tokens, p->heads_kv);
    return SDPA_B200_INVALID_ARG;
  }
  st = check_device();
  if (st != SDPA_B200_OK) return st;
  if (p->code == SDPA_B200_INT4) return launch_store4(*p, static_cast<cudaStream_t>(stream));
  StoreParams s;
  s.side[0] = {static_cast<const uint16_t*>(p->key), static_cast<uint8_t*>(p->k_cache), static_cast<float*>(p->k_scale), p->key_row_stride, p->key_head_stride, p->k_block_stride,
               p->k_head_stride, p->k_row_stride};
  s.side[1] = {static_cast<const uint16_t*>(p->value), static_cast<uint8_t*>(p->v_cache), static_cast<float*>(p->v_scale), p->value_row_stride, p->value_head_stride,
               p->v_block_stride, p->v_head_stride, p->v_row_stride};
  s.slots = p->slots;
  s.tokens = p->num_tokens;
  s.heads = p->heads_kv;
  s.shift = block_shift(p->block_size);
  s.num_slots = p->num_blocks << s.shift;
  // few tokens: a warp for each, whatever the runs are; many: windows that begin one or two runs of a block
  const int64_t units = 2 * static_cast<int64_t>(p->heads_kv);
  s.window = p->num_tokens * units <= 148 * 64 ? kWarps : p->block_size >= 64 ? 64 : 32;
  const int64_t ctas = (p->num_tokens + s.window - 1) / s.window * units;
  if (ctas > INT32_MAX) {
    set_error("cache_store: too many tokens (%d) for %d heads", p->num_tokens, p->heads_kv);
    return SDPA_B200_INVALID_ARG;
  }
  const unsigned grid = static_cast<unsigned>(ctas);
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const bool f16 = p->dtype == SDPA_B200_F16;
  cudaError_t err = cudaSuccess;
  auto launch = [&](auto dim, auto int8) {
    constexpr int kD = decltype(dim)::value;
    constexpr bool kInt8 = decltype(int8)::value;
    err = launch_behind(f16 ? store_kernel<kD, kInt8, true> : store_kernel<kD, kInt8, false>, dim3(grid), kWarps * 32, 0, cs, true, 1, s);
  };
  auto launch_dim = [&](auto dim) { p->code == SDPA_B200_INT8 ? launch(dim, std::true_type{}) : launch(dim, std::false_type{}); };
  p->head_dim == 64 ? launch_dim(std::integral_constant<int, 64>{}) : launch_dim(std::integral_constant<int, 128>{});
  if (err != cudaSuccess) {
    set_error("cache_store: launch failed: %s", cudaGetErrorString(err));
    return SDPA_B200_LAUNCH_FAILED;
  }
  count_launch();
  return SDPA_B200_OK;
}
