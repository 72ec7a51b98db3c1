// Keys and values of a serving step into the 4-bit paged cache. No counterpart in the reference, which has no paged cache.
//
// For every 32 elements of a token and head: scale = the smallest number of five significant bits, 2^-100 at least, with 7 * scale >= max |x|, code = round(x / scale), ties to even.
// Five bits, since 7 * 31 < 2^8: a code times its scale is then exact in bf16 (and f16, within its range), so that what attention streams, gathers and reads back is one number; that
// costs a step of 1/32 more on average. x has at most 11 bits, a scale 5: no quotient but a tie itself comes nearer than 2^-12 to the middle of two codes, so x * (1 / scale) with one
// correction step, which gives quotients of few bits exactly, rounds as the exact quotient does.
//
// Measured: 8192 tokens of 4 prompts, 8 heads of 128, bf16 beside their queries: 15.6 us with 8 elements a thread, divisions and a conversion for each element (155 instructions for 8 elements, 71% of the
// issue slots); 13.6 without the divisions; 10.6 with 16 elements a thread, two times; 10.0 with 16 once (4.3 TB/s), 12.5 four times. 64 tokens 3.7,
// which is a launch.
//
// A scale depends on its own 32 elements only: no runs to find, nothing read back, no order among tokens. A thread has 16 elements, two threads a scale.
#include <type_traits>

#include "cache_common.cuh"

namespace sdpa_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 16;  // elements of a thread

struct Store4Side {
  const uint16_t* in;
  uint8_t* cache;
  uint16_t* scale;
  int64_t in_row, in_head, block, head, row;
};

struct Store4Params {
  Store4Side side[2];  // keys, values
  const int32_t* slots;
  int tokens, heads, num_slots, shift;
  uint32_t heads_inv;  // row / heads = (high half of row * heads_inv + row) >> heads_log, for rows below 2^31
  int heads_log;
};

// A thread has a part of one row (a head of a token)
template <int kD, bool kF16>
__global__ void __launch_bounds__(kThreads) store4_kernel(const Store4Params p) {
  constexpr int kLanes = kD / kPer, kRowsAtOnce = kThreads / kLanes;
  constexpr uint32_t kInf = kF16 ? 0x7c00u : 0x7f80u;
  const Store4Side& x = p.side[blockIdx.x & 1];
  const int at = threadIdx.x % kLanes * kPer;
  const int row = static_cast<int>(blockIdx.x >> 1) * kRowsAtOnce + threadIdx.x / kLanes, t = (__umulhi(row, p.heads_inv) + row) >> p.heads_log, head = row - t * p.heads;
  launch_dependents();
  wait_for_previous_grid();
  uint4 w[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
  int slot = -1;
  if (t < p.tokens) {
    slot = p.slots[t];
    if (t + 1 < p.tokens && p.slots[t + 1] == slot) slot = -1;  // the same slot again with the next token: the later stays
    const uint4* src = reinterpret_cast<const uint4*>(x.in + t * x.in_row + head * x.in_head + at);
    w[0] = src[0], w[1] = src[1];
  }
  const uint32_t held[kPer / 2] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
  // 16-bit floats without their signs are ordered as integers, infinity and NaN behind all numbers
  uint32_t top = 0u;
#pragma unroll
  for (int e = 0; e < kPer / 2; ++e) top = __vmaxu2(top, held[e] & 0x7fff7fffu);
  top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top & 0xffffu, top >> 16);
  const bool bad = top >= kInf;
  // A little less than 1/7: what is 7 times a number of five bits does not get above it, and no other comes nearer than 2^-12 to one
  const float seventh = unpack_16x2<kF16>(top).x * 0x1.249248p-3f;
  const float scale = bad ? 1.f : fmaxf(__uint_as_float((__float_as_uint(seventh) + 0x7ffffu) & 0xfff80000u), 0x1p-100f);
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale));
  uint32_t packed[kPer / 8];
#pragma unroll
  for (int k = 0; k < kPer / 8; ++k) {
    uint32_t code[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 v = unpack_16x2<kF16>(held[4 * k + e]);
      const float2 q = mul2(v, make_float2(inv, inv));
      const float2 off = fma2(q, make_float2(-scale, -scale), v);
      const float2 n = add2(fma2(off, make_float2(inv, inv), q), make_float2(12582912.f, 12582912.f));  // 1.5 * 2^23 + x has x, rounded, in its low bits
      code[2 * e] = __float_as_uint(n.x);
      code[2 * e + 1] = __float_as_uint(n.y);
    }
    auto bytes = [&](int e) { return __byte_perm(__byte_perm(code[e], code[e + 2], 0x0040), __byte_perm(code[e + 4], code[e + 6], 0x0040), 0x5410); };
    packed[k] = (bytes(0) & 0x0f0f0f0fu) | (bytes(1) << 4 & 0xf0f0f0f0u);
    if (bad) packed[k] = 0u;
  }
  if (slot < 0 || slot >= p.num_slots) return;
  const int block = slot >> p.shift, place = slot & ((1 << p.shift) - 1);
  *reinterpret_cast<uint2*>(x.cache + block * x.block + head * x.head + place * x.row + at / 2) = make_uint2(packed[0], packed[1]);
  if (at % kScaleGroup == 0)
    x.scale[((((static_cast<int64_t>(block) * p.heads + head) << p.shift) + place) * kD + at) / kScaleGroup] = bad ? 0x7fc0u : static_cast<uint16_t>(__float_as_uint(scale) >> 16);
}

}  // namespace

int launch_store4(const sdpa_b200_cache_params& p, cudaStream_t stream) {
  Store4Params s;
  s.side[0] = {static_cast<const uint16_t*>(p.key), static_cast<uint8_t*>(p.k_cache), static_cast<uint16_t*>(p.k_scale), p.key_row_stride, p.key_head_stride,
               p.k_block_stride, p.k_head_stride, p.k_row_stride};
  s.side[1] = {static_cast<const uint16_t*>(p.value), static_cast<uint8_t*>(p.v_cache), static_cast<uint16_t*>(p.v_scale), p.value_row_stride, p.value_head_stride,
               p.v_block_stride, p.v_head_stride, p.v_row_stride};
  s.slots = p.slots;
  s.tokens = p.num_tokens;
  s.heads = p.heads_kv;
  s.shift = block_shift(p.block_size);
  s.num_slots = p.num_blocks << s.shift;
  for (s.heads_log = 0; (1 << s.heads_log) < p.heads_kv;) ++s.heads_log;
  s.heads_inv = static_cast<uint32_t>(((1ull << 32) * ((1ull << s.heads_log) - p.heads_kv)) / p.heads_kv + 1);
  const int64_t rows = static_cast<int64_t>(p.num_tokens) * p.heads_kv;
  const bool f16 = p.dtype == SDPA_B200_F16;
  cudaError_t err = cudaSuccess;
  auto launch = [&](auto dim) {
    constexpr int kD = decltype(dim)::value, kRowsOfCta = kThreads / (kD / kPer);
    const unsigned grid = static_cast<unsigned>(2 * ((rows + kRowsOfCta - 1) / kRowsOfCta));
    err = launch_behind(f16 ? store4_kernel<kD, true> : store4_kernel<kD, false>, dim3(grid), kThreads, 0, stream, true, 1, s);
  };
  p.head_dim == 64 ? launch(std::integral_constant<int, 64>{}) : launch(std::integral_constant<int, 128>{});
  if (err != cudaSuccess) {
    set_error("cache_store: launch failed: %s", cudaGetErrorString(err));
    return SDPA_B200_LAUNCH_FAILED;
  }
  count_launch();
  return SDPA_B200_OK;
}

}  // namespace sdpa_b200
