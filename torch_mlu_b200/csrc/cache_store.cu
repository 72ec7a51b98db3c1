// Keys and values of a serving step into the 8-bit paged cache. No counterpart in the reference, which has no paged cache.
//
// Per (block, head) that gets tokens: need = the smallest power of two at which the largest new element is a code, scale = max(old, need) where
// the block holds earlier tokens, code = round(x / scale). Decoding raises the scale of a block that fills up token by token; earlier tokens are then
// read, multiplied by old / scale and rounded again. With powers of two that costs e4m3 only what falls below its smallest numbers, and a
// dequantised element is exact in 16 bits.
//
// Bound by HBM for prompts (two bytes read and one written per element), by latency for decode steps. The tokens of one block stand next to each other,
// so a run of them is found from the slots alone: it begins where a token's block is not that of the token with a place in front. A warp takes (a run, a head,
// keys or values): the first pass over its rows gives the largest element, the second the codes.
#include "cache_common.cuh"

namespace sdpa_b200 {
namespace {

constexpr int kWarps = 4;

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
};

template <bool kF16>
__device__ __forceinline__ void to_floats(const uint4& w, float (&x)[8]) {
  const float2 a = unpack_16x2<kF16>(w.x), b = unpack_16x2<kF16>(w.y), c = unpack_16x2<kF16>(w.z), d = unpack_16x2<kF16>(w.w);
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y, x[4] = c.x, x[5] = c.y, x[6] = d.x, x[7] = d.y;
}

template <int kD, bool kInt8, bool kF16>
__global__ void __launch_bounds__(kWarps * 32) store_kernel(const StoreParams p) {
  constexpr int kLanes = kD / 8, kRows = 32 / kLanes;  // lanes per row, rows per step of the warp
  const int lane = threadIdx.x & 31, sub = lane / kLanes, at = lane % kLanes * 8;
  const int t0 = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int head = blockIdx.y >> 1;
  if (t0 >= p.tokens) return;
  auto block_of = [&](int t) {
    const int slot = p.slots[t];
    return slot < 0 || slot >= p.num_slots ? -1 : slot >> p.shift;
  };
  const int block = block_of(t0);
  if (block < 0) return;
  // first of its run? The nearest token in front that has a place, within 32
  const int front = lane < t0 ? block_of(t0 - 1 - lane) : -1;
  const unsigned placed = __ballot_sync(0xffffffffu, front >= 0), mine = __ballot_sync(0xffffffffu, front == block);
  if ((placed & -placed & mine) != 0) return;
  int n = 1;  // tokens of the run, and of those left out in between
  for (;;) {
    const int b = t0 + n + lane < p.tokens ? block_of(t0 + n + lane) : -1;
    const unsigned same = __ballot_sync(0xffffffffu, b == block), other = __ballot_sync(0xffffffffu, b >= 0 && b != block);
    const unsigned run = same & (other == 0 ? ~0u : (other & -other) - 1);  // in front of the first token of another block
    if (run != 0) n += 32 - __clz(run);
    if (run == 0 || other != 0) break;
  }
  const StoreSide& x = p.side[blockIdx.y & 1];
  const uint16_t* in = x.in + t0 * x.in_row + head * x.in_head + at;
  uint8_t* cache = x.cache + block * x.block + head * x.head + at;
  const int mask = (1 << p.shift) - 1, place = p.slots[t0] & mask;

  // ---- the largest finite element
  float largest = 0.f;
  bool broken = false;
  for (int r = sub; r < n; r += kRows) {
    if (block_of(t0 + r) < 0) continue;
    float v[8];
    to_floats<kF16>(*reinterpret_cast<const uint4*>(in + r * x.in_row), v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = fabsf(v[e]);
      if (a < INFINITY) largest = fmaxf(largest, a);
      else broken = true;
    }
  }
#pragma unroll
  for (int d = 1; d < 32; d *= 2) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, d));
  broken = __any_sync(0xffffffffu, broken);
  float* scale = x.scale + static_cast<int64_t>(block) * p.heads + head;
  const float need = scale_for<kInt8>(largest);
  float now = need;
  if (place > 0) {
    const float old = *scale;
    now = old >= need || isnan(old) ? old : need;
    if (now != old && !isnan(old)) {
      // ---- the scale has grown: earlier tokens are rounded again
      const float down = 1.f / now;  // a power of two: exact
      for (int r = sub; r < place; r += kRows) {
        const uint2 codes = *reinterpret_cast<const uint2*>(cache + r * x.row);
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
        *reinterpret_cast<uint2*>(cache + r * x.row) = make_uint2(values_to_codes<kInt8>(v[0], v[1], v[2], v[3]), values_to_codes<kInt8>(v[4], v[5], v[6], v[7]));
      }
    }
  }
  if (kInt8 && broken) now = __int_as_float(0x7fffffff);
  __syncwarp();  // every lane has read the old scale
  if (lane == 0) *scale = now;

  // ---- codes
  const bool exact = (__float_as_uint(now) & 0x7fffffu) == 0;  // a power of two: multiplying by the reciprocal is dividing
  const float inv = 1.f / now;
  for (int r = sub; r < n; r += kRows) {
    const int slot = p.slots[t0 + r];
    if (slot < 0 || slot >= p.num_slots || (r + 1 < n && p.slots[t0 + r + 1] == slot)) continue;  // the next token has the same place: that one stays
    float v[8];
    to_floats<kF16>(*reinterpret_cast<const uint4*>(in + r * x.in_row), v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = exact ? v[e] * inv : __fdiv_rn(v[e], now);
    *reinterpret_cast<uint2*>(cache + (slot & mask) * x.row) = make_uint2(values_to_codes<kInt8>(v[0], v[1], v[2], v[3]), values_to_codes<kInt8>(v[4], v[5], v[6], v[7]));
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
  st = check_device();
  if (st != SDPA_B200_OK) return st;
  StoreParams s;
  s.side[0] = {static_cast<const uint16_t*>(p->key), static_cast<uint8_t*>(p->k_cache), p->k_scale, p->key_row_stride, p->key_head_stride, p->k_block_stride,
               p->k_head_stride, p->k_row_stride};
  s.side[1] = {static_cast<const uint16_t*>(p->value), static_cast<uint8_t*>(p->v_cache), p->v_scale, p->value_row_stride, p->value_head_stride,
               p->v_block_stride, p->v_head_stride, p->v_row_stride};
  s.slots = p->slots;
  s.tokens = p->num_tokens;
  s.heads = p->heads_kv;
  s.shift = block_shift(p->block_size);
  s.num_slots = p->num_blocks << s.shift;
  const dim3 grid((p->num_tokens + kWarps - 1) / kWarps, 2 * p->heads_kv);
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const bool f16 = p->dtype == SDPA_B200_F16;
  auto launch = [&](auto dim, auto int8) {
    constexpr int kD = decltype(dim)::value;
    constexpr bool kInt8 = decltype(int8)::value;
    if (f16) store_kernel<kD, kInt8, true><<<grid, kWarps * 32, 0, cs>>>(s);
    else store_kernel<kD, kInt8, false><<<grid, kWarps * 32, 0, cs>>>(s);
  };
  auto launch_dim = [&](auto dim) { p->code == SDPA_B200_INT8 ? launch(dim, std::true_type{}) : launch(dim, std::false_type{}); };
  p->head_dim == 64 ? launch_dim(std::integral_constant<int, 64>{}) : launch_dim(std::integral_constant<int, 128>{});
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) {
    set_error("cache_store: launch failed: %s", cudaGetErrorString(err));
    return SDPA_B200_LAUNCH_FAILED;
  }
  count_launch();
  return SDPA_B200_OK;
}
