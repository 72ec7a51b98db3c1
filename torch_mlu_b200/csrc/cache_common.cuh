// The 8-bit codes of the paged cache (include/sdpa_b200.h): conversions from and to 16-bit and 32-bit values, argument checks.
#pragma once

#include "kernels.h"
#include "ptx_sm100.cuh"

namespace sdpa_b200 {

// four codes -> their values as f16 pairs, exact: bytes 0, 1 to `lo`, bytes 2, 3 to `hi`
template <bool kInt8>
__device__ __forceinline__ void codes_to_f16(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  if constexpr (kInt8) {
    // 0x6400 | (x ^ 0x80) is the f16 number 1024 + 128 + x
    const uint32_t u = codes ^ 0x80808080u;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(__byte_perm(u, 0x64646464u, 0x4140)), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(__byte_perm(u, 0x64646464u, 0x4342)), "r"(0x64806480u));
  } else {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}\n"
        : "=r"(lo), "=r"(hi)
        : "r"(codes));
  }
}
// the same for bytes 0, 2 and 1, 3: what a transposed 16-bit ldmatrix leaves is two neighbouring dimensions of each of two tokens
template <bool kInt8>
__device__ __forceinline__ void codes_to_f16_by_two(uint32_t codes, uint32_t& even, uint32_t& odd) {
  if constexpr (kInt8) {
    const uint32_t u = codes ^ 0x80808080u;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(even) : "r"(__byte_perm(u, 0x64646464u, 0x4240)), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(odd) : "r"(__byte_perm(u, 0x64646464u, 0x4341)), "r"(0x64806480u));
  } else {
    codes_to_f16<false>(__byte_perm(codes, 0u, 0x3120), even, odd);
  }
}

// The smallest power of two 2^k, k >= -100, at which `largest` (finite, not negative) is a code: at most 448 = 1.75 * 2^8 of e4m3, 127 = 1.984375 * 2^6 of int8.
template <bool kInt8>
__device__ __forceinline__ float scale_for(float largest) {
  const uint32_t bits = __float_as_uint(largest), part = bits & 0x7fffffu;
  int k = static_cast<int>(bits >> 23) - 127 - (kInt8 ? 6 : 8) + (part > (kInt8 ? 0x7e0000u : 0x600000u) ? 1 : 0);
  k = k < -100 ? -100 : k;
  return __uint_as_float(static_cast<uint32_t>(k + 127) << 23);
}

// four values in units of their scale -> codes, to the nearest, ties to even. Not a number or infinite: NaN of e4m3 (the hardware conversion would make
// infinity the largest code); int8 has none, its caller marks the scale.
template <bool kInt8>
__device__ __forceinline__ uint32_t values_to_codes(float a, float b, float c, float d) {
  if constexpr (kInt8) {
    auto one = [](float x) { return static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(x, -127.f), 127.f))) & 0xffu; };
    return one(a) | one(b) << 8 | one(c) << 16 | one(d) << 24;
  } else {
    auto fit = [](float x) { return fabsf(x) == INFINITY ? __int_as_float(0x7fffffff) : x; };
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}\n"
        : "=r"(r)
        : "f"(fit(a)), "f"(fit(b)), "f"(fit(c)), "f"(fit(d)));
    return r;
  }
}

// The same for finite values times `inv`, a power of two, that are known to be within the largest code.
template <bool kInt8>
__device__ __forceinline__ uint32_t values_to_codes_within(float a, float b, float c, float d, float inv) {
  if constexpr (kInt8) {
    // 1.5 * 2^23 + x has x, rounded, in its low bits
    auto one = [inv](float x) { return __float_as_uint(fmaf(x, inv, 12582912.f)); };
    return __byte_perm(__byte_perm(one(a), one(b), 0x0040), __byte_perm(one(c), one(d), 0x0040), 0x5410);
  } else {
    const float2 ab = mul2(make_float2(a, b), make_float2(inv, inv)), cd = mul2(make_float2(c, d), make_float2(inv, inv));
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}\n"
        : "=r"(r)
        : "f"(ab.x), "f"(ab.y), "f"(cd.x), "f"(cd.y));
    return r;
  }
}

// log2 of a block size, or -1
inline int block_shift(int block_size) {
  for (int shift = 4; shift <= 7; ++shift)
    if ((1 << shift) == block_size) return shift;
  return -1;
}

// What store and attention want of the cache itself. Touches no device.
inline int check_cache(const sdpa_b200_cache_params* p, const char* who) {
  if (p == nullptr) {
    set_error("%s: params is NULL", who);
    return SDPA_B200_INVALID_ARG;
  }
  if (p->code != SDPA_B200_E4M3 && p->code != SDPA_B200_INT8) {
    set_error("%s: codes must be e4m3 or int8 (code %d)", who, p->code);
    return SDPA_B200_UNSUPPORTED;
  }
  if (p->dtype != SDPA_B200_BF16 && p->dtype != SDPA_B200_F16) {
    set_error("%s: 16-bit tensors must be bf16 or f16 (dtype code %d)", who, p->dtype);
    return SDPA_B200_UNSUPPORTED;
  }
  if (p->head_dim != 64 && p->head_dim != 128) {
    set_error("%s: the 8-bit cache is built for head_dim 64 and 128 (got %d)", who, p->head_dim);
    return SDPA_B200_UNSUPPORTED;
  }
  if (block_shift(p->block_size) < 0) {
    set_error("%s: block_size must be 16, 32, 64 or 128 (got %d)", who, p->block_size);
    return SDPA_B200_INVALID_ARG;
  }
  if (p->num_blocks <= 0 || p->heads_kv <= 0 || static_cast<int64_t>(p->num_blocks) * p->block_size > INT32_MAX) {
    set_error("%s: num_blocks and heads_kv must be positive, num_blocks * block_size below 2^31 (got %d, %d)", who, p->num_blocks, p->heads_kv);
    return SDPA_B200_INVALID_ARG;
  }
  const void* bases[2] = {p->k_cache, p->v_cache};
  const int64_t strides[2][3] = {{p->k_block_stride, p->k_head_stride, p->k_row_stride}, {p->v_block_stride, p->v_head_stride, p->v_row_stride}};
  const int sizes[3] = {p->num_blocks, p->heads_kv, p->block_size};
  for (int x = 0; x < 2; ++x) {
    if (bases[x] == nullptr || (reinterpret_cast<uintptr_t>(bases[x]) & 15u) != 0) {
      set_error("%s: %s_cache must be a 16-byte aligned device pointer", who, x ? "v" : "k");
      return SDPA_B200_INVALID_ARG;
    }
    for (int i = 0; i < 3; ++i) {
      if (sizes[i] > 1 && (strides[x][i] < p->head_dim || strides[x][i] % 16 != 0 || strides[x][i] >= (int64_t(1) << 40))) {
        set_error("%s: %s_cache needs block / head / token strides that are multiples of 16 bytes and at least head_dim (got %lld)", who, x ? "v" : "k",
                  static_cast<long long>(strides[x][i]));
        return SDPA_B200_INVALID_ARG;
      }
    }
  }
  if (p->k_scale == nullptr || p->v_scale == nullptr || ((reinterpret_cast<uintptr_t>(p->k_scale) | reinterpret_cast<uintptr_t>(p->v_scale)) & 3u) != 0) {
    set_error("%s: k_scale and v_scale must be 4-byte aligned device pointers", who);
    return SDPA_B200_INVALID_ARG;
  }
  return SDPA_B200_OK;
}

}  // namespace sdpa_b200
