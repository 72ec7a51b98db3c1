// The codes of the paged cache (include/sdpa_b200.h): conversions from and to 16-bit and 32-bit values, argument checks.
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

// Four bits: eight codes, the even element in the low half of its byte, as their values. 0x6400 | u is the f16 number 1024 + u, with 16 u in its place 1024 + 16 u, u = code + 8
__device__ __forceinline__ void codes4_to_floats(uint32_t codes, float (&x)[8]) {
#pragma unroll
  for (int n = 0; n < 4; ++n) {  // elements n and n + 4
    const uint32_t w = n < 2 ? codes : codes >> 8;
    uint32_t h;
    if (n & 1) asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(h) : "r"((w & 0x00f000f0u) ^ 0x64806480u), "r"(0x2c002c00u), "r"(0xd480d480u));  // / 16 - 72
    else asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(h) : "r"((w & 0x000f000fu) ^ 0x64086408u), "r"(0x64086408u));                              // - 1032
    const float2 f = unpack_16x2<true>(h);
    x[n] = f.x;
    x[n + 4] = f.y;
  }
}

constexpr int kScaleGroup = 32;  // elements of a token and head that share a scale in a 4-bit cache

// kPer elements of a cache of any code, whose scale is one: 16, or 8 of 8 bits
template <int kCode, int kPer>
struct Span {
  static constexpr bool kFour = kCode == SDPA_B200_INT4;
  static constexpr int kWords = kPer * (kFour ? 4 : 8) / 32;
  static_assert(kWords == 2 || kWords == 4, "codes are read 8 or 16 bytes at a time");
  uint32_t codes[kWords];
  float scale;

  // Where elements from `at` on are: their codes, from those of the head's token on, and their scale
  static __device__ __forceinline__ int code_at(int at) { return kFour ? at / 2 : at; }
  static __device__ __forceinline__ int64_t scale_at(int block, int heads, int head, int place, int shift, int head_dim, int at) {
    const int64_t of_head = static_cast<int64_t>(block) * heads + head;
    return kFour ? ((of_head << shift) + place) * (head_dim / kScaleGroup) + at / kScaleGroup : of_head;
  }
  // From one head's scale to the next one's
  static __device__ __forceinline__ int scale_step(int shift, int head_dim) { return kFour ? (head_dim / kScaleGroup) << shift : 1; }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) codes[i] = 0u;
  }
  __device__ __forceinline__ void load(const uint8_t* codes_at, const void* scales, int64_t scale_index) {
    if constexpr (kWords == 4) {
      const uint4 w = *reinterpret_cast<const uint4*>(codes_at);
      codes[0] = w.x, codes[1] = w.y, codes[2] = w.z, codes[3] = w.w;
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(codes_at);
      codes[0] = w.x, codes[1] = w.y;
    }
    scale = kFour ? __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(scales)[scale_index]) << 16) : static_cast<const float*>(scales)[scale_index];
  }
  __device__ __forceinline__ void values(float (&x)[kPer]) const {
#pragma unroll
    for (int i = 0; i < kPer; i += 8) {
      float v[8];
      if constexpr (kFour) {
        codes4_to_floats(codes[i / 8], v);
      } else {
        uint32_t h[4];
        codes_to_f16<kCode == SDPA_B200_INT8>(codes[i / 4], h[0], h[1]);
        codes_to_f16<kCode == SDPA_B200_INT8>(codes[i / 4 + 1], h[2], h[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = unpack_16x2<true>(h[e]);
          v[2 * e] = f.x;
          v[2 * e + 1] = f.y;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i + e] = v[e];
    }
  }
};

// two elements in 16 bits, the largest number of the type where they are beyond it: a code is rounded, and the elements 65504 of f16 or 3.39e38 of bf16 come back as
// 2^16 or 2^128. NaN stays.
template <bool kF16>
__device__ __forceinline__ uint32_t pack_16x2_finite(float lo, float hi) {
  uint32_t r;
  if constexpr (kF16) asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// kPer elements times their scale as 16-bit numbers, 16 bytes at a time or 32, to where as many bytes are aligned
template <bool kF16, int kPer>
__device__ __forceinline__ void write_finite(uint16_t* to, const float (&v)[kPer], float scale) {
  uint32_t f[kPer / 2];
#pragma unroll
  for (int e = 0; e < kPer / 2; ++e) {
    const float2 x = mul2(make_float2(v[2 * e], v[2 * e + 1]), make_float2(scale, scale));
    f[e] = pack_16x2_finite<kF16>(x.x, x.y);
  }
  if constexpr (kPer == 16)
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(f[0]), "r"(f[1]), "r"(f[2]), "r"(f[3]), "r"(f[4]), "r"(f[5]), "r"(f[6]), "r"(f[7]) : "memory");
  else
    *reinterpret_cast<uint4*>(to) = make_uint4(f[0], f[1], f[2], f[3]);
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

// Store of 4-bit codes (cache4_store.cu), of arguments that have been checked
int launch_store4(const sdpa_b200_cache_params& p, cudaStream_t stream);

// Bytes of a token's codes of one head
inline int row_bytes(const sdpa_b200_cache_params& p) { return p.code == SDPA_B200_INT4 ? p.head_dim / 2 : p.head_dim; }

// What store, load and attention want of the cache itself. Touches no device.
inline int check_cache(const sdpa_b200_cache_params* p, const char* who) {
  if (p == nullptr) {
    set_error("%s: params is NULL", who);
    return SDPA_B200_INVALID_ARG;
  }
  if (p->code != SDPA_B200_E4M3 && p->code != SDPA_B200_INT8 && p->code != SDPA_B200_INT4) {
    set_error("%s: codes must be e4m3 or int8, or int4 (code %d)", who, p->code);
    return SDPA_B200_UNSUPPORTED;
  }
  if (p->dtype != SDPA_B200_BF16 && p->dtype != SDPA_B200_F16) {
    set_error("%s: 16-bit tensors must be bf16 or f16 (dtype code %d)", who, p->dtype);
    return SDPA_B200_UNSUPPORTED;
  }
  if (p->head_dim != 64 && p->head_dim != 128) {
    set_error("%s: the %d-bit cache is built for head_dim 64 and 128 (got %d)", who, p->code == SDPA_B200_INT4 ? 4 : 8, p->head_dim);
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
      if (sizes[i] > 1 && (strides[x][i] < row_bytes(*p) || strides[x][i] % 16 != 0 || strides[x][i] >= (int64_t(1) << 40))) {
        set_error("%s: %s_cache needs block / head / token strides that are multiples of 16 bytes and at least head_dim%s (got %lld)", who, x ? "v" : "k",
                  p->code == SDPA_B200_INT4 ? " / 2" : "",
                  static_cast<long long>(strides[x][i]));
        return SDPA_B200_INVALID_ARG;
      }
    }
  }
  const unsigned scale_align = p->code == SDPA_B200_INT4 ? 16 : 4;
  if (p->k_scale == nullptr || p->v_scale == nullptr || ((reinterpret_cast<uintptr_t>(p->k_scale) | reinterpret_cast<uintptr_t>(p->v_scale)) & (scale_align - 1)) != 0) {
    set_error("%s: k_scale and v_scale must be %u-byte aligned device pointers", who, scale_align);
    return SDPA_B200_INVALID_ARG;
  }
  return SDPA_B200_OK;
}

}  // namespace sdpa_b200
