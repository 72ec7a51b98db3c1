// Rotary positions with up to four axes (time, height, width): every row of q and k has its first rotary_dim elements turned, pair by pair, by
// angle_j = position[axis(j)] * inv_freq[j]. The gradient is the same turn backwards. No counterpart in the reference.
//
// The angles are the same for all heads of a token. A block takes a few tokens: its threads form the cosines and sines of those once into
// shared memory, then go over the (token, head, chunk) list, eight pairs a thread, with 16-byte loads and stores. The product of a position
// and a frequency is taken in 64 bits, where it is exact, and brought into [-1, 1] half turns there: at position 10^6 the 32-bit product is off by up to
// 0.03 radians. The rest, in 32 bits, is off by 2e-7.
#include "kernels.h"
#include "ptx_sm100.cuh"

namespace sdpa_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;

struct RotaryTensor {
  const uint16_t* in;
  uint16_t* out;
  int64_t in_batch, in_head, in_row, out_batch, out_head, out_row;
};

struct RotaryParams {
  RotaryTensor q, k;
  const void* positions;
  const float* inv_freq;
  int64_t pos_axis, pos_batch, pos_row;
  int64_t tokens;  // batch * length
  int length, heads_q, heads, head_dim, half;
  int axis_end[3];  // the first pair behind each axis but the last
  int tokens_per_block;
  int positions_64, interleaved;
  float scaling, sign;
};

// One 16-byte chunk of pairs: `a` and `b` hold the pairs' first and second elements of 8 pairs (halves apart), or eight elements = four pairs each
// (interleaved); `cs`: their cosines and sines.
template <bool kF16>
__device__ __forceinline__ uint32_t turn_word(uint32_t first, uint32_t second, const float2& cs0, const float2& cs1, uint32_t& second_out) {
  const float2 x = unpack_16x2<kF16>(first), y = unpack_16x2<kF16>(second);
  second_out = pack_16x2<kF16>(fmaf(x.x, cs0.y, y.x * cs0.x), fmaf(x.y, cs1.y, y.y * cs1.x));
  return pack_16x2<kF16>(fmaf(x.x, cs0.x, -y.x * cs0.y), fmaf(x.y, cs1.x, -y.y * cs1.y));
}
template <bool kF16>
__device__ __forceinline__ uint32_t turn_pair(uint32_t w, const float2& cs) {
  const float2 x = unpack_16x2<kF16>(w);
  return pack_16x2<kF16>(fmaf(x.x, cs.x, -x.y * cs.y), fmaf(x.x, cs.y, x.y * cs.x));
}

template <bool kF16>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  extern __shared__ float2 turns[];  // [tokens_per_block][half]: cosine, sine
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * p.tokens_per_block;
  const int tokens = static_cast<int>(min(static_cast<int64_t>(p.tokens_per_block), p.tokens - token0));
  for (int i = threadIdx.x; i < tokens * p.half; i += kThreads) {
    const int t = i / p.half, j = i - t * p.half;
    const int64_t token = token0 + t, b = token / p.length;
    const int axis = (j >= p.axis_end[0]) + (j >= p.axis_end[1]) + (j >= p.axis_end[2]);
    const int64_t at = axis * p.pos_axis + b * p.pos_batch + (token - b * p.length) * p.pos_row;
    const int64_t pos = p.positions_64 ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
    double x = static_cast<double>(pos) * static_cast<double>(p.inv_freq[j]) * 0.31830988618379067154;  // half turns
    x -= 2.0 * rint(0.5 * x);
    float s, c;
    sincospif(static_cast<float>(x), &s, &c);
    turns[i] = make_float2(c * p.scaling, s * p.scaling * p.sign);
  }
  __syncthreads();
  // chunks of a row: those of the pairs (16 elements each), then those that are copied (8 elements each)
  const int turned = p.half / 8, rest = (p.head_dim - 2 * p.half) / 8, chunks = turned + rest;
  const int per_token = p.heads * chunks;
  for (int i = threadIdx.x; i < tokens * per_token; i += kThreads) {
    const int t = i / per_token, r = i - t * per_token;
    const int h = r / chunks, c = r - h * chunks;
    const int64_t token = token0 + t, b = token / p.length, row = token - b * p.length;
    const bool is_q = h < p.heads_q;
    const RotaryTensor& x = is_q ? p.q : p.k;
    const int head = is_q ? h : h - p.heads_q;
    const uint16_t* in = x.in + b * x.in_batch + head * x.in_head + row * x.in_row;
    uint16_t* out = x.out + b * x.out_batch + head * x.out_head + row * x.out_row;
    if (c >= turned) {
      const int at = 2 * p.half + (c - turned) * 8;
      *reinterpret_cast<uint4*>(out + at) = *reinterpret_cast<const uint4*>(in + at);
      continue;
    }
    const float2* cs = turns + t * p.half + c * 8;
    const int at = p.interleaved ? c * 16 : c * 8, apart = p.interleaved ? 8 : p.half;
    uint4 u = *reinterpret_cast<const uint4*>(in + at), v = *reinterpret_cast<const uint4*>(in + at + apart);
    if (p.interleaved) {
      u.x = turn_pair<kF16>(u.x, cs[0]);
      u.y = turn_pair<kF16>(u.y, cs[1]);
      u.z = turn_pair<kF16>(u.z, cs[2]);
      u.w = turn_pair<kF16>(u.w, cs[3]);
      v.x = turn_pair<kF16>(v.x, cs[4]);
      v.y = turn_pair<kF16>(v.y, cs[5]);
      v.z = turn_pair<kF16>(v.z, cs[6]);
      v.w = turn_pair<kF16>(v.w, cs[7]);
    } else {
      u.x = turn_word<kF16>(u.x, v.x, cs[0], cs[1], v.x);
      u.y = turn_word<kF16>(u.y, v.y, cs[2], cs[3], v.y);
      u.z = turn_word<kF16>(u.z, v.z, cs[4], cs[5], v.z);
      u.w = turn_word<kF16>(u.w, v.w, cs[6], cs[7], v.w);
    }
    *reinterpret_cast<uint4*>(out + at) = u;
    *reinterpret_cast<uint4*>(out + at + apart) = v;
  }
}

int check_rows(const char* name, const void* in, const void* out, const int64_t (&s)[6], int batch, int heads, int length) {
  if (in == nullptr || out == nullptr) {
    set_error("rotary: %s is NULL", name);
    return SDPA_B200_INVALID_ARG;
  }
  if (((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) & 15u) != 0) {
    set_error("rotary: %s must be 16-byte aligned", name);
    return SDPA_B200_INVALID_ARG;
  }
  const int sizes[3] = {batch, heads, length};
  for (int i = 0; i < 6; ++i) {
    if (sizes[i % 3] > 1 && (s[i] < (i < 3 ? 0 : 8) || s[i] % 8 != 0)) {
      set_error("rotary: %s needs batch / head / row strides that are multiples of 8 elements, those of the result positive (got %lld)", name,
                static_cast<long long>(s[i]));
      return SDPA_B200_INVALID_ARG;
    }
  }
  return SDPA_B200_OK;
}

}  // namespace
}  // namespace sdpa_b200

extern "C" SDPA_B200_API int sdpa_b200_rotary(const sdpa_b200_rotary_params* p, void* stream) {
  using namespace sdpa_b200;
  if (p == nullptr) {
    set_error("rotary: params is NULL");
    return SDPA_B200_INVALID_ARG;
  }
  if (p->dtype != SDPA_B200_BF16 && p->dtype != SDPA_B200_F16) {
    set_error("rotary: q and k must be bf16 or f16 (dtype code %d)", p->dtype);
    return SDPA_B200_UNSUPPORTED;
  }
  if (p->batch <= 0 || p->length <= 0 || p->heads_q <= 0 || p->heads_k < 0) {
    set_error("rotary: batch, length and heads_q must be positive (got %d, %d, %d), heads_k not negative (%d)", p->batch, p->length, p->heads_q, p->heads_k);
    return SDPA_B200_INVALID_ARG;
  }
  if (p->head_dim <= 0 || p->head_dim % 8 != 0 || p->head_dim > 256) {
    set_error("rotary: head_dim must be a multiple of 8 and at most 256 (got %d)", p->head_dim);
    return SDPA_B200_INVALID_ARG;
  }
  if (p->rotary_dim <= 0 || p->rotary_dim % 16 != 0 || p->rotary_dim > p->head_dim) {
    set_error("rotary: rotary_dim must be a multiple of 16 and at most head_dim (got %d of %d)", p->rotary_dim, p->head_dim);
    return SDPA_B200_INVALID_ARG;
  }
  if (p->axes < 1 || p->axes > 4) {
    set_error("rotary: positions have one to four axes (got %d)", p->axes);
    return SDPA_B200_INVALID_ARG;
  }
  int64_t pairs = 0;
  for (int a = 0; a < p->axes; ++a) pairs = p->sections[a] < 0 ? -1000000 : pairs + p->sections[a];
  if (pairs != p->rotary_dim / 2) {
    set_error("rotary: sections must not be negative and add up to rotary_dim / 2 = %d", p->rotary_dim / 2);
    return SDPA_B200_INVALID_ARG;
  }
  if (p->positions == nullptr || p->inv_freq == nullptr) {
    set_error("rotary: positions and inv_freq must be given");
    return SDPA_B200_INVALID_ARG;
  }
  const int64_t qs[6] = {p->q_batch_stride, p->q_head_stride, p->q_row_stride, p->qo_batch_stride, p->qo_head_stride, p->qo_row_stride};
  const int64_t ks[6] = {p->k_batch_stride, p->k_head_stride, p->k_row_stride, p->ko_batch_stride, p->ko_head_stride, p->ko_row_stride};
  int st = check_rows("q", p->q, p->q_out, qs, p->batch, p->heads_q, p->length);
  if (st == SDPA_B200_OK && p->heads_k > 0) st = check_rows("k", p->k, p->k_out, ks, p->batch, p->heads_k, p->length);
  if (st != SDPA_B200_OK) return st;
  st = check_device();
  if (st != SDPA_B200_OK) return st;
  RotaryParams r;
  r.q = {static_cast<const uint16_t*>(p->q), static_cast<uint16_t*>(p->q_out), qs[0], qs[1], qs[2], qs[3], qs[4], qs[5]};
  r.k = {static_cast<const uint16_t*>(p->k), static_cast<uint16_t*>(p->k_out), ks[0], ks[1], ks[2], ks[3], ks[4], ks[5]};
  r.positions = p->positions;
  r.inv_freq = p->inv_freq;
  r.pos_axis = p->pos_axis_stride;
  r.pos_batch = p->pos_batch_stride;
  r.pos_row = p->pos_row_stride;
  r.tokens = static_cast<int64_t>(p->batch) * p->length;
  r.length = p->length;
  r.heads_q = p->heads_q;
  r.heads = p->heads_q + p->heads_k;
  r.head_dim = p->head_dim;
  r.half = p->rotary_dim / 2;
  int end = 0;
  for (int a = 0; a < 3; ++a) {
    if (a < p->axes) end += p->sections[a];
    r.axis_end[a] = a < p->axes - 1 ? end : kMaxPairs;
  }
  r.positions_64 = p->positions_64;
  r.interleaved = p->interleaved;
  r.scaling = p->scaling;
  r.sign = p->inverse ? -1.f : 1.f;
  r.tokens_per_block = r.tokens >= 2048 ? 4 : 1;
  const int64_t blocks = (r.tokens + r.tokens_per_block - 1) / r.tokens_per_block;
  if (blocks > 0x7fffffff) {
    set_error("rotary: too many tokens");
    return SDPA_B200_INVALID_ARG;
  }
  const size_t smem = static_cast<size_t>(r.tokens_per_block) * r.half * sizeof(float2);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p->dtype == SDPA_B200_F16) rotary_kernel<true><<<static_cast<unsigned>(blocks), kThreads, smem, s>>>(r);
  else rotary_kernel<false><<<static_cast<unsigned>(blocks), kThreads, smem, s>>>(r);
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) {
    set_error("rotary: launch failed: %s", cudaGetErrorString(err));
    return SDPA_B200_LAUNCH_FAILED;
  }
  count_launch();
  return SDPA_B200_OK;
}
