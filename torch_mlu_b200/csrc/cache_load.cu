// Tokens of requests out of the paged cache, as packed 16-bit keys and values. No counterpart in the reference, which has no paged cache.
//
// Row cu[b] + i is token first[b] + i of request b: code * scale, a product in 32 bits, rounded to 16. Bound by HBM: 4.5 or 8 bits read and 16 written per element.
// A CTA has 64 rows of some heads. It counts the requests that end in front of its first row with all threads at once; what stands behind is found from there.
// Measured, 8 heads of 128: 16 requests of 4096 to 8192 tokens out of 4 bits 113 us with each element converted by itself and each head's addresses anew, 88 now (5.2 TB/s); 8 of 8192 out of e4m3 62 (5.7 TB/s);
// 301 tokens 5.2 to 6.0, four latencies behind the launch, and the host. Eight elements a thread instead of 16 89 and 66, five CTAs on an SM by fewer registers 94 and 69.
#include <algorithm>
#include <type_traits>

#include "cache_common.cuh"

namespace sdpa_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kTokens = 64;  // of a CTA
constexpr int kPer = 16;     // elements of a thread: 32 bytes of the result

struct LoadParams {
  const uint8_t* cache[2];
  const void* scale[2];
  uint16_t* out[2];
  int64_t block[2], head[2], row[2];
  const int32_t* block_table;
  const int32_t* cu;
  const int32_t* first;  // or null
  int64_t table_stride;
  int batch, rows, heads, heads_each, max_blocks, num_blocks, shift;
};

template <int kD, int kCode, bool kF16>
__global__ void __launch_bounds__(kThreads) load_kernel(const LoadParams p) {
  constexpr int kLanes = kD / kPer, kRowsAtOnce = kThreads / kLanes, kTimes = kTokens / kRowsAtOnce;
  const int tid = threadIdx.x, at = tid % kLanes * kPer, row0 = blockIdx.x * kTokens;
  launch_dependents();
  wait_for_previous_grid();
  int ended = 0;  // requests that end at or in front of the CTA's first row
  for (int base = 0; base < p.batch; base += kThreads) ended += __syncthreads_count(base + tid < p.batch && p.cu[base + tid + 1] <= row0);
  int id[kTimes], place[kTimes];  // block; -1: none in the cache, -2: no request's row
#pragma unroll
  for (int i = 0; i < kTimes; ++i) {
    const int row = row0 + tid / kLanes + i * kRowsAtOnce;
    int b = ended;
    if (b < p.batch && p.cu[b + 1] <= row) {
      int behind = p.batch;
      for (++b; b < behind;) {
        const int mid = (b + behind) / 2;
        if (p.cu[mid + 1] <= row) b = mid + 1;
        else behind = mid;
      }
    }
    id[i] = -2;
    place[i] = 0;
    const int begin = b < p.batch ? p.cu[b] : 0;
    if (b < p.batch && row >= begin) {
      const int64_t token = static_cast<int64_t>(p.first ? p.first[b] : 0) + row - begin, page = token >> p.shift;
      id[i] = token >= 0 && page < p.max_blocks ? p.block_table[b * p.table_stride + page] : -1;
      if (id[i] < 0 || id[i] >= p.num_blocks) id[i] = -1;
      place[i] = static_cast<int>(token) & ((1 << p.shift) - 1);
    }
  }
  const int h0 = blockIdx.y * p.heads_each, h1 = min(h0 + p.heads_each, p.heads);
  const uint8_t* codes[kTimes][2];
  int64_t scale_at[kTimes];
#pragma unroll
  for (int i = 0; i < kTimes; ++i) {
#pragma unroll
    for (int x = 0; x < 2; ++x) codes[i][x] = p.cache[x] + id[i] * p.block[x] + h0 * p.head[x] + place[i] * p.row[x] + Span<kCode, kPer>::code_at(at);
    scale_at[i] = Span<kCode, kPer>::scale_at(id[i], p.heads, h0, place[i], p.shift, kD, at);
  }
#pragma unroll 2
  for (int h = h0; h < h1; ++h) {
    Span<kCode, kPer> w[kTimes][2];
#pragma unroll
    for (int i = 0; i < kTimes; ++i)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        w[i][x].clear();
        w[i][x].scale = id[i] == -1 ? __int_as_float(0x7fffffff) : 0.f;
        if (id[i] >= 0) w[i][x].load(codes[i][x], p.scale[x], scale_at[i]);
        codes[i][x] += p.head[x];
        if (x == 1) scale_at[i] += Span<kCode, kPer>::scale_step(p.shift, kD);
      }
#pragma unroll
    for (int i = 0; i < kTimes; ++i) {
      const int row = row0 + tid / kLanes + i * kRowsAtOnce;
      if (row >= p.rows) continue;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float scale = fabsf(w[i][x].scale) == INFINITY ? __int_as_float(0x7fffffff) : w[i][x].scale;
        float v[kPer];
        w[i][x].values(v);
        write_finite<kF16>(p.out[x] + (static_cast<int64_t>(row) * p.heads + h) * kD + at, v, scale);
      }
    }
  }
}

}  // namespace
}  // namespace sdpa_b200

extern "C" SDPA_B200_API int sdpa_b200_cache_load(const sdpa_b200_cache_params* p, void* stream) {
  using namespace sdpa_b200;
  int st = check_cache(p, "cache_load");
  if (st != SDPA_B200_OK) return st;
  if (p->num_tokens <= 0 || p->batch <= 0 || p->max_blocks <= 0 || p->table_stride < p->max_blocks) {
    set_error("cache_load: num_tokens, batch and max_blocks must be positive, a table row must hold max_blocks (got %d, %d, %d, %lld)", p->num_tokens, p->batch, p->max_blocks,
              static_cast<long long>(p->table_stride));
    return SDPA_B200_INVALID_ARG;
  }
  const void* words[3] = {p->block_table, p->cu_seqlens_k, p->first};
  for (int i = 0; i < 3; ++i) {
    if ((words[i] == nullptr && i < 2) || (reinterpret_cast<uintptr_t>(words[i]) & 3u) != 0) {
      set_error("cache_load: block_table and cu_seqlens_k must be given, and 4-byte aligned as first");
      return SDPA_B200_INVALID_ARG;
    }
  }
  const void* outs[2] = {p->key_out, p->value_out};
  for (int i = 0; i < 2; ++i) {
    if (outs[i] == nullptr || (reinterpret_cast<uintptr_t>(outs[i]) & 31u) != 0) {
      set_error("cache_load: %s must be a 32-byte aligned device pointer", i ? "value_out" : "key_out");
      return SDPA_B200_INVALID_ARG;
    }
  }
  if (p->num_tokens > INT32_MAX - kTokens) {
    set_error("cache_load: too many rows (%d)", p->num_tokens);
    return SDPA_B200_UNSUPPORTED;
  }
  st = check_device();
  if (st != SDPA_B200_OK) return st;
  LoadParams l;
  l.cache[0] = static_cast<const uint8_t*>(p->k_cache);
  l.cache[1] = static_cast<const uint8_t*>(p->v_cache);
  l.scale[0] = p->k_scale;
  l.scale[1] = p->v_scale;
  l.out[0] = static_cast<uint16_t*>(p->key_out);
  l.out[1] = static_cast<uint16_t*>(p->value_out);
  l.block[0] = p->k_block_stride, l.head[0] = p->k_head_stride, l.row[0] = p->k_row_stride;
  l.block[1] = p->v_block_stride, l.head[1] = p->v_head_stride, l.row[1] = p->v_row_stride;
  l.block_table = p->block_table;
  l.cu = p->cu_seqlens_k;
  l.first = p->first;
  l.table_stride = p->table_stride;
  l.batch = p->batch;
  l.rows = p->num_tokens;
  l.heads = p->heads_kv;
  l.max_blocks = p->max_blocks;
  l.num_blocks = p->num_blocks;
  l.shift = block_shift(p->block_size);
  const int64_t tiles = (static_cast<int64_t>(p->num_tokens) + kTokens - 1) / kTokens;
  // all heads a CTA where that fills the GPU: the rows' places are found once
  const int64_t wanted = std::max<int64_t>(1, tiles * p->heads_kv / (148 * 8));
  l.heads_each = static_cast<int>(std::max<int64_t>(std::min<int64_t>(wanted, p->heads_kv), (p->heads_kv + 65534) / 65535));
  const dim3 grid(static_cast<unsigned>(tiles), (p->heads_kv + l.heads_each - 1) / l.heads_each);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool f16 = p->dtype == SDPA_B200_F16;
  cudaError_t err = cudaSuccess;
  auto launch = [&](auto dim, auto code) {
    constexpr int kD = decltype(dim)::value, kCode = decltype(code)::value;
    err = launch_behind(f16 ? load_kernel<kD, kCode, true> : load_kernel<kD, kCode, false>, grid, kThreads, 0, s, true, 1, l);
  };
  auto launch_dim = [&](auto dim) {
    if (p->code == SDPA_B200_INT8) launch(dim, std::integral_constant<int, SDPA_B200_INT8>{});
    else if (p->code == SDPA_B200_INT4) launch(dim, std::integral_constant<int, SDPA_B200_INT4>{});
    else launch(dim, std::integral_constant<int, SDPA_B200_E4M3>{});
  };
  p->head_dim == 64 ? launch_dim(std::integral_constant<int, 64>{}) : launch_dim(std::integral_constant<int, 128>{});
  if (err != cudaSuccess) {
    set_error("cache_load: launch failed: %s", cudaGetErrorString(err));
    return SDPA_B200_LAUNCH_FAILED;
  }
  count_launch();
  return SDPA_B200_OK;
}
