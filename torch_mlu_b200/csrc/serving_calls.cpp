// The serving operators from tensors to launched kernels: bookkeeping of a step, the 8-bit paged cache, rotary positions with their gradient. Called by
// py_calls.cpp for kv_cache.py and rotary.py: a decode step's kernels run for a few microseconds each, and filling the parameter blocks through ctypes took
// the host 25 to 45 us a call. They are operators of b200_sdpa too, through which a call goes while somebody wants to see it (a tracer, a dispatch mode): what launched
// kernels beside a tracer would leave its results in the traced program as constants.
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/library.h>

#include <algorithm>
#include <cstdlib>

#include "torch_glue.h"

namespace b200_glue {

using at::Tensor;

namespace {

// A CUDA tensor with memory of its own: a wrapper (of torch.func, of a dispatch mode, without data) has nothing that a kernel could read.
void check_plain(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be on a CUDA device (this path has no CPU fallback)");
  constexpr c10::DispatchKeySet wrapped =
      c10::python_ks | c10::functorch_transforms_ks |
      c10::DispatchKeySet({c10::DispatchKey::Functionalize, c10::DispatchKey::Negative, c10::DispatchKey::Conjugate, c10::DispatchKey::ZeroTensor});
  TORCH_CHECK(!t.key_set().has_any(wrapped) && t.layout() == at::kStrided, name, " must be an ordinary tensor");
}

void check_ints(const Tensor& t, const char* name, const Tensor& like) {
  check_plain(t, name);
  TORCH_CHECK(t.scalar_type() == at::kInt && t.device() == like.device(), name, " must be an int32 tensor on the device of the others");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

void check_table(const Tensor& t, const Tensor& like) {
  check_plain(t, "block_table");
  TORCH_CHECK(t.dim() == 2 && t.scalar_type() == at::kInt && t.device() == like.device() && (t.stride(1) == 1 || t.size(1) == 1),
              "block_table must be int32 [requests, max_blocks] with contiguous rows, on the device of the others");
}

// rows of a table with one request, or none, may have any stride
int64_t table_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.size(1), 1); }

int32_t to_int32(int64_t n, const char* name) {
  TORCH_CHECK(n >= INT32_MIN && n <= INT32_MAX, name, " does not fit 32 bits (got ", n, ")");
  return static_cast<int32_t>(n);
}

// Autograd learns that a tensor has been written in place.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// What is differentiated forwards, or backwards, would be left out silently.
void check_no_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), "forward-mode differentiation of ", what, " is not implemented");
}

bool needs_grad(const Tensor& t) { return t.defined() && t.requires_grad() && at::GradMode::is_enabled(); }

// Whether a tracer, a dispatch mode, a functional transform or code below autograd is to see the operators of this thread. (Autocast has nothing to do with them, and inference
// mode, which switches autograd off too, is what servers run in.)
bool calls_are_seen() {
  const auto tls = c10::impl::tls_local_dispatch_key_set();
  return !(c10::default_included_set | c10::autocast_dispatch_keyset).has_all(tls.included_) ||
         (tls.excluded_.has(c10::DispatchKey::AutogradFunctionality) && !c10::InferenceMode::is_enabled()) ||
         c10::impl::TorchDispatchModeTLS::any_modes_set() || torch::jit::tracer::isTracing();
}

// What wraps a tensor (a functional transform, a fake tensor) has no rule for these operators
void check_all_plain(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors) check_plain(*t, "every argument");
}

template <class F>
auto operator_named(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

}  // namespace

namespace {

std::vector<Tensor> launch_plan(const Tensor& cached_lens, const Tensor& new_tokens, const Tensor& block_table, const Tensor& ring, const Tensor& ring_state,
                                int64_t block_size, int64_t num_tokens, bool in_place) {
  check_ints(cached_lens, "cached_lens", cached_lens);
  check_ints(new_tokens, "new_tokens", cached_lens);
  check_ints(ring, "ring", cached_lens);
  check_ints(ring_state, "ring_state", cached_lens);
  check_table(block_table, cached_lens);
  const int64_t B = block_table.size(0);
  TORCH_CHECK(cached_lens.dim() == 1 && cached_lens.size(0) == B && new_tokens.dim() == 1 && new_tokens.size(0) == B && ring.dim() == 1 && ring_state.dim() == 1 &&
                  ring_state.size(0) == 3,
              "cached_lens and new_tokens must be [requests], ring [num_blocks], ring_state [3]");
  TORCH_CHECK(num_tokens > 0, "num_tokens must be positive (got ", num_tokens, ")");
  c10::cuda::CUDAGuard guard(cached_lens.device());
  // the results are cut out of one allocation: five took the host longer than the step takes the GPU
  const int64_t sizes[5] = {in_place ? 0 : B, B + 1, num_tokens, num_tokens, in_place ? 0 : 3};
  const Tensor all = new_tensor({sizes[0] + sizes[1] + sizes[2] + sizes[3] + sizes[4]}, at::kInt, cached_lens);
  std::vector<Tensor> step;
  step.reserve(5);
  int64_t at = 0;
  for (const int64_t n : sizes) {
    Tensor x = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
    x.unsafeGetTensorImpl()->set_storage_offset(at);
    x.unsafeGetTensorImpl()->set_sizes_contiguous(n);
    step.push_back(std::move(x));
    at += n;
  }
  if (in_place) {
    step[0] = cached_lens;
    step[4] = ring_state;
  }
  sdpa_b200_plan_params p = {};
  p.cached_lens = cached_lens.data_ptr<int32_t>();
  p.new_tokens = new_tokens.data_ptr<int32_t>();
  p.block_table = block_table.data_ptr<int32_t>();
  p.ring = ring.data_ptr<int32_t>();
  p.ring_state = ring_state.data_ptr<int32_t>();
  p.seq_lens = step[0].data_ptr<int32_t>();
  p.cu_seqlens = step[1].data_ptr<int32_t>();
  p.positions = step[2].data_ptr<int32_t>();
  p.slots = step[3].data_ptr<int32_t>();
  p.next_state = step[4].data_ptr<int32_t>();
  p.table_stride = table_stride(block_table);
  p.batch = to_int32(B, "requests");
  p.max_blocks = to_int32(block_table.size(1), "max_blocks");
  p.num_blocks = to_int32(ring.size(0), "num_blocks");
  p.block_size = to_int32(block_size, "block_size");
  p.num_tokens = to_int32(num_tokens, "num_tokens");
  check_status(sdpa_b200_plan_step(&p, stream_of(cached_lens)), "sdpa_b200_plan_step");
  for (const Tensor* t : {&block_table, &ring}) written(*t);
  if (in_place) {
    written(cached_lens);
    written(ring_state);
  }
  return step;
}

using PlanResult = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;
PlanResult plan_operator(const Tensor& cached_lens, const Tensor& new_tokens, const Tensor& block_table, const Tensor& ring, const Tensor& ring_state, int64_t block_size,
                         int64_t num_tokens) {
  const auto r = launch_plan(cached_lens, new_tokens, block_table, ring, ring_state, block_size, num_tokens, false);
  return {r[0], r[1], r[2], r[3], r[4]};
}
std::tuple<Tensor, Tensor, Tensor> plan_operator_in_place(const Tensor& cached_lens, const Tensor& new_tokens, const Tensor& block_table, const Tensor& ring,
                                                          const Tensor& ring_state, int64_t block_size, int64_t num_tokens) {
  const auto r = launch_plan(cached_lens, new_tokens, block_table, ring, ring_state, block_size, num_tokens, true);
  return {r[1], r[2], r[3]};
}

}  // namespace

std::vector<Tensor> plan_step(const Tensor& cached_lens, const Tensor& new_tokens, const Tensor& block_table, const Tensor& ring, const Tensor& ring_state,
                              int64_t block_size, int64_t num_tokens, bool in_place) {
  if (!calls_are_seen()) return launch_plan(cached_lens, new_tokens, block_table, ring, ring_state, block_size, num_tokens, in_place);
  check_all_plain({&cached_lens, &new_tokens, &block_table, &ring, &ring_state});
  if (!in_place) {
    static auto op = operator_named<decltype(plan_operator)>("b200_sdpa::plan_step");
    const auto r = op.call(cached_lens, new_tokens, block_table, ring, ring_state, block_size, num_tokens);
    return {std::get<0>(r), std::get<1>(r), std::get<2>(r), std::get<3>(r), std::get<4>(r)};
  }
  static auto op = operator_named<decltype(plan_operator_in_place)>("b200_sdpa::plan_step_");
  const auto r = op.call(cached_lens, new_tokens, block_table, ring, ring_state, block_size, num_tokens);
  return {cached_lens, std::get<0>(r), std::get<1>(r), std::get<2>(r), ring_state};
}

namespace {

void cache_params(sdpa_b200_cache_params& p, const Tensor& x, const char* name, const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs) {
  check_plain(x, name);
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "16-bit tensors must be fp16 or bf16 (got ", x.scalar_type(), ")");
  check_plain(kc, "key_cache");
  check_plain(vc, "value_cache");
  TORCH_CHECK(kc.dim() == 4 && kc.sizes() == vc.sizes(), "key_cache and value_cache must both be [num_blocks, heads_kv, block_size, head_dim]");
  TORCH_CHECK((kc.scalar_type() == at::kFloat8_e4m3fn || kc.scalar_type() == at::kChar) && vc.scalar_type() == kc.scalar_type(),
              "the caches must both be float8_e4m3fn or int8");
  TORCH_CHECK(x.size(-1) == kc.size(3), "the caches must have the head_dim of the other tensors");
  for (const Tensor* t : {&kc, &vc})
    TORCH_CHECK(t->device() == x.device() && t->stride(3) == 1, "the caches must have a contiguous last dimension, on the device of the other tensors");
  for (const Tensor* t : {&ks, &vs}) {
    check_plain(*t, "a scale");
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(0) == kc.size(0) && t->size(1) == kc.size(1) && t->is_contiguous() && t->device() == x.device(),
                "key_scale and value_scale must be contiguous fp32 [num_blocks, heads_kv] on the device of the other tensors");
  }
  p.k_cache = kc.data_ptr();
  p.v_cache = vc.data_ptr();
  p.k_scale = ks.data_ptr<float>();
  p.v_scale = vs.data_ptr<float>();
  p.k_block_stride = kc.stride(0);
  p.k_head_stride = kc.stride(1);
  p.k_row_stride = kc.stride(2);
  p.v_block_stride = vc.stride(0);
  p.v_head_stride = vc.stride(1);
  p.v_row_stride = vc.stride(2);
  p.num_blocks = to_int32(kc.size(0), "num_blocks");
  p.heads_kv = to_int32(kc.size(1), "heads_kv");
  p.block_size = to_int32(kc.size(2), "block_size");
  p.head_dim = to_int32(kc.size(3), "head_dim");
  p.code = kc.scalar_type() == at::kChar ? SDPA_B200_INT8 : SDPA_B200_E4M3;
  p.dtype = x.scalar_type() == at::kHalf ? SDPA_B200_F16 : SDPA_B200_BF16;
}

void launch_store(const Tensor& key, const Tensor& value, const Tensor& slots, const Tensor& key_cache, const Tensor& value_cache, const Tensor& key_scale,
                 const Tensor& value_scale) {
  TORCH_CHECK(key.dim() == 3 && key.sizes() == value.sizes(), "key and value must both be [tokens, heads_kv, head_dim]");
  TORCH_CHECK(key.scalar_type() == value.scalar_type() && key.device() == value.device() && key.stride(2) == 1 && value.stride(2) == 1,
              "key and value must have the same dtype and device, and a contiguous last dimension");
  check_plain(value, "value");
  sdpa_b200_cache_params p = {};
  cache_params(p, key, "key", key_cache, value_cache, key_scale, value_scale);
  TORCH_CHECK(key.size(1) == key_cache.size(1), "the caches must have the heads of key and value");
  for (const Tensor* t : {&key, &value, &key_cache, &value_cache, &key_scale, &value_scale}) {
    TORCH_CHECK(!needs_grad(*t), "the cache keeps no gradient: store keys and values under torch.no_grad()");
    check_no_tangent(*t, "the cache");
  }
  check_ints(slots, "slots", key);
  TORCH_CHECK(slots.dim() == 1 && slots.size(0) == key.size(0), "slots must be [tokens]");
  if (key.size(0) == 0) return;
  TORCH_CHECK(p.k_cache != p.v_cache && p.k_scale != p.v_scale, "keys and values need caches and scales of their own");
  p.key = key.data_ptr();
  p.value = value.data_ptr();
  p.slots = slots.data_ptr<int32_t>();
  p.num_tokens = to_int32(key.size(0), "tokens");
  p.key_row_stride = key.stride(0);
  p.key_head_stride = key.stride(1);
  p.value_row_stride = value.stride(0);
  p.value_head_stride = value.stride(1);
  c10::cuda::CUDAGuard guard(key.device());
  check_status(sdpa_b200_cache_store(&p, stream_of(key)), "sdpa_b200_cache_store");
  for (const Tensor* t : {&key_cache, &value_cache, &key_scale, &value_scale}) written(*t);
}

std::tuple<Tensor, Tensor> launch_attention(const Tensor& query, const Tensor& key_cache, const Tensor& value_cache, const Tensor& key_scale,
                                           const Tensor& value_scale, const Tensor& block_table, const Tensor& seq_lens,
                                           const c10::optional<Tensor>& cu_seqlens, int64_t max_seqlen_q, c10::optional<int64_t> max_seqlen_k, bool causal,
                                           c10::optional<double> scale) {
  TORCH_CHECK(query.dim() == 3 && query.stride(2) == 1, "query must be [tokens, heads_q, head_dim] with a contiguous last dimension");
  sdpa_b200_cache_params p = {};
  cache_params(p, query, "query", key_cache, value_cache, key_scale, value_scale);
  check_table(block_table, query);
  const int64_t B = block_table.size(0), T = query.size(0), H = query.size(1);
  check_ints(seq_lens, "seq_lens", query);
  TORCH_CHECK(seq_lens.dim() == 1 && seq_lens.size(0) == B, "seq_lens must be [requests]");
  if (cu_seqlens.has_value()) {
    check_ints(*cu_seqlens, "cu_seqlens", query);
    TORCH_CHECK(cu_seqlens->dim() == 1 && cu_seqlens->size(0) == B + 1, "cu_seqlens must have requests + 1 entries");
  }
  for (const Tensor* t : {&query, &key_cache, &value_cache, &key_scale, &value_scale}) {
    TORCH_CHECK(!needs_grad(*t), "attention over the cache has no gradient: call it under torch.no_grad()");
    check_no_tangent(*t, "attention over the cache");
  }
  c10::cuda::CUDAGuard guard(query.device());
  Tensor out = new_tensor({T, H, query.size(2)}, query.scalar_type(), query), lse = new_tensor({H, T}, at::kFloat, query);
  if (query.numel() == 0) return {out, lse};
  p.q = query.data_ptr();
  p.out = out.data_ptr();
  p.lse = lse.data_ptr<float>();
  p.q_row_stride = query.stride(0);
  p.q_head_stride = query.stride(1);
  p.o_row_stride = out.stride(0);
  p.o_head_stride = out.stride(1);
  p.block_table = block_table.data_ptr<int32_t>();
  p.seq_lens = seq_lens.data_ptr<int32_t>();
  p.cu_seqlens_q = cu_seqlens.has_value() ? cu_seqlens->data_ptr<int32_t>() : nullptr;
  p.table_stride = table_stride(block_table);
  p.max_blocks = to_int32(block_table.size(1), "max_blocks");
  p.batch = to_int32(B, "requests");
  p.total_q = to_int32(T, "tokens");
  p.heads_q = to_int32(H, "heads_q");
  p.max_seqlen_q = to_int32(max_seqlen_q, "max_seqlen_q");
  p.max_seqlen_k = to_int32(max_seqlen_k.has_value() ? *max_seqlen_k : block_table.size(1) * key_cache.size(2), "max_seqlen_k");
  p.is_causal = causal;
  p.softmax_scale = static_cast<float>(scale_or_default(query, scale));
  p.device_status = reinterpret_cast<uint32_t*>(status_word(query.get_device()).data_ptr());
  size_t bytes = 0;
  check_status(sdpa_b200_cache_attention_workspace_bytes(&p, &bytes), "workspace query");
  const c10::DataPtr ws = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);  // back to torch's stream-ordered pool at the end of this call
  check_status(sdpa_b200_cache_attention(&p, ws.get(), bytes, stream_of(query)), "sdpa_b200_cache_attention");
  return {out, lse};
}

}  // namespace

void cache_store(const Tensor& key, const Tensor& value, const Tensor& slots, const Tensor& key_cache, const Tensor& value_cache, const Tensor& key_scale,
                 const Tensor& value_scale) {
  if (!calls_are_seen()) return launch_store(key, value, slots, key_cache, value_cache, key_scale, value_scale);
  check_all_plain({&key, &value, &slots, &key_cache, &value_cache, &key_scale, &value_scale});
  static auto op = operator_named<decltype(launch_store)>("b200_sdpa::cache_store_");
  op.call(key, value, slots, key_cache, value_cache, key_scale, value_scale);
}

std::tuple<Tensor, Tensor> cache_attention(const Tensor& query, const Tensor& key_cache, const Tensor& value_cache, const Tensor& key_scale,
                                           const Tensor& value_scale, const Tensor& block_table, const Tensor& seq_lens,
                                           const c10::optional<Tensor>& cu_seqlens, int64_t max_seqlen_q, c10::optional<int64_t> max_seqlen_k, bool causal,
                                           c10::optional<double> scale) {
  if (!calls_are_seen())
    return launch_attention(query, key_cache, value_cache, key_scale, value_scale, block_table, seq_lens, cu_seqlens, max_seqlen_q, max_seqlen_k, causal, scale);
  check_all_plain({&query, &key_cache, &value_cache, &key_scale, &value_scale, &block_table, &seq_lens});
  if (cu_seqlens.has_value()) check_plain(*cu_seqlens, "cu_seqlens");
  static auto op = operator_named<decltype(launch_attention)>("b200_sdpa::cache_attention");
  return op.call(query, key_cache, value_cache, key_scale, value_scale, block_table, seq_lens, cu_seqlens, max_seqlen_q, max_seqlen_k, causal, scale);
}

// ------------------------------------------------------------------------- rotary positions
namespace {

struct RotaryCall {
  std::vector<int64_t> sections;  // empty: positions have no axis dimension
  bool interleaved, inverse;
  double scaling;
};

void rotary_tensor(const Tensor& x, const char* name, const Tensor& q) {
  check_plain(x, name);
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "query and key must be bf16 or fp16 (", name, " is ", x.scalar_type(), ")");
  TORCH_CHECK(x.scalar_type() == q.scalar_type(), "query and key must be bf16 or fp16, both the same");
  TORCH_CHECK(x.dim() == q.dim() && x.device() == q.device() && x.size(-1) == q.size(-1), "query and key must agree in dimensions, device and head_dim");
  TORCH_CHECK(x.dim() != 3 || x.size(0) == q.size(0), "query and key must have the same tokens");
  TORCH_CHECK(x.dim() != 4 || (x.size(0) == q.size(0) && x.size(2) == q.size(2)), "query and key must have the same batch and length");
}

void strides_of(const Tensor& t, int64_t& batch, int64_t& head, int64_t& row) {
  batch = t.dim() == 4 ? t.stride(0) : 0;
  head = t.stride(1);
  row = t.stride(t.dim() == 4 ? 2 : 0);
}

// Whether two tensors whose elements are a row apart by the same strides have any in common: slices of one projection do not, overlapping ones do. (Other strides are not
// looked at.)
bool rows_overlap(const Tensor& x, const Tensor& y) {
  if (x.numel() == 0 || y.numel() == 0) return false;
  int64_t xs[3], ys[3];  // batch, head, row
  strides_of(x, xs[0], xs[1], xs[2]);
  strides_of(y, ys[0], ys[1], ys[2]);
  const bool packed = x.dim() == 3;
  const int64_t xn[3] = {packed ? 1 : x.size(0), x.size(1), x.size(packed ? 0 : 2)}, yn[3] = {xn[0], y.size(1), xn[2]}, width = x.size(-1);
  // where an element of x and one of y are the same, the distance of the tensors is a sum of n * stride with n from -(y's size - 1) to x's size - 1, and of less than a row
  struct Step {
    int64_t stride, least, most;
  };
  Step steps[3];
  int n_steps = 0;
  for (int i = 0; i < 3; ++i) {
    if (xn[i] == 1 && yn[i] == 1) continue;
    if (xn[i] > 1 && yn[i] > 1 && xs[i] != ys[i]) return false;
    steps[n_steps++] = {xn[i] > 1 ? xs[i] : ys[i], 1 - yn[i], xn[i] - 1};
  }
  std::sort(steps, steps + n_steps, [](const Step& a, const Step& b) { return a.stride > b.stride; });
  auto reaches = [&](auto&& self, int i, int64_t distance) -> bool {
    if (i == n_steps) return std::abs(distance) < width;
    const int64_t n = distance / steps[i].stride;  // strides are positive here; the nearest two and one on either side
    for (int64_t k = std::max(n - 1, steps[i].least); k <= std::min(n + 1, steps[i].most); ++k)
      if (self(self, i + 1, distance - k * steps[i].stride)) return true;
    return false;
  };
  return reaches(reaches, 0, (reinterpret_cast<intptr_t>(y.data_ptr()) - reinterpret_cast<intptr_t>(x.data_ptr())) / 2);
}

Tensor new_turned(const Tensor& x) {
  if (x.dim() == 3) return new_tensor(x.sizes(), x.scalar_type(), x);
  return new_tensor({x.size(0), x.size(2), x.size(1), x.size(3)}, x.scalar_type(), x).transpose(1, 2);
}

// `x` and, where it is defined, `y` turned into new tensors or in place
std::tuple<Tensor, Tensor> turn(const Tensor& x, const Tensor& y, const Tensor& positions, const Tensor& inv_freq, const RotaryCall& c, bool in_place) {
  const int64_t pairs = inv_freq.numel();
  c10::cuda::CUDAGuard guard(x.device());
  const Tensor xo = in_place ? x : new_turned(x), yo = !y.defined() || in_place ? y : new_turned(y);
  if (x.numel() == 0 && (!y.defined() || y.numel() == 0)) return {xo, yo};
  sdpa_b200_rotary_params p = {};
  const bool packed = x.dim() == 3;
  p.q = x.data_ptr();
  p.q_out = xo.data_ptr();
  strides_of(x, p.q_batch_stride, p.q_head_stride, p.q_row_stride);
  strides_of(xo, p.qo_batch_stride, p.qo_head_stride, p.qo_row_stride);
  if (y.defined()) {
    p.k = y.data_ptr();
    p.k_out = yo.data_ptr();
    strides_of(y, p.k_batch_stride, p.k_head_stride, p.k_row_stride);
    strides_of(yo, p.ko_batch_stride, p.ko_head_stride, p.ko_row_stride);
    p.heads_k = to_int32(y.size(1), "heads");
  }
  p.heads_q = to_int32(x.size(1), "heads");
  p.batch = to_int32(packed ? 1 : x.size(0), "batch");
  p.length = to_int32(packed ? x.size(0) : x.size(2), "length");
  p.head_dim = to_int32(x.size(-1), "head_dim");
  p.rotary_dim = to_int32(2 * pairs, "rotary_dim");
  p.positions = positions.data_ptr();
  p.positions_64 = positions.scalar_type() == at::kLong;
  p.inv_freq = inv_freq.data_ptr<float>();
  p.axes = c.sections.empty() ? 1 : static_cast<int32_t>(c.sections.size());
  p.sections[0] = static_cast<int32_t>(pairs);
  for (size_t i = 0; i < c.sections.size(); ++i) p.sections[i] = to_int32(c.sections[i], "a section");
  const int64_t first = c.sections.empty() ? 0 : 1, dims = positions.dim() - first;
  p.pos_axis_stride = first ? positions.stride(0) : 0;
  p.pos_batch_stride = dims == 2 && positions.size(first) > 1 ? positions.stride(first) : 0;
  p.pos_row_stride = positions.stride(-1);
  p.interleaved = c.interleaved;
  p.inverse = c.inverse;
  p.scaling = static_cast<float>(c.scaling);
  p.dtype = x.scalar_type() == at::kHalf ? SDPA_B200_F16 : SDPA_B200_BF16;
  check_status(sdpa_b200_rotary(&p, stream_of(x)), "sdpa_b200_rotary");
  return {xo, yo};
}

// The incoming gradient as the kernel can read it: multiples of 8 elements, 0 (an expanded one) among them
Tensor readable(const Tensor& x) {
  bool ok = x.stride(-1) == 1 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  for (int64_t i = 0; ok && i < x.dim() - 1; ++i) ok = x.size(i) == 1 || (x.stride(i) >= 0 && x.stride(i) % 8 == 0);
  return ok ? x : x.clone(at::MemoryFormat::Contiguous);
}

c10::optional<Tensor> if_defined(const Tensor& t) { return t.defined() ? c10::optional<Tensor>(t) : c10::nullopt; }

void check_rotary(const Tensor& query, const Tensor& key, const Tensor& positions, const Tensor& inv_freq, const std::vector<int64_t>& sections) {
  TORCH_CHECK(query.dim() == 3 || query.dim() == 4, "query must be packed [tokens, heads, head_dim] or [batch, heads, seq_len, head_dim]");
  rotary_tensor(query, "query", query);
  if (key.defined()) rotary_tensor(key, "key", query);
  for (const Tensor* t : {&query, &key}) TORCH_CHECK(!t->defined() || t->stride(-1) == 1, "query and key must have a contiguous last dimension");
  check_plain(inv_freq, "inv_freq");
  TORCH_CHECK(inv_freq.dim() == 1 && inv_freq.scalar_type() == at::kFloat && inv_freq.is_contiguous() && inv_freq.device() == query.device(),
              "inv_freq must be a contiguous fp32 vector of rotary_dim / 2 frequencies on the device of query");
  TORCH_CHECK(!needs_grad(inv_freq), "rotary positions have no gradient of inv_freq: detach it");
  for (const Tensor* t : {&query, &key, &inv_freq}) check_no_tangent(*t, "rotary positions");
  check_plain(positions, "positions");
  TORCH_CHECK((positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong) && positions.device() == query.device(),
              "positions must be int32 or int64, on the device of query");
  int64_t pairs = 0, least = 0;
  for (const int64_t n : sections) {
    pairs += n;
    least = std::min(least, n);
  }
  TORCH_CHECK(sections.empty() || (sections.size() <= 4 && least >= 0 && pairs == inv_freq.numel()),
              "sections must be one to four numbers of pairs that add up to rotary_dim / 2 = ", inv_freq.numel());
  // positions: [axes,] tokens, or [axes,] [batch or 1,] length
  const int64_t first = sections.empty() ? 0 : 1, dims = positions.dim() - first;
  TORCH_CHECK(first == 0 || (positions.dim() > 0 && positions.size(0) == static_cast<int64_t>(sections.size())), "positions must have ", sections.size(),
              " axes in front (got shape ", positions.sizes(), ")");
  if (query.dim() == 3) {
    TORCH_CHECK(dims == 1 && positions.size(first) == query.size(0), "positions must be ", first ? "[axes, tokens]" : "[tokens]", " (got shape ", positions.sizes(), ")");
  } else {
    TORCH_CHECK((dims == 1 || (dims == 2 && (positions.size(first) == 1 || positions.size(first) == query.size(0)))) && positions.size(-1) == query.size(2),
                "positions must be ", first ? "[axes, length] or [axes, batch, length]" : "[length] or [batch, length]", " (got shape ", positions.sizes(), ")");
  }
}

// An operator has no results that may be missing: one, or two with a key
std::vector<Tensor> rotary_operator(const Tensor& query, const c10::optional<Tensor>& key, const Tensor& positions, const Tensor& inv_freq, at::OptionalIntArrayRef sections,
                                    bool interleaved, double scaling, bool inverse) {
  const Tensor k = key.value_or(Tensor());
  const std::vector<int64_t> parts = sections.has_value() ? sections->vec() : std::vector<int64_t>();
  check_rotary(query, k, positions, inv_freq, parts);
  const auto r = turn(query, k, positions, inv_freq, {parts, interleaved, inverse, scaling}, false);
  if (!k.defined()) return {std::get<0>(r)};
  return {std::get<0>(r), std::get<1>(r)};
}

// turn() into new tensors, below autograd, seen by those who want to see it
std::tuple<Tensor, Tensor> turned(const Tensor& x, const Tensor& y, const Tensor& positions, const Tensor& inv_freq, const RotaryCall& c) {
  at::AutoDispatchBelowADInplaceOrView guard;
  if (!c10::impl::TorchDispatchModeTLS::any_modes_set() && !torch::jit::tracer::isTracing()) return turn(x, y, positions, inv_freq, c, false);
  static auto op = operator_named<decltype(rotary_operator)>("b200_sdpa::rotary_embedding");
  const auto r = op.call(x, if_defined(y), positions, inv_freq, c.sections.empty() ? at::OptionalIntArrayRef() : at::OptionalIntArrayRef(c.sections), c.interleaved, c.scaling, c.inverse);
  return {r[0], r.size() > 1 ? r[1] : Tensor()};
}

// The gradient of a turn is the turn backwards, itself an operator with a gradient.
struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const c10::optional<Tensor>& other,
                                                const Tensor& positions, const Tensor& inv_freq, std::vector<int64_t> sections, bool interleaved, bool inverse, double scaling) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions, inv_freq});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    ctx->saved_data["scaling"] = scaling;
    const Tensor y = other.value_or(Tensor());
    auto r = turned(x, y, positions, inv_freq, {std::move(sections), interleaved, inverse, scaling});
    if (!y.defined()) return {std::get<0>(r)};
    return {std::get<0>(r), std::get<1>(r)};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const RotaryCall c = {ctx->saved_data["sections"].toIntVector(), ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["inverse"].toBool(),
                          ctx->saved_data["scaling"].toDouble()};
    torch::autograd::variable_list result(8);
    std::vector<size_t> wanted;
    for (size_t i = 0; i < grads.size(); ++i)
      if (grads[i].defined() && ctx->needs_input_grad(i)) wanted.push_back(i);
    if (wanted.empty()) return result;
    Tensor g[2];
    for (size_t i = 0; i < wanted.size(); ++i) {
      check_plain(grads[wanted[i]], "an incoming gradient");
      g[i] = readable(grads[wanted[i]]);
    }
    std::tuple<Tensor, Tensor> r;
    if (needs_grad(g[0]) || needs_grad(g[1])) {
      const auto v = RotaryFunction::apply(g[0], if_defined(g[1]), saved[0], saved[1], c.sections, c.interleaved, c.inverse, c.scaling);
      r = {v[0], v.size() > 1 ? v[1] : Tensor()};
    } else {
      r = turned(g[0], g[1], saved[0], saved[1], c);
    }
    result[wanted[0]] = std::get<0>(r);
    if (wanted.size() > 1) result[wanted[1]] = std::get<1>(r);
    return result;
  }
};

std::vector<Tensor> rotary_with_grad(const Tensor& query, const c10::optional<Tensor>& key, const Tensor& positions, const Tensor& inv_freq, at::OptionalIntArrayRef sections,
                                     bool interleaved, double scaling, bool inverse) {
  const Tensor k = key.value_or(Tensor());
  const std::vector<int64_t> parts = sections.has_value() ? sections->vec() : std::vector<int64_t>();
  check_rotary(query, k, positions, inv_freq, parts);
  if (needs_grad(query) || needs_grad(k)) return RotaryFunction::apply(query, key, positions, inv_freq, parts, interleaved, inverse, scaling);
  const auto r = turned(query, k, positions, inv_freq, {parts, interleaved, inverse, scaling});
  if (!k.defined()) return {std::get<0>(r)};
  return {std::get<0>(r), std::get<1>(r)};
}

void rotary_operator_in_place(const Tensor& query, const c10::optional<Tensor>& key, const Tensor& positions, const Tensor& inv_freq, at::OptionalIntArrayRef sections,
                              bool interleaved, double scaling) {
  const Tensor k = key.value_or(Tensor());
  const std::vector<int64_t> parts = sections.has_value() ? sections->vec() : std::vector<int64_t>();
  check_rotary(query, k, positions, inv_freq, parts);
  TORCH_CHECK(!needs_grad(query) && !needs_grad(k), "rotary positions in place have no gradient: use rotary_embedding");
  for (const Tensor* t : {&query, &k}) {
    for (int64_t i = 0; t->defined() && i < t->dim(); ++i)
      TORCH_CHECK(t->size(i) <= 1 || t->stride(i) != 0, "rotary positions in place need elements of their own (a stride is 0)");
  }
  TORCH_CHECK(!k.defined() || !rows_overlap(query, k), "rotary positions in place: query and key are the same memory, or share some");
  turn(query, k, positions, inv_freq, {parts, interleaved, false, scaling}, true);
  for (const Tensor* t : {&query, &k})
    if (t->defined()) written(*t);
}

}  // namespace

std::tuple<Tensor, Tensor> rotary(const Tensor& query, const Tensor& key, const Tensor& positions, const Tensor& inv_freq, const std::vector<int64_t>& sections,
                                  bool interleaved, double scaling, bool in_place) {
  const bool seen = calls_are_seen();
  const at::OptionalIntArrayRef parts = sections.empty() ? at::OptionalIntArrayRef() : at::OptionalIntArrayRef(sections);
  if (in_place) {
    if (seen) {
      static auto op = operator_named<decltype(rotary_operator_in_place)>("b200_sdpa::rotary_embedding_");
      check_rotary(query, key, positions, inv_freq, sections);
      op.call(query, if_defined(key), positions, inv_freq, parts, interleaved, scaling);
    } else {
      rotary_operator_in_place(query, if_defined(key), positions, inv_freq, parts, interleaved, scaling);
    }
    return {query, key};
  }
  std::vector<Tensor> r;
  if (seen) {
    static auto op = operator_named<decltype(rotary_operator)>("b200_sdpa::rotary_embedding");
    check_rotary(query, key, positions, inv_freq, sections);  // a wrapped tensor has no rule here
    r = op.call(query, if_defined(key), positions, inv_freq, parts, interleaved, scaling, false);
  } else {
    r = rotary_with_grad(query, if_defined(key), positions, inv_freq, parts, interleaved, scaling, false);
  }
  return {r[0], r.size() > 1 ? r[1] : Tensor()};
}

}  // namespace b200_glue

TORCH_LIBRARY_FRAGMENT(b200_sdpa, m) {
  m.def("rotary_embedding(Tensor query, Tensor? key, Tensor positions, Tensor inv_freq, int[]? sections, bool interleaved, float scaling, bool inverse) -> Tensor[]");
  m.def("rotary_embedding_(Tensor(a!) query, Tensor(b!)? key, Tensor positions, Tensor inv_freq, int[]? sections, bool interleaved, float scaling) -> ()");
  m.def("plan_step(Tensor cached_lens, Tensor new_tokens, Tensor(a!) block_table, Tensor(b!) ring, Tensor ring_state, int block_size, int num_tokens) -> "
        "(Tensor seq_lens, Tensor cu_seqlens, Tensor positions, Tensor slots, Tensor next_state)");
  m.def("plan_step_(Tensor(a!) cached_lens, Tensor new_tokens, Tensor(b!) block_table, Tensor(c!) ring, Tensor(d!) ring_state, int block_size, int num_tokens) -> "
        "(Tensor cu_seqlens, Tensor positions, Tensor slots)");
  m.def("cache_store_(Tensor key, Tensor value, Tensor slots, Tensor(a!) key_cache, Tensor(b!) value_cache, Tensor(c!) key_scale, Tensor(d!) value_scale) -> ()");
  m.def("cache_attention(Tensor query, Tensor key_cache, Tensor value_cache, Tensor key_scale, Tensor value_scale, Tensor block_table, Tensor seq_lens, Tensor? cu_seqlens, "
        "int max_seqlen_q, int? max_seqlen_k, bool is_causal, float? scale) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(b200_sdpa, CUDA, m) {
  m.impl("rotary_embedding", b200_glue::rotary_operator);
  m.impl("rotary_embedding_", b200_glue::rotary_operator_in_place);
  m.impl("plan_step", b200_glue::plan_operator);
  m.impl("plan_step_", b200_glue::plan_operator_in_place);
  m.impl("cache_store_", b200_glue::launch_store);
  m.impl("cache_attention", b200_glue::launch_attention);
}

TORCH_LIBRARY_IMPL(b200_sdpa, AutogradCUDA, m) { m.impl("rotary_embedding", b200_glue::rotary_with_grad); }
