/*
 * sdpa_b200.h - C ABI of libsdpa_b200.so: scaled-dot-product attention forward, backward
 * and split-KV decode for NVIDIA B200 (sm_100a), written to stand where torch_mlu binds
 * Cambricon's closed attention library.
 *
 * What each entry point replaces in the reference (paths inside Cambricon/torch_mlu):
 *   sdpa_b200_fwd            <- mha_varlen_fwd, i.e. cnnlFlashAttentionForward_v2
 *                               torch_mlu/csrc/aten/operators/cnnl/internal/FlashAttention_internal.cpp:57-267
 *                               (declared cnnl_internal.h:1461-1476)
 *   sdpa_b200_bwd            <- mha_varlen_bwd, i.e. cnnlFlashAttentionBackward
 *                               .../internal/FlashAttention_internal.cpp:269-483 (cnnl_internal.h:1478-1495)
 *   sdpa_b200_*_workspace_bytes
 *                            <- cnnlGetFlashAttention{Forward,Backward}WorkspaceSize_v2
 *                               .../internal/FlashAttention_internal.cpp:215-230, 437-447
 *   sdpa_b200_status_string  <- TORCH_CNNL_CHECK's status-to-text, torch_mlu/csrc/aten/utils/exceptions.h:77-83
 *   sdpa_b200_dropout_keep_mask[_varlen]
 *                            <- the Philox state the reference hands to its kernel (cnnlRandGenerator / seed, offset,
 *                               .../internal/FlashAttention_internal.cpp:190-214): here the pattern itself, as bits
 *   bias / dbias fields      <- the attn_bias and grad_bias descriptors of mem_eff_fwd / mem_eff_bwd
 *                               (.../internal/FlashAttention_internal.cpp:485-904)
 *
 * Conventions
 *   - Plain C: pointers, sizes, one POD struct. No C++ or torch types cross this boundary.
 *   - Every pointer in sdpa_b200_params is a DEVICE pointer on the caller's current device.
 *   - The caller owns every buffer including the workspace; the library allocates no device
 *     memory and keeps no per-call state.
 *   - Calls enqueue work on `stream` and return without synchronising.
 *   - Errors are integer status codes; nothing throws, aborts or traps the device. A kernel
 *     whose internal wait runs out writes SDPA_B200_DEVICE_TIMEOUT into the first word of
 *     the workspace; sdpa_b200_read_device_status() fetches it (it synchronises the stream).
 *   - Layout: element strides for (batch, head, row); the head_dim stride must be 1.
 *       dense   : cu_seqlens_* == NULL, batch b / head h / row r of q lives at
 *                 q + b*q_batch_stride + h*q_head_stride + r*q_row_stride (any BHLD/BLHD view)
 *       varlen  : cu_seqlens_q/k are int32[batch+1] exclusive prefix sums; tensors are packed
 *                 [total_tokens, heads, head_dim]; *_batch_stride is ignored and row r of
 *                 sequence b is token cu_seqlens[b] + r.
 *   - lse (natural-log logsumexp of scale*QK^T over the visible keys, fp32):
 *       dense   : [batch, heads_q, seqlen_q] contiguous
 *       varlen  : [heads_q, total_q] contiguous (the buffer mha_varlen_fwd allocates,
 *                 FlashAttention_internal.cpp:129)
 *     A row with no visible key gets out = 0 and lse = +inf.
 *   - Causal masking is bottom-right aligned: key j is visible to query i when
 *     j <= i + seqlen_k - seqlen_q (the reference test oracle's rule,
 *     test/torch_ops/test_scaled_dot_product_attention.py:69). With seqlen_q == seqlen_k it is
 *     the usual lower triangle.
 *   - GQA/MQA: heads_q % heads_kv == 0; query head h reads KV head h / (heads_q/heads_kv)
 *     (FlashAttention_internal.cpp:117-124).
 */
#ifndef SDPA_B200_H_
#define SDPA_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SDPA_B200_VERSION 108

#if defined(__GNUC__)
#define SDPA_B200_API __attribute__((visibility("default")))
#else
#define SDPA_B200_API
#endif

/* status codes */
enum {
  SDPA_B200_OK = 0,
  SDPA_B200_INVALID_ARG = 1,    /* null pointer, bad shape, bad stride/alignment, workspace too small */
  SDPA_B200_UNSUPPORTED = 2,    /* valid request this build has no kernel for (dtype, head_dim > 128 with a bias, decode with bias) */
  SDPA_B200_LAUNCH_FAILED = 3,  /* CUDA reported an error while configuring or launching */
  SDPA_B200_DEVICE_TIMEOUT = 4, /* a bounded wait inside a kernel ran out (read back from workspace) */
  SDPA_B200_NO_DEVICE = 5       /* not an sm_100 device / no CUDA driver */
};

enum { SDPA_B200_BF16 = 0, SDPA_B200_F16 = 1 }; /* element type of q, k, v, out and gradients (the reference
                                                   takes the same two: sdp_utils.h:433-455) */

/* kernel selection for the forward entry point */
enum {
  SDPA_B200_KERNEL_AUTO = 0,    /* decode when max_seqlen_q is small, prefill otherwise */
  SDPA_B200_KERNEL_PREFILL = 1, /* TMA + tcgen05 tile kernel */
  SDPA_B200_KERNEL_DECODE = 2   /* split-KV streaming kernel */
};

typedef struct sdpa_b200_params {
  /* inputs */
  const void* q; /* bf16 */
  const void* k;
  const void* v;
  /* forward outputs (inputs of backward) */
  void* out;  /* bf16, same shape as q */
  float* lse; /* fp32, layout above */
  /* backward only */
  const void* dout; /* bf16, same shape/strides family as out */
  /* Gradients. Packed: rows of tokens that belong to no sequence (in front of cu_seqlens[0], behind cu_seqlens[batch]) are
   * set to zero. */
  void* dq;         /* bf16, shape of q */
  void* dk;         /* bf16, shape of k */
  void* dv;         /* bf16, shape of v */

  /* varlen: device int32[batch+1]; NULL for dense */
  const int32_t* cu_seqlens_q;
  const int32_t* cu_seqlens_k;

  int32_t batch;
  int32_t heads_q;
  int32_t heads_kv;
  int32_t head_dim;     /* a multiple of 8, at most 256 (SDPA_B200_KERNEL_DECODE: 64 or 128; with a bias: at most 128) */
  int32_t max_seqlen_q; /* dense: seqlen_q */
  int32_t max_seqlen_k; /* dense: seqlen_k */
  int32_t total_q;      /* varlen: rows of q/out; dense: ignored */
  int32_t total_k;      /* varlen: rows of k/v;   dense: ignored */

  /* element strides; head_dim stride is 1 */
  int64_t q_batch_stride, q_head_stride, q_row_stride;
  int64_t k_batch_stride, k_head_stride, k_row_stride;
  int64_t v_batch_stride, v_head_stride, v_row_stride;
  int64_t o_batch_stride, o_head_stride, o_row_stride;
  /* backward */
  int64_t do_batch_stride, do_head_stride, do_row_stride;
  int64_t dq_batch_stride, dq_head_stride, dq_row_stride;
  int64_t dk_batch_stride, dk_head_stride, dk_row_stride;
  int64_t dv_batch_stride, dv_head_stride, dv_row_stride;

  float softmax_scale; /* > 0; the reference default is 1/sqrt(head_dim), sdp_utils.h:40-47 */
  float dropout_p;     /* 0, or inside (0, 1) together with keep_rows / keep_cols */
  int32_t is_causal;
  int32_t dtype;      /* SDPA_B200_BF16 or SDPA_B200_F16 */
  int32_t kernel;     /* SDPA_B200_KERNEL_* (forward only) */
  int32_t num_splits; /* decode: 0 = choose; otherwise the number of KV splits */
  /* Dropout keep-masks written by sdpa_b200_dropout_keep_mask() (dense) or ..._varlen() (packed) for the same
   * batch, heads_q and sequence lengths; both NULL when dropout_p == 0. The forward reads keep_rows; the
   * backward reads both. */
  const uint32_t* keep_rows;
  const uint32_t* keep_cols;
  /* Additive attention bias of the memory-efficient operators (mem_eff_fwd / mem_eff_bwd,
   * FlashAttention_internal.cpp:485-904): out = softmax(scale * q k^T + bias) v. NULL = none. Same 16-bit
   * type as q; element strides for (batch, head, query row), 0 for a broadcast dimension; the key stride is 1.
   * Rows start 16-byte aligned (row stride a multiple of 8, or 0) and are readable up to the next multiple of
   * 8 keys. With packed (varlen) q / k / v the bias stays a [batch, heads_q, max_seqlen_q, max_seqlen_k] tensor:
   * sequence b reads bias[b, h, i, j] for its query i and key j counted from the start of the sequence. The
   * same holds for dbias and bias_t. */
  const void* bias;
  int64_t bias_batch_stride, bias_head_stride, bias_row_stride;
  /* Backward: gradient of the bias, [batch, heads_q, seqlen_q, dbias_row_stride >= seqlen_k rounded up to 8],
   * same type, or NULL. Elements the causal mask hides are not written: clear the buffer first.
   * Without a causal mask every element of a dense call's gradient is written; the padding behind seqlen_k need not be. */
  void* dbias;
  int64_t dbias_batch_stride, dbias_head_stride, dbias_row_stride;
  /* Backward, optional: the same bias with keys and queries exchanged, [batch, heads_q, seqlen_k, seqlen_q]
   * with unit query stride and the rules of `bias` for alignment and padding (strides for batch, head, key row).
   * The dK/dV kernel, whose threads own keys, then reads 16 bytes at a time instead of two. Not needed when the
   * bias does not depend on the query (bias_row_stride == 0). NULL = not given. */
  const void* bias_t;
  int64_t bias_t_batch_stride, bias_t_head_stride, bias_t_row_stride;
  /* Backward: 0 = whichever is faster for the sizes. That may be the fused kernel (up to head_dim 64), which forms
   * every tile's scores once and adds its dQ contributions into an fp32 workspace with floating-point reductions whose
   * order varies between launches (dK and dV are still summed in a fixed order). Non-zero = only kernels with a fixed
   * summation order throughout, so that the same call gives the same bits every time, with any workspace size. A call with
   * a bias takes only those too. Ignored by the forward. */
  int32_t deterministic;
  /* Forward (tile kernel): number of SMs the persistent kernel leaves free, for a kernel that is to run beside it on
   * another stream - a collective that reassembles the previous step's outputs, say. 0 = one CTA on every SM, which
   * keeps any other kernel out until the CTAs leave. At least one SM is always used. */
  int32_t sm_margin;
  /* Optional device word (4-byte aligned) that collects kernel status across calls: a kernel whose bounded wait
   * runs out stores SDPA_B200_DEVICE_TIMEOUT there. The library never clears it, so one word can watch a whole
   * stream of calls whose workspaces come and go; read it with sdpa_b200_read_device_status and clear it
   * yourself. NULL = the first word of the call's workspace, cleared at the start of each call. */
  uint32_t* device_status;
} sdpa_b200_params;

SDPA_B200_API int sdpa_b200_version(void);
SDPA_B200_API const char* sdpa_b200_status_string(int status);
/* Text of the last error raised on the calling thread (what was wrong and where). */
SDPA_B200_API const char* sdpa_b200_last_error(void);

/* Workspace size the matching call is best given for these params (>= 256 bytes; 256-byte aligned base required).
 * For the forward it is also the least it needs. The backward may leave dS there (up to 2 GiB; head dims above 64) and runs
 * with less as well, on slower kernels: sdpa_b200_bwd_workspace_least_bytes is the size below which it is refused. */
SDPA_B200_API int sdpa_b200_fwd_workspace_bytes(const sdpa_b200_params* p, size_t* bytes);
SDPA_B200_API int sdpa_b200_bwd_workspace_bytes(const sdpa_b200_params* p, size_t* bytes);
SDPA_B200_API int sdpa_b200_bwd_workspace_least_bytes(const sdpa_b200_params* p, size_t* bytes);

/* out, lse <- attention(q, k, v). `stream` is a cudaStream_t passed as void*. */
SDPA_B200_API int sdpa_b200_fwd(const sdpa_b200_params* p, void* workspace, size_t workspace_bytes, void* stream);

/* dq, dk, dv <- backward(dout, q, k, v, out, lse). */
SDPA_B200_API int sdpa_b200_bwd(const sdpa_b200_params* p, void* workspace, size_t workspace_bytes, void* stream);

/* Synchronises `stream`, reads the status word a kernel may have left in `workspace` (or in the word given as
 * sdpa_b200_params.device_status) and returns it in *device_status (SDPA_B200_OK or SDPA_B200_DEVICE_TIMEOUT). */
SDPA_B200_API int sdpa_b200_read_device_status(const void* workspace, void* stream, int* device_status);

/* Self-test of the time-out path every kernel of this library shares: launches one warp that waits, for at most
 * `budget_us` microseconds, on a shared-memory barrier nobody will ever arrive on - no copy or MMA is in flight -
 * then gives up exactly as the attention kernels do: it stores SDPA_B200_DEVICE_TIMEOUT into *device_status and
 * returns normally, leaving the context usable. No counterpart in the reference, whose vendor kernels report
 * nothing back from the device. */
SDPA_B200_API int sdpa_b200_selftest_wait_timeout(uint32_t* device_status, uint32_t budget_us, void* stream);

/* The same for a forward's grid with several CTAs per SM: each of `ctas` CTAs, one at a time per SM, adds 1 to *started and waits for at most `budget_us`
 * (up to 1000) microseconds; those that give up take the CTAs that have not started with them, so that the grid ends after one budget and *started
 * has grown by no more than the number of SMs. */
SDPA_B200_API int sdpa_b200_selftest_grid_timeout(uint32_t* device_status, uint32_t* started, uint32_t ctas, uint32_t budget_us, void* stream);

/* Split-KV decode (dense tensors, seqlen_q == 1) for callers that cannot allocate device memory
 * where they call it - inside an allocator or memory-pool callback, or after the process has
 * frozen its memory plan. No counterpart in the reference: its attention calls always take a
 * workspace from the caching allocator (FlashAttention_internal.cpp:215-230). The caller passes
 * inputs and outputs only; the split partials live in a fixed SDPA_B200_STATIC_SCRATCH_BYTES
 * array inside the library (held by every GPU that loads it). Requests whose partials exceed it
 * (batch * heads_q * num_splits * (head_dim + 1) * 4 bytes with num_splits > 1; with num_splits 0
 * they always fit) are refused with SDPA_B200_INVALID_ARG. The first call on each device looks the array's address up; make it outside stream capture. Calls
 * that overlap on one GPU race on the shared array - order them on one stream. */
#define SDPA_B200_STATIC_SCRATCH_BYTES (16u << 20)
SDPA_B200_API int sdpa_b200_decode_static(const sdpa_b200_params* p, void* stream);

/* Folds one partial attention result into an fp32 accumulator by the logsumexp rule (the combine
 * step of ring / context-parallel prefill; no counterpart in the reference, whose attention is
 * single-device):  lse' = log(exp(lse_acc) + exp(lse_part)),
 *                  o_acc' = o_acc*exp(lse_acc - lse') + o_part*exp(lse_part - lse').
 * o_acc [batch, heads, rows, head_dim] fp32 and lse_acc / lse_part [batch, heads, rows] fp32 are
 * contiguous; o_part is bf16 or f16 (`dtype`) with the given element strides (the `out` of
 * sdpa_b200_fwd).
 * Start an accumulator with lse_acc = -inf (o_acc may be uninitialised). */
SDPA_B200_API int sdpa_b200_merge_partial(float* o_acc, float* lse_acc, const void* o_part, const float* lse_part,
                                          int32_t batch, int32_t heads, int32_t rows, int32_t head_dim,
                                          int32_t dtype, int64_t part_batch_stride, int64_t part_head_stride,
                                          int64_t part_row_stride, void* stream);

/* Dropout pattern for one attention call, one bit per (query, key) pair, drawn from Philox4x32-10 with the
 * given seed and offset (the reference draws it inside its device kernel from such a pair,
 * FlashAttention_internal.cpp:190-214, and returns the pair so that the backward pass can repeat it; here the
 * caller generates the masks again from the pair before calling sdpa_b200_bwd, or keeps them).
 *   keep_rows: uint32 [batch*heads][Lq_pad][Lk_pad/32], bit (k & 31) of word (q, k >> 5) set = pair kept
 *   keep_cols: uint32 [batch*heads][Lk_pad][Lq_pad/32], bit (q & 31) of word (k, q >> 5): the transpose
 * Lq_pad / Lk_pad are the lengths rounded up to a multiple of 128; `heads` is heads_q. A pair is dropped with
 * probability round(dropout_p * 256) / 256; kept probabilities are scaled by 1 / (1 - dropout_p) in the
 * attention kernels. With `is_causal` (the bottom-right
 * aligned mask of the attention calls) 128 x 128 tiles that the mask hides completely are filled with zeros
 * instead of random bits; a call made with is_causal must be given masks made with it or without it, never the
 * other way round. */
SDPA_B200_API int sdpa_b200_dropout_keep_mask(uint64_t seed, uint64_t offset, float dropout_p, int32_t batch,
                                              int32_t heads, int32_t seqlen_q, int32_t seqlen_k, int32_t is_causal,
                                              uint32_t* keep_rows, uint32_t* keep_cols, void* stream);

/* The same pattern for packed (varlen) tensors: sequence b of the batch gets the bits batch index b would get
 * in the dense form, addressed by packed token index:
 *   keep_rows: uint32 [heads][total_q + 128][Lk_pad/32], row = packed query index, bit = key position inside
 *              the query's sequence;   keep_cols: uint32 [heads][total_k + 128][Lq_pad/32], the transpose.
 * Lq_pad / Lk_pad are max_seqlen_q / max_seqlen_k rounded up to 128. Both arrays must arrive zero-filled: only
 * words an attention kernel reads are written. */
SDPA_B200_API int sdpa_b200_dropout_keep_mask_varlen(uint64_t seed, uint64_t offset, float dropout_p, int32_t batch,
                                                     int32_t heads, const int32_t* cu_seqlens_q,
                                                     const int32_t* cu_seqlens_k, int32_t total_q, int32_t total_k,
                                                     int32_t max_seqlen_q, int32_t max_seqlen_k, int32_t is_causal,
                                                     uint32_t* keep_rows, uint32_t* keep_cols, void* stream);

/* Writes sdpa_b200_params.bias_t for a bias given as in sdpa_b200_params (16-bit elements, element strides, unit
 * key stride, row_stride != 0): out is [batch][heads][seqlen_k][out_row_stride], contiguous, out_row_stride a
 * multiple of 8 that holds seqlen_q; the padding is zero-filled. Pass batch = 1 (heads = 1) for a bias that is
 * broadcast along that dimension and give bias_t the stride 0 there. */
SDPA_B200_API int sdpa_b200_transpose_bias(const void* bias, int64_t batch_stride, int64_t head_stride, int64_t row_stride,
                                           int32_t batch, int32_t heads, int32_t seqlen_q, int32_t seqlen_k, void* out,
                                           int64_t out_row_stride, void* stream);

/* Writes a boolean attention mask (one byte per element, non-zero = the pair takes part, element strides, 0 for a broadcast
 * dimension) as the additive bias of 0 / -inf that sdpa_b200_params.bias takes: out is
 * [batch][heads][seqlen_q][out_row_stride] 16-bit elements of `dtype`, contiguous, out_row_stride a multiple of 8 that holds
 * seqlen_k; the padding is zero-filled. Pass 1 for a dimension the mask is broadcast along and give the bias the stride 0
 * there. */
SDPA_B200_API int sdpa_b200_mask_to_bias(const void* mask, int64_t batch_stride, int64_t head_stride, int64_t row_stride,
                                         int64_t key_stride, int32_t batch, int32_t heads, int32_t seqlen_q, int32_t seqlen_k,
                                         void* out, int64_t out_row_stride, int32_t dtype, void* stream);

/* Copies a bias of 16-bit elements (element strides, 0 for a broadcast dimension, any key stride) into rows that sdpa_b200_params.bias can be read
 * from: out is [batch][heads][seqlen_q][out_row_stride], contiguous, out_row_stride a multiple of 8 that holds seqlen_k; the padding is zero-filled. */
SDPA_B200_API int sdpa_b200_pad_bias(const void* bias, int64_t batch_stride, int64_t head_stride, int64_t row_stride,
                                     int64_t key_stride, int32_t batch, int32_t heads, int32_t seqlen_q, int32_t seqlen_k,
                                     void* out, int64_t out_row_stride, void* stream);

/* Sums a bias gradient (sdpa_b200_params.dbias: 16-byte aligned, strides that are multiples of 8, unit key stride, rows readable to the next multiple
 * of 8 keys) over the batches and / or the heads that the bias is broadcast along, in fp32. out is [batch or 1][heads or 1][seqlen_q][seqlen_k],
 * contiguous, of `dtype`. */
SDPA_B200_API int sdpa_b200_sum_bias_grad(const void* grad, int64_t batch_stride, int64_t head_stride, int64_t row_stride,
                                          int32_t batch, int32_t heads, int32_t seqlen_q, int32_t seqlen_k, int32_t over_batch,
                                          int32_t over_heads, void* out, int32_t dtype, void* stream);

/* ---- rotary positions -------------------------------------------------------------------------------------------------
 * q_out, k_out <- q, k with the first rotary_dim elements of every row turned by the angles of its token:
 *   angle_j = position[axis(j)] * inv_freq[j],  (x, y) -> scaling * (x cos - y sin, x sin + y cos)
 * over the pairs (j, j + rotary_dim / 2), or (2j, 2j + 1) with `interleaved`; the other elements are copied. axis(j) is the
 * section that pair j falls into, so that sections of time, height and width turn by three positions of a token. The angle is
 * formed in 64 bits, since in 32 that of a far position is lost. `inverse` turns by the negative angle: the gradient of q and k out
 * of that of the results. q_out / k_out may be q / k themselves. No counterpart in the reference, whose models bring their own. */
typedef struct sdpa_b200_rotary_params {
  const void* q;
  const void* k; /* NULL with heads_k == 0 */
  void* q_out;
  void* k_out;
  const void* positions; /* int32, or int64 with positions_64, aligned to them; [axes][batch][length] by the strides below, in elements */
  const float* inv_freq; /* [rotary_dim / 2] */
  int32_t batch, length, heads_q, heads_k;
  int32_t head_dim;    /* a multiple of 8, at most 256 */
  int32_t rotary_dim;  /* a multiple of 16, at most head_dim */
  int32_t axes;        /* 1 to 4 */
  int32_t sections[4]; /* pairs per axis, together rotary_dim / 2 */
  int32_t interleaved, inverse, positions_64;
  int32_t dtype; /* SDPA_B200_BF16 or SDPA_B200_F16 */
  float scaling;
  /* elements, multiples of 8; those of inputs may be 0 (broadcast) */
  int64_t q_batch_stride, q_head_stride, q_row_stride;
  int64_t k_batch_stride, k_head_stride, k_row_stride;
  int64_t qo_batch_stride, qo_head_stride, qo_row_stride;
  int64_t ko_batch_stride, ko_head_stride, ko_row_stride;
  int64_t pos_axis_stride, pos_batch_stride, pos_row_stride;
} sdpa_b200_rotary_params;

SDPA_B200_API int sdpa_b200_rotary(const sdpa_b200_rotary_params* p, void* stream);

/* ---- the paged cache --------------------------------------------------------------------------------------------------
 * Keys and values live in blocks of block_size tokens: codes [num_blocks][heads_kv][block_size][head_dim]; an element is code * scale.
 * 8 bits: e4m3 or int8, with one fp32 scale per block and head. 4 bits: whole numbers from -8 to 7, two in a byte, the even element in the low
 * half, with a bf16 scale for every 32 elements of a token and head, [num_blocks][heads_kv][block_size][head_dim / 32].
 * A request's token at position p is in the block block_table[request]
 * [p / block_size], at p % block_size; that place in the cache, block * block_size + p % block_size, is called its slot. No
 * counterpart in the reference, which has no paged cache. */
enum { SDPA_B200_E4M3 = 0, SDPA_B200_INT8 = 1, SDPA_B200_INT4 = 4 };

/* One serving step's bookkeeping. new_tokens[i] tokens are added to request i (negative: that many are taken back), and what it needs
 * or no longer needs of blocks moves between block_table and a ring of free ones. The ring holds ring_state[1] free blocks from index
 * ring_state[0] on, modulo num_blocks; blocks are taken at its front, request by request, page by page, and given back at its end.
 * Written: seq_lens[i] = cached_lens[i] + new_tokens[i]; cu_seqlens[batch + 1], the offsets of the requests' new tokens; positions and
 * slots of these num_tokens tokens, 0 and -1 behind the last one; the new blocks in block_table (entries behind a request's last block
 * mean nothing and are left as they are); blocks given back, in the ring; next_state.
 * All or nothing: where a request would get a negative length, more than max_blocks blocks or tokens behind num_tokens, next_state[2] is
 * -1 - (the first such request), where blocks are lacking their number, else 0; a step that is refused so changes nothing, and seq_lens,
 * cu_seqlens, positions, slots are those of a step without new tokens. seq_lens may be cached_lens and next_state may be ring_state. */
typedef struct sdpa_b200_plan_params {
  const int32_t* cached_lens; /* [batch] */
  const int32_t* new_tokens;  /* [batch] */
  int32_t* block_table;       /* [batch][table_stride], the first max_blocks of each row */
  int32_t* ring;              /* [num_blocks] */
  const int32_t* ring_state;  /* [3] */
  int32_t* seq_lens;          /* [batch] */
  int32_t* cu_seqlens;        /* [batch + 1] */
  int32_t* positions;         /* [num_tokens] */
  int32_t* slots;             /* [num_tokens] */
  int32_t* next_state;        /* [3] */
  int64_t table_stride;
  int32_t batch, max_blocks, num_blocks, block_size, num_tokens; /* block_size: 16, 32, 64 or 128; num_blocks * block_size < 2^31 */
} sdpa_b200_plan_params;

SDPA_B200_API int sdpa_b200_plan_step(const sdpa_b200_plan_params* p, void* stream);

typedef struct sdpa_b200_cache_params {
  /* codes by (block, head, token) strides in bytes, multiples of 16, head_dim contiguous; 16-byte aligned */
  void* k_cache;
  void* v_cache;
  void* k_scale; /* 8 bits: fp32 [num_blocks][heads_kv], those of V not negative; 4 bits: bf16 [num_blocks][heads_kv][block_size][head_dim / 32], 16-byte aligned */
  void* v_scale;
  int64_t k_block_stride, k_head_stride, k_row_stride;
  int64_t v_block_stride, v_head_stride, v_row_stride;
  int32_t num_blocks, block_size, heads_kv, head_dim; /* block_size: 16, 32, 64 or 128; head_dim: 64 or 128 */
  int32_t code;  /* SDPA_B200_E4M3, SDPA_B200_INT8 or SDPA_B200_INT4 */
  int32_t dtype; /* of key, value, q, out: SDPA_B200_BF16 or SDPA_B200_F16 */
  /* store */
  const void* key; /* [num_tokens][heads_kv][head_dim] by strides in elements, multiples of 8 */
  const void* value;
  int64_t key_row_stride, key_head_stride;
  int64_t value_row_stride, value_head_stride;
  const int32_t* slots;
  int32_t num_tokens;
  /* attention */
  int32_t batch;
  const void* q; /* [total_q][heads_q][head_dim] by strides in elements, multiples of 8 */
  void* out;
  float* lse; /* [heads_q][total_q] */
  int64_t q_row_stride, q_head_stride;
  int64_t o_row_stride, o_head_stride;
  const int32_t* block_table;  /* [batch][table_stride], the first max_blocks of each row */
  const int32_t* seq_lens;     /* [batch]: tokens of each request in the cache, those of q among them */
  const int32_t* cu_seqlens_q; /* [batch + 1]; NULL: one row of q per request */
  int64_t table_stride;
  int32_t max_blocks, heads_q, total_q;
  int32_t max_seqlen_q, max_seqlen_k; /* at least the longest request's */
  int32_t is_causal;                  /* bottom-right aligned, as everywhere here */
  float softmax_scale;
  uint32_t* device_status; /* as in sdpa_b200_params */
  /* load */
  void* key_out; /* [num_tokens][heads_kv][head_dim], contiguous, 32-byte aligned */
  void* value_out;
  const int32_t* first; /* [batch]: each request's first token; NULL: 0 */
  const int32_t* cu_seqlens_k; /* [batch + 1]: offsets of the requests' rows of key_out and value_out */
} sdpa_b200_cache_params;

/* Puts the keys and values of a step into the cache. 8 bits: every (block, head) that gets tokens has its scale raised to the smallest power of two
 * at which the largest of them is a code (448 for e4m3, 127 for int8), unless it is that large already; earlier tokens of the block are
 * rounded again to a scale that has grown. A block whose first place is written starts anew. Tokens with a negative slot, or one behind the
 * cache, are left out. The tokens of one block stand next to each other, with rising slots, as sdpa_b200_plan_step gives them (the same slot
 * twice in a row: the later token stays; fewer than 32 tokens that are left out may stand between them); a block that comes up again
 * behind tokens of another one is not allowed, since the two parts are worked on at the same time; keys and values have caches and scales of
 * their own for the same reason. A NaN or infinite element becomes NaN in e4m3; int8 has none, there the scale becomes NaN until the block
 * starts anew.
 * 4 bits: every 32 elements of a token and head get the smallest scale of five significant bits, 2^-100 at least, at which the largest of them is no more than 7 (a code times
 * such a scale is exact in 16 bits within the type's range); the code is the nearest whole number, the even one of two. A scale depends on nothing but its 32 elements. With a
 * NaN or infinite one among them it is NaN and the codes are 0. */
SDPA_B200_API int sdpa_b200_cache_store(const sdpa_b200_cache_params* p, void* stream);

/* key_out, value_out <- tokens of the requests: row cu_seqlens_k[b] + i is token first[b] + i of request b, found through block_table, max_blocks blocks a row. code * scale,
 * a product in 32 bits, is rounded to dtype; what is beyond its largest number is that number. NaN: a token in front of 0 or behind the table's row, a block number outside the cache, an
 * infinite or NaN scale. Rows in front of cu_seqlens_k[0] and behind the last request are filled with zeros. Offsets that fall, or leave the outputs, write nothing outside
 * them; a row that several requests claim belongs to one of them. */
SDPA_B200_API int sdpa_b200_cache_load(const sdpa_b200_cache_params* p, void* stream);

/* out, lse <- attention of each request's last rows of q over its tokens in the cache. A row without a visible key gets out = 0 and lse = +inf;
 * rows of q outside every request are left unwritten. NaN (with lse = +inf, as NaN rows have here): the rows that see a block number outside the
 * cache, or a scale of K that is infinite or NaN, and all rows of a request whose length passes the table's row. Nothing at or behind seq_lens
 * counts, whatever stands there. A NaN among the values, or a scale of V that is negative, infinite or NaN, may reach every row of its request
 * and kv head, as 0 * NaN. A scale of V below 2^-100, as of a block of zeros, counts as 2^-100 where rows are few; there a value counts down to
 * 2^-39 of the largest product of a weight and a scale of V in its row. In a 4-bit cache scales of V keep all their bits down to 2^-16 of the
 * largest among 64 neighbouring tokens, count down to 2^-24 of it and to 2^-100, and a weight times a scale counts down to 2^-38 of the largest product in its row of a weight and the largest
 * scale among its 64 tokens (11 bits of it down to 2^-28); they may be negative, and a scale of K or V that is infinite or NaN reaches only the rows that see its token.
 * Scores may be of any size that 32 bits hold where rows are few or softmax_scale is above 2^16; else below 2^27, and sums of values times weights of up to 2^8 must fit 32 bits, as in
 * the prefill kernel.
 * Where requests have many rows, codes * scales are brought to 16 bits, q's type, in the workspace, of as many requests at a time as fit 4 GiB
 * at max_seqlen_k tokens each: exact with scales that are powers of two, else rounded as by load, and within the type's range. What is beyond its
 * largest number is that number (f16: 65504; the code of an element from 63488 on may be 65536), and f16 loses what is below 2^-24, as of a
 * cache that was filled from bf16. */
SDPA_B200_API int sdpa_b200_cache_attention_workspace_bytes(const sdpa_b200_cache_params* p, size_t* bytes);
SDPA_B200_API int sdpa_b200_cache_attention(const sdpa_b200_cache_params* p, void* workspace, size_t workspace_bytes, void* stream);

/* How many of this library's kernels the calling process has launched so far. */
SDPA_B200_API uint64_t sdpa_b200_launch_count(void);

#ifdef __cplusplus
}
#endif
#endif /* SDPA_B200_H_ */
