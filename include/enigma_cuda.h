/* enigma_cuda.h — C ABI of libenigma_cuda.so, the B200 (sm_100a) backend of the
 * Enigma runtime.
 *
 * This library takes the place of the Swift/Metal runtime dylib
 * (enigma/runtime_dispatch/swift/libenigma_runtime.swift in the reference),
 * which Python binds with ctypes (enigma/runtime_dispatch/runtime.py:259-316).
 * Plain pointers and sizes only: device pointers are `void*` from
 * enigma_alloc (or any CUDA allocation), streams are `void*` holding a
 * cudaStream_t (NULL = the legacy default stream).
 *
 * Every function returns an int32 status:
 *    0  ENIGMA_OK
 *   -1  ENIGMA_ERR_LAUNCH   launch failed (the Swift runtime's "encoder" error)
 *   -2  ENIGMA_ERR_EXEC     execution error reported by the GPU
 *   -3  ENIGMA_ERR_TIMEOUT  a bounded device-side wait gave up
 *   -4  ENIGMA_ERR_BADARG   shape / pointer / alignment rejected before launch
 *   -5  ENIGMA_ERR_DEVICE   no usable sm_100 device
 * The message of the last failure on the calling thread is returned by
 * enigma_last_error.  -1 and -2 keep the Swift runtime's meaning
 * (libenigma_runtime.swift:146-175).
 */
#ifndef ENIGMA_CUDA_H
#define ENIGMA_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ENIGMA_OK 0
#define ENIGMA_ERR_LAUNCH (-1)
#define ENIGMA_ERR_EXEC (-2)
#define ENIGMA_ERR_TIMEOUT (-3)
#define ENIGMA_ERR_BADARG (-4)
#define ENIGMA_ERR_DEVICE (-5)

/* Element types (storage); accumulation is always fp32. */
#define ENIGMA_DTYPE_F32 0
#define ENIGMA_DTYPE_BF16 1

/* Kernel ids for enigma_dispatch (the recognizer in enigma/compiler maps a
 * traced @enigma.kernel to one of these). */
#define ENIGMA_KERNEL_RMSNORM 1   /* bufs: x, w, y            ip: rows, hidden, dtype   fp: eps */
#define ENIGMA_KERNEL_GEMM 2      /* bufs: A, B, C            ip: M, N, K, dtype, accumulate */
#define ENIGMA_KERNEL_SDPA 3      /* bufs: Q, K, V, O         ip: B, Hq, Hkv, Sq, Skv, D, causal, dtype  fp: scale */

/* ---- device / queue: replaces enigma_create_device, enigma_create_queue
 *      (libenigma_runtime.swift:10, :19) ---- */
int32_t enigma_init(int32_t device);
int32_t enigma_device_count(int32_t* count);
int32_t enigma_stream_create(void** stream);
int32_t enigma_stream_destroy(void* stream);
int32_t enigma_synchronize(void* stream);
int32_t enigma_last_error(char* buf, size_t len);
/* Name of the device kernel the last operator call on this thread chose (e.g.
 * "gemm_bf16_pair_kernel", "sdpa_fwd_tc_kernel"); "" before any call.  No
 * counterpart in the reference, whose Swift runtime runs one named pipeline per
 * dispatch (libenigma_runtime.swift:132-214): here one operator picks between
 * tensor-core and CUDA-core kernels by shape and alignment. */
int32_t enigma_last_kernel(char* buf, size_t len);

/* ---- capability queries: replace enigma_device_name,
 *      enigma_device_max_threadgroup_memory,
 *      enigma_device_max_threads_per_threadgroup, enigma_device_supports_family
 *      (libenigma_runtime.swift:223-260) ---- */
int32_t enigma_device_name(int32_t device, char* buf, size_t len);
int32_t enigma_device_attrs(int32_t device, int64_t* sm_count, int64_t* max_smem_per_block,
                            int64_t* max_threads_per_block, int64_t* total_mem_bytes,
                            int32_t* cc_major, int32_t* cc_minor);

/* ---- buffers: replace enigma_create_buffer, enigma_create_buffer_empty,
 *      enigma_buffer_contents, enigma_release (libenigma_runtime.swift:91-124, :216).
 *      Device memory is not host-visible, so "contents" becomes explicit copies. ---- */
int32_t enigma_alloc(void** ptr, size_t bytes);
int32_t enigma_free(void* ptr);
int32_t enigma_host_alloc(void** ptr, size_t bytes); /* pinned host memory */
int32_t enigma_host_free(void* ptr);
int32_t enigma_upload(void* dst_dev, const void* src_host, size_t bytes, void* stream);
int32_t enigma_download(void* dst_host, const void* src_dev, size_t bytes, void* stream);
int32_t enigma_memset(void* dst_dev, int32_t value, size_t bytes, void* stream);

/* ---- the hot-path operators (asynchronous on `stream`) ---- */

/* y = x * rsqrt(mean(x^2) + eps) * w per row; x, y [rows, hidden] row-major, w [hidden].
 * Replaces the dispatch of rmsnorm_kernel (examples/benchmark_rmsnorm.py:31-84)
 * and of rmsnorm (examples/metal/rmsnorm_handwritten.metal:4-46). */
int32_t enigma_rmsnorm(int32_t dtype, const void* x, const void* w, void* y, int64_t rows,
                       int64_t hidden, float eps, void* stream);

/* C[M,N] = A[M,K] * B[K,N], all row-major bf16, fp32 accumulate, bf16 out.
 * Replaces the dispatch of gemm_async (examples/async_copy_gemm.py:32-79);
 * semantics of enigma.gemm (enigma/ops/gemm.py:51-167) with beta = 0. */
int32_t enigma_gemm_bf16(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K,
                         void* stream);

/* O = softmax(scale * Q K^T [+ causal mask]) V per (batch, head); bf16 in and out,
 * Q/O [B, Hq, Sq, D], K/V [B, Hkv, Skv, D], GQA maps q-head h to kv-head h / (Hq/Hkv).
 * causal masks key j > query i + (Skv - Sq) (bottom-right aligned).
 * Replaces the dispatch of sdpa_enigma (examples/benchmark_sdpa.py:48-158),
 * fa_naive / fa_tv_kernel (examples/showcase_attention.py:31-125). */
int32_t enigma_sdpa_bf16(const void* Q, const void* K, const void* V, void* O, int64_t batch,
                         int64_t heads_q, int64_t heads_kv, int64_t seq_q, int64_t seq_kv,
                         int64_t head_dim, float scale, int32_t causal, void* stream);

/* C[i] = A[i] op B[i] for i < n; op 0 add, 1 sub, 2 mul, 3 max, 4 min; fp32 or bf16.
 * Replaces the dispatch of add_kernel (examples/vector_add_tv.py:13-55) and the
 * one-thread-per-element kernels of examples/vector_add.py.  Buffers 16-byte aligned
 * for the vector path (any alignment of the element size works, slower). */
int32_t enigma_elementwise(int32_t op, int32_t dtype, const void* A, const void* B, void* C,
                           int64_t n, void* stream);

/* fp32 reference-shape variants on CUDA cores (exact fp32 FMA accumulation):
 * C[M,N] (+)= A[M,K] * B[K,N] — replaces matmul_k4 / gemm_k4
 * (tests/metal/test_gemm_matmul_runtime.py:20-60); `accumulate` != 0 adds into C. */
int32_t enigma_gemm_f32(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K,
                        int32_t accumulate, void* stream);
/* The same with either operand transposed: A is [K, M] when trans_a, B is [N, K] when
 * trans_b — replaces the tile op enigma.gemm(A_s, B_s, C, M, N, K, transpose_A,
 * transpose_B) (enigma/ops/gemm.py:51-167; C += A @ B, C starting from the zero-filled
 * register tile, tests/metal/test_new_features_runtime.py:25-56). */
int32_t enigma_gemm_f32_trans(const void* A, const void* B, void* C, int64_t M, int64_t N,
                              int64_t K, int32_t trans_a, int32_t trans_b, int32_t accumulate,
                              void* stream);
/* fp32 attention, same layout and masking as enigma_sdpa_bf16 (showcase_attention.py:31-125,
 * benchmark_sdpa.py:48-150 with the KV de-interleaved). */
int32_t enigma_sdpa_f32(const void* Q, const void* K, const void* V, void* O, int64_t batch,
                        int64_t heads_q, int64_t heads_kv, int64_t seq_q, int64_t seq_kv,
                        int64_t head_dim, float scale, int32_t causal, void* stream);

/* Attention over strided views (CUDA cores, any head_dim <= 256): strides12 holds the
 * element strides (batch, head, sequence) of Q, K, V and O in that order; head_dim is
 * contiguous.  Lets reference layouts run without copies, e.g. the token-major Q/O
 * [tokens, heads, D] and the interleaved [kv_head, token, K|V] buffer of
 * examples/benchmark_sdpa.py:188-194. */
int32_t enigma_sdpa_strided(int32_t dtype, const void* Q, const void* K, const void* V, void* O,
                            int64_t batch, int64_t heads_q, int64_t heads_kv, int64_t seq_q,
                            int64_t seq_kv, int64_t head_dim, const int64_t* strides12,
                            float scale, int32_t causal, void* stream);
/* As enigma_sdpa_strided with an attention sink per query head (gpt-oss): sinks[h] is a
 * logit in the same units as scale * q.k that joins the softmax denominator only, i.e.
 * O = sum_j e^(s_j - M) v_j / (e^(sinks[h] - M) + sum_j e^(s_j - M)).  Replaces the
 * sink / running-max buffer `s` of examples/metal/sdpa_handwritten.metal:16-42 (m starts at
 * s[h], l at 1) and of sdpa_enigma (examples/benchmark_sdpa.py:64-72).  sinks may be NULL. */
int32_t enigma_sdpa_strided_sinks(int32_t dtype, const void* Q, const void* K, const void* V,
                                  void* O, int64_t batch, int64_t heads_q, int64_t heads_kv,
                                  int64_t seq_q, int64_t seq_kv, int64_t head_dim,
                                  const int64_t* strides12, float scale, int32_t causal,
                                  const float* sinks, void* stream);

/* ---- RMSNorm of host-resident rows (the reference's execute() path: host arrays in, host
 *      bytes out, runtime.py:318-421, for the RMSNorm of examples/benchmark_rmsnorm.py) ----
 * x_host [rows, hidden] -> y_host, w_host [hidden]; dtype ENIGMA_DTYPE_F32 or _BF16.  Rows go
 * through the GPU in chunks of chunk_rows on two streams (the caller's and a library-owned
 * one): chunk c's upload, kernel and download run in order on stream c % 2, so uploads,
 * kernels and downloads of neighbouring chunks overlap (host<->device copies are full
 * duplex).  x_host / y_host should be page-locked (enigma_host_alloc) for the copies to
 * overlap.  workspace: device memory of enigma_rmsnorm_host_workspace_bytes() bytes, 256-byte
 * aligned (w and two chunk buffers each way).  Synchronous: returns when y_host is written. */
int32_t enigma_rmsnorm_host_workspace_bytes(int32_t dtype, int64_t hidden, int64_t chunk_rows,
                                            size_t* bytes);
int32_t enigma_rmsnorm_host(int32_t dtype, const void* x_host, const void* w_host, void* y_host,
                            int64_t rows, int64_t hidden, float eps, void* workspace,
                            size_t workspace_bytes, int64_t chunk_rows, void* stream);

/* ---- one decoder-layer decode step (Qwen-style; the reference's qwen_fused megakernel,
 *      examples/qwen_megakernel.py:228-269, at BASELINE config 5 shapes) ----
 * x, out: [batch, hidden] bf16.  Weights bf16, row-major [in, out]:
 *   w_qkv [hidden, (heads_q + 2 heads_kv) * head_dim]   (q heads | k heads | v heads)
 *   w_o [heads_q * head_dim, hidden], w_gate_up [hidden, 2 * intermediate] (gate | up),
 *   w_down [intermediate, hidden]; w_in_norm / w_post_norm [hidden].
 * rope_cos / rope_sin: fp32 [head_dim] rotate-half tables for `position`.
 * k_cache / v_cache: bf16 [batch, heads_kv, cache_capacity, head_dim]; the step writes
 * the new token's k, v at `position` and attends over position + 1 keys.
 * head_dim must be 64; heads_q / heads_kv <= 8; hidden <= 2048; batch <= 128.
 * workspace: caller-owned device memory of enigma_decode_workspace_bytes() bytes. */
typedef struct enigma_decode_layer_desc {
  int64_t batch, hidden, heads_q, heads_kv, head_dim, intermediate, cache_capacity, position;
  float eps, attn_scale;
  const void *w_in_norm, *w_qkv, *w_o, *w_post_norm, *w_gate_up, *w_down;
  const float *rope_cos, *rope_sin;
  void *k_cache, *v_cache;
} enigma_decode_layer_desc;
int32_t enigma_decode_workspace_bytes(const enigma_decode_layer_desc* desc, size_t* bytes);
int32_t enigma_decode_layer_bf16(const enigma_decode_layer_desc* desc, const void* x, void* out,
                                 void* workspace, size_t workspace_bytes, void* stream);

/* The reference's own fp32 single-token layer (qwen_fused, examples/qwen_megakernel.py:
 * 228-269) with its buffer set: weights row-major [out, in] (y = W x); caches
 * [heads_kv, cache_total, head_dim] already holding the new token's k / v (as the
 * reference's host prepares them); norm_buf .. k_rope_buf are the reference's scratch
 * buffers and serve as the workspace.  fp32 throughout; head_dim even and <= 256. */
typedef struct enigma_qwen_decode_f32_desc {
  int64_t hidden, heads_q, heads_kv, head_dim, intermediate, cache_total;
  float eps, attn_scale;
  const float *x, *w_norm, *Wq, *Wk, *Wv, *w_q_norm, *w_k_norm, *cos_pos, *sin_pos;
  const float *k_cache, *v_cache, *Wo, *w_post, *Wg, *Wu, *Wd;
  float *norm_buf, *q_buf, *k_buf, *v_buf, *attn_buf, *mlp_buf, *post_buf, *q_rope_buf,
      *k_rope_buf, *out;
} enigma_qwen_decode_f32_desc;
int32_t enigma_qwen_decode_f32(const enigma_qwen_decode_f32_desc* desc, void* stream);

/* The same decode step without a caller-provided workspace, for callers that cannot
 * allocate device memory on this path: a serving loop that must never enter the
 * allocator, a plugin inside a host runtime that owns all device memory, code where an
 * allocation failure mid-step is not acceptable.  (No counterpart in the reference: its
 * Metal runtime always allocates buffers per call.)  The workspace is a fixed 16 MiB
 * device array inside this library, held on every GPU that loads it until the process
 * exits; a step that needs more (enigma_decode_workspace_bytes) is rejected with
 * ENIGMA_ERR_BADARG.  Its first call on a device looks up the array's device address once
 * (cudaGetSymbolAddress), so make that first call before any stream capture.  With lazy
 * module loading (CUDA's default) that first call is also when the driver loads this
 * library's device code on the device and commits the 16 MiB: it can fail for lack of
 * device memory, so make it during set-up.  Later calls allocate nothing.  A bounded wait
 * that runs out flags this entry's own static status word; enigma_synchronize and
 * enigma_take_device_status report it (ENIGMA_ERR_TIMEOUT) once and clear it.  All calls
 * share the array: calls that overlap on the GPU race, so serialize them on one stream. */
int32_t enigma_decode_layer_bf16_noalloc(const enigma_decode_layer_desc* desc, const void* x,
                                         void* out, void* stream);
/* Self-test of that reporting: the probe of enigma_check_timeout_path aimed at the
 * no-allocation entry's status word. */
int32_t enigma_decode_noalloc_check_timeout_path(int64_t polls, void* stream);

/* ---- serving: prompts of different lengths, and a cache in pages ----
 * (No counterpart in the reference, whose one decode example owns a dense cache of one
 * sequence, examples/qwen_megakernel.py:228-269.) */

/* Attention over whole prompts packed one after the other: sequence s owns lens_q[s] rows of
 * q [tokens_q, heads_q, head_dim] and lens_k[s] rows of k, v [tokens_k, heads_kv, head_dim].
 *   out_i = sum_j softmax_j(scale q_i . k_j) v_j  over the sequence's keys,
 * with causal j <= i + lens_k[s] - lens_q[s]; query head h reads kv head h / (heads_q /
 * heads_kv).  A row that sees no key gives zeros and lse -inf.  Token and head strides are
 * in elements, head_dim is contiguous; lse (may be NULL) is [tokens_q, heads_q], natural log.
 * Keys of other sequences are never read into a result, whatever they hold; a masked key of a
 * row's own sequence must be finite in v.  scale must be positive.
 *
 * enigma_sdpa_packed_plan (host only) lays out the work for these lengths, so a batch's layers
 * share one plan: which thread block does what, evenly, with long rows split over their keys
 * where there are few.  It writes *n_ints ints into plan[capacity] (plan NULL: only counts),
 * the first ENIGMA_PACKED_PLAN_HEADER of them the header.  The caller keeps the plan in device
 * memory (16-byte aligned) and gives the header with every call; a plan that splits rows needs a workspace of
 * enigma_sdpa_packed_workspace_bytes() bytes, 256-byte aligned. */
#define ENIGMA_PACKED_PLAN_HEADER 8
#define ENIGMA_PACKED_TILE_ROWS 128
int32_t enigma_sdpa_packed_plan(const int64_t* lens_q, const int64_t* lens_k, int64_t n_seqs,
                                int64_t heads_q, int64_t heads_kv, int32_t causal, int32_t* plan,
                                int64_t capacity, int64_t* n_ints);
int32_t enigma_sdpa_packed_workspace_bytes(const int32_t* header, int64_t head_dim, size_t* bytes);
typedef struct enigma_sdpa_packed_desc {
  int64_t tokens_q, tokens_k, heads_q, heads_kv, head_dim;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;
  float scale;
  int32_t causal, dtype, reserved;
  int32_t header[ENIGMA_PACKED_PLAN_HEADER];
  const int32_t* plan;
  const void *q, *k, *v;
  void* out;
  float* lse;
  void* workspace;
  size_t workspace_bytes;
} enigma_sdpa_packed_desc;
int32_t enigma_sdpa_packed(const enigma_sdpa_packed_desc* desc, void* stream);

/* One new token per sequence over a paged cache: q, out [batch, heads_q, head_dim]; pages
 * [pages, heads_kv, page, head_dim] (contiguous but for the page strides, in elements);
 * table [n_slots, table_width] int32 page numbers, lens [n_slots] int32 keys of each sequence;
 * sequence b uses row slots[b] (slots NULL: row b).  The first prefix_len keys are the same for
 * the whole batch: they are read through the row of sequence 0.  bf16 with heads of 64 or 128,
 * strides of multiples of 8 and 16-byte aligned buffers runs on the tensor cores, which read a
 * prefix once for every 256 rows (sequence, query head) of a kv head, in tables of at most 1536
 * keys once per sequence and kv head; other calls read it once per sequence and query head.  A
 * sequence attends to its first min(lens, table_width * page) keys; none gives zeros, and a slot
 * that does not exist has none.  A key whose table entry is no page is a key and a value of zeros.  Keys that
 * no sequence sees may hold anything; a prefix key that one sequence sees must be finite in v if
 * another is too short to see it.  scale is positive, page 16, 32, 64 or 128, batch <= 4096.  workspace: caller-owned device memory of
 * enigma_sdpa_shared_prefix_workspace_bytes() bytes, 256-byte aligned. */
typedef struct enigma_sdpa_shared_prefix_desc {
  int64_t batch, heads_q, heads_kv, head_dim, page, pages, table_width, n_slots, prefix_len;
  int64_t q_batch, q_head, o_batch, o_head, k_page, v_page;
  float scale;
  int32_t dtype;
  const int32_t *table, *lens, *slots;
  const void *q, *k_pages, *v_pages;
  void *out, *workspace;
  size_t workspace_bytes;
} enigma_sdpa_shared_prefix_desc;
int32_t enigma_sdpa_shared_prefix_workspace_bytes(const enigma_sdpa_shared_prefix_desc* desc,
                                                  size_t* bytes);
int32_t enigma_sdpa_shared_prefix(const enigma_sdpa_shared_prefix_desc* desc, void* stream);

/* A paged cache: k, v [layers, pages, heads_kv, page, head_dim]; table [slots, table_width]
 * (-1: none), lens [slots], refs [pages] (rows that hold the page; 0: free), status [1], all
 * int32 on the device.  Requests (n entries) are int32 device arrays.  New pages are the lowest
 * free ones in the order of the request.  A request that cannot be met changes nothing and
 * sets ENIGMA_CACHE_FULL or ENIGMA_CACHE_BAD_REQUEST in *status (a slot out of range or named
 * twice, a parent among the children, a length below the current one or past the table).
 *   fork     children[i] lets go of its pages and continues parents[i]: full pages are
 *            shared, the valid rows of a partly filled last page are copied to a new page.
 *   free     the slots let go of their pages.
 *   reserve  slots[i] grows to lens[i] tokens.
 *   write    rows of new_k / new_v (strides4: k token, k head, v token, v head, in elements)
 *            of one layer: rows cu[i] .. cu[i + 1] are tokens starts[i], ... of slots[i];
 *            a token without a page is left out and sets ENIGMA_CACHE_BAD_REQUEST.  A page that
 *            forks share (a full one) is written for all of them: appending never meets one,
 *            writing over earlier tokens may.
 *   compact  the n live pages take the numbers below n; rows are rewritten to match.
 *   copy_pages  whole pages src[i] -> dst[i], all layers; no page both source and destination
 *            (that is not checked, numbers out of range are).
 * workspace: enigma_kv_cache_workspace_bytes() bytes; calls that share it run in one order. */
#define ENIGMA_CACHE_FULL 1
#define ENIGMA_CACHE_BAD_REQUEST 2
#define ENIGMA_CACHE_MAX_REQUEST 8192   /* entries of one fork, free or reserve */
typedef struct enigma_kv_cache_desc {
  int64_t layers, pages, heads_kv, page, head_dim, elem_bytes, slots, table_width;
  void *k, *v;
  int32_t *table, *lens, *refs, *status;
  void* workspace;
  size_t workspace_bytes;
} enigma_kv_cache_desc;
int32_t enigma_kv_cache_workspace_bytes(const enigma_kv_cache_desc* desc, size_t* bytes);
int32_t enigma_kv_cache_fork(const enigma_kv_cache_desc* desc, const int32_t* parents,
                             const int32_t* children, int64_t n, void* stream);
int32_t enigma_kv_cache_free(const enigma_kv_cache_desc* desc, const int32_t* slots, int64_t n,
                             void* stream);
int32_t enigma_kv_cache_reserve(const enigma_kv_cache_desc* desc, const int32_t* slots,
                                const int32_t* lens, int64_t n, void* stream);
int32_t enigma_kv_cache_write(const enigma_kv_cache_desc* desc, int64_t layer, const void* new_k,
                              const void* new_v, const int64_t* strides4, const int32_t* slots,
                              const int32_t* starts, const int32_t* cu, int64_t n, int64_t tokens,
                              void* stream);
int32_t enigma_kv_cache_compact(const enigma_kv_cache_desc* desc, void* stream);
int32_t enigma_kv_cache_copy_pages(const enigma_kv_cache_desc* desc, const int32_t* src,
                                   const int32_t* dst, int64_t n, void* stream);

/* ---- rotary positions, and the paged cache in 8-bit codes ----
 * (No counterpart in the reference, whose decode example turns one token's heads by two given
 * tables inside its kernel, examples/qwen_megakernel.py:228-269.) */

/* Turns queries q [tokens, heads_q, head_dim] and keys k [tokens, heads_k, head_dim] (heads_k 0:
 * queries alone) to their positions in one launch.  Pair i of a head's first rotary_dim elements
 * (x[i], x[i + rotary_dim / 2]) in the half layout, (x[2i], x[2i + 1]) interleaved, turns by
 * positions[token] * turns[i] / 2^64 of a full turn and is multiplied by `factor`; the elements
 * behind are copied.  inverse != 0 turns back: the transpose of the same map, so its gradient.
 * Positions are int32 or int64 (position_bytes); turns [rotary_dim / 2] is a device array, a
 * frequency w in radians being round(w / 2 pi * 2^64) modulo 2^64.  Token and head strides in
 * elements, head_dim contiguous; an output may be its input, but not overlap it otherwise. */
#define ENIGMA_ROPE_HALF 0
#define ENIGMA_ROPE_INTERLEAVED 1
typedef struct enigma_rope_desc {
  int64_t tokens, heads_q, heads_k, head_dim, rotary_dim;
  int64_t q_token, q_head, k_token, k_head, oq_token, oq_head, ok_token, ok_head;
  float factor;
  int32_t dtype, layout, inverse, position_bytes, reserved;
  const void* positions;
  const uint64_t* turns;
  const void *q, *k;
  void *out_q, *out_k;
} enigma_rope_desc;
int32_t enigma_rope(const enigma_rope_desc* desc, void* stream);

/* A paged cache whose pages hold 8-bit codes (cache.elem_bytes 1; whole numbers in [-127, 127] or
 * e4m3 floats) with one fp32 scale for each ENIGMA_SCALE_BLOCK tokens of a page and head:
 * k_scale, v_scale [layers, pages, heads_kv, page / ENIGMA_SCALE_BLOCK]; a code stands for code *
 * scale.  head_dim is a multiple of 16 up to 256, page 16, 32, 64 or 128; pages are 16-byte aligned.
 * enigma_kv_cache_free and enigma_kv_cache_reserve take `cache` itself; fork, compact and
 * copy_pages are those of enigma_kv_cache_* with the scales moved along.
 *   write  as enigma_kv_cache_write, from rows of any type.  The scale of a block is the least
 *          power of two 2^e under which the block's largest magnitude (2^-110 if that is more) is at most
 *          127, or 448, and a code is the value over the scale, rounded to nearest (ties to
 *          even).  A write that starts behind a block's first token keeps the block's earlier
 *          tokens: its scale is the larger of the block's and the new tokens' (in magnitude: the
 *          block's may be any finite number, and stays where it is the larger one, the new codes
 *          being rounded from products with its fp32 reciprocal), and where it
 *          grows the earlier codes are rounded to it.  What a block held behind the last
 *          written token is lost.  A value that is not finite makes its block's scale NaN, until
 *          a write starts the block anew.  A page that forks share is not written
 *          (ENIGMA_CACHE_SHARED), nor is a block that two entries of a request name
 *          (ENIGMA_CACHE_BAD_REQUEST).
 *   read   rows cu[i] .. cu[i + 1] get the tokens starts[i], ... of slots[i]; a token that the slot does
 *          not hold gives zeros; rows before cu[0] and behind cu[n] are left as they were. */
#define ENIGMA_SCALE_BLOCK 16
#define ENIGMA_CODE_INT8 0
#define ENIGMA_CODE_E4M3 1
#define ENIGMA_CACHE_SHARED 4
typedef struct enigma_kv_cache_q8_desc {
  enigma_kv_cache_desc cache;
  float *k_scale, *v_scale;
  int32_t code, reserved;
} enigma_kv_cache_q8_desc;
int32_t enigma_kv_cache_q8_fork(const enigma_kv_cache_q8_desc* desc, const int32_t* parents,
                                const int32_t* children, int64_t n, void* stream);
int32_t enigma_kv_cache_q8_compact(const enigma_kv_cache_q8_desc* desc, void* stream);
int32_t enigma_kv_cache_q8_copy_pages(const enigma_kv_cache_q8_desc* desc, const int32_t* src,
                                      const int32_t* dst, int64_t n, void* stream);
/* Rows [tokens, heads_kv, head_dim] of one layer and the n entries of a request: what a write puts
 * into the cache, or where a read puts them.  Strides in elements. */
typedef struct enigma_kv_cache_rows {
  int64_t layer, n, tokens, k_token, k_head, v_token, v_head;
  int32_t dtype, reserved;
  void *k, *v;
  const int32_t *slots, *starts, *cu;
} enigma_kv_cache_rows;
int32_t enigma_kv_cache_q8_write(const enigma_kv_cache_q8_desc* desc, const enigma_kv_cache_rows* rows,
                                 void* stream);
int32_t enigma_kv_cache_q8_read(const enigma_kv_cache_q8_desc* desc, const enigma_kv_cache_rows* rows,
                                void* stream);

/* One new token per sequence over pages of 8-bit codes: q, out [batch, heads_q, head_dim] of type
 * dtype; k_pages, v_pages [pages, heads_kv, page, head_dim] codes, contiguous but for the page
 * strides (k_page, v_page, in codes, multiples of 16); k_scale, v_scale [pages, heads_kv, page /
 * ENIGMA_SCALE_BLOCK], contiguous but for theirs (ks_page, vs_page); scales are any finite numbers
 * (a weight times its v_scale is held to 2^-34 of the largest |v_scale| seen with it, 2^-40 in fp32).
 *   out = sum_j softmax_j(scale k_scale_j q . k_j) v_scale_j v_j
 * over the first min(lens, table_width * page) keys; tables, lens and slots as in
 * enigma_sdpa_shared_prefix: no keys, or a slot that does not exist, give zeros, and a key whose
 * table entry is no page is a key and a value of zeros.  A code or scale that is seen and is NaN
 * gives NaN; what no sequence sees may hold anything.  scale is positive, batch <= 4096, head_dim
 * a multiple of 16 up to 256, page 16, 32, 64 or 128; batch * table_width * page / 16 fits in int32.
 * workspace: caller-owned device memory of enigma_sdpa_quantized_workspace_bytes() bytes, 256-byte
 * aligned. */
typedef struct enigma_sdpa_quantized_desc {
  int64_t batch, heads_q, heads_kv, head_dim, page, pages, table_width, n_slots;
  int64_t q_batch, q_head, o_batch, o_head, k_page, v_page, ks_page, vs_page;
  float scale;
  int32_t dtype, code, reserved;
  const int32_t *table, *lens, *slots;
  const void *q, *k_pages, *v_pages;
  const float *k_scale, *v_scale;
  void *out, *workspace;
  size_t workspace_bytes;
} enigma_sdpa_quantized_desc;
int32_t enigma_sdpa_quantized_workspace_bytes(const enigma_sdpa_quantized_desc* desc, size_t* bytes);
int32_t enigma_sdpa_quantized(const enigma_sdpa_quantized_desc* desc, void* stream);

/* ---- generic dispatch by kernel id: replaces enigma_dispatch /
 *      enigma_dispatch_timed (libenigma_runtime.swift:132-214).
 *      grid / threads are Metal-style totals (threads per axis, not groups),
 *      accepted for interface parity and checked (no zero extent, at most 1024
 *      threads per threadgroup; NULL = not given); the kernels pick their own
 *      CTA shapes.
 *      dispatch_timed returns the device time of the launch in microseconds,
 *      measured with CUDA events on `stream`, and synchronizes. ---- */
int32_t enigma_dispatch(int32_t kernel_id, void* const* buffers, int32_t n_buffers,
                        const int64_t* iparams, int32_t n_iparams, const float* fparams,
                        int32_t n_fparams, const uint32_t* grid3, const uint32_t* threads3,
                        void* stream);
int32_t enigma_dispatch_timed(int32_t kernel_id, void* const* buffers, int32_t n_buffers,
                              const int64_t* iparams, int32_t n_iparams, const float* fparams,
                              int32_t n_fparams, const uint32_t* grid3, const uint32_t* threads3,
                              void* stream, double* elapsed_us);

/* ---- event timing (for benchmarks that time a sequence of launches) ---- */
int32_t enigma_event_create(void** ev);
int32_t enigma_event_destroy(void* ev);
int32_t enigma_event_record(void* ev, void* stream);
int32_t enigma_event_elapsed_ms(void* start, void* stop, float* ms);

/* Number of device-side timeouts flagged since the last call (and reset): the library's
 * per-device status word plus the no-allocation decode entry's word.  Allocates nothing. */
int32_t enigma_take_device_status(int32_t* timeouts);
/* Self-test of the timeout reporting: enqueues one CTA that waits on a barrier nothing
 * arrives on, gives up after `polls` polls (<= 2^24; microseconds) and flags the device status
 * word as the kernels' bounded waits do; the next enigma_synchronize then returns
 * ENIGMA_ERR_TIMEOUT and clears it, and the context stays usable. */
int32_t enigma_check_timeout_path(int64_t polls, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* ENIGMA_CUDA_H */
