// serving_abi.cu — C-ABI entry points of the serving operators (packed prompt attention, paged
// attention with a shared prefix, page operations, rotary positions, the cache in 8-bit codes).
// Validation happens here; the kernels check what only the device knows (page numbers, slots,
// lengths).
#include <algorithm>
#include <exception>
#include <vector>

#include "attn_serving.cuh"

namespace enigma_serving {
std::vector<int32_t> make_packed_plan(const int64_t* lens_q, const int64_t* lens_k, int64_t n,
                                      int group, int heads_kv, bool causal, int sms);
}

using enigma::set_error;

namespace {

inline cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

int32_t launch_status(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return ENIGMA_OK;
  set_error("%s launch failed: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
  return ENIGMA_ERR_LAUNCH;
}

int32_t bad(const char* msg) {
  set_error("bad argument: %s", msg);
  return ENIGMA_ERR_BADARG;
}

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

constexpr int64_t kInt31 = (1ll << 31) - 1;

int32_t check_heads(int64_t heads_q, int64_t heads_kv, int64_t head_dim) {
  if (heads_q <= 0 || heads_kv <= 0 || heads_q % heads_kv != 0)
    return bad("heads_q must be a positive multiple of heads_kv");
  if (heads_q > 65535) return bad("heads_q must be at most 65535");
  if (head_dim <= 0 || head_dim > 256) return bad("head_dim must be in [1, 256]");
  return ENIGMA_OK;
}

// The kernels take a row's maximum before they scale it.
bool good_scale(float s) { return s > 0.f && s < 1e30f; }

int32_t check_shared(const enigma_sdpa_shared_prefix_desc* d) {
  if (d == nullptr) return bad("sdpa_shared_prefix: desc is NULL");
  if (d->dtype != ENIGMA_DTYPE_F32 && d->dtype != ENIGMA_DTYPE_BF16)
    return bad("sdpa_shared_prefix: dtype");
  const int32_t e = check_heads(d->heads_q, d->heads_kv, d->head_dim);
  if (e != ENIGMA_OK) return e;
  if (d->batch < 0 || d->batch > 4096) return bad("sdpa_shared_prefix: batch must be in [0, 4096]");
  if (d->page != 16 && d->page != 32 && d->page != 64 && d->page != 128)
    return bad("sdpa_shared_prefix: page must be 16, 32, 64 or 128");
  if (d->pages <= 0 || d->table_width <= 0 || d->n_slots < 0 || (d->n_slots == 0 && d->batch > 0))
    return bad("sdpa_shared_prefix: pages, table_width and n_slots must be positive");
  if (d->pages > kInt31 / (d->heads_kv * d->page) || d->table_width > (kInt31 - 256) / d->page ||
      d->n_slots > kInt31)
    return bad("sdpa_shared_prefix: sizes must fit in int32");
  if (d->prefix_len < 0 || d->prefix_len > d->table_width * d->page)
    return bad("sdpa_shared_prefix: prefix_len must be in [0, table_width * page]");
  return ENIGMA_OK;
}

// map: only the page map is touched, whatever the pages hold.
int32_t check_cache(const enigma_kv_cache_desc* d, bool run, bool map = false) {
  if (d == nullptr) return bad("kv_cache: desc is NULL");
  if (d->layers <= 0 || d->pages <= 0 || d->heads_kv <= 0 || d->page <= 0 || d->head_dim <= 0 ||
      d->slots <= 0 || d->table_width <= 0)
    return bad("kv_cache: sizes must be positive");
  if (d->elem_bytes != 2 && d->elem_bytes != 4 && !(map && d->elem_bytes == 1))
    return bad("kv_cache: elem_bytes must be 2 or 4");
  if (d->slots > 262144) return bad("kv_cache: at most 262144 slots");
  if (d->pages > kInt31 || d->layers > kInt31 || d->heads_kv > kInt31 || d->page > kInt31 ||
      d->head_dim > (1 << 20) || d->table_width > (kInt31 - d->page) / d->page)
    return bad("kv_cache: sizes must fit in int32");
  if (!run) return ENIGMA_OK;
  if (d->k == nullptr || d->v == nullptr || d->table == nullptr || d->lens == nullptr ||
      d->refs == nullptr || d->status == nullptr)
    return bad("kv_cache: NULL buffer");
  if (!aligned(d->k, size_t(d->elem_bytes)) || !aligned(d->v, size_t(d->elem_bytes)))
    return bad("kv_cache: misaligned buffer");
  if (d->workspace == nullptr || !aligned(d->workspace, 4) ||
      d->workspace_bytes < enigma::kv_cache_workspace_bytes(*d))
    return bad("kv_cache: workspace must hold enigma_kv_cache_workspace_bytes() bytes");
  return ENIGMA_OK;
}

// Entries of one request: at most one per slot.
int32_t check_request(const enigma_kv_cache_desc* d, const void* a, const void* b, int64_t n,
                      bool map) {
  const int32_t e = check_cache(d, true, map);
  if (e != ENIGMA_OK) return e;
  if (n < 0 || n > d->slots) return bad("kv_cache: a request names each slot at most once");
  if (n > ENIGMA_CACHE_MAX_REQUEST) return bad("kv_cache: a request has at most 8192 entries");
  if (n > 0 && (a == nullptr || b == nullptr)) return bad("kv_cache: NULL request");
  return ENIGMA_OK;
}

bool good_page(int64_t page) { return page == 16 || page == 32 || page == 64 || page == 128; }

int32_t check_codes(int64_t head_dim, int64_t page, int32_t code) {
  if (head_dim <= 0 || head_dim > 256 || head_dim % 16 != 0)
    return bad("8-bit cache: head_dim must be a multiple of 16 up to 256");
  if (!good_page(page)) return bad("8-bit cache: page must be 16, 32, 64 or 128");
  if (code != ENIGMA_CODE_INT8 && code != ENIGMA_CODE_E4M3) return bad("8-bit cache: code");
  return ENIGMA_OK;
}

int32_t check_q8(const enigma_kv_cache_q8_desc* d) {
  if (d == nullptr) return bad("kv_cache_q8: desc is NULL");
  int32_t e = check_cache(&d->cache, true, true);
  if (e != ENIGMA_OK) return e;
  if (d->cache.elem_bytes != 1) return bad("kv_cache_q8: elem_bytes must be 1");
  if (d->cache.heads_kv > 65535) return bad("kv_cache_q8: heads_kv must be at most 65535");
  e = check_codes(d->cache.head_dim, d->cache.page, d->code);
  if (e != ENIGMA_OK) return e;
  if (d->k_scale == nullptr || d->v_scale == nullptr) return bad("kv_cache_q8: NULL buffer");
  if (!aligned(d->cache.k, 16) || !aligned(d->cache.v, 16) || !aligned(d->k_scale, 4) ||
      !aligned(d->v_scale, 4))
    return bad("kv_cache_q8: misaligned buffer");
  return ENIGMA_OK;
}

// The rows of a write or read.
int32_t check_rows(const enigma_kv_cache_q8_desc* d, const enigma_kv_cache_rows* w) {
  if (w == nullptr) return bad("kv_cache_q8: rows is NULL");
  if (w->layer < 0 || w->layer >= d->cache.layers) return bad("kv_cache_q8: layer out of range");
  if (w->dtype != ENIGMA_DTYPE_F32 && w->dtype != ENIGMA_DTYPE_BF16) return bad("kv_cache_q8: dtype");
  if (w->n < 0 || w->tokens < 0 || w->n > kInt31 - 256 || w->tokens > kInt31 - 256)
    return bad("kv_cache_q8: request size");
  if (w->tokens == 0) return ENIGMA_OK;
  if (w->n == 0) return bad("kv_cache_q8: rows without a slot");
  if (w->k == nullptr || w->v == nullptr || w->slots == nullptr || w->starts == nullptr ||
      w->cu == nullptr)
    return bad("kv_cache_q8: NULL request");
  if (w->k_token < 0 || w->k_head < 0 || w->v_token < 0 || w->v_head < 0)
    return bad("kv_cache_q8: negative stride");
  const size_t es = w->dtype == ENIGMA_DTYPE_F32 ? 4 : 2;
  if (!aligned(w->k, es) || !aligned(w->v, es) || !aligned(w->slots, 4) || !aligned(w->starts, 4) ||
      !aligned(w->cu, 4))
    return bad("kv_cache_q8: misaligned buffer");
  return ENIGMA_OK;
}

int32_t check_quantized(const enigma_sdpa_quantized_desc* d) {
  if (d == nullptr) return bad("sdpa_quantized: desc is NULL");
  if (d->dtype != ENIGMA_DTYPE_F32 && d->dtype != ENIGMA_DTYPE_BF16)
    return bad("sdpa_quantized: dtype");
  int32_t e = check_heads(d->heads_q, d->heads_kv, d->head_dim);
  if (e == ENIGMA_OK) e = check_codes(d->head_dim, d->page, d->code);
  if (e != ENIGMA_OK) return e;
  if (d->batch < 0 || d->batch > 4096) return bad("sdpa_quantized: batch must be in [0, 4096]");
  if (d->pages <= 0 || d->table_width <= 0 || d->n_slots < 0 || (d->n_slots == 0 && d->batch > 0))
    return bad("sdpa_quantized: pages, table_width and n_slots must be positive");
  if (d->pages > kInt31 / (d->heads_kv * d->page) || d->table_width > (kInt31 - 256) / d->page ||
      d->n_slots > kInt31)
    return bad("sdpa_quantized: sizes must fit in int32");
  // The kernel counts a batch's chunks of 16 keys or more, and up to four for a sequence's start, in 32
  // bits, a thread's share of all heads' too.
  const int64_t chunks = d->batch * (d->table_width * d->page / 16 + 5);
  if (chunks > kInt31 || double(chunks) * double(d->heads_q) > 1e12)
    return bad("sdpa_quantized: more keys than one call takes");
  return ENIGMA_OK;
}

}  // namespace

extern "C" {

int32_t enigma_sdpa_packed_plan(const int64_t* lens_q, const int64_t* lens_k, int64_t n_seqs,
                                int64_t heads_q, int64_t heads_kv, int32_t causal, int32_t* plan,
                                int64_t capacity, int64_t* n_ints) {
  if (n_ints == nullptr) return bad("sdpa_packed_plan: n_ints is NULL");
  if (n_seqs < 0 || (n_seqs > 0 && (lens_q == nullptr || lens_k == nullptr)))
    return bad("sdpa_packed_plan: NULL lengths");
  const int32_t e = check_heads(heads_q, heads_kv, 1);
  if (e != ENIGMA_OK) return e;
  int64_t total_q = 0, total_k = 0;
  for (int64_t s = 0; s < n_seqs; ++s) {
    if (lens_q[s] < 0 || lens_k[s] < 0) return bad("sdpa_packed_plan: negative length");
    if (lens_q[s] > kInt31 || lens_k[s] > kInt31) return bad("sdpa_packed_plan: too long");
    total_q += lens_q[s];
    total_k += lens_k[s];
    if (total_q > kInt31 - 256 || total_k > kInt31 - 256)
      return bad("sdpa_packed_plan: token counts must fit in int32");
  }
  try {
    const std::vector<int32_t> ints = enigma_serving::make_packed_plan(
        lens_q, lens_k, n_seqs, int(heads_q / heads_kv), int(heads_kv), causal != 0,
        enigma::sm_count());
    if (ints.empty()) return bad("sdpa_packed_plan: too much work for one plan");
    *n_ints = int64_t(ints.size());
    if (plan == nullptr) return ENIGMA_OK;
    if (capacity < *n_ints) return bad("sdpa_packed_plan: capacity is less than the plan");
    std::copy(ints.begin(), ints.end(), plan);
  } catch (const std::exception&) {
    return bad("sdpa_packed_plan: out of host memory");
  }
  return ENIGMA_OK;
}

int32_t enigma_sdpa_packed_workspace_bytes(const int32_t* header, int64_t head_dim, size_t* bytes) {
  if (header == nullptr || bytes == nullptr) return bad("sdpa_packed: NULL argument");
  if (head_dim <= 0 || head_dim > 256) return bad("head_dim must be in [1, 256]");
  const int64_t slots = header[enigma_serving::kSlots];
  if (slots < 0) return bad("sdpa_packed: not a plan's header");
  *bytes = size_t(slots) * ENIGMA_PACKED_TILE_ROWS * (size_t(head_dim) + 2) * sizeof(float);
  return ENIGMA_OK;
}

int32_t enigma_sdpa_packed(const enigma_sdpa_packed_desc* d, void* stream) {
  if (d == nullptr) return bad("sdpa_packed: desc is NULL");
  if (d->dtype != ENIGMA_DTYPE_F32 && d->dtype != ENIGMA_DTYPE_BF16)
    return bad("sdpa_packed: dtype");
  int32_t e = check_heads(d->heads_q, d->heads_kv, d->head_dim);
  if (e != ENIGMA_OK) return e;
  if (!good_scale(d->scale)) return bad("sdpa_packed: scale must be positive and finite");
  if (d->tokens_q < 0 || d->tokens_k < 0) return bad("sdpa_packed: negative size");
  if (d->tokens_q > kInt31 - 256 || d->tokens_k > kInt31 - 256)
    return bad("sdpa_packed: sizes must fit in int32");
  const int64_t strides[8] = {d->q_token, d->q_head, d->k_token, d->k_head,
                              d->v_token, d->v_head, d->o_token, d->o_head};
  for (int i = 0; i < 8; ++i)
    if (strides[i] < 0) return bad("sdpa_packed: negative stride");
  for (int i = 0; i < ENIGMA_PACKED_PLAN_HEADER; ++i)
    if (d->header[i] < 0) return bad("sdpa_packed: not a plan's header");
  if (d->tokens_q == 0 || d->header[enigma_serving::kItems] == 0) return ENIGMA_OK;
  if (d->plan == nullptr || d->q == nullptr || d->out == nullptr ||
      (d->tokens_k > 0 && (d->k == nullptr || d->v == nullptr)))
    return bad("sdpa_packed: NULL buffer");
  const size_t es = d->dtype == ENIGMA_DTYPE_F32 ? 4 : 2;
  if (!aligned(d->q, es) || !aligned(d->k, es) || !aligned(d->v, es) || !aligned(d->out, es) ||
      !aligned(d->lse, 4) || !aligned(d->plan, 16))
    return bad("sdpa_packed: misaligned buffer");
  size_t need = 0;
  e = enigma_sdpa_packed_workspace_bytes(d->header, d->head_dim, &need);
  if (e != ENIGMA_OK) return e;
  if (need > 0 &&
      (d->workspace == nullptr || !aligned(d->workspace, 256) || d->workspace_bytes < need))
    return bad("sdpa_packed: workspace must be 256-byte aligned and hold "
               "enigma_sdpa_packed_workspace_bytes() bytes");
  return launch_status(enigma::sdpa_packed_launch(*d, as_stream(stream)), "sdpa_packed");
}

int32_t enigma_sdpa_shared_prefix_workspace_bytes(const enigma_sdpa_shared_prefix_desc* d,
                                                  size_t* bytes) {
  const int32_t e = check_shared(d);
  if (e != ENIGMA_OK) return e;
  if (bytes == nullptr) return bad("sdpa_shared_prefix: bytes is NULL");
  *bytes = enigma::sdpa_shared_prefix_workspace(*d);
  return ENIGMA_OK;
}

int32_t enigma_sdpa_shared_prefix(const enigma_sdpa_shared_prefix_desc* d, void* stream) {
  const int32_t e = check_shared(d);
  if (e != ENIGMA_OK) return e;
  if (!good_scale(d->scale)) return bad("sdpa_shared_prefix: scale must be positive and finite");
  if (d->slots == nullptr && d->batch > d->n_slots)
    return bad("sdpa_shared_prefix: more sequences than table rows");
  if (d->q_batch < 0 || d->q_head < 0 || d->o_batch < 0 || d->o_head < 0 || d->k_page < 0 ||
      d->v_page < 0)
    return bad("sdpa_shared_prefix: negative stride");
  if (d->batch == 0) return ENIGMA_OK;
  if (d->q == nullptr || d->k_pages == nullptr || d->v_pages == nullptr || d->out == nullptr ||
      d->table == nullptr || d->lens == nullptr)
    return bad("sdpa_shared_prefix: NULL buffer");
  const size_t es = d->dtype == ENIGMA_DTYPE_F32 ? 4 : 2;
  if (!aligned(d->q, es) || !aligned(d->k_pages, es) || !aligned(d->v_pages, es) ||
      !aligned(d->out, es) || !aligned(d->table, 4) || !aligned(d->lens, 4) ||
      !aligned(d->slots, 4))
    return bad("sdpa_shared_prefix: misaligned buffer");
  const size_t need = enigma::sdpa_shared_prefix_workspace(*d);
  if (need > 0 && (d->workspace == nullptr || !aligned(d->workspace, 256) ||
                   d->workspace_bytes < need))
    return bad("sdpa_shared_prefix: workspace must be 256-byte aligned and hold "
               "enigma_sdpa_shared_prefix_workspace_bytes() bytes");
  return launch_status(enigma::sdpa_shared_prefix_launch(*d, as_stream(stream)),
                       "sdpa_shared_prefix");
}

int32_t enigma_kv_cache_workspace_bytes(const enigma_kv_cache_desc* d, size_t* bytes) {
  const int32_t e = check_cache(d, false, true);
  if (e != ENIGMA_OK) return e;
  if (bytes == nullptr) return bad("kv_cache: bytes is NULL");
  *bytes = enigma::kv_cache_workspace_bytes(*d);
  return ENIGMA_OK;
}

int32_t enigma_kv_cache_fork(const enigma_kv_cache_desc* d, const int32_t* parents,
                             const int32_t* children, int64_t n, void* stream) {
  const int32_t e = check_request(d, parents, children, n, false);
  if (e != ENIGMA_OK || n == 0) return e;
  return launch_status(enigma::kv_cache_fork(*d, parents, children, n, as_stream(stream)),
                       "kv_cache_fork");
}

int32_t enigma_kv_cache_free(const enigma_kv_cache_desc* d, const int32_t* slots, int64_t n,
                             void* stream) {
  const int32_t e = check_request(d, slots, slots, n, true);
  if (e != ENIGMA_OK || n == 0) return e;
  return launch_status(enigma::kv_cache_free(*d, slots, n, as_stream(stream)), "kv_cache_free");
}

int32_t enigma_kv_cache_reserve(const enigma_kv_cache_desc* d, const int32_t* slots,
                                const int32_t* lens, int64_t n, void* stream) {
  const int32_t e = check_request(d, slots, lens, n, true);
  if (e != ENIGMA_OK || n == 0) return e;
  return launch_status(enigma::kv_cache_reserve(*d, slots, lens, n, as_stream(stream)),
                       "kv_cache_reserve");
}

int32_t enigma_kv_cache_write(const enigma_kv_cache_desc* d, int64_t layer, const void* new_k,
                              const void* new_v, const int64_t* strides4, const int32_t* slots,
                              const int32_t* starts, const int32_t* cu, int64_t n, int64_t tokens,
                              void* stream) {
  const int32_t e = check_cache(d, true);
  if (e != ENIGMA_OK) return e;
  if (layer < 0 || layer >= d->layers) return bad("kv_cache: layer out of range");
  if (n < 0 || tokens < 0 || n > kInt31 || tokens > kInt31) return bad("kv_cache: request size");
  if (tokens == 0) return ENIGMA_OK;
  if (n == 0) return bad("kv_cache: rows without a slot");
  if (new_k == nullptr || new_v == nullptr || strides4 == nullptr || slots == nullptr ||
      starts == nullptr || cu == nullptr)
    return bad("kv_cache: NULL request");
  for (int i = 0; i < 4; ++i)
    if (strides4[i] < 0) return bad("kv_cache: negative stride");
  if (!aligned(new_k, size_t(d->elem_bytes)) || !aligned(new_v, size_t(d->elem_bytes)))
    return bad("kv_cache: misaligned buffer");
  return launch_status(enigma::kv_cache_write(*d, layer, new_k, new_v, strides4, slots, starts, cu,
                                              n, tokens, as_stream(stream)),
                       "kv_cache_write");
}

int32_t enigma_kv_cache_compact(const enigma_kv_cache_desc* d, void* stream) {
  const int32_t e = check_cache(d, true);
  if (e != ENIGMA_OK) return e;
  return launch_status(enigma::kv_cache_compact(*d, as_stream(stream)), "kv_cache_compact");
}

int32_t enigma_kv_cache_copy_pages(const enigma_kv_cache_desc* d, const int32_t* src,
                                   const int32_t* dst, int64_t n, void* stream) {
  const int32_t e = check_cache(d, true);
  if (e != ENIGMA_OK) return e;
  if (n < 0 || n > d->pages) return bad("kv_cache: more copies than pages");
  if (n == 0) return ENIGMA_OK;
  if (src == nullptr || dst == nullptr) return bad("kv_cache: NULL request");
  return launch_status(enigma::kv_cache_copy_pages(*d, src, dst, n, as_stream(stream)),
                       "kv_cache_copy_pages");
}

int32_t enigma_rope(const enigma_rope_desc* d, void* stream) {
  if (d == nullptr) return bad("rope: desc is NULL");
  if (d->dtype != ENIGMA_DTYPE_F32 && d->dtype != ENIGMA_DTYPE_BF16) return bad("rope: dtype");
  if (d->layout != ENIGMA_ROPE_HALF && d->layout != ENIGMA_ROPE_INTERLEAVED)
    return bad("rope: layout");
  if (d->position_bytes != 4 && d->position_bytes != 8)
    return bad("rope: positions are int32 or int64");
  if (d->heads_q <= 0 || d->heads_k < 0 || d->heads_q > 65535 || d->heads_k > 65535)
    return bad("rope: heads_q must be in [1, 65535], heads_k in [0, 65535]");
  if (d->head_dim <= 0 || d->head_dim > 4096) return bad("rope: head_dim must be in [1, 4096]");
  if (d->rotary_dim < 0 || d->rotary_dim > d->head_dim || d->rotary_dim % 2 != 0)
    return bad("rope: rotary_dim must be even and at most head_dim");
  if (d->tokens < 0 || d->tokens > kInt31 - 256) return bad("rope: token counts must fit in int32");
  const int64_t strides[8] = {d->q_token,  d->q_head,  d->k_token,  d->k_head,
                              d->oq_token, d->oq_head, d->ok_token, d->ok_head};
  for (int i = 0; i < 8; ++i)
    if (strides[i] < 0) return bad("rope: negative stride");
  if (d->tokens == 0) return ENIGMA_OK;
  if (d->positions == nullptr || (d->rotary_dim > 0 && d->turns == nullptr) || d->q == nullptr ||
      d->out_q == nullptr || (d->heads_k > 0 && (d->k == nullptr || d->out_k == nullptr)))
    return bad("rope: NULL buffer");
  const size_t es = d->dtype == ENIGMA_DTYPE_F32 ? 4 : 2;
  if (!aligned(d->q, es) || !aligned(d->k, es) || !aligned(d->out_q, es) ||
      !aligned(d->out_k, es) || !aligned(d->turns, 8) ||
      !aligned(d->positions, size_t(d->position_bytes)))
    return bad("rope: misaligned buffer");
  return launch_status(enigma::rope_launch(*d, as_stream(stream)), "rope");
}

int32_t enigma_kv_cache_q8_fork(const enigma_kv_cache_q8_desc* d, const int32_t* parents,
                                const int32_t* children, int64_t n, void* stream) {
  int32_t e = check_q8(d);
  if (e == ENIGMA_OK) e = check_request(&d->cache, parents, children, n, true);
  if (e != ENIGMA_OK || n == 0) return e;
  return launch_status(enigma::kv_cache_q8_fork(*d, parents, children, n, as_stream(stream)),
                       "kv_cache_q8_fork");
}

int32_t enigma_kv_cache_q8_compact(const enigma_kv_cache_q8_desc* d, void* stream) {
  const int32_t e = check_q8(d);
  if (e != ENIGMA_OK) return e;
  return launch_status(enigma::kv_cache_q8_compact(*d, as_stream(stream)), "kv_cache_q8_compact");
}

int32_t enigma_kv_cache_q8_copy_pages(const enigma_kv_cache_q8_desc* d, const int32_t* src,
                                      const int32_t* dst, int64_t n, void* stream) {
  const int32_t e = check_q8(d);
  if (e != ENIGMA_OK) return e;
  if (n < 0 || n > d->cache.pages) return bad("kv_cache_q8: more copies than pages");
  if (n == 0) return ENIGMA_OK;
  if (src == nullptr || dst == nullptr) return bad("kv_cache_q8: NULL request");
  return launch_status(enigma::kv_cache_q8_copy_pages(*d, src, dst, n, as_stream(stream)),
                       "kv_cache_q8_copy_pages");
}

int32_t enigma_kv_cache_q8_write(const enigma_kv_cache_q8_desc* d, const enigma_kv_cache_rows* rows,
                                 void* stream) {
  int32_t e = check_q8(d);
  if (e == ENIGMA_OK) e = check_rows(d, rows);
  if (e != ENIGMA_OK || rows->tokens == 0) return e;
  return launch_status(enigma::kv_cache_q8_write(*d, *rows, as_stream(stream)), "kv_cache_q8_write");
}

int32_t enigma_kv_cache_q8_read(const enigma_kv_cache_q8_desc* d, const enigma_kv_cache_rows* rows,
                                void* stream) {
  int32_t e = check_q8(d);
  if (e == ENIGMA_OK) e = check_rows(d, rows);
  if (e != ENIGMA_OK || rows->tokens == 0) return e;
  return launch_status(enigma::kv_cache_q8_read(*d, *rows, as_stream(stream)), "kv_cache_q8_read");
}

int32_t enigma_sdpa_quantized_workspace_bytes(const enigma_sdpa_quantized_desc* d, size_t* bytes) {
  const int32_t e = check_quantized(d);
  if (e != ENIGMA_OK) return e;
  if (bytes == nullptr) return bad("sdpa_quantized: bytes is NULL");
  *bytes = enigma::sdpa_quantized_workspace(*d);
  return ENIGMA_OK;
}

int32_t enigma_sdpa_quantized(const enigma_sdpa_quantized_desc* d, void* stream) {
  const int32_t e = check_quantized(d);
  if (e != ENIGMA_OK) return e;
  if (!good_scale(d->scale)) return bad("sdpa_quantized: scale must be positive and finite");
  if (d->slots == nullptr && d->batch > d->n_slots)
    return bad("sdpa_quantized: more sequences than table rows");
  if (d->q_batch < 0 || d->q_head < 0 || d->o_batch < 0 || d->o_head < 0 || d->k_page < 0 ||
      d->v_page < 0 || d->ks_page < 0 || d->vs_page < 0)
    return bad("sdpa_quantized: negative stride");
  if (d->batch == 0) return ENIGMA_OK;
  if (d->q == nullptr || d->k_pages == nullptr || d->v_pages == nullptr || d->out == nullptr ||
      d->k_scale == nullptr || d->v_scale == nullptr || d->table == nullptr || d->lens == nullptr)
    return bad("sdpa_quantized: NULL buffer");
  const size_t es = d->dtype == ENIGMA_DTYPE_F32 ? 4 : 2;
  if (!aligned(d->q, es) || !aligned(d->out, es) || !aligned(d->k_pages, 16) ||
      !aligned(d->v_pages, 16) || d->k_page % 16 != 0 || d->v_page % 16 != 0 ||
      !aligned(d->k_scale, 4) || !aligned(d->v_scale, 4) || !aligned(d->table, 4) ||
      !aligned(d->lens, 4) || !aligned(d->slots, 4))
    return bad("sdpa_quantized: misaligned buffer");
  const size_t need = enigma::sdpa_quantized_workspace(*d);
  if (need > 0 && (d->workspace == nullptr || !aligned(d->workspace, 256) ||
                   d->workspace_bytes < need))
    return bad("sdpa_quantized: workspace must be 256-byte aligned and hold "
               "enigma_sdpa_quantized_workspace_bytes() bytes");
  return launch_status(enigma::sdpa_quantized_launch(*d, as_stream(stream)), "sdpa_quantized");
}

}  // extern "C"
