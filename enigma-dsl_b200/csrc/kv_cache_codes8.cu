// kv_cache_codes8.cu — a paged cache in 8-bit codes: rows quantised as they are written, and read back.
//
// Codes and scales are those of codes8.cuh.  A write that starts inside a block of 16 tokens keeps
// the block's earlier tokens: the scale becomes the larger of the block's and what the new tokens
// need, and if it grows the earlier codes are rounded to it.  A write that starts a block, or
// goes on behind it, sets the scale from the new tokens alone: what the page held before, or a
// sequence that was cut short, does not count.  So a sequence's tokens are written in order, and
// what stands in a block behind the last written token means nothing.  A value that is not finite
// gives its block the scale NaN, until the block is started anew.
#include <algorithm>

#include "codes8.cuh"

namespace {

using namespace enigma_codes8;
using namespace enigma_sm100;

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Entry of packed row t: the last i in [0, n) with cu[i] <= t, found 32 ways at once.
__device__ __forceinline__ int entry_of(const int32_t* cu, int n, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, span = n;
  while (span > 1) {
    const int step = (span + 31) / 32, i = lo + (lane + 1) * step;
    const bool past = i >= lo + span || cu[i] > t;
    const int k = __ffs(__ballot_sync(0xffffffffu, past)) - 1;           // lane 31 is always past
    span = min(step, lo + span - (lo + k * step));
    lo += k * step;
  }
  return lo;
}

__device__ __forceinline__ void load4(const float* p, float (&x)[4], bool vec) {
  if (vec) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = p[i];
  }
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&x)[4], bool vec) {
  uint2 v;
  if (vec) {
    v = *reinterpret_cast<const uint2*>(p);
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    v = make_uint2(h[0] | uint32_t(h[1]) << 16, h[2] | uint32_t(h[3]) << 16);
  }
  x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
  x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
}

struct Write {
  uint8_t *k, *v;                        // the layer's pages
  float *ks, *vs;                        // and scales
  const void *new_k, *new_v;
  const int32_t *table, *refs, *slots, *starts, *cu;
  int32_t* status;
  int64_t k_token, k_head, v_token, v_head;
  int n, tokens, heads, slots_total, pages, width, page, d;
  bool vec;                              // rows can be read four elements at a time
};

// The rows of one block that one entry of the request writes.
struct Part {
  int t, rows, r0;                       // first packed row, their number, first row in the block
  int64_t block;                         // (page * heads) * blocks of a page + block in the page
};

// Blocks (c, y): the parts that begin in packed rows [16 c, 16 c + 16), 8 gridDim.y warps over their
// (part, K or V, head) triples.  A part begins with its entry, or on a block's first token.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(256) write_codes8_kernel(const Write w) {
  __shared__ Part s_part[kScaleBlock];
  __shared__ int s_found[kScaleBlock];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < kScaleBlock) s_found[threadIdx.x] = 0;
  griddep_launch_dependents();
  griddep_wait();
  __syncthreads();
  const int per_page = w.page / kScaleBlock;
  for (int x = warp; x < kScaleBlock; x += 8) {
    const int t = int(blockIdx.x) * kScaleBlock + x;
    if (t >= w.tokens) break;
    const int i = entry_of(w.cu, w.n, t);
    const int first = w.cu[i], end = min(w.cu[i + 1], w.tokens), slot = w.slots[i];
    const int64_t start = w.starts[i], pos = start + t - first;
    int fail = 0;
    if (t < first || t >= end || slot < 0 || slot >= w.slots_total || pos < 0 ||
        pos / w.page >= w.width)
      fail = ENIGMA_CACHE_BAD_REQUEST;
    const int r0 = int(pos % kScaleBlock);
    if (fail == 0 && t != max(first, 0) && r0 != 0) continue;            // in the middle of a part
    int at = -1;
    if (fail == 0) {
      at = w.table[int64_t(slot) * w.width + pos / w.page];
      if (at < 0 || at >= w.pages) fail = ENIGMA_CACHE_BAD_REQUEST;
      else if (w.refs[at] > 1) fail = ENIGMA_CACHE_SHARED;
    }
    if (fail == 0) {
      // Another entry of the same slot that touches this block would change it at the same time.
      const int64_t b0 = pos - r0, b1 = b0 + kScaleBlock;
      bool twice = false;
      for (int j = lane; j < w.n; j += 32)
        if (j != i && w.slots[j] == slot) {
          const int64_t s = w.starts[j], e = s + w.cu[j + 1] - int64_t(w.cu[j]);
          twice |= s < e && s < b1 && e > b0;
        }
      if (__any_sync(0xffffffffu, twice)) fail = ENIGMA_CACHE_BAD_REQUEST;
    }
    if (lane == 0) {
      if (fail != 0) {
        atomicOr(w.status, fail);
      } else {
        Part p;
        p.t = t;
        p.rows = min(kScaleBlock - r0, end - t);
        p.r0 = r0;
        p.block = int64_t(at) * w.heads * per_page + pos % w.page / kScaleBlock;
        s_part[x] = p;
        s_found[x] = 1;
      }
    }
  }
  __syncthreads();
  // The parts that there are, in the order of their rows: the same list in every block of a column.
  const uint32_t found = __ballot_sync(0xffffffffu, lane < kScaleBlock && s_found[lane % kScaleBlock]);
  const int quads = w.d / 4, step_r = 32 / quads, step_c = 32 % quads;
  const int units = __popc(found) * 2 * w.heads;
  for (int u = int(blockIdx.y) * 8 + warp; u < units; u += 8 * int(gridDim.y)) {
    const Part p = s_part[__fns(found, 0, u / (2 * w.heads) + 1)];
    const int rest = u % (2 * w.heads), head = rest >> 1;
    const bool is_v = rest & 1;
    const T* rows = is_v ? static_cast<const T*>(w.new_v) + p.t * w.v_token + head * w.v_head
                         : static_cast<const T*>(w.new_k) + p.t * w.k_token + head * w.k_head;
    const int64_t token = is_v ? w.v_token : w.k_token;
    const int64_t block = p.block + int64_t(head) * per_page;
    uint8_t* codes = (is_v ? w.v : w.k) + block * kScaleBlock * w.d;
    float* scale_at = (is_v ? w.vs : w.ks) + block;
    const float held = p.r0 > 0 ? *scale_at : 0.f;
    uint32_t top = 0;
    for (int r = lane / quads, c = lane % quads; r < p.rows;) {
      float x[4];
      load4(rows + r * token + 4 * c, x, w.vec);
#pragma unroll
      for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
      r += step_r;
      c += step_c;
      if (c >= quads) c -= quads, ++r;
    }
    top = __reduce_max_sync(0xffffffffu, top);
    const bool finite = top < 0x7f800000u && fabsf(held) < INFINITY;
    const float scale = finite ? fmaxf(held, scale_of<E4M3>(top)) : __uint_as_float(0x7fffffffu);
    const float inverse = finite ? 1.f / scale : 0.f;
    if (finite && held < scale) {                                        // (r0 = 0: there are none)
      for (int x = lane; x < p.r0 * quads; x += 32) {
        uint32_t* word = reinterpret_cast<uint32_t*>(codes) + x;
        const float2 lo = floats_of(halves_of<E4M3>(*word & 0xffffu));
        const float2 hi = floats_of(halves_of<E4M3>(*word >> 16));
        *word = codes_of<E4M3>(lo.x * held * inverse, lo.y * held * inverse, hi.x * held * inverse,
                               hi.y * held * inverse);
      }
    }
    for (int r = lane / quads, c = lane % quads; r < p.rows;) {
      float x[4];
      load4(rows + r * token + 4 * c, x, w.vec);
      *reinterpret_cast<uint32_t*>(codes + (p.r0 + r) * w.d + 4 * c) =
          finite ? codes_of<E4M3>(x[0] * inverse, x[1] * inverse, x[2] * inverse, x[3] * inverse) : 0u;
      r += step_r;
      c += step_c;
      if (c >= quads) c -= quads, ++r;
    }
    if (lane == 0) *scale_at = scale;
  }
}

struct Read {
  const uint8_t *k, *v;
  const float *ks, *vs;
  void *out_k, *out_v;
  const int32_t *table, *lens, *slots, *starts, *cu;
  int64_t k_token, k_head, v_token, v_head;
  int n, tokens, heads, slots_total, pages, width, page, d;
  bool vec;
};

__device__ __forceinline__ void store4(float* p, const float (&x)[4], bool vec) {
  if (vec) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = x[i];
  }
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float (&x)[4], bool vec) {
  if (vec) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = __float2bfloat16_rn(x[i]);
  }
}

// A warp per packed row; rows before the first entry and behind the last are left as they were, a
// token that the slot does not hold is zeros.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(256) read_codes8_kernel(const Read w) {
  const int lane = threadIdx.x & 31;
  const int quads = w.d / 4, row = w.heads * quads, per_page = w.page / kScaleBlock;
  griddep_launch_dependents();
  griddep_wait();
  for (int t = int(blockIdx.x) * 8 + (threadIdx.x >> 5); t < w.tokens; t += int(gridDim.x) * 8) {
    const int i = entry_of(w.cu, w.n, t);
    if (t < w.cu[i] || t >= w.cu[i + 1]) continue;
    const int slot = w.slots[i];
    const int64_t pos = int64_t(w.starts[i]) + t - w.cu[i];
    int at = -1;
    if (slot >= 0 && slot < w.slots_total && pos >= 0 && pos < w.lens[slot] &&
        pos / w.page < w.width)
      at = w.table[int64_t(slot) * w.width + pos / w.page];
    const bool has = at >= 0 && at < w.pages;
    for (int x = lane; x < 2 * row; x += 32) {
      const bool is_v = x >= row;
      const int y = is_v ? x - row : x, h = y / quads, c = y - h * quads;
      float f[4] = {0.f, 0.f, 0.f, 0.f};
      if (has) {
        const int64_t line = (int64_t(at) * w.heads + h) * w.page + pos % w.page;
        const uint32_t word = reinterpret_cast<const uint32_t*>((is_v ? w.v : w.k) + line * w.d)[c];
        const float s = (is_v ? w.vs : w.ks)[(int64_t(at) * w.heads + h) * per_page +
                                             pos % w.page / kScaleBlock];
        const float2 lo = floats_of(halves_of<E4M3>(word & 0xffffu));
        const float2 hi = floats_of(halves_of<E4M3>(word >> 16));
        f[0] = lo.x * s; f[1] = lo.y * s; f[2] = hi.x * s; f[3] = hi.y * s;
      }
      store4((is_v ? static_cast<T*>(w.out_v) + t * w.v_token + h * w.v_head
                   : static_cast<T*>(w.out_k) + t * w.k_token + h * w.k_head) + 4 * c, f, w.vec);
    }
  }
}

// Rows of four elements that can be moved at once.
bool vectors(int dtype, const void* k, const void* v, const int64_t* strides4) {
  const size_t es = dtype == ENIGMA_DTYPE_F32 ? 4 : 2;
  bool ok = aligned(k, 4 * es) && aligned(v, 4 * es);
  for (int i = 0; i < 4; ++i) ok = ok && strides4[i] % 4 == 0;
  return ok;
}

// The scales as pages of one row per head, which move with their codes.
enigma_kv_cache_desc scales_of(const enigma_kv_cache_q8_desc& d) {
  enigma_kv_cache_desc s = d.cache;
  s.k = d.k_scale;
  s.v = d.v_scale;
  s.head_dim = s.page / kScaleBlock;
  s.elem_bytes = 4;
  s.page = 1;
  return s;
}

}  // namespace

namespace enigma {

cudaError_t kv_cache_q8_fork(const enigma_kv_cache_q8_desc& d, const int32_t* parents,
                             const int32_t* children, int64_t n, cudaStream_t s) {
  const cudaError_t e = kv_cache_fork(d.cache, parents, children, n, s);
  return e == cudaSuccess ? kv_cache_copy_listed(scales_of(d), n, s) : e;
}

cudaError_t kv_cache_q8_compact(const enigma_kv_cache_q8_desc& d, cudaStream_t s) {
  const cudaError_t e = kv_cache_compact(d.cache, s);
  return e == cudaSuccess ? kv_cache_copy_listed(scales_of(d), d.cache.pages / 2, s) : e;
}

cudaError_t kv_cache_q8_copy_pages(const enigma_kv_cache_q8_desc& d, const int32_t* src,
                                   const int32_t* dst, int64_t n, cudaStream_t s) {
  const cudaError_t e = kv_cache_copy_pages(d.cache, src, dst, n, s);
  return e == cudaSuccess ? kv_cache_copy_pages(scales_of(d), src, dst, n, s) : e;
}

cudaError_t kv_cache_q8_write(const enigma_kv_cache_q8_desc& d, int64_t layer, int dtype,
                              const void* new_k, const void* new_v, const int64_t* strides4,
                              const int32_t* slots, const int32_t* starts, const int32_t* cu,
                              int64_t n, int64_t tokens, cudaStream_t s) {
  note_kernel("write_codes8_kernel");
  const enigma_kv_cache_desc& c = d.cache;
  const int64_t blocks = c.pages * c.heads_kv * (c.page / kScaleBlock);       // of a layer
  Write w;
  w.k = static_cast<uint8_t*>(c.k) + layer * blocks * kScaleBlock * c.head_dim;
  w.v = static_cast<uint8_t*>(c.v) + layer * blocks * kScaleBlock * c.head_dim;
  w.ks = d.k_scale + layer * blocks;
  w.vs = d.v_scale + layer * blocks;
  w.new_k = new_k;
  w.new_v = new_v;
  w.table = c.table;
  w.refs = c.refs;
  w.slots = slots;
  w.starts = starts;
  w.cu = cu;
  w.status = c.status;
  w.k_token = strides4[0];
  w.k_head = strides4[1];
  w.v_token = strides4[2];
  w.v_head = strides4[3];
  w.n = int(n);
  w.tokens = int(tokens);
  w.heads = int(c.heads_kv);
  w.slots_total = int(c.slots);
  w.pages = int(c.pages);
  w.width = int(c.table_width);
  w.page = int(c.page);
  w.d = int(c.head_dim);
  w.vec = vectors(dtype, new_k, new_v, strides4);
  const dim3 grid(unsigned((tokens + kScaleBlock - 1) / kScaleBlock), 4);
  const bool f32 = dtype == ENIGMA_DTYPE_F32, e4m3 = d.code == ENIGMA_CODE_E4M3;
  if (f32 && e4m3) return launch_dependent(write_codes8_kernel<float, true>, grid, 256, 0, s, w);
  if (f32) return launch_dependent(write_codes8_kernel<float, false>, grid, 256, 0, s, w);
  if (e4m3) return launch_dependent(write_codes8_kernel<__nv_bfloat16, true>, grid, 256, 0, s, w);
  return launch_dependent(write_codes8_kernel<__nv_bfloat16, false>, grid, 256, 0, s, w);
}

cudaError_t kv_cache_q8_read(const enigma_kv_cache_q8_desc& d, int64_t layer, int dtype, void* out_k,
                             void* out_v, const int64_t* strides4, const int32_t* slots,
                             const int32_t* starts, const int32_t* cu, int64_t n, int64_t tokens,
                             cudaStream_t s) {
  note_kernel("read_codes8_kernel");
  const enigma_kv_cache_desc& c = d.cache;
  const int64_t blocks = c.pages * c.heads_kv * (c.page / kScaleBlock);
  Read w;
  w.k = static_cast<const uint8_t*>(c.k) + layer * blocks * kScaleBlock * c.head_dim;
  w.v = static_cast<const uint8_t*>(c.v) + layer * blocks * kScaleBlock * c.head_dim;
  w.ks = d.k_scale + layer * blocks;
  w.vs = d.v_scale + layer * blocks;
  w.out_k = out_k;
  w.out_v = out_v;
  w.table = c.table;
  w.lens = c.lens;
  w.slots = slots;
  w.starts = starts;
  w.cu = cu;
  w.k_token = strides4[0];
  w.k_head = strides4[1];
  w.v_token = strides4[2];
  w.v_head = strides4[3];
  w.n = int(n);
  w.tokens = int(tokens);
  w.heads = int(c.heads_kv);
  w.slots_total = int(c.slots);
  w.pages = int(c.pages);
  w.width = int(c.table_width);
  w.page = int(c.page);
  w.d = int(c.head_dim);
  w.vec = vectors(dtype, out_k, out_v, strides4);
  const unsigned grid = unsigned(std::min<int64_t>((tokens + 7) / 8, int64_t(sm_count()) * 32));
  const bool f32 = dtype == ENIGMA_DTYPE_F32, e4m3 = d.code == ENIGMA_CODE_E4M3;
  if (f32 && e4m3) return launch_dependent(read_codes8_kernel<float, true>, grid, 256, 0, s, w);
  if (f32) return launch_dependent(read_codes8_kernel<float, false>, grid, 256, 0, s, w);
  if (e4m3) return launch_dependent(read_codes8_kernel<__nv_bfloat16, true>, grid, 256, 0, s, w);
  return launch_dependent(read_codes8_kernel<__nv_bfloat16, false>, grid, 256, 0, s, w);
}

}  // namespace enigma
