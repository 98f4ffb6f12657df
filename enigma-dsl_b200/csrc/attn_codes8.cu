// attn_codes8.cu — one new token per sequence over a paged cache held in 8-bit codes with a scale for
// each 16 tokens of a page and head (codes8.cuh):
//   out = sum_j softmax_j(c s_k(j) q . k_j) s_v(j) v_j  over the sequence's first len keys.
#include <cfloat>

#include "attn_serving.cuh"
#include "codes8.cuh"

namespace {

using namespace enigma_codes8;

struct Attend {
  const void* q;
  void* out;
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int32_t *table, *lens, *slots;
  int64_t q_batch, q_head, o_batch, o_head, k_page, v_page, ks_page, vs_page;
  int heads_q, group, d, page, pages, width, n_slots;
  float scale;
};

__device__ __forceinline__ float at(const float* p) { return *p; }
__device__ __forceinline__ float at(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

template <bool E4M3>
__device__ __forceinline__ float value_of(uint8_t code) {
  return floats_of(halves_of<E4M3>(code)).x;
}

// A block per (query head, sequence), its four warps on every fourth key; lane l has elements
// l, l + 32, ... of the head.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(128) attend_codes8_kernel(const Attend a) {
  __shared__ float s_m[4], s_l[4], s_o[4][256];
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kvh = h / a.group, parts = a.page / kScaleBlock;
  const int slot = a.slots ? a.slots[b] : b;
  const bool there = slot >= 0 && slot < a.n_slots;
  const int64_t most = int64_t(a.width) * a.page;
  const int len = there ? int(min(int64_t(max(a.lens[slot], 0)), most)) : 0;
  const T* q = static_cast<const T*>(a.q) + b * a.q_batch + h * a.q_head;
  float qv[8], o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int x = lane + 32 * i;
    qv[i] = x < a.d ? at(q + x) : 0.f;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int j = warp; j < len; j += 4) {
    const int p = a.table[int64_t(slot) * a.width + j / a.page], r = j % a.page;
    const bool has = p >= 0 && p < a.pages;              // a key without a page is zeros
    const int64_t row = (int64_t(kvh) * a.page + r) * a.d;
    const int block = kvh * parts + r / kScaleBlock;
    float s = 0.f;
    if (has) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int x = lane + 32 * i;
        if (x < a.d) s += qv[i] * value_of<E4M3>(a.k[p * a.k_page + row + x]);
      }
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
      s *= a.ks[p * a.ks_page + block] * a.scale;
    }
    const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;
    const float shrink = expf(m - base), w = expf(s - base);
    m = top;
    l = l * shrink + w;
    const float sv = has ? a.vs[p * a.vs_page + block] * w : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int x = lane + 32 * i;
      o[i] *= shrink;
      if (has && x < a.d) o[i] += sv * value_of<E4M3>(a.v[p * a.v_page + row + x]);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) s_o[warp][lane + 32 * i] = o[i];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  const float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f, w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = expf(s_m[i] - base);
    sum += w[i] * s_l[i];
  }
  T* out = static_cast<T*>(a.out) + b * a.o_batch + h * a.o_head;
  for (int x = threadIdx.x; x < a.d; x += 128) {
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) y += w[i] * s_o[i][x];
    put(out + x, sum == 0.f ? 0.f : y / sum);
  }
}

}  // namespace

namespace enigma {

size_t sdpa_quantized_workspace(const enigma_sdpa_quantized_desc&) { return 0; }

cudaError_t sdpa_quantized_launch(const enigma_sdpa_quantized_desc& d, cudaStream_t s) {
  note_kernel("attend_codes8_kernel");
  Attend a;
  a.q = d.q;
  a.out = d.out;
  a.k = static_cast<const uint8_t*>(d.k_pages);
  a.v = static_cast<const uint8_t*>(d.v_pages);
  a.ks = d.k_scale;
  a.vs = d.v_scale;
  a.table = d.table;
  a.lens = d.lens;
  a.slots = d.slots;
  a.q_batch = d.q_batch;
  a.q_head = d.q_head;
  a.o_batch = d.o_batch;
  a.o_head = d.o_head;
  a.k_page = d.k_page;
  a.v_page = d.v_page;
  a.ks_page = d.ks_page;
  a.vs_page = d.vs_page;
  a.heads_q = int(d.heads_q);
  a.group = int(d.heads_q / d.heads_kv);
  a.d = int(d.head_dim);
  a.page = int(d.page);
  a.pages = int(d.pages);
  a.width = int(d.table_width);
  a.n_slots = int(d.n_slots);
  a.scale = d.scale;
  const dim3 grid(unsigned(d.heads_q), unsigned(d.batch));
  const bool f32 = d.dtype == ENIGMA_DTYPE_F32, e4m3 = d.code == ENIGMA_CODE_E4M3;
  if (f32 && e4m3) attend_codes8_kernel<float, true><<<grid, 128, 0, s>>>(a);
  else if (f32) attend_codes8_kernel<float, false><<<grid, 128, 0, s>>>(a);
  else if (e4m3) attend_codes8_kernel<__nv_bfloat16, true><<<grid, 128, 0, s>>>(a);
  else attend_codes8_kernel<__nv_bfloat16, false><<<grid, 128, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace enigma
