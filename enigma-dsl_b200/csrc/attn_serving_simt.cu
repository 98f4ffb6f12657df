// attn_serving_simt.cu — packed and paged attention on CUDA cores: any head_dim <= 256, fp32 or
// bf16 storage, any strides and alignment.  The tensor-core kernels (attn_packed.cu,
// attn_paged.cu) take the bf16 shapes they can; these take the rest.
#include <algorithm>

#include "attn_serving.cuh"

namespace {

using enigma_serving::PackedItem;

__device__ __forceinline__ float load(const float* p) { return *p; }
__device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store(float* p, float v) { *p = v; }
__device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

constexpr int kMaxDPerLane = 8;        // head_dim <= 256
constexpr int kWarps = 8;

// Running softmax of one row held by a warp: lane holds elements lane, lane + 32, ... of the
// head; m is the running maximum, l the sum of e^(s - m), acc the weighted sum of V rows, all
// fp32.  Only keys the row sees are visited, so nothing behind a mask can reach it.
template <typename T>
struct Row {
  float q[kMaxDPerLane], acc[kMaxDPerLane];
  float m = -INFINITY, l = 0.f;
  __device__ void start(const T* p, int D, int lane, float scale) {
#pragma unroll
    for (int t = 0; t < kMaxDPerLane; ++t) {
      const int d = lane + 32 * t;
      q[t] = d < D ? load(p + d) * scale : 0.f;
      acc[t] = 0.f;
    }
  }
  __device__ void key(const T* k, const T* v, int D, int lane) {
    float s = 0.f;
#pragma unroll
    for (int t = 0; t < kMaxDPerLane; ++t) {
      const int d = lane + 32 * t;
      if (d < D) s = fmaf(q[t], load(k + d), s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float m_new = fmaxf(m, s);
    // A first key whose score is -inf keeps the empty state (no (-inf) - (-inf)).
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float corr = expf(m - base), p = expf(s - base);
    l = l * corr + p;
#pragma unroll
    for (int t = 0; t < kMaxDPerLane; ++t) {
      const int d = lane + 32 * t;
      if (d < D) acc[t] = fmaf(acc[t], corr, p * load(v + d));
    }
    m = m_new;
  }
};

// One warp per row of an item: rows (token, head) of both tiles, grid (items, parts).  Items that
// split a row's keys were made for the tensor-core kernel: the first of them does all here.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
packed_simt_kernel(const enigma_sdpa_packed_desc p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const PackedItem it = reinterpret_cast<const PackedItem*>(
      p.plan + p.header[enigma_serving::kItemsAt])[blockIdx.x];
  const int G = int(p.heads_q / p.heads_kv), D = int(p.head_dim), kvh = it.kvh;
  // An item that does not lie inside the tensors is no work of theirs.
  if (it.q0 < 0 || it.q0 + int64_t(it.lq) > p.tokens_q || it.k0 < 0 ||
      it.k0 + int64_t(it.lk) > p.tokens_k || it.t0 < 0 || kvh < 0 ||
      kvh >= p.heads_kv || it.j0 > 0)
    return;
  const int n = min((it.alt ? 1 : 2) * it.tokens, it.lq - it.t0) * G;
  const T* kb = static_cast<const T*>(p.k) + it.k0 * p.k_token + kvh * p.k_head;
  const T* vb = static_cast<const T*>(p.v) + it.k0 * p.v_token + kvh * p.v_head;
  for (int r = blockIdx.y * kWarps + warp; r < n; r += gridDim.y * kWarps) {
    const int t = it.t0 + r / G, h = kvh * G + r % G;
    const int64_t tok = int64_t(it.q0) + t;
    Row<T> row;
    row.start(static_cast<const T*>(p.q) + tok * p.q_token + h * p.q_head, D, lane, p.scale);
    const int last = p.causal ? min(it.lk - 1, t + it.lk - it.lq) : it.lk - 1;
    for (int64_t j = 0; j <= last; ++j) row.key(kb + j * p.k_token, vb + j * p.v_token, D, lane);
    const float inv = row.l == 0.f ? 0.f : 1.f / row.l;     // a row without keys gives zeros
    T* o = static_cast<T*>(p.out) + tok * p.o_token + h * p.o_head;
#pragma unroll
    for (int x = 0; x < kMaxDPerLane; ++x) {
      const int d = lane + 32 * x;
      if (d < D) store(o + d, row.acc[x] * inv);
    }
    if (p.lse != nullptr && lane == 0)
      p.lse[tok * p.heads_q + h] = row.m + logf(row.l);
  }
}

// One CTA per (sequence, query head); its warps take every kWarps-th key and merge at the end.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
paged_simt_kernel(const enigma_sdpa_shared_prefix_desc p) {
  __shared__ float s_m[kWarps], s_l[kWarps], s_acc[kWarps][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.x, D = int(p.head_dim);
  const int64_t b = blockIdx.y;
  const int kvh = h / int(p.heads_q / p.heads_kv);
  const int64_t slot = p.slots != nullptr ? p.slots[b] : b;
  const int64_t slot0 = p.slots != nullptr ? p.slots[0] : 0;
  const bool there = slot >= 0 && slot < p.n_slots && slot0 >= 0 && slot0 < p.n_slots;
  const int64_t len = there ? min(int64_t(max(p.lens[slot], 0)), p.table_width * p.page) : 0;
  Row<T> row;
  row.start(static_cast<const T*>(p.q) + b * p.q_batch + h * p.q_head, D, lane, p.scale);
  for (int64_t j = warp; j < len; j += kWarps) {
    const int64_t s = j < p.prefix_len ? slot0 : slot;
    const int at = p.table[s * p.table_width + j / p.page];
    if (at < 0 || at >= p.pages) continue;                  // not a page: no key
    const int64_t off = (kvh * p.page + j % p.page) * D;
    row.key(static_cast<const T*>(p.k_pages) + at * p.k_page + off,
            static_cast<const T*>(p.v_pages) + at * p.v_page + off, D, lane);
  }
#pragma unroll
  for (int x = 0; x < kMaxDPerLane; ++x) s_acc[warp][lane + 32 * x] = row.acc[x];
  if (lane == 0) {
    s_m[warp] = row.m;
    s_l[warp] = row.l;
  }
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w]);
  for (int w = 0; w < kWarps; ++w) L += s_m[w] == -INFINITY ? 0.f : s_l[w] * expf(s_m[w] - M);
  for (int d = threadIdx.x; d < D; d += kWarps * 32) {
    float o = 0.f;
    for (int w = 0; w < kWarps; ++w)
      if (s_m[w] != -INFINITY) o = fmaf(s_acc[w][d], expf(s_m[w] - M), o);
    store(static_cast<T*>(p.out) + b * p.o_batch + h * p.o_head + d, L == 0.f ? 0.f : o / L);
  }
}

}  // namespace

namespace enigma {

cudaError_t sdpa_packed_simt_launch(const enigma_sdpa_packed_desc& d, cudaStream_t s) {
  note_kernel("packed_simt_kernel");
  const dim3 grid(unsigned(d.header[enigma_serving::kItems]), 8);
  if (d.dtype == ENIGMA_DTYPE_F32) packed_simt_kernel<float><<<grid, kWarps * 32, 0, s>>>(d);
  else packed_simt_kernel<__nv_bfloat16><<<grid, kWarps * 32, 0, s>>>(d);
  return cudaGetLastError();
}

cudaError_t sdpa_paged_simt_launch(const enigma_sdpa_shared_prefix_desc& d, cudaStream_t s) {
  note_kernel("paged_simt_kernel");
  const dim3 grid(unsigned(d.heads_q), unsigned(d.batch));
  if (d.dtype == ENIGMA_DTYPE_F32) paged_simt_kernel<float><<<grid, kWarps * 32, 0, s>>>(d);
  else paged_simt_kernel<__nv_bfloat16><<<grid, kWarps * 32, 0, s>>>(d);
  return cudaGetLastError();
}

}  // namespace enigma
