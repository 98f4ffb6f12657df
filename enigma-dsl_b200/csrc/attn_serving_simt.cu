// attn_serving_simt.cu — packed and paged attention on CUDA cores: any head_dim <= 256, fp32 or
// bf16 storage, any strides and alignment.  The tensor-core kernels (attn_packed.cu,
// attn_paged.cu) take the bf16 shapes they can; these take the rest.
#include <algorithm>

#include "attn_serving.cuh"

namespace {

using enigma_serving::PackedGroup;
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

// ============================================================================ packed
// A CTA takes 64 rows (token, head) of an item against its keys, 64 at a time.  128 threads, each
// with 8 rows x 4 keys of S and 8 rows x DP / 16 columns of O, rows in pairs for the packed fp32
// FMA.  Q, K and P lie transposed in shared memory, so a step of either product reads 8 rows
// with two and 4 keys or columns with one 16-byte load for 32 multiply-adds.  Bound by the
// FMA pipe and, next to it, by shared memory.
constexpr int TR = 64, TK = 64, TT = 128;

template <int DP>
struct TileCfg {
  static constexpr int QT = DP * TR, KT = DP * (TK + 4), VT = TK * DP, PT = TK * TR;   // floats
  static constexpr int SMEM = (QT + (KT > PT ? KT : PT) + VT) * 4;
  static constexpr int CPT = DP / 16;                     // columns of O per thread
};

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u),
                     __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
}

// Elements d .. d + 3 of a row, zero past D.
template <typename T>
__device__ __forceinline__ float4 row4(const T* p, int d, int D, bool vec) {
  if (vec && d + 4 <= D) return load4(p + d);
  return make_float4(d < D ? load(p + d) : 0.f, d + 1 < D ? load(p + d + 1) : 0.f,
                     d + 2 < D ? load(p + d + 2) : 0.f, d + 3 < D ? load(p + d + 3) : 0.f);
}

template <typename T, int DP>
__global__ void __launch_bounds__(TT)
packed_simt_kernel(const enigma_sdpa_packed_desc p, const bool vec) {
  using C = TileCfg<DP>;
  extern __shared__ float4 smem4[];
  float* s_q = reinterpret_cast<float*>(smem4);           // [DP][TR]
  float* s_k = s_q + C::QT;                               // [DP][TK + 4]; then P [TK][TR]
  float* s_v = s_k + (C::KT > C::PT ? C::KT : C::PT);     // [TK][DP]
  const int tid = threadIdx.x;
  const PackedItem it = reinterpret_cast<const PackedItem*>(
      p.plan + p.header[enigma_serving::kItemsAt])[blockIdx.x];
  const int G = int(p.heads_q / p.heads_kv), D = int(p.head_dim), kvh = it.kvh;
  // An item that does not lie inside the tensors is no work of theirs.
  if (it.q0 < 0 || it.q0 + int64_t(it.lq) > p.tokens_q || it.k0 < 0 ||
      it.k0 + int64_t(it.lk) > p.tokens_k || it.t0 < 0 || kvh < 0 || kvh >= p.heads_kv ||
      it.slot >= p.header[enigma_serving::kSlots])
    return;
  const int n = min((it.alt ? 1 : 2) * it.tokens, it.lq - it.t0) * G;   // rows of the item
  const int r0 = blockIdx.y * TR;
  if (r0 >= n) return;
  const int off = p.causal ? it.lk - it.lq + 1 : it.lk;   // a token's keys: min(lk, token + off)
  const int t_last = it.t0 + (min(r0 + TR, n) - 1) / G;
  const int k_end = min(min(it.lk, t_last + off), it.j1 * 128);
  const T* kb = static_cast<const T*>(p.k) + it.k0 * p.k_token + kvh * p.k_head;
  const T* vb = static_cast<const T*>(p.v) + it.k0 * p.v_token + kvh * p.v_head;
  for (int x = tid; x < TR * (DP / 4); x += TT) {
    const int r = x % TR, d = x / TR * 4, row = r0 + r;
    float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < n)
      q = row4(static_cast<const T*>(p.q) + (int64_t(it.q0) + it.t0 + row / G) * p.q_token +
                   (kvh * G + row % G) * p.q_head, d, D, vec);
    s_q[d * TR + r] = q.x;
    s_q[(d + 1) * TR + r] = q.y;
    s_q[(d + 2) * TR + r] = q.z;
    s_q[(d + 3) * TR + r] = q.w;
  }
  const int rg = tid / 16, cg = tid % 16;                 // rows rg * 8 .., keys / columns cg * 4 ..
  int keys[8];                                            // keys each row sees
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int row = r0 + rg * 8 + r;
    keys[r] = row < n ? min(it.lk, it.t0 + row / G + off) : 0;
  }
  float2 o[4][C::CPT];
  float m[8], l[8];                                       // l: this thread's keys only
#pragma unroll
  for (int r = 0; r < 8; ++r) m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < C::CPT; ++c) o[r][c] = make_float2(0.f, 0.f);
  const float c_log2 = p.scale * 1.4426950408889634f;
  for (int k0 = it.j0 * 128; k0 < k_end; k0 += TK) {
    __syncthreads();
    // Keys past the end are zeros in K and V; their weights are zero too.
    for (int x = tid; x < TK * (DP / 4); x += TT) {
      const int key = x % TK, d = x / TK * 4;
      float4 k = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k0 + key < it.lk) k = row4(kb + (k0 + key) * p.k_token, d, D, vec);
      s_k[d * (TK + 4) + key] = k.x;
      s_k[(d + 1) * (TK + 4) + key] = k.y;
      s_k[(d + 2) * (TK + 4) + key] = k.z;
      s_k[(d + 3) * (TK + 4) + key] = k.w;
    }
    for (int x = tid; x < TK * (DP / 4); x += TT) {
      const int key = x / (DP / 4), d = x % (DP / 4) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k0 + key < it.lk) v = row4(vb + (k0 + key) * p.v_token, d, D, vec);
      *reinterpret_cast<float4*>(s_v + key * DP + d) = v;
    }
    __syncthreads();
    float2 s[4][4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[r][c] = make_float2(0.f, 0.f);
#pragma unroll 8
    for (int d = 0; d < DP; ++d) {
      const float4 qa = *reinterpret_cast<const float4*>(s_q + d * TR + rg * 8);
      const float4 qb = *reinterpret_cast<const float4*>(s_q + d * TR + rg * 8 + 4);
      const float4 k = *reinterpret_cast<const float4*>(s_k + d * (TK + 4) + cg * 4);
      const float2 q[4] = {{qa.x, qa.y}, {qa.z, qa.w}, {qb.x, qb.y}, {qb.z, qb.w}};
      const float kk[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r][c] = fma2(q[r], make_float2(kk[c], kk[c]), s[r][c]);
    }
    __syncthreads();                                      // K is read: P takes its place
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      float v[4];
      float mx = m[r];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        v[c] = (r & 1) ? s[r / 2][c].y : s[r / 2][c].x;
        if (k0 + cg * 4 + c >= keys[r]) v[c] = -INFINITY;
        mx = fmaxf(mx, v[c]);
      }
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float base = mx == -INFINITY ? 0.f : mx * c_log2;
      const float f = exp2f(m[r] * c_log2 - base);        // m = -inf: 0
      m[r] = mx;
      l[r] *= f;
#pragma unroll
      for (int c = 0; c < C::CPT; ++c) {
        if (r & 1) o[r / 2][c].y *= f;
        else o[r / 2][c].x *= f;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float e = exp2f(fmaf(v[c], c_log2, -base));
        l[r] += e;
        if (r & 1) s[r / 2][c].y = e;
        else s[r / 2][c].x = e;
      }
    }
    // Four rows at once; their place in a key's row is turned by the key's group, so that the 8
    // lanes of one store phase meet all banks.
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float4*>(s_k + (cg * 4 + c) * TR + (((rg * 2 + h) ^ (cg & 7)) * 4)) =
            make_float4(s[2 * h][c].x, s[2 * h][c].y, s[2 * h + 1][c].x, s[2 * h + 1][c].y);
    __syncthreads();
#pragma unroll 4
    for (int j = 0; j < TK; ++j) {
      const int turn = j >> 2 & 7;
      const float4 pa = *reinterpret_cast<const float4*>(s_k + j * TR + ((rg * 2) ^ turn) * 4);
      const float4 pb = *reinterpret_cast<const float4*>(s_k + j * TR + ((rg * 2 + 1) ^ turn) * 4);
      const float2 w[4] = {{pa.x, pa.y}, {pa.z, pa.w}, {pb.x, pb.y}, {pb.z, pb.w}};
#pragma unroll
      for (int c4 = 0; c4 < C::CPT; c4 += 4) {
        const float4 v = *reinterpret_cast<const float4*>(s_v + j * DP + c4 * 16 + cg * 4);
        const float vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            o[r][c4 + c] = fma2(w[r], make_float2(vv[c], vv[c]), o[r][c4 + c]);
      }
    }
  }
  float* opart = static_cast<float*>(p.workspace);
  float2* ml = reinterpret_cast<float2*>(opart + int64_t(p.header[enigma_serving::kSlots]) * 128 * D);
#pragma unroll
  for (int r = 0; r < 8; ++r) {
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
    const int row = r0 + rg * 8 + r;
    if (row >= n) continue;
    const int64_t tok = int64_t(it.q0) + it.t0 + row / G;
    const int h = kvh * G + row % G;
    const bool final = it.slot < 0;
    const float inv = !final ? 1.f : l[r] == 0.f ? 0.f : 1.f / l[r];   // no keys: zeros
    // Partial results: rows of the item's second tile go to the next slot, as do an alt item's
    // odd key tiles, which this kernel does not treat apart (that state is empty).
    const int tile = row / (it.tokens * G), in_tile = row - tile * it.tokens * G;
    const int64_t at = (int64_t(it.slot) + tile) * 128 + in_tile;
    T* out = static_cast<T*>(p.out) + tok * p.o_token + h * p.o_head;
#pragma unroll
    for (int c = 0; c < C::CPT; ++c) {
      const int d = c / 4 * 64 + cg * 4 + c % 4;
      const float v = ((r & 1) ? o[r / 2][c].y : o[r / 2][c].x) * inv;
      if (d < D) {
        if (final) store(out + d, v);
        else opart[at * D + d] = v;
      }
    }
    if (cg == 0) {
      if (!final) {
        ml[at] = make_float2(m[r] * c_log2, l[r]);
        if (it.alt) ml[at + 128] = make_float2(-INFINITY, 0.f);
      } else if (p.lse != nullptr) {
        p.lse[tok * p.heads_q + h] = (m[r] * c_log2 + log2f(l[r])) * 0.6931471805599453f;
      }
    }
  }
}

// Joins the partial results of split rows.  One warp per row; grid (groups, rows / 8).
template <typename T, int V>
__global__ void __launch_bounds__(256)
packed_join_kernel(const enigma_sdpa_packed_desc p) {
  const int lane = threadIdx.x & 31, D = int(p.head_dim), G = int(p.heads_q / p.heads_kv);
  const int r = int(blockIdx.y) * 8 + (threadIdx.x >> 5);       // row of the pair of tiles
  const PackedGroup g = reinterpret_cast<const PackedGroup*>(
      p.plan + p.header[enigma_serving::kGroupsAt])[blockIdx.x];
  const float* opart = static_cast<const float*>(p.workspace);
  const float2* ml =
      reinterpret_cast<const float2*>(opart + int64_t(p.header[enigma_serving::kSlots]) * 128 * D);
  const int state = r / 128, row = r % 128;
  const int tok = g.tok0 + state * g.tokens + row / G;
  if (row >= g.tokens * G || tok >= g.tok_end || tok >= p.tokens_q || (g.alt && state > 0)) return;
  const int n = g.alt ? 2 * g.parts : g.parts, step = (g.alt ? 1 : 2) * 128;
  const int64_t at = int64_t(g.slot + (g.alt ? 0 : state)) * 128 + row;
  enigma_serving::RowJoin<V> join;
  join.best(ml + at, step, n, lane);
  join.seal();
  join.add(ml + at, step, opart + at * D, int64_t(step) * D, n, D, lane);
  const int h = g.kvh * G + row % G;
  const float inv = join.l == 0.f ? 0.f : 1.f / join.l;
  T* out = static_cast<T*>(p.out) + tok * p.o_token + h * p.o_head;
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (lane + 32 * v < D) store(out + lane + 32 * v, join.acc[v] * inv);
  if (p.lse != nullptr && lane == 0)
    p.lse[int64_t(tok) * p.heads_q + h] =
        join.l == 0.f ? -INFINITY : (join.M + log2f(join.l)) * 0.6931471805599453f;
}

template <typename T>
void launch_join(const enigma_sdpa_packed_desc& d, const dim3 grid, cudaStream_t s) {
  if (d.head_dim <= 64) packed_join_kernel<T, 2><<<grid, 256, 0, s>>>(d);
  else if (d.head_dim <= 128) packed_join_kernel<T, 4><<<grid, 256, 0, s>>>(d);
  else packed_join_kernel<T, 8><<<grid, 256, 0, s>>>(d);
}

template <typename T, int DP>
cudaError_t launch_packed(const enigma_sdpa_packed_desc& d, cudaStream_t s) {
  using C = TileCfg<DP>;
  const cudaError_t e = cudaFuncSetAttribute(
      packed_simt_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  // Four elements at a time where every row starts on their boundary.
  const int64_t size = 4 * int64_t(sizeof(T));
  bool vec = true;
  for (const void* b : {d.q, d.k, d.v}) vec &= reinterpret_cast<uintptr_t>(b) % uintptr_t(size) == 0;
  for (const int64_t x : {d.q_token, d.q_head, d.k_token, d.k_head, d.v_token, d.v_head})
    vec &= x % 4 == 0;
  const int64_t group = d.heads_q / d.heads_kv;
  const int64_t rows = 2 * std::max<int64_t>(1, ENIGMA_PACKED_TILE_ROWS / group) * group;
  const dim3 grid(unsigned(d.header[enigma_serving::kItems]), unsigned((rows + TR - 1) / TR));
  packed_simt_kernel<T, DP><<<grid, TT, C::SMEM, s>>>(d, vec);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_packed(const enigma_sdpa_packed_desc& d, cudaStream_t s) {
  if (d.head_dim <= 64) return launch_packed<T, 64>(d, s);
  if (d.head_dim <= 128) return launch_packed<T, 128>(d, s);
  return launch_packed<T, 256>(d, s);
}

// ============================================================================ paged
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
  return d.dtype == ENIGMA_DTYPE_F32 ? launch_packed<float>(d, s)
                                     : launch_packed<__nv_bfloat16>(d, s);
}

cudaError_t sdpa_packed_join_launch(const enigma_sdpa_packed_desc& d, cudaStream_t s) {
  const int groups = d.header[enigma_serving::kGroups];
  if (groups == 0) return cudaSuccess;
  const dim3 grid(unsigned(groups), 2 * ENIGMA_PACKED_TILE_ROWS / 8);
  if (d.dtype == ENIGMA_DTYPE_F32) launch_join<float>(d, grid, s);
  else launch_join<__nv_bfloat16>(d, grid, s);
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
