// attn_serving_simt.cu — packed and paged attention on CUDA cores: any head_dim <= 256, fp32 or
// bf16 storage, any strides and alignment.  The tensor-core kernels (attn_packed.cu,
// attn_paged.cu) take the bf16 shapes they can; these take the rest.
#include <algorithm>

#include "attn_serving.cuh"

namespace {

using enigma_sm100::cluster_ctarank;
using enigma_sm100::cluster_sync;
using enigma_sm100::griddep_launch_dependents;
using enigma_sm100::griddep_wait;
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
  // n keys of zeros with values of zeros: their score is 0 (NaN where q is not finite, as q . 0).
  __device__ void zero_keys(int n) {
    float s = 0.f;
#pragma unroll
    for (int t = 0; t < kMaxDPerLane; ++t) s = fmaf(q[t], 0.f, s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float m_new = fmaxf(m, s), corr = expf(m - m_new);
    l = l * corr + float(n) * expf(s - m_new);
#pragma unroll
    for (int t = 0; t < kMaxDPerLane; ++t) acc[t] *= corr;
    m = m_new;
  }
};

// ============================================================================ packed
// A CTA takes 64 rows (token, head) of an item against its keys, TK at a time.  128 threads, each
// with 8 rows x TK / 16 keys of S and 8 rows x DP / 16 columns of O.  Products run on the packed
// fp32 FMA: S over pairs of the head dimension, so that neither operand has to be doubled, O over
// pairs of rows.  K of the next tile is fetched while the softmax and P V run, V while S does.
// What comes out of shared memory holds the products up: a warp's 16-byte load is 512 bytes through
// the SM's 128-byte port, even where lanes read the same, so S takes 12 loads = 48 cycles of it per
// warp for 64 FMAs = 140 cycles of one of four FMA pipes (192 against 140 for the four), O the same.
// 1772 tokens in 4 prompts, 14 / 2 heads of 64, causal: 126 us; 4096, 8 / 8: 547 us = 31 TFLOP/s, 2.4
// times what the FMAs need, of which the port explains 1.37; the rest (two barriers and a softmax
// between the products of a tile, 8 warps on an SM) is not taken apart.  Tiles of 8 x 8 per thread
// load less, but registers leave too few warps: 10 to 20 % more time.
constexpr int TR = 64, TT = 128;

template <int DP>
struct TileCfg {
  static constexpr int TK = DP <= 64 ? 64 : 32;           // keys per tile
  static constexpr int LD = DP + 4;                       // row of Q or K: 8 lanes meet all banks
  static constexpr int SMEM = (TR * LD + TK * LD + TK * DP + TK * TR) * 4;
  static constexpr int KPT = TK / 16, CPT = DP / 16;      // keys, columns of O per thread
  static constexpr int CTAS = DP <= 128 ? 2 : 1;   // per SM, by shared memory
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

// Four elements of a row to shared memory; fp32 rows of aligned tensors by an asynchronous copy
// (zeros where there is no row), waited for by rows_landed.
__device__ __forceinline__ void put4(float* dst, const float* p, int d, int D, bool vec, bool there) {
  if (vec && (d + 4 <= D || !there)) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                 ::"r"(enigma_sm100::smem_u32(dst)), "l"(there ? p + d : p), "r"(there ? 16 : 0)
                 : "memory");
  } else {
    *reinterpret_cast<float4*>(dst) = there ? row4(p, d, D, vec) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
}
__device__ __forceinline__ void put4(float* dst, const __nv_bfloat16* p, int d, int D, bool vec,
                                     bool there) {
  *reinterpret_cast<float4*>(dst) = there ? row4(p, d, D, vec) : make_float4(0.f, 0.f, 0.f, 0.f);
}
__device__ __forceinline__ void rows_landed() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// What CTA `rank` of the cluster has at this place of its shared memory.
__device__ __forceinline__ float2 peer2(const float2* p, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
               : "=f"(v.x), "=f"(v.y)
               : "r"(enigma_sm100::mapa_shared(enigma_sm100::smem_u32(p), uint32_t(rank)))
               : "memory");
  return v;
}
__device__ __forceinline__ float4 peer4(const float* p, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(enigma_sm100::mapa_shared(enigma_sm100::smem_u32(p), uint32_t(rank)))
               : "memory");
  return v;
}

// SPLIT: each block of rows is a cluster of `parts` CTAs, which share its keys (a kernel of its own:
// one for both took 3 % longer where nothing is split).
template <typename T, int DP, bool SPLIT>
__global__ void __launch_bounds__(TT, TileCfg<DP>::CTAS)
packed_simt_kernel(const enigma_sdpa_packed_desc p, const bool vec, const int row_blocks,
                   const int n_parts) {
  using C = TileCfg<DP>;
  constexpr int TK = C::TK, LD = C::LD, KPT = C::KPT;
  const int parts = SPLIT ? n_parts : 1;
  extern __shared__ float4 smem4[];
  griddep_launch_dependents();
  float* s_q = reinterpret_cast<float*>(smem4);           // [TR][LD]
  float* s_k = s_q + TR * LD;                             // [TK][LD]
  float* s_v = s_k + TK * LD;                             // [TK][DP]
  float* s_p = s_v + TK * DP;                             // [TK][TR]
  const int tid = threadIdx.x;
  const PackedItem it = reinterpret_cast<const PackedItem*>(
      p.plan + p.header[enigma_serving::kItemsAt])[blockIdx.x / (row_blocks * parts)];
  const int G = int(p.heads_q / p.heads_kv), D = int(p.head_dim), kvh = it.kvh;
  // An item that does not lie inside the tensors is no work of theirs.
  if (it.q0 < 0 || it.q0 + int64_t(it.lq) > p.tokens_q || it.k0 < 0 ||
      it.k0 + int64_t(it.lk) > p.tokens_k || it.t0 < 0 || kvh < 0 || kvh >= p.heads_kv ||
      it.slot >= p.header[enigma_serving::kSlots])
    return;
  const int n = min(2 * it.tokens, it.lq - it.t0) * G;    // rows of the item
  // An item's row blocks side by side: the heaviest items start first.
  const int r0 = int(blockIdx.x / parts % row_blocks) * TR;
  if (r0 >= n) return;
  const int off = p.causal ? it.lk - it.lq + 1 : it.lk;   // a token's keys: min(lk, token + off)
  const int t_last = it.t0 + (min(r0 + TR, n) - 1) / G;
  int k_begin = it.j0 * 128, k_end = min(min(it.lk, t_last + off), it.j1 * 128);
  if (SPLIT && k_begin < k_end) {        // this CTA's keys
    const int rank = int(cluster_ctarank()), tiles = (k_end - k_begin + TK - 1) / TK;
    k_end = min(k_end, k_begin + tiles * (rank + 1) / parts * TK);
    k_begin += tiles * rank / parts * TK;
  }
  const T* kb = static_cast<const T*>(p.k) + it.k0 * p.k_token + kvh * p.k_head;
  const T* vb = static_cast<const T*>(p.v) + it.k0 * p.v_token + kvh * p.v_head;
  // Keys past the end are zeros in K and V; their weights are zero too.
  auto fetch_k = [&](int k0) {
    for (int x = tid; x < TK * (DP / 4); x += TT) {
      const int key = x / (DP / 4), d = x % (DP / 4) * 4;
      const bool there = k0 + key < it.lk && d < D;
      put4(s_k + key * LD + d, there ? kb + (k0 + key) * p.k_token : kb, d, D, vec, there);
    }
  };
  auto fetch_v = [&](int k0) {
    for (int x = tid; x < TK * (DP / 4); x += TT) {
      const int key = x / (DP / 4), d = x % (DP / 4) * 4;
      const bool there = k0 + key < it.lk && d < D;
      put4(s_v + key * DP + d, there ? vb + (k0 + key) * p.v_token : vb, d, D, vec, there);
    }
  };
  for (int x = tid; x < TR * (DP / 4); x += TT) {
    const int r = x / (DP / 4), d = x % (DP / 4) * 4, row = r0 + r;
    float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < n)
      q = row4(static_cast<const T*>(p.q) + (int64_t(it.q0) + it.t0 + row / G) * p.q_token +
                   (kvh * G + row % G) * p.q_head, d, D, vec);
    *reinterpret_cast<float4*>(s_q + r * LD + d) = q;
  }
  if (k_begin < k_end) {
    fetch_k(k_begin);
    fetch_v(k_begin);
  }
  const int rg = tid / 16, cg = tid % 16;    // rows rg * 8 .., keys cg + 16 c, columns cg * 4 ..
  int keys[8];                               // keys each row sees
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int row = r0 + rg * 8 + r;
    keys[r] = row < n ? min(it.lk, it.t0 + row / G + off) : 0;
  }
  float2 o[4][C::CPT];
  float m[8], l[8];                          // l: this thread's keys only
#pragma unroll
  for (int r = 0; r < 8; ++r) m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < C::CPT; ++c) o[r][c] = make_float2(0.f, 0.f);
  const float c_log2 = p.scale * 1.4426950408889634f;
  for (int k0 = k_begin; k0 < k_end; k0 += TK) {
    rows_landed();                           // K (and, one tile late, nothing else)
    __syncthreads();
    if (k0 > k_begin) fetch_v(k0);           // the last tile's P V is done
    asm volatile("cp.async.commit_group;" ::: "memory");
    float2 s2[8][KPT];                       // sums over even and odd elements
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int c = 0; c < KPT; ++c) s2[r][c] = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
      float4 k[KPT];
#pragma unroll
      for (int c = 0; c < KPT; ++c)
        k[c] = *reinterpret_cast<const float4*>(s_k + (cg + 16 * c) * LD + d);
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float4 q = *reinterpret_cast<const float4*>(s_q + (rg * 8 + r) * LD + d);
#pragma unroll
        for (int c = 0; c < KPT; ++c)
          s2[r][c] = fma2(make_float2(q.x, q.y), make_float2(k[c].x, k[c].y), s2[r][c]);
#pragma unroll
        for (int c = 0; c < KPT; ++c)
          s2[r][c] = fma2(make_float2(q.z, q.w), make_float2(k[c].z, k[c].w), s2[r][c]);
      }
    }
    __syncthreads();                         // K is read
    if (k0 + TK < k_end) fetch_k(k0 + TK);
    float e[8][KPT];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      float mx = m[r];
#pragma unroll
      for (int c = 0; c < KPT; ++c) {
        e[r][c] = s2[r][c].x + s2[r][c].y;
        if (k0 + cg + 16 * c >= keys[r]) e[r][c] = -INFINITY;
        mx = fmaxf(mx, e[r][c]);
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
      for (int c = 0; c < KPT; ++c) {
        e[r][c] = exp2f(fmaf(e[r][c], c_log2, -base));
        l[r] += e[r][c];
      }
    }
    // Four rows at once; their place in a key's row is turned by the key, so that the 8 lanes of
    // one store phase meet all banks.
#pragma unroll
    for (int c = 0; c < KPT; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float4*>(s_p + (cg + 16 * c) * TR + (((rg * 2 + h) ^ (cg & 7)) * 4)) =
            make_float4(e[4 * h][c], e[4 * h + 1][c], e[4 * h + 2][c], e[4 * h + 3][c]);
    if (k0 + TK < k_end)                     // V, but not the K tile just asked for
      asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 1;" ::: "memory");
    else
      rows_landed();
    __syncthreads();
#pragma unroll 4
    for (int j = 0; j < TK; ++j) {
      const float4 pa = *reinterpret_cast<const float4*>(s_p + j * TR + ((rg * 2) ^ (j & 7)) * 4);
      const float4 pb = *reinterpret_cast<const float4*>(s_p + j * TR + ((rg * 2 + 1) ^ (j & 7)) * 4);
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
  if (SPLIT) {
    // Each CTA's state into its own shared memory, over Q and K; then each joins its share of the
    // rows, reading the others' in their order.
    float2* s_ml = reinterpret_cast<float2*>(s_k);        // [TR]
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 8; ++r) {
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
      const int row = rg * 8 + r;
      // (Nothing but NaN scores: a sum of NaN, no maximum.)
      if (cg == 0)
        s_ml[row] = make_float2(m[r] == -INFINITY ? (l[r] == 0.f ? -INFINITY : 0.f) : m[r] * c_log2,
                                l[r]);
#pragma unroll
      for (int c = 0; c < C::CPT; ++c)
        s_q[row * LD + c / 4 * 64 + cg * 4 + c % 4] = (r & 1) ? o[r / 2][c].y : o[r / 2][c].x;
    }
    cluster_sync();
    const int share = TR / parts, first = int(cluster_ctarank()) * share;
    for (int x = tid; x < share * (DP / 4); x += TT) {
      const int in_block = first + x / (DP / 4), d = x % (DP / 4) * 4, row = r0 + in_block;
      if (row >= n || d >= D) continue;
      float M = -INFINITY, L = 0.f;
      for (int y = 0; y < parts; ++y) M = fmaxf(M, peer2(s_ml + in_block, y).x);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int y = 0; y < parts; ++y) {
        const float2 a = peer2(s_ml + in_block, y);
        if (a.x == -INFINITY) continue;                   // saw no key
        const float f = exp2f(a.x - M);
        const float4 v = peer4(s_q + in_block * LD + d, y);
        acc.x = fmaf(v.x, f, acc.x);
        acc.y = fmaf(v.y, f, acc.y);
        acc.z = fmaf(v.z, f, acc.z);
        acc.w = fmaf(v.w, f, acc.w);
        L = fmaf(a.y, f, L);
      }
      const int64_t tok = int64_t(it.q0) + it.t0 + row / G;
      const int h = kvh * G + row % G;
      const int tile = row / (it.tokens * G), in_tile = row - tile * it.tokens * G;
      const int64_t at = (int64_t(it.slot) + tile) * 128 + in_tile;
      const bool final = it.slot < 0;
      const float inv = !final ? 1.f : L == 0.f ? 0.f : 1.f / L;
      const float vv[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
      T* out = static_cast<T*>(p.out) + tok * p.o_token + h * p.o_head + d;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (d + c >= D) continue;
        if (final) store(out + c, vv[c]);
        else opart[at * D + d + c] = vv[c];
      }
      if (d == 0) {
        if (!final) ml[at] = make_float2(M, L);
        else if (p.lse != nullptr)
          p.lse[tok * p.heads_q + h] = (M + log2f(L)) * 0.6931471805599453f;
      }
    }
    cluster_sync();                          // the others have read
    return;
  }
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
    // Partial results: rows of the item's second tile go to the next slot.
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
        // (Nothing but NaN scores: a sum of NaN, no maximum.  The part is not empty.)
        ml[at] = make_float2(m[r] == -INFINITY && l[r] != 0.f ? 0.f : m[r] * c_log2, l[r]);
      } else if (p.lse != nullptr) {
        p.lse[tok * p.heads_q + h] = (m[r] * c_log2 + log2f(l[r])) * 0.6931471805599453f;
      }
    }
  }
}

// Joins the partial results of split rows: O = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i, always in
// the same order.  A warp takes four rows: 8 lanes each have a row's (m, l), and the four rows'
// loads of a part are in flight together (one row per warp: the loads' latency is the time, 13 us
// for 72 pairs of tiles in 2 parts).  grid (groups, rows / 32).
template <typename T, int V>
__global__ void __launch_bounds__(256)
packed_join_kernel(const enigma_sdpa_packed_desc p, const bool parts_blocked) {
  constexpr int R = 4;
  const int lane = threadIdx.x & 31, D = int(p.head_dim), G = int(p.heads_q / p.heads_kv);
  const int r0 = (int(blockIdx.y) * 8 + (threadIdx.x >> 5)) * R;   // first row, of 2 * 128
  const PackedGroup g = reinterpret_cast<const PackedGroup*>(
      p.plan + p.header[enigma_serving::kGroupsAt])[blockIdx.x];
  const float* opart = static_cast<const float*>(p.workspace);
  const float2* ml =
      reinterpret_cast<const float2*>(opart + int64_t(p.header[enigma_serving::kSlots]) * 128 * D);
  const int state = r0 / 128;
  const int row0 = r0 % 128, mine = row0 + (lane >> 3);            // this lane's row of (m, l)
  const int tok = g.tok0 + state * g.tokens + mine / G;
  // (A group that does not lie inside the tensors or the parts is none of theirs.)
  const bool live = mine < g.tokens * G && tok >= 0 && tok < g.tok_end && tok < p.tokens_q &&
                    g.kvh >= 0 && g.kvh < p.heads_kv && g.slot >= 0 &&
                    g.slot + 2 * int64_t(g.parts) <= p.header[enigma_serving::kSlots];
  if (!__any_sync(0xffffffffu, live)) return;
  const int n = g.parts;
  const int64_t step = 2 * 128, at = int64_t(g.slot + state) * 128;
  // Element d of row r of a part: [d / 8][r][d % 8] (blocked) or [r][d].
  const bool blocked = sizeof(T) == 2 && parts_blocked;     // fp32 parts never are
  const int row = blocked ? 8 : D, v_step = blocked ? 4 * 128 * 8 : 32;
  const int lane_at = blocked ? lane / 8 * 128 * 8 + lane % 8 : lane;
  griddep_wait();                                                  // the parts are written
  float M = -INFINITY, l = 0.f;
  float acc[R][V];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int v = 0; v < V; ++v) acc[r][v] = 0.f;
  if (live)
    for (int i = lane & 7; i < n; i += 8) M = fmaxf(M, ml[at + mine + i * step].x);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  for (int i0 = 0; i0 < n; i0 += 8) {
    const int i = i0 + (lane & 7);
    const float2 x = live && i < n ? ml[at + mine + i * step] : make_float2(-INFINITY, 0.f);
    const float w = x.x == -INFINITY ? 0.f : exp2f(x.x - M);       // this part saw no key: 0
    if (w != 0.f) l = fmaf(x.y, w, l);
    const int here = min(8, n - i0);
    for (int y = 0; y < here; ++y) {
      float f[R], o[R][V];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        f[r] = __shfl_sync(0xffffffffu, w, r * 8 + y);
        const float* from = opart + (at + (i0 + y) * step) * D + (row0 + r) * row + lane_at;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          o[r][v] = 0.f;
          if (f[r] != 0.f && lane + 32 * v < D) o[r][v] = from[v * v_step];
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v) acc[r][v] = fmaf(o[r][v], f[r], acc[r][v]);
    }
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  const int h = g.kvh * G + mine % G;
  if (p.lse != nullptr && live && (lane & 7) == 0)
    p.lse[int64_t(tok) * p.heads_q + h] =
        l == 0.f ? -INFINITY : (M + log2f(l)) * 0.6931471805599453f;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t to = int64_t(tok) * p.o_token + int64_t(h) * p.o_head;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float s = __shfl_sync(0xffffffffu, inv, r * 8);
    const int64_t to_row = __shfl_sync(0xffffffffu, to, r * 8);
    if (__shfl_sync(0xffffffffu, live ? 1 : 0, r * 8) == 0) continue;
    T* out = static_cast<T*>(p.out) + to_row;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (lane + 32 * v < D) store(out + lane + 32 * v, acc[r][v] * s);
  }
}

template <typename T>
cudaError_t launch_join(const enigma_sdpa_packed_desc& d, const dim3 grid, bool blocked, cudaStream_t s) {
  if (d.head_dim <= 64) return enigma::launch_dependent(packed_join_kernel<T, 2>, grid, 256, 0, s, d, blocked);
  if (d.head_dim <= 128) return enigma::launch_dependent(packed_join_kernel<T, 4>, grid, 256, 0, s, d, blocked);
  return enigma::launch_dependent(packed_join_kernel<T, 8>, grid, 256, 0, s, d, blocked);
}

template <typename T, int DP>
cudaError_t launch_packed(const enigma_sdpa_packed_desc& d, cudaStream_t s) {
  using C = TileCfg<DP>;
  // Four elements at a time where every row starts on their boundary.
  const int64_t size = 4 * int64_t(sizeof(T));
  bool vec = true;
  for (const void* b : {d.q, d.k, d.v}) vec &= reinterpret_cast<uintptr_t>(b) % uintptr_t(size) == 0;
  for (const int64_t x : {d.q_token, d.q_head, d.k_token, d.k_head, d.v_token, d.v_head})
    vec &= x % 4 == 0;
  const int64_t group = d.heads_q / d.heads_kv;
  const int64_t rows = 2 * std::max<int64_t>(1, ENIGMA_PACKED_TILE_ROWS / group) * group;
  const int row_blocks = int((rows + TR - 1) / TR);
  const int64_t blocks = int64_t(d.header[enigma_serving::kItems]) * row_blocks;
  if (blocks > (int64_t(1) << 31) - 1) return cudaErrorInvalidConfiguration;
  // Where twice as many blocks would still be at most two rounds of what the SMs hold, clusters split
  // each one's keys, into parts of 128 keys or more (30 tokens against 2000 keys, 8 / 2 heads of 64:
  // 60 -> 30 us; 295 against 1258, 14 / 2 of 128: 129 -> 78, and unsplit with one round as the limit;
  // four rounds: 96).
  int parts = 1;
  while (parts < 8 && blocks * parts * 2 <= 2 * int64_t(enigma::sm_count()) * C::CTAS &&
         d.header[enigma_serving::kLongest] >= 2 * parts)
    parts *= 2;
  const auto kernel = parts > 1 ? packed_simt_kernel<T, DP, true> : packed_simt_kernel<T, DP, false>;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(unsigned(blocks * parts));
  c.blockDim = dim3(TT);
  c.dynamicSmemBytes = C::SMEM;
  c.stream = s;
  cudaLaunchAttribute a[1];
  a[0].id = cudaLaunchAttributeClusterDimension;
  a[0].val.clusterDim.x = unsigned(parts);
  a[0].val.clusterDim.y = a[0].val.clusterDim.z = 1;
  c.attrs = a;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, d, vec, row_blocks, parts);
}

template <typename T>
cudaError_t launch_packed(const enigma_sdpa_packed_desc& d, cudaStream_t s) {
  if (d.head_dim <= 64) return launch_packed<T, 64>(d, s);
  if (d.head_dim <= 128) return launch_packed<T, 128>(d, s);
  return launch_packed<T, 256>(d, s);
}

// ============================================================================ paged
// One CTA per (sequence, query head); its warps take every kWarps-th key and merge at the end.  A key
// without a page is one of zeros, as TMA reads it for the tensor-core kernels.  The simple form: every
// query head reads K and V, the prefix too, for itself, a key costs a warp one dependent chain (dot
// product, five shuffles, two exponentials, rescale), and long rows are not split.  That chain is the
// time, not memory: 16 sequences of 1 to 8191 keys, 32 / 8 heads of 128, fp32: 1808 us against 82 for
// the bytes; one of 22250 keys: 4809 against 28.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
paged_simt_kernel(const enigma_sdpa_shared_prefix_desc p) {
  __shared__ float s_m[kWarps], s_l[kWarps], s_acc[kWarps][256];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.x, D = int(p.head_dim);
  const int64_t b = blockIdx.y;
  const int kvh = h / int(p.heads_q / p.heads_kv);
  const int64_t slot = p.slots != nullptr ? p.slots[b] : b;
  const int64_t slot0 = p.slots != nullptr ? p.slots[0] : 0;      // the prefix is read through it
  const bool there = slot >= 0 && slot < p.n_slots, there0 = slot0 >= 0 && slot0 < p.n_slots;
  const int64_t len = there ? min(int64_t(max(p.lens[slot], 0)), p.table_width * p.page) : 0;
  Row<T> row;
  row.start(static_cast<const T*>(p.q) + b * p.q_batch + h * p.q_head, D, lane, p.scale);
  int zeros = 0;                                            // keys of this warp without a page
  int64_t j = warp;
  if (!there0 && j < min(len, p.prefix_len)) {
    zeros = int((min(len, p.prefix_len) - j + kWarps - 1) / kWarps);
    j += int64_t(zeros) * kWarps;
  }
  for (; j < len; j += kWarps) {
    const int64_t s = j < p.prefix_len ? slot0 : slot;
    const int at = p.table[s * p.table_width + j / p.page];
    if (at < 0 || at >= p.pages) {                          // not a page: reads as zeros
      ++zeros;
      continue;
    }
    const int64_t off = (kvh * p.page + j % p.page) * D;
    row.key(static_cast<const T*>(p.k_pages) + at * p.k_page + off,
            static_cast<const T*>(p.v_pages) + at * p.v_page + off, D, lane);
  }
  if (zeros > 0) row.zero_keys(zeros);
#pragma unroll
  for (int x = 0; x < kMaxDPerLane; ++x) s_acc[warp][lane + 32 * x] = row.acc[x];
  if (lane == 0) {
    s_m[warp] = row.m;
    s_l[warp] = row.l;
  }
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w]);
  // A warp without keys has l = 0; one with nothing but NaN scores has no maximum either, but l = NaN.
  for (int w = 0; w < kWarps; ++w) L += s_l[w] == 0.f ? 0.f : s_l[w] * expf(s_m[w] - M);
  for (int d = threadIdx.x; d < D; d += kWarps * 32) {
    float o = 0.f;
    for (int w = 0; w < kWarps; ++w)
      if (s_l[w] != 0.f) o = fmaf(s_acc[w][d], expf(s_m[w] - M), o);
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

cudaError_t sdpa_packed_join_launch(const enigma_sdpa_packed_desc& d, bool blocked, cudaStream_t s) {
  const int groups = d.header[enigma_serving::kGroups];
  if (groups == 0) return cudaSuccess;
  const dim3 grid(unsigned(groups), 2 * ENIGMA_PACKED_TILE_ROWS / 32);
  return d.dtype == ENIGMA_DTYPE_F32 ? launch_join<float>(d, grid, blocked, s)
                                     : launch_join<__nv_bfloat16>(d, grid, blocked, s);
}

cudaError_t sdpa_paged_simt_launch(const enigma_sdpa_shared_prefix_desc& d, cudaStream_t s) {
  note_kernel("paged_simt_kernel");
  const dim3 grid(unsigned(d.heads_q), unsigned(d.batch));
  if (d.dtype == ENIGMA_DTYPE_F32) paged_simt_kernel<float><<<grid, kWarps * 32, 0, s>>>(d);
  else paged_simt_kernel<__nv_bfloat16><<<grid, kWarps * 32, 0, s>>>(d);
  return cudaGetLastError();
}

}  // namespace enigma
