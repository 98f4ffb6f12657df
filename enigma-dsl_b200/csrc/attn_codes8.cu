// attn_codes8.cu — one new token per sequence over a paged cache held in 8-bit codes with a scale for
// each 16 tokens of a page and head (codes8.cuh):
//   out = sum_j softmax_j(c s_k(j) q . k_j) s_v(j) v_j  over the sequence's first len keys.
//
// Bound by memory: a key costs 2 D bytes and a few scales, read once for all query heads of its kv
// head.  The work is the flattened list of (unit, chunk of KEYS keys), unit = (sequence, kv head, up to
// 8 NT of its query heads); warp w of W takes the contiguous range [w n, (w + 1) n), n = ceil(T / W), so
// every SM streams as much, whatever the lengths are.  Each warp has a ring of its own in shared memory
// that it fills with cp.async (16 bytes a lane) and empties by itself: no barrier until the end, and
// nothing to wait for but its own copies.  A unit that lies within one warp's range is finished
// there.  The others leave pieces (maximum, sum, unnormalised O): the block joins its warps' pieces
// after its only barrier, and what goes past a block's ends is joined by join_codes8_kernel.
//
// Both products are m16n8k16 with fp16 operands and fp32 sums, which hold every code exactly; keys
// or the head's elements are the 16-row side, the query heads (8) the narrow one:
//   S^T [keys, heads] = K Q^T,   O^T [elements, heads] += V^T P^T.
// The order of a product's inner index is free as long as both operands share it, and so is which
// rows stand where: so a lane's operands are 16 consecutive bytes of a key's row in both products,
// no fragment needs a transposing load, and V's pairs of keys are made by byte permutations before
// they are converted.  Scores take s_k in fp32.  s_v goes into P relative to the chunk's larger
// one, which is applied to the chunk's product in fp32, as is exp2(chunk's maximum - running maximum):
// P is at most 2^15, its largest value exactly, so rounding it to fp16 costs 2^-11 of the weight, or
// 2^-40 of the chunk's largest.  fp32 queries and P are two fp16 numbers each (2^-22, or the same
// 2^-40).  Queries are brought to [2^11, 2^12) by a power of two per head.
#include <algorithm>
#include <atomic>

#include "attn_serving.cuh"
#include "codes8.cuh"

namespace {

using namespace enigma_codes8;
using namespace enigma_sm100;

constexpr int WARPS = 8;
constexpr int THREADS = WARPS * 32;
constexpr int SLOTS = WARPS + 2;         // pieces of a block in the workspace: its warps' first ones,
constexpr int BEFORE = WARPS;            // what it has of a unit that began in another block,
constexpr int AFTER = WARPS + 1;         // and of one that goes on in the next

template <int DT, int NT>
struct Cfg {
  static constexpr int KEYS = DT == 256 ? 16 : 32;       // of a chunk
  static constexpr int MT = KEYS / 16;                    // 16-key tiles, scale blocks
  static constexpr int TILE = KEYS * DT;                  // bytes of K or V
  static constexpr int STAGES = DT == 64 ? 6 : 3;
  static constexpr int RING = STAGES * 2 * TILE;          // 24 KB a warp
  static constexpr int TILES = DT / 16;                   // 16-element tiles of O
  static constexpr int HEADS = 8 * NT;
  static constexpr int PIECE = (TILES * NT * 4) * 32;     // floats of O in fragment order
  static constexpr int SLOT = PIECE + 2 * HEADS;          // and maxima and sums
};

struct Attend {
  const void* q;
  void* out;
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int32_t *table, *lens, *slots;
  int64_t q_batch, q_head, o_batch, o_head, k_page, v_page, ks_page, vs_page;
  int batch, heads_kv, group, blocks, d, page_shift, pages, width, n_slots;
  int whole;                             // a block per unit: nothing to join
  float scale_log2;
  bool q_vec, o_vec;                     // rows of q, out on 16 bytes
  float* pieces;                         // [block][SLOTS][SLOT]
  int2* links;                           // [block]: unit that goes on behind it, blocks it spans
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;"
               ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turn_8x8(uint32_t x) {   // an 8 x 8 fragment, transposed
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_halves(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// The same and what it leaves over, as halves.
__device__ __forceinline__ uint32_t split_halves(float lo, float hi, uint32_t* rest) {
  const uint32_t r = pack_halves(lo, hi);
  const float2 f = floats_of(r);
  *rest = pack_halves(lo - f.x, hi - f.y);
  return r;
}
// Maximum or sum over the lanes that hold the same heads.
__device__ __forceinline__ float max_over_keys(float x) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ float sum_over_keys(float x) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
// 0 where nothing was seen, so that no difference of infinities is taken.
__device__ __forceinline__ float base_of(float top) { return top == -INFINITY ? 0.f : top; }

// Where chunk c (16 bytes) of row r is in a tile.  Eight lanes that load at once must find eight
// different 16-byte columns of a 128-byte line: of K, lanes of two neighbouring rows and four
// neighbouring chunks; of V, of two neighbouring chunks and every second of eight rows.
template <int DT>
__device__ __forceinline__ uint32_t k_at(int r, int c) {
  if (DT == 64) return uint32_t(r * 64 + c * 16);
  return uint32_t(r * DT + ((c ^ (((r & 1) << 2) | ((r >> 1) & 3))) << 4));
}
template <int DT>
__device__ __forceinline__ uint32_t v_at(int r, int c) {
  if (DT == 64) return uint32_t((r >> 1) * 128 + (((((r & 1) << 2) + c) ^ (r & 6)) << 4));
  return uint32_t(r * DT + ((c ^ (r & 7)) << 4));
}

__device__ __forceinline__ int len_at(const Attend& a, int b) {
  const int slot = a.slots ? a.slots[b] : b;
  if (slot < 0 || slot >= a.n_slots) return 0;
  return int(min(int64_t(max(a.lens[slot], 0)), int64_t(a.width) << a.page_shift));
}

// A place in the work list: chunk j of the n of a unit.
struct Place {
  int b, u, j, n, len;
  int64_t row;                           // first entry of the sequence's table row
};

__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// Two neighbouring elements of a head's result.
template <typename T>
__device__ __forceinline__ void store_pair(T* p, float x, float y, bool vec) {
  if (sizeof(T) == 2 && vec) {
    *reinterpret_cast<uint32_t*>(p) = pack_bf16x2(x, y);
  } else if (vec) {
    *reinterpret_cast<float2*>(p) = make_float2(x, y);
  } else {
    store1(p, x);
    store1(p + 1, y);
  }
}

// First element of O's tile m that lane (g, t) has, in rows g and g + 8: e and e + 1.
template <int DT>
__device__ __forceinline__ int element_of(int m, int g) {
  if (DT == 64) return 8 * g + 2 * m;
  return DT == 128 || m < 8 ? 16 * g + 2 * m : 128 + 16 * g + 2 * (m - 8);
}

template <typename T>
__device__ __forceinline__ T* out_row(const Attend& a, int b, int u, int head) {
  const int kvh = u / a.blocks;
  return static_cast<T*>(a.out) + b * a.o_batch + int64_t(kvh * a.group + head) * a.o_head;
}

// T: of queries and results; DT: the head's elements, rounded up; NT: tiles of 8 query heads.
template <typename T, bool E4M3, int DT, int NT>
__global__ void __launch_bounds__(THREADS, 1) attend_codes8_kernel(const Attend a) {
  using C = Cfg<DT, NT>;
  constexpr bool SPLIT = sizeof(T) == 4;
  constexpr int MT = C::MT, KEYS = C::KEYS;
  extern __shared__ __align__(128) uint8_t smem[];       // rings, chunks before each b, lengths
  __shared__ float s_scale[WARPS][C::STAGES][2 * MT];
  __shared__ float s_m[WARPS][C::HEADS], s_l[WARPS][C::HEADS];   // of the pieces in the rings
  __shared__ int s_unit[2 * WARPS], s_ends[2 * WARPS];   // pieces in order: a warp's first, its last
  __shared__ int s_warp[WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * C::RING;
  const uint32_t ring_at = smem_u32(ring);
  int* s_starts = reinterpret_cast<int*>(smem + WARPS * C::RING);        // [batch + 1]
  int* s_len = s_starts + a.batch + 1;                                    // [batch]
  const int per_b = a.heads_kv * a.blocks;
  griddep_launch_dependents();
  if (tid < 2 * WARPS) s_unit[tid] = -1;
  if (a.d < DT)                          // columns that no copy fills
    for (int x = tid; x < WARPS * C::RING / 16; x += THREADS)
      reinterpret_cast<uint4*>(smem)[x] = make_uint4(0, 0, 0, 0);
  griddep_wait();

  // The warp's range [x0, x1) of the list (whole: of the block's unit), per of them a warp.
  int64_t x0, x1, per;
  Place in;
  if (a.whole) {
    in.b = int(blockIdx.x) / per_b;
    in.u = int(blockIdx.x) - in.b * per_b;
    in.len = len_at(a, in.b);
    in.n = (in.len + KEYS - 1) / KEYS;
    if (in.len == 0) {
      const int hb = in.u % a.blocks * C::HEADS, heads = min(C::HEADS, a.group - hb);
      for (int x = tid; x < heads * a.d; x += THREADS)
        store1(out_row<T>(a, in.b, in.u, hb + x / a.d) + x % a.d, 0.f);
      return;
    }
    per = (in.n + WARPS - 1) / WARPS;
    x0 = min(warp * per, int64_t(in.n));
    x1 = min(x0 + per, int64_t(in.n));
    in.j = int(x0);
    __syncthreads();
  } else {
    int run = 0;
    for (int b0 = 0; b0 < a.batch; b0 += THREADS) {
      const int b = b0 + tid;
      int v = 0;
      if (b < a.batch) {
        const int len = len_at(a, b);
        s_len[b] = len;
        v = (len + KEYS - 1) / KEYS;
      }
      int x = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) s_warp[warp] = x;
      __syncthreads();
      int before = run;
      for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += s_warp[w];
        run += s_warp[w];
      }
      if (b < a.batch) s_starts[b] = before + x - v;
      __syncthreads();
    }
    if (tid == 0) s_starts[a.batch] = run;
    __syncthreads();
    const int64_t total = int64_t(run) * per_b;
    per = (total + int64_t(gridDim.x) * WARPS - 1) / (int64_t(gridDim.x) * WARPS);
    x0 = min((int64_t(blockIdx.x) * WARPS + warp) * per, total);
    x1 = min(x0 + per, total);
    if (x0 < x1) {
      int lo = 0, hi = a.batch;          // the last b with starts[b] * per_b <= x0
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (int64_t(s_starts[mid]) * per_b <= x0) lo = mid;
        else hi = mid;
      }
      in.b = lo;
      in.len = s_len[lo];
      in.n = s_starts[lo + 1] - s_starts[lo];
      const int64_t within = x0 - int64_t(s_starts[lo]) * per_b;
      in.u = int(within / in.n);
      in.j = int(within - int64_t(in.u) * in.n);
    }
    // Sequences without keys are in nobody's range.
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x)
      if (s_len[b] == 0)
        for (int x = tid; x < a.heads_kv * a.group * a.d; x += THREADS)
          store1(static_cast<T*>(a.out) + b * a.o_batch + int64_t(x / a.d) * a.o_head + x % a.d, 0.f);
  }

  auto find_row = [&](Place& p) {
    p.row = int64_t(a.slots ? a.slots[p.b] : p.b) * a.width;
  };
  auto advance = [&](Place& p) {         // (called only where another chunk of the range follows)
    if (++p.j < p.n) return;
    p.j = 0;
    if (++p.u < per_b) return;
    p.u = 0;
    do {
      ++p.b;
      p.n = s_starts[p.b + 1] - s_starts[p.b];
    } while (p.n == 0);
    p.len = s_len[p.b];
    find_row(p);
  };
  // Asks for a chunk's codes and scales; keys behind the last and without a page are zeros.
  const int page_mask = (1 << a.page_shift) - 1, parts = (page_mask + 1) / kScaleBlock;
  const int chunks = a.d >> 4;           // 16-byte chunks of a row
  auto issue = [&](const Place& p, int stage) {
    const int kvh = p.u / a.blocks;
    const uint32_t kd = ring_at + stage * 2 * C::TILE, vd = kd + C::TILE;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int key0 = p.j * KEYS + 16 * i, live = min(16, p.len - key0);
      const int page = live > 0 ? a.table[p.row + (key0 >> a.page_shift)] : -1;
      const bool has = page >= 0 && page < a.pages;
      const int in_page = key0 & page_mask;
      const int64_t at = has ? (int64_t(kvh) * (page_mask + 1) + in_page) * a.d : 0;
      const uint8_t* k = a.k + (has ? page * a.k_page + at : 0);
      const uint8_t* v = a.v + (has ? page * a.v_page + at : 0);
      constexpr int PER = DT / 16, ROWS = 32 / PER;          // chunks of a row, rows at once
      const int c = lane % PER;
#pragma unroll
      for (int r0 = 0; r0 < 16; r0 += ROWS) {
        const int r = r0 + lane / PER;
        const uint32_t bytes = has && r < live ? 16 : 0;
        const int64_t from = bytes ? int64_t(r) * a.d + c * 16 : 0;
        if (c < chunks) {
          cp_async16(kd + k_at<DT>(16 * i + r, c), k + from, bytes);
          cp_async16(vd + v_at<DT>(16 * i + r, c), v + from, bytes);
        }
      }
      if (lane < 2) {
        const float* s = lane ? a.vs : a.ks;
        const int64_t where = page * (lane ? a.vs_page : a.ks_page) + kvh * parts + in_page / kScaleBlock;
        cp_async4(smem_u32(&s_scale[warp][stage][lane * MT + i]), s + (has ? where : 0), has ? 4 : 0);
      }
    }
  };

  uint32_t qf[NT][DT / 16][SPLIT ? 4 : 2];               // queries: both halves of the inner index
  float cq[NT][2];                                       // what brings a head's scores to log2 units
  float m[NT][2], l[NT][2], o[C::TILES][NT][4];
  auto load_queries = [&](const Place& p) {
    const int kvh = p.u / a.blocks, hb = (p.u - kvh * a.blocks) * C::HEADS;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int head = hb + nt * 8 + g;
      const T* row = static_cast<const T*>(a.q) + p.b * a.q_batch + int64_t(kvh * a.group + head) * a.q_head;
      float x[DT / 64][16];
      uint32_t top = 0;
#pragma unroll
      for (int jj = 0; jj < DT / 64; ++jj) {
        const int e = 64 * jj + 16 * t;
        const bool there = head < a.group && e < a.d;
        if (there && a.q_vec) {
#pragma unroll
          for (int i = 0; i < int(sizeof(T)); ++i) {         // 16 elements: 2 or 4 times 16 bytes
            const uint4 w = *reinterpret_cast<const uint4*>(row + e + i * (16 / int(sizeof(T))));
            const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              if (SPLIT) {
                x[jj][(4 * i + y) & 15] = __uint_as_float(v[y]);
              } else {
                x[jj][(8 * i + 2 * y) & 15] = __uint_as_float(v[y] << 16);
                x[jj][(8 * i + 2 * y + 1) & 15] = __uint_as_float(v[y] & 0xffff0000u);
              }
            }
          }
        } else {
#pragma unroll
          for (int y = 0; y < 16; ++y) x[jj][y] = there ? float(row[e + y]) : 0.f;
        }
#pragma unroll
        for (int y = 0; y < 16; ++y) top = max(top, __float_as_uint(x[jj][y]) & 0x7fffffffu);
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = max(27, int(top >> 23));                 // biased; 2^-100 at least
      const float up = __uint_as_float(uint32_t(127 + 127 + 11 - e) << 23);
      const float back = __uint_as_float(uint32_t(max(e - 11, 1)) << 23) * a.scale_log2;
#pragma unroll
      for (int i = 0; i < 2; ++i) cq[nt][i] = __shfl_sync(0xffffffffu, back, (2 * t + i) * 4);
#pragma unroll
      for (int jj = 0; jj < DT / 64; ++jj)
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float lo = x[jj][4 * s + 2 * i] * up, hi = x[jj][4 * s + 2 * i + 1] * up;
            if (SPLIT) qf[nt][4 * jj + s][i] = split_halves(lo, hi, &qf[nt][4 * jj + s][(2 + i) % (SPLIT ? 4 : 2)]);
            else qf[nt][4 * jj + s][i] = pack_halves(lo, hi);
          }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[nt][i] = -INFINITY;
        l[nt][i] = 0.f;
      }
#pragma unroll
      for (int x = 0; x < C::TILES; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[x][nt][i] = 0.f;
    }
  };

  auto compute = [&](const Place& p, int stage) {
    const uint32_t kd = ring_at + stage * 2 * C::TILE, vd = kd + C::TILE;
    const float* sc = s_scale[warp][stage];
    float s[MT][NT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[i][nt][x] = 0.f;
#pragma unroll
    for (int jj = 0; jj < DT / 64; ++jj) {
      if (64 * jj >= a.d) break;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint4 x = lds128(kd + k_at<DT>(16 * i + g, 4 * jj + t));
        const uint4 y = lds128(kd + k_at<DT>(16 * i + g + 8, 4 * jj + t));
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          uint32_t f[4];
          halves_of4<E4M3>(xs[z], &f[0], &f[2]);
          halves_of4<E4M3>(ys[z], &f[1], &f[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(s[i][nt], f, qf[nt][4 * jj + z][0], qf[nt][4 * jj + z][1]);
            if (SPLIT) mma_f16(s[i][nt], f, qf[nt][4 * jj + z][2 % (SPLIT ? 4 : 2)],
                               qf[nt][4 * jj + z][3 % (SPLIT ? 4 : 2)]);
          }
        }
      }
    }
    // V's codes while the scores are weighed: keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of each tile.
    constexpr int WORDS = DT / 32;
    uint32_t vw[MT][4][WORDS];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const int r = 16 * i + 2 * t + (z & 1) + 8 * (z >> 1);
        if (DT == 64) {
          const uint2 w = lds64(vd + v_at<DT>(r, g >> 1) + (g & 1) * 8);
          vw[i][z][0] = w.x;
          vw[i][z][1] = w.y;
        } else {
#pragma unroll
          for (int h = 0; h < DT / 128; ++h) {
            const uint4 w = lds128(vd + v_at<DT>(r, g + 8 * h));
            vw[i][z][(4 * h) % WORDS] = w.x;
            vw[i][z][(4 * h + 1) % WORDS] = w.y;
            vw[i][z][(4 * h + 2) % WORDS] = w.z;
            vw[i][z][(4 * h + 3) % WORDS] = w.w;
          }
        }
      }
    const bool last = (p.j + 1) * KEYS > p.len;              // some of its keys do not count
    float top_v = 0.f, ratio[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) top_v = fmaxf(top_v, fabsf(sc[MT + i]));
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const float x = sc[MT + i];
      ratio[i] = x == 0.f ? 0.f : fabsf(x) == top_v ? copysignf(1.f, x) : x / top_v;
    }
    uint32_t pf[MT][NT][SPLIT ? 4 : 2];
    float fresh[NT][2];
    bool grown = false;
    float shrink[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          s[i][nt][x] *= sc[i] * cq[nt][x & 1];
          if (last && p.j * KEYS + 16 * i + g + 8 * (x >> 1) >= p.len) s[i][nt][x] = -INFINITY;
          top[x & 1] = fmaxf(top[x & 1], s[i][nt][x]);
        }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        top[x] = max_over_keys(top[x]);
        const float now = fmaxf(m[nt][x], top[x]), base = base_of(now);
        grown |= now != m[nt][x];
        shrink[nt][x] = ex2(m[nt][x] - base);
        fresh[nt][x] = ex2(top[x] - base);
        m[nt][x] = now;
        top[x] = 15.f - base_of(top[x]);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        float w[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          w[x] = ex2(s[i][nt][x] + top[x & 1]);
          sum[x & 1] += w[x];
          w[x] *= ratio[i];
        }
        if (SPLIT) {
          uint32_t r0, r1;
          pf[i][nt][0] = turn_8x8(split_halves(w[0], w[1], &r0));
          pf[i][nt][1] = turn_8x8(split_halves(w[2], w[3], &r1));
          pf[i][nt][2 % (SPLIT ? 4 : 2)] = turn_8x8(r0);
          pf[i][nt][3 % (SPLIT ? 4 : 2)] = turn_8x8(r1);
        } else {
          pf[i][nt][0] = turn_8x8(pack_halves(w[0], w[1]));
          pf[i][nt][1] = turn_8x8(pack_halves(w[2], w[3]));
        }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        l[nt][x] = l[nt][x] * shrink[nt][x] + sum[x] * fresh[nt][x];
        fresh[nt][x] *= top_v;
      }
    }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int x = 0; x < C::TILES; ++x)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[x][nt][i] *= shrink[nt][i & 1];
    }
#pragma unroll
    for (int z = 0; z < WORDS; ++z)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float acc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 4; ++x) acc[nt][x] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          uint32_t f[4];
          halves_of4<E4M3>(__byte_perm(vw[i][0][z], vw[i][1][z], half ? 0x7362 : 0x5140), &f[0], &f[1]);
          halves_of4<E4M3>(__byte_perm(vw[i][2][z], vw[i][3][z], half ? 0x7362 : 0x5140), &f[2], &f[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(acc[nt], f, pf[i][nt][0], pf[i][nt][1]);
            if (SPLIT) mma_f16(acc[nt], f, pf[i][nt][2 % (SPLIT ? 4 : 2)], pf[i][nt][3 % (SPLIT ? 4 : 2)]);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            o[2 * z + half][nt][x] = fmaf(acc[nt][x], fresh[nt][x & 1], o[2 * z + half][nt][x]);
      }
  };

  if (x0 < x1) {
    find_row(in);
    Place at = in;
    int64_t asked = x0;
    auto next = [&](int stage) {
      if (asked < x1) {
        issue(in, stage);
        if (++asked < x1) advance(in);
      }
      cp_commit();
    };
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; ++s) next(s);
    int st = 0, to = C::STAGES - 1;
    bool fresh = true, began = false;
    for (int64_t x = x0; x < x1; ++x) {
      if (fresh) {
        load_queries(at);
        began = at.j == 0;
        fresh = false;
      }
      cp_wait<C::STAGES - 2>();
      __syncwarp();                      // every lane's copies, and nobody reads the stage before
      next(to);
      compute(at, st);
      st = st + 1 == C::STAGES ? 0 : st + 1;
      to = to + 1 == C::STAGES ? 0 : to + 1;
      const bool end = at.j + 1 == at.n, over = x + 1 == x1;
      if (end || over) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int y = 0; y < 2; ++y) l[nt][y] = sum_over_keys(l[nt][y]);
        if (began && end) {              // all of the unit
          const int hb = at.u % a.blocks * C::HEADS;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int head = hb + nt * 8 + 2 * t + y;
              if (head >= a.group) continue;
              T* row = out_row<T>(a, at.b, at.u, head);
              const float sum = l[nt][y], inv = 1.f / sum;
#pragma unroll
              for (int mt = 0; mt < C::TILES; ++mt) {
                const int e = element_of<DT>(mt, g);
                if (e < a.d)
                  store_pair(row + e, sum == 0.f ? 0.f : o[mt][nt][y] * inv,
                             sum == 0.f ? 0.f : o[mt][nt][2 + y] * inv, a.o_vec);
              }
            }
        } else {
          // A first piece that others follow goes to the workspace, a last one where the copies were.
          __syncwarp();
          float* to_o = over ? reinterpret_cast<float*>(ring)
                             : a.pieces + (int64_t(blockIdx.x) * SLOTS + warp) * C::SLOT;
          float* to_m = over ? s_m[warp] : to_o + C::PIECE;
          float* to_l = over ? s_l[warp] : to_m + C::HEADS;
#pragma unroll
          for (int mt = 0; mt < C::TILES; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int y = 0; y < 4; ++y) to_o[((mt * NT + nt) * 4 + y) * 32 + lane] = o[mt][nt][y];
          if (g == 0)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                to_m[nt * 8 + 2 * t + y] = m[nt][y];
                to_l[nt * 8 + 2 * t + y] = l[nt][y];
              }
          if (lane == 0) {
            s_unit[2 * warp + over] = at.b * per_b + at.u;
            s_ends[2 * warp + over] = (began ? 1 : 0) | (end ? 2 : 0);
          }
        }
        fresh = true;
      }
      if (!over) advance(at);
    }
  }
  __syncthreads();

  // The warps' pieces, unit by unit.
  if (!a.whole && tid == 0) a.links[blockIdx.x] = make_int2(0, 0);
  for (int i0 = 0; i0 < 2 * WARPS;) {
    const int unit = s_unit[i0];
    if (unit < 0) {
      ++i0;
      continue;
    }
    int i1 = i0 + 1, tail = i0;
    while (i1 < 2 * WARPS && (s_unit[i1] < 0 || s_unit[i1] == unit)) {
      if (s_unit[i1] >= 0) tail = i1;
      ++i1;
    }
    const bool began = s_ends[i0] & 1, end = s_ends[tail] & 2;
    const int b = unit / per_b, u = unit - b * per_b, hb = u % a.blocks * C::HEADS;
    float* to = a.pieces + (int64_t(blockIdx.x) * SLOTS + (began ? AFTER : BEFORE)) * C::SLOT;
    for (int x = warp; x < C::TILES * NT; x += WARPS) {
      const int mt = x / NT, nt = x % NT, h0 = nt * 8 + 2 * t;
      float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f}, acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (int i = i0; i <= tail; ++i) {
        if (s_unit[i] < 0) continue;
        const float* piece = a.pieces + (int64_t(blockIdx.x) * SLOTS + (i >> 1)) * C::SLOT;
        const float* pm = i & 1 ? s_m[i >> 1] : piece + C::PIECE;
        top[0] = fmaxf(top[0], pm[h0]);
        top[1] = fmaxf(top[1], pm[h0 + 1]);
      }
      for (int i = i0; i <= tail; ++i) {
        if (s_unit[i] < 0) continue;
        const float* piece = a.pieces + (int64_t(blockIdx.x) * SLOTS + (i >> 1)) * C::SLOT;
        const float* pm = i & 1 ? s_m[i >> 1] : piece + C::PIECE;
        const float* pl = i & 1 ? s_l[i >> 1] : piece + C::PIECE + C::HEADS;
        const float* po = i & 1 ? reinterpret_cast<const float*>(smem + (i >> 1) * C::RING) : piece;
        float w[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          w[y] = ex2(pm[h0 + y] - base_of(top[y]));
          sum[y] += pl[h0 + y] * w[y];
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[y] += po[((mt * NT + nt) * 4 + y) * 32 + lane] * w[y & 1];
      }
      if (began && end) {
        const int e = element_of<DT>(mt, g);
#pragma unroll
        for (int y = 0; y < 2; ++y)
          if (hb + h0 + y < a.group && e < a.d)
            store_pair(out_row<T>(a, b, u, hb + h0 + y) + e, sum[y] == 0.f ? 0.f : acc[y] / sum[y],
                       sum[y] == 0.f ? 0.f : acc[2 + y] / sum[y], a.o_vec);
      } else {
#pragma unroll
        for (int y = 0; y < 4; ++y) to[((mt * NT + nt) * 4 + y) * 32 + lane] = acc[y];
        if (mt == 0 && g == 0)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            to[C::PIECE + h0 + y] = top[y];
            to[C::PIECE + C::HEADS + h0 + y] = sum[y];
          }
      }
    }
    if (began && !end && tid == 0) {     // (the last unit of the block: written after the zero above)
      const int64_t n = s_starts[b + 1] - s_starts[b];
      const int64_t stop = int64_t(s_starts[b]) * per_b + (u + 1) * n;
      a.links[blockIdx.x] = make_int2(unit, int((stop - 1) / (per * WARPS)) - int(blockIdx.x) + 1);
    }
    i0 = i1;
  }
}

// Block (c, x): tile x of O of the unit that began in block c and went on behind it.  Its warps take
// every eighth part, then the block joins the warps.
template <typename T, int DT, int NT>
__global__ void __launch_bounds__(THREADS) join_codes8_kernel(const Attend a) {
  using C = Cfg<DT, NT>;
  __shared__ float s_o[WARPS][4][32], s_m[WARPS][8], s_l[WARPS][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int mt = int(blockIdx.y) / NT, nt = int(blockIdx.y) % NT, h0 = nt * 8 + 2 * t;
  griddep_launch_dependents();
  griddep_wait();
  const int2 link = a.links[blockIdx.x];
  if (link.y == 0) return;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = warp; i < link.y; i += WARPS) {
    const float* piece =
        a.pieces + (int64_t(blockIdx.x + i) * SLOTS + (i == 0 ? AFTER : BEFORE)) * C::SLOT;
    float x[4], pm[2], pl[2];
#pragma unroll
    for (int y = 0; y < 4; ++y) x[y] = piece[((mt * NT + nt) * 4 + y) * 32 + lane];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      pm[y] = piece[C::PIECE + h0 + y];
      pl[y] = piece[C::PIECE + C::HEADS + h0 + y];
    }
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const float top = fmaxf(m[y], pm[y]), was = ex2(m[y] - base_of(top)), is = ex2(pm[y] - base_of(top));
      m[y] = top;
      l[y] = l[y] * was + pl[y] * is;
      acc[y] = acc[y] * was + x[y] * is;
      acc[2 + y] = acc[2 + y] * was + x[2 + y] * is;
    }
  }
#pragma unroll
  for (int y = 0; y < 4; ++y) s_o[warp][y][lane] = acc[y];
  if (g == 0)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      s_m[warp][2 * t + y] = m[y];
      s_l[warp][2 * t + y] = l[y];
    }
  __syncthreads();
  if (warp >= 2) return;                 // warp y: the lanes' head 2 t + y
  const int y = warp, n = min(WARPS, link.y);
  float top = -INFINITY, sum = 0.f, e0 = 0.f, e1 = 0.f;
  for (int w = 0; w < n; ++w) top = fmaxf(top, s_m[w][2 * t + y]);
  for (int w = 0; w < n; ++w) {
    const float is = ex2(s_m[w][2 * t + y] - base_of(top));
    sum += s_l[w][2 * t + y] * is;
    e0 += s_o[w][y][lane] * is;
    e1 += s_o[w][2 + y][lane] * is;
  }
  const int per_b = a.heads_kv * a.blocks, b = link.x / per_b, u = link.x - b * per_b;
  const int head = u % a.blocks * C::HEADS + h0 + y, e = element_of<DT>(mt, g);
  if (head < a.group && e < a.d)
    store_pair(out_row<T>(a, b, u, head) + e, sum == 0.f ? 0.f : e0 / sum, sum == 0.f ? 0.f : e1 / sum,
               a.o_vec);
}

// Tiles of 8 query heads that a unit takes: two for groups of more than 8, where their registers
// fit (fp32 queries and heads of 256 have as much in one).
int tiles_of(const enigma_sdpa_quantized_desc& d) {
  return d.heads_q / d.heads_kv > 8 && d.head_dim <= 128 && d.dtype == ENIGMA_DTYPE_BF16 ? 2 : 1;
}

int64_t units_of(const enigma_sdpa_quantized_desc& d) {
  const int64_t heads = 8 * tiles_of(d), group = d.heads_q / d.heads_kv;
  return d.batch * d.heads_kv * ((group + heads - 1) / heads);
}

// A block per unit, or the even split and a join.
bool whole(const enigma_sdpa_quantized_desc& d) {
  const int64_t sms = enigma::sm_count(), units = units_of(d);
  const int64_t bytes = 2 * d.head_dim * d.page * d.table_width;         // of the longest unit there may be
  return units <= sms && bytes * (sms - units) / sms <= (110 << 10);
}

size_t slot_floats(const enigma_sdpa_quantized_desc& d) {
  const size_t dt = d.head_dim <= 64 ? 64 : d.head_dim <= 128 ? 128 : 256, heads = 8 * tiles_of(d);
  return heads * dt + 2 * heads;
}

template <typename T, bool E4M3, int DT, int NT>
cudaError_t launch(const enigma_sdpa_quantized_desc& d, Attend a, cudaStream_t s) {
  using C = Cfg<DT, NT>;
  a.blocks = (a.group + C::HEADS - 1) / C::HEADS;
  a.whole = whole(d) ? 1 : 0;
  const int sms = enigma::sm_count();
  const size_t smem = size_t(WARPS) * C::RING + (a.whole ? 0 : (2 * size_t(d.batch) + 1) * 4);
  auto* kernel = attend_codes8_kernel<T, E4M3, DT, NT>;
  static std::atomic<uint64_t> ready{0};                     // devices where the attribute is set
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(dev < 64 && (ready.load() >> dev & 1))) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             WARPS * C::RING + (2 * 4096 + 1) * 4);
    if (e == cudaSuccess && dev < 64) ready.fetch_or(uint64_t(1) << dev);
  }
  if (e != cudaSuccess) return e;
  a.links = static_cast<int2*>(d.workspace);
  a.pieces = static_cast<float*>(d.workspace) + (sms * 2 + 63) / 64 * 64;
  const unsigned grid = a.whole ? unsigned(units_of(d)) : unsigned(sms);
  e = enigma::launch_dependent(kernel, grid, THREADS, smem, s, a);
  if (e != cudaSuccess || a.whole) return e;
  return enigma::launch_dependent(join_codes8_kernel<T, DT, NT>, dim3(grid, C::TILES * NT), THREADS, 0, s,
                                  a);
}

template <typename T, bool E4M3>
cudaError_t launch_sizes(const enigma_sdpa_quantized_desc& d, const Attend& a, cudaStream_t s) {
  if (d.head_dim > 128) return launch<T, E4M3, 256, 1>(d, a, s);
  if (sizeof(T) == 2 && tiles_of(d) == 2)
    return d.head_dim > 64 ? launch<__nv_bfloat16, E4M3, 128, 2>(d, a, s)
                           : launch<__nv_bfloat16, E4M3, 64, 2>(d, a, s);
  return d.head_dim > 64 ? launch<T, E4M3, 128, 1>(d, a, s) : launch<T, E4M3, 64, 1>(d, a, s);
}

}  // namespace

namespace enigma {

size_t sdpa_quantized_workspace(const enigma_sdpa_quantized_desc& d) {
  if (d.batch == 0 || whole(d)) return 0;
  const size_t sms = size_t(sm_count());
  return ((sms * 2 + 63) / 64 * 64 + sms * SLOTS * slot_floats(d)) * sizeof(float);
}

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
  a.batch = int(d.batch);
  a.heads_kv = int(d.heads_kv);
  a.group = int(d.heads_q / d.heads_kv);
  a.d = int(d.head_dim);
  a.page_shift = d.page == 16 ? 4 : d.page == 32 ? 5 : d.page == 64 ? 6 : 7;
  a.pages = int(d.pages);
  a.width = int(d.table_width);
  a.n_slots = int(d.n_slots);
  a.scale_log2 = d.scale * 1.4426950408889634f;
  const bool f32 = d.dtype == ENIGMA_DTYPE_F32, e4m3 = d.code == ENIGMA_CODE_E4M3;
  const int64_t es = f32 ? 4 : 2;
  a.q_vec = reinterpret_cast<uintptr_t>(d.q) % 16 == 0 && d.q_batch * es % 16 == 0 &&
            d.q_head * es % 16 == 0;
  a.o_vec = reinterpret_cast<uintptr_t>(d.out) % 16 == 0 && d.o_batch * es % 16 == 0 &&
            d.o_head * es % 16 == 0;
  if (f32) return e4m3 ? launch_sizes<float, true>(d, a, s) : launch_sizes<float, false>(d, a, s);
  return e4m3 ? launch_sizes<__nv_bfloat16, true>(d, a, s) : launch_sizes<__nv_bfloat16, false>(d, a, s);
}

}  // namespace enigma
