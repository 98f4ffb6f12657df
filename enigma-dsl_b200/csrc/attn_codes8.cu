// attn_codes8.cu — one new token per sequence over a paged cache held in 8-bit codes with a scale for
// each 16 tokens of a page and head (codes8.cuh):
//   out = sum_j softmax_j(c s_k(j) q . k_j) s_v(j) v_j  over the sequence's first len keys.
//
// Bound by memory: a key costs 2 D bytes and a few scales, read once for all query heads of its kv
// head.  The work is the flattened list of T entries, a unit's start and its chunks of KEYS keys, unit =
// (sequence, kv head, up to H of its query heads); warp w of W takes the contiguous range
// [w T / W, (w + 1) T / W), so every SM streams as much, whatever the lengths are.  Each warp has a ring
// of its own in shared memory that it fills with cp.async (16 bytes a lane) and empties by itself: no
// barrier until the end, and nothing to wait for but its own copies.  A unit that lies within one
// warp's range is finished there.  The others leave pieces (maximum, sum, unnormalised O): the block
// joins its warps' pieces after its only barrier, and what goes past a block's ends is joined by
// join_codes8_kernel.
// Measured, replayed from a graph: 192 contexts of 500 to 8000 keys, 8 kv heads of 128, bf16: 272 us, 6.2
// TB/s of codes and scales.  16 of 1 to 8191 keys: 33.4 us, 4.0 TB/s, of which the keys take 20; the rest
// is the launches (2 us), the ranges (2), the joins in the blocks (3) and behind them (3), and the
// first chunk's way.  64 of 2049 keys, 2 heads of 64: 11.1 us.  One of 131071, fp32: 56 us, 4.8 TB/s, bound by
// instructions: each product is made twice, P's exponentials and splits are as many as in bf16.
// The matrix instructions are the warp's, not the SM's asynchronous ones: a decode step has one to 16
// rows a key, and what counts is that codes go from their copy to an operand without another pass
// through shared memory.
//
// Both products are m16n8k16 with fp16 operands and fp32 sums, which hold every code exactly; keys
// or the head's elements are the 16-row side, the query heads (8) the narrow one:
//   S^T [keys, heads] = K Q^T,   O^T [elements, heads] += V^T P^T.
// The order of a product's inner index is free as long as both operands share it, and so is which
// rows stand where: so a lane's operands are 16 consecutive bytes of a key's row in both products,
// no fragment needs a transposing load, and V's pairs of keys are made by byte permutations before
// they are converted.  Scores take s_k in fp32, P takes s_v.
//
// bf16: O accumulates in the products' own registers.  P = exp2(s - m) s_v / v0 2^9 with a reference m
// that follows the running maximum once a score passes it by 4, and v0 the largest |s_v|, followed
// once another passes it fourfold: P < 2^15, so most chunks change no reference, need no maximum
// over the lanes and rescale nothing.  Rounding P to fp16 costs 2^-11 of the weight, or 2^-34 of a weight
// of one.  fp32: queries and P are two fp16 numbers each (2^-22), for up to 4 heads in columns beside each
// other, so that one product serves both (one context of 131071: 56 us, 65 with two products); a
// chunk's P is relative to its own largest score and s_v, times 2^15, and what brings it to the running
// maximum is applied to the chunk's product in fp32, so that small weights keep theirs whatever came
// before (2^-40 of the chunk's largest).  Queries are brought to [2^11, 2^12) by a power of two per
// head.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "codes8.cuh"

namespace {

using namespace enigma_codes8;
using namespace enigma_sm100;

template <typename T, int DT, int H>
struct Cfg {
  static constexpr int NT = (H + 7) / 8;                  // tiles of 8 columns
  // The work list's unit starts count as STARTS chunks: loading its queries and writing its result takes a
  // warp about as long (16 of 1 to 8191 keys, heads of 128: 33.4 us, 35.4 with one, 33.6 with three, but
  // 192 long contexts 0.9 % longer with three; heads of 256, 42.4, 43.8 with two).  A block gets LEAST
  // entries or more, if the list has as many: so it has a chunk, and a unit's pieces are in consecutive
  // blocks.
  static constexpr int STARTS = DT > 128 ? 4 : 2;
  static constexpr int LEAST = STARTS + 2;
  // As many warps as their registers leave room for: O, queries and a chunk's operands.  12 against 8:
  // 192 long contexts of heads of 128 272 us, 288; 16 ragged ones 33, 36; fp32 heads of 64, 47 x 4096
  // keys, 49, 54.  Two tiles of heads of 128 need 8: 42 us (64 x 4096 keys, 2 kv heads), 57 with 10.
  static constexpr int WARPS = NT == 1 && DT < 256 || DT * NT <= 128 ? 12 : 8;
  static constexpr int THREADS = WARPS * 32;
  static constexpr int SLOTS = WARPS + 2;                // pieces of a block in the workspace: its warps'
  static constexpr int BEFORE = WARPS;                   // first ones, what it has of a unit that began
  static constexpr int AFTER = WARPS + 1;                // in another block, and of one that goes on
  static constexpr int MAIN = DT < 128 ? 64 : DT;         // elements of a row's first part, and pieces of
  static constexpr int TAILS = (DT - MAIN) / 16;          // 16 behind it, which tiles hold apart
  static constexpr int KEYS = TAILS ? 32 : 4096 / DT;     // of a chunk: up to 4 KB of K, as much of V
  static constexpr int MT = KEYS / 16;                    // 16-key tiles, scale blocks
  static constexpr int TILE = KEYS * DT;                  // bytes of K or V
  static constexpr int STAGES = (192 << 10) / (WARPS * 2 * TILE);
  static constexpr int RING = STAGES * 2 * TILE;          // of a warp
  static constexpr int TILES = DT / 16;                   // 16-element tiles of O
  static constexpr int HEADS = H, COLS = 8 * NT;
  static constexpr int PIECE = (TILES * NT * 4) * 32;     // floats of O in fragment order
  static constexpr int SLOT = PIECE + 2 * COLS;           // and maxima and sums
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
  int fast;                              // rows of DT codes: copies at constant offsets
  float* pieces;                         // [block][SLOTS][SLOT]
  int2* links;                           // [block]: unit that goes on behind it, blocks it spans
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;"
               ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// The same with offsets that the instruction holds.
template <int TO, int FROM>
__device__ __forceinline__ void cp_async16_at(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0+%2], [%1+%3], 16;"
               ::"r"(dst), "l"(src), "n"(TO), "n"(FROM) : "memory");
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
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same from zero.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
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

// Where chunk c (16 bytes) of row r is in a tile (of its first part: DT is MAIN here).  Eight lanes that
// load at once must find eight different 16-byte columns of a 128-byte line: of K, lanes of two
// neighbouring rows and four neighbouring chunks; of V, of two neighbouring chunks and every second
// of eight rows.
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

// x / y, in 32 bits where that is enough (a 64-bit division takes several times as long).
__device__ __forceinline__ int64_t quotient(int64_t x, uint32_t y) {
  return x >> 32 ? x / y : int64_t(uint32_t(x) / y);
}

// A place in the work list: chunk j of the n of a unit; entries left in the warp's range.
struct Place {
  int b, u, j, n, len, left;
  const int32_t* row;                    // the sequence's table row
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

// N copies of 16 bytes a lane, STEP bytes apart in memory and, but for the swizzle's form, INTO in the tile.
template <int N, int FORMS, int STEP, int INTO, int Y = 0>
__device__ __forceinline__ void copy_rows(const uint32_t (&to)[FORMS], uint32_t plus, const uint8_t* from) {
  if constexpr (Y < N) {
    constexpr int TO = Y / FORMS * FORMS * INTO;
    cp_async16_at<TO, Y * STEP>(to[Y % FORMS] + plus, from);
    copy_rows<N, FORMS, STEP, INTO, Y + 1>(to, plus, from);
  }
}

// First element of O's tile m that lane (g, t) has, in rows g and g + 8: e and e + 1.
template <int DT>
__device__ __forceinline__ int element_of(int m, int g) {
  if (DT < 128) return m < 4 ? 8 * g + 2 * m : 16 * m + 2 * g;
  return DT == 128 || m < 8 ? 16 * g + 2 * m : 128 + 16 * g + 2 * (m - 8);
}

template <typename T>
__device__ __forceinline__ T* out_row(const Attend& a, int b, int u, int head) {
  const int kvh = u / a.blocks;
  return static_cast<T*>(a.out) + b * a.o_batch + int64_t(kvh * a.group + head) * a.o_head;
}

// What a block's warps left, in order: a warp's first piece, its last.
template <typename C>
struct Pieces {
  alignas(16) float2 ml[2 * C::WARPS][C::COLS];           // maximum, sum
  int unit[2 * C::WARPS], ends[2 * C::WARPS];            // -1: none; 1: has its unit's first key, 2: the last
  int2 at[2 * C::WARPS];                                  // sequence, and unit of the sequence
};

// T: of queries and results; DT: the head's elements, rounded up; H: query heads of a unit.
template <typename T, bool E4M3, int DT, int H>
__global__ void __launch_bounds__(Cfg<T, DT, H>::THREADS, 1)
    attend_codes8_kernel(const __grid_constant__ Attend a) {
  using C = Cfg<T, DT, H>;
  constexpr bool SPLIT = sizeof(T) == 4, BESIDE = H == 4;
  static_assert(!BESIDE || SPLIT);
  constexpr int STARTS = C::STARTS, LEAST = C::LEAST;
  constexpr int MAIN = C::MAIN, TAILS = C::TAILS, TAIL = C::KEYS * 16;   // (bytes of a tail in a tile)
  constexpr int MT = C::MT, NT = C::NT, KEYS = C::KEYS, WARPS = C::WARPS, THREADS = C::THREADS;
  constexpr int PARTS = SPLIT && !BESIDE ? 4 : 2;            // registers of an operand: inner index, two parts
  extern __shared__ __align__(128) uint8_t smem[];       // rings, list entries before each b, last chunks
  __shared__ __align__(16) float s_scale[WARPS][C::STAGES][2 * MT];
  __shared__ Pieces<C> s_pieces;
  __shared__ int s_warp[WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * C::RING;
  const uint32_t ring_at = smem_u32(ring);
  int* s_starts = reinterpret_cast<int*>(smem + WARPS * C::RING);        // [batch + 1]
  uint8_t* s_rest = reinterpret_cast<uint8_t*>(s_starts + a.batch + 1);   // [batch] keys of the last chunk
  const int per_b = a.heads_kv * a.blocks;
  griddep_launch_dependents();
  if (tid < 2 * WARPS) s_pieces.unit[tid] = -1;
  if (a.d < DT)                          // columns that no copy fills
    for (int x = tid; x < WARPS * C::RING / 16; x += THREADS)
      reinterpret_cast<uint4*>(smem)[x] = make_uint4(0, 0, 0, 0);
  griddep_wait();

  // The warp's part of the list (whole: of the block's unit, chunks alone).
  Place in;
  in.left = 0;
  int64_t total = 0, used = 1;           // entries in all, blocks that take some
  auto set_sequence = [&](Place& p) {
    p.n = s_starts[p.b + 1] - s_starts[p.b] - STARTS;
    p.len = (p.n - 1) * KEYS + s_rest[p.b];
    p.row = a.table + int64_t(a.slots ? a.slots[p.b] : p.b) * a.width;
  };
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
    in.row = a.table + int64_t(a.slots ? a.slots[in.b] : in.b) * a.width;
    in.j = int(int64_t(in.n) * warp / WARPS);
    in.left = int(int64_t(in.n) * (warp + 1) / WARPS) - in.j;
    __syncthreads();
  } else {
    int run = 0;
    for (int b0 = 0; b0 < a.batch; b0 += THREADS) {
      const int b = b0 + tid;
      int v = 0;
      if (b < a.batch) {
        const int len = len_at(a, b), n = (len + KEYS - 1) / KEYS;
        s_rest[b] = uint8_t(len - (n - 1) * KEYS);
        v = n > 0 ? n + STARTS : 0;
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
    total = int64_t(run) * per_b;
    used = max(int64_t(1), min(int64_t(gridDim.x), quotient(total, LEAST)));
    const uint32_t w = blockIdx.x * WARPS + warp, of = uint32_t(used) * WARPS;
    const int64_t each = quotient(total, of);
    const uint32_t more = uint32_t(total - each * of);       // (below of: grids are small)
    const int64_t x0 = each * w + w * more / of;
    if (blockIdx.x < used) in.left = int(each + (w + 1) * more / of - w * more / of);
    if (in.left > 0) {
      int lo = 0, hi = a.batch;          // the last b with starts[b] * per_b <= x0
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (int64_t(s_starts[mid]) * per_b <= x0) lo = mid;
        else hi = mid;
      }
      in.b = lo;
      set_sequence(in);
      const int64_t within = x0 - int64_t(s_starts[lo]) * per_b;
      in.u = int(quotient(within, in.n + STARTS));
      const int entry = int(within - int64_t(in.u) * (in.n + STARTS));
      in.j = max(entry - STARTS, 0);
      in.left -= max(STARTS - entry, 0);
    }
    // Sequences without keys are in nobody's range.
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x)
      if (s_starts[b + 1] == s_starts[b])
        for (int x = tid; x < a.heads_kv * a.group * a.d; x += THREADS)
          store1(static_cast<T*>(a.out) + b * a.o_batch + int64_t(x / a.d) * a.o_head + x % a.d, 0.f);
  }

  auto query_row = [&](const Place& p, int head) {
    const int kvh = p.u / a.blocks;
    return static_cast<const T*>(a.q) + p.b * a.q_batch +
           int64_t(kvh * a.group + (p.u - kvh * a.blocks) * C::HEADS + head) * a.q_head;
  };
  auto heads_of = [&](const Place& p) { return min(C::HEADS, a.group - p.u % a.blocks * C::HEADS); };
  // The next chunk of the range, if there is one (left > 0).
  auto advance = [&](Place& p) {
    --p.left;
    if (++p.j < p.n) return;
    p.left -= STARTS;
    if (p.left <= 0) return;
    p.j = 0;
    if (++p.u < per_b) return;
    p.u = 0;
    do ++p.b; while (s_starts[p.b + 1] == s_starts[p.b]);
    set_sequence(p);
  };

  // Asks for a chunk's codes and scales; keys behind the last and without a page are zeros.  A lane's
  // copies go to places that differ by constants, but for the swizzle, which takes two forms.
  const int page_mask = (1 << a.page_shift) - 1, parts = (page_mask + 1) / kScaleBlock;
  const int chunks = a.d >> 4;           // 16-byte chunks of a row
  constexpr int PER = MAIN / 16, ROWS = 32 / PER;              // of a row; rows that the lanes copy at once
  constexpr int FORMS = ROWS == 8 ? 1 : 8 / ROWS;            // the swizzles take the rows' low three bits
  const int lane_r = lane / PER, lane_c = lane % PER;
  uint32_t k_to[FORMS], v_to[FORMS];
#pragma unroll
  for (int y = 0; y < FORMS; ++y) {
    k_to[y] = ring_at + k_at<MAIN>(y * ROWS + lane_r, lane_c);
    v_to[y] = ring_at + C::TILE + v_at<MAIN>(y * ROWS + lane_r, lane_c);
  }
  const int lane_from = lane_r * DT + lane_c * 16;
  const uint32_t tail_to = ring_at + KEYS * MAIN + lane * 16;
  auto issue = [&](const Place& p, int stage) {
    const int kvh = p.u / a.blocks, key0 = p.j * KEYS, live = p.len - key0;
    const uint32_t to = stage * 2 * C::TILE;
    const bool one = page_mask + 1 >= KEYS;                  // all keys of the chunk in a page
    for (int i = 0; i < MT; i += one ? MT : 1) {
      const int n = one ? KEYS : 16, from0 = 16 * i, here = live - from0;
      const int page = here > 0 ? p.row[(key0 + from0) >> a.page_shift] : -1;
      const bool has = page >= 0 && page < a.pages;
      const int in_page = (key0 + from0) & page_mask;
      const int64_t at = (int64_t(kvh) * (page_mask + 1) + in_page) * a.d;
      if (a.fast && one && has && here >= KEYS) {
        const uint8_t* k = a.k + page * a.k_page + at;
        const uint8_t* v = a.v + page * a.v_page + at;
        copy_rows<KEYS / ROWS, FORMS, ROWS * DT, ROWS * MAIN>(k_to, to, k + lane_from);
        copy_rows<KEYS / ROWS, FORMS, ROWS * DT, ROWS * MAIN>(v_to, to, v + lane_from);
#pragma unroll
        for (int c = 0; c < TAILS; ++c) {                    // (chunks of 32 keys: a lane a row)
          cp_async16(tail_to + to + c * TAIL, k + lane * DT + MAIN + 16 * c, 16);
          cp_async16(tail_to + to + C::TILE + c * TAIL, v + lane * DT + MAIN + 16 * c, 16);
        }
      } else if (a.fast && has && here >= n) {
        const uint8_t* k = a.k + page * a.k_page + at;
        const uint8_t* v = a.v + page * a.v_page + at;
        copy_rows<16 / ROWS, FORMS, ROWS * DT, ROWS * MAIN>(k_to, to + from0 * MAIN, k + lane_from);
        copy_rows<16 / ROWS, FORMS, ROWS * DT, ROWS * MAIN>(v_to, to + from0 * MAIN, v + lane_from);
        if (TAILS && lane < 16)
#pragma unroll
          for (int c = 0; c < TAILS; ++c) {
            cp_async16(tail_to + to + from0 * 16 + c * TAIL, k + lane * DT + MAIN + 16 * c, 16);
            cp_async16(tail_to + to + from0 * 16 + C::TILE + c * TAIL, v + lane * DT + MAIN + 16 * c, 16);
          }
      } else {
        const uint8_t* k = a.k + (has ? page * a.k_page + at : 0);
        const uint8_t* v = a.v + (has ? page * a.v_page + at : 0);
#pragma unroll 1
        for (int r = lane_r; r < n; r += ROWS) {
          const uint32_t bytes = has && r < here ? 16 : 0;
          const int64_t from = bytes ? int64_t(r) * a.d + lane_c * 16 : 0;
          if (lane_c < chunks) {
            cp_async16(ring_at + to + k_at<MAIN>(from0 + r, lane_c), k + from, bytes);
            cp_async16(ring_at + to + C::TILE + v_at<MAIN>(from0 + r, lane_c), v + from, bytes);
          }
        }
        if (TAILS && lane < n)
#pragma unroll
          for (int c = 0; c < TAILS; ++c) {                  // (n is at most 32 here)
            const uint32_t bytes = has && lane < here ? 16 : 0;
            const int from = bytes ? lane * DT + MAIN + 16 * c : 0;
            cp_async16(tail_to + to + from0 * 16 + c * TAIL, k + from, bytes);
            cp_async16(tail_to + to + from0 * 16 + C::TILE + c * TAIL, v + from, bytes);
          }
      }
      const int x = lane % MT;
      if (lane < 2 * MT && (one || x == i)) {
        const bool is_v = lane >= MT, there = has && (one ? 16 * x < here : true);
        const int64_t where = page * (is_v ? a.vs_page : a.ks_page) + kvh * parts +
                              in_page / kScaleBlock + (one ? x : 0);
        cp_async4(smem_u32(&s_scale[warp][stage][lane]), (is_v ? a.vs : a.ks) + (there ? where : 0),
                  there ? 4 : 0);
      }
    }
  };

  uint32_t qf[NT][DT / 16][PARTS];       // queries
  float cq[NT][2];                       // what brings a head's scores to log2 units
  float m[NT][2], l[NT][2], o[C::TILES][NT][4];
  float v0 = 0.f, to_v0 = 0.f;           // bf16: O is in units of v0 2^-9, to_v0 = 2^9 / v0
  auto load_queries = [&](const Place& p) {
    const int heads = heads_of(p);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int head = BESIDE ? g & 3 : nt * 8 + g;
      const T* row = query_row(p, head);
      float x[MAIN / 64][16], tail[TAILS + 1][4];
      uint32_t top = 0;
#pragma unroll
      for (int jj = 0; jj < MAIN / 64; ++jj) {
        const int e = 64 * jj + 16 * t;
        const bool there = head < heads && e < a.d;
        if (a.q_vec) {
#pragma unroll
          for (int i = 0; i < int(sizeof(T)); ++i) {         // 16 elements: 2 or 4 times 16 bytes
            uint4 w = make_uint4(0, 0, 0, 0);
            if (there) w = *reinterpret_cast<const uint4*>(row + e + i * (16 / int(sizeof(T))));
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
#pragma unroll
      for (int c = 0; c < TAILS; ++c)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          tail[c][y] = head < heads ? float(row[MAIN + 16 * c + 4 * t + y]) : 0.f;
          top = max(top, __float_as_uint(tail[c][y]) & 0x7fffffffu);
        }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = max(27, int(top >> 23));                 // biased; 2^-100 at least
      const float up = __uint_as_float(uint32_t(127 + 127 + 11 - e) << 23);
      const float back = __uint_as_float(uint32_t(max(e - 11, 1)) << 23) * a.scale_log2;
#pragma unroll
      for (int i = 0; i < 2; ++i) cq[nt][i] = __shfl_sync(0xffffffffu, back, (2 * t + i) * 4);
      auto pack = [&](int k16, int i, float lo, float hi) {
        uint32_t rest;
        qf[nt][k16][i] = SPLIT ? split_halves(lo * up, hi * up, &rest) : pack_halves(lo * up, hi * up);
        if (BESIDE && g >= 4) qf[nt][k16][i] = rest;
        if (PARTS == 4) qf[nt][k16][(2 + i) % PARTS] = rest;
      };
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int jj = 0; jj < MAIN / 64; ++jj)
#pragma unroll
          for (int s = 0; s < 4; ++s) pack(4 * jj + s, i, x[jj][4 * s + 2 * i], x[jj][4 * s + 2 * i + 1]);
#pragma unroll
        for (int c = 0; c < TAILS; ++c) pack(MAIN / 16 + c, i, tail[c][2 * i], tail[c][2 * i + 1]);
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
    v0 = to_v0 = 0.f;
  };

  auto compute = [&](const Place& p, int stage) {
    const uint32_t kd = ring_at + stage * 2 * C::TILE, vd = kd + C::TILE;
    float sc[2 * MT];                    // s_k, s_v of the chunk's blocks
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) sc[i] = s_scale[warp][stage][i];
    float s[MT][NT][4];
    // 16 elements of tile i's keys, words x of key g and y of key g + 8.
    auto add_scores = [&](int i, int k16, uint32_t x, uint32_t y) {
      uint32_t f[4];
      halves_of4<E4M3>(x, &f[0], &f[2]);
      halves_of4<E4M3>(y, &f[1], &f[3]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (k16 == 0) mma_f16_first(s[i][nt], f, qf[nt][0][0], qf[nt][0][1]);
        else mma_f16(s[i][nt], f, qf[nt][k16][0], qf[nt][k16][1]);
        if (PARTS == 4) mma_f16(s[i][nt], f, qf[nt][k16][2 % PARTS], qf[nt][k16][3 % PARTS]);
      }
    };
#pragma unroll
    for (int jj = 0; jj < MAIN / 64; ++jj) {
      if (64 * jj >= a.d) break;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint4 x = lds128(kd + k_at<MAIN>(16 * i + g, 4 * jj + t));
        const uint4 y = lds128(kd + k_at<MAIN>(16 * i + g + 8, 4 * jj + t));
        add_scores(i, 4 * jj, x.x, y.x);
        add_scores(i, 4 * jj + 1, x.y, y.y);
        add_scores(i, 4 * jj + 2, x.z, y.z);
        add_scores(i, 4 * jj + 3, x.w, y.w);
      }
    }
#pragma unroll
    for (int c = 0; c < TAILS; ++c)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint32_t at = kd + KEYS * MAIN + c * TAIL + (16 * i + g) * 16 + 4 * t;
        add_scores(i, MAIN / 16 + c, lds32(at), lds32(at + 8 * 16));
      }
    // V's codes while the scores are weighed: keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of each tile.
    constexpr int WORDS = MAIN / 32;
    uint32_t vw[MT][4][WORDS + TAILS];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const int r = 16 * i + 2 * t + (z & 1) + 8 * (z >> 1);
        if (MAIN == 64) {
          const uint2 w = lds64(vd + v_at<MAIN>(r, g >> 1) + (g & 1) * 8);
          vw[i][z][0] = w.x;
          vw[i][z][1] = w.y;
        } else {
#pragma unroll
          for (int h = 0; h < MAIN / 128; ++h) {
            const uint4 w = lds128(vd + v_at<MAIN>(r, g + 8 * h));
            vw[i][z][(4 * h) % WORDS] = w.x;
            vw[i][z][(4 * h + 1) % WORDS] = w.y;
            vw[i][z][(4 * h + 2) % WORDS] = w.z;
            vw[i][z][(4 * h + 3) % WORDS] = w.w;
          }
        }
#pragma unroll
        for (int c = 0; c < TAILS; ++c)
          vw[i][z][WORDS + c] = lds16(vd + KEYS * MAIN + c * TAIL + r * 16 + 2 * g);
      }
    float top_v = 0.f;
#pragma unroll
    for (int i = 0; i < MT; ++i) top_v = fmaxf(top_v, fabsf(sc[MT + i]));
    // Scores in log2 units, and each lane's largest.
    float top[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const float c[2] = {sc[i] * cq[nt][0], sc[i] * cq[nt][1]};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (BESIDE) s[i][nt][x] += __shfl_xor_sync(0xffffffffu, s[i][nt][x], 2);
          s[i][nt][x] *= c[x & 1];
        }
      }
    if ((p.j + 1) * KEYS > p.len) {                          // some keys do not count
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (p.j * KEYS + 16 * i + g + 8 * x >= p.len)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[i][nt][2 * x] = s[i][nt][2 * x + 1] = -INFINITY;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        top[nt][x] = fmaxf(s[0][nt][x], s[0][nt][2 + x]);
#pragma unroll
        for (int i = 1; i < MT; ++i) top[nt][x] = fmaxf(top[nt][x], fmaxf(s[i][nt][x], s[i][nt][2 + x]));
      }
    uint32_t pf[MT][NT][PARTS];
    float fresh[NT][2];                  // fp32: what brings the chunk's product to O's units
    if (SPLIT) {
      float ratio[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const float x = sc[MT + i];
        ratio[i] = x == 0.f ? 0.f : fabsf(x) == top_v ? copysignf(1.f, x) : x / top_v;
      }
      bool grown = false;
      float shrink[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float here = max_over_keys(top[nt][x]);
          const float now = fmaxf(m[nt][x], here), base = base_of(now);
          grown |= now != m[nt][x];
          shrink[nt][x] = ex2(m[nt][x] - base);
          fresh[nt][x] = ex2(here - base);
          m[nt][x] = now;
          top[nt][x] = 15.f - base_of(here);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          float w[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            w[x] = ex2(s[i][nt][x] + top[nt][x & 1]);
            sum[x & 1] += w[x];
            w[x] *= ratio[i];
          }
          uint32_t r0, r1, h0 = split_halves(w[0], w[1], &r0), h1 = split_halves(w[2], w[3], &r1);
          if (BESIDE && t >= 2) h0 = r0, h1 = r1;
          pf[i][nt][0] = turn_8x8(h0);
          pf[i][nt][1] = turn_8x8(h1);
          if (PARTS == 4) {
            pf[i][nt][2 % PARTS] = turn_8x8(r0);
            pf[i][nt][3 % PARTS] = turn_8x8(r1);
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
    } else {
      bool past = top_v > 4.f * v0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) past |= top[nt][x] > m[nt][x] + 4.f;
      if (__any_sync(0xffffffffu, past)) {                   // new references
        float shrink[NT][2], change = 1.f;
        if (top_v > v0) {
          const float was = v0;
          v0 = fmaxf(top_v, 0x1p-100f);
          to_v0 = 512.f / v0;
          change = was / v0;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float now = fmaxf(m[nt][x], max_over_keys(top[nt][x]));
            shrink[nt][x] = ex2(m[nt][x] - base_of(now));
            m[nt][x] = now;
            l[nt][x] *= shrink[nt][x];
            shrink[nt][x] *= change;
          }
#pragma unroll
        for (int x = 0; x < C::TILES; ++x)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[x][nt][i] *= shrink[nt][i & 1];
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float base[2] = {base_of(m[nt][0]), base_of(m[nt][1])};
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const float r = sc[MT + i] * to_v0;
          float w[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            w[x] = ex2(s[i][nt][x] - base[x & 1]);
            l[nt][x & 1] += w[x];
          }
          pf[i][nt][0] = turn_8x8(pack_halves(w[0] * r, w[1] * r));
          pf[i][nt][1] = turn_8x8(pack_halves(w[2] * r, w[3] * r));
        }
      }
    }
    // A tile of O: two bytes of each key's word z.
    auto add_tile = [&](int tile, int z, uint32_t bytes) {
      float acc[NT][4];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        uint32_t f[4];
        halves_of4<E4M3>(__byte_perm(vw[i][0][z], vw[i][1][z], bytes), &f[0], &f[1]);
        halves_of4<E4M3>(__byte_perm(vw[i][2][z], vw[i][3][z], bytes), &f[2], &f[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (!SPLIT) {
            mma_f16(o[tile][nt], f, pf[i][nt][0], pf[i][nt][1]);
            continue;
          }
          if (i == 0) mma_f16_first(acc[nt], f, pf[i][nt][0], pf[i][nt][1]);
          else mma_f16(acc[nt], f, pf[i][nt][0], pf[i][nt][1]);
          if (PARTS == 4) mma_f16(acc[nt], f, pf[i][nt][2 % PARTS], pf[i][nt][3 % PARTS]);
        }
      }
      if (SPLIT)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[tile][nt][x] = fmaf(acc[nt][x], fresh[nt][x & 1], o[tile][nt][x]);
    };
#pragma unroll
    for (int z = 0; z < WORDS; ++z) {
      add_tile(2 * z, z, 0x5140);
      add_tile(2 * z + 1, z, 0x7362);
    }
#pragma unroll
    for (int c = 0; c < TAILS; ++c) add_tile(2 * WORDS + c, WORDS + c, 0x5140);
  };

  if (in.left > 0) {
    Place at = in;
    auto next = [&](int stage) {
      if (in.left > 0) {
        issue(in, stage);
        const int u = in.u, b = in.b;
        advance(in);
        if (in.left > 0 && (in.u != u || in.b != b) && g < heads_of(in))   // its queries, ahead
          for (int x = t * 64; x < a.d * int(sizeof(T)); x += 256)
            asm volatile("prefetch.global.L1 [%0];" ::"l"(reinterpret_cast<const uint8_t*>(query_row(in, g)) + x));
      }
      cp_commit();
    };
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; ++s) next(s);
    int st = 0, to = C::STAGES - 1;
    bool fresh = true, began = false;
    while (at.left > 0) {
      if (fresh) {
        load_queries(at);
        began = at.j == 0;
        fresh = false;
      }
      cp_wait<C::STAGES - 2>();
      __syncwarp();                      // every lane's copies, and nobody reads the stage before
      // (Asking for a chunk as soon as the codes before it are in registers, in the middle of a chunk's
      // work, has more in flight but is slower: 292 against 272 us for 192 long contexts.)
      next(to);
      to = to + 1 == C::STAGES ? 0 : to + 1;
      compute(at, st);
      st = st + 1 == C::STAGES ? 0 : st + 1;
      const bool end = at.j + 1 == at.n;
      const bool over = at.left - 1 - (end && !a.whole ? STARTS : 0) <= 0;
      if (end || over) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int y = 0; y < 2; ++y) l[nt][y] = sum_over_keys(l[nt][y]);
        if (BESIDE)                      // both parts of P
#pragma unroll
          for (int mt = 0; mt < C::TILES; ++mt)
#pragma unroll
            for (int y = 0; y < 4; ++y) o[mt][0][y] += __shfl_xor_sync(0xffffffffu, o[mt][0][y], 2);
        const float unit = SPLIT ? 1.f : v0 * (1.f / 512.f);
        if (began && end) {              // all of the unit
          const int heads = heads_of(at), hb = at.u % a.blocks * C::HEADS;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int head = nt * 8 + 2 * t + y;
              if (head >= heads) continue;
              T* row = out_row<T>(a, at.b, at.u, hb + head);
              const float f = l[nt][y] == 0.f ? 0.f : unit / l[nt][y];
#pragma unroll
              for (int mt = 0; mt < C::TILES; ++mt) {
                const int e = element_of<DT>(mt, g);
                if (e < a.d) store_pair(row + e, o[mt][nt][y] * f, o[mt][nt][2 + y] * f, a.o_vec);
              }
            }
        } else {
          // A first piece that others follow goes to the workspace, a last one where the copies were.
          __syncwarp();
          const int i = 2 * warp + over;
          float* to_o = over ? reinterpret_cast<float*>(ring)
                             : a.pieces + (int64_t(blockIdx.x) * C::SLOTS + warp) * C::SLOT;
#pragma unroll
          for (int mt = 0; mt < C::TILES; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int y = 0; y < 4; ++y) to_o[((mt * NT + nt) * 4 + y) * 32 + lane] = o[mt][nt][y] * unit;
          if (g == 0)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int y = 0; y < 2; ++y)
                s_pieces.ml[i][nt * 8 + 2 * t + y] = make_float2(m[nt][y], l[nt][y]);
          if (lane == 0) {
            s_pieces.unit[i] = at.b * per_b + at.u;
            s_pieces.ends[i] = (began ? 1 : 0) | (end ? 2 : 0);
            s_pieces.at[i] = make_int2(at.b, at.u);
          }
        }
        fresh = true;
      }
      advance(at);
    }
  }
  __syncthreads();

  // The pieces of each unit: to the result, or to a piece of the block's.
  if (!a.whole && tid == 0) a.links[blockIdx.x] = make_int2(0, 0);
  const int mine = lane < 2 * WARPS ? s_pieces.unit[lane] : -1;
  const uint32_t all = __ballot_sync(0xffffffffu, mine >= 0);
  float* own = a.pieces + int64_t(blockIdx.x) * C::SLOTS * C::SLOT;
  // A warp per (unit, tile of O): the lane's two heads' largest maximum, then what each piece adds.
  int turn = warp;
  for (uint32_t rest = all; rest != 0;) {
    const int first = __ffs(rest) - 1, unit = s_pieces.unit[first];
    const uint32_t these = __ballot_sync(0xffffffffu, mine == unit);
    rest &= ~these;
    const int2 where = s_pieces.at[first];
    const int b = where.x, u = where.y;
    const bool began = s_pieces.ends[first] & 1, end = s_pieces.ends[31 - __clz(these)] & 2;
    int x = turn;
    for (; x < C::TILES * NT; x += WARPS) {
      const int mt = x / NT, nt = x % NT, h0 = nt * 8 + 2 * t;
      float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f}, acc[4] = {0.f, 0.f, 0.f, 0.f};
      uint32_t bits = these;
      if (__popc(these) > 6) {           // many: all last pieces at once, those of other units as nothing
        float4 ml[WARPS];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          ml[w] = *reinterpret_cast<const float4*>(&s_pieces.ml[2 * w + 1][h0]);
          if (!(these >> (2 * w + 1) & 1)) ml[w] = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
          top[0] = fmaxf(top[0], ml[w].x);
          top[1] = fmaxf(top[1], ml[w].z);
        }
        const float base[2] = {base_of(top[0]), base_of(top[1])};
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const bool one = these >> (2 * w + 1) & 1;
          const float* po = reinterpret_cast<const float*>(smem + w * C::RING) + x * 128 + lane;
          const float f[2] = {ex2(ml[w].x - base[0]), ex2(ml[w].z - base[1])};
          sum[0] += ml[w].y * f[0];
          sum[1] += ml[w].w * f[1];
#pragma unroll
          for (int y = 0; y < 4; ++y) acc[y] += (one ? po[y * 32] : 0.f) * f[y & 1];
        }
        bits &= 0x55555555u;             // (a unit has at most one piece that others followed)
      }
      // One after the other, the next one's loads ahead.
      float v[4];
      float4 ml = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
      auto load = [&](int i) {
        const float* po = i & 1 ? reinterpret_cast<const float*>(smem + (i >> 1) * C::RING)
                                : own + (i >> 1) * C::SLOT;
#pragma unroll
        for (int y = 0; y < 4; ++y) v[y] = po[x * 128 + y * 32 + lane];
        ml = *reinterpret_cast<const float4*>(&s_pieces.ml[i][h0]);
      };
      if (bits != 0) load(__ffs(bits) - 1);
#pragma unroll 1
      while (bits != 0) {
        const float now[2] = {fmaxf(top[0], ml.x), fmaxf(top[1], ml.z)};
        const float base[2] = {base_of(now[0]), base_of(now[1])};
        const float was[2] = {ex2(top[0] - base[0]), ex2(top[1] - base[1])};
        const float is[2] = {ex2(ml.x - base[0]), ex2(ml.z - base[1])};
        sum[0] = sum[0] * was[0] + ml.y * is[0];
        sum[1] = sum[1] * was[1] + ml.w * is[1];
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[y] = acc[y] * was[y & 1] + v[y] * is[y & 1];
        top[0] = now[0];
        top[1] = now[1];
        bits &= bits - 1;
        if (bits != 0) load(__ffs(bits) - 1);
      }
      if (began && end) {
        const int hb = u % a.blocks * C::HEADS, e = element_of<DT>(mt, g);
#pragma unroll
        for (int y = 0; y < 2; ++y)
          if (h0 + y < C::HEADS && hb + h0 + y < a.group && e < a.d) {
            const float f = sum[y] == 0.f ? 0.f : 1.f / sum[y];
            store_pair(out_row<T>(a, b, u, hb + h0 + y) + e, acc[y] * f, acc[2 + y] * f, a.o_vec);
          }
      } else {
        float* to = own + (began ? C::AFTER : C::BEFORE) * C::SLOT;
#pragma unroll
        for (int y = 0; y < 4; ++y) to[x * 128 + lane + y * 32] = acc[y];
        if (mt == 0 && g == 0)
#pragma unroll
          for (int y = 0; y < 2; ++y)
            reinterpret_cast<float2*>(to + C::PIECE)[h0 + y] = make_float2(top[y], sum[y]);
      }
    }
    turn = x - C::TILES * NT;            // the warps that had nothing to do come first in the next unit
    if (began && !end && tid == 0) {     // (the last unit of the block: written after the zero above)
      const int64_t entries = s_starts[b + 1] - s_starts[b];
      const int64_t stop = int64_t(s_starts[b]) * per_b + (u + 1) * entries;
      const int last = int((stop * used - 1) / total);                   // the block that has its end
      a.links[blockIdx.x] = make_int2(unit, last - int(blockIdx.x) + 1);
    }
  }
}

// Block (c, x): tile x of O of the unit that began in block c and went on behind it.  Its warps take
// every eighth part, then the block joins the warps.
template <typename T, int DT, int H>
__global__ void __launch_bounds__(256) join_codes8_kernel(const Attend a) {
  using C = Cfg<T, DT, H>;
  constexpr int WARPS = 8, NT = C::NT;
  __shared__ float s_o[WARPS][4][32], s_m[WARPS][8], s_l[WARPS][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int mt = int(blockIdx.y) / NT, nt = int(blockIdx.y) % NT, h0 = nt * 8 + 2 * t;
  griddep_launch_dependents();
  griddep_wait();
  // The first part is asked for before it is known whether there is one.
  const int2 link = a.links[blockIdx.x];
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, acc[4] = {0.f, 0.f, 0.f, 0.f};
  float x[4], pm[2], pl[2];
  auto load = [&](int i) {
    const int block = min(int(blockIdx.x) + i, int(gridDim.x) - 1);
    const float* piece = a.pieces + (int64_t(block) * C::SLOTS + (i == 0 ? C::AFTER : C::BEFORE)) * C::SLOT;
#pragma unroll
    for (int y = 0; y < 4; ++y) x[y] = piece[((mt * NT + nt) * 4 + y) * 32 + lane];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const float2 ml = reinterpret_cast<const float2*>(piece + C::PIECE)[h0 + y];
      pm[y] = ml.x;
      pl[y] = ml.y;
    }
  };
  load(warp);
  if (link.y == 0) return;
  for (int i = warp; i < link.y;) {
    const float y0 = x[0], y1 = x[1], y2 = x[2], y3 = x[3];
    const float qm[2] = {pm[0], pm[1]}, ql[2] = {pl[0], pl[1]};
    i += WARPS;
    if (i < link.y) load(i);
    float was[2], is[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const float top = fmaxf(m[y], qm[y]);
      was[y] = ex2(m[y] - base_of(top));
      is[y] = ex2(qm[y] - base_of(top));
      m[y] = top;
      l[y] = l[y] * was[y] + ql[y] * is[y];
    }
    acc[0] = acc[0] * was[0] + y0 * is[0];
    acc[1] = acc[1] * was[1] + y1 * is[1];
    acc[2] = acc[2] * was[0] + y2 * is[0];
    acc[3] = acc[3] * was[1] + y3 * is[1];
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
  if (h0 + y < C::HEADS && head < a.group && e < a.d)
    store_pair(out_row<T>(a, b, u, head) + e, sum == 0.f ? 0.f : e0 / sum, sum == 0.f ? 0.f : e1 / sum,
               a.o_vec);
}

// Query heads that a unit takes.  16 where the group is larger than 8, so that codes are read and
// converted once for two tiles (2 kv heads for 32: 95 x 4096 keys of 128 58 us against 69, 190 of 64 57
// against 70), but where registers have no room for them: heads of 256, and fp32.  4 in fp32 where the
// group is no larger: both parts of a query and of P in one tile (one context of 131071: 56 us, 65).
int unit_heads(const enigma_sdpa_quantized_desc& d) {
  const int64_t group = d.heads_q / d.heads_kv;
  if (d.dtype == ENIGMA_DTYPE_F32) return group > 4 ? 8 : 4;
  return group > 8 && d.head_dim <= 128 ? 16 : 8;
}

int64_t units_of(const enigma_sdpa_quantized_desc& d) {
  const int64_t heads = unit_heads(d), group = d.heads_q / d.heads_kv;
  return d.batch * d.heads_kv * ((group + heads - 1) / heads);
}

// A block per unit, or the even split and a join.  The host knows the table's width, not the lengths: a
// block per unit, which saves the ranges and the joins, where the longest unit there may be is
// small, the larger the fewer SMs it leaves idle.  us, heads of 128, all of the longest length or
// of 1 to it:
//   8 units (heads of 64) of 128 KB: 7.8, 7.6 (split 8.6, 8.4); 256 KB: 10.2, 10.0 (9.0, 8.8)
//   64 of 256 KB: 11.7, 11.3 (13.3, 10.9);           512 KB: 17.0, 16.6 (15.8, 13.7)
//   128 of 512 KB: 17.8, 17.0 (21.5, 17.0);          1 MB: 29.9, 27.2 (33.8, 22.1)
bool whole(const enigma_sdpa_quantized_desc& d) {
  const int64_t sms = enigma::sm_count(), units = units_of(d);
  const int64_t bytes = 2 * d.head_dim * d.page * d.table_width;         // of the longest unit there may be
  return units <= sms && bytes * (5 * sms - 4 * units) / (5 * sms) <= (170 << 10);
}

// Calls f with the elements of a head that the kernel is made for: 80 and 96 by themselves (38 x 4096
// keys, 8 heads of 80: 58 us, 75 as heads of 128), others rounded up.
template <int H, typename F>
auto with_elements(int64_t head_dim, F f) {
  using std::integral_constant;
  if (head_dim <= 64) return f(integral_constant<int, 64>{});
  if (head_dim == 80) return f(integral_constant<int, 80>{});
  if (head_dim == 96) return f(integral_constant<int, 96>{});
  if constexpr (H <= 8)
    if (head_dim > 128) return f(integral_constant<int, 256>{});
  return f(integral_constant<int, 128>{});
}

// Calls f with the type of queries and the heads of a unit.
template <typename F>
auto with_heads(const enigma_sdpa_quantized_desc& d, F f) {
  using std::integral_constant;
  const int heads = unit_heads(d);
  if (d.dtype == ENIGMA_DTYPE_F32)
    return heads == 4 ? f(0.f, integral_constant<int, 4>{}) : f(0.f, integral_constant<int, 8>{});
  return heads == 16 ? f(__nv_bfloat16{}, integral_constant<int, 16>{})
                     : f(__nv_bfloat16{}, integral_constant<int, 8>{});
}

// Floats of the workspace that a block's pieces take.
size_t block_floats(const enigma_sdpa_quantized_desc& d) {
  return with_heads(d, [&](auto type, auto heads) {
    return with_elements<heads.value>(d.head_dim, [&](auto elements) {
      using C = Cfg<decltype(type), elements.value, heads.value>;
      return size_t(C::SLOTS) * C::SLOT;
    });
  });
}

template <typename T, bool E4M3, int DT, int H>
cudaError_t launch(const enigma_sdpa_quantized_desc& d, Attend a, cudaStream_t s) {
  using C = Cfg<T, DT, H>;
  a.blocks = (a.group + C::HEADS - 1) / C::HEADS;
  a.whole = whole(d) ? 1 : 0;
  a.fast = a.d == DT;
  const int sms = enigma::sm_count();
  const size_t smem = size_t(C::WARPS) * C::RING + (a.whole ? 0 : size_t(d.batch) * 5 + 4);
  auto* kernel = attend_codes8_kernel<T, E4M3, DT, H>;
  static std::atomic<uint64_t> ready{0};                     // devices where the attribute is set
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(dev < 64 && (ready.load() >> dev & 1))) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             C::WARPS * C::RING + 4096 * 5 + 4);
    if (e == cudaSuccess && dev < 64) ready.fetch_or(uint64_t(1) << dev);
  }
  if (e != cudaSuccess) return e;
  a.links = static_cast<int2*>(d.workspace);
  a.pieces = static_cast<float*>(d.workspace) + (sms * 2 + 63) / 64 * 64;
  const unsigned grid = a.whole ? unsigned(units_of(d)) : unsigned(sms);
  e = enigma::launch_dependent(kernel, grid, C::THREADS, smem, s, a);
  if (e != cudaSuccess || a.whole) return e;
  return enigma::launch_dependent(join_codes8_kernel<T, DT, H>, dim3(grid, C::TILES * C::NT), 256, 0, s,
                                  a);
}

template <bool E4M3>
cudaError_t launch_any(const enigma_sdpa_quantized_desc& d, const Attend& a, cudaStream_t s) {
  return with_heads(d, [&](auto type, auto heads) {
    return with_elements<heads.value>(d.head_dim, [&](auto elements) {
      return launch<decltype(type), E4M3, elements.value, heads.value>(d, a, s);
    });
  });
}

}  // namespace

namespace enigma {

size_t sdpa_quantized_workspace(const enigma_sdpa_quantized_desc& d) {
  if (d.batch == 0 || whole(d)) return 0;
  const size_t sms = size_t(sm_count());
  return ((sms * 2 + 63) / 64 * 64 + sms * block_floats(d)) * sizeof(float);
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
  return e4m3 ? launch_any<true>(d, a, s) : launch_any<false>(d, a, s);
}

}  // namespace enigma
