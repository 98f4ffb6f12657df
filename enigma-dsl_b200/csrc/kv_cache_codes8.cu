// kv_cache_codes8.cu — a paged cache in 8-bit codes: rows quantised as they are written, and read back.
//
// Codes and scales are those of codes8.cuh.  A write that starts inside a block of 16 tokens keeps
// the block's earlier tokens: the scale becomes the larger (in magnitude) of the block's and what the new
// tokens need, and if it grows the earlier codes are rounded to it.  A write that starts a block, or
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

// Elements of a row that are moved at once, 16 bytes of them.
template <typename T>
constexpr int kVec = 16 / int(sizeof(T));

// Four elements from 16 or 8 loaded bytes, from element 4 y on.
__device__ __forceinline__ void four_of(const uint4& v, int, float (&x)[4], float) {
  x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y);
  x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void four_of(const uint4& v, int y, float (&x)[4], __nv_bfloat16) {
  const uint32_t a = y ? v.z : v.x, b = y ? v.w : v.y;
  x[0] = __uint_as_float(a << 16); x[1] = __uint_as_float(a & 0xffff0000u);
  x[2] = __uint_as_float(b << 16); x[3] = __uint_as_float(b & 0xffff0000u);
}

// 16 bytes of a row, whatever its alignment.
template <typename T, bool VEC>
__device__ __forceinline__ uint4 load_vec(const T* p) {
  if (VEC) return *reinterpret_cast<const uint4*>(p);
  uint4 v;
  if (sizeof(T) == 4) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p);
    v = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    v = make_uint4(h[0] | uint32_t(h[1]) << 16, h[2] | uint32_t(h[3]) << 16, h[4] | uint32_t(h[5]) << 16,
                   h[6] | uint32_t(h[7]) << 16);
  }
  return v;
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_vec(T* p, const uint4& v) {
  if (VEC) {
    *reinterpret_cast<uint4*>(p) = v;
  } else if (sizeof(T) == 4) {
    uint32_t* w = reinterpret_cast<uint32_t*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else {
    uint16_t* h = reinterpret_cast<uint16_t*>(p);
    h[0] = uint16_t(v.x); h[1] = uint16_t(v.x >> 16); h[2] = uint16_t(v.y); h[3] = uint16_t(v.y >> 16);
    h[4] = uint16_t(v.z); h[5] = uint16_t(v.z >> 16); h[6] = uint16_t(v.w); h[7] = uint16_t(v.w >> 16);
  }
}

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

struct Rows {
  const int32_t *table, *slots, *starts, *cu;
  int64_t k_token, k_head, v_token, v_head;
  int n, tokens, heads, slots_total, pages, width, page_shift, d;
};

// An entry of a request, and its rows [first, end).
struct Entry {
  int index, slot, start, first, end;
};

// The entries of the packed rows t0 .. t0 + 15, for lanes 0 to 15 (and again for the others): a search
// for the first, then one look at it and the 31 entries behind; where more of those begin within
// these rows (empty ones may), a search for each row.
__device__ __forceinline__ Entry entries_of(const Rows& r, int t0) {
  const int lane = threadIdx.x & 31, x = lane % kScaleBlock;
  const int e0 = entry_of(r.cu, r.n, t0), j = min(e0 + lane, r.n - 1);
  const int first = r.cu[j], end = r.cu[j + 1], slot = r.slots[j], start = r.starts[j];
  int at = 0;                            // the row's entry - e0
#pragma unroll
  for (int y = 0; y < kScaleBlock; ++y) {
    const uint32_t past = __ballot_sync(0xffffffffu, lane > 0 && e0 + lane < r.n && first <= t0 + y);
    if (x == y) at = past ? 31 - __clz(past) : 0;
  }
  Entry e;
  e.index = e0 + at;
  e.first = __shfl_sync(0xffffffffu, first, at);
  e.end = __shfl_sync(0xffffffffu, end, at);
  e.slot = __shfl_sync(0xffffffffu, slot, at);
  e.start = __shfl_sync(0xffffffffu, start, at);
  if (__any_sync(0xffffffffu, at == 31)) {                   // perhaps further on
    int mine = 0;
    for (int y = 0; y < kScaleBlock; ++y) {
      const int i = entry_of(r.cu, r.n, t0 + y);
      if (x == y) mine = i;
    }
    e = {mine, r.slots[mine], r.starts[mine], r.cu[mine], r.cu[mine + 1]};
  }
  return e;
}

struct Write {
  Rows r;
  uint8_t *k, *v;                        // the layer's pages
  float *ks, *vs;                        // and scales
  const void *new_k, *new_v;
  const int32_t* refs;
  int32_t* status;
};

// The rows of one block that one entry of the request writes.
struct Part {
  int t, rows, r0;                       // first packed row, their number, first row in the block
  int entry, slot;
  int64_t block;                         // of the first head: (page * heads) * blocks of a page + block in it
  int64_t first;                         // position of the block's first row in the sequence
};

// One block of one head: what is new of it, and where it is.
template <typename T>
struct Block {
  const T* rows;                         // the first new row
  int64_t token;                         // from one row to the next
  uint8_t* codes;
  float* scale;
  int n, r0;                             // new rows, the first one's place in the block; n 0: none
};

// Blocks by P warps, of which this is the q-th: the scale that old and new rows need, and their codes.  NV:
// vectors of 16 bytes that a lane has of a block's new rows; those of all N blocks are loaded at
// once.  tops: where P > 1 warps tell each other their largest magnitude, not those of the call before.
template <typename T, bool E4M3, bool VEC, int NV, int N, int P = 1>
__device__ __forceinline__ void write_blocks(const Block<T> (&b)[N], int d, int q = 0, uint32_t* tops = nullptr) {
  static_assert(P == 1 || N == 1);
  constexpr int E = kVec<T>;
  const int lane = threadIdx.x & 31, cols = d / E, step_r = 32 / cols, step_c = 32 - step_r * cols;
  const int v_first = lane + 32 * NV * q, r_first = v_first / cols, c_first = v_first - r_first * cols;
  float held[N];
  uint4 x[N][NV];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    held[k] = b[k].r0 > 0 ? *b[k].scale : 0.f;
    int r = r_first, c = c_first;        // (a row past the last is the last again)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[k][i] = load_vec<T, VEC>(b[k].rows + max(min(r, b[k].n - 1), 0) * b[k].token + c * E);
      r += step_r;
      c += step_c;
      if (c >= cols) c -= cols, ++r;
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    if (b[k].n == 0) continue;
    uint32_t top = 0;                    // bits of the largest magnitude
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t v[4] = {x[k][i].x, x[k][i].y, x[k][i].z, x[k][i].w};
#pragma unroll
      for (int y = 0; y < 4; ++y)
        top = E == 8 ? __vmaxu2(top, v[y] & 0x7fff7fffu) : max(top, v[y] & 0x7fffffffu);
    }
    if (E == 8) top = max(top & 0xffff0000u, top << 16);
    top = __reduce_max_sync(0xffffffffu, top);
    if (P > 1) {
      if (lane == 0) tops[q] = top;
      asm volatile("bar.sync %0, %1;" ::"r"(1 + int(threadIdx.x) / (32 * P)), "n"(32 * P) : "memory");
#pragma unroll
      for (int y = 0; y < P; ++y) top = max(top, tops[y]);
    }
    // Scales compare by magnitude: a block of a cache made elsewhere may have a negative one, which stays as it
    // is where it is large enough.
    const float need = scale_of<E4M3>(top);
    const bool finite = top < 0x7f800000u && fabsf(held[k]) < INFINITY, grows = fabsf(held[k]) < need;
    const float scale = !finite ? __uint_as_float(0x7fffffffu) : grows ? need : held[k];
    const float inverse = finite ? 1.f / scale : 0.f;
    if (finite && grows) {               // (r0 = 0: there are no old rows)
      for (int w = lane + 32 * q; w < b[k].r0 * (d / 4); w += 32 * P) {
        uint32_t* word = reinterpret_cast<uint32_t*>(b[k].codes) + w;
        uint32_t lo, hi;
        halves_of4<E4M3>(*word, &lo, &hi);
        const float2 f = floats_of(lo), g = floats_of(hi);
        const float h = held[k];
        *word = codes_of<E4M3>(f.x * h, f.y * h, g.x * h, g.y * h, inverse);
      }
    }
    int r = r_first, c = c_first;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint32_t out[E / 4];
#pragma unroll
      for (int y = 0; y < E / 4; ++y) {
        float f[4];
        four_of(x[k][i], y, f, T(0.f));
        out[y] = finite ? codes_of<E4M3>(f[0], f[1], f[2], f[3], inverse) : 0u;
      }
      if (r < b[k].n) {
        uint32_t* to = reinterpret_cast<uint32_t*>(b[k].codes + (b[k].r0 + r) * d + c * E);
        if (E == 8) *reinterpret_cast<uint2*>(to) = make_uint2(out[0], out[E / 4 - 1]);
        else *to = out[0];
      }
      r += step_r;
      c += step_c;
      if (c >= cols) c -= cols, ++r;
    }
    if (lane == 0 && q == 0) *b[k].scale = scale;
  }
}

constexpr int WWARPS = 8;

// Blocks (c, y): the parts that begin in packed rows [16 c, 16 c + 16), WWARPS gridDim.y warps over their
// (part, K or V, head) triples.  A part begins with its entry, or on a block's first token.  Bound
// by memory for prompts; the request's look-ups, five loads that wait for one another, are made
// once for 16 rows, a lane each, and hidden by the other blocks of the SM.  8 heads of 128, bf16, replayed:
// 32768 tokens 40 us (5.0 TB/s of rows and codes), 8192 12.4; 256 single tokens 6.3 us, nearly all of it
// the look-ups.  4096 single tokens take 23 us, 19 without the look for clashes, which every block
// makes among all entries (47 where each slot was compared with each part).
// A block's rows of more than 8 vectors a lane are shared by P warps: their registers then leave room for as
// many warps as those of shorter rows (5448 fp32 tokens of 8 heads of 256: 23 us, 38 with a warp
// alone; but bf16 heads of 128, which fit, 45 against 42 when shared by two).
template <typename T, bool E4M3, bool VEC, int NV, int P>
__global__ void __launch_bounds__(WWARPS * 32, 32 / WWARPS) write_codes8_kernel(const __grid_constant__ Write w) {
  __shared__ Part s_part[kScaleBlock];
  __shared__ uint32_t s_found, s_twice;                    // parts there are, parts that another entry changes
  __shared__ uint32_t s_own;                               // entries from s_first on that clash with no part
  __shared__ int s_first;                                  // the block's first entry
  __shared__ int s_few;                                    // no part has more than 32 vectors: 1; 64: 2
  __shared__ uint32_t s_tops[2][WWARPS];
  __shared__ __align__(16) uint32_t s_slots[128];          // bit s % 4096: slot s may be a part's
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t0 = int(blockIdx.x) * kScaleBlock;
  const int threads = int(blockDim.x), warps = threads >> 5;
  const Rows& r = w.r;
  const int page = 1 << r.page_shift, per_page = page / kScaleBlock;
  griddep_launch_dependents();
  griddep_wait();
  // Entries' slots that a thread loads at once, at first while the parts are looked up.  (Four: 4096 single tokens
  // 22.9 against 23.4 us, 1024 9.0 both, but 16 prompts written and read 48.3 against 47.9.)
  constexpr int AHEAD = 2;
  int slots[AHEAD];
  auto load_slots = [&](int j) {         // (an entry past the last is the last again)
#pragma unroll
    for (int y = 0; y < AHEAD; ++y) slots[y] = r.slots[min(j + y * threads, r.n - 1)];
  };
  if (r.n > 1) load_slots(threadIdx.x);
  if (warp == 0) {
    const int x = lane % kScaleBlock, t = t0 + x;
    reinterpret_cast<uint4*>(s_slots)[lane] = make_uint4(0, 0, 0, 0);
    __syncwarp();
    const Entry e = entries_of(r, t0);
    int fail = 0;
    Part p;
    bool found = false;
    if (t < r.tokens && lane < kScaleBlock) {
      const int first = e.first, end = min(e.end, r.tokens);
      p.slot = e.slot;
      const int64_t pos = int64_t(e.start) + t - first;
      if (t < first || t >= end || p.slot < 0 || p.slot >= r.slots_total || pos < 0 ||
          pos >> r.page_shift >= r.width)
        fail = ENIGMA_CACHE_BAD_REQUEST;
      p.t = t;
      p.r0 = int(pos & (kScaleBlock - 1));
      p.rows = min(kScaleBlock - p.r0, end - t);
      p.entry = e.index;
      p.first = pos - p.r0;
      if (fail == 0 && (t == max(first, 0) || p.r0 == 0)) {              // else in the middle of a part
        const int at = r.table[int64_t(p.slot) * r.width + (pos >> r.page_shift)];
        if (at < 0 || at >= r.pages) fail = ENIGMA_CACHE_BAD_REQUEST;
        else if (w.refs[at] > 1) fail = ENIGMA_CACHE_SHARED;
        found = fail == 0;
        p.block = int64_t(at) * r.heads * per_page + (pos & (page - 1)) / kScaleBlock;
      }
      if (fail != 0) atomicOr(w.status, fail);
    }
    const uint32_t all = __ballot_sync(0xffffffffu, found);
    if (found) {
      s_part[__popc(all & ((1u << lane) - 1u))] = p;
      if (r.n > 1) atomicOr(&s_slots[p.slot >> 5 & 127], 1u << (p.slot & 31));
    }
    // Parts of one slot are of one entry as a rule, which clashes with none of them then.
    const int e0 = __shfl_sync(0xffffffffu, e.index, 0);
    uint32_t own = 0;
    if (r.n > 1) {
      const uint32_t by_slot = __match_any_sync(0xffffffffu, found ? p.slot : -1 - lane);
      const uint32_t by_entry = __match_any_sync(0xffffffffu, found ? p.entry : -1 - lane);
      own = __reduce_or_sync(0xffffffffu, found && by_slot == by_entry && p.entry - e0 < 32
                                              ? 1u << (p.entry - e0) : 0u);
    }
    const uint32_t longest = __reduce_max_sync(0xffffffffu, found ? uint32_t(p.rows * r.d) : 0u);
    if (lane == 0) {
      s_found = (1u << __popc(all)) - 1u;
      s_twice = 0;
      s_own = own;
      s_first = e0;
      s_few = longest <= 32 * kVec<T> ? 1 : longest <= 64 * kVec<T> ? 2 : 0;
    }
  }
  __syncthreads();
  const int parts = __popc(s_found);
  // Another entry of the same slot that touches the block would change it at the same time.
  if (r.n > 1) {
    for (int j0 = threadIdx.x; j0 < r.n;) {
#pragma unroll
      for (int y = 0; y < AHEAD; ++y) {
        const int j = j0 + y * threads, slot = slots[y];
        if (j >= r.n || !(s_slots[slot >> 5 & 127] >> (slot & 31) & 1)) continue;
        if (uint32_t(j - s_first) < 32 && (s_own >> (j - s_first) & 1)) continue;
#pragma unroll 1
        for (int x = 0; x < parts; ++x)
          if (s_part[x].slot == slot && s_part[x].entry != j) {
            const int64_t s = r.starts[j], e = s + r.cu[j + 1] - int64_t(r.cu[j]);
            if (s < e && s < s_part[x].first + kScaleBlock && e > s_part[x].first) {
              atomicOr(&s_twice, 1u << x);
              atomicOr(w.status, ENIGMA_CACHE_BAD_REQUEST);
            }
          }
      }
      j0 += AHEAD * threads;
      if (j0 < r.n) load_slots(j0);
    }
    __syncthreads();
  }
  const uint32_t found = s_found & ~s_twice;
  const int units = parts * 2 * r.heads;
  auto block_of = [&](int u) {
    Block<T> b;
    const int x = min(u, units - 1) / (2 * r.heads), rest = min(u, units - 1) - x * 2 * r.heads;
    const int head = rest >> 1;
    const Part& p = s_part[x];
    const bool is_v = rest & 1;
    const int64_t block = p.block + int64_t(head) * per_page;
    b.token = is_v ? r.v_token : r.k_token;
    b.rows = static_cast<const T*>(is_v ? w.new_v : w.new_k) + p.t * b.token +
             head * (is_v ? r.v_head : r.k_head);
    b.codes = (is_v ? w.v : w.k) + block * kScaleBlock * r.d;
    b.scale = (is_v ? w.vs : w.ks) + block;
    b.n = u < units && (found >> x & 1) ? p.rows : 0;
    b.r0 = p.r0;
    return b;
  };
  if (units == 0) return;
  const int stride = warps * int(gridDim.y), u0 = int(blockIdx.y) * warps + warp;
  if (s_few == 1) {                      // single tokens: four blocks at once, a vector a lane
    for (int u = u0; u < units; u += 4 * stride) {
      const Block<T> b[4] = {block_of(u), block_of(u + stride), block_of(u + 2 * stride),
                             block_of(u + 3 * stride)};
      write_blocks<T, E4M3, VEC, 1, 4>(b, r.d);
    }
  } else if (s_few == 2) {
    for (int u = u0; u < units; u += 2 * stride) {
      const Block<T> b[2] = {block_of(u), block_of(u + stride)};
      write_blocks<T, E4M3, VEC, 2, 2>(b, r.d);
    }
  } else {
    int turn = 0;
    for (int u = u0 / P; u < units; u += stride / P) {       // (P divides `warps`)
      const Block<T> b[1] = {block_of(u)};
      write_blocks<T, E4M3, VEC, NV, 1, P>(b, r.d, warp % P, &s_tops[turn][warp / P * P]);
      if (b[0].n > 0) turn ^= 1;         // (where the warps met)
    }
  }
}

struct Read {
  Rows r;
  const uint8_t *k, *v;
  const float *ks, *vs;
  void *out_k, *out_v;
  const int32_t* lens;
};

// Blocks (c, y): packed rows [16 c, 16 c + 16): their look-ups as above, then a warp per row or piece of
// one, its lanes along the heads, READ vectors of K and of V at once.  Rows before the first entry and
// behind the last are left as they were, a token that the slot does not hold is zeros.  Bound by memory:
// 32768 tokens of 8 heads of 128, bf16, 36 us (5.6 TB/s of codes and rows), 8192 9.0; 256 single tokens
// 4.5 us, the look-ups.
template <typename T, bool E4M3, bool VEC, int READ>
__global__ void __launch_bounds__(WWARPS * 32) read_codes8_kernel(const __grid_constant__ Read w) {
  constexpr int E = kVec<T>;
  __shared__ int64_t s_line[kScaleBlock];                  // of the first head: page * heads * page size + row
  __shared__ int s_kind[kScaleBlock];                      // 0: no row, 1: zeros, 2: a token
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t0 = int(blockIdx.x) * kScaleBlock;
  const Rows& r = w.r;
  const int page = 1 << r.page_shift, per_page = page / kScaleBlock;
  griddep_launch_dependents();
  griddep_wait();
  if (warp == 0) {
    const int t = t0 + lane % kScaleBlock;
    const Entry e = entries_of(r, t0);
    if (lane < kScaleBlock) {
      int kind = 0;
      if (t < r.tokens && t >= e.first && t < e.end) {
        const int slot = e.slot;
        const int64_t pos = int64_t(e.start) + t - e.first;
        kind = 1;
        if (slot >= 0 && slot < r.slots_total && pos >= 0 && pos >> r.page_shift < r.width) {
          const int at = r.table[int64_t(slot) * r.width + (pos >> r.page_shift)];
          if (pos < w.lens[slot] && at >= 0 && at < r.pages) {
            kind = 2;
            s_line[lane] = int64_t(at) * r.heads * page + (pos & (page - 1));
          }
        }
      }
      s_kind[lane] = kind;
    }
  }
  __syncthreads();
  const int cols = r.d / E, items = r.heads * cols, step_h = 32 / cols, step_c = 32 - step_h * cols;
  const int h_first = lane / cols, c_first = lane - h_first * cols;
  const int pieces = (items + 32 * READ - 1) / (32 * READ) * kScaleBlock;          // of all rows: K and V together
  for (int i = int(blockIdx.y) * WWARPS + warp; i < pieces; i += WWARPS * int(gridDim.y)) {
    const int x = i % kScaleBlock, kind = s_kind[x];
    if (kind == 0) continue;
    const int t = t0 + x;
    const int64_t line = kind == 2 ? s_line[x] : 0;
    const uint8_t* codes[2] = {w.k + line * r.d, w.v + line * r.d};
    const float* scales[2] = {w.ks + line / kScaleBlock, w.vs + line / kScaleBlock};   // (pages are whole blocks)
    T* out[2] = {static_cast<T*>(w.out_k) + t * r.k_token, static_cast<T*>(w.out_v) + t * r.v_token};
    const int64_t out_head[2] = {r.k_head, r.v_head};
    int h0 = h_first, c0 = c_first;
    if (i >= kScaleBlock) {
      const int first = i / kScaleBlock * 32 * READ + lane;
      h0 = first / cols;
      c0 = first - h0 * cols;
    }
    int h = h0, c = c0;
    uint32_t code[2][READ][E / 4];
    float scale[2][READ];
#pragma unroll
    for (int y = 0; y < READ; ++y) {                       // (a head past the last is the last again)
      const int head = min(h, r.heads - 1);
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const uint32_t* from = reinterpret_cast<const uint32_t*>(codes[z] + int64_t(head) * page * r.d + c * E);
        if (E == 8) {
          const uint2 v = *reinterpret_cast<const uint2*>(from);
          code[z][y][0] = v.x;
          code[z][y][E / 4 - 1] = v.y;
        } else {
          code[z][y][0] = *from;
        }
        scale[z][y] = scales[z][head * per_page];
      }
      h += step_h;
      c += step_c;
      if (c >= cols) c -= cols, ++h;
    }
    h = h0;
    c = c0;
#pragma unroll
    for (int y = 0; y < READ; ++y) {
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        uint32_t words[4];
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
          uint32_t lo, hi;
          halves_of4<E4M3>(code[z][y][i], &lo, &hi);
          const float2 a = floats_of(lo), b = floats_of(hi);
          const float f = scale[z][y];
          if (E == 8) {
            words[(2 * i) & 3] = pack_bf16x2(a.x * f, a.y * f);
            words[(2 * i + 1) & 3] = pack_bf16x2(b.x * f, b.y * f);
          } else {
            words[0] = __float_as_uint(a.x * f);
            words[1] = __float_as_uint(a.y * f);
            words[2] = __float_as_uint(b.x * f);
            words[3] = __float_as_uint(b.y * f);
          }
        }
        uint4 v = make_uint4(words[0], words[1], words[2], words[3]);
        if (kind == 1) v = make_uint4(0, 0, 0, 0);
        if (h < r.heads) store_vec<T, VEC>(out[z] + h * out_head[z] + c * E, v);
      }
      h += step_h;
      c += step_c;
      if (c >= cols) c -= cols, ++h;
    }
  }
}

// Rows that can be moved 16 bytes at a time.
bool vectors(const enigma_kv_cache_rows& w) {
  const int64_t all = w.k_token | w.k_head | w.v_token | w.v_head, es = w.dtype == ENIGMA_DTYPE_F32 ? 4 : 2;
  return aligned(w.k, 16) && aligned(w.v, 16) && all * es % 16 == 0;
}

Rows rows_of(const enigma_kv_cache_desc& c, const enigma_kv_cache_rows& w) {
  Rows r;
  r.table = c.table;
  r.slots = w.slots;
  r.starts = w.starts;
  r.cu = w.cu;
  r.k_token = w.k_token;
  r.k_head = w.k_head;
  r.v_token = w.v_token;
  r.v_head = w.v_head;
  r.n = int(w.n);
  r.tokens = int(w.tokens);
  r.heads = int(c.heads_kv);
  r.slots_total = int(c.slots);
  r.pages = int(c.pages);
  r.width = int(c.table_width);
  r.page_shift = c.page == 16 ? 4 : c.page == 32 ? 5 : c.page == 64 ? 6 : 7;
  r.d = int(c.head_dim);
  return r;
}

// Blocks that share a column, 16 packed rows whose look-ups each of them makes: one where the columns alone
// fill the GPU with `per_sm` blocks an SM, else as many as fill it, or twice as many where a warp
// still has two of the column's `tasks` then; never more than have one of at most `most`, nor more than
// eight whose warps then have four or less.  (8192 tokens, 8 heads of 128, written: 12.3 us with one, 12.5 with
// two; 4096: 10.4, 8.0, four 8.4; 8192 tokens of 32 heads read: 42, 38; 5448 fp32 tokens of 8 heads of
// 256 written: 32, 27, three 24; 64 single tokens of 2 heads of 64: 7.3, 5.8, eight 5.0; 256 of 8 of 128: 18,
// 11, eight 6.4, 32 7.1.)
dim3 shared(int64_t columns, int64_t per_sm, int64_t tasks, int64_t most) {
  const int64_t fill = enigma::sm_count() * per_sm / columns;
  const int64_t twice = std::min(tasks / (2 * WWARPS), enigma::sm_count() * per_sm * 2 / columns);
  const int64_t enough = std::min(most / WWARPS, std::max<int64_t>(8, most / (4 * WWARPS)));
  const int64_t share = std::max<int64_t>(1, std::max(std::min(enough, fill), twice));
  return dim3(unsigned(columns), unsigned(std::min<int64_t>(share, 65535)));
}

template <typename T, bool E4M3, bool VEC>
cudaError_t launch_write(const Write& w, cudaStream_t s) {
  const int vectors = w.r.d * int(sizeof(T)) / 32;         // of a lane, if a warp has all of 16 new rows
  const int warps = vectors <= 8 ? 1 : vectors <= 16 ? 2 : 4;
  const int64_t columns = (int64_t(w.r.tokens) + kScaleBlock - 1) / kScaleBlock;
  // (Part, K or V, head) triples of a column: where it is one part, and where the entries are as short as they
  // may be and begin anywhere.
  const int64_t units = int64_t(2) * w.r.heads * warps;
  const int64_t parts = w.r.n == 1 ? 1 : std::min<int64_t>(kScaleBlock, 2 + w.r.n / columns);
  const dim3 grid = shared(columns, 4, units, units * parts);
  // Long requests take blocks of 4 warps, of which fewer wait for the look-ups: 32768 tokens of 2 heads of 64
  // 8.8 us, 12.9 with 8, of 8 heads of 128 40, 42; but 12000 21 against 17.
  const unsigned threads = columns > enigma::sm_count() * 12 ? 128 : 256;
  auto* kernel = vectors <= 4    ? write_codes8_kernel<T, E4M3, VEC, 4, 1>
                 : vectors == 5  ? write_codes8_kernel<T, E4M3, VEC, 5, 1>             // (heads of 80)
                 : warps == 1    ? write_codes8_kernel<T, E4M3, VEC, 8, 1>
                 : vectors == 10 ? write_codes8_kernel<T, E4M3, VEC, 5, 2>
                                 : write_codes8_kernel<T, E4M3, VEC, 8, 2>;
  if constexpr (sizeof(T) == 4)
    if (warps == 4) kernel = write_codes8_kernel<T, E4M3, VEC, 8, 4>;
  return enigma::launch_dependent(kernel, grid, threads, 0, s, w);
}

template <typename T, bool E4M3, bool VEC>
cudaError_t launch_read(const Read& w, cudaStream_t s) {
  const int64_t columns = (int64_t(w.r.tokens) + kScaleBlock - 1) / kScaleBlock;
  const int64_t items = int64_t(w.r.heads) * w.r.d / kVec<T>;            // of a row
  // Vectors of a lane at once: no more than there are, and as many bytes of codes in flight in fp32 (4096
  // tokens of 8 heads of 128 9.3 us, 11.6 with 4; bf16, 32768 tokens, 36 us, 53 with 8).
  int at_once = items <= 32 ? 1 : 4;
  auto* kernel = at_once == 1 ? read_codes8_kernel<T, E4M3, VEC, 1> : read_codes8_kernel<T, E4M3, VEC, 4>;
  if constexpr (sizeof(T) == 4)
    if (items > 128) {
      kernel = read_codes8_kernel<T, E4M3, VEC, 8>;
      at_once = 8;
    }
  const int64_t pieces = kScaleBlock * ((items + 32 * at_once - 1) / (32 * at_once));
  return enigma::launch_dependent(kernel, shared(columns, at_once == 1 ? 8 : 4, pieces, pieces), 256, 0, s, w);
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

cudaError_t kv_cache_q8_write(const enigma_kv_cache_q8_desc& d, const enigma_kv_cache_rows& rows,
                              cudaStream_t s) {
  note_kernel("write_codes8_kernel");
  const enigma_kv_cache_desc& c = d.cache;
  const int64_t blocks = c.pages * c.heads_kv * (c.page / kScaleBlock);       // of a layer
  Write w;
  w.r = rows_of(c, rows);
  w.k = static_cast<uint8_t*>(c.k) + rows.layer * blocks * kScaleBlock * c.head_dim;
  w.v = static_cast<uint8_t*>(c.v) + rows.layer * blocks * kScaleBlock * c.head_dim;
  w.ks = d.k_scale + rows.layer * blocks;
  w.vs = d.v_scale + rows.layer * blocks;
  w.new_k = rows.k;
  w.new_v = rows.v;
  w.refs = c.refs;
  w.status = c.status;
  const bool vec = vectors(rows), e4m3 = d.code == ENIGMA_CODE_E4M3;
  using B = __nv_bfloat16;
  if (rows.dtype == ENIGMA_DTYPE_F32)
    return e4m3 ? (vec ? launch_write<float, true, true>(w, s) : launch_write<float, true, false>(w, s))
                : (vec ? launch_write<float, false, true>(w, s) : launch_write<float, false, false>(w, s));
  return e4m3 ? (vec ? launch_write<B, true, true>(w, s) : launch_write<B, true, false>(w, s))
              : (vec ? launch_write<B, false, true>(w, s) : launch_write<B, false, false>(w, s));
}

cudaError_t kv_cache_q8_read(const enigma_kv_cache_q8_desc& d, const enigma_kv_cache_rows& rows,
                             cudaStream_t s) {
  note_kernel("read_codes8_kernel");
  const enigma_kv_cache_desc& c = d.cache;
  const int64_t blocks = c.pages * c.heads_kv * (c.page / kScaleBlock);
  Read w;
  w.r = rows_of(c, rows);
  w.k = static_cast<const uint8_t*>(c.k) + rows.layer * blocks * kScaleBlock * c.head_dim;
  w.v = static_cast<const uint8_t*>(c.v) + rows.layer * blocks * kScaleBlock * c.head_dim;
  w.ks = d.k_scale + rows.layer * blocks;
  w.vs = d.v_scale + rows.layer * blocks;
  w.out_k = rows.k;
  w.out_v = rows.v;
  w.lens = c.lens;
  const bool vec = vectors(rows), e4m3 = d.code == ENIGMA_CODE_E4M3;
  using B = __nv_bfloat16;
  if (rows.dtype == ENIGMA_DTYPE_F32)
    return e4m3 ? (vec ? launch_read<float, true, true>(w, s) : launch_read<float, true, false>(w, s))
                : (vec ? launch_read<float, false, true>(w, s) : launch_read<float, false, false>(w, s));
  return e4m3 ? (vec ? launch_read<B, true, true>(w, s) : launch_read<B, true, false>(w, s))
              : (vec ? launch_read<B, false, true>(w, s) : launch_read<B, false, false>(w, s));
}

}  // namespace enigma
