// attn_paged.cu — one new token per sequence over a paged cache with a shared prefix.
//
// The prefix is a matrix product: all sequences' heads of a kv head's group against the same
// keys (attn_tc.cuh, split over the keys so that every SM has a part).  Each sequence's own
// keys are read once for few rows, which is bound by memory: paged_decode_kernel streams them.
// Both leave partial results (maximum, sum, unnormalised O); paged_join_kernel joins them.
#include <algorithm>
#include <mutex>
#include <new>

#include "attn_tc.cuh"

namespace {

using namespace enigma_tc;

// ============================================================================ own keys
// The work is the flattened list of (unit, 64-key chunk) pairs, unit = (sequence, kv head, block
// of up to 16 query heads); CTA c of P takes the contiguous range [c T / P, (c + 1) T / P), so
// every SM streams the same number of chunks whatever the lengths are.  A producer warp loads
// chunks by TMA (one box per page and 64 columns) into a ring; two warps take 32 keys each of
// the even chunks, two of the odd ones.  Both products have the keys or the elements as the
// 16-row operand and the heads, at most 16, as the 8-column one: S^T = K Q^T, O^T += V^T P^T with
// P^T's fragments turned by movmatrix.  For up to 8 heads that is half the products and half the
// registers of the form with the heads as rows (128 sequences of 1 to 1024 keys, 32 / 8 heads of
// 128: 52.9 -> 50.4 us, 5.3 TB/s; next to a shared prefix, where it has a third of the SMs, 32768
// shared keys and those: 117.5 -> 109.5).  Statistics and O in fp32; P is rounded to bf16,
// as the product takes it, its sum is of the unrounded values.  At the end of a unit's run of
// chunks each warp stores its state, in slot (c + u) * 4 + warp (segments in order advance c or
// u, so the slots are distinct): merging the warps first would cost two barriers and a second pass
// per run, four partials of a few KB next to a run's 100 KB and more of K and V cost less.
constexpr int CHUNK = 64;
constexpr int DWARPS = 4;
constexpr int DTHREADS = (DWARPS + 1) * 32;
constexpr int WKEYS = 32;                    // keys of a chunk that one warp takes
constexpr int ROWS = 16;                     // query heads of a unit
constexpr int PAGES = 128;                   // page numbers looked up at once

template <int D>
struct DCfg {
  static constexpr int ATOMS = D / 64;
  static constexpr int TILE = CHUNK * D * 2;            // one of K or V
  static constexpr int CTAS = D == 64 ? 3 : 2;            // on an SM, with STAGES each
  static constexpr int STAGES = 4 - D / 128;
  static constexpr int DEEP = D == 64 ? 12 : 6;           // one CTA on an SM
};

struct DecodeParams {
  const __nv_bfloat16* q;
  int64_t q_batch, q_head;
  const int32_t *table, *lens, *slots;
  int batch, heads_kv, group, blocks, rows;  // blocks of `rows` <= 16 heads per group
  int width, n_slots, pages, page_shift, box_shift, prefix, base;
  int fold;                                  // the prefix's keys are read here too
  // DIRECT: where the result goes; or, part: one partial result per unit, slot = unit
  __nv_bfloat16* out;
  int64_t o_batch, o_head;
  int part;
  float scale_log2;
  float* opart;                              // [slot][rows][D]
  float2* ml;                                // [slot][rows]
  int32_t* starts;                           // [batch + 1] chunks (of one unit) before b
  uint32_t* status;
  int stages;
};

// Element c (16 bytes) of row r in a 128-byte-swizzled tile.
__device__ __forceinline__ uint32_t sw128(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turn_8x8(uint32_t x) {   // an 8 x 8 fragment, transposed
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Sum over the lanes that hold the same heads.
__device__ __forceinline__ float over_keys(float x) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
// Barrier over the DWARPS consumer warps; whether all say yes.
__device__ __forceinline__ bool warps_all(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %1, 0;\n\t"
      "barrier.cta.red.and.pred b, 1, %2, a;\n\tselp.u32 %0, 1, 0, b;\n\t}"
      : "=r"(all) : "r"(ok ? 1u : 0u), "n"(DWARPS * 32) : "memory");
  return all != 0;
}

// floor(n c / P) for n c < 2^53 without a 64-bit division.
__device__ __forceinline__ int64_t share(int64_t n, int64_t c, int64_t P) {
  const int64_t x = n * c;
  int64_t q = int64_t(double(x) / double(P));
  if ((q + 1) * P <= x) ++q;
  if (q * P > x) --q;
  return q;
}

// The CTA that owns chunk x of T over P CTAs.
__device__ __forceinline__ int owner(int64_t x, int64_t T, int64_t P) {
  return int(((x + 1) * P - 1) / T);
}

// Chunks of a sequence: of the prefix, if it is read here, then of its own keys (from `base`, the
// prefix's end rounded down to a chunk).
__device__ __forceinline__ int prefix_chunks(const DecodeParams& p, int len) {
  return p.fold ? (min(len, p.prefix) + CHUNK - 1) / CHUNK : 0;
}
__device__ __forceinline__ int chunks_of(const DecodeParams& p, int len) {
  return prefix_chunks(p, len) + (len > p.prefix ? (len - p.base + CHUNK - 1) / CHUNK : 0);
}

// Chunk j of a sequence: its first key, and the keys [lo, hi) that count.
struct Chunk {
  int key0, lo, hi, seq;       // seq: whose table row holds its pages
};
__device__ __forceinline__ Chunk chunk_at(const DecodeParams& p, int b, int len, int np, int j) {
  Chunk c;                     // np: chunks of the prefix
  if (j < np) {
    c.key0 = j * CHUNK;
    c.lo = 0;
    c.hi = min(len, p.prefix);
    c.seq = 0;
  } else {
    c.key0 = p.base + (j - np) * CHUNK;
    c.lo = p.prefix;
    c.hi = len;
    c.seq = b;
  }
  return c;
}

// Where the prefix kernel left the partial results of sequence b's heads of kv head kvh: n rows of
// its [slot][128], `step` apart; head h of the group is row at + h.
struct PrefixRows {
  int64_t at;
  int n, step;
};
__device__ __forceinline__ PrefixRows prefix_rows(int splits, int tokens, int row_tiles, int pairs,
                                                  int group, int b, int kvh) {
  PrefixRows r = {0, 0, 0};
  if (splits == 0) return r;
  const int tile = b / tokens, pair = tile >> 1;
  const bool alt = 2 * pair + 1 >= row_tiles;
  r.n = alt ? 2 * splits : splits;
  r.step = (alt ? 1 : 2) * BM;
  r.at = (int64_t(kvh * pairs + pair) * splits * 2 + (alt ? 0 : (tile & 1))) * BM +
         (b - tile * tokens) * group;
  return r;
}

// A run of one unit's chunks.
struct Segment {
  int b, kvh, block, unit;
  int j0, n;                    // first chunk within the unit, number of chunks
};

// The segment that begins at chunk x of the CTA's range [x, end).  starts[b] * units_per_b is
// the first chunk of sequence b.
__device__ __forceinline__ Segment segment_at(const int* starts, int batch, int per_b, int blocks,
                                              int64_t x, int64_t end) {
  int lo = 0, hi = batch;       // the last b with starts[b] * per_b <= x
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (int64_t(starts[mid]) * per_b <= x) lo = mid;
    else hi = mid;
  }
  Segment s;
  s.b = lo;
  const int n = starts[lo + 1] - starts[lo];
  const int64_t in_b = x - int64_t(starts[lo]) * per_b;
  const int u = int(in_b / n);
  s.j0 = int(in_b - int64_t(u) * n);
  s.kvh = u / blocks;
  s.block = u - s.kvh * blocks;
  s.unit = lo * per_b + u;
  s.n = int(min(int64_t(n - s.j0), end - x));
  return s;
}

// DIRECT: a CTA per unit, which writes the final result, or the unit's one partial result; no
// work list.  NT: tiles of 8 heads.
template <int D, bool DIRECT, int NT>
__global__ void __launch_bounds__(DTHREADS, DCfg<D>::CTAS)
paged_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const DecodeParams p) {
  using C = DCfg<D>;
  const int ST = p.stages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  int* s_starts = reinterpret_cast<int*>(ring + ST * 2 * C::TILE);    // [batch + 1]
  int* s_len = s_starts + p.batch + 1;                                // [batch]
  __shared__ uint64_t full[C::DEEP][2], empty[C::DEEP];   // a stage's chunks for either team
  __shared__ float s_m[DWARPS][ROWS], s_l[DWARPS][ROWS];    // DIRECT
  __shared__ int s_warp[DWARPS + 1], s_pages[PAGES];
  __shared__ int s_loads;                    // chunks asked for, when the producer is done; else -1
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t most = int64_t(p.width) << p.page_shift;
  griddep_launch_dependents();

  if (tid == 0) s_loads = -1;
  if (tid < ST) {
    mbar_init(&full[tid][0], 1);
    mbar_init(&full[tid][1], 1);
    mbar_init(&empty[tid], 2);               // the chunk's two warps
    fence_barrier_init();
  }
  if (tid == DWARPS * 32) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  const int per_b = p.heads_kv * p.blocks;
  int64_t c0 = 0, c1 = 0;
  Segment unit = {};                         // DIRECT: unit blockIdx.x
  int unit_len = 0;
  if (DIRECT) {
    unit.b = int(blockIdx.x) / per_b;
    const int u = int(blockIdx.x) - unit.b * per_b;
    unit.kvh = u / p.blocks;
    unit.block = u - unit.kvh * p.blocks;
    unit_len = len_of(p.lens, p.slots, p.n_slots, most, unit.b);
    unit.n = chunks_of(p, unit_len);
    c1 = unit.n;
    if (unit.n == 0) {                       // no keys: zeros, or a part that says so
      const int rows = min(p.rows, p.group - unit.block * p.rows);
      if (p.part) {
        if (tid < rows) p.ml[int64_t(blockIdx.x) * p.rows + tid] = make_float2(-INFINITY, 0.f);
        griddep_wait();
        return;
      }
      __nv_bfloat16* to = p.out + unit.b * p.o_batch +
                          int64_t(unit.kvh * p.group + unit.block * p.rows) * p.o_head;
      for (int x = tid; x < rows * (D / 8); x += DTHREADS)
        *reinterpret_cast<uint4*>(to + x / (D / 8) * p.o_head + x % (D / 8) * 8) =
            make_uint4(0, 0, 0, 0);
      return;
    }
    __syncthreads();
  } else {
    // Chunk counts before each sequence.
    int run = 0;
    for (int b0 = 0; b0 < p.batch; b0 += DTHREADS) {
      const int b = b0 + tid;
      int v = 0;
      if (b < p.batch) {
        const int len = len_of(p.lens, p.slots, p.n_slots, most, b);
        s_len[b] = len;
        v = chunks_of(p, len);
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
      for (int w = 0; w < warp; ++w) before += s_warp[w];
      if (b < p.batch) s_starts[b] = before + x - v;
      for (int w = 0; w <= DWARPS; ++w) run += s_warp[w];
      __syncthreads();
    }
    if (tid == 0) s_starts[p.batch] = run;
    __syncthreads();
    if (blockIdx.x == 0)
      for (int b = tid; b <= p.batch; b += DTHREADS) p.starts[b] = s_starts[b];
    const int64_t T = int64_t(run) * per_b;
    const int64_t P = min(int64_t(gridDim.x), T);
    // This kernel reads nothing of the prefix kernel's, with which it shares the SMs, but the join
    // waits only for this one: so it ends after that one.
    if (int64_t(blockIdx.x) >= P) {
      griddep_wait();
      return;
    }
    c0 = share(T, blockIdx.x, P);
    c1 = share(T, int64_t(blockIdx.x) + 1, P);
  }
  auto segment = [&](int64_t at) {
    return DIRECT ? unit : segment_at(s_starts, p.batch, per_b, p.blocks, at, c1);
  };

  if (warp == DWARPS) {
    // ---------------------------------------------------------------- producer
    // One lane issues all boxes of a chunk; each lane its own was no faster.
    const int per_shift = 6 - p.box_shift, per = 1 << per_shift;   // boxes per chunk
    const int ahead = PAGES >> per_shift;                            // chunks looked up at once
    // Stages, parities and places in the look-up are counted on: a division here, in a warp with
    // nothing else to run, holds up every chunk (16 sequences of 512 shared keys, 8 kv heads of 128:
    // 14.6 us with five of them, 12.3 without).
    int st = 0, wraps = 0, team = 0;
    for (int64_t at = c0; at < c1;) {
      const Segment s = segment(at);
      const int len = DIRECT ? unit_len : s_len[s.b], np = prefix_chunks(p, len);
      int in = ahead;
      for (int j = s.j0; j < s.j0 + s.n; ++j) {
        const Chunk c = chunk_at(p, s.b, len, np, j);
        const int key0 = c.key0;
        const int boxes = (min(CHUNK, c.hi - key0) + (1 << p.box_shift) - 1) >> p.box_shift;
        // Page numbers of the next `ahead` chunks at once: one look-up per chunk, even if made a
        // chunk ahead, leaves the ring waiting for the table's latency.
        if (in == ahead) {
          in = 0;
          __syncwarp();
#pragma unroll
          for (int y = 0; y < PAGES; y += 32) {
            const int jj = j + ((y + lane) >> per_shift);
            if (jj < s.j0 + s.n) {
              const Chunk cc = chunk_at(p, s.b, len, np, jj);
              const int key = cc.key0 + (((y + lane) & (per - 1)) << p.box_shift);
              s_pages[y + lane] = page_at(p.table, p.slots, p.n_slots, p.width, p.pages, cc.seq,
                                          key >> p.page_shift);
            }
          }
          __syncwarp();
        }
        if (!__all_sync(0xffffffffu, mbar_wait(&empty[st], (wraps & 1) ^ 1, p.status))) {
          at = c1;
          break;
        }
        uint64_t* bar = &full[st][team];
        if (elect_one()) {
          mbar_arrive_expect_tx(bar, (uint32_t(2 * boxes * C::ATOMS) * 128u) << p.box_shift);
          for (int x = 0; x < boxes; ++x) {
            const int page = s_pages[in * per + x];
            const int row = (key0 + (x << p.box_shift)) & ((1 << p.page_shift) - 1);
            uint8_t* dst = ring + 2 * st * C::TILE + ((x << p.box_shift) * 128);
#pragma unroll
            for (int a = 0; a < C::ATOMS; ++a) {
              tma_load_4d(dst + a * CHUNK * 128, &tmK, bar, a * 64, row, s.kvh, page);
              tma_load_4d(dst + C::TILE + a * CHUNK * 128, &tmV, bar, a * 64, row, s.kvh, page);
            }
          }
        }
        __syncwarp();
        ++in;
        team ^= 1;
        if (++st == ST) st = 0, ++wraps;
      }
      at += s.n;
    }
    if (lane == 0) *static_cast<volatile int*>(&s_loads) = wraps * ST + st;
    griddep_wait();
    return;
  }

  // ------------------------------------------------------------------ consumers
  // A wait ran out (status is set): the copies in flight land before the block ends.
  auto give_up = [&] {
    int loads = -1;
    for (uint32_t i = 0; i < kSpinLimit && loads < 0; ++i) {
      loads = *static_cast<volatile int*>(&s_loads);
      if ((i & 1023u) == 1023u) __nanosleep(64);
    }
    for (int n = max(0, loads - ST); n < loads; ++n) {
      const int uses = ST % 2 == 0 ? n / ST : n / ST >> 1;  // of this barrier before (see below)
      mbar_drain(&full[n % ST][n & 1], uses & 1);
    }
  };
  const int g = lane >> 2, quad = lane & 3;
  const int team = warp >> 1;                               // takes every second chunk
  int turn = 0, st = -1, wraps = 0;                         // whose chunk is next, its stage
  for (int64_t at = c0; at < c1;) {
    const Segment s = segment(at);
    const int len = DIRECT ? unit_len : s_len[s.b], np = prefix_chunks(p, len);
    const int rows = min(p.rows, p.group - s.block * p.rows);
    uint32_t q[D / 16][NT][2];                              // Q^T: head g, elements 2 quad ..
    {
      const __nv_bfloat16* qb = p.q + s.b * p.q_batch +
                                int64_t(s.kvh * p.group + s.block * p.rows) * p.q_head;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = t * 8 + g, d = kk * 16 + quad * 2 + e * 8;
            q[kk][t][e] =
                row < rows ? *reinterpret_cast<const uint32_t*>(qb + row * p.q_head + d) : 0u;
          }
    }
    // A lane's heads: t * 8 + 2 quad + {0, 1}; of O^T the elements dd * 16 + g + {0, 8}.
    float o[D / 16][NT][4];
#pragma unroll
    for (int dd = 0; dd < D / 16; ++dd)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[dd][t][e] = 0.f;
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) m[t][h] = -INFINITY, l[t][h] = 0.f;
    bool ok = true;
    for (int j = s.j0; j < s.j0 + s.n; ++j) {
      if (++st == ST) st = 0, ++wraps;
      turn ^= 1;
      if ((turn ^ 1) != team) continue;
      // A team sees its own chunks only, so each has its own barrier per stage: the parity of
      // one that also counted the other team's could be a phase old.
      const int uses = ST % 2 == 0 ? wraps : wraps >> 1;    // of this barrier before
      ok = __all_sync(0xffffffffu, mbar_wait(&full[st][team], uses & 1, p.status));
      if (!ok) break;
      uint8_t* tile_k = ring + 2 * st * C::TILE;
      uint8_t* tile_v = tile_k + C::TILE;
      const Chunk ch = chunk_at(p, s.b, len, np, j);
      const int row0 = (warp & 1) * WKEYS;                  // this warp's first row of the chunk
      const int key0 = ch.key0 + row0;
      float sc[WKEYS / 16][NT][4];                          // S^T: keys g and g + 8 of each 16
#pragma unroll
      for (int n = 0; n < WKEYS / 16; ++n)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[n][t][e] = 0.f;
      const int mi = lane >> 3, mr = lane & 7;              // ldmatrix: matrix, row
      const uint32_t ka = smem_u32(tile_k);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int n = 0; n < WKEYS / 16; ++n) {
          uint32_t a[4];
          ldsm_x4(ka + (kk / 4) * CHUNK * 128 +
                      sw128(row0 + n * 16 + (mi & 1) * 8 + mr, (kk % 4) * 2 + (mi >> 1)), a);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_16816(sc[n][t], a, q[kk][t][0], q[kk][t][1]);
        }
      if (key0 + WKEYS > ch.hi || key0 < ch.lo) {           // warp-uniform
#pragma unroll
        for (int n = 0; n < WKEYS / 16; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + n * 16 + g + (e >> 1) * 8;
#pragma unroll
            for (int t = 0; t < NT; ++t)
              if (key >= ch.hi || key < ch.lo) sc[n][t][e] = -INFINITY;
          }
        // Rows past the end hold whatever the page or the ring held, rows of the prefix
        // whatever this sequence's page has there: 0 * NaN must not be.
        for (int x = lane; x < WKEYS * 8 * C::ATOMS; x += 32) {
          const int row = (x >> 3) % WKEYS;
          if (key0 + row >= ch.hi || key0 + row < ch.lo)
            *reinterpret_cast<uint4*>(tile_v + x / (WKEYS * 8) * CHUNK * 128 +
                                      (row0 + row) * 128 + (x & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();                           // before the next TMA write here
        __syncwarp();
      }
      float mc[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = m[t][h];
#pragma unroll
          for (int n = 0; n < WKEYS / 16; ++n) mx = max3f(mx, sc[n][t][h], sc[n][t][2 + h]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          mc[t][h] = mx == -INFINITY ? 0.f : mx * p.scale_log2;
          const float f = ex2(m[t][h] * p.scale_log2 - mc[t][h]);   // m = -inf: 0
          m[t][h] = mx;
          l[t][h] *= f;
          if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll
            for (int dd = 0; dd < D / 16; ++dd) {
              o[dd][t][h] *= f;
              o[dd][t][2 + h] *= f;
            }
          }
        }
      const uint32_t va = smem_u32(tile_v);
#pragma unroll
      for (int n = 0; n < WKEYS / 16; ++n) {
        uint32_t pb[NT][2];                                 // P^T: head g, keys 2 quad .. and + 8
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float e0 = ex2(fmaf(sc[n][t][2 * e], p.scale_log2, -mc[t][0]));
            const float e1 = ex2(fmaf(sc[n][t][2 * e + 1], p.scale_log2, -mc[t][1]));
            l[t][0] += e0;                                  // this lane's share of the sums
            l[t][1] += e1;
            pb[t][e] = turn_8x8(pack_bf16x2(e0, e1));
          }
#pragma unroll
        for (int dd = 0; dd < D / 16; ++dd) {
          uint32_t a[4];
          ldsm_x4_trans(va + (dd / 4) * CHUNK * 128 +
                            sw128(row0 + n * 16 + (mi >> 1) * 8 + mr, (dd % 4) * 2 + (mi & 1)), a);
#pragma unroll
          for (int t = 0; t < NT; ++t) mma_16816(o[dd][t], a, pb[t][0], pb[t][1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
    if (DIRECT) {
      // The ring is idle once every warp is here: it takes the warps' states, each thread sums
      // two columns of a row over the warps, in their order.
      if (!warps_all(ok)) return give_up();
      constexpr int LD = D + 4;                             // a store's 32 lanes meet 32 banks
      float* s_o = reinterpret_cast<float*>(ring);          // [DWARPS][NT * 8][LD]
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = t * 8 + quad * 2 + h;
          const float sum = over_keys(l[t][h]);
          if (g == 0) {
            s_m[warp][row] = m[t][h] == -INFINITY ? (sum == 0.f ? -INFINITY : 0.f)
                                                  : m[t][h] * p.scale_log2;
            s_l[warp][row] = sum;
          }
          if (row >= rows) continue;
#pragma unroll
          for (int dd = 0; dd < D / 16; ++dd)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              s_o[(warp * NT * 8 + row) * LD + dd * 16 + g + e * 8] = o[dd][t][2 * e + h];
        }
      warps_all(true);
      for (int x = tid; x < rows * (D / 4); x += DWARPS * 32) {
        const int row = x / (D / 4), d = x % (D / 4) * 4;
        float M = s_m[0][row];
#pragma unroll
        for (int w = 1; w < DWARPS; ++w) M = fmaxf(M, s_m[w][row]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float L = 0.f;
#pragma unroll
        for (int w = 0; w < DWARPS; ++w) {
          if (s_m[w][row] == -INFINITY) continue;           // saw no key: o is not written
          const float f = ex2(s_m[w][row] - M);
          const float4 v = *reinterpret_cast<const float4*>(s_o + (w * NT * 8 + row) * LD + d);
          acc.x = fmaf(v.x, f, acc.x);
          acc.y = fmaf(v.y, f, acc.y);
          acc.z = fmaf(v.z, f, acc.z);
          acc.w = fmaf(v.w, f, acc.w);
          L = fmaf(s_l[w][row], f, L);
        }
        if (p.part) {
          const int64_t at_part = int64_t(blockIdx.x) * p.rows + row;
          *reinterpret_cast<float4*>(p.opart + at_part * D + d) = acc;
          if (d == 0) p.ml[at_part] = make_float2(M, L);
        } else {
          const float inv = L == 0.f ? 0.f : 1.f / L;
          const int64_t at_out = s.b * p.o_batch +
                                 int64_t(s.kvh * p.group + s.block * p.rows + row) * p.o_head + d;
          *reinterpret_cast<uint2*>(p.out + at_out) = make_uint2(
              pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
        }
      }
      return;
    }
    if (!ok) return give_up();
    const int64_t slot = (int64_t(blockIdx.x) + s.unit) * DWARPS + warp;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = t * 8 + quad * 2 + h;
        const float sum = over_keys(l[t][h]);
        if (row >= rows) continue;
        // None of its keys: only says so.  (Nothing but NaN scores: a sum of NaN, no maximum.)
        const bool none = m[t][h] == -INFINITY && sum == 0.f;
        if (g == 0)
          p.ml[slot * p.rows + row] =
              none ? make_float2(-INFINITY, 0.f)
                   : make_float2(m[t][h] == -INFINITY ? 0.f : m[t][h] * p.scale_log2, sum);
        if (none) continue;
        float* to = p.opart + (slot * p.rows + row) * D + g;
#pragma unroll
        for (int dd = 0; dd < D / 16; ++dd)
#pragma unroll
          for (int e = 0; e < 2; ++e) to[dd * 16 + e * 8] = o[dd][t][2 * e + h];
      }
    at += s.n;
  }
}

// ============================================================================ join
struct JoinParams {
  __nv_bfloat16* out;
  int64_t o_batch, o_head;
  int batch, heads_q, heads_kv, group;
  // prefix: pairs x splits items, two states each (0 splits: no prefix)
  const float* p_opart;                    // [slot][D / 8][128][8]
  const float2* p_ml;
  int pairs, splits, row_tiles, tokens;
  // own keys
  const float* d_opart;
  const float2* d_ml;
  const int32_t* starts;                   // NULL: one part per unit
  int blocks, rows, ctas;
};

// Joins a row's partial results,
//   O = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i, M = max_i m_i (m in log2 units),
// the prefix's in their order, then the own ones.  It is all latency (L2 answers in half a
// microsecond): 16 parts' rows are in flight together, the first 16 already beside their (m, l).  A
// part that saw no key (m = -inf) may hold anything.  A warp per (sequence, query head) where a row
// has a few dozen parts; WARPS of them, joined in their order, where few rows have hundreds (one
// sequence of 22250 keys, 15 / 3 heads of 64, 600 parts a row: 68 -> 14 us;
// two of 40000 shared keys, 8 / 1 heads of 128: 38 -> 18).
constexpr int kManyParts = 48, kJoinWarps = 16;

template <int D, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32) paged_join_kernel(const JoinParams p) {
  constexpr int V = D / 32, BATCH = 16;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t id = WARPS == 1 ? blockIdx.x * 4 + warp : blockIdx.x;   // batch * heads_q < 2^28
  if (id >= uint32_t(p.batch) * uint32_t(p.heads_q)) return;
  const int b = int(id / uint32_t(p.heads_q)), h = int(id - uint32_t(b) * uint32_t(p.heads_q));
  const int kvh = h / p.group, gh = h - kvh * p.group;
  const PrefixRows pr = prefix_rows(p.splits, p.tokens, p.row_tiles, p.pairs, p.group, b, kvh);
  const int64_t p_at = pr.at + gh;
  const float* p_from = p.p_opart + p_at / BM * BM * D + (lane * V / 8 * BM + p_at % BM) * 8 +
                        lane * V % 8;
  const int per_b = p.heads_kv * p.blocks, block = gh / p.rows, u = kvh * p.blocks + block;
  const int64_t unit = int64_t(b) * per_b + u;
  int n_d = 1;
  int64_t d_at = unit * p.rows + (gh - block * p.rows);
  griddep_wait();
  if (p.starts != nullptr) {
    // The slots of the CTAs that hold the unit's chunks.
    const int64_t T = int64_t(p.starts[p.batch]) * per_b;
    const int start = p.starts[b], chunks = p.starts[b + 1] - start;
    n_d = 0;
    if (chunks > 0) {
      const int64_t x0 = int64_t(start) * per_b + int64_t(u) * chunks;
      const int64_t P = min(int64_t(p.ctas), T);
      const int first = owner(x0, T, P), last = owner(x0 + chunks - 1, T, P);
      n_d = (last - first + 1) * DWARPS;
      d_at = (int64_t(first) + unit) * DWARPS * p.rows + (gh - block * p.rows);
    }
  }
  // This warp's parts [i0, i0 + n).
  const int all = pr.n + n_d;
  const int per = WARPS == 1 ? all : (all + WARPS * BATCH - 1) / (WARPS * BATCH) * BATCH;
  const int i0 = WARPS == 1 ? 0 : warp * per, n = min(all - i0, per);
  auto row_at = [&](int i) {                       // row of part i in its workspace
    return i < pr.n ? p_at + int64_t(i) * pr.step : d_at + int64_t(i - pr.n) * p.rows;
  };
  auto ml_at = [&](int i) { return __ldcg((i0 + i < pr.n ? p.p_ml : p.d_ml) + row_at(i0 + i)); };
  float v[BATCH][V];
  auto fetch = [&](int base) {
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      if (base + u >= n) break;
      const int i = i0 + base + u;
      const float* from = i < pr.n ? p_from + int64_t(i) * pr.step * D
                                   : p.d_opart + row_at(i) * D + lane * V;
      if constexpr (V == 4) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(from));
        v[u][0] = x.x, v[u][1] = x.y, v[u][2] = x.z, v[u][3] = x.w;
      } else {
        const float2 x = __ldcg(reinterpret_cast<const float2*>(from));
        v[u][0] = x.x, v[u][1] = x.y;
      }
    }
  };
  fetch(0);
  float2 mine = lane < n ? ml_at(lane) : make_float2(-INFINITY, 0.f);
  float M = mine.x;
  for (int i = lane + 32; i < n; i += 32) M = fmaxf(M, ml_at(i).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  float acc[V] = {}, l = 0.f, w = 0.f;
  for (int base = 0; base < n; base += BATCH) {
    if (base > 0) fetch(base);
    if (base % 32 == 0) {
      if (base > 0) mine = base + lane < n ? ml_at(base + lane) : make_float2(-INFINITY, 0.f);
      w = mine.x == -INFINITY ? 0.f : ex2(mine.x - M);
      if (w != 0.f) l = fmaf(w, mine.y, l);        // this lane's parts
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const float f = __shfl_sync(0xffffffffu, w, (base + u) & 31);
      if (base + u < n && f != 0.f) {
#pragma unroll
        for (int x = 0; x < V; ++x) acc[x] = fmaf(v[u][x], f, acc[x]);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if constexpr (WARPS > 1) {
    __shared__ float s_m[WARPS], s_l[WARPS], s_acc[WARPS][D];
    if (lane == 0) s_m[warp] = M, s_l[warp] = l;
#pragma unroll
    for (int x = 0; x < V; ++x) s_acc[warp][lane * V + x] = acc[x];
    __syncthreads();
    if (warp > 0) return;
    for (int y = 1; y < WARPS; ++y) M = fmaxf(M, s_m[y]);
    l = 0.f;
#pragma unroll
    for (int x = 0; x < V; ++x) acc[x] = 0.f;
    for (int y = 0; y < WARPS; ++y) {
      if (s_m[y] == -INFINITY) continue;           // no key among its parts
      const float f = ex2(s_m[y] - M);
      l = fmaf(s_l[y], f, l);
#pragma unroll
      for (int x = 0; x < V; ++x) acc[x] = fmaf(s_acc[y][lane * V + x], f, acc[x]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __nv_bfloat16* out = p.out + b * p.o_batch + h * p.o_head + lane * V;
#pragma unroll
  for (int x = 0; x < V; x += 2)
    *reinterpret_cast<uint32_t*>(out + x) = pack_bf16x2(acc[x] * inv, acc[x + 1] * inv);
}

// ============================================================================ host
bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// The tensor-core kernels take bf16 heads of 64 or 128 whose rows TMA can address (base and
// strides multiples of 16 bytes), and a group that fits a tile.
bool tc_takes(const enigma_sdpa_shared_prefix_desc& d) {
  const int64_t st[6] = {d.q_batch, d.q_head, d.o_batch, d.o_head, d.k_page, d.v_page};
  for (int i = 0; i < 6; ++i)
    if (st[i] % 8 != 0 || st[i] <= 0 || st[i] >= (int64_t(1) << 39)) return false;
  return d.dtype == ENIGMA_DTYPE_BF16 && (d.head_dim == 64 || d.head_dim == 128) &&
         d.heads_q / d.heads_kv <= BM && aligned_to(d.q, 16) && aligned_to(d.k_pages, 16) &&
         aligned_to(d.v_pages, 16) && aligned_to(d.out, 16);
}

int log2_of(int64_t x) {
  int n = 0;
  while ((int64_t(1) << n) < x) ++n;
  return n;
}

constexpr int64_t kFoldBytes = 128ll << 20, kDirectKeys = 1536;
// Work of less is done one after the other: two streams cost four more host calls, 10 us.  (32
// sequences, 4096 shared and up to 512 own keys, 8 kv heads of 128: 19 us side by side, 26 one after
// the other; 128, 32768 and 1024: 104 / 129; 8, 2048 and 128: 12.1 / 13.4.)
constexpr double kBesideUs = 3.0, kStepUs = 1.9;

struct Layout {
  int group, tokens, row_tiles, pairs, splits, prefix;    // prefix part
  int blocks, rows, ctas;                                 // own part
  bool fold, direct, beside;
  size_t p_opart, p_ml, d_opart, d_ml, starts, total;     // byte offsets
};

Layout layout_of(const enigma_sdpa_shared_prefix_desc& d) {
  Layout y = {};
  const int sms = enigma::sm_count();
  y.group = int(d.heads_q / d.heads_kv);
  y.tokens = std::max(1, BM / y.group);
  // One sequence shares its prefix with nobody.
  y.prefix = d.batch > 1 ? int(d.prefix_len) : 0;
  y.row_tiles = int((d.batch + y.tokens - 1) / y.tokens);
  y.pairs = (y.row_tiles + 1) / 2;
  const int tiles = (y.prefix + BN - 1) / BN;
  // Short rows (by the table's width: lengths are on the device): one CTA per unit reads all its
  // keys, the prefix's too, and writes the result; no second launch, no partial results.  Measured (graph, us, so / with the prefix apart): 4 x 512
  // shared keys, 2 kv heads of 64: 7.4 / 11.3; 16 x 512, 8 of 128: 8.2 / 12.1; 32 x 1024: 13.3 /
  // 15.8; with longer rows a CTA's chain of chunks is what lasts: 8 x 1400: 13.7 / 11.7 (two launches
  // more, 4 us of the host), 8 x 2048: 17.4 / 14.1, 8 x 2048, 2 of 64: 15.3 / 11.2.
  const int64_t most = d.table_width * d.page;
  y.fold = y.prefix > 0 && most <= kDirectKeys &&
           d.batch * y.prefix * d.heads_kv * d.head_dim * 4 <= kFoldBytes;
  // A CTA per unit reads the own keys where no row has room for many of them; else they are split over
  // the SMs (32 x 4096 shared and up to 512 own keys in a table of 4608: 19.5 us, of 8192: 37).  Where the prefix is apart, a third launch joins the parts of both.
  y.direct = y.fold || most - y.prefix <= kDirectKeys;
  y.blocks = (y.group + ROWS - 1) / ROWS;
  y.rows = (y.group + y.blocks - 1) / y.blocks;
  const int64_t d_units = d.batch * d.heads_kv * y.blocks;
  if (tiles > 0 && !y.fold) {
    // The prefix is bound by the tensor cores, the own keys by memory, which a few SMs can keep
    // busy: so each gets SMs by its work, side by side.  A step of the prefix (128 keys for 256 rows)
    // takes 1.9 us; an SM draws 0.06 MB/us of own keys beside it, of which half of what the table has
    // room for is taken as the number, and 0.3 us go to a unit's start.  The number of parts, of two
    // tiles or more, is the one whose later end is the earliest; over nine shapes, each table as wide
    // as its longest sequence, within 1 % (6 % at most) of the best number measured for each, SMs in
    // proportion to the two works 7 % (13 %).
    const int64_t units = int64_t(d.heads_kv) * y.pairs;
    const double own = double(d_units) * 0.3 + double(d.batch * d.heads_kv) *
                                                   double(most - y.prefix) / 2 *
                                                   double(d.head_dim) * 4 / 6e4;
    const int limit = int(std::max<int64_t>(1, std::min<int64_t>(sms / units, (tiles + 1) / 2)));
    const double half = (y.row_tiles % 2) * 0.5;              // an odd tile fills half an item
    y.beside = y.direct &&
               (kStepUs * double(d.heads_kv) * tiles * (y.pairs - half) + own) / sms > kBesideUs;
    y.splits = limit;
    if (y.beside) {
      double best = INFINITY;
      for (int n = 1; n <= limit && n * units < sms; ++n) {
        const double end = std::max(kStepUs * double((tiles + n - 1) / n), own / double(sms - n * units));
        if (end < best) best = end, y.splits = n;
      }
    }
  }
  const int64_t p_slots = int64_t(d.heads_kv) * y.pairs * y.splits * 2;
  y.ctas = y.direct ? int(d_units) : sms * (d.head_dim == 64 ? DCfg<64>::CTAS : DCfg<128>::CTAS);
  const int64_t d_slots = !y.direct      ? (int64_t(y.ctas) + d_units) * DWARPS
                          : y.splits > 0 ? d_units
                                         : 0;
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t here = at;
    at += (size_t(bytes) + 255) & ~size_t(255);
    return here;
  };
  y.p_opart = take(p_slots * BM * d.head_dim * 4);
  y.p_ml = take(p_slots * BM * 8);
  y.d_opart = take(d_slots * y.rows * d.head_dim * 4);
  y.d_ml = take(d_slots * y.rows * 8);
  y.starts = take(y.direct ? 0 : (d.batch + 1) * 4);
  y.total = at;
  return y;
}

bool pages_map(CUtensorMap* m, const void* base, const enigma_sdpa_shared_prefix_desc& d,
               int64_t page_stride, int box_rows) {
  const cuuint64_t dims[4] = {cuuint64_t(d.head_dim), cuuint64_t(d.page), cuuint64_t(d.heads_kv),
                              cuuint64_t(d.pages)};
  const cuuint64_t strides[3] = {cuuint64_t(d.head_dim * 2), cuuint64_t(d.page * d.head_dim * 2),
                                 cuuint64_t(page_stride * 2)};
  const cuuint32_t box[4] = {64, cuuint32_t(box_rows), 1, 1};
  return make_map(m, base, 4, dims, strides, box);
}

// A second stream and the events for a fork to it and back; one call holds it at a time.  A stream
// that joined a capture belongs to it until the capture ends, so captured calls have their own: a
// call outside the capture, or in another one, must not meet it.
struct Side {
  cudaStream_t stream;
  cudaEvent_t fork, back;
  Side* next;
};
std::mutex side_mu;
Side* side_free[64][2];                                     // by device; not captured, captured

class SideHold {
 public:
  ~SideHold() {
    if (side_ == nullptr) return;
    std::lock_guard<std::mutex> lk(side_mu);
    side_->next = *list_;
    *list_ = side_;
  }
  // For work that goes back to stream s.
  cudaError_t take(cudaStream_t s) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && dev >= 64) e = cudaErrorInvalidDevice;
    if (e != cudaSuccess) return e;
    cudaStreamCaptureStatus state;
    unsigned long long id = 0;
    e = cudaStreamGetCaptureInfo(s, &state, &id);
    if (e != cudaSuccess) return e;
    const bool captured = state != cudaStreamCaptureStatusNone;
    list_ = &side_free[dev][captured];
    {
      std::lock_guard<std::mutex> lk(side_mu);
      for (Side** at = list_; *at != nullptr; at = &(*at)->next) {
        if (captured) {                                     // free, or in the same capture
          unsigned long long its = 0;
          if (cudaStreamGetCaptureInfo((*at)->stream, &state, &its) != cudaSuccess ||
              (state != cudaStreamCaptureStatusNone && its != id))
            continue;
        }
        side_ = *at;
        *at = side_->next;
        return cudaSuccess;
      }
    }
    Side* made = new (std::nothrow) Side{};
    if (made == nullptr) return cudaErrorMemoryAllocation;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // this is no part of a capture
    cudaThreadExchangeStreamCaptureMode(&mode);
    e = cudaStreamCreateWithFlags(&made->stream, cudaStreamNonBlocking);
    if (e == cudaSuccess) e = cudaEventCreateWithFlags(&made->fork, cudaEventDisableTiming);
    if (e == cudaSuccess) e = cudaEventCreateWithFlags(&made->back, cudaEventDisableTiming);
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (e == cudaSuccess) {
      side_ = made;
      return e;
    }
    if (made->fork != nullptr) cudaEventDestroy(made->fork);
    if (made->stream != nullptr) cudaStreamDestroy(made->stream);
    delete made;
    return e;
  }
  const Side& operator*() const { return *side_; }

 private:
  Side* side_ = nullptr;
  Side** list_ = nullptr;
};

template <int D>
cudaError_t launch(const enigma_sdpa_shared_prefix_desc& d, cudaStream_t s) {
  const Layout y = layout_of(d);
  uint8_t* ws = static_cast<uint8_t*>(d.workspace);
  uint32_t* status = enigma::device_status();
  if (status == nullptr) return cudaErrorMemoryAllocation;      // the bounded waits need it
  const int box_rows = int(std::min<int64_t>(d.page, 64));
  CUtensorMap mk, mv;
  if (!pages_map(&mk, d.k_pages, d, d.k_page, box_rows) ||
      !pages_map(&mv, d.v_pages, d, d.v_page, box_rows))
    return cudaErrorInvalidValue;
  const float scale_log2 = d.scale * 1.4426950408889634f;
  const int page_shift = log2_of(d.page), box_shift = log2_of(box_rows);
  cudaError_t e;
  SideHold side;
  if (y.beside) {
    e = side.take(s);
    if (e == cudaSuccess) e = cudaEventRecord((*side).fork, s);
    if (e != cudaSuccess) return e;
  }
  if (y.splits > 0) {
    CUtensorMap mq;
    const cuuint64_t dims[3] = {cuuint64_t(D), cuuint64_t(d.heads_q), cuuint64_t(d.batch)};
    const cuuint64_t strides[2] = {cuuint64_t(d.q_head * 2), cuuint64_t(d.q_batch * 2)};
    const cuuint32_t box[3] = {64, cuuint32_t(y.group), cuuint32_t(y.tokens)};
    if (!make_map(&mq, d.q, 3, dims, strides, box)) return cudaErrorInvalidValue;
    e = prepare_kernel<D, true>();
    if (e != cudaSuccess) return e;
    Params p = {};
    p.scale_log2 = scale_log2;
    p.group = y.group;
    p.tokens = y.tokens;
    p.status = status;
    p.opart = reinterpret_cast<float*>(ws + y.p_opart);
    p.ml = reinterpret_cast<float2*>(ws + y.p_ml);
    p.table = d.table;
    p.lens = d.lens;
    p.slots = d.slots;
    p.width = int(d.table_width);
    p.n_slots = int(d.n_slots);
    p.pages = int(d.pages);
    p.page_shift = page_shift;
    p.box_shift = box_shift;
    p.prefix = y.prefix;
    p.batch = int(d.batch);
    p.heads_kv = int(d.heads_kv);
    p.pairs = y.pairs;
    p.splits = y.splits;
    p.row_tiles = y.row_tiles;
    const int tiles = (y.prefix + BN - 1) / BN;
    p.per_split = tiles / y.splits;
    p.extra = tiles % y.splits;
    const int items = int(d.heads_kv) * y.pairs * y.splits;
    attn_tc_kernel<D, true><<<unsigned(items), THREADS, Cfg<D>::SMEM, s>>>(mq, mk, mv, p, items);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  DecodeParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(d.q);
  p.q_batch = d.q_batch;
  p.q_head = d.q_head;
  p.table = d.table;
  p.lens = d.lens;
  p.slots = d.slots;
  p.batch = int(d.batch);
  p.heads_kv = int(d.heads_kv);
  p.group = y.group;
  p.blocks = y.blocks;
  p.rows = y.rows;
  p.width = int(d.table_width);
  p.n_slots = int(d.n_slots);
  p.pages = int(d.pages);
  p.page_shift = page_shift;
  p.box_shift = box_shift;
  p.prefix = y.prefix;
  p.base = y.prefix / CHUNK * CHUNK;
  p.fold = y.fold;
  p.out = static_cast<__nv_bfloat16*>(d.out);
  p.o_batch = d.o_batch;
  p.o_head = d.o_head;
  p.part = y.splits > 0;
  p.scale_log2 = scale_log2;
  p.opart = reinterpret_cast<float*>(ws + y.d_opart);
  p.ml = reinterpret_cast<float2*>(ws + y.d_ml);
  p.starts = reinterpret_cast<int32_t*>(ws + y.starts);
  p.status = status;
  // A CTA that has the SM to itself needs the whole ring to cover the loads' latency.
  p.stages = y.direct && y.ctas <= enigma::sm_count() ? DCfg<D>::DEEP : DCfg<D>::STAGES;
  const int smem = p.stages * 2 * DCfg<D>::TILE + 1024 + (y.direct ? 0 : int(2 * d.batch + 1) * 4);
  const auto kernel = y.rows <= 8 ? (y.direct ? paged_decode_kernel<D, true, 1>
                                          : paged_decode_kernel<D, false, 1>)
                              : (y.direct ? paged_decode_kernel<D, true, 2>
                                          : paged_decode_kernel<D, false, 2>);
  {
    static std::atomic<uint64_t> ready{0};                  // devices where the attribute is set
    int dev = 0;
    e = cudaGetDevice(&dev);
    if (e == cudaSuccess && !(dev < 64 && (ready.load() >> dev & 1))) {
      const auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
      const int unit = DCfg<D>::DEEP * 2 * DCfg<D>::TILE + 1024;
      const int list = DCfg<D>::STAGES * 2 * DCfg<D>::TILE + 1024 + 8193 * 4;
      e = cudaFuncSetAttribute(paged_decode_kernel<D, true, 1>, attr, unit);
      if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_decode_kernel<D, true, 2>, attr, unit);
      if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_decode_kernel<D, false, 1>, attr, list);
      if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_decode_kernel<D, false, 2>, attr, list);
      if (e == cudaSuccess && dev < 64) ready.fetch_or(uint64_t(1) << dev);
    }
    if (e != cudaSuccess) return e;
  }
  if (y.beside) {
    // On a second stream, after the work before this call and before the join, which waits for it
    // even if the launch failed: a stream that captures must come back.
    e = cudaStreamWaitEvent((*side).stream, (*side).fork, 0);
    if (e != cudaSuccess) return e;
    kernel<<<unsigned(y.ctas), DTHREADS, smem, (*side).stream>>>(mk, mv, p);
    e = cudaGetLastError();
    cudaError_t back = cudaEventRecord((*side).back, (*side).stream);
    if (back == cudaSuccess) back = cudaStreamWaitEvent(s, (*side).back, 0);
    if (e == cudaSuccess) e = back;
  } else if (y.splits > 0) {
    e = enigma::launch_dependent(kernel, unsigned(y.ctas), DTHREADS, smem, s, mk, mv, p);
  } else {
    kernel<<<unsigned(y.ctas), DTHREADS, smem, s>>>(mk, mv, p);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess || (y.direct && y.splits == 0)) return e;
  JoinParams j = {};
  j.out = static_cast<__nv_bfloat16*>(d.out);
  j.o_batch = d.o_batch;
  j.o_head = d.o_head;
  j.batch = int(d.batch);
  j.heads_q = int(d.heads_q);
  j.heads_kv = int(d.heads_kv);
  j.group = y.group;
  j.p_opart = reinterpret_cast<const float*>(ws + y.p_opart);
  j.p_ml = reinterpret_cast<const float2*>(ws + y.p_ml);
  j.pairs = y.pairs;
  j.splits = y.splits;
  j.row_tiles = y.row_tiles;
  j.tokens = y.tokens;
  j.d_opart = p.opart;
  j.d_ml = p.ml;
  j.starts = y.direct ? nullptr : p.starts;
  j.blocks = y.blocks;
  j.rows = y.rows;
  j.ctas = y.ctas;
  // Parts of a row: the prefix's (twice as many where one row tile has two softmax states), and four
  // of each range that its unit's own keys lie in.
  const int64_t rows = d.batch * d.heads_q, units = d.batch * d.heads_kv * y.blocks;
  const int64_t parts = y.splits * (y.row_tiles % 2 + 1) +
                        (y.direct ? 1 : (y.ctas / units + 1) * DWARPS);
  const bool many = parts > kManyParts && rows <= 4 * enigma::sm_count();
  const auto join = many ? paged_join_kernel<D, kJoinWarps> : paged_join_kernel<D, 1>;
  const unsigned grid = unsigned(many ? rows : (rows + 3) / 4), threads = many ? kJoinWarps * 32 : 128;
  if (y.beside) {
    join<<<grid, threads, 0, s>>>(j);
    return cudaGetLastError();
  }
  return enigma::launch_dependent(join, grid, threads, 0, s, j);
}

}  // namespace

namespace enigma {

size_t sdpa_shared_prefix_workspace(const enigma_sdpa_shared_prefix_desc& d) {
  return d.batch > 0 && (d.head_dim == 64 || d.head_dim == 128) &&
                 d.dtype == ENIGMA_DTYPE_BF16 && d.heads_q / d.heads_kv <= BM
             ? layout_of(d).total
             : 0;
}

cudaError_t sdpa_shared_prefix_launch(const enigma_sdpa_shared_prefix_desc& d, cudaStream_t s) {
  if (!tc_takes(d)) return sdpa_paged_simt_launch(d, s);
  note_kernel(layout_of(d).splits > 0 ? "attn_tc_kernel" : "paged_decode_kernel");
  return d.head_dim == 128 ? launch<128>(d, s) : launch<64>(d, s);
}

}  // namespace enigma
