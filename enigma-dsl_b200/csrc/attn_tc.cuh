// attn_tc.cuh — attention on the sm_100a tensor cores for the serving operators.
//
//   O_r = sum_j softmax_j(scale q_r . k_j) v_j,   keys j < lim(r)
//
// A row r is one (token, query head) of a kv head's group: a tile takes `tokens` = 128 / G
// tokens with all G heads of their group, so every row of a tile reads the same K and V, a
// short sequence does not pay a tile per head, and a causal tile's rows end within
// `tokens` keys of each other.  A work item is two row tiles (256 rows) of one kv head and a
// range of 128-key tiles; or (paged, alt) one row tile twice, the even key tiles with one softmax
// state and the odd ones with the other, when there is no second row tile to fill the SM.  An alt
// item is its CTA's only one and the rings are even, so a state meets the same stages throughout
// and waits for every phase of their barriers.
//
//   warp 0      TMA: both Q tiles, then K and V tiles into rings of C::STAGES
//   warps 1, 2  one thread each issues the tcgen05.mma of softmax state i = warp - 1:
//               S_i = Q_i K_j^T, O_i += P_i V_j (P from TMEM over S_i's columns); the tensor
//               core works for one state while the other's softmax runs
//   warps 4-7, 8-11   softmax of the two tiles, one thread per row, fp32
//
// What bounds it: per 128 keys of both tiles the tensor core needs 2048 cycles and the
// exponential units 2048 (256 x 128 at 16 a cycle), each tile's chain S -> softmax -> P V -> S
// about 3500.  So the two states work in turns: one weighs its tile (its exponentials) while the
// other's products run.  Without turns they fall into step, both at the exponentials and then
// both waiting for the tensor core: 4300 cycles a step against 3550 (8192 tokens, 32 / 8 heads of
// 128, causal: 573 -> 457 us = 1200 TFLOP/s; one issuing thread for both states, in turns or not,
// 573 to 583 us).  The turn passes on after kHandOver of the 128 keys: 96 keys 457 us, 64 479,
// 80 480, all 128 482.
//
// The softmax takes the running maximum that the tiles before left and starts its exponentials
// at once; this tile's maximum is found beside them and only has to show that no weight exceeds
// 2^kGrow.  If one does, O and the sum are rescaled and the tile's exponentials are done again.
// Any base within fp32's range gives the same quotient, so this is exact (the maximum first:
// 463 us).  Not kept: a degree-4 polynomial on the FMA pipe for 1/8, 1/4, 3/8 of the exponentials
// (480, 511, 535 us: a turn is bound by one warp's instructions); the row sum after P's release
// (467 us); P released once, or at 96 keys (470 us).
//
// P is rounded to bf16, the operand type of the PV product; sums, maxima and O stay fp32.
// Every mbarrier wait is bounded (sm100.cuh).  Whether or not one ran out, a block ends only when its
// copies have landed and its products are done.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>

#include "attn_serving.cuh"

namespace enigma_tc {

using namespace enigma_sm100;

constexpr int BM = 128;            // rows per tile (two tiles per item)
constexpr int BN = 128;            // keys per tile
constexpr int THREADS = 384;       // warpgroup 0: TMA, 2 MMA, idle; WG 1, 2: softmax
// Register split: 384 x 168 at launch; warpgroup 0 drops to 104, the softmax warpgroups rise to
// 200: 128 * 104 + 256 * 200 = 384 * 168 exactly.
constexpr int LAUNCH_REGS = 168, WG0_REGS = 104, SOFTMAX_REGS = 200;
static_assert(128 * WG0_REGS + 256 * SOFTMAX_REGS <= THREADS * LAUNCH_REGS, "register split");
constexpr int kHandOver = 96;      // keys of a tile weighed when the other state's turn begins
constexpr float kGrow = 24.f;      // log2 units a weight may exceed 1 by before a rescale

template <int D>
struct Cfg {
  static constexpr int STAGES = D == 64 ? 4 : 2;
  static constexpr int Q_BYTES = BM * D * 2;
  static constexpr int KV_BYTES = BN * D * 2;
  static constexpr int ATOMS = D / 64;           // 128-byte swizzle atoms along D
  static constexpr int SMEM = 2 * Q_BYTES + 2 * STAGES * KV_BYTES + 1024 + 512;
  static constexpr uint32_t TMEM_COLS = 512;     // S0 | S1 | O0 | O1
  static constexpr uint32_t O_COL = 2 * BN;
};

struct Params {
  float scale_log2;
  int group, tokens;               // G, tokens per row tile (G * tokens <= 128)
  uint32_t* status;
  float* opart;                    // [slot][D / 8][128][8] fp32, not normalised
  float2* ml;                      // [slot][128] (maximum in log2 units, sum)
  // packed prompts
  const int32_t *offsets, *list;   // each CTA's range of items, the items
  __nv_bfloat16* out;
  float* lse;
  int64_t o_token, o_head;
  int heads_q, causal, tokens_q, tokens_k;
  int slots_end;                   // slots of partial results, at least 1
  int one;                         // each CTA has exactly one item
  // paged prefix
  const int32_t *table, *lens, *slots;
  int width, n_slots, pages, page_shift, box_shift, prefix, batch, heads_kv;
  int pairs, splits, row_tiles;
  int per_split, extra;            // key tiles of a part; the first `extra` have one more
};

// One item, as every role sees it.
struct Work {
  int tok0, tok_end;     // first token of tile 0; end of the sequence (batch)
  int kvh, k0, lk;       // kv head, first key row, number of keys
  int off;               // a token's keys: min(lk, token - seq0 + off); off >= lk: all
  int seq0;
  int j0;                // first key tile
  int cnt0, cnt1;        // key tiles of each softmax state
  int all;               // key tiles streamed
  bool alt;
  int slot;              // first partial slot, or -1: final result
};

template <bool PAGED>
__device__ __forceinline__ Work make_work(const Params& p, int t) {
  Work w;
  if (PAGED) {
    const int split = t % p.splits, unit = t / p.splits;
    const int pair = unit % p.pairs;
    w.kvh = unit / p.pairs;
    w.tok0 = pair * 2 * p.tokens;
    w.tok_end = p.batch;
    w.seq0 = 0;
    w.k0 = 0;
    w.lk = p.prefix;
    w.off = p.prefix;
    w.j0 = split * p.per_split + min(split, p.extra);
    w.all = p.per_split + (split < p.extra ? 1 : 0);
    w.alt = 2 * pair + 1 >= p.row_tiles;
    w.cnt0 = w.alt ? (w.all + 1) / 2 : w.all;
    w.cnt1 = w.alt ? w.all / 2 : w.all;
    w.slot = 2 * t;
  } else {
    const int4* it = reinterpret_cast<const int4*>(p.list) +
                     int64_t(t) * (enigma_serving::kItemInts / 4);
    const int4 a = __ldg(it), b = __ldg(it + 1), c = __ldg(it + 2);
    // q0 lq k0 lk | t0 tokens j0 j1 | kvh slot - -
    w.seq0 = a.x;
    w.tok0 = a.x + b.x;
    // An item that does not lie inside the tensors (a plan made for others) has no rows here.
    const bool in = a.x >= 0 && b.x >= 0 && c.x >= 0 && c.x < p.heads_kv && c.y + 1 < p.slots_end;
    w.tok_end = in ? a.x + a.y : w.tok0;
    w.k0 = a.z;
    w.lk = a.w;
    w.off = p.causal ? a.w - a.y + 1 : a.w;
    w.kvh = c.x;
    w.alt = false;
    w.slot = c.y;
    w.j0 = b.z;
    auto tiles = [&](int first) {
      const int last = min(first + p.tokens, w.tok_end) - 1;
      const int keys = p.causal ? min(w.lk, last - w.seq0 + w.off) : w.lk;
      const int end = first < w.tok_end && keys > 0 ? (keys + BN - 1) / BN : 0;
      return max(min(end, b.w) - b.z, 0);
    };
    w.cnt0 = tiles(w.tok0);
    w.cnt1 = tiles(w.tok0 + p.tokens);
    w.all = max(w.cnt0, w.cnt1);
  }
  return w;
}

// ------------------------------------------------------------------ packed fp32 math
__device__ __forceinline__ float2 f2fma(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 f2add(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 4-D tiled load (pages: head_dim, row, kv head, page).
__device__ __forceinline__ void tma_load_4d(void* dst, const void* desc, uint64_t* bar, int32_t c0,
                                            int32_t c1, int32_t c2, int32_t c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(desc)), "r"(smem_u32(bar)), "r"(c0),
        "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// 32 bytes, a sector.
__device__ __forceinline__ void store_32b(float* to, const uint32_t* x) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(to), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]),
                 "r"(x[6]), "r"(x[7])
               : "memory");
}

// The number of a page, or `pages` (out of the tensor map's range: reads as zeros) where the
// table holds none.
__device__ __forceinline__ int page_at(const int32_t* table, const int32_t* slots, int n_slots,
                                       int width, int pages, int seq, int col) {
  const int slot = slots != nullptr ? slots[seq] : seq;
  if (slot < 0 || slot >= n_slots || col >= width) return pages;
  const int at = table[int64_t(slot) * width + col];
  return at < 0 || at >= pages ? pages : at;
}

// Keys of sequence b.
__device__ __forceinline__ int len_of(const int32_t* lens, const int32_t* slots, int n_slots,
                                      int64_t most, int b) {
  const int slot = slots != nullptr ? slots[b] : b;
  if (slot < 0 || slot >= n_slots) return 0;
  const int n = lens[slot];
  return n < 0 ? 0 : int(n < most ? n : most);
}

template <int D, bool PAGED>
__global__ void __launch_bounds__(THREADS, 1)
attn_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
               const __grid_constant__ CUtensorMap tmV, const Params p, const int items) {
  using C = Cfg<D>;
  constexpr int ST = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                                   // Q0 | Q1
  uint8_t* sK = sQ + 2 * C::Q_BYTES;
  uint8_t* sV = sK + ST * C::KV_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + ST * C::KV_BYTES);
  uint64_t* q_full = bars;                   // [2] one Q tile per softmax state
  uint64_t* q_empty = q_full + 2;            // [2] the item's last S product has read Q_i
  uint64_t* k_full = q_empty + 2;            // [ST]
  uint64_t* k_empty = k_full + ST;
  uint64_t* v_full = k_empty + ST;
  uint64_t* v_empty = v_full + ST;
  uint64_t* s_full = v_empty + ST;            // [2] one per softmax state
  uint64_t* p_full = s_full + 2;             // [2 states][2 halves of the keys]
  uint64_t* o_done = p_full + 4;             // [2]
  uint64_t* o_free = o_done + 2;             // [2] the epilogue has read O_i
  uint64_t* turn = o_free + 2;               // [2] state i may take the exponential units
  uint64_t* idle = turn + 2;                 // [2] a wait ran out: the products of state i are done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(idle + 2);
  __shared__ int loads[4], gave_up;          // K, V, Q_0, Q_1 tiles asked for; a wait ran out

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  griddep_launch_dependents();               // the next kernel may take SMs that are free
  // Packed: the plan lists each CTA's items.  Paged: one item per CTA.
  const bool one = PAGED || p.one;
  const int t_begin = one ? int(blockIdx.x) : __ldg(p.offsets + blockIdx.x);
  const int t_end = one ? min(t_begin + 1, items) : __ldg(p.offsets + blockIdx.x + 1);

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    for (int s = 0; s < ST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 2);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 128);
      mbar_init(&p_full[2 * i + 1], 128);
      mbar_init(&o_done[i], 1);
      mbar_init(&o_free[i], 128);
      mbar_init(&turn[i], 4);
      mbar_init(&idle[i], 1);
    }
    fence_barrier_init();
    gave_up = 0;
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(WG0_REGS));
    if (warp == 0) {
      // ------------------------------------------------------------ TMA producer
      int jg = 0;                            // key tiles loaded so far
      int k_loads = 0, v_loads = 0;          // tiles asked for
      int q_items[2] = {0, 0};               // items with work per softmax state
      bool ok = true;
      const uint32_t q_bytes = uint32_t(p.group * p.tokens) * 128u;   // one atom of a Q tile
      for (int t = t_begin; t < t_end && ok; ++t) {
        const Work w = make_work<PAGED>(p, t);
        if (w.all == 0) continue;
        auto load_q = [&](int i, int n) {    // an alt item's one tile goes to both states
          if (n == 0) return true;
          if (q_items[i] > 0 &&
              !__all_sync(0xffffffffu, mbar_wait(&q_empty[i], (q_items[i] - 1) & 1, p.status)))
            return false;
          ++q_items[i];
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full[i], q_bytes * C::ATOMS);
#pragma unroll
            for (int a = 0; a < C::ATOMS; ++a)
              tma_load_3d(sQ + i * C::Q_BYTES + a * BM * 128, &tmQ, &q_full[i], a * 64,
                          w.kvh * p.group, w.tok0 + (w.alt ? 0 : i * p.tokens));
          }
          __syncwarp();
          return true;
        };
        ok = load_q(0, w.cnt0);
        if (!ok) break;
        // Paged: lane x knows the page of box x of the next tiles; the table is read two tiles ahead.
        // One lane issues all boxes, each lane its own was no faster; nor does it help to ask for
        // later tiles' bytes in L2 (128 sequences, 32768 shared keys: 111 us with, 105 without).
        int at_next = p.pages, at_after = p.pages;   // of tiles j, j + 1
        const bool looks = PAGED && lane < (BN >> p.box_shift);
        auto look_up = [&](int j) {          // the j-th tile of the item; none past its end
          if (!looks || j >= w.all) return p.pages;
          return page_at(p.table, p.slots, p.n_slots, p.width, p.pages, 0,
                         ((w.j0 + j) * BN + (lane << p.box_shift)) >> p.page_shift);
        };
        if (PAGED) {
          at_next = look_up(0);
          at_after = look_up(1);
        }
        for (int j = 0; j < w.all; ++j, ++jg) {
          const int s = jg % ST;
          const uint32_t ph = (jg / ST) & 1;
          const int key0 = (w.j0 + j) * BN;
          int boxes = 0;
          int at_now = 0;
          if (PAGED) {
            boxes = (min(BN, w.lk - key0) + (1 << p.box_shift) - 1) >> p.box_shift;
            at_now = at_next;
            at_next = at_after;
            at_after = look_up(j + 2);
          }
          const uint32_t bytes = PAGED ? (uint32_t(boxes * C::ATOMS) * 128u) << p.box_shift
                                       : uint32_t(C::KV_BYTES);
          auto load = [&](const CUtensorMap* map, uint8_t* dst, uint64_t* full, uint64_t* empty) {
            if (!__all_sync(0xffffffffu, mbar_wait(empty, ph ^ 1, p.status))) return false;
            if (lane == 0) mbar_arrive_expect_tx(full, bytes);
            __syncwarp();
            if (PAGED) {
              for (int x = 0; x < boxes; ++x) {
                const int page = __shfl_sync(0xffffffffu, at_now, x);
                const int row = (key0 + (x << p.box_shift)) & ((1 << p.page_shift) - 1);
                if (elect_one()) {
#pragma unroll
                  for (int a = 0; a < C::ATOMS; ++a)
                    tma_load_4d(dst + a * BN * 128 + ((x << p.box_shift) * 128), map, full, a * 64,
                                row, w.kvh, page);
                }
                __syncwarp();
              }
            } else if (lane == 0) {
#pragma unroll
              for (int a = 0; a < C::ATOMS; ++a)
                tma_load_3d(dst + a * BN * 128, map, full, a * 64, w.kvh, w.k0 + key0);
            }
            __syncwarp();
            return true;
          };
          ok = load(&tmK, sK + s * C::KV_BYTES, &k_full[s], &k_empty[s]);
          if (!ok) break;
          k_loads = jg + 1;
          ok = (j > 0 || load_q(1, w.cnt1)) &&
               load(&tmV, sV + s * C::KV_BYTES, &v_full[s], &v_empty[s]);
          if (!ok) break;
          v_loads = jg + 1;
        }
      }
      if (lane == 0) {
        loads[0] = k_loads;
        loads[1] = v_loads;
        loads[2] = q_items[0];
        loads[3] = q_items[1];
        if (!ok) gave_up = 1;
      }
      __syncwarp();
    } else if (warp <= 2) {
      // ------------------------------------------------------------ MMA issuers
      // Warp 1 + i issues for softmax state i: S_0 | PV_0 S_1 | PV_1 S_2 ...  Each state's
      // products wait for its own softmax only; the tensor core takes them as they come.
      if (lane == 0) {
        const int i = warp - 1;
        constexpr uint32_t idesc_s = idesc_bf16_f32(BM, BN, false, false);
        constexpr uint32_t idesc_o = idesc_bf16_f32(BM, D, false, true);
        const uint32_t s_tmem = tmem + uint32_t(i * BN), o_tmem = tmem + C::O_COL + uint32_t(i * D);
        const uint64_t dk0 = smem_desc_sw128(smem_u32(sK), 16, 1024);
        const uint64_t dv0 = smem_desc_sw128(smem_u32(sV), BN * 128, 1024);
        const uint64_t dq = smem_desc_sw128(smem_u32(sQ) + uint32_t(i) * C::Q_BYTES, 16, 1024);
        int jg = 0, pv = 0, items_done = 0;  // items_done: with work for this state
        bool ok = true;
        for (int t = t_begin; t < t_end && ok; ++t) {
          const Work w = make_work<PAGED>(p, t);
          if (w.all == 0) continue;
          const int n = i == 0 ? w.cnt0 : w.cnt1;
          // A stage is free again after one arrival from each issuer; the only user of an
          // alt item's stage arrives twice.
          auto release = [&](uint64_t* empty) {
            mma_commit(empty);
            if (w.alt) mma_commit(empty);
          };
          int st = jg + (w.alt ? i : 0);
          const int step = w.alt ? 2 : 1;
          auto issue_s = [&](int at) {
            const int sk = at % ST;
            tc_fence_after();
            const uint64_t dk = dk0 + uint64_t((sk * C::KV_BYTES) >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint64_t off = uint64_t(((kk / 4) * (BM * 128) + (kk % 4) * 32) >> 4);
              mma_bf16_ss(s_tmem, dq + off, dk + off, idesc_s, kk != 0 ? 1u : 0u);
            }
            mma_commit(&s_full[i]);
          };
          if (n > 0) {
            ok = mbar_wait(&q_full[i], items_done & 1, p.status) &&
                 mbar_wait(&k_full[st % ST], (st / ST) & 1, p.status);
            if (!ok) break;
            issue_s(st);
            if (n == 1) mma_commit(&q_empty[i]);
            release(&k_empty[st % ST]);
          }
          for (int j = 0; j < n; ++j, st += step) {
            const int sv = st % ST, next = st + step;
            // What the products of this step need besides P, before P is waited for.
            ok = mbar_wait(&v_full[sv], (st / ST) & 1, p.status) &&
                 (j + 1 == n || mbar_wait(&k_full[next % ST], (next / ST) & 1, p.status)) &&
                 (j > 0 || items_done == 0 || mbar_wait(&o_free[i], (items_done - 1) & 1, p.status));
            if (!ok) break;
            const uint64_t dv = dv0 + uint64_t((sv * C::KV_BYTES) >> 4);
            // P arrives in two halves of the keys, so the first half's products start while
            // the softmax finishes the second.
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              ok = mbar_wait(&p_full[2 * i + half], pv & 1, p.status);
              if (!ok) break;
              tc_fence_after();
#pragma unroll
              for (int kk = half * 4; kk < half * 4 + 4; ++kk)
                mma_bf16_ts(o_tmem, s_tmem + kk * 8, dv + uint64_t((kk * 2048) >> 4), idesc_o,
                            (j | kk) != 0 ? 1u : 0u);
            }
            if (!ok) break;
            ++pv;
            if (j + 1 == n) {
              mma_commit(&o_done[i]);
            } else {
              issue_s(next);
              if (j + 2 == n) mma_commit(&q_empty[i]);    // the item's last S was just issued
              release(&k_empty[next % ST]);
            }
            release(&v_empty[sv]);
          }
          if (!ok) break;
          if (n > 0) ++items_done;
          // Key tiles that only the other state needs.
          if (!w.alt) {
            for (int j = n; j < w.all; ++j, ++st) {
              ok = mbar_wait(&k_full[st % ST], (st / ST) & 1, p.status);
              if (!ok) break;
              mbar_arrive(&k_empty[st % ST]);
              ok = mbar_wait(&v_full[st % ST], (st / ST) & 1, p.status);
              if (!ok) break;
              mbar_arrive(&v_empty[st % ST]);
            }
          }
          jg += w.all;
        }
        if (!ok) gave_up = 1;
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
    // ------------------------------------------------------------ softmax / epilogue
    const int ti = (warp - 4) >> 2;           // softmax state of this warpgroup
    const int quarter = warp & 3;             // TMEM lane quarter this warp may access
    const int r = quarter * 32 + lane;        // row of the tile owned by this thread
    const uint32_t lane_off = uint32_t(quarter * 32) << 16;
    const uint32_t s_addr = tmem + lane_off + uint32_t(ti * BN);
    const uint32_t o_addr = tmem + lane_off + C::O_COL + uint32_t(ti * D);
    const float c = p.scale_log2;
    const int r_tok = r / p.group, r_head = r - r_tok * p.group;
    int sg = 0, acc_items = 0;                // S tiles seen, items whose O accumulated
    int jg = 0;                               // key tiles streamed before this item
    int turns = 0;                            // turns taken
    if (ti == 1 && lane == 0) mbar_arrive(&turn[0]);   // state 0 begins
    bool ok = true;
    for (int t = t_begin; t < t_end && ok; ++t) {
      Work w = make_work<PAGED>(p, t);
      const int n_my = ti == 0 ? w.cnt0 : w.cnt1;
      const int tok = w.tok0 + (w.alt ? 0 : ti * p.tokens) + r_tok;
      const bool live = r_tok < p.tokens && tok < w.tok_end && (PAGED || tok < p.tokens_q);
      int keys = 0;                           // keys this row sees
      if (live) {
        keys = PAGED ? min(w.lk, len_of(p.lens, p.slots, p.n_slots,
                                        int64_t(p.width) << p.page_shift, tok))
                     : min(w.lk, tok - w.seq0 + w.off);
      }
      // From here on the keys that any row of the item sees, where sequences end before the
      // prefix does.  Looked for only where no row of this warp sees all of them.
      if (PAGED && !__any_sync(0xffffffffu, live && keys == w.lk)) {
        int most = 0;
        const int end = min(w.tok0 + 2 * p.tokens, w.tok_end);
        for (int b = w.tok0 + lane; b < end; b += 32)
          most = max(most, len_of(p.lens, p.slots, p.n_slots, int64_t(p.width) << p.page_shift, b));
        w.lk = min(w.lk, __reduce_max_sync(0xffffffffu, most));
      }
      float m_used = -INFINITY, l = 0.f;      // m in raw score units
      const int both = min(w.cnt0, w.cnt1);   // tiles that both states have: taken in turns
      for (int j = 0; j < n_my; ++j, ++sg) {
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[ti], sg & 1, p.status));
        if (!ok) break;
        tc_fence_after();
        float x[BN];
#pragma unroll
        for (int k = 0; k < BN; k += 32) tmem_ld32(s_addr + k, reinterpret_cast<uint32_t*>(&x[k]));
        tmem_wait_ld();
        const int tile = w.alt ? 2 * j + ti : j;     // within the item
        const int lim = keys - (w.j0 + tile) * BN;
        // Warp-uniform: the loop below holds warp-collective tcgen05.st.  Rows of no token
        // are left as they are; nobody reads their result.
        if (__any_sync(0xffffffffu, live && lim < BN)) {
#pragma unroll
          for (int k = 0; k < BN; ++k) x[k] = (k < lim) ? x[k] : -INFINITY;
        }
        float2 sum2[4];
        float mq[4];
        auto row_max = [&](int k0, int k1) {       // folds x[k0 .. k1) into mq
#pragma unroll
          for (int k = k0; k < k1; k += 8)
#pragma unroll
            for (int u = 0; u < 4; ++u) mq[u] = max3f(mq[u], x[k + u], x[k + 4 + u]);
        };
        // p = 2^(s c - m c) in fp32 for 16 keys, summed in fp32, stored as bf16 pairs.
        auto weigh = [&](int k, float2 cc, float2 nmc) {
          uint32_t pk[8];
#pragma unroll
          for (int t2 = 0; t2 < 8; ++t2) {
            const float2 y = f2fma(make_float2(x[k + 2 * t2], x[k + 2 * t2 + 1]), cc, nmc);
            const float2 e = make_float2(ex2(y.x), ex2(y.y));
            sum2[t2 & 3] = f2add(sum2[t2 & 3], e);
            pk[t2] = pack_bf16x2(e.x, e.y);
          }
          tmem_st8(s_addr + k / 2, pk);
        };
        const float2 cc = make_float2(c, c);
        float2 nmc;
        auto rebase = [&](float m_new, bool need) {    // warp-uniform call
          const float f = need ? ex2((m_used - m_new) * c) : 1.0f;   // m_used = -inf: f = 0
          l *= f;
          if (j > 0) {
            // "S_i(j) done" implies PV_i(j-1) done (commit order), so O is complete here.
#pragma unroll 1
            for (int k = 0; k < D; k += 16) {
              uint32_t o[16];
              tmem_ld16(o_addr + k, o);
              tmem_wait_ld();
              uint32_t lo[8], hi[8];
#pragma unroll
              for (int t2 = 0; t2 < 8; ++t2) {
                lo[t2] = __float_as_uint(__uint_as_float(o[t2]) * f);
                hi[t2] = __float_as_uint(__uint_as_float(o[8 + t2]) * f);
              }
              tmem_st8(o_addr + k, lo);
              tmem_st8(o_addr + k + 8, hi);
            }
            tmem_wait_st();
          }
          if (need) m_used = m_new;
        };
        if (j == 0) {
#pragma unroll
          for (int u = 0; u < 4; ++u) mq[u] = -INFINITY;
          row_max(0, BN);
          m_used = max3f(mq[0], mq[1], fmaxf(mq[2], mq[3]));
        }
        if (j < both) {
          ok = __all_sync(0xffffffffu, mbar_wait(&turn[ti], turns & 1, p.status));
          if (!ok) break;
          ++turns;
        }
#pragma unroll 1
        for (int pass = 0; ; ++pass) {
          const float mc = (m_used == -INFINITY) ? 0.f : m_used * c;
          nmc = make_float2(-mc, -mc);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            sum2[u] = make_float2(0.f, 0.f);
            mq[u] = -INFINITY;
          }
#pragma unroll
          for (int k = 0; k < BN / 2; k += 16) {
            weigh(k, cc, nmc);
            row_max(2 * k, 2 * k + 32);
          }
          const float mx = max3f(mq[0], mq[1], fmaxf(mq[2], mq[3]));
          const bool need = (mx - m_used) * c > kGrow;    // m_used = -inf and a key: true
          if (pass > 0 || !__any_sync(0xffffffffu, need)) break;
          rebase(mx, need);
        }
        // What lies behind the last key that is seen (a neighbour's tokens, a page's unwritten
        // rows) may be NaN in V, and 0 * NaN would reach the sum.  Row r is cleared here,
        // before P is released; the stage stays until PV has read it.
        const int end = w.lk - (w.j0 + tile) * BN;
        if (end < BN) {
          const int st = jg + tile, s = st % ST;
          ok = __all_sync(0xffffffffu, mbar_wait(&v_full[s], (st / ST) & 1, p.status));
          if (!ok) break;
          if (r >= end) {
#pragma unroll
            for (int y = 0; y < D / 8; ++y)
              *reinterpret_cast<uint4*>(sV + s * C::KV_BYTES + (y / 8) * BN * 128 + r * 128 +
                                        (y % 8) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[2 * ti]);
#pragma unroll
        for (int k = BN / 2; k < BN; k += 16) {
          if (k == kHandOver && j < both && lane == 0) mbar_arrive(&turn[1 - ti]);
          weigh(k, cc, nmc);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[2 * ti + 1]);
        const float2 s01 = f2add(sum2[0], sum2[1]), s23 = f2add(sum2[2], sum2[3]);
        l += (s01.x + s23.x) + (s01.y + s23.y);
      }
      if (!ok) break;
      jg += w.all;
      if (n_my > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(&o_done[ti], acc_items & 1, p.status));
        if (!ok) break;
        tc_fence_after();
      }
      const bool none = n_my == 0 || keys <= 0;     // the row saw nothing
      if (w.slot < 0) {
        const float inv = none || l == 0.f ? 0.f : 1.0f / l;
        const int h = w.kvh * p.group + r_head;
        const int64_t row = live ? int64_t(tok) : 0;
        __nv_bfloat16* o_row = p.out + row * p.o_token + int64_t(live ? h : 0) * p.o_head;
        if (p.lse != nullptr && live)
          p.lse[row * p.heads_q + h] =
              none ? -INFINITY : (m_used * c + log2f(l)) * 0.6931471805599453f;
#pragma unroll 1
        for (int k = 0; k < D; k += 16) {
          uint32_t o[16];
          if (n_my > 0) {  // warp-uniform: the collective load runs on every lane
            tmem_ld16(o_addr + k, o);
            tmem_wait_ld();
          }
          uint32_t u[8];
#pragma unroll
          for (int t2 = 0; t2 < 8; ++t2)
            u[t2] = none ? 0u : pack_bf16x2(__uint_as_float(o[2 * t2]) * inv,
                                            __uint_as_float(o[2 * t2 + 1]) * inv);
          if (live) {
            reinterpret_cast<uint4*>(o_row + k)[0] = make_uint4(u[0], u[1], u[2], u[3]);
            reinterpret_cast<uint4*>(o_row + k)[1] = make_uint4(u[4], u[5], u[6], u[7]);
          }
        }
      } else {
        const int64_t row = int64_t(w.slot + ti) * BM + r;
        // (A row of nothing but NaN scores has l = NaN and no maximum: it is not empty.)
        if (live)
          p.ml[row] = none || l == 0.f ? make_float2(-INFINITY, 0.f)
                                       : make_float2(m_used == -INFINITY ? 0.f : m_used * c, l);
        if (n_my > 0) {
          // A warp's rows side by side, a sector each: with rows of D floats each of a warp's stores
          // met 32 lines (32 sequences, 4096 shared and up to 512 own keys, 32 / 8 heads of 128:
          // 21.7 -> 19.8 us; 1325 new tokens against 1 to 4096 keys, split: 60.6 -> 58.8).
          float* to = p.opart + int64_t(w.slot + ti) * BM * D + r * 8;
#pragma unroll 1
          for (int k = 0; k < D; k += 32) {
            uint32_t o[32];
            tmem_ld32(o_addr + k, o);
            tmem_wait_ld();
            if (live && !none) {
#pragma unroll
              for (int t2 = 0; t2 < 32; t2 += 8) store_32b(to + (k + t2) * BM, o + t2);
            }
          }
        }
      }
      if (n_my > 0) {
        // O_i has been read: the next item's first PV may overwrite it.
        tc_fence_before();
        mbar_arrive(&o_free[ti]);
        ++acc_items;
      }
    }
    if (!ok) gave_up = 1;
  }

  tc_fence_before();
  __syncthreads();
  if (gave_up != 0) {
    // What was asked for and nobody waited for, before its shared memory and TMEM go back.
    if (warp == 0) {
      for (int n = max(0, loads[0] - ST); n < loads[0]; ++n)
        mbar_drain(&k_full[n % ST], (n / ST) & 1);
      for (int n = max(0, loads[1] - ST); n < loads[1]; ++n)
        mbar_drain(&v_full[n % ST], (n / ST) & 1);
      for (int i = 0; i < 2; ++i)
        if (loads[2 + i] > 0) mbar_drain(&q_full[i], (loads[2 + i] - 1) & 1);
    } else if (warp <= 2 && lane == 0) {
      mma_commit(&idle[warp - 1]);
      mbar_drain(&idle[warp - 1], 0);
    } else if (warp >= 4) {
      tmem_wait_st();
    }
    tc_fence_before();
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// ------------------------------------------------------------------ host side
inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (fn == nullptr) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }
  return fn;
}

// bf16 map of `rank` dimensions, innermost contiguous; strides in bytes of dimensions 1, ...
inline bool make_map(CUtensorMap* m, const void* base, int rank, const cuuint64_t* dims,
                     const cuuint64_t* strides, const cuuint32_t* box) {
  auto fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, cuuint32_t(rank), const_cast<void*>(base), dims,
            strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Launch attributes of one instantiation (shared memory, registers enough for the split), set
// once per device: they outlast the call, and setting them costs a microsecond.
template <int D, bool PAGED>
cudaError_t prepare_kernel() {
  const auto kernel = attn_tc_kernel<D, PAGED>;
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && (ready.load() >> dev & 1)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::SMEM);
  if (e != cudaSuccess) return e;
  cudaFuncAttributes fa;
  e = cudaFuncGetAttributes(&fa, kernel);
  if (e != cudaSuccess) return e;
  if (fa.numRegs < LAUNCH_REGS) return cudaErrorInvalidConfiguration;
  if (dev < 64) ready.fetch_or(uint64_t(1) << dev);
  return cudaSuccess;
}

}  // namespace enigma_tc
