// attn_serving.cuh — argument blocks shared by the serving attention kernels: prompts of
// different lengths packed into one tensor, and single tokens over a paged cache.
#pragma once
#include "common.cuh"

namespace enigma_serving {

// The plan of a packed batch (enigma_sdpa_packed_plan), as ints: the header, n_ctas + 1 offsets
// (thread block c works through items [offset[c], offset[c + 1])), the items, the groups.
enum PlanHeader { kItems, kCtas, kSlots, kGroups, kItemsAt, kGroupsAt, kInts, kReserved };
constexpr int kOffsetsAt = ENIGMA_PACKED_PLAN_HEADER;

// One work item: the rows (token, query head of one kv head's group) of up to two consecutive
// tiles of a sequence, and the 128-key tiles [j0, j1) it covers.
struct PackedItem {
  int q0, lq;        // the sequence's first query row in the packed tensor, its length
  int k0, lk;        // the same of its keys
  int t0;            // first token of the item's first tile, within the sequence
  int tokens;        // tokens in each of its (at most) two tiles
  int j0, j1;
  int kvh;
  int slot;          // first of its two tiles' partial results, or -1: it computes the final one
  int pad[2];
};
constexpr int kItemInts = sizeof(PackedItem) / 4;

// The items of one pair of tiles whose keys were split: partial results slot, slot + 2, ... of
// `parts` items make the first tile's rows, slot + 1, slot + 3, ... the second's.
struct PackedGroup {
  int tok0, tok_end;  // first token of the first tile, end of the sequence (packed rows)
  int tokens, kvh;
  int slot, parts, pad[2];
};
constexpr int kGroupInts = sizeof(PackedGroup) / 4;

// Joins partial results of one row, a warp's work:
//   O = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i, M = max_i m_i (m in log2 units),
// always in the same order.  add() folds n partials in, `ml` + i * ml_step and `o` + i * o_step
// (D floats, lane takes every 32nd); best() must have seen the same ones first.  The lanes
// load 32 pairs (m, l) at once and 8 partials' rows are in flight together: one after the other
// the loads' latency is the whole time (20 partials: 24 us, now 3).  A partial that saw no key
// (m = -inf) may hold anything.
template <int V>
struct RowJoin {
  float acc[V] = {};
  float M = -INFINITY, l = 0.f;
  __device__ void best(const float2* ml, int64_t ml_step, int n, int lane) {
    for (int i = lane; i < n; i += 32) M = fmaxf(M, ml[i * ml_step].x);
  }
  __device__ void seal() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  }
  __device__ void add(const float2* ml, int64_t ml_step, const float* o, int64_t o_step, int n, int D,
                      int lane) {
    for (int i0 = 0; i0 < n; i0 += 32) {
      const float2 mine = i0 + lane < n ? ml[(i0 + lane) * ml_step] : make_float2(-INFINITY, 0.f);
      const float w = mine.x == -INFINITY ? 0.f : exp2f(mine.x - M);
      float part = w == 0.f ? 0.f : w * mine.y;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) part += __shfl_xor_sync(0xffffffffu, part, x);
      l += part;
      const int here = min(32, n - i0);
      for (int i = 0; i < here; i += 8) {
        float f[8], v[8][V];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          f[u] = __shfl_sync(0xffffffffu, w, (i + u) & 31);
          if (i + u >= here) f[u] = 0.f;
#pragma unroll
          for (int x = 0; x < V; ++x) {
            v[u][x] = 0.f;
            if (f[u] != 0.f && lane + 32 * x < D) v[u][x] = o[(i0 + i + u) * o_step + lane + 32 * x];
          }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
          for (int x = 0; x < V; ++x) acc[x] = fmaf(v[u][x], f[u], acc[x]);
      }
    }
  }
};

}  // namespace enigma_serving
