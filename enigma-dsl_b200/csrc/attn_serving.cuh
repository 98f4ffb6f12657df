// attn_serving.cuh — argument blocks shared by the serving attention kernels: prompts of
// different lengths packed into one tensor, and single tokens over a paged cache.
#pragma once
#include "common.cuh"

namespace enigma_serving {

// The plan of a packed batch (enigma_sdpa_packed_plan), as ints: the header, n_ctas + 1 offsets
// (thread block c works through items [offset[c], offset[c + 1])), the items, the groups.  kLongest:
// 128-key tiles of the longest item.
enum PlanHeader { kItems, kCtas, kSlots, kGroups, kItemsAt, kGroupsAt, kInts, kLongest };
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

}  // namespace enigma_serving
