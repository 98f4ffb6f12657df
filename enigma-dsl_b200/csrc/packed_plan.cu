// packed_plan.cu — the work list of the packed attention (host code).
//
// Items are dealt out heaviest first, each to the thread block with the least work so far, so
// the SMs finish within about one light item of each other without a shared counter; the order
// is fixed, and so are the results.  Where the batch has too few rows to fill the SMs, long key
// ranges are split into parts whose partial results are joined afterwards.
#include <algorithm>
#include <cstring>
#include <queue>
#include <vector>

#include "attn_serving.cuh"

namespace enigma_serving {

namespace {

// Cost of an item in steps of one 128-key tile for both row tiles: its start (Q, first S) and
// its epilogue take about as long as kItemCost steps.
constexpr int64_t kItemCost = 2;
// A part keeps at least this many key tiles: each part writes and the join reads 256 rows of
// fp32 partial results.
constexpr int64_t kMinPart = 4;

// Ints that the items may take in all.
constexpr int64_t kMaxInts = int64_t(1) << 30;

int64_t steps(const PackedItem& it) { return std::max(0, it.j1 - it.j0); }

}  // namespace

// Empty if the plan's counts do not fit in 31 bits.
std::vector<int32_t> make_packed_plan(const int64_t* lens_q, const int64_t* lens_k, int64_t n,
                                      int group, int heads_kv, bool causal, int sms) {
  const int64_t tokens = std::max(1, ENIGMA_PACKED_TILE_ROWS / group);
  std::vector<PackedItem> pairs;
  int64_t q0 = 0, k0 = 0, total = 0, longest = 0;
  for (int64_t s = 0; s < n; ++s) {
    const int64_t lq = lens_q[s], lk = lens_k[s];
    for (int64_t t0 = 0; t0 < lq; t0 += 2 * tokens) {
      PackedItem p;
      std::memset(&p, 0, sizeof(p));
      p.q0 = int(q0);
      p.lq = int(lq);
      p.k0 = int(k0);
      p.lk = int(lk);
      p.t0 = int(t0);
      p.tokens = int(tokens);
      const int64_t last = std::min(t0 + 2 * tokens, lq) - 1;
      const int64_t keys = causal ? std::min(lk, last + lk - lq + 1) : lk;
      p.j1 = keys > 0 ? int((keys + 127) / 128) : 0;
      p.slot = -1;
      total += (steps(p) + kItemCost) * heads_kv;
      longest = std::max(longest, steps(p) + kItemCost);
      pairs.push_back(p);
      // Refused before the list is made: it may not fit in the host's memory either.
      if (int64_t(pairs.size()) > kMaxInts / kItemInts / heads_kv) return {};
    }
    q0 += lq;
    k0 += lk;
  }
  // Split only where one item would outlast the others: parts of about an SM's fair share.
  const int64_t share = (total + sms - 1) / sms;
  const bool split = group <= ENIGMA_PACKED_TILE_ROWS && longest > share + share / 2;
  const int64_t part = std::max(kMinPart, share);
  std::vector<PackedItem> items;
  std::vector<PackedGroup> groups;
  int64_t slots = 0;
  for (const PackedItem& p : pairs) {
    for (int h = 0; h < heads_kv; ++h) {
      PackedItem it = p;
      it.kvh = h;
      const int64_t tiles = it.j1;
      const int64_t parts = split ? std::max<int64_t>(1, (tiles + part - 1) / part) : 1;
      if (parts == 1) {
        items.push_back(it);
        continue;
      }
      PackedGroup g;
      std::memset(&g, 0, sizeof(g));
      g.tok0 = it.q0 + it.t0;
      g.tok_end = it.q0 + it.lq;
      g.tokens = it.tokens;
      g.kvh = h;
      g.slot = int(slots);
      g.parts = int(parts);
      groups.push_back(g);
      for (int64_t x = 0; x < parts; ++x) {
        it.j0 = int(tiles * x / parts);
        it.j1 = int(tiles * (x + 1) / parts);
        it.slot = int(slots);
        slots += 2;
        items.push_back(it);
      }
      if (int64_t(items.size()) > kMaxInts / kItemInts) return {};
    }
  }
  // Heaviest first (equal ones in order: neighbours share K and V), each to the least loaded.
  std::stable_sort(items.begin(), items.end(), [](const PackedItem& x, const PackedItem& y) {
    return steps(x) > steps(y);
  });
  const int ctas = int(std::min<int64_t>(sms, int64_t(items.size())));
  std::vector<std::vector<int>> lists;
  lists.resize(size_t(ctas));
  using Load = std::pair<int64_t, int>;
  std::priority_queue<Load, std::vector<Load>, std::greater<Load>> least;
  for (int c = 0; c < ctas; ++c) least.push({0, c});
  for (size_t i = 0; i < items.size(); ++i) {
    Load l = least.top();
    least.pop();
    lists[size_t(l.second)].push_back(int(i));
    l.first += steps(items[i]) + kItemCost;
    least.push(l);
  }
  const int64_t items_at = (kOffsetsAt + ctas + 1 + 3) / 4 * 4;
  const int64_t groups_at = items_at + int64_t(items.size()) * kItemInts;
  std::vector<int32_t> out(size_t(groups_at + int64_t(groups.size()) * kGroupInts), 0);
  out[kItems] = int32_t(items.size());
  out[kCtas] = ctas;
  out[kSlots] = int32_t(slots);
  out[kGroups] = int32_t(groups.size());
  out[kItemsAt] = int32_t(items_at);
  out[kGroupsAt] = int32_t(groups_at);
  out[kInts] = int32_t(out.size());
  out[kLongest] = items.empty() ? 0 : int32_t(steps(items[0]));
  int32_t* to = out.data() + items_at;
  int done = 0;
  for (int c = 0; c < ctas; ++c) {
    out[size_t(kOffsetsAt + c)] = done;
    for (int i : lists[size_t(c)]) {
      std::memcpy(to, &items[size_t(i)], sizeof(PackedItem));
      to += kItemInts;
      ++done;
    }
  }
  out[size_t(kOffsetsAt + ctas)] = done;
  if (!groups.empty())
    std::memcpy(out.data() + groups_at, groups.data(), groups.size() * sizeof(PackedGroup));
  return out;
}

}  // namespace enigma_serving
