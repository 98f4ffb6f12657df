// kv_cache.cu — the page map of a paged key/value cache and the page copies it asks for.
//
// A cache holds `pages` pages of `page` tokens for each layer; a sequence (slot) owns a row of
// the table: the page of its tokens [c * page, (c + 1) * page) in column c, -1 past its end.
// refs[p] counts the rows that hold page p; a page with refs 0 is free.  Only full pages are
// shared: a fork copies the partly filled last page, so a slot may append without looking
// whether somebody else reads the page.
//
// Every change of the map is one launch of one 8-CTA cluster (cache_map_kernel): "check the
// request", "change refs" and "write rows" need each other's results, and a cluster barrier (well
// under a microsecond) is the cheapest way to order them.  It is bound by the latency of its
// dependent loads (request -> lengths | table rows | refs | free list), so each is made once, the
// request is kept in shared memory, and every CTA lists the free pages for itself instead of
// waiting for the others' counts.  New pages are the lowest free ones, in the order of the
// request, so the result does not depend on timing.  A request that is malformed or does not fit
// changes nothing but the status word.
#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace {

using namespace enigma_sm100;

constexpr int MAP_CTAS = 8;
constexpr int MAP_THREADS = 1024;
constexpr int WS_HEAD = 64;            // ints before the lists: [0] = number of page copies
constexpr int MAX_REQUEST = ENIGMA_CACHE_MAX_REQUEST;

enum Mode { kFork, kFree, kReserve };

struct Map {
  int32_t *table, *lens, *refs, *status;
  int32_t* ws;                         // WS_HEAD + 4 lists of `cap` ints
  int64_t cap;                         // max(slots, pages)
  int slots, pages, width, page;
  __host__ __device__ int32_t* src() const { return ws + WS_HEAD; }
  __host__ __device__ int32_t* dst() const { return src() + cap; }
  __host__ __device__ int32_t* fill() const { return dst() + cap; }
  __host__ __device__ int32_t* freed() const { return fill() + cap; }
};

// Exclusive prefix sum of v over the block (MAP_THREADS threads); *total gets the sum.
__device__ int block_scan(int v, int* s_warp, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int t = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += y;
    }
    s_warp[lane] = t;
  }
  __syncthreads();
  const int before = warp > 0 ? s_warp[warp - 1] : 0;
  *total = s_warp[31];
  __syncthreads();
  return before + x - v;
}

// Publishes one int of this CTA to every CTA of the cluster (slot `rank` of their s_all).
__device__ __forceinline__ void publish(int* s_all, uint32_t rank, int v) {
  if (threadIdx.x < MAP_CTAS) {
    const uint32_t a = mapa_shared(smem_u32(s_all + rank), threadIdx.x);
    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
  }
}

__device__ __forceinline__ int pages_of(int len, int page) {
  return int((uint32_t(len) + uint32_t(page) - 1u) / uint32_t(page));
}

// a: parents (fork) or slots; b: children (fork) or target lengths (reserve).
template <int MODE>
__global__ void __cluster_dims__(MAP_CTAS, 1, 1) __launch_bounds__(MAP_THREADS, 1)
cache_map_kernel(const Map m, const int32_t* __restrict__ a, const int32_t* __restrict__ b, int n) {
  extern __shared__ int s_req[];                 // [n] each: slot, parent or target, tokens, start
  int *s_slot = s_req, *s_other = s_req + n, *s_len = s_req + 2 * n, *s_start = s_req + 3 * n;
  uint32_t* s_bits = reinterpret_cast<uint32_t*>(s_req + 4 * n);    // one bit per slot: named
  __shared__ int s_warp[32];
  __shared__ unsigned long long s_need;          // pages asked for: may be more than an int holds
  const uint32_t rank = cluster_ctarank();
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = int(rank) * (MAP_THREADS / 32) + (tid >> 5);     // of the cluster
  constexpr int WARPS = MAP_CTAS * MAP_THREADS / 32;
  griddep_launch_dependents();
  for (int i = tid; i < (m.slots + 31) / 32; i += MAP_THREADS) s_bits[i] = 0;
  if (tid == 0) s_need = 0;
  griddep_wait();

  // Check the request; every CTA does it for itself and comes to the same answer, since
  // nothing is written before the barrier that follows.  s_len: tokens of the parent (fork), of
  // the slot (free, reserve).
  bool bad = false;
  for (int i = tid; i < n; i += MAP_THREADS) {
    const int c = MODE == kFork ? b[i] : a[i];
    const int other = MODE == kFork ? a[i] : MODE == kReserve ? b[i] : 0;
    const int from = MODE == kFork ? other : c;
    const bool in = c >= 0 && c < m.slots && from >= 0 && from < m.slots;
    const int len = in ? m.lens[from] : 0;
    bad |= !in || len < 0 || int64_t(len) > int64_t(m.width) * m.page;
    if (MODE == kReserve) bad |= other < len || int64_t(other) > int64_t(m.width) * m.page;
    s_slot[i] = c;
    s_other[i] = other;
    s_len[i] = len;
  }
  __syncthreads();
  for (int i = tid; i < n; i += MAP_THREADS) {
    const int c = s_slot[i];
    const uint32_t bit = 1u << (c & 31);
    if (c >= 0 && c < m.slots) bad |= (atomicOr(&s_bits[c >> 5], bit) & bit) != 0;   // named twice
  }
  if (MODE == kFork) {
    __syncthreads();
    for (int i = tid; i < n; i += MAP_THREADS) {
      const int p = s_other[i];
      bad |= p >= 0 && p < m.slots && (s_bits[p >> 5] >> (p & 31) & 1u);   // a parent among them
    }
  }
  if (__syncthreads_or(bad)) {
    if (rank == 0 && tid == 0) {
      atomicOr(m.status, ENIGMA_CACHE_BAD_REQUEST);
      m.ws[0] = 0;
    }
    return;
  }
  cluster_sync();

  // References: children (or freed slots) let go of their pages, parents' full pages gain one.  A
  // warp per entry, its lanes along the row.
  auto change_refs = [&](int by) {
    for (int i = warp; i < n; i += WARPS) {
      int32_t* row = m.table + int64_t(s_slot[i]) * m.width;
      const int32_t* from = m.table + int64_t(s_other[i]) * m.width;
      const int full = MODE == kFork ? s_len[i] / m.page : 0;
      for (int col = lane; col < m.width; col += 32) {
        const int e = row[col];
        const int f = col < full ? from[col] : -1;
        if (e >= 0 && e < m.pages) atomicAdd(&m.refs[e], -by);
        if (f >= 0 && f < m.pages) atomicAdd(&m.refs[f], by);
        if (MODE == kFree) row[col] = -1;
      }
      if (MODE == kFree && lane == 0) m.lens[s_slot[i]] = 0;
    }
  };
  if (MODE != kReserve) change_refs(1);
  if (MODE == kFree) return;

  // Pages each entry needs, and where its first one is in the list.
  int need = 0;
  for (int i0 = 0; i0 < n; i0 += MAP_THREADS) {
    const int i = i0 + tid;
    int w = 0, got = 0;
    if (i < n)
      w = MODE == kFork ? (s_len[i] % m.page ? 1 : 0)
                        : pages_of(s_other[i], m.page) - pages_of(s_len[i], m.page);
    if (w > 0) atomicAdd(&s_need, static_cast<unsigned long long>(w));
    const int at = need + block_scan(w, s_warp, &got);
    if (i < n) s_start[i] = at;
    need += got;                                 // (wraps only where s_need says "does not fit")
  }
  if (MODE == kFork) cluster_sync();             // every change of refs is made (reserve: none was)

  // The `need` lowest free pages.  A thread looks at a run of pages; refs were changed by
  // atomics, so they are read from L2.  Every CTA writes the same list.
  const int per = (m.pages + MAP_THREADS - 1) / MAP_THREADS;
  const int p0 = min(tid * per, m.pages), p1 = min(p0 + per, m.pages);
  int mine = 0, total = 0;
  for (int p = p0; p < p1; ++p) mine += __ldcg(&m.refs[p]) == 0;
  int at = block_scan(mine, s_warp, &total);
  if (s_need > static_cast<unsigned long long>(total)) {   // does not fit: as it was
    cluster_sync();                              // everyone has counted
    if (MODE == kFork) change_refs(-1);
    if (rank == 0 && tid == 0) {
      atomicOr(m.status, ENIGMA_CACHE_FULL);
      m.ws[0] = 0;
    }
    return;
  }
  for (int p = p0; p < p1 && at < need && mine > 0; ++p)
    if (__ldcg(&m.refs[p]) == 0) m.freed()[at++] = p;
  if (rank == 0 && tid == 0) m.ws[0] = MODE == kFork ? need : 0;
  cluster_sync();                                // refs are read, the list is written

  for (int i = warp; i < n; i += WARPS) {
    int32_t* row = m.table + int64_t(s_slot[i]) * m.width;
    const int start = s_start[i];
    if (MODE == kFork) {
      const int32_t* from = m.table + int64_t(s_other[i]) * m.width;
      const int len = s_len[i], full = len / m.page, part = len % m.page;
      for (int col = lane; col < m.width; col += 32) {
        int e = col <= full ? from[col] : -1;
        if (col == full) {
          if (part) {
            m.src()[start] = e;
            e = __ldcg(&m.freed()[start]);
            m.dst()[start] = e;
            m.fill()[start] = part;
            m.refs[e] = 1;
          } else {
            e = -1;
          }
        }
        row[col] = e;
      }
      if (lane == 0) m.lens[s_slot[i]] = len;
    } else {
      const int held = pages_of(s_len[i], m.page), want = pages_of(s_other[i], m.page);
      for (int col = held + lane; col < want; col += 32) {
        const int e = __ldcg(&m.freed()[start + col - held]);
        m.refs[e] = 1;
        row[col] = e;
      }
      if (lane == 0) m.lens[s_slot[i]] = s_other[i];
    }
  }
}

// The n live pages take the numbers below n: live pages at or above n move, in order, to the
// holes below n.  Lists source, destination (whole pages) and rewrites refs and the table.
__global__ void __cluster_dims__(MAP_CTAS, 1, 1) __launch_bounds__(MAP_THREADS, 1)
cache_compact_kernel(const Map m) {
  __shared__ int s_warp[32];
  __shared__ int s_all[MAP_CTAS], s_low[MAP_CTAS];
  const uint32_t rank = cluster_ctarank();
  const int tid = threadIdx.x, gtid = int(rank) * MAP_THREADS + tid;
  constexpr int GT = MAP_CTAS * MAP_THREADS;
  const int per = (m.pages + MAP_CTAS - 1) / MAP_CTAS;
  const int p0 = min(int(rank) * per, m.pages), p1 = min(p0 + per, m.pages);
  griddep_launch_dependents();
  griddep_wait();
  cluster_sync();                      // every CTA runs before its shared memory is written
  int mine = 0, counted = 0;
  for (int p = p0 + tid; p < p1; p += MAP_THREADS) mine += m.refs[p] > 0;
  block_scan(mine, s_warp, &counted);
  publish(s_all, rank, counted);
  cluster_sync();
  int live = 0;
#pragma unroll
  for (int r = 0; r < MAP_CTAS; ++r) live += s_all[r];
  // Live pages below `live` stay; the number of the others is the number of holes.
  mine = 0;
  for (int p = p0 + tid; p < min(p1, live); p += MAP_THREADS) mine += m.refs[p] > 0;
  block_scan(mine, s_warp, &counted);
  publish(s_low, rank, counted);
  cluster_sync();
  int low = 0, before = 0;             // live pages below `live`; live pages below p0
#pragma unroll
  for (int r = 0; r < MAP_CTAS; ++r) {
    low += s_low[r];
    if (r < int(rank)) before += s_all[r];
  }
  int32_t* remap = m.freed();
  for (int q = p0; q < p1; q += MAP_THREADS) {
    const int p = q + tid;
    const bool in = p < p1;
    const bool is_live = in && m.refs[p] > 0;
    int got = 0;
    const int below = before + block_scan(is_live ? 1 : 0, s_warp, &got);   // live pages below p
    before += got;
    if (in) {
      remap[p] = p;
      if (p < live && !is_live) m.dst()[p - below] = p;
      if (p >= live && is_live) m.src()[below - low] = p;
    }
  }
  cluster_sync();
  const int moved = live - low;
  for (int i = gtid; i < moved; i += GT) {
    const int s = __ldcg(&m.src()[i]), d = __ldcg(&m.dst()[i]);
    remap[s] = d;
    m.refs[d] = m.refs[s];
    m.refs[s] = 0;
    m.fill()[i] = m.page;
  }
  if (gtid == 0) m.ws[0] = moved;
  cluster_sync();
  const int64_t cells = int64_t(m.slots) * m.width;
  for (int64_t x = gtid; x < cells; x += GT) {
    const int e = m.table[x];
    if (e >= 0 && e < m.pages) {
      const int to = __ldcg(&remap[e]);
      if (to != e) m.table[x] = to;
    }
  }
}

// ------------------------------------------------------------------------------ page copies
struct Copy {
  uint8_t *k, *v;
  const int32_t *src, *dst, *fill;     // fill NULL: whole pages
  const int32_t* count;                // on the device: copies to make
  int32_t* status;
  int64_t layer_bytes;                 // one layer of K (or V)
  int64_t head_bytes;                  // one head of a page
  int layers, heads, pages, page, row_bytes;      // row_bytes: head_dim * element size
};

// Pages that a caller names: checked as a whole before any is copied; ws[0] = copies to make.
__global__ void __launch_bounds__(MAP_THREADS)
cache_copy_check_kernel(const int32_t* __restrict__ src, const int32_t* __restrict__ dst, int n,
                        int pages, int32_t* ws, int32_t* status) {
  griddep_launch_dependents();
  griddep_wait();
  bool bad = false;
  for (int i = threadIdx.x; i < n; i += MAP_THREADS) {
    const int s = src[i], d = dst[i];
    bad |= s < 0 || s >= pages || d < 0 || d >= pages;
  }
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0) {
    ws[0] = bad ? 0 : n;
    if (bad) atomicOr(status, ENIGMA_CACHE_BAD_REQUEST);
  }
}

// Units of one (copy, layer, K or V, head): fill * row_bytes contiguous bytes.  Bound by HBM; small
// blocks and many of them, so that the hardware keeps all SMs' requests going: 128 threads, up
// to 256 blocks per SM 6.4 TB/s (1 GB moved, read and written; 8 blocks of 256 threads per SM:
// 5.8), while as many blocks as there could be copies costs their start (131072: 5.4).
constexpr int COPY_THREADS = 128;
template <typename V>
__global__ void __launch_bounds__(COPY_THREADS) cache_copy_kernel(const Copy c) {
  griddep_launch_dependents();
  griddep_wait();
  const int64_t units = int64_t(*c.count) * c.layers * 2 * c.heads;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int head = int(u % c.heads);
    int64_t r = u / c.heads;
    uint8_t* base = (r & 1) ? c.v : c.k;
    r >>= 1;
    const int layer = int(r % c.layers), i = int(r / c.layers);
    const int s = c.src[i], d = c.dst[i];
    if (s < 0 || s >= c.pages || d < 0 || d >= c.pages) {
      if (threadIdx.x == 0) atomicOr(c.status, ENIGMA_CACHE_BAD_REQUEST);
      continue;
    }
    const int rows = c.fill != nullptr ? c.fill[i] : c.page;
    const int64_t page_bytes = c.head_bytes * c.heads;
    uint8_t* at = base + layer * c.layer_bytes + head * c.head_bytes;
    const V* from = reinterpret_cast<const V*>(at + s * page_bytes);
    V* to = reinterpret_cast<V*>(at + d * page_bytes);
    const int vecs = int(int64_t(rows) * c.row_bytes / int64_t(sizeof(V)));
    // Four loads in flight before their stores (the two may not overlap, which the compiler
    // cannot know).
    for (int x = threadIdx.x; x < vecs; x += 4 * COPY_THREADS) {
      V v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (x + u * COPY_THREADS < vecs) v[u] = from[x + u * COPY_THREADS];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (x + u * COPY_THREADS < vecs) to[x + u * COPY_THREADS] = v[u];
    }
  }
}

// ------------------------------------------------------------------------ new tokens' rows
struct Write {
  uint8_t *k, *v;                      // the layer's pages
  const uint8_t *new_k, *new_v;
  const int32_t *table, *slots, *starts, *cu;
  int32_t* status;
  int64_t k_token, k_head, v_token, v_head;   // byte strides of the new rows
  int64_t head_bytes;
  int n, tokens, heads, slots_total, pages, width, page, row_bytes;
};

// One warp per token, its lanes along the rows of K, then V.  The row's first loads are made before
// its place is known: sequence (cu is searched 32 ways at once), table, page, store.
template <typename V>
__global__ void __launch_bounds__(256) cache_write_kernel(const Write w) {
  const int lane = threadIdx.x & 31;
  const int warps = int(gridDim.x) * 8;
  const int per = w.row_bytes / int(sizeof(V)), row = w.heads * per;     // vectors: head, token
  griddep_launch_dependents();
  griddep_wait();
  for (int t = int(blockIdx.x) * 8 + (threadIdx.x >> 5); t < w.tokens; t += warps) {
    auto source = [&](int x) {
      const bool is_v = x >= row;
      const int y = is_v ? x - row : x, h = y / per, e = y - h * per;
      return reinterpret_cast<const V*>(is_v ? w.new_v + t * w.v_token + h * w.v_head
                                             : w.new_k + t * w.k_token + h * w.k_head) + e;
    };
    V first = V();
    if (lane < 2 * row) first = *source(lane);
    // The last i in [0, n) with cu[i] <= t, in [lo, lo + span).
    int lo = 0, span = w.n;
    while (span > 1) {
      const int step = (span + 31) / 32, i = lo + (lane + 1) * step;
      const bool past = i >= lo + span || w.cu[i] > t;
      const int k = __ffs(__ballot_sync(0xffffffffu, past)) - 1;         // lane 31 is always past
      span = min(step, lo + span - (lo + k * step));
      lo += k * step;
    }
    const int slot = w.slots[lo];
    const int64_t pos = int64_t(w.starts[lo]) + t - w.cu[lo];
    int at = -1;
    if (t >= w.cu[0] && t < w.cu[w.n] && slot >= 0 && slot < w.slots_total && pos >= 0 &&
        pos / w.page < w.width)
      at = w.table[int64_t(slot) * w.width + pos / w.page];
    if (at < 0 || at >= w.pages) {
      if (lane == 0) atomicOr(w.status, ENIGMA_CACHE_BAD_REQUEST);
      continue;
    }
    const int64_t to = at * w.head_bytes * w.heads + (pos % w.page) * w.row_bytes;
    for (int x = lane; x < 2 * row; x += 32) {
      const bool is_v = x >= row;
      const int y = is_v ? x - row : x, h = y / per, e = y - h * per;
      const V v = x == lane ? first : *source(x);
      reinterpret_cast<V*>((is_v ? w.v : w.k) + to + h * w.head_bytes)[e] = v;
    }
  }
}

Map make_map(const enigma_kv_cache_desc& d) {
  Map m;
  m.table = d.table;
  m.lens = d.lens;
  m.refs = d.refs;
  m.status = d.status;
  m.ws = static_cast<int32_t*>(d.workspace);
  m.cap = std::max(d.slots, d.pages);
  m.slots = int(d.slots);
  m.pages = int(d.pages);
  m.width = int(d.table_width);
  m.page = int(d.page);
  return m;
}

bool a16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// *count copies (on the device), at most n.
cudaError_t launch_copy(const enigma_kv_cache_desc& d, const int32_t* src, const int32_t* dst,
                        const int32_t* fill, const int32_t* count, int64_t n, cudaStream_t s) {
  Copy c;
  c.k = static_cast<uint8_t*>(d.k);
  c.v = static_cast<uint8_t*>(d.v);
  c.src = src;
  c.dst = dst;
  c.fill = fill;
  c.count = count;
  c.status = d.status;
  c.row_bytes = int(d.head_dim * d.elem_bytes);
  c.head_bytes = d.page * c.row_bytes;
  c.layer_bytes = d.pages * d.heads_kv * c.head_bytes;
  c.layers = int(d.layers);
  c.heads = int(d.heads_kv);
  c.pages = int(d.pages);
  c.page = int(d.page);
  const int64_t units = n * d.layers * 2 * d.heads_kv;
  const unsigned grid = unsigned(std::min<int64_t>(units, int64_t(enigma::sm_count()) * 256));
  if (grid == 0) return cudaSuccess;
  if (c.row_bytes % 16 == 0 && a16(d.k) && a16(d.v))
    return enigma::launch_dependent(cache_copy_kernel<uint4>, grid, COPY_THREADS, 0, s, c);
  return enigma::launch_dependent(cache_copy_kernel<uint16_t>, grid, COPY_THREADS, 0, s, c);
}

template <int MODE>
cudaError_t launch_map(const enigma_kv_cache_desc& d, const int32_t* a, const int32_t* b, int64_t n,
                       cudaStream_t s) {
  const size_t smem = size_t(n) * 16 + size_t((d.slots + 31) / 32) * 4;
  static std::atomic<uint64_t> ready{0};                    // devices where the attribute is set
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && !(dev < 64 && (ready.load() >> dev & 1))) {
    e = cudaFuncSetAttribute(cache_map_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             MAX_REQUEST * 16 + 262144 / 8);
    if (e == cudaSuccess && dev < 64) ready.fetch_or(uint64_t(1) << dev);
  }
  if (e != cudaSuccess) return e;
  return enigma::launch_dependent(cache_map_kernel<MODE>, MAP_CTAS, MAP_THREADS, smem, s, make_map(d),
                                  a, b, int(n));
}

}  // namespace

namespace enigma {

size_t kv_cache_workspace_bytes(const enigma_kv_cache_desc& d) {
  return size_t(WS_HEAD + 4 * std::max(d.slots, d.pages)) * sizeof(int32_t);
}

cudaError_t kv_cache_fork(const enigma_kv_cache_desc& d, const int32_t* parents,
                          const int32_t* children, int64_t n, cudaStream_t s) {
  note_kernel("cache_map_kernel");
  const cudaError_t e = launch_map<kFork>(d, parents, children, n, s);
  if (e != cudaSuccess) return e;
  const Map m = make_map(d);
  return launch_copy(d, m.src(), m.dst(), m.fill(), m.ws, n, s);
}

cudaError_t kv_cache_free(const enigma_kv_cache_desc& d, const int32_t* slots, int64_t n,
                          cudaStream_t s) {
  note_kernel("cache_map_kernel");
  return launch_map<kFree>(d, slots, nullptr, n, s);
}

cudaError_t kv_cache_reserve(const enigma_kv_cache_desc& d, const int32_t* slots,
                             const int32_t* lens, int64_t n, cudaStream_t s) {
  note_kernel("cache_map_kernel");
  return launch_map<kReserve>(d, slots, lens, n, s);
}

cudaError_t kv_cache_compact(const enigma_kv_cache_desc& d, cudaStream_t s) {
  note_kernel("cache_compact_kernel");
  const Map m = make_map(d);
  const cudaError_t e =
      enigma::launch_dependent(cache_compact_kernel, MAP_CTAS, MAP_THREADS, 0, s, m);
  if (e != cudaSuccess) return e;
  // At most half of the pages move: each moved page has a hole of its own.
  return launch_copy(d, m.src(), m.dst(), nullptr, m.ws, d.pages / 2, s);
}

cudaError_t kv_cache_copy_pages(const enigma_kv_cache_desc& d, const int32_t* src,
                                const int32_t* dst, int64_t n, cudaStream_t s) {
  note_kernel("cache_copy_kernel");
  const Map m = make_map(d);
  const cudaError_t e = enigma::launch_dependent(cache_copy_check_kernel, 1, MAP_THREADS, 0, s, src,
                                                 dst, n, d.pages, m.ws, d.status);
  return e == cudaSuccess ? launch_copy(d, src, dst, nullptr, m.ws, n, s) : e;
}

cudaError_t kv_cache_write(const enigma_kv_cache_desc& d, int64_t layer, const void* new_k,
                           const void* new_v, const int64_t* strides4, const int32_t* slots,
                           const int32_t* starts, const int32_t* cu, int64_t n, int64_t tokens,
                           cudaStream_t s) {
  note_kernel("cache_write_kernel");
  Write w;
  w.row_bytes = int(d.head_dim * d.elem_bytes);
  w.head_bytes = d.page * w.row_bytes;
  const int64_t layer_bytes = d.pages * d.heads_kv * w.head_bytes;
  w.k = static_cast<uint8_t*>(d.k) + layer * layer_bytes;
  w.v = static_cast<uint8_t*>(d.v) + layer * layer_bytes;
  w.new_k = static_cast<const uint8_t*>(new_k);
  w.new_v = static_cast<const uint8_t*>(new_v);
  w.table = d.table;
  w.slots = slots;
  w.starts = starts;
  w.cu = cu;
  w.status = d.status;
  w.k_token = strides4[0] * d.elem_bytes;
  w.k_head = strides4[1] * d.elem_bytes;
  w.v_token = strides4[2] * d.elem_bytes;
  w.v_head = strides4[3] * d.elem_bytes;
  w.n = int(n);
  w.tokens = int(tokens);
  w.heads = int(d.heads_kv);
  w.slots_total = int(d.slots);
  w.pages = int(d.pages);
  w.width = int(d.table_width);
  w.page = int(d.page);
  const unsigned grid =
      unsigned(std::min<int64_t>((tokens + 7) / 8, int64_t(sm_count()) * 8));
  const bool vec = w.row_bytes % 16 == 0 && a16(w.k) && a16(w.v) && a16(new_k) && a16(new_v) &&
                   w.k_token % 16 == 0 && w.k_head % 16 == 0 && w.v_token % 16 == 0 &&
                   w.v_head % 16 == 0;
  return vec ? enigma::launch_dependent(cache_write_kernel<uint4>, grid, 256, 0, s, w)
             : enigma::launch_dependent(cache_write_kernel<uint16_t>, grid, 256, 0, s, w);
}

}  // namespace enigma
