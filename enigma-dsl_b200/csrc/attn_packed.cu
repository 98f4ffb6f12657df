// attn_packed.cu — attention over packed prompts: the tensor-core kernel of attn_tc.cuh over the
// plan's items, and the join of rows whose keys the plan split.
#include <algorithm>

#include "attn_tc.cuh"

namespace {

using namespace enigma_tc;
using namespace enigma_serving;

// Joins the partial results of split rows: O = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i, in
// the order of the parts.  One warp per row; grid (groups, row blocks).
template <int D>
__global__ void __launch_bounds__(256)
packed_join_kernel(const PackedGroup* __restrict__ groups, const float* __restrict__ opart,
                   const float2* __restrict__ ml, const Params p) {
  const int lane = threadIdx.x & 31;
  const int r = int(blockIdx.y) * 8 + (threadIdx.x >> 5);       // row of the pair of tiles
  const PackedGroup g = groups[blockIdx.x];
  const int state = r / BM, row = r % BM;
  const int tok = g.tok0 + state * g.tokens + row / p.group;
  if (row >= g.tokens * p.group || tok >= g.tok_end || (g.alt && state > 0)) return;
  const int n = g.alt ? 2 * g.parts : g.parts, step = g.alt ? 1 : 2;
  const int64_t first = g.slot + (g.alt ? 0 : state);
  float M = -INFINITY;
  for (int i = lane; i < n; i += 32) M = fmaxf(M, ml[(first + i * step) * BM + row].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  constexpr int V = D / 32;
  float acc[V] = {};
  float l = 0.f;
  for (int i = 0; i < n; ++i) {
    const int64_t at = (first + i * step) * BM + row;
    const float2 x = ml[at];
    if (x.x == -INFINITY) continue;                             // this part saw no key
    const float f = ex2(x.x - M);
    l = fmaf(x.y, f, l);
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = fmaf(opart[at * D + lane * V + v], f, acc[v]);
  }
  const int h = g.kvh * p.group + row % p.group;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __nv_bfloat16* out = p.out + tok * p.o_token + h * p.o_head + lane * V;
#pragma unroll
  for (int v = 0; v < V; v += 2)
    *reinterpret_cast<uint32_t*>(out + v) = pack_bf16x2(acc[v] * inv, acc[v + 1] * inv);
  if (p.lse != nullptr && lane == 0)
    p.lse[int64_t(tok) * p.heads_q + h] =
        l == 0.f ? -INFINITY : (M + log2f(l)) * 0.6931471805599453f;
}

bool a16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// The tensor-core kernel takes bf16 heads of 64 or 128 whose rows TMA can address: base and
// strides multiples of 16 bytes (8 elements), and a group that fits a tile.
bool tc_takes(const enigma_sdpa_packed_desc& d) {
  const int64_t st[8] = {d.q_token, d.q_head, d.k_token, d.k_head,
                         d.v_token, d.v_head, d.o_token, d.o_head};
  for (int i = 0; i < 8; ++i)
    if (st[i] % 8 != 0 || st[i] <= 0 || st[i] >= (int64_t(1) << 39)) return false;
  return d.dtype == ENIGMA_DTYPE_BF16 && (d.head_dim == 64 || d.head_dim == 128) &&
         d.tokens_k > 0 && d.heads_q / d.heads_kv <= BM && a16(d.q) && a16(d.k) && a16(d.v) &&
         a16(d.out);
}

// [head_dim, heads, tokens] with boxes of 64 x `heads` x `tokens`.
bool rows_map(CUtensorMap* m, const void* base, int64_t D, int64_t heads, int64_t tokens,
              int64_t head_stride, int64_t token_stride, int box_heads, int box_tokens) {
  const cuuint64_t dims[3] = {cuuint64_t(D), cuuint64_t(heads), cuuint64_t(tokens)};
  const cuuint64_t strides[2] = {cuuint64_t(head_stride * 2), cuuint64_t(token_stride * 2)};
  const cuuint32_t box[3] = {64, cuuint32_t(box_heads), cuuint32_t(box_tokens)};
  return make_map(m, base, 3, dims, strides, box);
}

template <int D>
cudaError_t launch(const enigma_sdpa_packed_desc& d, cudaStream_t s) {
  const int group = int(d.heads_q / d.heads_kv), tokens = std::max(1, BM / group);
  CUtensorMap mq, mk, mv;
  if (!rows_map(&mq, d.q, D, d.heads_q, d.tokens_q, d.q_head, d.q_token, group, tokens) ||
      !rows_map(&mk, d.k, D, d.heads_kv, d.tokens_k, d.k_head, d.k_token, 1, BN) ||
      !rows_map(&mv, d.v, D, d.heads_kv, d.tokens_k, d.v_head, d.v_token, 1, BN))
    return cudaErrorInvalidValue;
  cudaError_t e = prepare_kernel<D, false>();
  if (e != cudaSuccess) return e;
  Params p = {};
  p.scale_log2 = d.scale * 1.4426950408889634f;
  p.group = group;
  p.tokens = tokens;
  p.status = enigma::device_status();
  if (p.status == nullptr) return cudaErrorMemoryAllocation;   // the bounded waits need it
  p.opart = static_cast<float*>(d.workspace);
  p.ml = reinterpret_cast<float2*>(p.opart + int64_t(d.header[kSlots]) * BM * D);
  p.offsets = d.plan + kOffsetsAt;
  p.list = d.plan + d.header[kItemsAt];
  p.out = static_cast<__nv_bfloat16*>(d.out);
  p.lse = d.lse;
  p.o_token = d.o_token;
  p.o_head = d.o_head;
  p.heads_q = int(d.heads_q);
  p.causal = d.causal != 0;
  p.tokens_q = int(d.tokens_q);
  p.tokens_k = int(d.tokens_k);
  attn_tc_kernel<D, false><<<unsigned(d.header[kCtas]), THREADS, Cfg<D>::SMEM, s>>>(
      mq, mk, mv, p, d.header[kItems]);
  e = cudaGetLastError();
  if (e != cudaSuccess || d.header[kGroups] == 0) return e;
  packed_join_kernel<D><<<dim3(unsigned(d.header[kGroups]), 2 * BM / 8), 256, 0, s>>>(
      reinterpret_cast<const PackedGroup*>(d.plan + d.header[kGroupsAt]), p.opart, p.ml, p);
  return cudaGetLastError();
}

}  // namespace

namespace enigma {

cudaError_t sdpa_packed_launch(const enigma_sdpa_packed_desc& d, cudaStream_t s) {
  if (!tc_takes(d)) return sdpa_packed_simt_launch(d, s);
  note_kernel("attn_tc_kernel");
  return d.head_dim == 128 ? launch<128>(d, s) : launch<64>(d, s);
}

}  // namespace enigma
