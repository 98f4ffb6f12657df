// attn_packed.cu — attention over packed prompts: the tensor-core kernel of attn_tc.cuh over the
// plan's items, or the CUDA-core one, then the join of rows whose keys the plan split.
#include <algorithm>

#include "attn_tc.cuh"

namespace {

using namespace enigma_tc;
using namespace enigma_serving;

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
  p.heads_kv = int(d.heads_kv);
  p.slots_end = std::max(1, d.header[kSlots]);
  p.causal = d.causal != 0;
  p.one = d.header[kItems] == d.header[kCtas];
  p.tokens_q = int(d.tokens_q);
  p.tokens_k = int(d.tokens_k);
  attn_tc_kernel<D, false><<<unsigned(d.header[kCtas]), THREADS, Cfg<D>::SMEM, s>>>(
      mq, mk, mv, p, d.header[kItems]);
  return cudaGetLastError();
}

}  // namespace

namespace enigma {

cudaError_t sdpa_packed_launch(const enigma_sdpa_packed_desc& d, cudaStream_t s) {
  cudaError_t e;
  const bool tc = tc_takes(d);
  if (!tc) {
    e = sdpa_packed_simt_launch(d, s);
  } else {
    note_kernel("attn_tc_kernel");
    e = d.head_dim == 128 ? launch<128>(d, s) : launch<64>(d, s);
  }
  return e == cudaSuccess ? sdpa_packed_join_launch(d, tc, s) : e;
}

}  // namespace enigma
