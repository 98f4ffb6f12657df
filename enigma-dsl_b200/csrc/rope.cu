// rope.cu — rotary positions of queries and keys in one launch.
//
// Pair i of a head's first `rotary` elements turns by the angle p * w_i:
//   a' = f (a cos - b sin),  b' = f (b cos + a sin)
// with (a, b) = (x_i, x_{i + rotary / 2}) in the half layout, (x_{2i}, x_{2i+1}) interleaved; the
// elements behind are copied.  The turn back (the transpose, which is also the gradient) has -sin.
//
// Angles: turns[i] is w_i / 2 pi as a 64-bit binary fraction, so p * turns[i] modulo 2^64 is the
// angle modulo a full turn, exactly, for any position; rounding starts at its conversion to fp32.
// (An fp32 product p * w_i is off by p * w_i * 2^-24 radians: 0.06 at a position of a million.)
#include "common.cuh"

namespace {

using namespace enigma_sm100;

struct Rope {
  const void *q, *k, *positions;
  void *out_q, *out_k;
  const uint64_t* turns;
  int64_t q_token, q_head, k_token, k_head, oq_token, oq_head, ok_token, ok_head;
  int64_t tokens;
  int heads_q, heads, d, rotary;         // heads: of q and k
  float factor, sign;                    // sign: -1 turns back
  int wide;                              // positions of 64 bits
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// (f cos, f sin) of position * turns.
__device__ __forceinline__ float2 turn_of(uint64_t position, uint64_t turns, float factor, float sign) {
  const float half_turns = __ll2float_rn(int64_t(position * turns)) * 0x1p-63f;
  float s, c;
  sincospif(half_turns, &s, &c);
  return make_float2(c * factor, s * factor * sign);
}

// A block per token; a thread per pair (or element behind them), for all heads.
template <typename T>
__global__ void __launch_bounds__(256) rope_kernel(const Rope r, bool half) {
  const int64_t t = blockIdx.x;
  const uint64_t p = r.wide ? static_cast<const uint64_t*>(r.positions)[t]
                            : uint64_t(int64_t(static_cast<const int32_t*>(r.positions)[t]));
  const int pairs = r.rotary / 2;
  for (int i = threadIdx.x; i < pairs + r.d - r.rotary; i += 256) {
    const bool turn = i < pairs;
    const int a = !turn ? r.rotary + i - pairs : half ? i : 2 * i, b = half ? i + pairs : a + 1;
    const float2 cs = turn ? turn_of(p, r.turns[i], r.factor, r.sign) : make_float2(1.f, 0.f);
    for (int h = 0; h < r.heads; ++h) {
      const bool is_q = h < r.heads_q;
      const int g = is_q ? h : h - r.heads_q;
      const T* x = is_q ? static_cast<const T*>(r.q) + t * r.q_token + g * r.q_head
                        : static_cast<const T*>(r.k) + t * r.k_token + g * r.k_head;
      T* y = is_q ? static_cast<T*>(r.out_q) + t * r.oq_token + g * r.oq_head
                  : static_cast<T*>(r.out_k) + t * r.ok_token + g * r.ok_head;
      if (!turn) {
        y[a] = x[a];
        continue;
      }
      const float u = to_f(x[a]), v = to_f(x[b]);
      put(y + a, u * cs.x - v * cs.y);
      put(y + b, v * cs.x + u * cs.y);
    }
  }
}

}  // namespace

namespace enigma {

cudaError_t rope_launch(const enigma_rope_desc& d, cudaStream_t s) {
  note_kernel("rope_kernel");
  Rope r;
  r.q = d.q;
  r.k = d.k;
  r.positions = d.positions;
  r.out_q = d.out_q;
  r.out_k = d.out_k;
  r.turns = d.turns;
  r.q_token = d.q_token;
  r.q_head = d.q_head;
  r.k_token = d.k_token;
  r.k_head = d.k_head;
  r.oq_token = d.oq_token;
  r.oq_head = d.oq_head;
  r.ok_token = d.ok_token;
  r.ok_head = d.ok_head;
  r.tokens = d.tokens;
  r.heads_q = int(d.heads_q);
  r.heads = int(d.heads_q + d.heads_k);
  r.d = int(d.head_dim);
  r.rotary = int(d.rotary_dim);
  r.factor = d.factor;
  r.sign = d.inverse ? -1.f : 1.f;
  r.wide = d.position_bytes == 8;
  const bool half = d.layout == ENIGMA_ROPE_HALF;
  if (d.dtype == ENIGMA_DTYPE_F32) rope_kernel<float><<<unsigned(d.tokens), 256, 0, s>>>(r, half);
  else rope_kernel<__nv_bfloat16><<<unsigned(d.tokens), 256, 0, s>>>(r, half);
  return cudaGetLastError();
}

}  // namespace enigma
