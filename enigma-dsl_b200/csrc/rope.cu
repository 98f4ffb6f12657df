// rope.cu — rotary positions of queries and keys in one launch.
//
// Pair i of a head's first `rotary` elements turns by the angle p * w_i:
//   a' = f (a cos - b sin),  b' = f (b cos + a sin)
// with (a, b) = (x_i, x_{i + rotary / 2}) in the half layout, (x_{2i}, x_{2i+1}) interleaved; the
// elements behind are copied.  The turn back (the transpose, which is also the gradient) has -sin.
//
// Angles: turns[i] is w_i / 2 pi as a 64-bit binary fraction, so p * turns[i] modulo 2^64 is the
// angle modulo a full turn without any rounding of its own, for any position.  What is off is the
// frequency (made from 64-bit floats: 2^-52 of itself, and half a unit) and the angle's conversion to
// fp32 (pi 2^-24 radians), which is the larger part up to p * w_i of about 2^29.
// (An fp32 product p * w_i is off by p * w_i * 2^-24 radians: 0.06 at a position of a million.)
#include <algorithm>

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
  int parts, part_heads;                 // warps of a token, heads of each
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

// E elements of a head, as one access of 16 bytes at most.
template <typename T, int E>
struct alignas(sizeof(T) * E > 16 ? 16 : sizeof(T) * E) Vec {
  T x[E];
};

// Turns x (and y, the pairs' second elements, where they are apart) by the angles.
template <int E, int PAIRS>
__device__ __forceinline__ void turn_pairs(Vec<float, E>& x, Vec<float, E>& y, const float2 (&angle)[PAIRS]) {
  constexpr bool TWO = PAIRS == E;
#pragma unroll
  for (int e = 0; e < PAIRS; ++e) {
    float& v = TWO ? x.x[e] : x.x[(2 * e) % E];
    float& w = TWO ? y.x[e] : x.x[(2 * e + 1) % E];
    const float f = v, g = w;
    v = f * angle[e].x - g * angle[e].y;
    w = g * angle[e].x + f * angle[e].y;
  }
}
template <int E, int PAIRS>
__device__ __forceinline__ void turn_pairs(Vec<__nv_bfloat16, E>& x, Vec<__nv_bfloat16, E>& y,
                                           const float2 (&angle)[PAIRS]) {
  Vec<float, E> f, g;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    f.x[e] = to_f(x.x[e]);
    g.x[e] = PAIRS == E ? to_f(y.x[e]) : 0.f;
  }
  turn_pairs<E, PAIRS>(f, g, angle);
  if constexpr (E == 1) {
    put(&x.x[0], f.x[0]);
    put(&y.x[0], g.x[0]);
  } else {
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      reinterpret_cast<uint32_t*>(&x)[e / 2] = pack_bf16x2(f.x[e], f.x[e + 1]);
      if (PAIRS == E) reinterpret_cast<uint32_t*>(&y)[e / 2] = pack_bf16x2(g.x[e], g.x[e + 1]);
    }
  }
}

// A warp takes a token, or the heads of one part of it where tokens are few.  It makes the angles
// once, into shared memory; then a lane keeps one unit's (E pairs in the half layout, a vector of
// either half, or two vectors of the elements that are copied, from either half of those; interleaved
// a vector of E / 2 pairs or of copied ones) and turns that unit of every head, or of every second,
// third, ... where a head has less than 32 units: neighbouring lanes touch neighbouring memory.  Bound by
// memory: 8192 tokens of 40 heads of 128, bf16, 28.1 us, 6.0 TB/s; half of each head turned 26.4 for
// 150 MB (39.7 where copied elements had a lane for each vector).  BATCH heads' loads are in flight at
// once, the first through the making of the angles.  They are straight-line code, heads past the last
// being the last again: loads under a condition, or asked for one by one as others arrive, waited for
// one another (42 to 83 us).
// 5 heads (30 us then; 2, 3, 4: 30.5, 30.1, 31.3), or 2 where a warp has no more rounds (64 tokens of
// 16 heads of 64: 2.5 against 2.9 us).
constexpr int WARPS = 4;
constexpr int ANGLE_BYTES = 48 << 10;    // of a block

template <typename T, int E, bool HALF, int BATCH>
__global__ void __launch_bounds__(WARPS * 32) rope_kernel(const __grid_constant__ Rope r) {
  using V = Vec<T, E>;
  constexpr bool TWO = HALF || E == 1;   // a pair's elements come in two vectors
  constexpr int PAIRS = TWO ? E : E / 2;
  extern __shared__ __align__(16) float2 s_angles[];
  const int pairs = r.rotary / 2, turned = pairs / PAIRS;
  const int rest = r.d - r.rotary, units = turned + (TWO ? (rest / E + 1) / 2 : rest / E);
  const int lane = threadIdx.x & 31, warps = int(blockDim.x) >> 5;
  float2* angles = s_angles + (threadIdx.x >> 5) * ((pairs + 1) & ~1);
  const int groups = max(1, 32 / units);                 // heads at once
  griddep_launch_dependents();
  griddep_wait();
  const int64_t w = int64_t(blockIdx.x) * warps + (threadIdx.x >> 5);
  if (w >= r.tokens * r.parts) return;
  const int64_t t = r.parts == 1 ? w : w / r.parts;
  const int h_lo = int(w - t * r.parts) * r.part_heads, h_hi = min(h_lo + r.part_heads, r.heads);
  bool made = false;
  for (int u0 = 0; u0 < units; u0 += 32) {               // (once, but for heads of more than 32 units)
    const int group = units <= 32 ? min(lane / units, groups - 1) : 0;
    const int u = min(u0 + lane - group * units, units - 1);
    const bool has = units <= 32 ? lane < groups * units : u0 + lane < units, turn = u < turned;
    const int e0 = !turn ? r.rotary + (u - turned) * E : HALF || !TWO ? u * E : 2 * u;
    const int apart = !turn ? rest / 2 : HALF ? pairs : 1;
    const T* q = static_cast<const T*>(r.q) + t * r.q_token + e0;
    const T* k = static_cast<const T*>(r.k) + t * r.k_token + e0 - r.heads_q * r.k_head;
    T* out_q = static_cast<T*>(r.out_q) + t * r.oq_token + e0;
    T* out_k = static_cast<T*>(r.out_k) + t * r.ok_token + e0 - r.heads_q * r.ok_head;
    float2 angle[PAIRS];
    for (int h0 = h_lo; h0 < h_hi; h0 += BATCH * groups) {
      V x[BATCH], y[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int h = min(h0 + i * groups + group, h_hi - 1);
        const bool is_q = h < r.heads_q;
        const T* from = (is_q ? q : k) + h * (is_q ? r.q_head : r.k_head);
        x[i] = *reinterpret_cast<const V*>(from);
        if (TWO) y[i] = *reinterpret_cast<const V*>(from + apart);
      }
      if (h0 == h_lo) {
        if (!made) {
          const uint64_t p = r.wide ? static_cast<const uint64_t*>(r.positions)[t]
                                    : uint64_t(int64_t(static_cast<const int32_t*>(r.positions)[t]));
          for (int i = lane; i < pairs; i += 32) angles[i] = turn_of(p, r.turns[i], r.factor, r.sign);
          made = true;
          __syncwarp();
        }
#pragma unroll
        for (int e = 0; e < PAIRS; ++e) angle[e] = turn ? angles[u * PAIRS + e] : make_float2(1.f, 0.f);
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int h = h0 + i * groups + group;
        const bool is_q = h < r.heads_q;
        T* to = (is_q ? out_q : out_k) + h * (is_q ? r.oq_head : r.ok_head);
        const V was = x[i], was_y = y[i];
        turn_pairs<E, PAIRS>(x[i], y[i], angle);
        if (!has || h >= h_hi) continue;
        if (turn) {
          *reinterpret_cast<V*>(to) = x[i];
          if (TWO) *reinterpret_cast<V*>(to + apart) = y[i];
        } else if (to != (is_q ? q : k) + h * (is_q ? r.q_head : r.k_head)) {
          *reinterpret_cast<V*>(to) = was;                   // (bits that no arithmetic has seen)
          if (TWO) *reinterpret_cast<V*>(to + apart) = was_y;
        }
      }
    }
  }
}

// The largest vector, 16 bytes at most, that divides what every access starts at.
int vector_of(const enigma_rope_desc& d) {
  const int64_t es = d.dtype == ENIGMA_DTYPE_F32 ? 4 : 2;
  const bool half = d.layout == ENIGMA_ROPE_HALF;
  int64_t all = half ? d.rotary_dim / 2 | (d.head_dim - d.rotary_dim) / 2 : d.rotary_dim;
  all |= d.head_dim | d.rotary_dim | d.q_token | d.q_head | d.oq_token | d.oq_head;
  uintptr_t at = reinterpret_cast<uintptr_t>(d.q) | reinterpret_cast<uintptr_t>(d.out_q);
  if (d.heads_k > 0) {
    all |= d.k_token | d.k_head | d.ok_token | d.ok_head;
    at |= reinterpret_cast<uintptr_t>(d.k) | reinterpret_cast<uintptr_t>(d.out_k);
  }
  int e = int(16 / es);
  while (e > 1 && (all % e != 0 || at % uintptr_t(e * es) != 0)) e /= 2;
  return e;
}

template <typename T, int E>
cudaError_t launch(const enigma_rope_desc& d, Rope r, cudaStream_t s) {
  const bool half = d.layout == ENIGMA_ROPE_HALF;
  const int64_t rest = (r.d - r.rotary) / E;
  const int64_t units = half || E == 1 ? r.rotary / 2 / E + (rest + 1) / 2 : r.rotary / E + rest;
  // Parts of a token where there are fewer than 16 warps an SM, of at least one round of heads.
  const int64_t sms = enigma::sm_count(), groups = std::max<int64_t>(1, 32 / units);
  const int64_t rounds = (r.heads + groups - 1) / groups;
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(rounds, sms * 16 / std::max<int64_t>(1, d.tokens)));
  r.part_heads = int((rounds + parts - 1) / parts * groups);
  r.parts = (r.heads + r.part_heads - 1) / r.part_heads;
  const int64_t bytes = std::max<int64_t>(16, (r.rotary / 2 + 1) / 2 * 16);
  const int64_t work = d.tokens * r.parts;
  const int64_t warps = std::min<int64_t>(work >= sms * WARPS ? WARPS : 1, ANGLE_BYTES / bytes);
  const unsigned grid = unsigned((work + warps - 1) / warps);
  auto* kernel = r.part_heads <= 2 * groups
                     ? (half ? rope_kernel<T, E, true, 2> : rope_kernel<T, E, false, 2>)
                     : (half ? rope_kernel<T, E, true, 5> : rope_kernel<T, E, false, 5>);
  return enigma::launch_dependent(kernel, grid, unsigned(warps * 32), size_t(warps * bytes), s, r);
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
  const int e = vector_of(d);
  if (d.dtype == ENIGMA_DTYPE_F32)
    return e == 4 ? launch<float, 4>(d, r, s) : e == 2 ? launch<float, 2>(d, r, s) : launch<float, 1>(d, r, s);
  return e == 8   ? launch<__nv_bfloat16, 8>(d, r, s)
         : e == 4 ? launch<__nv_bfloat16, 4>(d, r, s)
         : e == 2 ? launch<__nv_bfloat16, 2>(d, r, s)
                  : launch<__nv_bfloat16, 1>(d, r, s);
}

}  // namespace enigma
