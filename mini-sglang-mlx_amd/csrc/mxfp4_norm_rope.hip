// Per-head RMS norm of q and k, rotary embedding of both, and the store of k and v in a pool of 4 bits (mxfp4.h), in one pass.
//
//   y   = w x / sqrt(mean(x^2) + eps)                                    (per head)
//   o_i = y_i cos(t_i) - y_{i+d/2} sin(t_i),  o_{i+d/2} = y_i sin(t_i) + y_{i+d/2} cos(t_i)
//   t_i = position base^(-i / (d/2))                                     (rotate-half form, rotary_dim = d)
//   q_out[t, h] = bf16(o(q[t, h]));  the pool's row of slot out_loc[t] = the codes of o(k[t, h]) and v[t, h]
//
// Everything between the inputs and the one rounding at the end is held in 32 bits, with no rounding to bf16 on the way.  The codes
// of k make two things matter that a bf16 result forgives.  A code falls by the last bit of a value next to a border: the mean
// and its root are therefore taken in 64 bits, and the products behind them are single roundings of 32 in the order above, so the
// result does not depend on how lanes add.  And angles reach 10^6 radians, where 32 bits are 0.03 off: the turns
// position * base^(-i / (d/2)) / 2 pi are a product of 64 bits, their fraction is exact, and sine and cosine of what is left, at most an
// eighth of a turn, are Taylor sums in 64 bits.  (64-bit products issue as fast as 32-bit ones here.)
//
// HBM-bound: q, k and v are read once, q and the codes written once.  Sixteen lanes own one token's head: lane j holds elements E j .. E j + E - 1
// of both halves (E = d / 32), so the rotation pairs are lane-local; a block of 32 dims is 32 / E of them.  The same lanes take K and V of
// a head, since V that is not finite is noted in K's block bytes.  A group of lanes walks a chunk of the token's heads, and the angles are made once
// per chunk.
#include <math.h>

#include <type_traits>

#include "msgl_internal.h"
#include "mxfp4.h"

namespace msgl {
namespace {

constexpr int kGroupLanes = 16;
constexpr int kThreads = 256;

template <int D>
struct Params {
  const uint16_t *q, *k, *v, *q_weight, *k_weight;
  const int32_t *positions, *out_loc;
  uint16_t* q_out;
  unsigned char *codes, *scales;
  int64_t q_stride0, k_stride0, v_stride0, codes_stride, scales_stride, num_slots;
  uint32_t items, chunks, per_group;  // (token, chunk of heads)
  int32_t n_q, n_kv;
  double eps;
  double turns[D / 2];  // base^(-i / (d/2)) / 2 pi
};

__device__ __forceinline__ double dpp_sum16(double v) {
  auto add = [&](auto control) {
    constexpr int C = decltype(control)::value;
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint64_t o = (uint64_t)(uint32_t)dpp<C>((int)(u >> 32)) << 32 | (uint32_t)dpp<C>((int)(uint32_t)u);
    v += __builtin_bit_cast(double, o);
  };
  add(std::integral_constant<int, 0xB1>{});
  add(std::integral_constant<int, 0x4E>{});
  add(std::integral_constant<int, 0x141>{});
  add(std::integral_constant<int, 0x140>{});
  return v;
}

// 1 / sqrt(x) to the last bits of a double: the hardware's estimate and two steps of Newton's method
__device__ __forceinline__ double reciprocal_root(double x) {
  double y = __builtin_amdgcn_rsq(x);
#pragma unroll
  for (int i = 0; i < 2; ++i) y = fma(0.5 * y, fma(-x * y, y, 1.0), y);
  return x == __builtin_inf() ? 0.0 : y;
}

// Sine and cosine of so many turns
__device__ __forceinline__ void sine_cosine(double turns, float* sine, float* cosine) {
  const double part = turns - rint(turns);  // exact, as is what is left of it beside a whole quarter
  const double quarter = rint(4.0 * part);
  const double t = 6.283185307179586476925 * fma(-0.25, quarter, part), z = t * t;
  double s = 1.0 / 6227020800.0, c = -1.0 / 87178291200.0;  // 1 / 13!, -1 / 14!: what follows is below 3e-14
  s = fma(z, s, -1.0 / 39916800.0);
  c = fma(z, c, 1.0 / 479001600.0);
  s = fma(z, s, 1.0 / 362880.0);
  c = fma(z, c, -1.0 / 3628800.0);
  s = fma(z, s, -1.0 / 5040.0);
  c = fma(z, c, 1.0 / 40320.0);
  s = fma(z, s, 1.0 / 120.0);
  c = fma(z, c, -1.0 / 720.0);
  s = fma(z, s, -1.0 / 6.0);
  c = fma(z, c, 1.0 / 24.0);
  s = fma(t * z, s, t);
  c = fma(z, fma(z, c, -0.5), 1.0);
  const int n = (int)quarter & 3;
  const float fs = (float)s, fc = (float)c;
  const float a = (n & 1) ? fc : fs, b = (n & 1) ? fs : fc;
  *sine = (n & 2) ? -a : a;
  *cosine = (n == 1 || n == 2) ? -b : b;
}

template <int E>
struct Half;  // E bf16 values as one load
template <>
struct Half<4> { typedef u32x2_t type; };
template <>
struct Half<8> { typedef u32x4_t type; };

template <int D>
__global__ __launch_bounds__(kThreads) void norm_rope_store_mxfp4_kernel(Params<D> p) {
  constexpr int E = D / 32, kBlockLanes = kMxBlock / E;
  using V = typename Half<E>::type;
  const int j = threadIdx.x & (kGroupLanes - 1);
  const uint32_t item = blockIdx.x * (kThreads / kGroupLanes) + threadIdx.x / kGroupLanes;
  if (item >= p.items) return;  // whole groups leave together, and nothing crosses groups
  const uint32_t token = item / p.chunks, chunk = item - token * p.chunks;
  const int n_heads = p.n_q + p.n_kv, h_begin = chunk * p.per_group, h_end = min(h_begin + (int)p.per_group, n_heads);
  const int off = j * E;
  struct Row {
    V lo, hi;
  };
  auto fetch = [&](const uint16_t* row) { return Row{*reinterpret_cast<const V*>(row + off), *reinterpret_cast<const V*>(row + D / 2 + off)}; };
  auto value = [](const V& r, int e) {
    const uint32_t w = r[e >> 1];
    return __builtin_bit_cast(float, (e & 1) ? w & 0xffff0000u : w << 16);
  };
  const double position = (double)p.positions[token];
  const int64_t slot = p.out_loc[token];
  float cs[E], sn[E];
#pragma unroll
  for (int e = 0; e < E; ++e) sine_cosine(position * p.turns[off + e], &sn[e], &cs[e]);

  // x: in order the E values of the lower half and those of the upper
  auto load = [&](const uint16_t* row, float (&x)[2 * E]) {
    const Row r = fetch(row);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      x[e] = value(r.lo, e);
      x[E + e] = value(r.hi, e);
    }
  };
  auto rotate = [&](float (&x)[2 * E], const uint16_t* weight) {
#pragma clang fp contract(off)
    float w[2 * E];
    load(weight, w);
    double ss = 0.0;
#pragma unroll
    for (int e = 0; e < 2 * E; ++e) ss = fma((double)x[e], (double)x[e], ss);
    ss = dpp_sum16(ss);
    const float factor = (float)reciprocal_root(ss * (1.0 / D) + p.eps);
#pragma unroll
    for (int e = 0; e < 2 * E; ++e) x[e] = w[e] * (x[e] * factor);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float a = x[e], b = x[E + e];
      x[e] = a * cs[e] - b * sn[e];
      x[E + e] = a * sn[e] + b * cs[e];
    }
  };
  // The codes of a row at `codes` and its block bytes at `scales`; poison: the row counts as zeros, `mark`: and its block bytes say so
  auto store = [&](const float (&in)[2 * E], unsigned char* codes, unsigned char* scales, bool poison, bool mark) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float x[8], amax = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        x[e] = poison ? 0.f : in[half * E + e];
        amax = fmaxf(amax, fabsf(x[e]));
      }
      amax = fmaxf(amax, dpp<0xB1>(amax));
      amax = fmaxf(amax, dpp<0x4E>(amax));
      if constexpr (kBlockLanes == 8) amax = fmaxf(amax, dpp<0x141>(amax));
      const int byte = mx_block_byte(amax);
      const uint32_t word = mx_codes8(x, byte);
      unsigned char* to = codes + half * (D / 4) + j * (E / 2);
      if constexpr (E == 8) *reinterpret_cast<uint32_t*>(to) = word;
      else *reinterpret_cast<uint16_t*>(to) = (uint16_t)word;
      if (j % kBlockLanes == 0) scales[half * (D / 64) + j / kBlockLanes] = (unsigned char)(poison && mark ? kMxNotFinite : byte);
    }
  };
  auto any_not_finite = [&](const float (&x)[2 * E]) {
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 2 * E; ++e) bad |= (__builtin_bit_cast(uint32_t, x[e]) & 0x7f800000u) == 0x7f800000u;
    return bad;
  };

  for (int h = h_begin; h < h_end; ++h) {
    if (h < p.n_q) {
      float x[2 * E];
      load(p.q + token * p.q_stride0 + h * D, x);
      rotate(x, p.q_weight);
      uint16_t* dst = p.q_out + ((int64_t)token * p.n_q + h) * D + off;
      V lo, hi;
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        lo[e >> 1] = pack_bf16x2(x[e], x[e + 1]);
        hi[e >> 1] = pack_bf16x2(x[E + e], x[E + e + 1]);
      }
      *reinterpret_cast<V*>(dst) = lo;
      *reinterpret_cast<V*>(dst + D / 2) = hi;
    } else {
      const int kvh = h - p.n_q;
      float k[2 * E], v[2 * E];
      load(p.k + token * p.k_stride0 + kvh * D, k);
      load(p.v + token * p.v_stride0 + kvh * D, v);
      rotate(k, p.k_weight);
      const uint64_t group = 0xffffull << (lane_id() & ~(kGroupLanes - 1));
      const bool poison = (__ballot(any_not_finite(k) || any_not_finite(v)) & group) != 0;
      if ((uint64_t)slot >= (uint64_t)p.num_slots) continue;
      unsigned char* codes = p.codes + slot * p.codes_stride + kvh * D;
      unsigned char* scales = p.scales + slot * p.scales_stride + kvh * (D / 16);
      store(k, codes, scales, poison, true);
      store(v, codes + D / 2, scales + D / 32, poison, false);
    }
  }
}

template <int D>
int launch(const Mxfp4NormRopeArgs& a, hipStream_t stream) {
  Params<D> p{};
  p.q = static_cast<const uint16_t*>(a.q);
  p.k = static_cast<const uint16_t*>(a.k);
  p.v = static_cast<const uint16_t*>(a.v);
  p.q_weight = static_cast<const uint16_t*>(a.q_weight);
  p.k_weight = static_cast<const uint16_t*>(a.k_weight);
  p.positions = a.positions;
  p.out_loc = a.out_loc;
  p.q_out = static_cast<uint16_t*>(a.q_out);
  p.codes = static_cast<unsigned char*>(a.pool.codes);
  p.scales = static_cast<unsigned char*>(a.pool.scales);
  p.q_stride0 = a.q_stride0;
  p.k_stride0 = a.k_stride0;
  p.v_stride0 = a.v_stride0;
  p.codes_stride = a.pool.codes_stride0;
  p.scales_stride = a.pool.scales_stride0;
  p.num_slots = a.pool.num_slots;
  p.n_q = (int32_t)a.n_q;
  p.n_kv = (int32_t)a.pool.n_kv;
  p.eps = a.eps;
  // base^(-1 / (d/2)) and its powers: 80-bit products, off by less than a step of a double at the last
  const long double step = powl((long double)a.rope_base, -2.0L / D);
  long double turn = 0.159154943091895335768883763372514362L;  // 1 / 2 pi
  for (int i = 0; i < D / 2; ++i, turn *= step) p.turns[i] = (double)turn;
  // one head per group until its workgroups fill the chip twice over: few tokens are the chain of one group's loads
  const int64_t n_heads = a.n_q + a.pool.n_kv;
  p.per_group = a.n_tokens * n_heads <= 512 * (kThreads / kGroupLanes) ? 1 : 8;
  p.chunks = (uint32_t)((n_heads + p.per_group - 1) / p.per_group);
  const int64_t items = a.n_tokens * p.chunks, per_block = kThreads / kGroupLanes;
  if (items >= (int64_t)1 << 31) return MSGL_ERR_SHAPE;
  p.items = (uint32_t)items;
  return launch_kernel(norm_rope_store_mxfp4_kernel<D>, dim3((unsigned)((items + per_block - 1) / per_block)), dim3(kThreads), stream, p);
}

}  // namespace

int launch_norm_rope_store_mxfp4(const Mxfp4NormRopeArgs& a, hipStream_t stream) {
  return a.pool.head_dim == 128 ? launch<128>(a, stream) : launch<256>(a, stream);
}

}  // namespace msgl
