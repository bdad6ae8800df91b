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
// HBM-bound: q, k and v are read once, q and the codes written once.  d / 16 lanes own one token's head: lane j holds elements 8 j .. 8 j + 7 of both
// halves, so the rotation pairs are lane-local, a block of 32 dims is four lanes, and the lanes of a wave take neighbouring heads: whole lines.
// The same lanes take K and V of a head, since V that is not finite is noted in K's block bytes.  Sines and cosines are made once per
// workgroup and token, a pair to a thread, and lie in LDS.
#include <math.h>

#include <type_traits>

#include "msgl_internal.h"
#include "mxfp4.h"

namespace msgl {
namespace {

constexpr int kThreads = 256;
constexpr int kManyTokens = 4;  // of a workgroup, where there are many

template <int D>
struct Params {
  const uint16_t *q, *k, *v, *q_weight, *k_weight;
  const int32_t *positions, *out_loc;
  uint16_t* q_out;
  unsigned char *codes, *scales;
  int64_t q_stride0, k_stride0, v_stride0, codes_stride, scales_stride, num_slots;
  int32_t n_tokens, n_q, n_kv;
  uint32_t chunks;  // workgroups to a token's heads
  double eps;
  double turns[D / 2];  // base^(-i / (d/2)) / 2 pi
};

template <int C>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)(uint32_t)dpp<C>((int)(u >> 32)) << 32 | (uint32_t)dpp<C>((int)(uint32_t)u));
}
template <int LANES>  // 8 or 16
__device__ __forceinline__ double sum_over(double v) {
  v += dpp64<0xB1>(v);
  v += dpp64<0x4E>(v);
  v += dpp64<0x141>(v);
  if constexpr (LANES == 16) v += dpp64<0x140>(v);
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

// 16 values of a lane: 8 of the lower half of a head and 8 of the upper
struct Row {
  u32x4_t lo, hi;
};
__device__ __forceinline__ void values_of(const Row& r, float (&x)[16]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t l = r.lo[e >> 1], h = r.hi[e >> 1];
    x[e] = __builtin_bit_cast(float, (e & 1) ? l & 0xffff0000u : l << 16);
    x[8 + e] = __builtin_bit_cast(float, (e & 1) ? h & 0xffff0000u : h << 16);
  }
}
// The bits of the largest of a half's values; what is not finite is above all others
__device__ __forceinline__ uint32_t largest(const float (&x)[16], int half) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __builtin_bit_cast(uint32_t, x[8 * half + e]) & 0x7fffffffu);
  return top;
}

template <int D, int TOKENS>
__global__ __launch_bounds__(kThreads) void norm_rope_store_mxfp4_kernel(Params<D> p) {
  constexpr int kLanes = D / 16, kGroups = kThreads / kLanes / TOKENS;  // groups of lanes to a token
  __shared__ __attribute__((aligned(16))) float2 angles[TOKENS][D / 2];
  const uint32_t block = blockIdx.x / p.chunks, chunk = blockIdx.x - block * p.chunks;
  const int group = threadIdx.x / kLanes, j = threadIdx.x % kLanes;
  const int first = (int)block * TOKENS, sub = group / kGroups;
  const int token = min(first + sub, p.n_tokens - 1);  // of the last again, where there are no more: nothing is stored
  const bool live = first + sub < p.n_tokens;
  const int off = j * 8, units = p.n_q + p.n_kv;
  const uint16_t *q = p.q + token * p.q_stride0 + off, *k = p.k + token * p.k_stride0 + off, *v = p.v + token * p.v_stride0 + off;
  auto load = [](const uint16_t* row) { return Row{ld_global_b128(row), ld_global_b128(row + D / 2)}; };
  // a unit: a q head, or K and V of a kv head.  The lanes of a wave have neighbouring units, and the next ones' rows are under way
  struct Unit {
    Row a, b;
  };
  auto fetch = [&](int u) {
    Unit x{};
    if (u < p.n_q) {
      x.a = load(q + u * D);
    } else if (u < units) {
      x.a = load(k + (u - p.n_q) * D);
      x.b = load(v + (u - p.n_q) * D);
    }
    return x;
  };
  const int step = kGroups * (int)p.chunks;
  int u = (int)chunk * kGroups + group % kGroups;
  Unit next = fetch(u);
  const int64_t slot = p.out_loc[token];
  float q_weight[16], k_weight[16];
  values_of(load(p.q_weight + off), q_weight);
  values_of(load(p.k_weight + off), k_weight);
#pragma unroll
  for (int at = threadIdx.x; at < TOKENS * (D / 2); at += kThreads) {
    const int t = at / (D / 2), pair = at % (D / 2);
    float2 a;
    sine_cosine((double)p.positions[min(first + t, p.n_tokens - 1)] * p.turns[pair], &a.y, &a.x);
    angles[t][pair] = a;
  }
  __syncthreads();
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = angles[sub][off + e].x;
    sn[e] = angles[sub][off + e].y;
  }

  auto rotate = [&](float (&x)[16], const float (&w)[16]) {
#pragma clang fp contract(off)
    double lo = 0.0, hi = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo = fma((double)x[e], (double)x[e], lo);
      hi = fma((double)x[8 + e], (double)x[8 + e], hi);
    }
    const float factor = (float)reciprocal_root(sum_over<kLanes>(lo + hi) * (1.0 / D) + p.eps);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = w[e] * (x[e] * factor);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = x[e], b = x[8 + e];
      x[e] = a * cs[e] - b * sn[e];
      x[8 + e] = a * sn[e] + b * cs[e];
    }
  };
  for (; u < units; u += step) {
    const Unit now = next;
    next = fetch(u + step);
    float x[16];
    values_of(now.a, x);
    if (u < p.n_q) {
      rotate(x, q_weight);
      if (!live) continue;
      uint16_t* dst = p.q_out + ((int64_t)token * p.n_q + u) * D + off;
      u32x4_t lo, hi;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
        hi[e] = pack_bf16x2(x[8 + 2 * e], x[8 + 2 * e + 1]);
      }
      st_global_b128(dst, lo);
      st_global_b128(dst + D / 2, hi);
    } else {
      rotate(x, k_weight);
      float y[16];
      values_of(now.b, y);
      uint32_t top[4] = {largest(x, 0), largest(x, 1), largest(y, 0), largest(y, 1)};
      const uint64_t mine = ((1ull << kLanes) - 1) << (lane_id() & ~(kLanes - 1));
      const bool poison = (__ballot(max(max(top[0], top[1]), max(top[2], top[3])) >= 0x7f800000u) & mine) != 0;
#pragma unroll
      for (int h = 0; h < 4; ++h) {  // the block's
        top[h] = max(top[h], (uint32_t)dpp<0xB1>((int)top[h]));
        top[h] = max(top[h], (uint32_t)dpp<0x4E>((int)top[h]));
      }
      if (!live || (uint64_t)slot >= (uint64_t)p.num_slots) continue;
      unsigned char* codes = p.codes + slot * p.codes_stride + (u - p.n_q) * D;
      unsigned char* scales = p.scales + slot * p.scales_stride + (u - p.n_q) * (D / 16);
#pragma unroll
      for (int h = 0; h < 4; ++h) {  // K's halves, V's halves
        float z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = poison ? 0.f : h < 2 ? x[8 * h + e] : y[8 * (h - 2) + e];
        const int byte = mx_block_byte(poison ? 0u : top[h]);
        *reinterpret_cast<uint32_t*>(codes + h * (D / 4) + j * 4) = mx_codes8(z, byte);
        if ((j & 3) == 0) scales[h * (D / 64) + (j >> 2)] = (unsigned char)(poison && h < 2 ? kMxNotFinite : byte);
      }
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
  // A workgroup has four tokens where that fills the chip twice over: it makes their angles with all its threads.  Else a token or a part of its heads
  const bool many = a.n_tokens >= 2 * kManyTokens * (int64_t)device_cus();
  constexpr int kUnits = kThreads / (D / 16);
  p.n_tokens = (int32_t)a.n_tokens;
  p.chunks = many ? 1u : (uint32_t)((a.n_q + a.pool.n_kv + kUnits - 1) / kUnits);
  const int64_t blocks = many ? (a.n_tokens + kManyTokens - 1) / kManyTokens : a.n_tokens * p.chunks;
  if (a.n_tokens > 0x7fffffffLL || blocks > 0x7fffffffLL) return MSGL_ERR_SHAPE;
  return launch_kernel(many ? norm_rope_store_mxfp4_kernel<D, kManyTokens> : norm_rope_store_mxfp4_kernel<D, 1>, dim3((unsigned)blocks), dim3(kThreads), stream, p);
}

}  // namespace

int launch_norm_rope_store_mxfp4(const Mxfp4NormRopeArgs& a, hipStream_t stream) {
  return a.pool.head_dim == 128 ? launch<128>(a, stream) : launch<256>(a, stream);
}

}  // namespace msgl
