// A wave's attention over a K/V pool in 4 bits (mxfp4.h): some keys of a request for all columns (query, q head) that share a kv head.
//
//   out[c] = sum_j w_cj v_j / sum_j w_cj,  w_cj = exp(sm_scale q_c . k_j - m_c),  over the keys j that column c sees
//
// Bound by memory: a key of a kv head is D + D / 16 bytes, of its request 4 more, and everything a column needs is computed from one pass
// over them with the running maximum m and sum.  Whose keys a wave takes: mxfp4_attention.hip.
//
// One wave, 32 keys:
//   S^T = K Q^T    mfma 16x16x32, keys on M.  Lane (r, g) of the operand holds 32 dims of its key, block 4 h + g of half h: 16 bytes of codes and one
//                  block byte.  Four products take 8 dims of every block each, which is an order of the contraction like any other, and Q is
//                  read in the same.
//   O^T += V^T P^T mfma 16x16x32, dims on M.  Lane (r, g) reads dims 8 r .. 8 r + 7 of half h, one word, of each of the 8 keys of group g, and turns the 8 x 8 values
//                  over after the conversion.  Row 4 a + i of product u of S^T is key 8 a + of_group(4 u + i), so the
//                  weights of group g's keys are the ones that its lanes hold.
// The conversion multiplies by the block's factor on the way (one instruction for two values), so codes cost what 16-bit values would.
// Weights are rounded to the type of q for the second product (half a step, 2^-8 and 2^-11 of a weight, as the 16-bit pool's
// kernels do; for what half does not reach see kLift); scores, sums and accumulators have 32 bits, and so do the partials.
#pragma once
#include <type_traits>

#include "mxfp4.h"
#include "prefill_tile_common.h"
#include "splitkv_tiles.h"

namespace msgl {

struct MxParams : SplitKvParams {
  int32_t negate;  // scale_log2e is positive: with a scale below zero (-1) the scores of -q count, with none (1) those of zeros
};

template <int D, int NCT>
struct MxColumns {
  u32x4_t q[NCT][D / 32];      // [4 h + c]: dims 128 h + 32 g + 8 c ..
  int lo[NCT], hi[NCT];        // first and last visible key of this lane's column in each tile of 16
  int all_lo, all_hi;          // keys inside are visible to every column
  float m[NCT], l[NCT];        // the reference of the weights (base 2; 0 before the first key) less kLift; this lane's part of their sum
  float top[NCT];              // the reference, or -infinity before the first key
  f32x4_t o[NCT][D / 128][8];  // [h][n][i]: dim 128 h + 8 (4 g + i) + n
};

template <int D>
struct MxTile {  // 32 keys as they lie in the pool
  u32x4_t k[D / 128][2];
  uint32_t k_byte[D / 128][2];
  uint32_t v[D / 128][8], v_byte[D / 128][8];
};

// The factor of a block as the conversion wants it.  Half reaches 65504 = 2^16 (1 - 2^-11) while a block that holds that much has the unit 2^14 and codes up to
// 6: K and V come in at half their size there, and scores and results are doubled.  Byte 0, of a slot that nobody stored, stays 0: its codes are zeros.
template <bool F16, bool IS_K>
__device__ __forceinline__ float block_factor(uint32_t byte) {
  if constexpr (!F16) return mx_scale(byte);
  else if constexpr (IS_K) return mx_scale(byte == kMxNotFinite ? byte : max(byte, 1u) - 1);
  else return mx_scale(max(byte, 1u) - 1);
}
template <bool F16>
constexpr float kBack = F16 ? 2.f : 1.f;

// Weights are 2^(kLift + score - reference), and the reference moves where a score is more than kReach above it.  Half holds 11 bits of a number from 2^-14 on,
// steps of 2^-24 below, and 65504: from 2^13 to 2^15 for the largest weight of a wave's keys, the others keep their 11 bits down to 2^-27 of it, and
// are off by at most 2^-38 of it below.  (At 1, as in bf16, which has the range, a key 17 above all others in the exponent left nothing of them.)
template <bool F16>
constexpr float kLift = F16 ? 13.f : 0.f;
template <bool F16>
constexpr float kReach = F16 ? 2.f : kLazy;

template <int D, int NCT, bool F16>
__device__ __forceinline__ void start_mx_columns(const MxParams& p, const ReqInfo& r, int kvh, int t_end, MxColumns<D, NCT>& c_) {
  const int t16 = lane_id() & 15, g = lane_id() >> 4;
  const int ncols = r.q_len * p.group;
  int all_lo = 0, all_hi = 0x7fffffff;
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    const int col = ct * 16 + t16;
    const bool valid = col < ncols;
    const int qi = valid ? query_of(p, col) : 0;
    const int hh = valid ? col - qi * p.group : 0;
    const uint16_t* qrow = p.q + (int64_t)(r.q_start + qi) * p.q_stride0 + (kvh * p.group + hh) * D + g * 32;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      c_.q[ct][s] = u32x4_t{0u, 0u, 0u, 0u};
      if (valid) c_.q[ct][s] = ld_global_b128(qrow + (s >> 2) * 128 + (s & 3) * 8);
      if (p.negate != 0) c_.q[ct][s] = p.negate < 0 ? c_.q[ct][s] ^ 0x80008000u : u32x4_t{0u, 0u, 0u, 0u};
    }
    const int qpos = r.prefix + qi;
    int lo = (p.window > 0) ? qpos - p.window + 1 : 0;
    int hi = min(p.is_cross ? r.kv_len - 1 : min(qpos, r.kv_len - 1), t_end - 1);
    if (valid) {
      all_lo = max(all_lo, lo);
      all_hi = min(all_hi, hi);
    } else {
      lo = 1;
      hi = 0;
    }
    c_.lo[ct] = lo;
    c_.hi[ct] = hi;
  }
  c_.all_lo = __builtin_amdgcn_readfirstlane(row_max16(all_lo));
  c_.all_hi = __builtin_amdgcn_readfirstlane(~row_max16(~all_hi));
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    c_.m[ct] = 0.f;
    c_.top[ct] = kNegInf;
    c_.l[ct] = 0.f;
#pragma unroll
    for (int h = 0; h < D / 128; ++h)
#pragma unroll
      for (int n = 0; n < 8; ++n) c_.o[ct][h][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
}

// Where the 32 keys of a tile lie in a wave's stage of LDS, and who takes them to registers.  A load moves 1 KiB: whole slots of a head (8 at
// head_dim 128, 4 at 256), 16 bytes a lane, which come to lie one behind the other; the 16-byte pieces of a row are exchanged among
// themselves so that the 16 lanes of a read find theirs in different banks.
//   row(key), piece c at place c ^ turn(key) of its row
// Keys of a lane group's 8, in the order n = 4 u + i in which S^T has them (row 4 a + i of product u): of_group(n).
template <int D>
struct Place;
template <>
struct Place<128> {
  static constexpr int kLoads = 4, kScaleLoads = 1, kLanes = 8;  // lanes to a row in a load
  static __device__ __forceinline__ constexpr int of_group(int n) { return (n & 1) + 4 * ((n >> 1) & 1) + 2 * (n >> 2); }
  // load u, lanes 8 j ..: key 4 j + u
  static __device__ __forceinline__ int key(int u, int j) { return 4 * j + u; }
  static __device__ __forceinline__ constexpr int row(int key) { return 8 * (key & 3) + (key >> 2); }
  static __device__ __forceinline__ constexpr int turn(int key) { return ((key >> 3) & 3) | ((key & 1) << 2); }
  // What a lane reads, as the sum of its own part and one of the instruction: lane (4 a + i, g) piece g of key 8 a + of_group(4 u + i), ...
  static __device__ __forceinline__ int k_lane(int a, int i, int g) { return (8 * (i & 1) + 2 * a + (i >> 1)) * 128 + ((g ^ a) + 4 * (i & 1)) * 16; }
  static __device__ __forceinline__ int k_lane_h(int a, int i, int g) { return k_lane(a, i, g); }
  static __device__ __forceinline__ constexpr int k_of(int u) { return 16 * 128 * u; }
  static __device__ __forceinline__ int k_byte(int a, int i, int g) { return (8 * a + of_group(i)) * 8 + g; }
  // ... and word 4 a + i of V of key 8 g + of_group(n)
  static __device__ __forceinline__ int v_lane(int a, int i, int g) { return 2 * g * 128 + (a ^ g) * 16 + i * 4; }
  static __device__ __forceinline__ constexpr int v_of(int n, int) { return (8 * ((n & 1) + 2 * (n >> 2)) + ((n >> 1) & 1)) * 128 + (n & 1 ? 0 : 64); }
};
template <>
struct Place<256> {
  static constexpr int kLoads = 8, kScaleLoads = 2, kLanes = 16;
  static __device__ __forceinline__ constexpr int of_group(int n) { return n; }
  static __device__ __forceinline__ int key(int u, int j) { return 8 * j + u; }
  static __device__ __forceinline__ constexpr int row(int key) { return 4 * (key & 7) + (key >> 3); }
  static __device__ __forceinline__ constexpr int turn(int key) { return (key >> 3) | ((key & 3) << 2); }
  static __device__ __forceinline__ int k_lane(int a, int i, int g) { return (4 * i + a) * 256 + (4 * i + (g ^ a)) * 16; }
  static __device__ __forceinline__ int k_lane_h(int a, int i, int g) { return (4 * i + a) * 256 + (4 * (i ^ 1) + (g ^ a)) * 16; }
  static __device__ __forceinline__ constexpr int k_of(int u) { return 16 * 256 * u; }
  static __device__ __forceinline__ int k_byte(int a, int i, int g) { return (8 * a + i) * 16 + g; }
  static __device__ __forceinline__ int v_lane(int a, int i, int g) { return g * 256 + (a ^ g) * 16 + i * 4; }
  static __device__ __forceinline__ constexpr int v_of(int n, int h) { return 4 * n * 256 + ((2 + h) ^ (n & 3)) * 64; }
};

// sum + both weights of a pair
template <bool F16>
__device__ __forceinline__ float add_weights(uint32_t pair, float sum) {
  if constexpr (F16) return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, pair), f16x2_t{(_Float16)1.f, (_Float16)1.f}, sum, false);
  else return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pair), kOnes, sum, false);
}

// Keys tb .. tb + 31 for the columns in `c_`
template <int D, int NCT, bool F16>
__device__ __forceinline__ void compute_mx_tile(const SplitKvParams& p, const MxTile<D>& t, int tb, MxColumns<D, NCT>& c_) {
  const int g = lane_id() >> 4;
  f32x4_t s[2][NCT];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) s[u][ct] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int h = 0; h < D / 128; ++h) {
      const float factor = block_factor<F16, true>(t.k_byte[h][u]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const u32x4_t k = mx_values8<F16>(t.k[h][u][c], factor);
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) s[u][ct] = mfma_16x16x32_raw<F16>(k, c_.q[ct][4 * h + c], s[u][ct]);
      }
    }
  const bool need_mask = (tb < c_.all_lo) || (tb + 31 > c_.all_hi);
  u32x4_t pb[NCT];
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    float x[8];  // of key tb + 8 g + of_group(n)
#pragma unroll
    for (int n = 0; n < 8; ++n) x[n] = s[n >> 2][ct][n & 3];
    if (need_mask) {
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int key = tb + 8 * g + Place<D>::of_group(n);
        if (key < c_.lo[ct] || key > c_.hi[ct]) x[n] = kNegInf;
      }
    }
    const float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))) * p.scale_log2e;
    // The reference moves only where a score is far beyond it: weights up to 2^kReach are as exact as those up to 1
    if (__any(mx > c_.top[ct] + kReach<F16>)) {
      const float top = fmaxf(c_.top[ct], max_across<32>(max_across<16>(mx)));
      const float m = top == kNegInf ? 0.f : top;
      const float alpha = fast_exp2(c_.top[ct] - m);
      c_.top[ct] = top;
      c_.m[ct] = m - kLift<F16>;
      c_.l[ct] *= alpha;
#pragma unroll
      for (int h = 0; h < D / 128; ++h)
#pragma unroll
        for (int n = 0; n < 8; ++n) c_.o[ct][h][n] *= alpha;
    }
#pragma unroll
    for (int n = 0; n < 8; ++n) x[n] = fast_exp2(__builtin_fmaf(x[n], p.scale_log2e, -c_.m[ct]));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pb[ct][i] = pack_16x2<F16>(x[2 * i], x[2 * i + 1]);
      c_.l[ct] = add_weights<F16>(pb[ct][i], c_.l[ct]);  // the ones that multiply V
    }
  }
#pragma unroll
  for (int h = 0; h < D / 128; ++h) {
    u32x4_t v[8];
#pragma unroll
    for (int n = 0; n < 8; ++n) v[n] = mx_values8<F16>(t.v[h][n], block_factor<F16, false>(t.v_byte[h][n]));
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      u32x4_t vt;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = v[2 * i][n >> 1], b = v[2 * i + 1][n >> 1];
        vt[i] = (n & 1) ? pack_hi16(a, b) : pack_lo16(a, b);
      }
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) c_.o[ct][h][n] = mfma_16x16x32_raw<F16>(vt, pb[ct], c_.o[ct][h][n]);
    }
  }
}

// A wave's LDS: stages of codes and block bytes, and the slot ids of tiles to come.
template <int D>
struct WaveLds {
  // Tiles on their way while one is computed: more do not come faster.  (16 requests of 32-128 K keys 209 us with one, 219 with three; 32 under a window 15.6,
  // 17.2 and with seven 22.5: the LDS for them is taken from other workgroups of the CU.)
  static constexpr int kAhead = 1, kStages = kAhead + 1;
  static constexpr int kIdsAhead = kAhead + 1, kIdTiles = 2 * kStages;  // ids are asked for so many tiles before their tile is
  static_assert((kStages & (kStages - 1)) == 0 && kIdTiles >= kAhead + kIdsAhead + 1);
  static constexpr int kCodes = 32 * D, kScales = 32 * (D / 16), kStage = kCodes + kScales, kIds = kStages * kStage;
  unsigned char bytes[kIds + kIdTiles * 256];
};

template <int D>
__device__ __forceinline__ void send_tile_ids(uint32_t lds0, const int32_t* idx, int tile, int last) {
  using L = WaveLds<D>;
  lds_direct_b32(lds0 + L::kIds + (uint32_t)(tile & (L::kIdTiles - 1)) * 256u, idx, (uint32_t)min(tile * 32 + (lane_id() & 31), last) * 4u);
}
// In front of attend_mx_keys(), which waits for them
template <int D>
__device__ __forceinline__ void send_first_ids(const MxParams& p, const ReqInfo& r, int t_begin, int t_end, unsigned char* lds) {
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)MSGL_LDS_PTR(unsigned char, lds));
  for (int tile = 0; tile < WaveLds<D>::kIdsAhead; ++tile) send_tile_ids<D>(lds0, p.kv_indices + r.kv_start + t_begin, tile, t_end - t_begin - 1);
}

// At most N loads of the wave under way, and none of its reads of LDS: the stage that the next loads write has been read.
template <int N>
__device__ __forceinline__ void wait_tile() {
  static_assert(N >= 0 && N < 64, "vmcnt is a 6-bit field");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));
  asm volatile("" ::: "memory");
}

// Keys [t_begin, t_end) of request `r`, in order, for the columns in `c_`; `lds`: the wave's own, so nobody else is waited for.
// The ids of its first tiles are under way (send_first_ids).  Everything comes by loads that write LDS, of which the compiler knows nothing: tile i is there when no more of them than those issued
// behind its last are under way.  Each iteration issues the same number, in the same order: codes and block bytes of the tile kAhead on, ids of the tile kAhead +
// kIdsAhead on.  Keys past the end are the last one again, and masked.
template <int D, int NCT, bool F16, int WALK>
__device__ __forceinline__ void attend_mx_keys(const SplitKvParams& p, const ReqInfo& r, int kvh, int t_begin, int t_end, unsigned char* lds,
                                               MxColumns<D, NCT>& c_) {
  using P = Place<D>;
  using L = WaveLds<D>;
  constexpr int kAhead = L::kAhead, kStages = L::kStages, kIdsAhead = L::kIdsAhead, kIdTiles = L::kIdTiles;
  constexpr int kIssued = P::kLoads + P::kScaleLoads + 1;
  constexpr int kScaleWords = D / 64;  // of 4 bytes, of a key
  using Offset = typename std::conditional<(WALK & kWide) != 0, uint64_t, uint32_t>::type;
  const int lane = lane_id(), t16 = lane & 15, g = lane >> 4, a = t16 >> 2, i = t16 & 3;
  const unsigned char* codes = reinterpret_cast<const unsigned char*>(p.k_cache) + kvh * D;
  const unsigned char* scales = reinterpret_cast<const unsigned char*>(p.v_cache) + kvh * (D / 16);
  const int32_t* idx = p.kv_indices + r.kv_start + t_begin;
  const int last = t_end - t_begin - 1, n_tiles = (last >> 5) + 1;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)MSGL_LDS_PTR(unsigned char, lds));
  const auto shared = MSGL_LDS_PTR(unsigned char, lds);
  const uint32_t codes_stride = (uint32_t)p.k_stride0, scales_stride = (uint32_t)p.v_stride0;
  auto offset = [](uint32_t slot, uint32_t stride) -> Offset {
    if constexpr (WALK & kWide) return (uint64_t)slot * stride;
    else return __umul24(slot, stride);  // both below 2^24 here
  };

  const int j = lane / P::kLanes, piece = lane % P::kLanes;
  auto send_ids = [&](int tile) { send_tile_ids<D>(lds0, idx, tile, last); };
  auto send_tile = [&](int tile) {
    const uint32_t stage = lds0 + (uint32_t)(tile & (kStages - 1)) * L::kStage;
    const auto ids = shared + L::kIds + (tile & (kIdTiles - 1)) * 256;
    uint32_t slot[P::kLoads];
#pragma unroll
    for (int q = 0; q < P::kLoads; q += 4) {
      const u32x4_t four = *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>(ids + P::key(q, j) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) slot[q + e] = min(four[e], p.max_slot);
    }
    uint32_t scale_slot[P::kScaleLoads];
#pragma unroll
    for (int q = 0; q < P::kScaleLoads; ++q)
      scale_slot[q] = min(*reinterpret_cast<const __attribute__((address_space(3))) uint32_t*>(ids + ((64 / kScaleWords) * q + lane / kScaleWords) * 4), p.max_slot);
#pragma unroll
    for (int u = 0; u < P::kLoads; ++u) {
      const Offset from = offset(slot[u], codes_stride) + (uint32_t)((piece ^ P::turn(P::key(u, j))) * 16);
      if constexpr (WALK & kStream) lds_stream_b128(stage + u * 1024u, codes, from);
      else lds_direct_b128(stage + u * 1024u, codes, from);
    }
#pragma unroll
    for (int q = 0; q < P::kScaleLoads; ++q)
      lds_direct_b32(stage + L::kCodes + q * 256u, scales, offset(scale_slot[q], scales_stride) + (uint32_t)(lane % kScaleWords) * 4u);
  };
  wait_all_vm();
#pragma unroll
  for (int tile = 0; tile < kAhead; ++tile) {
    send_tile(tile);
    send_ids(tile + kIdsAhead);
  }
  for (int tile = 0; tile < n_tiles; ++tile) {
    wait_tile<(kAhead - 1) * kIssued + 1>();
    send_tile(tile + kAhead);
    send_ids(tile + kAhead + kIdsAhead);
    const auto at = shared + (tile & (kStages - 1)) * L::kStage;
    const auto k_at = at + P::k_lane(a, i, g), v_at = at + P::v_lane(a, i, g);
    const auto kb_at = at + L::kCodes + P::k_byte(a, i, g), vb_at = at + L::kCodes + 8 * g * (D / 16) + D / 32 + a;
    MxTile<D> t;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int h = 0; h < D / 128; ++h) {
        t.k[h][u] = *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>((h == 0 ? k_at : at + P::k_lane_h(a, i, g)) + P::k_of(u));
        t.k_byte[h][u] = kb_at[(P::of_group(4 * u) - P::of_group(0)) * (D / 16) + 4 * h];
      }
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int h = 0; h < D / 128; ++h) {
        t.v[h][n] = *reinterpret_cast<const __attribute__((address_space(3))) uint32_t*>(v_at + P::v_of(n, h));
        t.v_byte[h][n] = vb_at[P::of_group(n) * (D / 16) + 4 * h];
      }
    compute_mx_tile<D, NCT, F16>(p, t, t_begin + tile * 32, c_);
  }
  wait_all_vm();  // what is still under way writes LDS that the next keys want
}

}  // namespace msgl
