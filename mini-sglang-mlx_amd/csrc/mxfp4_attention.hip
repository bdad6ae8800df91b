// Attention over a K/V pool in 4 bits for decode and short query blocks: mxfp4_tiles.h, one workgroup to a share of a request's keys for one to eight kv heads.
//
// Each request's visible keys are cut into equal shares, as many in all as there are workgroups that the card holds at once, one to a CU; the waves of a
// workgroup take a head each, or cut a head's share again and meet in LDS; and of a request that several shares hold the workgroup that counts last puts
// the partials together.  One launch, and nobody waits for anybody: a merge in a launch of its own took 8 us of small calls and 12 of 32 requests of 32 columns,
// and equal parts of the stream of all keys, which begin and end inside requests, as long as whole shares or longer (64 requests of 8 K keys 109
// us against 107, 8 of 4 K 18.7 against 15.5).  Partials and counts travel at agent scope; a count word carries the launch's number
// (launch_number.h), so the workspace needs no clearing, and is left as of a launch that never happened, so a replay counts anew.
//
// Bound by memory: 16 requests of 32-128 K keys of 8 heads of 128, 6.3 TB/s; 64 of 1-8 K 5.5.
#include <cmath>
#include <utility>

#include "agent_scope.h"
#include "launch_number.h"
#include "mxfp4_tiles.h"

namespace msgl {
namespace {

struct ShareParams : MxParams {
  unsigned long long* counts;     // [query block][batch][head_groups][kCountWords]: shares done
  unsigned long long nonce;       // launch_number.h
  int32_t shares;                 // as many as there may be ..
  float min_len;                  // .. if that makes none shorter
  int32_t wave_shift;             // log2 of the waves on a head's share
};

// A share's place: number `share` of the `n_shares` of request b, number `item` of the launch
struct MxShare {
  ReqInfo r;
  int b, share, n_shares, item;
};
// How requests are cut: the shortest length of a share, min_len at least, with which there are no more shares than fit on the card at once.  It is between
// total / shares and what is enough when every request loses a whole share to its end, and the wave that wants to know looks for it there: 64 requests at a
// time, which stay in registers up to kCached of them.  (Beyond those the outer end is taken.)  Where even a share to a request is too many, each has one.
constexpr int kCached = 512;
// (The quotient of floats may take an exact one a share too far, never two; `max_shares` of the launch has room for a share more of every request that has keys.)
__device__ __forceinline__ int shares_of(int visible, float per_len) { return (int)ceilf((float)visible * per_len); }

// All lanes must call; false past the last share.
__device__ __forceinline__ bool find_mx_share(const ShareParams& p, int item, MxShare* x) {
  const int lane = lane_id();
  auto visible_of = [&](const ReqInfo& r, int b0) { return b0 + lane < p.batch && r.q_len > 0 ? max(r.hi - r.lo, 0) : 0; };
  auto request_at = [&](int b0) { return request_info(p, min(b0 + lane, p.batch - 1)); };
  const ReqInfo first64 = request_at(0);
  int visible[kCached / kWave];
  visible[0] = visible_of(first64, 0);
  int total = wave_sum(visible[0]), some = __popcll(__ballot(visible[0] > 0));
#pragma unroll
  for (int c = 1; c < kCached / kWave; ++c) {
    visible[c] = 0;
    if (c * kWave >= p.batch) continue;
    visible[c] = visible_of(request_at(c * kWave), c * kWave);
    total += wave_sum(visible[c]);
    some += __popcll(__ballot(visible[c] > 0));
  }
  for (int b0 = kCached; b0 < p.batch && some < p.shares; b0 += kWave) {
    const int n = visible_of(request_at(b0), b0);
    total += wave_sum(n);
    some += __popcll(__ballot(n > 0));
  }
  if (some >= p.shares) {
    if (item >= p.batch) return false;
    *x = {request_info(p, item), item, 0, 1, (int)(blockIdx.y * (gridDim.x / p.head_groups)) + item};
    return true;
  }
  auto fit = [&](float len) {
    const float per_len = __builtin_amdgcn_rcpf(len);
    int n = 0;
#pragma unroll
    for (int c = 0; c < kCached / kWave; ++c)
      if (c * kWave < p.batch) n += shares_of(visible[c], per_len);
    return wave_sum(n) <= p.shares;
  };
  float len = fmaxf((float)total * __builtin_amdgcn_rcpf((float)p.shares), p.min_len);  // from here ..
  float most = fmaxf((float)total * __builtin_amdgcn_rcpf((float)(p.shares - some)), p.min_len);  // .. to here
  if (p.batch > kCached) {
    len = most;
  } else if (!fit(len)) {
    while (most > len * (1.f + 1.f / 32)) {
      const float mid = 0.5f * (len + most);
      if (fit(mid)) most = mid;
      else len = mid;
    }
    len = most;
  }
  const float per_len = __builtin_amdgcn_rcpf(len);
  int base = 0;
  auto here = [&](int n_visible, int b0, auto&& request) {
    // a request without visible keys has one empty share: its rows are zero
    const int n = b0 + lane < p.batch ? max(shares_of(n_visible, per_len), 1) : 0;
    const int incl = wave_inclusive_scan(n), sum = __builtin_amdgcn_readlane(incl, kWave - 1), first = base + incl - n;
    base += sum;
    if (item >= base) return false;
    const int src = __builtin_amdgcn_readfirstlane(__ffsll((long long)__ballot(item >= first && item < first + n)) - 1);
    x->r = request(src);
    x->b = b0 + src;
    x->share = item - __builtin_amdgcn_readlane(first, src);
    x->n_shares = __builtin_amdgcn_readlane(n, src);
    x->item = blockIdx.y * (gridDim.x / p.head_groups) + item;
    return true;
  };
  if (here(visible[0], 0, [&](int src) {
        ReqInfo r;
        r.kv_start = __builtin_amdgcn_readlane(first64.kv_start, src);
        r.kv_len = __builtin_amdgcn_readlane(first64.kv_len, src);
        r.q_start = __builtin_amdgcn_readlane(first64.q_start, src);
        r.q_len = __builtin_amdgcn_readlane(first64.q_len, src);
        r.prefix = __builtin_amdgcn_readlane(first64.prefix, src);
        r.lo = __builtin_amdgcn_readlane(first64.lo, src);
        r.hi = __builtin_amdgcn_readlane(first64.hi, src);
        r.rows = __builtin_amdgcn_readlane(first64.rows, src);
        return r;
      }))
    return true;
#pragma unroll
  for (int c = 1; c < kCached / kWave; ++c) {
    if (c * kWave >= p.batch) return false;
    if (here(visible[c], c * kWave, [&](int src) { return request_info(p, c * kWave + src); })) return true;
  }
  for (int b0 = kCached; b0 < p.batch; b0 += kWave)
    if (here(visible_of(request_at(b0), b0), b0, [&](int src) { return request_info(p, b0 + src); })) return true;
  return false;
}

// The LDS of a workgroup: a wave's stages, and in their place, when its keys are done, its accumulators.
template <int D, int NCT>
struct WavePart {
  static constexpr int kBlock = 16 * NCT * 8 + 8;  // floats of 8 dims: [col][8], padded
  float o[D / 8][kBlock];
};
template <int D, int NCT, int NW>
struct MxLds {
  static constexpr int kWaveBytes = (std::max(sizeof(WaveLds<D>), sizeof(WavePart<D, NCT>)) + 255) / 256 * 256;
  unsigned char wave[NW][kWaveBytes];
  float2 state[NW][16 * NCT];  // (reference, sum) of a wave's columns
  int last;
};

template <typename F, int... I>
__device__ __forceinline__ void each(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}

// A wave's place in its workgroup: waves on a head, which head, which of its waves
struct MxWave {
  int waves, sub, sw, threads, me;  // threads on a head, this one's number
  __device__ __forceinline__ explicit MxWave(const ShareParams& p) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    waves = 1 << p.wave_shift;
    sub = wave >> p.wave_shift;
    sw = wave & (waves - 1);
    threads = 64 << p.wave_shift;
    me = (int)threadIdx.x - sub * threads;
  }
};
// A wave's keys of a share
struct MxRange {
  int begin, end;
  __device__ __forceinline__ MxRange(const ShareParams& p, const MxShare& x, const MxWave& w) {
    const int per = ((x.r.hi - x.r.lo + x.n_shares - 1) / x.n_shares + 31) & ~31;
    const int s_begin = min(x.r.lo + x.share * per, x.r.hi), s_end = min(s_begin + per, x.r.hi);
    const int per_wave = (((per + w.waves - 1) >> p.wave_shift) + 31) & ~31;
    begin = min(s_begin + w.sw * per_wave, s_end);
    end = min(begin + per_wave, s_end);
  }
};

// Four dims of a column of the result
template <int D, bool F16>
__device__ __forceinline__ void leave_quad(const ShareParams& p, const ReqInfo& r, int kvh, int col, int d4, f32x4_t o) {
  const int qi = query_of(p, col);
  uint16_t* dst = p.out + ((int64_t)(r.q_start + qi) * p.n_q + kvh * p.group + (col - qi * p.group)) * D + d4;
  *reinterpret_cast<u32x2_t*>(dst) = u32x2_t{pack_16x2<F16>(o[0], o[1]), pack_16x2<F16>(o[2], o[3])};
}

// The waves of a head, whose accumulators and state are in LDS: the rows, if the share is all of the request, else its partial.
template <int D, int NCT, bool F16, int NW>
__device__ __forceinline__ void put_waves_together(const ShareParams& p, const MxLds<D, NCT, NW>& lds, const MxShare& x, int hg, const MxWave& w) {
  constexpr int kQuads = D / 4;  // a thread's unit of work: 4 dims of one column
  const int t16 = lane_id() & 15, kvh = hg * p.nwh + w.sub, ncols = x.r.q_len * p.group;
  const int64_t row0 = ((int64_t)x.item * p.n_kv + kvh) * p.cols;
  const Partials own(p.part_o + row0 * D, (uint32_t)(ncols * D * 4));
  // Every wave's part of a quad is asked for before the first is used.  The lanes of a row of 16 work on one column: lane i has
  // wave i's reference and sum, and its weight goes to the others by DPP.
  auto with = [&](auto n_waves) {
    constexpr int W = decltype(n_waves)::value;
    for (int it = w.me; it < ncols * kQuads; it += w.threads) {
      const int col = it / kQuads, d4 = (it - col * kQuads) * 4;
      float2 ml = lds.state[w.sub * W + min(t16, W - 1)][col];
      f32x4_t o[W];
#pragma unroll
      for (int i = 0; i < W; ++i)
        o[i] = *reinterpret_cast<const f32x4_t*>(&reinterpret_cast<const WavePart<D, NCT>*>(lds.wave[w.sub * W + i])->o[d4 >> 3][col * 8 + (d4 & 7)]);
      if (t16 >= W) ml = float2{kNegInf, 0.f};
      const float top = row_max16(ml.x), m = top == kNegInf ? 0.f : top;
      const float e = fast_exp2(ml.x - m);  // 0 for a wave without visible keys
      // a wave that saw nothing but NaN has no reference and a sum that is NaN, with any weight
      const float l = row_sum16(e * ml.y);
      f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
      each([&](auto i) { acc += of_row_lane<decltype(i)::value>(e) * o[decltype(i)::value]; }, std::make_integer_sequence<int, W>{});
      acc *= l > 0.f ? kBack<F16> / l : 0.f;  // (NaN: the accumulators are that too)
      if (x.n_shares == 1) {
        leave_quad<D, F16>(p, x.r, kvh, col, d4, acc);
      } else {
        own.store(16u * (uint32_t)it, acc);
        // NaN: any weight above zero takes the partial's NaN into the merged row
        if (d4 == 0)
          __hip_atomic_store(p.part_lse + row0 + col, l > 0.f ? m + __log2f(l) : l == 0.f ? kNegInf : 0.f, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  };
  if (w.waves == 4) with(std::integral_constant<int, 4>{});
  else if (w.waves == 2) with(std::integral_constant<int, 2>{});
  else with(std::integral_constant<int, 1>{});
}

// The partials of all shares of a request, by log-sum-exp: its rows.
template <int D, bool F16>
__device__ __forceinline__ void put_shares_together(const ShareParams& p, const MxShare& x, int hg, const MxWave& w) {
  constexpr int kQuads = D / 4;
  const int t16 = lane_id() & 15, kvh = hg * p.nwh + w.sub, ncols = x.r.q_len * p.group, n_shares = x.n_shares;
  const int64_t step = (int64_t)p.n_kv * p.cols;  // rows from one share to the next
  const int64_t first = ((int64_t)(x.item - x.share) * p.n_kv + kvh) * p.cols;
  const uint32_t step_bytes = (uint32_t)(step * (D * 4));
  const Partials all(p.part_o + first * D, (uint32_t)n_shares * step_bytes);
  const float* const lse_from = p.part_lse + first;
  // U shares of Q quads at a time; the lanes of a row of 16 work on the same columns
  auto with = [&](auto in_flight, auto quads) {
    constexpr int U = decltype(in_flight)::value, Q = decltype(quads)::value;
    const int n_quads = ncols * kQuads;
    for (int it = w.me; it < n_quads; it += Q * w.threads) {
      float top[Q], l[Q];
      f32x4_t acc[Q];
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        top[q] = kNegInf;
        l[q] = 0.f;
        acc[q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      }
      for (int s0 = 0; s0 < n_shares; s0 += U) {  // shares past the last one: the last again, not used; quads likewise
        const int mine = min(s0 + min(t16, U - 1), n_shares - 1);
        float lse[Q];
        f32x4_t o[Q][U];
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const int at = min(it + q * w.threads, n_quads - kQuads + (it & (kQuads - 1)));
          lse[q] = __hip_atomic_load(lse_from + mine * step + at / kQuads, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
          for (int u = 0; u < U; ++u) o[q][u] = all.load(16u * (uint32_t)at, (uint32_t)min(s0 + u, n_shares - 1) * step_bytes);
        }
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          if (t16 >= U || s0 + t16 >= n_shares) lse[q] = kNegInf;
          const float now = fmaxf(top[q], row_max16(lse[q])), m = now == kNegInf ? 0.f : now;
          const float old = fast_exp2(top[q] - m), e = fast_exp2(lse[q] - m);
          acc[q] *= old;
          l[q] = l[q] * old + row_sum16(e);
          top[q] = now;
          each([&](auto u) {
            if (s0 + decltype(u)::value < n_shares) acc[q] += of_row_lane<decltype(u)::value>(e) * o[q][decltype(u)::value];
          }, std::make_integer_sequence<int, U>{});
        }
      }
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int at = it + q * w.threads, col = at / kQuads;
        if (at < n_quads) leave_quad<D, F16>(p, x.r, kvh, col, (at - col * kQuads) * 4, acc[q] * (l[q] > 0.f ? 1.0f / l[q] : 0.f));
      }
    }
  };
  using std::integral_constant;
  if (n_shares <= 4) with(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  else if (n_shares <= 8) with(integral_constant<int, 8>{}, integral_constant<int, 2>{});
  else with(integral_constant<int, 16>{}, integral_constant<int, 1>{});
}

template <int D, int NCT, bool F16, int WALK, int NW>
__global__ __launch_bounds__(64 * NW, (D == 128 && NCT <= 2) || NCT == 1 ? 2 : 1) void mxfp4_attention_kernel(ShareParams p) {
  using Lds = MxLds<D, NCT, NW>;
  __shared__ __attribute__((aligned(256))) Lds lds;
  const int t16 = lane_id() & 15, g = lane_id() >> 4;
  p.q_begin = blockIdx.y * p.max_len_extend;
  const int item = blockIdx.x / p.head_groups, hg = blockIdx.x - item * p.head_groups;
  MxShare x;
  if (!find_mx_share(p, item, &x)) return;
  unsigned long long* const word = p.counts + (((int64_t)blockIdx.y * p.batch + x.b) * p.head_groups + hg) * kCountWords;
  if (x.n_shares > 1 && threadIdx.x == 0) open_count(word, p.nonce);
  const MxWave w(p);
  unsigned char* const mine = lds.wave[w.sub * w.waves + w.sw];
  const MxRange keys(p, x, w);
  if (keys.begin < keys.end) send_first_ids<D>(p, x.r, keys.begin, keys.end, mine);
  const int ncols = x.r.q_len * p.group, kvh = hg * p.nwh + w.sub;
  MxColumns<D, NCT> c_;
  start_mx_columns<D, NCT, F16>(p, x.r, kvh, keys.end, c_);
  if (keys.begin < keys.end) attend_mx_keys<D, NCT, F16, WALK>(p, x.r, kvh, keys.begin, keys.end, mine, c_);
  // ---- the waves of a head meet in LDS
  auto& part = *reinterpret_cast<WavePart<D, NCT>*>(mine);
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    const float l = sum_across<32>(sum_across<16>(c_.l[ct]));
    const int col = ct * 16 + t16;
    if (col >= ncols) continue;
    if (g == 0) lds.state[w.sub * w.waves + w.sw][col] = float2{c_.top[ct], l};
#pragma unroll
    for (int h = 0; h < D / 128; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f32x4_t w0, w1;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          w0[n] = c_.o[ct][h][n][i];
          w1[n] = c_.o[ct][h][4 + n][i];
        }
        float* dst = &part.o[h * 16 + 4 * g + i][col * 8];
        *reinterpret_cast<f32x4_t*>(dst) = w0;
        *reinterpret_cast<f32x4_t*>(dst + 4) = w1;
      }
  }
  __syncthreads();
  put_waves_together<D, NCT, F16, NW>(p, lds, x, hg, w);
  if (x.n_shares == 1) return;
  wait_all_vm();  // this wave's partials are where every CU sees them
  __syncthreads();
  if (threadIdx.x == 0) {
    const bool last = count_one(word, p.nonce) == x.n_shares - 1;
    if (last) st_agent(word, 0ull);  // as of a launch that never happened: the next replay counts anew
    lds.last = last;
  }
  __syncthreads();
  if (lds.last) put_shares_together<D, F16>(p, x, hg, w);
}

template <int D, int NCT, int NW, bool F16>
int launch_walk(const ShareParams& p, dim3 grid, hipStream_t stream) {
  auto launch = [&](auto w) {
    return launch_kernel(mxfp4_attention_kernel<D, NCT, F16, decltype(w)::value, NW>, grid, dim3(64 * NW), stream, p);
  };
  return p.walk == (kStream | kWide) ? launch(std::integral_constant<int, kStream | kWide>{})
         : p.walk == kStream         ? launch(std::integral_constant<int, kStream>{})
         : p.walk == kWide           ? launch(std::integral_constant<int, kWide>{})
                                     : launch(std::integral_constant<int, kNarrow>{});
}

// Columns that a workgroup's waves hold, and the blocks of queries, with all their q heads of a kv head, that a request's are cut into: each reads the keys anew.
constexpr int64_t most_columns(int64_t head_dim) { return head_dim == 128 ? 64 : 32; }
struct QueryBlocks {
  int64_t blocks, queries, cols;  // queries and columns of one
  QueryBlocks(int64_t group, int64_t head_dim, int64_t max_len_extend) {
    const int64_t most = std::max<int64_t>(most_columns(head_dim) / group, 1);
    blocks = (max_len_extend + most - 1) / most;
    queries = (max_len_extend + blocks - 1) / blocks;
    cols = queries * group;
  }
};

// How a launch is cut: waves of a workgroup, kv heads of one, shares that fit on the card at once and the most that there can be.
struct Plan {
  int waves, heads, min_len;
  int64_t shares, max_shares;
};
int64_t shares_at_once(int64_t batch, int64_t n_kv, int heads, int64_t blocks, bool two_to_a_cu) {
  const int64_t shares = std::max<int64_t>(device_cus() / (n_kv / heads * blocks), 1);
  return two_to_a_cu && batch > shares ? 2 * shares : shares;
}
// Which of them, by what a launch takes for each, in us, of the average request:
//   bytes     at 6 TB/s with 4 heads to a workgroup, whose lines lie side by side, in 1.25 of that with 2 and 1.7 with 1; 8 waves of 8 heads, 1 KiB a slot, are
//             faster still; longer by the CUs that get none (16 requests of 64 K keys, 8 heads: 200 us with 8, 220 with 4, 259 with 2, 379 with 1)
//             Two tiles of columns are bound by their arithmetic as well, and want two waves to a SIMD: 8 waves of 4 heads 0.98, of 2 1.2 (32 requests of 4 K keys, 32
//             columns: 4 heads with 4 waves 51.1 us, with 8 48.4, 2 heads 51.5 and 49.6)
//   a wave    0.018 a key and tile of columns, where there is little else (one request of 2 K keys, 4 heads 13.7 us, 2 10.3, 1 8.6)
//   the merge 3, and 2 a trip of the loop in put_shares_together(), of which the more heads a workgroup has the more shares there are and the fewer threads to a head (16 of 4 K
//             keys, 64 columns: 4 heads 91.4, 1 head 57.7; 32 columns of head_dim 256 81.7 and 35.1)
// Lengths count by their mean alone: what a long request among many short ones takes is not in it.
Plan plan_of(int64_t batch, int64_t keys, int64_t n_kv, int64_t head_dim, const QueryBlocks& q) {
  const int64_t cols = q.cols;
  const float wave_key = 0.018f * (float)((cols + 15) / 16);
  // More requests than CUs for them: two workgroups to a CU, so that the longest can be cut (300 requests of 500-1500 keys, 8 heads: 109.7 and 79.0 us).  Where a
  // CU has a share for every request it takes one (256 of 1-3 K: 119 and 133).
  const bool one_tile = cols <= 16 && head_dim == 128, two_tiles = cols <= (head_dim == 128 ? 32 : 16);  // LDS and registers for 16 and for 8 waves
  Plan best{};
  float least = 0.f;
  auto consider = [&](int waves, int heads, float rate, int min_len) {
    const int64_t shares = shares_at_once(batch, n_kv, heads, q.blocks, one_tile || (two_tiles && waves == 4));
    const float request = (float)keys / (float)batch;
    const float len = std::max(request / std::max((float)shares / (float)batch, 1.f), (float)min_len);
    const int n = std::max((int)(request / len + 0.5f), 1);
    const float loops = (float)(cols * head_dim / 4) / (float)(64 * waves / heads) / (n <= 4 ? 4.f : n <= 8 ? 2.f : 1.f);
    const float idle = std::max((float)shares / (float)(n * batch), 1.f);
    const float uneven = shares <= batch ? 1.15f : 1.f;  // nothing is cut: the longest request decides
    const float stream = std::max((float)(keys * n_kv * head_dim * q.blocks) * (17.f / 16.f / 6e6f) * rate * idle * uneven, wave_key * len * (float)heads / (float)waves);
    const float cost = stream + (n > 1 ? 3.f + 2.f * loops * std::ceil((float)n / 16.f) : 0.f);
    if (best.waves != 0 && cost >= least) return;
    least = cost;
    best = {waves, heads, min_len, shares, 0};
  };
  for (int min_len = 128; min_len <= (cols <= 16 ? 128 : 1024); min_len *= 2) {
    consider(4, 1, 1.7f, min_len);
    if (n_kv % 2 == 0) consider(4, 2, 1.25f, min_len);
    if (n_kv % 4 == 0) consider(4, 4, 1.f, min_len);
    if (head_dim != 128 || cols > 32) continue;  // (8 waves' accumulators are no room for)
    if (n_kv % 8 == 0) consider(8, 8, 0.93f, min_len);
    if (cols <= 16) continue;
    if (n_kv % 2 == 0) consider(8, 2, 1.2f, min_len);
    if (n_kv % 4 == 0) consider(8, 4, 0.98f, min_len);
  }
  best.max_shares = best.shares + batch;
  return best;
}
size_t counts_bytes(int64_t batch, int64_t n_kv, int64_t blocks) { return (size_t)(blocks * batch * n_kv) * kCountWords * sizeof(unsigned long long); }

}  // namespace

// Short query blocks: those in few enough blocks of queries, each of which reads and converts the keys again, that unpacking them for the 16-bit pool's
// kernels takes longer.  32 requests of 4 K keys of 8 heads, 8 q heads each, us with the codes read and unpacked: 16 queries (2 blocks) 168 and 305, 24 (3)
// 274 and 319, 32 (4) 320 and 336, 8 of 2 K 52 and 50; 2 heads of 256: 8 queries (2) 57 and 153, 16 (4) 95 and 165, 32 (8) 168 and 202, 8 of 4 K 48 and 52.
bool mxfp4_reads_codes(int64_t group, int64_t head_dim, int64_t max_len_extend) {
  const QueryBlocks q(group, head_dim, max_len_extend);
  return q.cols <= most_columns(head_dim) && q.blocks <= (head_dim == 128 ? 3 : 8);
}

// For every plan: which one it is may depend on a window
size_t mxfp4_attention_workspace_bytes(int64_t batch, int64_t n_q, int64_t n_kv, int64_t head_dim, int64_t max_len_extend) {
  const QueryBlocks q(n_q / n_kv, head_dim, max_len_extend);
  int64_t most = 0;
  for (int heads = 1; heads <= (q.cols <= 32 ? 8 : 4) && n_kv % heads == 0; heads *= 2) most = std::max(most, shares_at_once(batch, n_kv, heads, q.blocks, true));
  most += batch;
  return counts_bytes(batch, n_kv, q.blocks) + (size_t)(q.blocks * most * n_kv * q.cols) * (size_t)(head_dim + 1) * sizeof(float);
}

int launch_mxfp4_attention(const Mxfp4AttentionArgs& a, hipStream_t stream) {
  const int64_t n_kv = a.pool.n_kv, d = a.pool.head_dim;
  const QueryBlocks q(a.n_q / n_kv, d, a.max_len_extend);
  const int64_t cols = q.cols;
  if (cols < 1 || cols > most_columns(d) || q.blocks > 65535) return MSGL_ERR_SHAPE;
  if (a.f16 && cols > 16) return MSGL_ERR_DTYPE;
  const int64_t keys = visible_keys(a.batch, a.total_kv, a.window, q.queries, a.is_cross != 0);
  const Plan plan = plan_of(a.batch, keys, n_kv, d, q);
  ShareParams p{};
  p.q = static_cast<const uint16_t*>(a.q);
  p.k_cache = static_cast<const uint16_t*>(a.pool.codes);  // as bytes, strides too
  p.v_cache = static_cast<const uint16_t*>(a.pool.scales);
  p.k_stride0 = a.pool.codes_stride0;
  p.v_stride0 = a.pool.scales_stride0;
  p.kv_indptr = a.kv_indptr;
  p.kv_indices = a.kv_indices;
  p.qo_indptr = a.qo_indptr;
  p.prefix_lens = a.prefix_lens;
  p.out = static_cast<uint16_t*>(a.out);
  p.q_stride0 = a.n_q * d;
  p.batch = (int32_t)a.batch;
  p.n_q = (int32_t)a.n_q;
  p.n_kv = (int32_t)n_kv;
  p.group = (int32_t)(a.n_q / n_kv);
  p.per_group = 65535u / (uint32_t)p.group + 1u;
  p.cols = (int32_t)cols;
  p.max_len_extend = (int32_t)q.queries;
  p.q_cap = a.max_len_extend;
  p.f16 = a.f16;
  p.is_cross = a.is_cross;
  p.window = a.window;
  p.max_slot = (uint32_t)(a.pool.num_slots - 1);
  p.negate = a.sm_scale < 0.f ? -1 : a.sm_scale == 0.f ? 1 : 0;
  p.scale_log2e = a.sm_scale == 0.f ? 1.f : std::fabs(a.sm_scale) * kLog2e * (a.f16 ? 2.f : 1.f);
  const int64_t stride = std::max(a.pool.codes_stride0, a.pool.scales_stride0);
  const bool wide = a.pool.num_slots > 1 << 24 || stride >= 1 << 24 || (uint64_t)a.pool.num_slots * (uint64_t)stride >= (1ull << 32);
  p.walk = (wide ? kWide : kNarrow) | (streams(keys * n_kv * (d + d / 16)) ? kStream : kNarrow);
  p.nwh = plan.heads;
  p.head_groups = (int32_t)(n_kv / plan.heads);
  p.shares = (int32_t)plan.shares;
  p.min_len = (float)plan.min_len;
  p.wave_shift = __builtin_ctz((unsigned)(plan.waves / plan.heads));
  p.counts = static_cast<unsigned long long*>(a.workspace);
  p.part_o = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + counts_bytes(a.batch, n_kv, q.blocks));
  p.part_lse = p.part_o + (size_t)(plan.max_shares * q.blocks) * (size_t)(n_kv * cols) * (size_t)d;
  p.nonce = next_launch_number();
  const int64_t units = plan.max_shares * p.head_groups;
  if (units > 0x7fffffffLL) return MSGL_ERR_SHAPE;
  const dim3 grid((unsigned)units, (unsigned)q.blocks);
  const int nct = (int)((cols + 15) / 16);
  auto launch = [&](auto dim, auto tiles, auto half) {
    constexpr int D = decltype(dim)::value, NCT = decltype(tiles)::value;
    constexpr bool F16 = decltype(half)::value;
    if constexpr (D == 128 && NCT <= 2) {
      if (plan.waves == 8) return launch_walk<D, NCT, 8, F16>(p, grid, stream);
    }
    return launch_walk<D, NCT, 4, F16>(p, grid, stream);
  };
  using std::integral_constant;
  if (d == 128) {
    if (a.f16) return launch(integral_constant<int, 128>{}, integral_constant<int, 1>{}, std::true_type{});
    if (nct == 1) return launch(integral_constant<int, 128>{}, integral_constant<int, 1>{}, std::false_type{});
    if (nct == 2) return launch(integral_constant<int, 128>{}, integral_constant<int, 2>{}, std::false_type{});
    return launch(integral_constant<int, 128>{}, integral_constant<int, 4>{}, std::false_type{});
  }
  if (a.f16) return launch(integral_constant<int, 256>{}, integral_constant<int, 1>{}, std::true_type{});
  if (nct == 1) return launch(integral_constant<int, 256>{}, integral_constant<int, 1>{}, std::false_type{});
  return launch(integral_constant<int, 256>{}, integral_constant<int, 2>{}, std::false_type{});
}

}  // namespace msgl
