// The stream of visible keys that is cut into equal segments (paged_splitkv.hip, mxfp4_attention.hip): where a segment
// begins, and where the partials lie that the merge kernels of paged_splitkv.hip put together.
#pragma once
#include "splitkv_tiles.h"

namespace msgl {

// Where dim `dim` of column `col` of the partial of (item, kv head) number `block` lives.  Blocks
// of 8 dims are the outer index and columns the inner one: in the attention kernel's accumulator
// layout the 16 lanes of a row group hold the same 8 dims of 16 consecutive columns, so one store
// instruction writes 32 contiguous bytes per lane and 512 contiguous bytes per row group.  (With
// the column as the outer index every lane of a store wrote 16 bytes of a different 512-byte row:
// 64 partial cache lines per instruction, and the partial stores of a share cost as much as
// several microseconds of streaming.)
__device__ __forceinline__ int64_t partial_offset(int64_t block, int cols, int col, int dim, int D) {
  return (block * cols * (int64_t)D) + ((int64_t)(dim >> 3) * cols + col) * 8 + (dim & 7);
}

// A request with visible keys takes their number of positions in the stream plus `boundary`
// positions without tokens behind them.  Starting on the next request costs a workgroup a fixed
// time (its geometry, Q rows, slot ids and first tiles are three dependent memory round trips, and
// the load pipeline drains and refills): measured 8-9 us, the time of about a hundred tokens, and the
// kernel ends when its slowest workgroup does.  Charging the boundary to the segment that crosses it
// gives that workgroup fewer tokens; a segment that ends or starts inside the empty positions just
// has less to do or starts at the next request.
__device__ __forceinline__ int stream_length(const SplitKvParams& p, int visible) {
  return visible > 0 ? visible + p.boundary : 0;
}

// Segments are a multiple of 64 positions long, one trip of the tile loop.  (Multiples of 16 or 32
// fill the last few segments that rounding up to 64 leaves without work, but give every share a
// partly filled trip: measured 0.5-1 % slower on the decode and verify shapes.)
__device__ __forceinline__ int segment_length(int total, int n_seg, int min_seg) {
  const int even = ((total + n_seg - 1) / n_seg + 63) / 64 * 64;
  return max(even, min_seg);
}

// Wave-cooperative: length of the stream, and the request that holds stream position
// `seg * seg_len` (its keys or the empty positions behind them) together with the stream position
// of that request's first key.
// Returns false when the segment starts beyond the stream.  All lanes must call.
__device__ __forceinline__ bool locate_segment(const SplitKvParams& p, int seg, int* seg_len,
                                               int* total_out, int* req, int* req_vstart) {
  const int lane = lane_id();
  int total = 0, n = 0, incl = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kWave) {
    const int b = b0 + lane;
    n = 0;
    if (b < p.batch) {
      const ReqInfo r = request_info(p, b);
      n = stream_length(p, r.hi - r.lo);
    }
    incl = wave_inclusive_scan(n);
    total += __shfl(incl, kWave - 1, kWave);
  }
  total = max(total - p.boundary, 0);  // nothing follows the last request: its empty positions go
  const int len = segment_length(total, p.n_seg, p.min_seg);
  *seg_len = len;
  *total_out = total;
  const int pos = seg * len;
  if (pos >= total) return false;
  int base = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kWave) {
    if (p.batch > kWave) {  // more than one batch of requests: recompute this batch
      const int b = b0 + lane;
      n = 0;
      if (b < p.batch) {
        const ReqInfo r = request_info(p, b);
        n = stream_length(p, r.hi - r.lo);
      }
      incl = wave_inclusive_scan(n);
    }
    const int batch_total = __shfl(incl, kWave - 1, kWave);
    if (pos < base + batch_total) {
      const int first = base + incl - n;
      const bool hit = (pos >= first) && (pos < first + n);
      const int src = __ffsll((long long)__ballot(hit)) - 1;
      *req = b0 + src;
      *req_vstart = __shfl(first, src, kWave);
      return true;
    }
    base += batch_total;
  }
  return false;
}

// Puts the fp32 partials of a launch together (every field of `p` that the kernels of paged_splitkv.hip read set as launch_splitkv() sets it;
// f16: the result's type) and writes zeros where a request sees no key.
int launch_fp32_merge(const SplitKvParams& p, int64_t head_dim, hipStream_t stream);

}  // namespace msgl
