// Rows of a K/V pool in 4 bits (mxfp4.h): the store, the way back, and the store with the q/k norm and the rotary embedding in front.
//
// All three move bytes: a token's K and V of a head are 4 D bytes in 16 bits and D + D / 16 in the pool.
#include "msgl_internal.h"
#include "mxfp4.h"

namespace msgl {
namespace {

constexpr int kThreads = 256;
// Rows of a thread, on their way at once: 11.6 K rows of 8 heads of 128 take 12.7 us to be stored and 10.2 to be loaded with two, 14.0 and 11.7 with one,
// 14.0 and 10.8 with four; 64 K of them 67.6 us (5.0 TB/s) to be unpacked with four in a loop, 91 with one.
constexpr int kRows = 2, kUnpackRows = 4;

__device__ __forceinline__ float value16(uint32_t w, int half, bool f16) {
  const uint32_t h = half ? w >> 16 : w & 0xffffu;
  return f16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h) : __builtin_bit_cast(float, h << 16);
}
// Or over the 16 lanes' four groups of four, whose lanes agree
__device__ __forceinline__ uint32_t or_of_blocks(uint32_t v) {
  v |= (uint32_t)dpp<0x124>((int)v);  // the lane 4 below, with rotation
  return v | (uint32_t)dpp<0x128>((int)v);
}

struct StoreParams {
  unsigned char *codes, *scales;
  const int32_t* indices;
  const uint16_t *k, *v;
  int64_t codes_stride, scales_stride, k_stride0, v_stride0, num_slots;  // of the pool in bytes
  uint32_t items, n_kv;                                                  // (row, kv head)
};

// D / 4 lanes to a (row, kv head), half of them K's and half V's, 8 dims each; a block is 4 lanes.
template <int D, bool F16>
__global__ __launch_bounds__(kThreads) void store_mxfp4_kernel(StoreParams p) {
  constexpr int kRowLanes = D / 8, kLanes = 2 * kRowLanes, kAtOnce = kThreads / kLanes;
  const int lane = threadIdx.x % kLanes, of_v = lane / kRowLanes, j = lane % kRowLanes;
  const uint32_t first = blockIdx.x * (kAtOnce * kRows) + threadIdx.x / kLanes;
  uint32_t head[kRows];
  int64_t slot[kRows];
  u32x4_t raw[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const uint32_t item = min(first + u * kAtOnce, p.items - 1);  // lanes of no item stay for the exchanges
    const uint32_t row = item / p.n_kv;
    head[u] = item - row * p.n_kv;
    raw[u] = ld_global_b128((of_v ? p.v + row * p.v_stride0 : p.k + row * p.k_stride0) + head[u] * D + j * 8);
    slot[u] = p.indices[row];
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    float x[8];
    uint32_t top = 0;  // the largest value's bits, with what is not finite above all others
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = value16(raw[u][e >> 1], e & 1, F16);
      top = max(top, __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu);
    }
    // one lane's is everybody's of the (row, kv head)
    const uint64_t of_item = kLanes == 64 ? ~0ull : ((1ull << (kLanes & 63)) - 1) << (lane_id() & ~(kLanes - 1) & 63);
    const bool poison = (__ballot(top >= 0x7f800000u) & of_item) != 0;
    top = max(top, (uint32_t)dpp<0xB1>((int)top));
    top = max(top, (uint32_t)dpp<0x4E>((int)top));
    if (poison) {
      top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
    }
    const int byte = mx_block_byte(top);
    const uint32_t codes = mx_codes8(x, byte);
    const uint32_t scales = or_of_blocks((uint32_t)(poison && !of_v ? kMxNotFinite : byte) << (8 * ((lane >> 2) & 3)));
    if (first + u * kAtOnce < p.items && (uint64_t)slot[u] < (uint64_t)p.num_slots) {
      *reinterpret_cast<uint32_t*>(p.codes + slot[u] * p.codes_stride + head[u] * D + lane * 4) = codes;
      if ((lane & 15) == 0)
        *reinterpret_cast<uint32_t*>(p.scales + slot[u] * p.scales_stride + head[u] * (D / 16) + (lane >> 4) * 4) = scales;
    }
  }
}

struct LoadParams {
  const unsigned char *codes, *scales;
  const int32_t* indices;
  uint16_t *k, *v;
  int64_t codes_stride, scales_stride;
  uint32_t items, n_kv, max_slot;
};

template <int D, bool F16>
__global__ __launch_bounds__(kThreads) void load_mxfp4_kernel(LoadParams p) {
  constexpr int kRowLanes = D / 8, kLanes = 2 * kRowLanes, kAtOnce = kThreads / kLanes;
  const int lane = threadIdx.x % kLanes, of_v = lane / kRowLanes, j = lane % kRowLanes;
  const uint32_t first = blockIdx.x * (kAtOnce * kRows) + threadIdx.x / kLanes;
  uint32_t item[kRows], head[kRows], slot[kRows], codes[kRows], byte[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    item[u] = min(first + u * kAtOnce, p.items - 1);
    const uint32_t row = item[u] / p.n_kv;
    head[u] = item[u] - row * p.n_kv;
    slot[u] = min((uint32_t)p.indices[row], p.max_slot);
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    codes[u] = *reinterpret_cast<const uint32_t*>(p.codes + slot[u] * p.codes_stride + head[u] * D + lane * 4);
    byte[u] = p.scales[slot[u] * p.scales_stride + head[u] * (D / 16) + (lane >> 2)];
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    if (first + u * kAtOnce >= p.items) return;
    st_global_b128((of_v ? p.v : p.k) + (int64_t)item[u] * D + j * 8, mx_values8<F16>(codes[u], mx_scale(byte[u])));
  }
}

struct UnpackParams {
  const unsigned char *codes, *scales;
  const int32_t *kv_indptr, *kv_indices, *prefix_lens;
  uint16_t *k, *v;
  int32_t* numbers;
  int64_t codes_stride, scales_stride;
  int32_t batch, total_kv, window, per_request;  // workgroups to a request, 0: they share all positions out
  uint32_t n_kv, max_slot;
};

// The listed rows as bf16 for the tile kernels, D / 4 lanes to a (position, kv head).  Those read whole tiles of 64 keys from the one that
// holds a query's first visible key on, up to the request's last key, and V of a key that the mask hides meets a weight of zero: it has to be there.
template <int D>
__global__ __launch_bounds__(kThreads) void unpack_mxfp4_kernel(UnpackParams p) {
  constexpr int kRowLanes = D / 8, kLanes = 2 * kRowLanes, kAtOnce = kThreads / kLanes;
  const int lane = threadIdx.x % kLanes, of_v = lane / kRowLanes, j = lane % kRowLanes;
  int64_t begin = 0, end = p.total_kv, step = gridDim.x, first = blockIdx.x;
  if (p.per_request > 0) {
    const int b = blockIdx.x / p.per_request;
    first = blockIdx.x - b * p.per_request;
    step = p.per_request;
    const int start = p.kv_indptr[b];
    end = min((int64_t)p.kv_indptr[b + 1], end);
    begin = start + (max(p.prefix_lens[b] - p.window + 1, 0) & ~127);
  }
  const uint32_t items = (uint32_t)max(end - begin, (int64_t)0) * p.n_kv;
  for (uint32_t at0 = (uint32_t)first * kAtOnce * kUnpackRows + threadIdx.x / kLanes; at0 < items; at0 += (uint32_t)step * kAtOnce * kUnpackRows) {
    uint32_t row[kUnpackRows], head[kUnpackRows], codes[kUnpackRows], byte[kUnpackRows];
#pragma unroll
    for (int u = 0; u < kUnpackRows; ++u) {
      const uint32_t at = min(at0 + u * kAtOnce, items - 1);
      const uint32_t r = at / p.n_kv;
      row[u] = (uint32_t)begin + r;
      head[u] = at - r * p.n_kv;
    }
    uint32_t slot[kUnpackRows];
#pragma unroll
    for (int u = 0; u < kUnpackRows; ++u) slot[u] = min((uint32_t)p.kv_indices[row[u]], p.max_slot);
#pragma unroll
    for (int u = 0; u < kUnpackRows; ++u) {
      codes[u] = *reinterpret_cast<const uint32_t*>(p.codes + slot[u] * p.codes_stride + head[u] * D + lane * 4);
      byte[u] = p.scales[slot[u] * p.scales_stride + head[u] * (D / 16) + (lane >> 2)];
    }
#pragma unroll
    for (int u = 0; u < kUnpackRows; ++u) {
      if (at0 + u * kAtOnce >= items) break;
      st_global_b128((of_v ? p.v : p.k) + ((int64_t)row[u] * p.n_kv + head[u]) * D + j * 8, mx_values8<false>(codes[u], mx_scale(byte[u])));
      if (head[u] == 0 && lane == 0) p.numbers[row[u]] = (int32_t)row[u];
    }
  }
}

}  // namespace

int launch_unpack_mxfp4(const Mxfp4UnpackArgs& a, hipStream_t stream) {
  UnpackParams p{};
  p.codes = static_cast<const unsigned char*>(a.pool.codes);
  p.scales = static_cast<const unsigned char*>(a.pool.scales);
  p.kv_indptr = a.kv_indptr;
  p.kv_indices = a.kv_indices;
  p.prefix_lens = a.prefix_lens;
  p.k = static_cast<uint16_t*>(a.k);
  p.v = static_cast<uint16_t*>(a.v);
  p.numbers = a.numbers;
  p.codes_stride = a.pool.codes_stride0;
  p.scales_stride = a.pool.scales_stride0;
  p.batch = (int32_t)a.batch;
  p.total_kv = (int32_t)a.total_kv;
  p.window = a.window;
  p.n_kv = (uint32_t)a.pool.n_kv;
  p.max_slot = (uint32_t)(a.pool.num_slots - 1);
  if (a.total_kv * a.pool.n_kv > 0x7fffffffLL) return MSGL_ERR_SHAPE;
  const int64_t at_once = kUnpackRows * (kThreads / (a.pool.head_dim / 4)), most = 16 * (int64_t)device_cus();
  auto blocks = [&](int64_t keys) { return std::max<int64_t>(1, (keys * a.pool.n_kv + at_once - 1) / at_once); };
  int64_t grid = std::min(blocks(a.total_kv), most);
  if (a.window > 0) {
    const int64_t each = std::min(blocks((int64_t)a.window + a.max_len_extend + 128), std::max<int64_t>(1, most / a.batch));
    p.per_request = (int32_t)each;
    grid = each * a.batch;
  }
  if (grid > 0x7fffffffLL) return MSGL_ERR_SHAPE;
  const auto kernel = a.pool.head_dim == 128 ? unpack_mxfp4_kernel<128> : unpack_mxfp4_kernel<256>;
  return launch_kernel(kernel, dim3((unsigned)grid), dim3(kThreads), stream, p);
}

int launch_store_mxfp4(const Mxfp4StoreArgs& a, hipStream_t stream) {
  const int64_t items = a.length * a.pool.n_kv, per_block = kRows * (kThreads / (a.pool.head_dim / 4));
  if (items >= (int64_t)1 << 31) return MSGL_ERR_SHAPE;
  StoreParams p{};
  p.codes = static_cast<unsigned char*>(a.pool.codes);
  p.scales = static_cast<unsigned char*>(a.pool.scales);
  p.indices = a.indices;
  p.k = static_cast<const uint16_t*>(a.k);
  p.v = static_cast<const uint16_t*>(a.v);
  p.codes_stride = a.pool.codes_stride0;
  p.scales_stride = a.pool.scales_stride0;
  p.k_stride0 = a.k_stride0;
  p.v_stride0 = a.v_stride0;
  p.num_slots = a.pool.num_slots;
  p.items = (uint32_t)items;
  p.n_kv = (uint32_t)a.pool.n_kv;
  const auto kernel = a.pool.head_dim == 128 ? (a.f16 ? store_mxfp4_kernel<128, true> : store_mxfp4_kernel<128, false>)
                                             : (a.f16 ? store_mxfp4_kernel<256, true> : store_mxfp4_kernel<256, false>);
  return launch_kernel(kernel, dim3((unsigned)((items + per_block - 1) / per_block)), dim3(kThreads), stream, p);
}

int launch_load_mxfp4(const Mxfp4LoadArgs& a, hipStream_t stream) {
  const int64_t items = a.length * a.pool.n_kv, per_block = kRows * (kThreads / (a.pool.head_dim / 4));
  if (items >= (int64_t)1 << 31) return MSGL_ERR_SHAPE;
  LoadParams p{};
  p.codes = static_cast<const unsigned char*>(a.pool.codes);
  p.scales = static_cast<const unsigned char*>(a.pool.scales);
  p.indices = a.indices;
  p.k = static_cast<uint16_t*>(a.k);
  p.v = static_cast<uint16_t*>(a.v);
  p.codes_stride = a.pool.codes_stride0;
  p.scales_stride = a.pool.scales_stride0;
  p.items = (uint32_t)items;
  p.n_kv = (uint32_t)a.pool.n_kv;
  p.max_slot = (uint32_t)(a.pool.num_slots - 1);
  const auto kernel = a.pool.head_dim == 128 ? (a.f16 ? load_mxfp4_kernel<128, true> : load_mxfp4_kernel<128, false>)
                                             : (a.f16 ? load_mxfp4_kernel<256, true> : load_mxfp4_kernel<256, false>);
  return launch_kernel(kernel, dim3((unsigned)((items + per_block - 1) / per_block)), dim3(kThreads), stream, p);
}

}  // namespace msgl
