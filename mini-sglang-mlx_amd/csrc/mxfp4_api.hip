// extern "C" entry points of include/msgl_mxfp4_cache.h: argument checks, and which kernels a prefill call takes.
#include <algorithm>

#include "msgl_internal.h"

namespace {

using msgl::Mxfp4Pool;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_dtype(int32_t dtype, bool f16_ok) {
  return dtype == MSGL_DTYPE_BF16 || (f16_ok && dtype == MSGL_DTYPE_F16) ? MSGL_OK : MSGL_ERR_DTYPE;
}
int check_sizes(int64_t n_kv, int64_t d, int64_t num_slots, int64_t codes_stride0, int64_t scales_stride0) {
  if (d != 128 && d != 256) return MSGL_ERR_HEAD_DIM;
  if (n_kv <= 0 || n_kv > (1 << 20) || num_slots <= 0 || num_slots > 0x80000000ll) return MSGL_ERR_SHAPE;
  if (codes_stride0 < n_kv * d || scales_stride0 < n_kv * (d / 16)) return MSGL_ERR_SHAPE;
  if (codes_stride0 > 0xffffffffll || scales_stride0 > 0xffffffffll) return MSGL_ERR_SHAPE;  // of 32 bits in the attention's walk
  return MSGL_OK;
}
int check_pool(const Mxfp4Pool& pool) {
  if (!pool.codes || !pool.scales) return MSGL_ERR_NULL_POINTER;
  if (!aligned16(pool.codes) || reinterpret_cast<uintptr_t>(pool.scales) % 8 || pool.codes_stride0 % 16 || pool.scales_stride0 % 8) return MSGL_ERR_ALIGNMENT;
  return MSGL_OK;
}
Mxfp4Pool pool_of(const void* codes, const void* scales, int64_t codes_stride0, int64_t scales_stride0, int64_t num_slots, int64_t n_kv, int64_t d) {
  return Mxfp4Pool{const_cast<void*>(codes), const_cast<void*>(scales), codes_stride0, scales_stride0, num_slots, n_kv, d};
}
// Of attention: the partials of a request, which a share's workgroup addresses by 32 bits, are at most 32 KiB a kv head and share, and there are
// at most 4096 + 2 n_kv of those.
constexpr int64_t kMostKvHeads = 1 << 15;
int check_heads(int64_t n_q, int64_t n_kv) {
  if (n_q <= 0 || n_kv > kMostKvHeads) return MSGL_ERR_SHAPE;
  return n_q % n_kv != 0 ? MSGL_ERR_HEAD_RATIO : MSGL_OK;
}

// The unpacked rows of a prefill call, in front of the tile kernels' own workspace.
struct Unpacked {
  size_t k, v, numbers, rest;  // offsets
};
Unpacked unpacked(int64_t total_kv, int64_t n_kv, int64_t d) {
  auto whole = [](size_t bytes) { return (bytes + 255) / 256 * 256; };
  const size_t rows = whole((size_t)total_kv * n_kv * d * 2);
  return Unpacked{0, rows, 2 * rows, 2 * rows + whole((size_t)total_kv * sizeof(int32_t))};
}
constexpr int64_t kMostKeys = (int64_t)1 << 30;  // listed: a wave's place among a share's ids is 32 bits of bytes
bool reads_pool(int64_t n_q, int64_t n_kv, int64_t d, int64_t max_len_extend) { return msgl::mxfp4_reads_codes(n_q / n_kv, d, max_len_extend); }

}  // namespace

extern "C" {

int msgl_store_kv_cache_mxfp4(void* kv_codes, void* kv_scales, const int32_t* indices, const void* k, const void* v, int64_t length,
                              int64_t num_kv_heads, int64_t head_dim, int64_t num_slots, int64_t codes_stride0,
                              int64_t scales_stride0, int64_t k_stride0, int64_t v_stride0, int32_t dtype, void* stream) {
  if (length < 0) return MSGL_ERR_SHAPE;
  if (const int rc = check_sizes(num_kv_heads, head_dim, num_slots, codes_stride0, scales_stride0)) return rc;
  if (const int rc = check_dtype(dtype, true)) return rc;
  if (k_stride0 < num_kv_heads * head_dim || v_stride0 < num_kv_heads * head_dim) return MSGL_ERR_SHAPE;
  if (length == 0) return MSGL_OK;
  msgl::Mxfp4StoreArgs a{};
  a.pool = pool_of(kv_codes, kv_scales, codes_stride0, scales_stride0, num_slots, num_kv_heads, head_dim);
  if (!indices || !k || !v) return MSGL_ERR_NULL_POINTER;
  if (const int rc = check_pool(a.pool)) return rc;
  if (!aligned16(k) || !aligned16(v) || k_stride0 % 8 || v_stride0 % 8) return MSGL_ERR_ALIGNMENT;
  a.indices = indices;
  a.k = k;
  a.v = v;
  a.length = length;
  a.k_stride0 = k_stride0;
  a.v_stride0 = v_stride0;
  a.f16 = dtype == MSGL_DTYPE_F16;
  return msgl::launch_store_mxfp4(a, static_cast<hipStream_t>(stream));
}

int msgl_load_kv_cache_mxfp4(const void* kv_codes, const void* kv_scales, const int32_t* indices, void* k, void* v, int64_t length,
                             int64_t num_kv_heads, int64_t head_dim, int64_t num_slots, int64_t codes_stride0,
                             int64_t scales_stride0, int32_t dtype, void* stream) {
  if (length < 0) return MSGL_ERR_SHAPE;
  if (const int rc = check_sizes(num_kv_heads, head_dim, num_slots, codes_stride0, scales_stride0)) return rc;
  if (const int rc = check_dtype(dtype, true)) return rc;
  if (length == 0) return MSGL_OK;
  msgl::Mxfp4LoadArgs a{};
  a.pool = pool_of(kv_codes, kv_scales, codes_stride0, scales_stride0, num_slots, num_kv_heads, head_dim);
  if (!indices || !k || !v) return MSGL_ERR_NULL_POINTER;
  if (const int rc = check_pool(a.pool)) return rc;
  if (!aligned16(k) || !aligned16(v)) return MSGL_ERR_ALIGNMENT;
  a.indices = indices;
  a.k = k;
  a.v = v;
  a.length = length;
  a.f16 = dtype == MSGL_DTYPE_F16;
  return msgl::launch_load_mxfp4(a, static_cast<hipStream_t>(stream));
}

int msgl_qk_norm_rope_store_mxfp4(const void* q, const void* k, const void* v, int64_t q_stride0, int64_t k_stride0, int64_t v_stride0,
                                  const void* q_weight, const void* k_weight, const int32_t* positions, const int32_t* out_loc,
                                  void* q_out, void* kv_codes, void* kv_scales, int64_t codes_stride0, int64_t scales_stride0,
                                  int64_t num_slots, int64_t n_tokens, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                  double rms_norm_eps, double rope_base, int32_t dtype, void* stream) {
  if (n_tokens < 0 || num_q_heads <= 0 || num_q_heads > (1 << 20)) return MSGL_ERR_SHAPE;
  if (const int rc = check_sizes(num_kv_heads, head_dim, num_slots, codes_stride0, scales_stride0)) return rc;
  if (const int rc = check_dtype(dtype, false)) return rc;
  if (!(rope_base > 1.0) || !(rope_base < 1e300) || !(rms_norm_eps >= 0.0)) return MSGL_ERR_SHAPE;
  if (q_stride0 < num_q_heads * head_dim || k_stride0 < num_kv_heads * head_dim || v_stride0 < num_kv_heads * head_dim) return MSGL_ERR_SHAPE;
  if (n_tokens == 0) return MSGL_OK;
  msgl::Mxfp4NormRopeArgs a{};
  a.pool = pool_of(kv_codes, kv_scales, codes_stride0, scales_stride0, num_slots, num_kv_heads, head_dim);
  if (!q || !k || !v || !q_weight || !k_weight || !positions || !out_loc || !q_out) return MSGL_ERR_NULL_POINTER;
  if (const int rc = check_pool(a.pool)) return rc;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(q_weight) || !aligned16(k_weight) || !aligned16(q_out) || q_stride0 % 8 ||
      k_stride0 % 8 || v_stride0 % 8)
    return MSGL_ERR_ALIGNMENT;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.positions = positions;
  a.out_loc = out_loc;
  a.q_out = q_out;
  a.q_stride0 = q_stride0;
  a.k_stride0 = k_stride0;
  a.v_stride0 = v_stride0;
  a.n_tokens = n_tokens;
  a.n_q = num_q_heads;
  a.eps = rms_norm_eps;
  a.rope_base = rope_base;
  return msgl::launch_norm_rope_store_mxfp4(a, static_cast<hipStream_t>(stream));
}

size_t msgl_paged_decode_mxfp4_workspace_bytes(int64_t batch, int64_t total_kv, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim) {
  if (batch <= 0 || total_kv < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0) return 0;
  return msgl::mxfp4_attention_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim, 1);
}

int msgl_paged_decode_attention_mxfp4(const void* q, const void* kv_codes, const void* kv_scales, const int32_t* kv_indptr,
                                      const int32_t* kv_indices, void* out, void* workspace, size_t workspace_bytes, int64_t batch,
                                      int64_t total_kv, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                      int64_t num_slots, int64_t codes_stride0, int64_t scales_stride0, float sm_scale, int32_t dtype,
                                      void* stream) {
  if (batch < 0 || total_kv < 0 || batch > 0x7fffffffLL || total_kv > kMostKeys) return MSGL_ERR_SHAPE;
  if (const int rc = check_sizes(num_kv_heads, head_dim, num_slots, codes_stride0, scales_stride0)) return rc;
  if (const int rc = check_heads(num_q_heads, num_kv_heads)) return rc;
  if (num_q_heads / num_kv_heads > 16) return MSGL_ERR_GROUP_TOO_LARGE;
  if (const int rc = check_dtype(dtype, true)) return rc;
  if (batch == 0) return MSGL_OK;
  msgl::Mxfp4AttentionArgs a{};
  a.pool = pool_of(kv_codes, kv_scales, codes_stride0, scales_stride0, num_slots, num_kv_heads, head_dim);
  if (!q || !out || !kv_indptr || (total_kv > 0 && !kv_indices)) return MSGL_ERR_NULL_POINTER;
  if (const int rc = check_pool(a.pool)) return rc;
  if (!aligned16(q) || !aligned16(out)) return MSGL_ERR_ALIGNMENT;
  if (!workspace || !aligned16(workspace) ||
      workspace_bytes < msgl::mxfp4_attention_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim, 1))
    return MSGL_ERR_WORKSPACE;
  a.q = q;
  a.kv_indptr = kv_indptr;
  a.kv_indices = kv_indices;
  a.out = out;
  a.workspace = workspace;
  a.batch = batch;
  a.total_kv = total_kv;
  a.n_q = num_q_heads;
  a.sm_scale = sm_scale;
  a.max_len_extend = 1;
  a.f16 = dtype == MSGL_DTYPE_F16;
  return msgl::launch_mxfp4_attention(a, static_cast<hipStream_t>(stream));
}

size_t msgl_paged_prefill_mxfp4_workspace_bytes(int64_t batch, int64_t total_q, int64_t total_kv, int64_t num_q_heads, int64_t num_kv_heads,
                                                int64_t head_dim, int64_t max_len_extend) {
  if (batch <= 0 || total_q < 0 || total_kv < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 || max_len_extend <= 0) return 0;
  if (reads_pool(num_q_heads, num_kv_heads, head_dim, max_len_extend))
    return msgl::mxfp4_attention_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim, max_len_extend);
  return std::max<size_t>(256, unpacked(total_kv, num_kv_heads, head_dim).rest +
                                   msgl_paged_prefill_workspace_bytes(batch, total_q, total_kv, num_q_heads, num_kv_heads, head_dim, max_len_extend));
}

int msgl_paged_prefill_attention_mxfp4(const void* q, const void* kv_codes, const void* kv_scales, const int32_t* qo_indptr,
                                       const int32_t* kv_indptr, const int32_t* kv_indices, const int32_t* prefix_lens, void* out,
                                       void* workspace, size_t workspace_bytes, int64_t batch, int64_t total_q, int64_t total_kv,
                                       int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int64_t num_slots,
                                       int64_t codes_stride0, int64_t scales_stride0, float sm_scale, int32_t max_len_extend,
                                       int32_t is_cross_attention, int32_t sliding_window_size, int32_t dtype, void* stream) {
  if (const int rc = check_sizes(num_kv_heads, head_dim, num_slots, codes_stride0, scales_stride0)) return rc;
  if (const int rc = check_heads(num_q_heads, num_kv_heads)) return rc;
  if (sliding_window_size < 0) return MSGL_ERR_WINDOW;
  if (batch <= 0) return MSGL_ERR_BATCH;
  if (total_q < 0 || total_kv < 0 || batch > 0x7fffffffLL || total_q > 0x7fffffffLL || total_kv > kMostKeys) return MSGL_ERR_SHAPE;
  if (const int rc = check_dtype(dtype, false)) return rc;
  if (total_q == 0 || max_len_extend <= 0) return MSGL_OK;
  const Mxfp4Pool pool = pool_of(kv_codes, kv_scales, codes_stride0, scales_stride0, num_slots, num_kv_heads, head_dim);
  if (!q || !out || !qo_indptr || !kv_indptr || !prefix_lens || (total_kv > 0 && !kv_indices)) return MSGL_ERR_NULL_POINTER;
  if (const int rc = check_pool(pool)) return rc;
  if (!aligned16(q) || !aligned16(out)) return MSGL_ERR_ALIGNMENT;
  if (!workspace || !aligned16(workspace) ||
      workspace_bytes < msgl_paged_prefill_mxfp4_workspace_bytes(batch, total_q, total_kv, num_q_heads, num_kv_heads, head_dim, max_len_extend))
    return MSGL_ERR_WORKSPACE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (reads_pool(num_q_heads, num_kv_heads, head_dim, max_len_extend)) {
    if (batch * max_len_extend > 0x7fffffffLL) return MSGL_ERR_SHAPE;
    msgl::Mxfp4AttentionArgs a{};
    a.pool = pool;
    a.q = q;
    a.kv_indptr = kv_indptr;
    a.kv_indices = kv_indices;
    a.qo_indptr = qo_indptr;
    a.prefix_lens = prefix_lens;
    a.out = out;
    a.workspace = workspace;
    a.batch = batch;
    a.total_kv = total_kv;
    a.n_q = num_q_heads;
    a.sm_scale = sm_scale;
    a.max_len_extend = max_len_extend;
    a.is_cross = is_cross_attention ? 1 : 0;
    a.window = sliding_window_size;
    return msgl::launch_mxfp4_attention(a, s);
  }
  const Unpacked at = unpacked(total_kv, num_kv_heads, head_dim);
  char* ws = static_cast<char*>(workspace);
  msgl::Mxfp4UnpackArgs u{};
  u.pool = pool;
  u.kv_indptr = kv_indptr;
  u.kv_indices = kv_indices;
  u.prefix_lens = prefix_lens;
  u.k = ws + at.k;
  u.v = ws + at.v;
  u.numbers = reinterpret_cast<int32_t*>(ws + at.numbers);
  u.batch = batch;
  u.total_kv = total_kv;
  u.window = is_cross_attention ? 0 : sliding_window_size;
  u.max_len_extend = max_len_extend;
  if (total_kv > 0)
    if (const int rc = msgl::launch_unpack_mxfp4(u, s)) return rc;
  const int64_t row = num_kv_heads * head_dim;
  return msgl_paged_prefill_attention(q, u.k, u.v, qo_indptr, kv_indptr, u.numbers, prefix_lens, out, ws + at.rest, workspace_bytes - at.rest, batch,
                                      total_q, total_kv, num_q_heads, num_kv_heads, head_dim, total_kv, row, row, sm_scale, max_len_extend,
                                      is_cross_attention, sliding_window_size, dtype, stream);
}

}  // extern "C"
