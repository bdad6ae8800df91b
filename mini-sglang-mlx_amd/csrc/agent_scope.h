// What workgroups of one launch leave for each other, whichever XCD they run on: partials, counts (paged_shares.hip, mxfp4_attention.hip).
#pragma once
#include "msgl_device.h"

namespace msgl {

__device__ __forceinline__ void st_agent(unsigned long long* p, unsigned long long v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long ld_agent(const unsigned long long* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// 16 bytes of the partials at agent scope.  (As two 8-byte accesses, the largest there are of atomics, each of them walks all
// the lines that the wave's 16-byte pieces lie in: 24 loads of a thread took 1.5 K cycles to be issued, 48 of head_dim 256 3.8 K.)
constexpr int kAgentScope = 16;  // sc1
struct Partials {
  __amdgpu_buffer_rsrc_t at;
  __device__ __forceinline__ Partials(float* from, uint32_t bytes) : at(__builtin_amdgcn_make_buffer_rsrc(from, 0, bytes, 0x00020000)) {}
  __device__ __forceinline__ f32x4_t load(uint32_t lane_at, uint32_t share_at) const {
    return __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(at, (int)lane_at, (int)share_at, kAgentScope));
  }
  __device__ __forceinline__ void store(uint32_t lane_at, f32x4_t v) const {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, v), at, (int)lane_at, 0, kAgentScope);
  }
};

// Counting in a launch's word (launch_number.h), which may hold anything before.  All that count ask nothing of each other: open() at the start
// makes the word this launch's if the one before it left it as it should, with 0, and nobody waits for that; then one() is one addition.  (Sixteen that find
// a word that is not theirs at the same time, and each try until their own count is in it, took 16 us.)
constexpr int kCountWords = 16;  // 8-byte words from one that is counted in to the next: a line each

__device__ __forceinline__ void open_count(unsigned long long* word, unsigned long long nonce) {
  unsigned long long left = 0;
  __hip_atomic_compare_exchange_strong(word, &left, nonce << 16, __ATOMIC_RELAXED, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// What the launch had counted before
__device__ __forceinline__ int count_one(unsigned long long* word, unsigned long long nonce) {
  for (;;) {
    unsigned long long now = __hip_atomic_fetch_add(word, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if ((now >> 16) == nonce) return (int)(now & 0xffff);
    // an addition to a word that was not this launch's did not count: the first to see it makes it so, and is counted with that
    ++now;
    do {
      if (__hip_atomic_compare_exchange_strong(word, &now, nonce << 16 | 1ull, __ATOMIC_RELAXED, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) return 0;
    } while ((now >> 16) != nonce);
  }
}

}  // namespace msgl
