// Device-side access to a paged key-value cache (include/kq.h: kq_kv).
#pragma once
#include "kq_device.h"
#include "kq_internal.h"

namespace kq {

// Cache element types.  bf16 is held as its bits.
struct KvF16 { typedef _Float16 T; static constexpr int id = KQ_KV_F16; };
struct KvBf16 { typedef uint16_t T; static constexpr int id = KQ_KV_BF16; };
struct KvI8 { typedef int8_t T; static constexpr int id = KQ_KV_I8; };

// fp32 -> bf16 bits, to nearest even; a NaN keeps its top bits and stays one.
__device__ __forceinline__ uint32_t bf16_rne(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
    return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}

// The positions of a request with a tree that are there: those ahead of its tree, and T more.
__device__ __forceinline__ int tree_length(const AttnArgs& a, int base) {
    return base < 0 ? 0 : min(min(base, a.max_len) + a.T, a.max_len);
}

}  // namespace kq
