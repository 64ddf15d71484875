// The format of a cache held in 4 bits (see include/b200gptq.h): checks, and a row's words in the kernels.
#pragma once

#include "attn.cuh"

namespace b200gptq {

constexpr int kCacheMost = 1 << 29;      // of every size, so that positions and their differences are ints

inline int cache4_check(const b200gptq_cache4& c) {
    if (c.dtype != B200GPTQ_F16 && c.dtype != B200GPTQ_BF16) return B200GPTQ_ERR_SHAPE;
    if (c.batch < 1 || c.kv_heads < 1 || c.max_seq < 1 || (c.hd != 64 && c.hd != 128) || (c.group != 32 && c.group != 64)) return B200GPTQ_ERR_SHAPE;
    if (c.batch > kCacheMost || c.kv_heads > kCacheMost || c.max_seq > kCacheMost) return B200GPTQ_ERR_TOO_LARGE;
    return B200GPTQ_OK;
}
inline int cache4_check_memory(const b200gptq_cache4& c) {
    if (!c.k || !c.v || !c.k_scales || !c.v_scales) return B200GPTQ_ERR_NULL_POINTER;
    uintptr_t codes = reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v),
              constants = reinterpret_cast<uintptr_t>(c.k_scales) | reinterpret_cast<uintptr_t>(c.v_scales);
    for (int i = 0; i < 3; ++i) {
        codes |= (uintptr_t)(c.k_stride[i] | c.v_stride[i]);
        constants |= (uintptr_t)(2 * (c.k_scale_stride[i] | c.v_scale_stride[i]));
    }
    return (codes & 15u) || (constants & (uintptr_t)(4 * (c.hd / c.group) - 1)) ? B200GPTQ_ERR_ALIGNMENT : B200GPTQ_OK;
}

// Lane u of the HD / 8 that share a row has word (HD / 64) (u % 8) + u / 8 of it: dims a .. a + 3 in its fields 0, 4, 1, 5 and dims a + 32 .. a + 35 in 2, 6, 3, 7,
// with a = 64 (u / 8) + 4 (u % 8).  x[0 .. 3] are the former, x[4 .. 7] the latter.
__device__ __forceinline__ void cache4_codes(uint32_t w, unsigned (&c)[8]) {
    c[0] = w & 15u; c[2] = w >> 4 & 15u; c[4] = w >> 8 & 15u; c[6] = w >> 12 & 15u;
    c[1] = w >> 16 & 15u; c[3] = w >> 20 & 15u; c[5] = w >> 24 & 15u; c[7] = w >> 28;
}

}  // namespace b200gptq
