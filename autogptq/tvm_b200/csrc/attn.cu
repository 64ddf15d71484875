// b200gptq_attn: checks of the arguments and choice of the kernel.  See include/b200gptq.h.
#include <algorithm>
#include <cstdlib>

#include "attn.h"
#include "common.cuh"

namespace b200gptq {

bool attn_pdl_enabled() {
    static const bool on = [] {
        const char* e = std::getenv("B200GPTQ_PDL");
        return !(e && e[0] == '0');
    }();
    return on;
}

namespace {

constexpr int kMost = 1 << 29;      // of every size, so that positions and their differences are ints

int check_sizes(const b200gptq_attn_args& a) {
    if (a.dtype != B200GPTQ_F16 && a.dtype != B200GPTQ_BF16) return B200GPTQ_ERR_SHAPE;
    if (a.batch < 1 || a.tokens < 1 || a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads || (a.hd != 64 && a.hd != 128)) return B200GPTQ_ERR_SHAPE;
    if (a.max_seq < 1 || a.prefix < 0 || a.window < 0 || a.sinks < 0 || (a.window && a.prefix) || (!a.window && a.sinks)) return B200GPTQ_ERR_SHAPE;
    if (a.batch > kMost || a.tokens > kMost || a.heads > kMost || a.max_seq > kMost || a.prefix > kMost || a.window > kMost || a.sinks > kMost ||
        (long long)a.batch * a.tokens > kMost || (long long)a.batch * a.tokens * (a.heads / a.kv_heads) > kMost ||
        (long long)a.batch * a.tokens * a.heads > 0x7fffffff)
        return B200GPTQ_ERR_TOO_LARGE;
    return B200GPTQ_OK;
}

AttnPlan plan_of(const b200gptq_attn_args& a) {
    AttnPlan p = {};
    const long long rows = (long long)a.tokens * (a.heads / a.kv_heads), all = rows * a.batch, sms = sm_count();
    // 64 rows of a key head or more: the tcgen05 kernel, which has all keys of a tile in one CTA; fewer: the rows kernel, which splits them over CTAs.  Measured
    // (32 / 8 heads of 128, us, tcgen05 kernel and rows kernel).  Many sequences: 64 behind 500 positions, 32 rows 45 and 54, 60 rows 47 and 98; 8 with a
    // window of 4096, 32 rows 39 and 46, 64 rows 41 and 77, 128 rows 43 and 145.  One sequence has few tiles, and the rows kernel stays ahead up to some 256 rows: behind
    // 16384, 64 rows 120 and 80, 128 rows 131 and 73, 256 rows 132 and 132, 800 rows 133 and 478; window 4096, 64 rows 39 and 34, 128 rows 41 and 26, 256
    // rows 41 and 40, 800 rows 42 and 129.  The rule is the many sequences'; one that knows tiles and keys, and a tcgen05 kernel that splits the keys, are not there.
    if (rows >= 64 && attn_tiles_maps(a, false) && (!a.prefix || attn_tiles_maps(a, true))) {
        p.tiles = true;
        return p;
    }
    // Warps per tile of rows: as many as the SMs hold (16 each, or 8 where a tile has more than 8 rows), a block of 16 keys for each at least.
    const long long tile = rows <= 8 ? 8 : rows <= 16 ? 16 : 32, held = sms * (rows <= 8 ? 16 : 8), units = (rows + tile - 1) / tile * a.kv_heads * a.batch;
    // The prefix among each sequence's keys: `again` bytes more, from L2, or before, with two more launches.  Single tokens, us, among and before: 8 sequences,
    // 8 key heads of 128, 500 positions (14 MB) 8.0 and 12.1; 4, 32 key heads, 500 (25 MB) 9.4 and 11.6; 5, 8 key heads, 2000 (33 MB) 13.9 and 13.8; 8 of them
    // (57 MB) 14.1 and 15.0; 16 (123 MB) 22.7 and 14.8; 2, 8 key heads, 16384 (67 MB) 39.3 and 24.5; 64, 8 key heads, 500 (129 MB) 24.2 and 13.0.
    const double again = (double)(a.batch - 1) * a.kv_heads * a.prefix * a.hd * 4;
    const bool apart = a.prefix && again > 32e6;
    const long long keys = (a.window ? std::min<long long>(a.max_seq, (long long)a.window + a.sinks + a.tokens) : a.max_seq) + (apart ? 0 : a.prefix);
    long long warps = rows > 8 ? 8 : keys < 256 ? 1 : 2;
    while (warps < 8 * kAttnMaxSplit && units * warps * 2 <= held && keys >= warps * 2 * 16) warps *= 2;
    if (apart) {
        p.prefix_tiles = all > 32 && attn_tiles_maps(a, true);
        if (p.prefix_tiles) {
            const long long blocks = (a.prefix + kAttnTilesKeys - 1) / kAttnTilesKeys, ctas = (all + 255) / 256 * a.kv_heads;
            // SMs by bytes, the caches taken to be half full, a third at least: the sequences' own launch runs on the others.  32 / 8 heads of 128, us,
            // this share, every SM for the prefix, and without the third: 32 sequences, 8192 keys before 130 of 640 each, 19.6, 25.7 and 19.6; 64, 4096 before
            // 500 of 1024, 55.4, 57.5 and 45.5; 48, 12000 before 150 of 2048, 44.2, 38.0 and 70.6.  (How full the caches are is known on the device only.)
            const double share = std::max(1. / 3, a.prefix / (a.prefix + 0.5 * a.batch * a.max_seq));
            p.parts = (int)std::max<long long>(1, std::min(std::min<long long>((long long)(sms * share) / ctas, kAttnMaxParts), blocks / 4));
        } else {
            const long long ctas = (all <= 16 ? 1 : (all + 31) / 32) * a.kv_heads;
            p.parts = (int)std::max<long long>(1, std::min<long long>(std::min<long long>(2 * sms / ctas, kAttnMaxParts), a.prefix / 128));
        }
    }
    // (beside the tcgen05 kernel an SM has registers for four warps)
    const long long most = rows <= 8 && p.prefix_tiles ? 4 : 8;
    p.warps = rows <= 8 ? (int)std::min(warps, most) : 8;
    p.own = (int)std::max(1LL, std::min<long long>(warps / most, kAttnMaxSplit));
    return p;
}

size_t scratch_bytes(const b200gptq_attn_args& a, const AttnPlan& p) {
    return (size_t)(p.parts ? p.parts + 1 : 0) * a.batch * a.tokens * a.heads * (a.hd + 2) * sizeof(float);
}

}  // namespace
}  // namespace b200gptq

using namespace b200gptq;

extern "C" {

B200GPTQ_API int64_t b200gptq_attn_workspace_bytes(const b200gptq_attn_args* args) {
    if (!args) return B200GPTQ_ERR_NULL_POINTER;
    const int st = check_sizes(*args);
    return st != B200GPTQ_OK ? st : (int64_t)scratch_bytes(*args, plan_of(*args));
}

B200GPTQ_API int b200gptq_attn(const b200gptq_attn_args* args, void* workspace, size_t workspace_bytes, void* stream) {
    if (!args) return B200GPTQ_ERR_NULL_POINTER;
    const b200gptq_attn_args& a = *args;
    const int st = check_sizes(a);
    if (st != B200GPTQ_OK) return st;
    if (!a.q || !a.k_cache || !a.v_cache || !a.out || !a.pos || (a.prefix && (!a.k_prefix || !a.v_prefix))) return B200GPTQ_ERR_NULL_POINTER;
    uintptr_t bits = 0;
    for (const void* p : {a.q, a.k_cache, a.v_cache, (const void*)a.out}) bits |= reinterpret_cast<uintptr_t>(p);
    if (a.prefix) bits |= reinterpret_cast<uintptr_t>(a.k_prefix) | reinterpret_cast<uintptr_t>(a.v_prefix);
    for (int i = 0; i < 3; ++i) bits |= (uintptr_t)(2 * (a.q_stride[i] | a.out_stride[i] | a.k_stride[i] | a.v_stride[i]));
    if (a.prefix)
        for (int i = 0; i < 2; ++i) bits |= (uintptr_t)(2 * (a.k_prefix_stride[i] | a.v_prefix_stride[i]));
    if (bits & 15u) return B200GPTQ_ERR_ALIGNMENT;
    if ((reinterpret_cast<uintptr_t>(a.pos) | reinterpret_cast<uintptr_t>(a.counts)) & 7u || reinterpret_cast<uintptr_t>(a.status) & 3u) return B200GPTQ_ERR_ALIGNMENT;
    const AttnPlan p = plan_of(a);
    const size_t need = scratch_bytes(a, p);
    if (need && (!workspace || workspace_bytes < need)) return B200GPTQ_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) & 15u) return B200GPTQ_ERR_ALIGNMENT;
    const cudaStream_t at = static_cast<cudaStream_t>(stream);
    float* part = static_cast<float*>(workspace);
    if (p.tiles) return attn_tiles_dispatch(a, at);
    if (p.prefix_tiles) {
        const int before = attn_tiles_prefix(a, part, p.parts, at);
        if (before != B200GPTQ_OK) return before;
    }
    return attn_rows_dispatch(a, part, p, at);
}

}  // extern "C"
