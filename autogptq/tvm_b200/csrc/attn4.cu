// b200gptq_attn_cache: checks of the arguments and choice of the kernel.  See include/b200gptq.h.
#include <algorithm>

#include "attn4.h"
#include "cache4.cuh"

namespace b200gptq {
namespace {

int check_sizes(const b200gptq_attn_cache_args& a) {
    const int st = cache4_check(a.cache);
    if (st != B200GPTQ_OK) return st;
    if (a.tokens < 1 || a.heads < 1 || a.heads % a.cache.kv_heads || a.window < 0 || a.sinks < 0 || (!a.window && a.sinks)) return B200GPTQ_ERR_SHAPE;
    const long long group = a.heads / a.cache.kv_heads;
    if (a.tokens > kCacheMost || a.heads > kCacheMost || a.window > kCacheMost || a.sinks > kCacheMost || (long long)a.cache.batch * a.tokens > kCacheMost ||
        (long long)a.cache.batch * a.tokens * group > kCacheMost || (long long)a.cache.batch * a.tokens * a.heads > 0x7fffffff ||
        (long long)a.cache.batch * a.cache.kv_heads > kCacheMost)
        return B200GPTQ_ERR_TOO_LARGE;
    return B200GPTQ_OK;
}

Attn4Plan plan_of(const b200gptq_attn_cache_args& a) {
    Attn4Plan p = {};
    const long long rows = (long long)a.tokens * (a.heads / a.cache.kv_heads), sms = sm_count();
    if (rows >= 64) {
        p.read = true;
        return p;
    }
    p.tiles8 = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
    const long long units = (rows + 8 * p.tiles8 - 1) / (8 * p.tiles8) * a.cache.kv_heads * a.cache.batch, held = sms * (p.tiles8 == 1 ? 2 : 1);
    const long long keys = a.window ? std::min<long long>(a.cache.max_seq, (long long)a.window + a.sinks + a.tokens) : a.cache.max_seq;
    while (p.split_bits < 3 && units << (p.split_bits + 1) <= held && keys >> (p.split_bits + 1) >= 128) ++p.split_bits;
    p.flat = keys > 2048;
    p.ctas = (int)held;
    return p;
}

int64_t scratch_bytes(const b200gptq_attn_cache_args& a, const Attn4Plan& p) {
    if (p.read) return (int64_t)a.cache.batch * a.cache.kv_heads * a.cache.max_seq * a.cache.hd * 4;
    return p.flat ? 2LL * kAttn4Warps * p.ctas * 8 * p.tiles8 * (a.cache.hd + 2) * (int)sizeof(float) : 0;
}

}  // namespace
}  // namespace b200gptq

using namespace b200gptq;

extern "C" {

B200GPTQ_API int64_t b200gptq_attn_cache_workspace_bytes(const b200gptq_attn_cache_args* args) {
    if (!args) return B200GPTQ_ERR_NULL_POINTER;
    const int st = check_sizes(*args);
    if (st != B200GPTQ_OK) return st;
    const double most = 4.0 * args->cache.batch * args->cache.kv_heads * args->cache.max_seq * args->cache.hd;
    const Attn4Plan p = plan_of(*args);
    return p.read && most > 9e18 ? B200GPTQ_ERR_TOO_LARGE : scratch_bytes(*args, p);
}

B200GPTQ_API int b200gptq_attn_cache(const b200gptq_attn_cache_args* args, void* workspace, size_t workspace_bytes, void* stream) {
    const int64_t need = b200gptq_attn_cache_workspace_bytes(args);
    if (need < 0) return (int)need;
    const b200gptq_attn_cache_args& a = *args;
    if (!a.q || !a.out || !a.pos) return B200GPTQ_ERR_NULL_POINTER;
    int st = cache4_check_memory(a.cache);
    if (st != B200GPTQ_OK) return st;
    uintptr_t bits = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out);
    for (int i = 0; i < 3; ++i) bits |= (uintptr_t)(2 * (a.q_stride[i] | a.out_stride[i]));
    if (bits & 15u) return B200GPTQ_ERR_ALIGNMENT;
    // (the rows kernel multiplies rows and their steps, in bytes, in 32 bits each)
    for (int64_t step : {a.cache.k_stride[2], a.cache.v_stride[2], 2 * a.cache.k_scale_stride[2], 2 * a.cache.v_scale_stride[2]})
        if (step < 0 || step > 0xffffffffLL) return B200GPTQ_ERR_TOO_LARGE;
    if ((reinterpret_cast<uintptr_t>(a.pos) | reinterpret_cast<uintptr_t>(a.counts)) & 7u || reinterpret_cast<uintptr_t>(a.status) & 3u) return B200GPTQ_ERR_ALIGNMENT;
    if (need && (!workspace || workspace_bytes < (size_t)need)) return B200GPTQ_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) & 15u) return B200GPTQ_ERR_ALIGNMENT;
    const Attn4Plan p = plan_of(a);
    const cudaStream_t at = static_cast<cudaStream_t>(stream);
    const b200gptq_cache4& c = a.cache;
    Attn4Args all = {};
    all.cache = c;
    b200gptq_attn_args& f = all.attn;
    f.q = a.q; f.out = a.out; f.pos = a.pos; f.counts = a.counts; f.status = a.status;
    std::copy(a.q_stride, a.q_stride + 3, f.q_stride);
    std::copy(a.out_stride, a.out_stride + 3, f.out_stride);
    f.dtype = c.dtype; f.batch = c.batch; f.tokens = a.tokens; f.heads = a.heads; f.kv_heads = c.kv_heads; f.hd = c.hd; f.max_seq = c.max_seq;
    f.window = a.window; f.sinks = a.sinks; f.pos_each = a.pos_each; f.scale = a.scale;
    if (!p.read) return attn4_rows_dispatch(all, static_cast<float*>(workspace), p, at);
    f.k_cache = workspace;
    f.v_cache = static_cast<char*>(workspace) + need / 2;
    const int64_t stride[3] = {(int64_t)c.kv_heads * c.max_seq * c.hd, (int64_t)c.max_seq * c.hd, c.hd};
    std::copy(stride, stride + 3, f.k_stride);
    std::copy(stride, stride + 3, f.v_stride);
    if (!attn_tiles_maps(f, false)) return B200GPTQ_ERR_TOO_LARGE;
    st = attn4_read_back(all, workspace, static_cast<char*>(workspace) + need / 2, at);
    return st != B200GPTQ_OK ? st : attn_tiles_dispatch(f, at);
}

}  // extern "C"
