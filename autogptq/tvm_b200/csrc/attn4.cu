// b200gptq_attn_cache: checks of the arguments and choice of the kernel.  See include/b200gptq.h.
#include <algorithm>
#include <cmath>

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

// Rows of the cache that the tokens of a sequence may see between them.
int seen_rows(const b200gptq_attn_cache_args& a) {
    return a.window ? (int)std::min<long long>(a.cache.max_seq, (long long)a.window + a.sinks + a.tokens - 1) : a.cache.max_seq;
}

// What is read back at once: `pairs` key heads of sequences, in turns of equal size.  (Turns that leave the rows in L2 until they have been multiplied are no gain: 2
// chunks of 512 behind 3500, 72 heads of 128, 311 MB at once 244 us, 4 turns of 18 heads, whose tiles fill the SMs once, 266.)
struct Turns {
    int batch, heads;                         // sequences and key heads of a turn
    int64_t bytes;                            // their rows in 16 bits, and where these are not all of the cache's the positions among them
    Turns(const b200gptq_attn_cache_args& a, long long pairs) {
        const b200gptq_cache4& c = a.cache;
        auto even = [](long long all, long long fit) {         // the smallest size with as few turns
            const long long turns = (all + fit - 1) / fit;
            return (int)((all + turns - 1) / turns);
        };
        if (pairs >= c.batch) { batch = c.batch; heads = even(c.kv_heads, pairs / c.batch); }
        else { batch = even(c.batch, pairs); heads = 1; }
        bytes = (int64_t)batch * heads * rows_of(a) + positions(a, batch);
    }
    static int64_t rows_of(const b200gptq_attn_cache_args& a) { return 4LL * seen_rows(a) * a.cache.hd; }
    static int64_t positions(const b200gptq_attn_cache_args& a, long long n) { return seen_rows(a) < a.cache.max_seq ? (8 * n + 15) / 16 * 16 : 0; }
    // As many as have 1 GB: the cache is in 4 bits because memory is short, and a second one of 16 bits beside it would not be.  (What that costs where a turn has fewer tiles
    // than there are SMs: 4 chunks of 128 tokens behind 100000 in caches of 131072, 2.1 GB at once 1280 us, three turns 2700.)
    static Turns wanted(const b200gptq_attn_cache_args& a) { return Turns(a, std::max(1LL, 1000000000LL / (long long)rows_of(a))); }
    // As many as a scratch of so many bytes has room for, which may be more or less; 0 bytes where it has for none.
    static Turns in(const b200gptq_attn_cache_args& a, size_t bytes) {
        const long long all = (long long)std::min<size_t>(bytes, (size_t)1 << 60) - positions(a, 1), pairs = all / (rows_of(a) + 8);
        Turns t(a, std::max(1LL, pairs));
        if (bytes < (size_t)t.bytes) t.bytes = 0;
        return t;
    }
};

Attn4Plan plan_of(const b200gptq_attn_cache_args& a) {
    Attn4Plan p = {};
    const long long rows = (long long)a.tokens * (a.heads / a.cache.kv_heads), sms = sm_count();
    const long long keys = seen_rows(a), pairs = (long long)a.cache.batch * a.cache.kv_heads;
    // Read back from 64 rows per key head on (as b200gptq_attn does), and otherwise where the sizes make one way much the longer, by rates in us that were measured at 128
    // dims: the rows kernel does 5900 keys of a tile of 32 rows in one, a CTA of the tcgen05 kernel 128 keys of its 128 rows, 8500 rows are read back.  32 / 8 heads of
    // 128, us, read back and not: 1 sequence behind 16000 positions, 16 tokens 137 and 56, 64 tokens 147 and 139, 200 tokens 148 and 490; behind 30000, 12
    // tokens 249 and 69; 4 sequences behind 8000, 16 tokens 95 and 96; 16 behind 30000, in three turns, 1091; 16 behind 3000, 12 tokens 82 and 111 to 149; 30 behind 300, 12 tokens 29 and 53; 8 behind 900, 16 tokens
    // 23 and 24; 64 behind 300, 8 tokens 58 and 57.
    p.read = rows >= 64;
    if (rows > 16) {
        const Turns t = Turns::wanted(a);
        const long long turns = (long long)((a.cache.batch + t.batch - 1) / t.batch) * ((a.cache.kv_heads + t.heads - 1) / t.heads);
        const double size = (double)keys * a.cache.hd / 128, direct = (double)((rows + 31) / 32) * pairs * size / 5900,
                     read = (double)(turns * (((rows + 127) / 128 * t.batch * t.heads + sms - 1) / sms)) * size / 128 + pairs * size / 8500;
        if (std::fabs(direct - read) > 10) p.read = read < direct;
    }
    if (p.read) return p;
    // A tile has 8, 16 or 32 rows.  Two CTAs of 8 rows fit an SM, one of more.
    p.tiles8 = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
    const long long units = (rows + 8 * p.tiles8 - 1) / (8 * p.tiles8) * pairs, held = sms * (p.tiles8 == 1 ? 2 : 1);
    // As many CTAs for a tile as the SMs hold, a part for each warp at least.
    while (p.split_bits < 3 && units << (p.split_bits + 1) <= held && keys >> (p.split_bits + 1) >= 128) ++p.split_bits;
    // Even runs of all keys, and a second launch whose work grows with the number of tiles, where a warp of a cluster has many parts, as the longest text has them.  Single
    // tokens, 32 / 8 heads of 128 (with 8 rows), us, runs and clusters: 1 text of 4000 12.6 and 8.2, of 16000 18.6 and 18.6, of 131000 57 and 117; 16 texts of
    // 200 to 4000 28 and 24, of 900 to 15900 62 and 78 (all of 15900: 99 and 96); 32 of 900 to 15900 111 and 149, 40 137 and 164; 64 of 200 to 4000 94 and 64, of 900 to 7900
    // 139 and 120.  16 rows: 2 texts of 16000 26 and 46, 16 of 900 to 7900 57 and 66.  32 rows: 1 of 30000 45 and 69, 8 of 900 to 7900 64 and 71, 16 of 900 to 3900 84 and 70.
    p.flat = 6 * (keys >> (p.split_bits + 7)) > 72 + units;
    p.ctas = (int)held;
    return p;
}

int64_t scratch_bytes(const b200gptq_attn_cache_args& a, const Attn4Plan& p) {
    if (p.read) return Turns::wanted(a).bytes;
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
    return scratch_bytes(*args, plan_of(*args));
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
    const Attn4Plan p = plan_of(a);
    Turns turn = Turns::in(a, workspace_bytes);
    if (workspace_bytes >= (size_t)need && turn.bytes < need) turn = Turns::wanted(a);
    if (need && (!workspace || (workspace_bytes < (size_t)need && !(p.read && turn.bytes)))) return B200GPTQ_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) & 15u) return B200GPTQ_ERR_ALIGNMENT;
    const cudaStream_t at_stream = static_cast<cudaStream_t>(stream);
    const b200gptq_cache4& c = a.cache;
    Attn4Args all = {};
    all.cache = c;
    b200gptq_attn_args& f = all.attn;
    f.q = a.q; f.out = a.out; f.pos = a.pos; f.counts = a.counts; f.status = a.status;
    std::copy(a.q_stride, a.q_stride + 3, f.q_stride);
    std::copy(a.out_stride, a.out_stride + 3, f.out_stride);
    f.dtype = c.dtype; f.batch = c.batch; f.tokens = a.tokens; f.heads = a.heads; f.kv_heads = c.kv_heads; f.hd = c.hd; f.max_seq = c.max_seq;
    f.window = a.window; f.sinks = a.sinks; f.pos_each = a.pos_each; f.scale = a.scale;
    if (!p.read) return attn4_rows_dispatch(all, static_cast<float*>(workspace), p, at_stream);
    const int group = a.heads / c.kv_heads, rows = seen_rows(a);
    const int64_t half = (int64_t)turn.batch * turn.heads * Turns::rows_of(a) / 2;
    char* const values = static_cast<char*>(workspace) + half;
    int64_t* const moved = rows < c.max_seq ? reinterpret_cast<int64_t*>(values + half) : nullptr;
    f.k_stride[2] = f.v_stride[2] = c.hd;
    f.k_stride[1] = f.v_stride[1] = (int64_t)rows * c.hd;
    f.k_stride[0] = f.v_stride[0] = turn.heads * f.k_stride[1];
    f.max_seq = rows;
    if (!attn_tiles_maps(f, false)) return B200GPTQ_ERR_TOO_LARGE;
    f.max_seq = c.max_seq;
    for (int b = 0; b < c.batch; b += turn.batch)
        for (int h = 0; h < c.kv_heads; h += turn.heads) {
            Attn4Args part = all;
            part.cache.batch = part.attn.batch = std::min(turn.batch, c.batch - b);
            part.cache.kv_heads = part.attn.kv_heads = std::min(turn.heads, c.kv_heads - h);
            part.attn.heads = part.attn.kv_heads * group;
            auto at = [&](const void* p, const int64_t (&stride)[3], int size) { return const_cast<char*>(static_cast<const char*>(p)) + (b * stride[0] + h * stride[1]) * size; };
            part.cache.k = at(c.k, c.k_stride, 1);
            part.cache.v = at(c.v, c.v_stride, 1);
            part.cache.k_scales = at(c.k_scales, c.k_scale_stride, 2);
            part.cache.v_scales = at(c.v_scales, c.v_scale_stride, 2);
            part.attn.q = static_cast<const char*>(a.q) + (b * a.q_stride[0] + (int64_t)h * group * a.q_stride[2]) * 2;
            part.attn.out = static_cast<char*>(a.out) + (b * a.out_stride[0] + (int64_t)h * group * a.out_stride[2]) * 2;
            if (a.pos_each) part.attn.pos = a.pos + b;
            if (a.counts) part.attn.counts = a.counts + b;
            st = attn4_read_back(part, workspace, values, rows, moved, at_stream);
            part.attn.k_cache = workspace;
            part.attn.v_cache = values;
            part.attn.max_seq = rows;
            part.attn.k_stride[0] = part.attn.v_stride[0] = part.attn.kv_heads * part.attn.k_stride[1];
            if (moved) { part.attn.pos = moved; part.attn.pos_each = 1; }
            if (st == B200GPTQ_OK) st = attn_tiles_dispatch(part.attn, at_stream);
            if (st != B200GPTQ_OK) return st;
        }
    return B200GPTQ_OK;
}

}  // extern "C"
