// b200gptq_attn_cache for few query rows per key head: the single tokens of a decode step (and short runs of them) over a cache held in 4 bits.
//
//   K = zK + sK cK,  V = zV + sV cV  (zero, scale and code by row and group of dims),   S = Q K^T,  w = softmax(scale S),  O = w V
//
// A row of the cache is 68 to 80 bytes for 128 dims and has to be multiplied by up to 8, 16 or 32 rows of Q, so bytes and instructions bound it alike, and the codes go
// to the tensor cores as they are: a field of four bits that is masked in place, at bits 0 .. 3 or 4 .. 7 of 16, is the fp16 number c 2^-24 or 16 c 2^-24 (subnormal,
// exact), so eight codes cost a shift and four masks.  Scales and zeros are applied beside the products:
//   S(key, row) = sum over groups of  sK (q . cK) + zK (sum of q)      one product chain per group, then two fp32 FMAs
//   O(dim, row) = sum over keys of  (w sV) cV + w zV                   w sV is what is rounded to fp16; w zV is summed in fp32, per group
// Q is scaled by a power of two per row (to below 2^15, exact for what is above 2^-38 of the row's largest; so bf16 queries are exact in fp16), w sV by one per
// warp that follows the largest scale seen, so neither leaves fp16's range.
//
// Every warp takes blocks of 16 keys on its own, through a ring of cp.async stages in shared memory.  Keys are the 16 of m16n8k16, rows the 8: 8 bytes (128
// dims: 16) of a key are the operand of S as they lie, two keys' words paired by byte permutations that of O (include/b200gptq.h has the order of the codes).
// Rows are only rescaled when a score is more than 2^8 above the maximum in use (no weight is above 2^8; fp32 sums).
//
// FLAT: the blocks of all sequences and key heads lie one behind the other, and each CTA takes an even run of them, whatever the texts' lengths, which are known
// on the device only.  Where a run ends inside a (sequence, key head) the sums go to scratch, and a second launch adds them up in order.
// Otherwise a cluster of 1 to 8 CTAs shares a (sequence, key head), and they add up through distributed shared memory.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "attn4.h"
#include "cache4.cuh"

namespace b200gptq {
namespace {

constexpr int kBlock = 16, kWarps = 8, kThreads = kWarps * 32, kStages = 4;
constexpr float kGrow = 8.f;             // log2 of what a score may be above the maximum in use
constexpr unsigned kLow = 0x000f000fu, kHigh = 0x00f000f0u;

__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {      // of an 8 x 8 matrix of 16-bit values, a pair of a row per lane
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void st_cluster(const float* local, int rank, float v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(v) : "memory");
}
template <int N> __device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
template <int N> struct Words { uint32_t w[N]; };
template <int N> __device__ __forceinline__ Words<N> lds(uint32_t at) {
    Words<N> r;
    if constexpr (N == 4) asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]) : "r"(at));
    else if constexpr (N == 2) asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "r"(at));
    else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r.w[0]) : "r"(at));
    return r;
}

// One block of 16 keys in shared memory, in bytes: codes of K as they lie; codes of V, 16 bytes at a time, where each 128 bytes (2 or 4 rows) are permuted so that
// the lanes of a load (rows 2c) meet no bank twice; constants of K and of V.
template <int HD, int GS> struct Stage {
    static constexpr int row = HD / 2, groups = HD / GS, constants = 4 * groups, k = 0, v = kBlock * row, kc = 2 * kBlock * row, vc = kc + kBlock * constants,
                         total = vc + kBlock * constants;
    __device__ static __forceinline__ int v_at(int r, int byte) {
        const int line = r * row / 128, chunk = (r * row % 128 + byte) / 16;
        return v + line * 128 + ((chunk ^ (2 * (line & (HD == 128 ? 3 : 1)))) * 16 + byte % 16);
    }
};

// Shared memory, in floats: the ring [warp][stage], over which the warps' sums [warp][row][HD + 4] come to lie; their maxima and denominators; the slices that the
// CTAs of the cluster push [split][row][HD / splits] with maxima and denominators; a flag per row; the rows' places (q, out); sums of q by group and row, factor of a
// row; the operand made of Q.
template <int HD, int GS, int NT> struct Lay {
    static constexpr int R = 8 * NT, LD = HD + 4, ring = kWarps * kStages * Stage<HD, GS>::total / 4, sums = kWarps * R * LD, ml = ring > sums ? ring : sums,
                         slice = ml + 2 * kWarps * R, slice_ml = slice + R * HD, flags = slice_ml + 2 * kAttn4MaxSplit * R, places = flags + R, qsum = places + 4 * R,
                         factor = qsum + 4 * R, where = factor + R, q = where + 8, total = q + NT * (HD / 32) * 32 * 4;
    static_assert(places % 2 == 0 && q % 4 == 0 && slice % 4 == 0, "");
};

// Blocks of a sequence: those that its tokens see between them; one at least where there are tokens, since their rows get zeros when they see nothing.
struct Span { AttnRange range; int p0, count, n_s, nb; };
__device__ __forceinline__ Span span_of(const Attn4Args& a, int b) {
    Span s;
    s.p0 = attn_pos(a.attn, b);
    s.count = attn_count(a.attn, b);
    s.range = attn_range(s.p0, s.p0 + max(s.count, 1) - 1, a.attn.window ? a.attn.window : 1 << 30, a.attn.sinks, a.attn.max_seq);
    s.n_s = (s.range.s_end + kBlock - 1) / kBlock;
    s.nb = s.count ? max(1, s.n_s + (s.range.w_end - s.range.w_start + kBlock - 1) / kBlock) : 0;
    return s;
}
// Of the CTAs of a FLAT launch, number i begins with block total * i / ctas.
__device__ __forceinline__ long long flat_begin(long long total, int i, int ctas) { return total * i / ctas; }

// The sequence in which block `at` of the flat order lies, and the block with which that sequence begins; the total where at < 0.  All threads of a CTA
// call it; `where` has room for 8 floats.
struct Found { int b; long long begin, total; };
__device__ Found flat_find(const Attn4Args& a, int units, int cta, int ctas, long long offset, long long* where) {
    __shared__ long long scan[kWarps + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Found f = {0, 0, 0};
    for (int b = threadIdx.x; b < a.attn.batch; b += kThreads) f.total += (long long)span_of(a, b).nb * units;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) f.total += __shfl_xor_sync(0xffffffffu, f.total, o);
    if (lane == 0) scan[warp] = f.total;
    __syncthreads();
    f.total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) f.total += scan[w];
    __syncthreads();
    const long long at = flat_begin(f.total, cta, ctas) + offset;
    if (threadIdx.x == 0) { where[0] = -1; where[1] = 0; }
    long long before = 0;
    for (int b0 = 0; b0 < a.attn.batch; b0 += kThreads) {
        const int b = b0 + threadIdx.x;
        const long long mine = b < a.attn.batch ? (long long)span_of(a, b).nb * units : 0;
        long long sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        if (lane == 31) scan[warp] = sum;
        __syncthreads();
        long long lower = before, all = before;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) lower += scan[w];
            all += scan[w];
        }
        if (at >= lower + sum - mine && at < lower + sum) { where[0] = b; where[1] = lower + sum - mine; }
        before = all;
        __syncthreads();
        if (before > at) break;
    }
    f.b = (int)where[0];
    f.begin = where[1];
    return f;
}

// The row once more by one warp, a few keys at a time and only those that it sees: see attn_row_again in attn.cuh, of which this is the plain form (all dims of
// the row that are not finite are done again).  A lane owns a word of every key, eight dims; the warp has 2 or 4 keys at a time.
template <typename T, int HD, int GS>
__device__ __noinline__ void attn4_row_again(const Attn4Args& a, int b, int t, int head, int p, int d0, int d1) {
    constexpr int LANES = HD / 8, KEYS = 32 / LANES, NG = HD / GS;
    const int lane = threadIdx.x & 31, u = lane % LANES, g = u & 7, h = u >> 3, kh = head / (a.attn.heads / a.attn.kv_heads), d = 64 * h + 4 * g;
    const int window = a.attn.window ? a.attn.window : 1 << 30;
    const b200gptq_cache4& c = a.cache;
    T* out = static_cast<T*>(a.attn.out) + b * a.attn.out_stride[0] + t * a.attn.out_stride[1] + head * a.attn.out_stride[2];
    const T* q = static_cast<const T*>(a.attn.q) + b * a.attn.q_stride[0] + t * a.attn.q_stride[1] + head * a.attn.q_stride[2];
    const uint8_t *k = static_cast<const uint8_t*>(c.k) + b * c.k_stride[0] + kh * c.k_stride[1], *v = static_cast<const uint8_t*>(c.v) + b * c.v_stride[0] + kh * c.v_stride[1];
    const T *ks = static_cast<const T*>(c.k_scales) + b * c.k_scale_stride[0] + kh * c.k_scale_stride[1],
            *vs = static_cast<const T*>(c.v_scales) + b * c.v_scale_stride[0] + kh * c.v_scale_stride[1];
    const int word = (HD / 64) * g + h, ga = h * NG / (HD / 64), gb = GS == 64 ? ga : 2 * h + 1;
    auto row = [&](const uint8_t* codes, const T* constants, float (&x)[8]) {
        unsigned code[8];
        cache4_codes(reinterpret_cast<const uint32_t*>(codes)[word], code);
        const float2 fa = Half<T>::unpack(reinterpret_cast<const uint32_t*>(constants)[ga]), fb = Half<T>::unpack(reinterpret_cast<const uint32_t*>(constants)[gb]);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = e < 4 ? fmaf((float)code[e], fa.x, fa.y) : fmaf((float)code[e], fb.x, fb.y);
    };
    float qf[8], acc[8], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) { qf[e] = Half<T>::wide(q[d + e % 4 + 32 * (e / 4)]) * a.attn.scale * kLog2e; acc[e] = 0.f; }
    const AttnRange r = attn_range(p, p, window, a.attn.sinks, a.attn.max_seq);
    auto keys = [&](int begin, int end) {
        for (int j0 = begin; j0 < end; j0 += KEYS) {
            const int j = j0 + lane / LANES;
            float x[8], y[8], s = 0.f;
            row(k + min(j, end - 1) * c.k_stride[2], ks + min(j, end - 1) * c.k_scale_stride[2], x);
            row(v + min(j, end - 1) * c.v_stride[2], vs + min(j, end - 1) * c.v_scale_stride[2], y);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(qf[e], x[e], s);
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (j >= end) continue;               // (whole groups of lanes; the shuffles above are before it, those below after the loop)
            const float up = fmaxf(m, s), safe = up == -INFINITY ? 0.f : up, corr = exp2_fast(m - safe), w = exp2_fast(s - safe);
            m = up;
            l = l * corr + w;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, y[e], acc[e] * corr);
        }
        __syncwarp();
    };
    keys(0, r.s_end);
    keys(r.w_start, r.w_end);
    float top = m;
#pragma unroll
    for (int o = LANES; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float corr = exp2_fast(m - (top == -INFINITY ? 0.f : top));
    l *= corr;
#pragma unroll
    for (int o = LANES; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        acc[e] *= corr;
#pragma unroll
        for (int o = LANES; o < 32; o <<= 1) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], o);
        const int at = d + e % 4 + 32 * (e / 4);
        if (lane < LANES && at >= d0 && at < d1 && !isfinite(Half<T>::wide(out[at]))) out[at] = Half<T>::round(l != 0.f ? acc[e] / l : 0.f);
    }
}

template <typename T, int HD, int GS, int NT, bool FLAT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1)
attn4_rows_kernel(const __grid_constant__ Attn4Args a, float* __restrict__ part, int split_bits, int row_tiles, int G, const __grid_constant__ Attn4Divisors by) {
    using L = Lay<HD, GS, NT>;
    using St = Stage<HD, GS>;
    constexpr int R = 8 * NT, NG = HD / GS, HH = HD / 64, KW = HD / 32, VW = HD / 64;      // words of a key per lane, for S and for O
    extern __shared__ __align__(16) float sm[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int window = a.attn.window ? a.attn.window : 1 << 30, splits = FLAT ? 1 : 1 << split_bits, units = a.attn.kv_heads * row_tiles;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(sm) + warp * kStages * St::total;
    auto token_of = [&](int idx) { return (int)over((unsigned)idx, by.group); };       // of row idx
    if (!FLAT && splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");

    const unsigned per_unit = blockIdx.x >> split_bits;
    const int split = FLAT ? 0 : blockIdx.x - (per_unit << split_bits);
    int b = 0, tile = 0, kh = 0;
    long long cur = 0, begin = 0, hi = 0, seq = 0;             // FLAT: the next block, the first one and the end of the run, the sequence's first
    if constexpr (FLAT) {
        const Found f = flat_find(a, units, blockIdx.x, gridDim.x, 0, reinterpret_cast<long long*>(sm + L::where));
        begin = cur = flat_begin(f.total, blockIdx.x, gridDim.x);
        hi = flat_begin(f.total, blockIdx.x + 1, gridDim.x);
        b = f.b;
        seq = f.begin;
        if (cur >= hi) return;
    } else {
        const unsigned unit = over(per_unit, by.row_tiles);
        tile = per_unit - unit * row_tiles;
        b = over(unit, by.kv_heads);
        kh = unit - b * a.attn.kv_heads;
    }
    Span span = span_of(a, b);
    while (true) {
        // ---- what is to be done: blocks first .. last of a (sequence, key head, tile of rows) ----
        int first, last, n_unit = 0;
        bool complete = true;
        if constexpr (FLAT) {
            n_unit = (int)((cur - seq) / span.nb);
            first = (int)(cur - seq - (long long)n_unit * span.nb);
            last = (int)min((long long)span.nb, first + (hi - cur));
            kh = n_unit / row_tiles;
            tile = n_unit - kh * row_tiles;
            complete = first == 0 && last == span.nb;
        } else {
            first = (int)((long long)span.nb * split >> split_bits);
            last = (int)((long long)span.nb * (split + 1) >> split_bits);
        }
        const int row0 = tile * R, nrows = min(R, span.count * G - row0);
        if (nrows <= 0) {                         // padding
            if constexpr (!FLAT) return;          // (every CTA of the cluster)
        } else {
        const AttnRange range = span.range;
        const int p_lo = span.p0 + token_of(row0), p_hi = span.p0 + token_of(row0 + nrows - 1);
        const uint8_t *kb = static_cast<const uint8_t*>(a.cache.k) + b * a.cache.k_stride[0] + kh * a.cache.k_stride[1],
                      *vb = static_cast<const uint8_t*>(a.cache.v) + b * a.cache.v_stride[0] + kh * a.cache.v_stride[1];
        const T *kcb = static_cast<const T*>(a.cache.k_scales) + b * a.cache.k_scale_stride[0] + kh * a.cache.k_scale_stride[1],
                *vcb = static_cast<const T*>(a.cache.v_scales) + b * a.cache.v_scale_stride[0] + kh * a.cache.v_scale_stride[1];
        auto block = [&](int i, int& j0, int& end) {
            j0 = i < span.n_s ? kBlock * i : range.w_start + kBlock * (i - span.n_s);
            end = i < span.n_s ? range.s_end : range.w_end;
        };
        // (rows behind the end of the range: its last row again, or row 0 of a range that is empty, with weight zero)
        auto fetch = [&](int i, int stage) {
            if (i < last) {
                int j0, end;
                block(i, j0, end);
                const int top = max(min(end, a.attn.max_seq) - 1, 0);       // (an empty range may lie behind the cache)
                const uint32_t at = ring + stage * St::total;
                constexpr int CHUNKS = St::row / 16;
#pragma unroll
                for (int x = 0; x < kBlock * CHUNKS / 32; ++x) {
                    const int r = (lane + 32 * x) / CHUNKS, byte = (lane + 32 * x) % CHUNKS * 16;
                    const long long j = min(j0 + r, top);
                    copy_async<16>(at + St::k + r * St::row + byte, kb + j * a.cache.k_stride[2] + byte);
                    copy_async<16>(at + St::v_at(r, byte), vb + j * a.cache.v_stride[2] + byte);
                }
                const long long j = min(j0 + (lane & 15), top);
                const T* from = lane < 16 ? kcb + j * a.cache.k_scale_stride[2] : vcb + j * a.cache.v_scale_stride[2];
                copy_async<St::constants>(at + (lane < 16 ? St::kc : St::vc) + (lane & 15) * St::constants, from);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        int i = first + warp;
#pragma unroll
        for (int s = 0; s < kStages - 1; ++s) fetch(i + s * kWarps, s);
        // ---- the rows' places, the operand made of Q, its sums ----
        long long* places = reinterpret_cast<long long*>(sm + L::places);
        if (threadIdx.x < R) {
            const int idx = row0 + min((int)threadIdx.x, nrows - 1), t = token_of(idx), head = kh * G + idx - t * G;
            places[threadIdx.x] = b * a.attn.q_stride[0] + t * a.attn.q_stride[1] + head * a.attn.q_stride[2];
            places[R + threadIdx.x] = b * a.attn.out_stride[0] + t * a.attn.out_stride[1] + head * a.attn.out_stride[2];
            reinterpret_cast<int*>(sm + L::flags)[threadIdx.x] = 0;
        }
        __syncthreads();
        // eight dims (32 y + 8 c ..) of row r per thread: HD / 8 threads of a warp share a row
        for (int x = threadIdx.x; x < R * HD / 8; x += kThreads) {
            const int r = x / (HD / 8), e8 = x % (HD / 8), y = e8 >> 2;
            const uint4 raw = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.attn.q) + places[r] + 8 * e8));
            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
            float f[8], most = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 two = Half<T>::unpack(w[e]);
                f[2 * e] = two.x; f[2 * e + 1] = two.y;
                most = fmaxf(most, fmaxf(fabsf(two.x), fabsf(two.y)));
            }
#pragma unroll
            for (int o = 1; o < HD / 8; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            int up = 15;
            if (most > 0.f && most < INFINITY) frexpf(most, &up);
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f[e] = ldexpf(f[e], 15 - up);
                sum += f[e];
            }
#pragma unroll
            for (int o = 1; o < GS / 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (e8 % (GS / 8) == 0) sm[L::qsum + (e8 / (GS / 8)) * R + r] = ldexpf(sum, -24);
            if (e8 == 0) sm[L::factor + r] = ldexpf(a.attn.scale * kLog2e, 24 + up - 15);
            *reinterpret_cast<uint4*>(sm + L::q + (((r >> 3) * KW + y) * 32 + (r & 7) * 4 + (e8 & 3)) * 4) =
                make_uint4(Half<__half>::pack(f[0], f[1]), Half<__half>::pack(f[2] * 0.0625f, f[3] * 0.0625f), Half<__half>::pack(f[4], f[5]),
                           Half<__half>::pack(f[6] * 0.0625f, f[7] * 0.0625f));
        }
        __syncthreads();
        // Rows of the lane: 8 t + 2 c and + 1
        float acc[NT][4 * HH][4], zacc[NT][2][NG], m[NT][2], l[NT][2], factor[NT][2], limit = 0.f, inverse = 0.f;
        int pr[NT][2];
        uint4 qr[NT <= 2 ? NT : 1][KW];
        float qs[NT <= 2 ? NT : 1][NG][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int n = 0; n < 4 * HH; ++n) acc[t][n][0] = acc[t][n][1] = acc[t][n][2] = acc[t][n][3] = 0.f;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                m[t][r] = -INFINITY; l[t][r] = 0.f;
                factor[t][r] = sm[L::factor + 8 * t + 2 * c + r];
                pr[t][r] = span.p0 + token_of(row0 + min(8 * t + 2 * c + r, nrows - 1));
#pragma unroll
                for (int n = 0; n < NG; ++n) {
                    zacc[t][r][n] = 0.f;
                    if constexpr (NT <= 2) qs[t][n][r] = sm[L::qsum + n * R + 8 * t + 2 * c + r];
                }
            }
            if constexpr (NT <= 2)
#pragma unroll
                for (int y = 0; y < KW; ++y) qr[t][y] = *reinterpret_cast<const uint4*>(sm + L::q + ((t * KW + y) * 32 + lane) * 4);
        }
        for (int stage = 0; i < last; i += kWarps) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            __syncwarp();
            fetch(i + (kStages - 1) * kWarps, stage == 0 ? kStages - 1 : stage - 1);
            const uint32_t at = ring + stage * St::total;
            stage = stage + 1 == kStages ? 0 : stage + 1;
            int j0, end;
            block(i, j0, end);
            // every row of the tile sees the whole block
            const bool whole = j0 + kBlock <= end && j0 + kBlock - 1 <= p_lo && (j0 > p_hi - window || j0 + kBlock <= a.attn.sinks);
            // ---- S: keys g (0, 1) and g + 8 (2, 3), rows 2 c and 2 c + 1 ----
            float s[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
            {
                const Words<KW> k0 = lds<KW>(at + St::k + g * St::row + 4 * KW * c), k1 = lds<KW>(at + St::k + (g + 8) * St::row + 4 * KW * c);
                const Words<NG> c0 = lds<NG>(at + St::kc + g * St::constants), c1 = lds<NG>(at + St::kc + (g + 8) * St::constants);
                float d[NT][4];
#pragma unroll
                for (int y = 0; y < KW; ++y) {        // 32 dims
                    if (GS == 32 || !(y & 1)) {
#pragma unroll
                        for (int t = 0; t < NT; ++t) d[t][0] = d[t][1] = d[t][2] = d[t][3] = 0.f;
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t w0 = k0.w[HH * x + (y >> 1)] >> (y & 1 ? 8 : 0), w1 = k1.w[HH * x + (y >> 1)] >> (y & 1 ? 8 : 0);
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            uint32_t b0, b1;
                            if constexpr (NT <= 2) {
                                b0 = x ? qr[t][y].z : qr[t][y].x;
                                b1 = x ? qr[t][y].w : qr[t][y].y;
                            } else {
                                const uint2 two = *reinterpret_cast<const uint2*>(sm + L::q + ((t * KW + y) * 32 + lane) * 4 + 2 * x);
                                b0 = two.x;
                                b1 = two.y;
                            }
                            mma16(d[t], w0 & kLow, w1 & kLow, w0 & kHigh, w1 & kHigh, b0, b1);
                        }
                    }
                    if (GS == 32 || (y & 1)) {
                        const int n = GS == 32 ? y : y >> 1;
                        const float2 f0 = Half<T>::unpack(c0.w[n]), f1 = Half<T>::unpack(c1.w[n]);       // (scale, zero)
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                float sum;
                                if constexpr (NT <= 2) sum = qs[t][n][e & 1];
                                else sum = sm[L::qsum + n * R + 8 * t + 2 * c + (e & 1)];
                                s[t][e] = fmaf(e < 2 ? f0.x : f1.x, d[t][e], fmaf(e < 2 ? f0.y : f1.y, sum, s[t][e]));
                            }
                    }
                }
            }
            // ---- constants of V; those of keys behind the end count for nothing ----
            const Words<NG> u0 = lds<NG>(at + St::vc + g * St::constants), u1 = lds<NG>(at + St::vc + (g + 8) * St::constants);
            float sv[2][NG], zv[2][NG], widest = 0.f;
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                const float2 f0 = Half<T>::unpack(u0.w[n]), f1 = Half<T>::unpack(u1.w[n]);
                sv[0][n] = f0.x; zv[0][n] = f0.y; sv[1][n] = f1.x; zv[1][n] = f1.y;
                if (!whole) {
                    if (j0 + g >= end) sv[0][n] = zv[0][n] = 0.f;
                    if (j0 + g + 8 >= end) sv[1][n] = zv[1][n] = 0.f;
                }
                widest = fmaxf(widest, fmaxf(sv[0][n], sv[1][n]));
            }
            bool grow = widest > 8.f * limit;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[t][e] *= factor[t][e & 1];
                    if (!whole) {
                        const int j = j0 + g + 8 * (e >> 1);
                        s[t][e] = j < end && attn_sees(pr[t][e & 1], j, window, a.attn.sinks) ? s[t][e] : -INFINITY;
                    }
                }
                grow = grow || fmaxf(s[t][0], s[t][2]) - m[t][0] > kGrow || fmaxf(s[t][1], s[t][3]) - m[t][1] > kGrow;
            }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) widest = fmaxf(widest, __shfl_xor_sync(0xffffffffu, widest, o));
                float shrink = 1.f;
                if (widest > limit) {                 // the power of two at or below it
                    const float now = fminf(fmaxf(__uint_as_float(__float_as_uint(widest) & 0x7f800000u), 0x1p-100f), 0x1p126f);
                    shrink = limit == 0.f ? 0.f : limit / now;
                    limit = now;
                    inverse = 1.f / now;
                }
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float up = fmaxf(fmaxf(s[t][r], s[t][2 + r]), m[t][r]);
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, o));
                        const float corr = up == -INFINITY ? 1.f : exp2_fast(m[t][r] - up), both = corr * shrink;
                        m[t][r] = up;
                        l[t][r] *= corr;
#pragma unroll
                        for (int n = 0; n < NG; ++n) zacc[t][r][n] *= corr;
#pragma unroll
                        for (int n = 0; n < 4 * HH; ++n) { acc[t][n][r] *= both; acc[t][n][2 + r] *= both; }
                    }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float safe = m[t][r] == -INFINITY ? 0.f : m[t][r];
                    s[t][r] = exp2_fast(s[t][r] - safe);
                    s[t][2 + r] = exp2_fast(s[t][2 + r] - safe);
                    l[t][r] += s[t][r] + s[t][2 + r];
#pragma unroll
                    for (int n = 0; n < NG; ++n) zacc[t][r][n] = fmaf(s[t][r], zv[0][n], fmaf(s[t][2 + r], zv[1][n], zacc[t][r][n]));
                }
            // ---- O: codes of keys 2c, 2c + 1 and 2c + 8, 2c + 9 in pairs ----
            Words<VW> v[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) v[n] = lds<VW>(at + St::v_at(2 * c + (n & 1) + 4 * (n & 2), 4 * VW * g));
#pragma unroll
            for (int h = 0; h < HH; ++h) {
                const uint32_t x[2][2] = {{__byte_perm(v[0].w[h], v[1].w[h], 0x5410u), __byte_perm(v[2].w[h], v[3].w[h], 0x5410u)},
                                          {__byte_perm(v[0].w[h], v[1].w[h], 0x7632u), __byte_perm(v[2].w[h], v[3].w[h], 0x7632u)}};
                uint32_t b0[NT], b1[NT];
#pragma unroll
                for (int y = 0; y < 2; ++y) {         // dims 64 h + 32 y + 4 g + {0, 2} and {1, 3}
                    if (GS == 32 || y == 0) {
                        const int n = GS == 32 ? 2 * h + y : h;
                        const float w0 = sv[0][n] * inverse, w1 = sv[1][n] * inverse;
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            b0[t] = transposed(Half<__half>::pack(s[t][0] * w0, s[t][1] * w0));
                            b1[t] = transposed(Half<__half>::pack(s[t][2] * w1, s[t][3] * w1));
                        }
                    }
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const uint32_t k01 = x[z][0] >> (8 * y), k89 = x[z][1] >> (8 * y);
#pragma unroll
                        for (int t = 0; t < NT; ++t) mma16(acc[t][4 * h + 2 * y + z], k01 & kLow, k01 & kHigh, k89 & kLow, k89 & kHigh, b0[t], b1[t]);
                    }
                }
            }
        }
        // ---- the warps' sums: rows, four adjacent dims each ----
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();                          // (the ring has been read)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = 8 * t + 2 * c + r;
                float sum = l[t][r];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
                for (int n = 0; n < NG; ++n)
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) zacc[t][r][n] += __shfl_xor_sync(0xffffffffu, zacc[t][r][n], o);
                if (row < nrows) {
                    if (g == 0) { sm[L::ml + 2 * (warp * R + row)] = m[t][r]; sm[L::ml + 2 * (warp * R + row) + 1] = sum; }
#pragma unroll
                    for (int h = 0; h < HH; ++h)
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const float z = zacc[t][r][GS == 32 ? 2 * h + y : h];
                            const float *even = acc[t][4 * h + 2 * y], *odd = acc[t][4 * h + 2 * y + 1];
                            // (fields at bits 4 .. 7 were 16 times as large)
                            *reinterpret_cast<float4*>(sm + (warp * R + row) * L::LD + 64 * h + 32 * y + 4 * g) =
                                make_float4(fmaf(even[r] * 0x1p24f, limit, z), fmaf(odd[r] * 0x1p24f, limit, z), fmaf(even[2 + r] * 0x1p20f, limit, z), fmaf(odd[2 + r] * 0x1p20f, limit, z));
                        }
                }
            }
        __syncthreads();
        if (!FLAT && splits > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");      // (all CTAs of the cluster run)
        // ---- the CTA's sums: to the scratch or out, or slice by slice to the CTAs of the cluster ----
        const int slice = FLAT ? HD : HD >> split_bits;
        constexpr int HD_BITS = HD == 128 ? 7 : 6;
        int* flags = reinterpret_cast<int*>(sm + L::flags);
        float* run = FLAT ? part + (2LL * blockIdx.x + (cur != begin)) * R * (HD + 2) : nullptr;
        for (int x = threadIdx.x; x < nrows * (HD / 4); x += kThreads) {
            const int row = x / (HD / 4), d = x % (HD / 4) * 4;
            float cm = -INFINITY, cl = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) cm = fmaxf(cm, sm[L::ml + 2 * (w * R + row)]);
            const float safe = cm == -INFINITY ? 0.f : cm;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float e = exp2_fast(sm[L::ml + 2 * (w * R + row)] - safe);
                const float4 f = *reinterpret_cast<const float4*>(sm + (w * R + row) * L::LD + d);
                cl += sm[L::ml + 2 * (w * R + row) + 1] * e;
                o.x += f.x * e; o.y += f.y * e; o.z += f.z * e; o.w += f.w * e;
            }
            if (FLAT && !complete) {
                *reinterpret_cast<float4*>(run + row * HD + d) = o;
                if (d == 0) *reinterpret_cast<float2*>(run + R * HD + 2 * row) = make_float2(cm, cl);
            } else if (FLAT || splits == 1) {
                const bool none = cl == 0.f;
                float f[4] = {none ? 0.f : o.x / cl, none ? 0.f : o.y / cl, none ? 0.f : o.z / cl, none ? 0.f : o.w / cl};
                if (settle<T>(f) && isfinite(cl)) flags[row] = 1;
                *reinterpret_cast<uint2*>(static_cast<T*>(a.attn.out) + places[R + row] + d) = make_uint2(Half<T>::pack(f[0], f[1]), Half<T>::pack(f[2], f[3]));
            } else {
                const float f[4] = {o.x, o.y, o.z, o.w};
                const int to = d >> (HD_BITS - split_bits);        // (a slice has 8 dims at least)
#pragma unroll
                for (int e = 0; e < 4; ++e) st_cluster(sm + L::slice + (split * R + row) * slice + d + e - to * slice, to, f[e]);
                if (d - to * slice == 0) {
                    st_cluster(sm + L::slice_ml + 2 * (split * R + row), to, cm);
                    st_cluster(sm + L::slice_ml + 2 * (split * R + row) + 1, to, cl);
                }
            }
        }
        if (!FLAT && splits > 1) {
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
            for (int x = threadIdx.x; x < nrows * (slice / 4); x += kThreads) {       // this CTA's slice of the dims
                const int row = x >> (HD_BITS - split_bits - 2), d = (x - row * (slice / 4)) * 4;
                const float2* ml = reinterpret_cast<const float2*>(sm + L::slice_ml) + row;
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                float tm = -INFINITY, tl = 0.f;
                for (int r = 0; r < splits; ++r) tm = fmaxf(tm, ml[r * R].x);
                const float safe = tm == -INFINITY ? 0.f : tm;
                for (int r = 0; r < splits; ++r) {
                    const float e = exp2_fast(ml[r * R].x - safe);
                    const float4 f = *reinterpret_cast<const float4*>(sm + L::slice + (r * R + row) * slice + d);
                    tl += ml[r * R].y * e;
                    o.x += f.x * e; o.y += f.y * e; o.z += f.z * e; o.w += f.w * e;
                }
                const bool none = tl == 0.f;
                float f[4] = {none ? 0.f : o.x / tl, none ? 0.f : o.y / tl, none ? 0.f : o.z / tl, none ? 0.f : o.w / tl};
                if (settle<T>(f) && isfinite(tl)) flags[row] = 1;
                *reinterpret_cast<uint2*>(static_cast<T*>(a.attn.out) + places[R + row] + split * slice + d) = make_uint2(Half<T>::pack(f[0], f[1]), Half<T>::pack(f[2], f[3]));
            }
        }
        // A weight of zero times a NaN, of a key that the row does not see: the row is done again.  (Not where the denominator is not finite: then a score
        // that the row sees is a NaN.)
        __syncthreads();
        if (complete)
            for (int row = warp; row < nrows; row += kWarps)
                if (flags[row]) {
                    const int idx = row0 + row, t = token_of(idx);
                    attn4_row_again<T, HD, GS>(a, b, t, kh * G + idx - t * G, span.p0 + t, FLAT ? 0 : split * slice, FLAT ? HD : (split + 1) * slice);
                }
        }
        if constexpr (!FLAT) {
            return;
        } else {
            cur += last - first;
            if (cur >= hi) return;
            __syncthreads();                      // (the sums and flags have been read)
            while (cur >= seq + (long long)span.nb * units) {
                seq += (long long)span.nb * units;
                span = span_of(a, ++b);
            }
        }
    }
}

// The runs of each (sequence, key head, tile of rows) in which a run of the FLAT launch ends: CTA i takes the one in which run i does, if that is the first there.
template <typename T, int HD, int GS, int NT>
__global__ void __launch_bounds__(kThreads)
attn4_sum_kernel(const __grid_constant__ Attn4Args a, const float* __restrict__ part, int row_tiles, int G, int ctas, const __grid_constant__ Attn4Divisors by) {
    constexpr int R = 8 * NT;
    __shared__ long long where[4];
    __shared__ int flags[R];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int units = a.attn.kv_heads * row_tiles, warp = threadIdx.x >> 5;
    const Found f = flat_find(a, units, blockIdx.x + 1, ctas, 0, where);
    const long long at = flat_begin(f.total, blockIdx.x + 1, ctas);
    if (f.b < 0) return;
    const Span span = span_of(a, f.b);
    const int n_unit = (int)((at - f.begin) / span.nb), kh = n_unit / row_tiles, tile = n_unit - kh * row_tiles;
    const long long start = f.begin + (long long)n_unit * span.nb, end = start + span.nb, mine = flat_begin(f.total, blockIdx.x, ctas);
    if (at == start || mine > start) return;                  // run i ends where the next one begins, or did not begin this one
    if (mine == at) return;                                   // (an empty run)
    const int row0 = tile * R, nrows = min(R, span.count * G - row0);
    if (nrows <= 0) return;
    int runs = 1;                                             // runs blockIdx.x .. + runs - 1
    while (flat_begin(f.total, blockIdx.x + runs, ctas) < end) ++runs;
    if (threadIdx.x < R) flags[threadIdx.x] = 0;
    __syncthreads();
    auto slot = [&](int r) { return part + (2LL * (blockIdx.x + r) + (r == 0 && mine != start)) * R * (HD + 2); };
    for (int x = threadIdx.x; x < nrows * (HD / 4); x += kThreads) {
        const int row = x / (HD / 4), d = x % (HD / 4) * 4;
        float tm = -INFINITY, tl = 0.f;
        for (int r = 0; r < runs; ++r)
            if (r == 0 || flat_begin(f.total, blockIdx.x + r, ctas) < flat_begin(f.total, blockIdx.x + r + 1, ctas)) tm = fmaxf(tm, slot(r)[R * HD + 2 * row]);
        const float safe = tm == -INFINITY ? 0.f : tm;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r = 0; r < runs; ++r) {
            if (r > 0 && flat_begin(f.total, blockIdx.x + r, ctas) >= flat_begin(f.total, blockIdx.x + r + 1, ctas)) continue;
            const float2 ml = *reinterpret_cast<const float2*>(slot(r) + R * HD + 2 * row);
            const float4 p = *reinterpret_cast<const float4*>(slot(r) + row * HD + d);
            const float e = exp2_fast(ml.x - safe);
            tl += ml.y * e;
            o.x += p.x * e; o.y += p.y * e; o.z += p.z * e; o.w += p.w * e;
        }
        const bool none = tl == 0.f;
        float v[4] = {none ? 0.f : o.x / tl, none ? 0.f : o.y / tl, none ? 0.f : o.z / tl, none ? 0.f : o.w / tl};
        if (settle<T>(v) && isfinite(tl)) flags[row] = 1;
        const int idx = row0 + row, t = (int)over((unsigned)idx, by.group), head = kh * G + idx - t * G;
        *reinterpret_cast<uint2*>(static_cast<T*>(a.attn.out) + f.b * a.attn.out_stride[0] + t * a.attn.out_stride[1] + head * a.attn.out_stride[2] + d) =
            make_uint2(Half<T>::pack(v[0], v[1]), Half<T>::pack(v[2], v[3]));
    }
    __syncthreads();
    for (int row = warp; row < nrows; row += kWarps)
        if (flags[row]) {
            const int idx = row0 + row, t = (int)over((unsigned)idx, by.group);
            attn4_row_again<T, HD, GS>(a, f.b, t, kh * G + idx - t * G, span.p0 + t, 0, HD);
        }
}

template <typename T, int HD, int GS, int NT, bool FLAT>
int run(const Attn4Args& a, float* part, const Attn4Plan& p, cudaStream_t stream) {
    static std::once_flag once[64];
    static cudaError_t result[64];
    auto* kernel = attn4_rows_kernel<T, HD, GS, NT, FLAT>;
    constexpr int smem = Lay<HD, GS, NT>::total * 4;
    int dev = 0;
    B200GPTQ_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return B200GPTQ_ERR_TOO_LARGE;
    std::call_once(once[dev], [&] { result[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    B200GPTQ_CUDA_TRY(result[dev]);
    const int G = a.attn.heads / a.attn.kv_heads;
    const long long tiles = ((long long)a.attn.tokens * G + 8 * NT - 1) / (8 * NT), ctas = FLAT ? p.ctas : tiles * a.attn.kv_heads * a.attn.batch << p.split_bits;
    if (ctas > 0x7fffffff) return B200GPTQ_ERR_TOO_LARGE;
    const Attn4Divisors by = {Divisor(tiles), Divisor(a.attn.kv_heads), Divisor(G)};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (attn_pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    if (!FLAT && p.split_bits) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = 1 << p.split_bits;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        cfg.numAttrs = n + 1;
    }
    B200GPTQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a, part, FLAT ? 0 : p.split_bits, (int)tiles, G, by));
    if (!FLAT || ctas < 2) return B200GPTQ_OK;
    cfg.gridDim = dim3((unsigned)ctas - 1);
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = n;
    B200GPTQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, attn4_sum_kernel<T, HD, GS, NT>, a, (const float*)part, (int)tiles, G, (int)ctas, by));
    return B200GPTQ_OK;
}

template <typename T, int HD, int GS>
int run_rows(const Attn4Args& a, float* part, const Attn4Plan& p, cudaStream_t stream) {
    if (p.tiles8 == 1) return p.flat ? run<T, HD, GS, 1, true>(a, part, p, stream) : run<T, HD, GS, 1, false>(a, part, p, stream);
    if (p.tiles8 == 2) return p.flat ? run<T, HD, GS, 2, true>(a, part, p, stream) : run<T, HD, GS, 2, false>(a, part, p, stream);
    return p.flat ? run<T, HD, GS, 4, true>(a, part, p, stream) : run<T, HD, GS, 4, false>(a, part, p, stream);
}

template <typename T>
int run_type(const Attn4Args& a, float* part, const Attn4Plan& p, cudaStream_t stream) {
    if (a.cache.hd == 128) return a.cache.group == 32 ? run_rows<T, 128, 32>(a, part, p, stream) : run_rows<T, 128, 64>(a, part, p, stream);
    return a.cache.group == 32 ? run_rows<T, 64, 32>(a, part, p, stream) : run_rows<T, 64, 64>(a, part, p, stream);
}

}  // namespace

int attn4_rows_dispatch(const Attn4Args& a, float* part, const Attn4Plan& p, cudaStream_t stream) {
    return a.attn.dtype == B200GPTQ_F16 ? run_type<__half>(a, part, p, stream) : run_type<__nv_bfloat16>(a, part, p, stream);
}

}  // namespace b200gptq
