// b200gptq_attn_cache for few query rows per key head: the single tokens of a decode step (and short runs of them) over a cache held in 4 bits.
//
//   K = zK + sK cK,  V = zV + sV cV  (zero, scale and code by row and group of dims),   S = Q K^T,  w = softmax(scale S),  O = w V
//
// A row of the cache is 68 to 80 bytes for 128 dims and has to be multiplied by up to 8, 16 or 32 rows of Q, so bytes and instructions bound it alike, and the codes go
// to the tensor cores as they are: a field of four bits that is masked in place, at bits 0 .. 3 or 4 .. 7 of 16, is the fp16 number c 2^-24 or 16 c 2^-24 (subnormal,
// exact), so eight codes cost a shift and four masks.  Scales and zeros are applied beside the products:
//   S(key, row) = sum over groups of  sK (q . cK) + zK (sum of q)      one product chain per group, then an fp32 FMA; the zeros in a product of their own, with
//                                                                      the sums of q in two numbers each (16 bits or more together)
//   O(dim, row) = sum over keys of  (w sV) (cV - 8) + w (zV + 8 sV)    w sV is what is rounded to fp16, and codes of both signs make half of its error of codes from 0 to 15
//                                                                      (by one subtraction in fp16, exact); the second term is summed in fp32, per group
// Q is scaled by a power of two per row (to below 2^15, exact for what is above 2^-38 of the row's largest; so bf16 queries are exact in fp16).  So is w sV, per
// row and group of dims: the largest so far lies between 2^6 and 2^16, so what becomes a subnormal number is off by 2^-31 of it at most.  (One power per warp that followed the largest
// scale alone was wrong: a key of large scale, whatever its weight, or another group's, took the low bits of all others.)  They are 16 bits each, since there are no
// registers left for numbers, and what the sums are in: while weights shrink with a growing maximum, sums stay and their units shrink.
//
// Every warp takes parts of 16 keys on its own, through a ring of cp.async stages in shared memory.  Keys are the 16 of m16n8k16, rows the 8: 8 bytes (128
// dims: 16) of a key are the operand of S as they lie, two keys' words paired by byte permutations that of O (include/b200gptq.h has the order of the codes).
// Rows are only rescaled when a score is more than 8 (log2) above the maximum in use (no weight is above 2^-16; fp32 sums), and then to a weight of 2^-24 for the
// largest: a power of two, which w sV does not round.  (A maximum rounded up to a whole number made all factors powers of two, and the distance of single tokens from 64 bits 2.9e-4 instead of 2.2e-4.)
//
// attn4_cluster_kernel: a cluster of 1 to 8 CTAs shares a (sequence, key head, tile of rows), and they add up through distributed shared memory.
// attn4_flat_kernel: for many keys per tile.  The parts of all sequences and key heads lie one behind the other, and each WARP takes an even run of them, whatever the texts'
// lengths, which are known on the device only.  Where a run ends inside a (sequence, key head) the sums go to scratch, of the eight warps together where the whole CTA is in
// one, and a second launch adds them up in order.  (A run for each CTA, whose warps shared a sequence's part of it: 16 texts of 900 to 15900 tokens, 32 / 8 heads, 66 us and SMs
// idle for a quarter of it, at the ends of sequences and at the end; sums of single warps alone: 1 text of 16000 26 us, with those of CTAs 19.)
//
// Measured (32 / 8 heads of 128): those 16 texts 62 us, 2.8 TB/s; 1 text of 700, 32 heads, 7.4; 2 texts of 16000 and 16 rows 28.8, 1 and 64 rows 56 (26.8 and 48.6
// with a power of two per warp; one copy of the products in a loop, instead of a branch with a second one: 16 texts 69).  A part takes 480 instructions, 60 % of the issue slots of the SMs are in use and half
// of the integer pipe's, and neither memory (42 %) nor the tensor pipe: what is left over are the waits of 4 warps per scheduler for each other's chains (loads from shared memory,
// products, exponentials).
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "attn4.h"
#include "cache4.cuh"

namespace b200gptq {
namespace {

constexpr int kPart = 16, kWarps = kAttn4Warps, kThreads = kWarps * 32, kStages = 4;
constexpr float kGrow = 8.f;             // log2 of what a score may be above the maximum in use
constexpr float kBelow = 24.f;           // log2 of what that maximum's weight lies below 1, so that a million of bf16's largest values add up in fp32
constexpr unsigned kLow = 0x000f000fu, kHigh = 0x00f000f0u;

__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same without a sum before it.
__device__ __forceinline__ void mma16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
template <typename T> __device__ __forceinline__ void mma8_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
    else
        asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
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
template <int N, int OFF = 0> __device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0 + %2], [%1], 16;" ::"r"(dst), "l"(src), "n"(OFF) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0 + %3], [%1], %2;" ::"r"(dst), "l"(src), "n"(N), "n"(OFF) : "memory");
}
template <int N> struct Words { uint32_t w[N]; };
template <int N, int OFF> __device__ __forceinline__ Words<N> lds(uint32_t at) {       // (the offset in the instruction)
    Words<N> r;
    if constexpr (N == 4) asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4 + %5];" : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]) : "r"(at), "n"(OFF));
    else if constexpr (N == 2) asm volatile("ld.shared.v2.b32 {%0,%1}, [%2 + %3];" : "=r"(r.w[0]), "=r"(r.w[1]) : "r"(at), "n"(OFF));
    else asm volatile("ld.shared.b32 %0, [%1 + %2];" : "=r"(r.w[0]) : "r"(at), "n"(OFF));
    return r;
}

// A part in shared memory, in bytes: codes of K as they lie; codes of V, 16 bytes at a time, where each 128 bytes (2 or 4 rows) are permuted so that
// the lanes of a load (rows 2c) meet no bank twice; constants of K and of V.
template <int HD, int GS> struct Stage {
    static constexpr int row = HD / 2, groups = HD / GS, constants = 4 * groups, k = 0, v = kPart * row, kc = 2 * kPart * row, vc = kc + kPart * constants,
                         total = vc + kPart * constants;
    __host__ __device__ static constexpr int v_at(int r, int byte) {
        const int line = r * row / 128, chunk = (r * row % 128 + byte) / 16;
        return v + line * 128 + ((chunk ^ (2 * (line & (HD == 128 ? 3 : 1)))) * 16 + byte % 16);
    }
};

// Shared memory, in floats.  A warp's ring, and with 32 rows its operand made of Q, which registers do not hold (a slot for each lane).  attn4_cluster_kernel, over the
// rings: the warps' sums [warp][row][HD + 4]; behind them their maxima and denominators, the slices that the CTAs of the cluster push [split][row][HD / splits] with maxima
// and denominators, a flag per row.
template <int HD, int GS, int NT> struct Lay {
    static constexpr int R = 8 * NT, LD = HD + 4, q = kStages * Stage<HD, GS>::total / 4, warp = q + (NT == 4 ? NT * (HD / 32) * 32 * 4 : 0), rings = kWarps * warp,
                         sums = kWarps * R * LD, ml = rings > sums ? rings : sums, slice = ml + 2 * kWarps * R, slice_ml = slice + R * HD,
                         flags = slice_ml + 2 * kAttn4MaxSplit * R, total = flags + R;
    static_assert(slice % 4 == 0 && q % 4 == 0 && warp % 4 == 0, "");
};

// Two codes less 8, in units of 2^-24 (or 16 times that): exact.
template <unsigned EIGHT> __device__ __forceinline__ uint32_t centred(uint32_t codes) {
    constexpr uint32_t eight = EIGHT | EIGHT << 16;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&codes), *reinterpret_cast<const __half2*>(&eight));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// a b and a b + c, each of two.
__device__ __forceinline__ float2 times(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 u, v;\n\tmov.b64 u, {%2, %3};\n\tmov.b64 v, {%4, %5};\n\tmul.rn.f32x2 u, u, v;\n\tmov.b64 {%0, %1}, u;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 times_plus(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 u, v, w;\n\tmov.b64 u, {%2, %3};\n\tmov.b64 v, {%4, %5};\n\tmov.b64 w, {%6, %7};\n\tfma.rn.f32x2 u, u, v, w;\n\tmov.b64 {%0, %1}, u;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }
// 2^e; 0 below fp32's normal numbers.
__device__ __forceinline__ float power(int e) { return e < -126 ? 0.f : __uint_as_float((unsigned)(e + 127) << 23); }

// Parts of a sequence: those that its tokens see between them; one at least where there are tokens, since their rows get zeros when they see nothing.
struct Span { AttnRange range; int p0, count, n_s, nb; };
__device__ __forceinline__ Span span_of(const Attn4Args& a, int b) {
    Span s;
    s.p0 = attn_pos(a.attn, b);
    s.count = attn_count(a.attn, b);
    s.range = attn_range(s.p0, s.p0 + max(s.count, 1) - 1, a.attn.window ? a.attn.window : 1 << 30, a.attn.sinks, a.attn.max_seq);
    s.n_s = (s.range.s_end + kPart - 1) / kPart;
    s.nb = s.count ? max(1, s.n_s + (s.range.w_end - s.range.w_start + kPart - 1) / kPart) : 0;
    return s;
}

// What a warp does: parts first, first + step .. below last of a (sequence, key head, tile of rows).
struct Job { int b, kh, row0, nrows, first, last, step; };

// A warp's sums: of rows 8 t + 2 c and + 1; O without the zeros, in units of 2^-24 / fit (dims 64 h + 32 y + 4 g + {0, 2} in acc[4 h + 2 y], {1, 3} in the next), and what the zeros
// add, by group, of the lane's keys.  fit: what w sV is multiplied by, a power of two for each row and group, whose upper 16 bits are all of it.
template <int HD, int GS, int NT> struct Sums {
    static constexpr int HH = HD / 64, NG = HD / GS;
    static constexpr unsigned kFitMost = 0x7e807e80u;            // 2^126: times a weight still a number
    float acc[NT][4 * HH][4], m[NT][2], l[NT][2];
    float2 zacc[NT][NG];                          // (x, y: r = 0, 1)
    unsigned fit[NT][NG];                         // (lower half, upper half)

    static __device__ __forceinline__ int field(unsigned both, int r) { return (int)(r ? both >> 23 : both >> 7 & 0xffu); }       // the exponent's
    static __device__ __forceinline__ float2 numbers(unsigned both) { return make_float2(__uint_as_float(both << 16), __uint_as_float(both & 0xffff0000u)); }
    // Row (t, r)'s sums of group n are multiplied by f.
    __device__ __forceinline__ void scale(int t, int r, int n, float f) {
#pragma unroll
        for (int x = 0; x < GS / 16; ++x) {
            float (&a)[4] = acc[t][GS / 16 * n + x];
            a[r] *= f;
            a[2 + r] *= f;
        }
    }

    // The lanes' shares of denominators and zeros added up.
    __device__ __forceinline__ void settle_lanes() {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    l[t][r] += __shfl_xor_sync(0xffffffffu, l[t][r], o);
#pragma unroll
                    for (int n = 0; n < NG; ++n) (r ? zacc[t][n].y : zacc[t][n].x) += __shfl_xor_sync(0xffffffffu, r ? zacc[t][n].y : zacc[t][n].x, o);
                }
    }
    // Dims 64 h + 32 y + 4 g .. of row r.  (Fields at bits 4 .. 7 were 16 times as large.)
    __device__ __forceinline__ float4 four(int t, int r, int h, int y) const {
        const int n = GS == 32 ? 2 * h + y : h;
        const float z = r ? zacc[t][n].y : zacc[t][n].x, limit = power(127 - field(fit[t][n], r));
        const float *even = acc[t][4 * h + 2 * y], *odd = acc[t][4 * h + 2 * y + 1];
        return make_float4(fmaf(even[r] * 0x1p24f, limit, z), fmaf(odd[r] * 0x1p24f, limit, z), fmaf(even[2 + r] * 0x1p20f, limit, z), fmaf(odd[2 + r] * 0x1p20f, limit, z));
    }
};

template <typename T, int HD, int GS, int NT>
__device__ __forceinline__ void run_parts(const Attn4Args& a, const Job& job, const Span& span, int G, const Divisor& by_group, uint32_t* own, Sums<HD, GS, NT>& sums) {
    using St = Stage<HD, GS>;
    using L = Lay<HD, GS, NT>;
    constexpr int NG = HD / GS, HH = HD / 64, KW = HD / 32, VW = HD / 64;      // words of a key per lane, for S and for O
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3, window = a.attn.window ? a.attn.window : 1 << 30;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(own);
    auto token_of = [&](int idx) { return (int)over((unsigned)idx, by_group); };       // of row idx
    const AttnRange range = span.range;
    const int p_lo = span.p0 + token_of(job.row0), p_hi = span.p0 + token_of(job.row0 + job.nrows - 1), last = job.last;
    const uint8_t *kb = static_cast<const uint8_t*>(a.cache.k) + job.b * a.cache.k_stride[0] + job.kh * a.cache.k_stride[1],
                  *vb = static_cast<const uint8_t*>(a.cache.v) + job.b * a.cache.v_stride[0] + job.kh * a.cache.v_stride[1];
    const T *kcb = static_cast<const T*>(a.cache.k_scales) + job.b * a.cache.k_scale_stride[0] + job.kh * a.cache.k_scale_stride[1],
            *vcb = static_cast<const T*>(a.cache.v_scales) + job.b * a.cache.v_scale_stride[0] + job.kh * a.cache.v_scale_stride[1];
    // A lane's share of a part: 16 bytes of row lane / CHUNKS (128 dims: and of the row 8 further on) of K and of V, the constants of row lane % 16 of K or V.
    constexpr int CHUNKS = St::row / 16;
    const unsigned k_step = (unsigned)a.cache.k_stride[2], v_step = (unsigned)a.cache.v_stride[2],
                   c_step = 2u * (unsigned)(lane < 16 ? a.cache.k_scale_stride[2] : a.cache.v_scale_stride[2]);
    const int r = lane / CHUNKS, byte = lane % CHUNKS * 16;
    const uint8_t *kl = kb + byte, *vl = vb + byte, *cl = reinterpret_cast<const uint8_t*>(lane < 16 ? kcb : vcb);
    const uint32_t k_to = St::k + r * St::row + byte, v_to = St::v_at(r, byte), c_to = (lane < 16 ? St::kc : St::vc) + (lane & 15) * St::constants;
    static_assert(HD == 64 || (Stage<128, GS>::v_at(9, 16) - Stage<128, GS>::v_at(1, 16) == 512), "");
    // The parts lie in two ranges of rows, the sinks and the window; the ring is filled anew for the second.  (Rows behind the end of a range may be read, with weight
    // zero, those behind the cache not.)
    const int most_row = a.attn.max_seq - 1;
    auto fetch = [&](int j0, int behind, uint32_t at) {
        if (j0 < behind) {
            const unsigned j = min(j0 + r, most_row);
            copy_async<16>(at + k_to, kl + (unsigned long long)j * k_step);
            copy_async<16>(at + v_to, vl + (unsigned long long)j * v_step);
            if constexpr (HD == 128) {
                const unsigned j8 = min(j0 + r + 8, most_row);
                copy_async<16, 512>(at + k_to, kl + (unsigned long long)j8 * k_step);
                copy_async<16, 512>(at + v_to, vl + (unsigned long long)j8 * v_step);
            }
            copy_async<St::constants>(at + c_to, cl + (unsigned long long)(unsigned)min(j0 + (lane & 15), most_row) * c_step);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    bool sink = job.first < span.n_s;
    int j0, behind;                               // first row of the warp's next part, a row behind its last one's first
    auto enter = [&](int first) {                 // part `first` of the job's, in the range that it lies in
        j0 = sink ? kPart * first : range.w_start + kPart * (first - span.n_s);
        behind = sink ? kPart * min(last, span.n_s) : range.w_start + kPart * (last - span.n_s);
#pragma unroll
        for (int s = 0; s < kStages; ++s) fetch(j0 + s * kPart * job.step, behind, ring + s * St::total);
    };
    enter(job.first);
    // ---- the operand made of Q: lane (g, c) has dims 32 y + 8 c .. of row 8 t + g, scaled by a power of two, the third and fourth of four by 1 / 16; sums by group ----
    uint4 qr[NT <= 2 ? NT : 1][KW];
    uint4* q_at = reinterpret_cast<uint4*>(own + L::q) + lane;
    uint32_t qz[NT];
    float factor[NT][2];
    float (&acc)[NT][4 * HH][4] = sums.acc, (&m)[NT][2] = sums.m, (&l)[NT][2] = sums.l;
    float2 (&zacc)[NT][NG] = sums.zacc;
    using Fit = Sums<HD, GS, NT>;
    unsigned (&fit)[NT][NG] = sums.fit;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int idx = job.row0 + min(8 * t + g, job.nrows - 1), tok = token_of(idx), head = job.kh * G + idx - tok * G;
        const T* q = static_cast<const T*>(a.attn.q) + job.b * a.attn.q_stride[0] + tok * a.attn.q_stride[1] + head * a.attn.q_stride[2] + 8 * c;
        uint4 raw[KW];
        float most = 0.f;
#pragma unroll
        for (int y = 0; y < KW; ++y) raw[y] = __ldcg(reinterpret_cast<const uint4*>(q + 32 * y));
#pragma unroll
        for (int y = 0; y < KW; ++y) {
            const uint32_t w[4] = {raw[y].x, raw[y].y, raw[y].z, raw[y].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 two = Half<T>::unpack(w[e]);
                most = fmaxf(most, fmaxf(fabsf(two.x), fabsf(two.y)));
            }
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        int up = 15;
        if (most > 0.f && most < INFINITY) frexpf(most, &up);
        // (2^(15 - up) in two factors: bf16's smallest numbers need more than fp32 has)
        const float scale0 = __int_as_float((127 + (15 - up) / 2) << 23), scale1 = __int_as_float((127 + 15 - up - (15 - up) / 2) << 23);
        float of[NG];
#pragma unroll
        for (int y = 0; y < KW; ++y) {
            const uint32_t w[4] = {raw[y].x, raw[y].y, raw[y].z, raw[y].w};
            float f[8], sum = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 two = Half<T>::unpack(w[e]);
                f[2 * e] = two.x * scale0 * scale1;
                f[2 * e + 1] = two.y * scale0 * scale1;
                sum += f[2 * e] + f[2 * e + 1];
            }
            const uint4 made = make_uint4(Half<__half>::pack(f[0], f[1]), Half<__half>::pack(f[2] * 0.0625f, f[3] * 0.0625f), Half<__half>::pack(f[4], f[5]),
                                          Half<__half>::pack(f[6] * 0.0625f, f[7] * 0.0625f));
            if constexpr (NT <= 2) qr[t][y] = made;
            else q_at[(t * KW + y) * 32] = made;
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (GS == 64 && (y & 1)) of[y >> 1] += sum;
            else of[GS == 64 ? y >> 1 : y] = sum;
        }
        // the sums in two numbers each, times 2^-6: factors 0 .. NG - 1 and NG .. 2 NG - 1 of the eight of a product; lane (g, c) has factors 2 c and 2 c + 1
        float upper[2], lower[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float sum = (NG == 4 ? (c & 1 ? of[(2 + e) % NG] : of[e % NG]) : of[e % NG]) * 0x1p-6f;
            upper[e] = Half<T>::wide(Half<T>::round(sum));
            lower[e] = sum - upper[e];
        }
        if constexpr (NG == 4) qz[t] = c < 2 ? Half<T>::pack(upper[0], upper[1]) : Half<T>::pack(lower[0], lower[1]);
        else if constexpr (NG == 2) qz[t] = c == 0 ? Half<T>::pack(upper[0], upper[1]) : c == 1 ? Half<T>::pack(lower[0], lower[1]) : 0u;
        else qz[t] = c == 0 ? Half<T>::pack(upper[0], lower[0]) : 0u;
        const float mine = ldexpf(a.attn.scale * kLog2e, 24 + up - 15);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            m[t][e] = -INFINITY; l[t][e] = 0.f;
            factor[t][e] = __shfl_sync(0xffffffffu, mine, 4 * (2 * c + e));
        }
#pragma unroll
        for (int n = 0; n < NG; ++n) { zacc[t][n] = both(0.f); fit[t][n] = Fit::kFitMost; }
#pragma unroll
        for (int n = 0; n < 4 * HH; ++n) acc[t][n][0] = acc[t][n][1] = acc[t][n][2] = acc[t][n][3] = 0.f;
    }
    // The lane's places in a part: codes and constants of keys g and g + 8, zeros, codes of keys 2c, 2c + 8 and 2c + 1, 2c + 9.
    const uint32_t k_lane = St::k + g * St::row + 4 * KW * c, c_lane = St::kc + g * St::constants, z_lane = c_lane + (NG == 4 ? 8 * (c & 1) : 0),
                   even_lane = St::v_at(2 * c, 4 * VW * g), odd_lane = St::v_at(2 * c + 1, 4 * VW * g);
    const int step = kPart * job.step;
    bool fresh = true;                            // the warp's first part: all sums are zero
    while (true) {
    // Parts that begin between these rows are seen as a whole by all rows of the tile.
    const int end = sink ? range.s_end : range.w_end, whole_from = sink ? 0 : p_hi - window + 1, whole_to = min(sink ? min(end, a.attn.sinks) : end, p_lo + 1) - kPart;
    for (uint32_t from = ring; j0 < behind; j0 += step) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        __syncwarp();
        const bool whole = j0 >= whole_from && j0 <= whole_to;
        const uint32_t k_from = from + k_lane, c_from = from + c_lane, z_from = from + z_lane, even_from = from + even_lane, odd_from = from + odd_lane;
        // ---- S: keys g (0, 1) and g + 8 (2, 3), rows 2 c and 2 c + 1 ----
        float s[NT][4];
        {
            // the zeros of groups 2 (c % 2) and + 1 (where there are fewer groups: of those there are), the same for both halves of a sum of q
            const Words<NG == 1 ? 1 : 2> z0 = lds<NG == 1 ? 1 : 2, 0>(z_from),
                                         z1 = lds<NG == 1 ? 1 : 2, 8 * St::constants>(z_from);
            const uint32_t a0 = __byte_perm(z0.w[0], z0.w[NG == 1 ? 0 : 1], 0x7632u), a1 = __byte_perm(z1.w[0], z1.w[NG == 1 ? 0 : 1], 0x7632u);
            const Words<KW> k0 = lds<KW, 0>(k_from), k1 = lds<KW, 8 * St::row>(k_from);
            const Words<NG> c0 = lds<NG, 0>(c_from), c1 = lds<NG, 8 * St::constants>(c_from);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                mma8_first<T>(s[t], a0, a1, qz[t]);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][e] *= 0x1p-18f;
            }
            float d[NT][4];
#pragma unroll
            for (int y = 0; y < KW; ++y) {        // 32 dims
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
                            const uint2 two = reinterpret_cast<const uint2*>(q_at + (t * KW + y) * 32)[x];
                            b0 = two.x;
                            b1 = two.y;
                        }
                        if (x == 0 && (GS == 32 || !(y & 1))) mma16_first(d[t], w0 & kLow, w1 & kLow, w0 & kHigh, w1 & kHigh, b0, b1);
                        else mma16(d[t], w0 & kLow, w1 & kLow, w0 & kHigh, w1 & kHigh, b0, b1);
                    }
                }
                if (GS == 32 || (y & 1)) {
                    const int n = GS == 32 ? y : y >> 1;
                    const float f0 = Half<T>::unpack(c0.w[n]).x, f1 = Half<T>::unpack(c1.w[n]).x;
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            const float2 two = times_plus(both(e ? f1 : f0), make_float2(d[t][e], d[t][e + 1]), make_float2(s[t][e], s[t][e + 1]));
                            s[t][e] = two.x;
                            s[t][e + 1] = two.y;
                        }
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][e] *= factor[t][e & 1];
        }
        if (!whole) {
            __syncwarp();                         // (so that it stays a branch: with predicates instead each part took 45 instructions more)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = j0 + g + 8 * (e >> 1), p = span.p0 + token_of(job.row0 + min(8 * t + 2 * c + (e & 1), job.nrows - 1));
                    s[t][e] = j < end && attn_sees(p, j, window, a.attn.sinks) ? s[t][e] : -INFINITY;
                }
        }
        bool grow = false;
        float top[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                top[t][r] = fmaxf(s[t][r], s[t][2 + r]);
                grow = grow || top[t][r] - m[t][r] > kGrow - kBelow;
            }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                int down[2];
                float2 corr, rest;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float up = top[t][r];
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, o));
                    up += kBelow;
                    const float by = up - m[t][r];           // (infinite where there was nothing, or a score is infinite: what there was counts for nothing)
                    const bool moves = by > kGrow;
                    if (moves) m[t][r] = up;
                    down[r] = moves ? (int)fminf(ceilf(by), 255.f) : 0;
                    (r ? corr.y : corr.x) = moves ? exp2_fast(-by) : 1.f;
                    (r ? rest.y : rest.x) = moves ? exp2_fast((float)down[r] - by) : 1.f;
                    if (!fresh) l[t][r] *= r ? corr.y : corr.x;
                }
                if (fresh) continue;
#pragma unroll
                for (int n = 0; n < NG; ++n) {    // what was the largest w sV is smaller by as much: units of the sums shrink so too, by the power of two that is next
                    const unsigned old = fit[t][n], now = __vminu2(old + ((unsigned)down[0] << 7 | (unsigned)down[1] << 23), Fit::kFitMost);
                    zacc[t][n] = times(zacc[t][n], corr);
                    fit[t][n] = now;
#pragma unroll
                    for (int r = 0; r < 2; ++r) sums.scale(t, r, n, power(Fit::field(now, r) - Fit::field(old, r) - down[r]) * (r ? rest.y : rest.x));
                }
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float safe = m[t][r] == -INFINITY ? 0.f : m[t][r];
                {
                    s[t][r] = exp2_fast(s[t][r] - safe);
                    s[t][2 + r] = exp2_fast(s[t][2 + r] - safe);
                    l[t][r] += s[t][r] + s[t][2 + r];
                }
            }
        // ---- O: codes of keys 2c, 2c + 1 and 2c + 8, 2c + 9 in pairs ----
        {
            // constants of V; those of keys behind the end count for nothing
            const Words<NG> u0 = lds<NG, kPart * St::constants>(c_from), u1 = lds<NG, (kPart + 8) * St::constants>(c_from);
            float sv[2][NG];
            {
                float zv[2][NG];
#pragma unroll
                for (int n = 0; n < NG; ++n) {
                    const float2 f0 = Half<T>::unpack(u0.w[n]), f1 = Half<T>::unpack(u1.w[n]);
                    sv[0][n] = f0.x; zv[0][n] = fmaf(8.f, f0.x, f0.y); sv[1][n] = f1.x; zv[1][n] = fmaf(8.f, f1.x, f1.y);
                }
                if (!whole) {
                    __syncwarp();
#pragma unroll
                    for (int n = 0; n < NG; ++n) {
                        if (j0 + g >= end) sv[0][n] = zv[0][n] = 0.f;
                        if (j0 + g + 8 >= end) sv[1][n] = zv[1][n] = 0.f;
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int n = 0; n < NG; ++n)
                        zacc[t][n] = times_plus(make_float2(s[t][0], s[t][1]), both(zv[0][n]), times_plus(make_float2(s[t][2], s[t][3]), both(zv[1][n]), zacc[t][n]));
            }
            // w sV as operands, of as many groups at once as registers hold
            constexpr int ONCE = NT <= 2 ? NG : 1, EIGHT = St::v_at(8, 0) - St::v_at(0, 0);
            Words<VW> v[4];
#pragma unroll
            for (int n0 = 0; n0 < NG; n0 += ONCE) {
                uint32_t b0[NT][ONCE], b1[NT][ONCE];
                auto products = [&] {             // (the weight first: a large scale alone may pass fp32 in units for small products)
                    __half2 most = __float2half2_rn(0.f);        // (a NaN, 0 times an infinity that is not seen, counts for nothing)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int i = 0; i < ONCE; ++i) {
                            const int n = n0 + i;
                            const float2 f = Fit::numbers(fit[t][n]),
                                         p0 = times(times(make_float2(s[t][0], s[t][1]), f), both(sv[0][n])),
                                         p1 = times(times(make_float2(s[t][2], s[t][3]), f), both(sv[1][n]));
                            b0[t][i] = Half<__half>::pack(p0.x, p0.y);
                            b1[t][i] = Half<__half>::pack(p1.x, p1.y);
                            most = __hmax2(most, __hmax2(__habs2(*reinterpret_cast<const __half2*>(&b0[t][i])), __habs2(*reinterpret_cast<const __half2*>(&b1[t][i]))));
                        }
                    return most;
                };
                if (__any_sync(0xffffffffu, !__hble2(products(), __float2half2_rn(32768.f)))) {      // units in which the largest product is 2^6 or a little more
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int i = 0; i < ONCE; ++i) {         // (of each row: upper halves of numbers, whose order is theirs)
                            const int n = n0 + i;
                            const float2 p0 = times(make_float2(s[t][0], s[t][1]), both(sv[0][n])), p1 = times(make_float2(s[t][2], s[t][3]), both(sv[1][n]));
                            const float x = fmaxf(fmaxf(fabsf(p0.x), fabsf(p1.x)), 0.f), y = fmaxf(fmaxf(fabsf(p0.y), fabsf(p1.y)), 0.f);
                            unsigned large = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632u);
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) large = __vmaxu2(large, __shfl_xor_sync(0xffffffffu, large, o));
                            // (exponent fields: 127 for 1, so 254 + 6 less that of the largest)
                            const unsigned old = fit[t][n], now = __vminu2(old, (260u << 7 | 260u << 23) - (large & 0x7f807f80u));
                            fit[t][n] = now;
                            if (!fresh)
#pragma unroll
                                for (int r = 0; r < 2; ++r) sums.scale(t, r, n, power(Fit::field(now, r) - Fit::field(old, r)));
                        }
                    products();
                }
                if (n0 == 0) { v[0] = lds<VW, 0>(even_from); v[1] = lds<VW, 0>(odd_from); v[2] = lds<VW, EIGHT>(even_from); v[3] = lds<VW, EIGHT>(odd_from); }
#pragma unroll
                for (int i = 0; i < ONCE; ++i) {
                    const int n = n0 + i, h = GS == 32 ? n >> 1 : n;
                    const uint32_t x[2][2] = {{__byte_perm(v[0].w[h], v[1].w[h], 0x5410u), __byte_perm(v[2].w[h], v[3].w[h], 0x5410u)},
                                              {__byte_perm(v[0].w[h], v[1].w[h], 0x7632u), __byte_perm(v[2].w[h], v[3].w[h], 0x7632u)}};
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        b0[t][i] = transposed(b0[t][i]);
                        b1[t][i] = transposed(b1[t][i]);
                    }
#pragma unroll
                    for (int y = GS == 32 ? n & 1 : 0; y < (GS == 32 ? (n & 1) + 1 : 2); ++y)        // dims 64 h + 32 y + 4 g + {0, 2} and {1, 3}
#pragma unroll
                        for (int z = 0; z < 2; ++z) {
                            const uint32_t k01 = x[z][0] >> (8 * y), k89 = x[z][1] >> (8 * y);
                            const uint32_t a0 = centred<8>(k01 & kLow), a1 = centred<128>(k01 & kHigh), a2 = centred<8>(k89 & kLow), a3 = centred<128>(k89 & kHigh);
#pragma unroll
                            for (int t = 0; t < NT; ++t) mma16(acc[t][4 * h + 2 * y + z], a0, a1, a2, a3, b0[t][i], b1[t][i]);
                        }
                }
            }
        }
        fresh = false;
        __syncwarp();                             // (the part has been read)
        fetch(j0 + kStages * step, behind, from);
        from = from + St::total == ring + kStages * St::total ? ring : from + St::total;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // on to the window: the job's first part behind the sinks
    if (!sink || last <= span.n_s) break;
    __syncwarp();                                 // (the ring has been read)
    sink = false;
    enter(job.first + (span.n_s - job.first + job.step - 1) / job.step * job.step);
    }
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

template <typename T, int HD, int GS, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1)
attn4_cluster_kernel(const __grid_constant__ Attn4Args a, int split_bits, int row_tiles, int G, const __grid_constant__ Attn4Divisors by) {
    using L = Lay<HD, GS, NT>;
    constexpr int R = 8 * NT, HH = HD / 64;
    extern __shared__ __align__(16) float sm[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3, splits = 1 << split_bits;
    if (splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const unsigned per_unit = blockIdx.x >> split_bits, unit = over(per_unit, by.row_tiles), b = over(unit, by.kv_heads);
    const int split = blockIdx.x - (per_unit << split_bits), kh = unit - b * a.attn.kv_heads;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const Span span = span_of(a, b);
    Job job = {(int)b, kh, (int)(per_unit - unit * row_tiles) * R, 0, (int)((long long)span.nb * split >> split_bits) + warp, (int)((long long)span.nb * (split + 1) >> split_bits), kWarps};
    job.nrows = min(R, span.count * G - job.row0);
    const int nrows = job.nrows;
    if (nrows <= 0) return;                       // padding: every CTA of the cluster leaves
    int* flags = reinterpret_cast<int*>(sm + L::flags);
    if (threadIdx.x < R) flags[threadIdx.x] = 0;
    Sums<HD, GS, NT> sums;
    run_parts<T, HD, GS, NT>(a, job, span, G, by.group, reinterpret_cast<uint32_t*>(sm + warp * L::warp), sums);
    sums.settle_lanes();
    __syncthreads();                              // (the rings have been read)
    // ---- the warps' sums: rows, four adjacent dims each ----
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = 8 * t + 2 * c + r;
            if (row < nrows) {
                if (g == 0) { sm[L::ml + 2 * (warp * R + row)] = sums.m[t][r]; sm[L::ml + 2 * (warp * R + row) + 1] = sums.l[t][r]; }
#pragma unroll
                for (int h = 0; h < HH; ++h)
#pragma unroll
                    for (int y = 0; y < 2; ++y) *reinterpret_cast<float4*>(sm + (warp * R + row) * L::LD + 64 * h + 32 * y + 4 * g) = sums.four(t, r, h, y);
            }
        }
    __syncthreads();
    if (splits > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");      // (all CTAs of the cluster run)
    // ---- the CTA's sums: out, or slice by slice to the CTAs of the cluster ----
    const int slice = HD >> split_bits;
    constexpr int HD_BITS = HD == 128 ? 7 : 6;
    auto out_of = [&](int row) {
        const int idx = job.row0 + row, t = (int)over((unsigned)idx, by.group), head = kh * G + idx - t * G;
        return static_cast<T*>(a.attn.out) + b * a.attn.out_stride[0] + t * a.attn.out_stride[1] + head * a.attn.out_stride[2];
    };
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
        if (splits == 1) {
            const bool none = cl == 0.f;
            float f[4] = {none ? 0.f : o.x / cl, none ? 0.f : o.y / cl, none ? 0.f : o.z / cl, none ? 0.f : o.w / cl};
            if (settle<T>(f) && isfinite(cl)) flags[row] = 1;
            *reinterpret_cast<uint2*>(out_of(row) + d) = make_uint2(Half<T>::pack(f[0], f[1]), Half<T>::pack(f[2], f[3]));
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
    if (splits > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        for (int x = threadIdx.x; x < nrows * (slice / 4); x += kThreads) {           // this CTA's slice of the dims
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
            *reinterpret_cast<uint2*>(out_of(row) + split * slice + d) = make_uint2(Half<T>::pack(f[0], f[1]), Half<T>::pack(f[2], f[3]));
        }
    }
    // A weight of zero times a NaN, of a key that the row does not see: the row is done again.  (Not where the denominator is not finite: then a score that the row
    // sees is a NaN.)
    __syncthreads();
    for (int row = warp; row < nrows; row += kWarps)
        if (flags[row]) {
            const int idx = job.row0 + row, t = (int)over((unsigned)idx, by.group);
            attn4_row_again<T, HD, GS>(a, b, t, kh * G + idx - t * G, span.p0 + t, split * slice, (split + 1) * slice);
        }
}

// ---- the parts of all sequences and key heads one behind the other ----
__device__ __forceinline__ long long divided(long long n, int d) {       // n >= 0, d > 0 (a division of 64 bits takes some 100 instructions)
    return n >> 32 ? n / d : (long long)((unsigned)n / (unsigned)d);
}
// The runs: the first `more` have `each` + 1 parts, the others `each`.
struct Runs {
    long long each;
    int more;
    __device__ __forceinline__ Runs(long long total, int runs) : each(divided(total, runs)), more((int)(total - each * runs)) {}
    __device__ __forceinline__ long long begin(int i) const { return each * i + min(i, more); }
    // The run that has part `at` of them.
    __device__ __forceinline__ int of(long long at) const {
        const long long longer = (each + 1) * more;
        return at < longer ? (int)divided(at, (int)(each + 1)) : more + (int)divided(at - longer, (int)each);
    }
};
// The sequences' parts as a warp sees them, 32 sequences at a time; `units`: key heads times tiles of rows, which have the same parts each.
struct Parts {
    long long mine, to, before;               // of the lane's sequence; with those before it among the 32; before these
    int b0;

    __device__ __forceinline__ void look(const Attn4Args& a, int units, int first) {
        const int lane = threadIdx.x & 31;
        b0 = first;
        mine = b0 + lane < a.attn.batch ? (long long)span_of(a, b0 + lane).nb * units : 0;
        to = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, to, o);
            if (lane >= o) to += x;
        }
    }
    // Leaves the first 32 sequences, so that there is nothing to be looked at again where there are no more.
    __device__ __forceinline__ long long all(const Attn4Args& a, int units) {
        long long sum = 0;
        for (int first = (a.attn.batch - 1) / 32 * 32; first >= 0; first -= 32) {
            look(a, units, first);
            sum += __shfl_sync(0xffffffffu, to, 31);
        }
        before = 0;
        return sum;
    }
    __device__ __forceinline__ void next(const Attn4Args& a, int units) {
        const long long sum = before + __shfl_sync(0xffffffffu, to, 31);
        look(a, units, b0 + 32);
        before = sum;
    }
    // The part with which lane who's sequence begins.
    __device__ __forceinline__ long long begin_of(int who) const { return before + __shfl_sync(0xffffffffu, to - mine, who); }
};
// Scratch of a run: what it did of the (sequence, key head, tile) in which it began, and of that in which it ended.
template <int HD, int NT> __device__ __forceinline__ float* scratch_of(float* part, int run, bool second) { return part + (2LL * run + second) * (8 * NT * (HD + 2)); }

template <typename T, int HD, int GS, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1)
attn4_flat_kernel(const __grid_constant__ Attn4Args a, float* __restrict__ part, int row_tiles, int G, const __grid_constant__ Attn4Divisors by) {
    using L = Lay<HD, GS, NT>;
    constexpr int R = 8 * NT, HH = HD / 64;
    extern __shared__ __align__(16) float sm[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3, units = a.attn.kv_heads * row_tiles, runs = gridDim.x * kWarps,
              run = blockIdx.x * kWarps + warp;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    Parts parts;
    const Runs by_run(parts.all(a, units), runs);
    const long long begin = by_run.begin(run), end = by_run.begin(run + 1), cta_begin = by_run.begin(run - warp), cta_end = by_run.begin(run - warp + kWarps);
    if (cta_begin >= cta_end) return;
    unsigned hit;
    while (!(hit = __ballot_sync(0xffffffffu, parts.mine && parts.before + parts.to > cta_begin))) parts.next(a, units);
    Job job;
    job.b = parts.b0 + __ffs(hit) - 1;
    long long sequence = parts.begin_of(__ffs(hit) - 1);         // the part with which it begins
    // All that the CTA does may lie in one (sequence, key head, tile): then its warps add up and leave one set of sums.
    const int nb0 = (int)divided(__shfl_sync(0xffffffffu, parts.mine, __ffs(hit) - 1), units), unit0 = (int)divided(cta_begin - sequence, nb0);
    const bool together = cta_end <= sequence + (long long)(unit0 + 1) * nb0;
    if (!together) {
        if (begin >= end) return;
        while (!(hit = __ballot_sync(0xffffffffu, parts.mine && parts.before + parts.to > begin))) parts.next(a, units);
        job.b = parts.b0 + __ffs(hit) - 1;
        sequence = parts.begin_of(__ffs(hit) - 1);
    }
    float* sums_at = sm + warp * L::warp;         // in place of the ring: [row][HD + 4], maximum and denominator behind a row
    static_assert(R * L::LD <= L::warp, "");
    if (together && begin >= end && lane < R) *reinterpret_cast<float2*>(sums_at + lane * L::LD + HD) = make_float2(-INFINITY, 0.f);
    for (long long cur = begin; cur < end;) {
        const Span span = span_of(a, job.b);
        if (cur >= sequence + (long long)span.nb * units) {      // the next sequence
            sequence += (long long)span.nb * units;
            ++job.b;
            continue;
        }
        const int unit = (int)divided(cur - sequence, span.nb);
        job.kh = (int)over((unsigned)unit, by.row_tiles);
        job.row0 = (unit - job.kh * row_tiles) * R;
        job.nrows = min(R, span.count * G - job.row0);
        job.first = (int)(cur - sequence - (long long)unit * span.nb);
        job.last = (int)min((long long)span.nb, job.first + (end - cur));
        job.step = 1;
        const bool second = cur != begin;
        cur += job.last - job.first;
        if (job.nrows <= 0) continue;             // padding
        Sums<HD, GS, NT> sums;
        run_parts<T, HD, GS, NT>(a, job, span, G, by.group, reinterpret_cast<uint32_t*>(sm + warp * L::warp), sums);
        sums.settle_lanes();
        __syncwarp();                             // (the ring has been read)
        if (together || job.first > 0 || job.last < span.nb) {
            float* to = together ? sums_at : scratch_of<HD, NT>(part, run, second);
            const int row_step = together ? L::LD : HD;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int row = 8 * t + 2 * c + r;
                    if (row >= job.nrows) continue;
                    if (g == 0) *reinterpret_cast<float2*>(to + (together ? row * L::LD + HD : R * HD + 2 * row)) = make_float2(sums.m[t][r], sums.l[t][r]);
#pragma unroll
                    for (int h = 0; h < HH; ++h)
#pragma unroll
                        for (int y = 0; y < 2; ++y) *reinterpret_cast<float4*>(to + row * row_step + 64 * h + 32 * y + 4 * g) = sums.four(t, r, h, y);
                }
            continue;
        }
        unsigned bad[NT][2];                      // lanes with a result that is not finite beside a denominator that is
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = 8 * t + 2 * c + r, idx = job.row0 + min(row, job.nrows - 1), tok = (int)over((unsigned)idx, by.group), head = job.kh * G + idx - tok * G;
                T* out = static_cast<T*>(a.attn.out) + job.b * a.attn.out_stride[0] + tok * a.attn.out_stride[1] + head * a.attn.out_stride[2];
                const float l = sums.l[t][r];
                const bool none = l == 0.f;
                bool odd = false;
#pragma unroll
                for (int h = 0; h < HH; ++h)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const float4 o = sums.four(t, r, h, y);
                        float f[4] = {none ? 0.f : o.x / l, none ? 0.f : o.y / l, none ? 0.f : o.z / l, none ? 0.f : o.w / l};
                        odd = settle<T>(f) || odd;
                        if (row < job.nrows) *reinterpret_cast<uint2*>(out + 64 * h + 32 * y + 4 * g) = make_uint2(Half<T>::pack(f[0], f[1]), Half<T>::pack(f[2], f[3]));
                    }
                bad[t][r] = __ballot_sync(0xffffffffu, odd && isfinite(l) && row < job.nrows);
            }
        __syncwarp();
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r)
                for (int x = 0; x < 4 && bad[t][r]; ++x)
                    if (bad[t][r] & 0x11111111u << x) {
                        const int idx = job.row0 + 8 * t + 2 * x + r, tok = (int)over((unsigned)idx, by.group);
                        attn4_row_again<T, HD, GS>(a, job.b, tok, job.kh * G + idx - tok * G, span.p0 + tok, 0, HD);
                    }
    }
    if (!together) return;
    __syncthreads();
    const int row0 = (unit0 - (int)over((unsigned)unit0, by.row_tiles) * row_tiles) * R, nrows = min(R, attn_count(a.attn, job.b) * G - row0);
    float* to = scratch_of<HD, NT>(part, run - warp, false);
    for (int x = threadIdx.x; x < nrows * (HD / 4); x += kThreads) {
        const int row = x / (HD / 4), d = x % (HD / 4) * 4;
        float cm = -INFINITY, cl = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) cm = fmaxf(cm, sm[w * L::warp + row * L::LD + HD]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float2 ml = *reinterpret_cast<const float2*>(sm + w * L::warp + row * L::LD + HD);
            if (ml.x == -INFINITY) continue;      // (nothing seen, or no part)
            const float e = exp2_fast(ml.x - cm);
            const float4 f = *reinterpret_cast<const float4*>(sm + w * L::warp + row * L::LD + d);
            cl += ml.y * e;
            o.x += f.x * e; o.y += f.y * e; o.z += f.z * e; o.w += f.w * e;
        }
        *reinterpret_cast<float4*>(to + row * HD + d) = o;
        if (d == 0) *reinterpret_cast<float2*>(to + R * HD + 2 * row) = make_float2(cm, cl);
    }
}

// A CTA for each row: the runs that share its (sequence, key head, tile), taken in turn by the warps (64 dims: halves of warps), which add up at the end, in order.
// What lies before the wait was written before the launch in front of this one let it start, when all its CTAs had waited themselves; the loads by-pass L1.
template <typename T, int HD, int GS, int NT>
__global__ void __launch_bounds__(kThreads)
attn4_sum_kernel(const __grid_constant__ Attn4Args a, float* __restrict__ part, int row_tiles, int G, int runs, const __grid_constant__ Attn4Divisors by) {
    constexpr int R = 8 * NT, LANES = HD / 4, TAKERS = kThreads / LANES, DEEP = 4;
    __shared__ float4 sum[TAKERS][LANES];
    __shared__ float2 ml[TAKERS];
    const int units = a.attn.kv_heads * row_tiles, taker = threadIdx.x / LANES, d = threadIdx.x % LANES * 4;
    const unsigned unit_all = blockIdx.x / R, per_kh = over(unit_all, by.row_tiles), b = over(per_kh, by.kv_heads);
    const int row = blockIdx.x % R, tile = unit_all - per_kh * row_tiles, kh = per_kh - b * a.attn.kv_heads, idx = tile * R + row;
    const Span span = span_of(a, b);
    const bool there = idx < span.count * G;
    Parts parts;
    const Runs by_run(parts.all(a, units), runs);
    while (parts.b0 + 32 <= (int)b) parts.next(a, units);
    const long long start = parts.begin_of((int)b - parts.b0) + (long long)(kh * row_tiles + tile) * span.nb, end = start + span.nb;
    // What there is: sums of runs, or of CTAs where all that a CTA did is in this unit; `early` runs, `ctas` CTAs from `cta` on, `late` runs.
    const int first = there ? by_run.of(start) : 0, last = there ? by_run.of(end - 1) : 0, cta0 = first / kWarps, cta1 = last / kWarps;
    auto inside = [&](int i) { return by_run.begin(i * kWarps) >= start && by_run.begin(i * kWarps + kWarps) <= end; };
    const bool in0 = inside(cta0), in1 = inside(cta1);
    const int early = in0 ? 0 : min(last + 1, (cta0 + 1) * kWarps) - first, cta = in0 ? cta0 : cta0 + 1, ctas = max(0, (in1 ? cta1 : cta1 - 1) - cta + 1),
              late = cta1 > cta0 && !in1 ? last - cta1 * kWarps + 1 : 0, records = early + ctas + late;
    const bool whole = !in0 && first == last;
    const bool second = by_run.begin(first) < start;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    if (!there || whole) return;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = taker; i0 < records; i0 += DEEP * TAKERS) {
        float2 of[DEEP];
        float4 v[DEEP];
        float up = m;
#pragma unroll
        for (int x = 0; x < DEEP; ++x) {
            const int i = i0 + x * TAKERS;
            const bool has = i < records;
            const int r = !has ? (early ? first : cta * kWarps) : i < early ? first + i : i < early + ctas ? (cta + i - early) * kWarps : cta1 * kWarps + i - early - ctas;
            const float* from = scratch_of<HD, NT>(part, r, r == first && second);
            of[x] = __ldcg(reinterpret_cast<const float2*>(from + R * HD + 2 * row));
            v[x] = __ldcg(reinterpret_cast<const float4*>(from + row * HD + d));
            if (!has) of[x] = make_float2(-INFINITY, 0.f);
            up = fmaxf(up, of[x].x);
        }
        const float safe = up == -INFINITY ? 0.f : up, corr = exp2_fast(m - safe);
        m = up;
        l *= corr;
        o.x *= corr; o.y *= corr; o.z *= corr; o.w *= corr;
#pragma unroll
        for (int x = 0; x < DEEP; ++x) {
            if (of[x].x == -INFINITY) continue;               // (nothing seen, or nothing there)
            const float e = exp2_fast(of[x].x - safe);
            l += of[x].y * e;
            o.x += v[x].x * e; o.y += v[x].y * e; o.z += v[x].z * e; o.w += v[x].w * e;
        }
    }
    sum[taker][d / 4] = o;
    if (d == 0) ml[taker] = make_float2(m, l);
    __syncthreads();
    if (threadIdx.x >= 32) return;
    float tm = -INFINITY, tl = 0.f;
#pragma unroll
    for (int x = 0; x < TAKERS; ++x) tm = fmaxf(tm, ml[x].x);
    const float safe = tm == -INFINITY ? 0.f : tm;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < TAKERS; ++x) {
        const float e = exp2_fast(ml[x].x - safe);
        const float4 v = sum[x][d / 4];
        tl += ml[x].y * e;
        o.x += v.x * e; o.y += v.y * e; o.z += v.z * e; o.w += v.w * e;
    }
    const bool none = tl == 0.f;
    float f[4] = {none ? 0.f : o.x / tl, none ? 0.f : o.y / tl, none ? 0.f : o.z / tl, none ? 0.f : o.w / tl};
    const bool bad = settle<T>(f);
    const int t = (int)over((unsigned)idx, by.group), head = kh * G + idx - t * G;
    if (threadIdx.x < LANES)
        *reinterpret_cast<uint2*>(static_cast<T*>(a.attn.out) + b * a.attn.out_stride[0] + t * a.attn.out_stride[1] + head * a.attn.out_stride[2] + d) =
            make_uint2(Half<T>::pack(f[0], f[1]), Half<T>::pack(f[2], f[3]));
    __syncwarp();
    if (__any_sync(0xffffffffu, bad && isfinite(tl))) attn4_row_again<T, HD, GS>(a, b, t, head, span.p0 + t, 0, HD);      // (as in attn4_cluster_kernel)
}

// A kernel's limit of shared memory, once per device.
struct Allowed {
    std::once_flag once[64];
    cudaError_t result[64];
    template <typename Kernel> int shared(Kernel* kernel, int bytes) {
        int dev = 0;
        B200GPTQ_CUDA_TRY(cudaGetDevice(&dev));
        if (dev < 0 || dev >= 64) return B200GPTQ_ERR_TOO_LARGE;
        std::call_once(once[dev], [&] { result[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
        B200GPTQ_CUDA_TRY(result[dev]);
        return B200GPTQ_OK;
    }
};

template <typename T, int HD, int GS, int NT>
int run(const Attn4Args& a, float* part, const Attn4Plan& p, cudaStream_t stream) {
    static Allowed cluster_allowed, flat_allowed;
    constexpr int smem = Lay<HD, GS, NT>::total * 4, flat_smem = Lay<HD, GS, NT>::rings * 4;
    const int G = a.attn.heads / a.attn.kv_heads;
    const long long tiles = ((long long)a.attn.tokens * G + 8 * NT - 1) / (8 * NT), units = tiles * a.attn.kv_heads * a.attn.batch, ctas = p.flat ? p.ctas : units << p.split_bits;
    if (ctas > 0x7fffffff || units * 8 * NT > 0x7fffffff) return B200GPTQ_ERR_TOO_LARGE;
    const Attn4Divisors by = {Divisor(tiles), Divisor(a.attn.kv_heads), Divisor(G)};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kThreads);
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
    if (!p.flat) {
        auto* kernel = attn4_cluster_kernel<T, HD, GS, NT>;
        const int st = cluster_allowed.shared(kernel, smem);
        if (st != B200GPTQ_OK) return st;
        cfg.dynamicSmemBytes = smem;
        if (p.split_bits) {
            attr[n].id = cudaLaunchAttributeClusterDimension;
            attr[n].val.clusterDim.x = 1 << p.split_bits;
            attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
            cfg.numAttrs = n + 1;
        }
        B200GPTQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a, p.split_bits, (int)tiles, G, by));
        return B200GPTQ_OK;
    }
    auto* kernel = attn4_flat_kernel<T, HD, GS, NT>;
    const int st = flat_allowed.shared(kernel, flat_smem);
    if (st != B200GPTQ_OK) return st;
    cfg.dynamicSmemBytes = flat_smem;
    B200GPTQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a, part, (int)tiles, G, by));
    cfg.gridDim = dim3((unsigned)(units * 8 * NT));
    cfg.dynamicSmemBytes = 0;
    B200GPTQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, attn4_sum_kernel<T, HD, GS, NT>, a, part, (int)tiles, G, (int)ctas * kWarps, by));
    return B200GPTQ_OK;
}

template <typename T, int HD, int GS>
int run_rows(const Attn4Args& a, float* part, const Attn4Plan& p, cudaStream_t stream) {
    return p.tiles8 == 1 ? run<T, HD, GS, 1>(a, part, p, stream) : p.tiles8 == 2 ? run<T, HD, GS, 2>(a, part, p, stream) : run<T, HD, GS, 4>(a, part, p, stream);
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
