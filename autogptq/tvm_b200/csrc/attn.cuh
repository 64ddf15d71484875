// What the two kernels of b200gptq_attn share: the types' conversions, what a query sees, and the slow exact row.
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"

namespace b200gptq {

constexpr float kLog2e = 1.4426950408889634f;

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994): with s = ceil(log2 d) and
// m = floor(2^32 (2^s - d) / d) + 1 it is (high word of m n + n) / 2^s.  The kernels divide where they start, by numbers that the host knows: a
// division there took 50 to 200 ns, one of 64 bits more, in launches of 3 to 20 us.
struct Divisor {
    unsigned m, s;
    explicit Divisor(long long d = 1) : s(0) {
        while (1LL << s < d) ++s;
        m = (unsigned)((((1LL << s) - d) << 32) / d + 1);
    }
};
__device__ __forceinline__ unsigned over(unsigned n, const Divisor& d) { return (__umulhi(n, d.m) + n) >> d.s; }

template <typename T> struct Half;       // the two 16-bit types
template <> struct Half<__half> {
    __device__ static __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    __device__ static __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
    __device__ static __forceinline__ __half round(float a) { return __float2half_rn(a); }
    __device__ static __forceinline__ float wide(__half a) { return __half2float(a); }
    static constexpr float kTop = 65504.f;
};
template <> struct Half<__nv_bfloat16> {
    __device__ static __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    __device__ static __forceinline__ float2 unpack(uint32_t u) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u)); }
    __device__ static __forceinline__ __nv_bfloat16 round(float a) { return __float2bfloat16_rn(a); }
    __device__ static __forceinline__ float wide(__nv_bfloat16 a) { return __bfloat162float(a); }
    static constexpr float kTop = 3.4028235e38f;      // (of fp32: values near bf16's largest number pass its range as they are added up)
};

// N results of a row, before they are rounded; whether one of them is not finite.  A mean of values is no larger than the largest of them, but with weights that
// are rounded and a sum that is not it can pass fp16's largest number by 2^-11, which rounds to infinity: it is that number then.  (All are looked at
// together: two chunks of 512 of 72 heads 61.2 us; 62.2 with each one held by itself, 60.4 with none.)
template <typename T, int N> __device__ __forceinline__ bool settle(float (&f)[N]) {
    bool odd = false, bad = false;
#pragma unroll
    for (int x = 0; x < N; ++x) odd = odd || !(fabsf(f[x]) <= Half<T>::kTop);
    if (odd)
#pragma unroll
        for (int x = 0; x < N; ++x) {
            if (isfinite(f[x])) f[x] = fminf(fmaxf(f[x], -Half<T>::kTop), Half<T>::kTop);
            else bad = true;
        }
    return bad;
}

__device__ __forceinline__ float exp2_fast(float x) {       // 2^x; 0 for -infinity
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Position of token 0 of sequence b.  Positions far outside the cache behave like those just outside (all sizes are 2^29 at most: with a window what
// lies 2^30 out has left the cache behind; without, where a window of 2^30 stands for none, tokens up to 2^29 - 1 further on still see row 0).
__device__ __forceinline__ int attn_pos(const b200gptq_attn_args& a, int b) {
    const long long p = __ldcg(reinterpret_cast<const long long*>(a.pos) + (a.pos_each ? b : 0));
    return (int)max(min(p, a.window ? 1LL << 30 : 1LL << 29), -(1LL << 30));
}
__device__ __forceinline__ int attn_count(const b200gptq_attn_args& a, int b) {
    if (!a.counts) return a.tokens;
    const long long n = __ldcg(reinterpret_cast<const long long*>(a.counts) + b);
    return (int)max(min(n, (long long)a.tokens), 0LL);
}
// Whether the query at position p sees row j >= 0 of its cache (window is at least 1 here; no window: 2^30).
__device__ __forceinline__ bool attn_sees(int p, int j, int window, int sinks) { return j <= p && (j > p - window || j < sinks); }

// Rows of a cache that the queries at positions p_lo .. p_hi see between them: [0, s_end) and [w_start, w_end), which do not overlap.
struct AttnRange { int s_end, w_start, w_end; };
__device__ __forceinline__ AttnRange attn_range(int p_lo, int p_hi, int window, int sinks, int max_seq) {
    AttnRange r;
    r.w_end = max(0, min(p_hi + 1, max_seq));
    r.w_start = max(0, p_lo - window + 1);
    r.s_end = max(0, min(sinks, r.w_end));
    if (r.w_start <= r.s_end) r.w_start = r.s_end = 0;
    r.w_end = max(r.w_end, r.w_start);
    return r;
}

// One query row by one warp, a few keys at a time, skipping the rows that it does not see.  The tiles of both kernels multiply weights of zero with whatever
// the rows hold that other queries of the tile see: where that gives a NaN or an infinity the row is done again here.  A lane owns HD / 32 dims.
// Whether there is anything to do is looked at first, since one such value in a row that all see (a sink) sends every row of a long prompt here:
//   * the dims that came out finite are right, and so is an infinity in fp16: 2^8 times the largest fp16 number, 2^29 times over, is far from fp32's end, so it
//     is that of values which the row sees, with weights that are not zero, and of one sign;
//   * a dim in which the row sees a NaN is one.  Those are looked for without the scores, a few rows of V at a time.
// One prompt of 8192, 32 / 8 heads of 128, window 4096 (0.36 ms) with one value per key head that is not finite: in a sink 0.57 (NaN) and 0.47 ms (infinity
// in fp16), 231 where every row was done again one key at a time; in the middle 32 and 21 ms, 176 so; an infinity in bf16, whose rows are all done again, 131.
template <typename T, int HD>
__device__ __noinline__ void attn_row_again(const b200gptq_attn_args& a, int b, int t, int head, int p, int d0, int d1) {
    constexpr int D = HD / 32, kAgain = 8;    // keys whose loads are on their way at once
    const int lane = threadIdx.x & 31, kh = head / (a.heads / a.kv_heads), window = a.window ? a.window : 1 << 30;
    T* out = static_cast<T*>(a.out) + b * a.out_stride[0] + t * a.out_stride[1] + head * a.out_stride[2];
    const AttnRange r = attn_range(p, p, window, a.sinks, a.max_seq);
    const T *kp = static_cast<const T*>(a.k_prefix) + kh * a.k_prefix_stride[0] + lane * D,
            *vp = static_cast<const T*>(a.v_prefix) + kh * a.v_prefix_stride[0] + lane * D;
    const T *kc = static_cast<const T*>(a.k_cache) + b * a.k_stride[0] + kh * a.k_stride[1] + lane * D,
            *vc = static_cast<const T*>(a.v_cache) + b * a.v_stride[0] + kh * a.v_stride[1] + lane * D;
    unsigned open = 0;                        // dims of the lane that are not known yet
#pragma unroll
    for (int e = 0; e < D; ++e) {
        const int d = lane * D + e;
        const float f = d >= d0 && d < d1 ? Half<T>::wide(out[d]) : 0.f;
        if (isnan(f) || (isinf(f) && !std::is_same<T, __half>::value)) open |= 1u << e;
    }
    auto known = [&](const T* v, long long stride, int j, int end) {
        for (; __any_sync(0xffffffffu, open) && j < end; j += kAgain)
#pragma unroll
            for (int u = 0; u < kAgain; ++u) {
                const uint32_t* row = reinterpret_cast<const uint32_t*>(v + min(j + u, end - 1) * stride);
#pragma unroll
                for (int e = 0; e < D; e += 2) {
                    const float2 f = Half<T>::unpack(row[e / 2]);
                    if (isnan(f.x)) open &= ~(1u << e);
                    if (isnan(f.y)) open &= ~(2u << e);
                }
            }
    };
    known(vp, a.v_prefix_stride[1], 0, a.prefix);
    known(vc, a.v_stride[2], 0, r.s_end);
    known(vc, a.v_stride[2], r.w_start, r.w_end);
    if (!__any_sync(0xffffffffu, open)) return;
    const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + t * a.q_stride[1] + head * a.q_stride[2] + lane * D;
    float qf[D], acc[D], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < D; ++e) { qf[e] = Half<T>::wide(q[e]) * a.scale * kLog2e; acc[e] = 0.f; }
    auto keys = [&](const T* k, long long k_stride, const T* v, long long v_stride, int j, int end) {
        for (; j < end; j += kAgain) {
            uint32_t kw[kAgain][D / 2], vw[kAgain][D / 2];
            float s[kAgain], up = m;
#pragma unroll
            for (int u = 0; u < kAgain; ++u) {
                const long long at = min(j + u, end - 1);
#pragma unroll
                for (int e = 0; e < D / 2; ++e) {
                    kw[u][e] = reinterpret_cast<const uint32_t*>(k + at * k_stride)[e];
                    vw[u][e] = reinterpret_cast<const uint32_t*>(v + at * v_stride)[e];
                }
            }
#pragma unroll
            for (int u = 0; u < kAgain; ++u) {
                s[u] = 0.f;
#pragma unroll
                for (int e = 0; e < D; e += 2) {
                    const float2 f = Half<T>::unpack(kw[u][e / 2]);
                    s[u] = fmaf(qf[e + 1], f.y, fmaf(qf[e], f.x, s[u]));
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
#pragma unroll
                for (int u = 0; u < kAgain; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], o);
#pragma unroll
            for (int u = 0; u < kAgain; ++u)
                if (j + u < end) up = fmaxf(up, s[u]);
            const float safe = up == -INFINITY ? 0.f : up, corr = exp2_fast(m - safe);
            m = up;
            l *= corr;
#pragma unroll
            for (int e = 0; e < D; ++e) acc[e] *= corr;
#pragma unroll
            for (int u = 0; u < kAgain; ++u)
                if (j + u < end) {
                    const float w = exp2_fast(s[u] - safe);
                    l += w;
#pragma unroll
                    for (int e = 0; e < D; e += 2) {
                        const float2 f = Half<T>::unpack(vw[u][e / 2]);
                        acc[e] = fmaf(w, f.x, acc[e]);
                        acc[e + 1] = fmaf(w, f.y, acc[e + 1]);
                    }
                }
        }
    };
    keys(kp, a.k_prefix_stride[1], vp, a.v_prefix_stride[1], 0, a.prefix);
    keys(kc, a.k_stride[2], vc, a.v_stride[2], 0, r.s_end);
    keys(kc, a.k_stride[2], vc, a.v_stride[2], r.w_start, r.w_end);
#pragma unroll
    for (int e = 0; e < D; ++e) {
        if (open >> e & 1u) out[lane * D + e] = Half<T>::round(l != 0.f ? acc[e] / l : 0.f);       // (a NaN stays one)
    }
}

}  // namespace b200gptq
