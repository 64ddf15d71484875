// b200gptq_cache_write and b200gptq_cache_read: a KV cache held in 4 bits, see include/b200gptq.h.
//
//   zero = min x,  scale = (max x - min x) / 15,  code = round((x - zero) / scale);   value = zero + scale * code
//
// Four lanes share a row: lane c has 8 dims of each 32, which are the codes of adjacent words (16 bytes of the row, 8 for 64 dims), 16 bytes of 16-bit values at a
// time. They meet in two shuffles per group for its minimum and maximum, of pairs of 16-bit numbers. A code is first taken from the product with 1 / scale, which
// is off by less than 2^-18, and divided out only where that is nearer than that to the middle between two codes.
// Bound by the bytes of long prompts and by the launch for a decode step.  Measured: a prompt of 8192, 32 / 8 heads of 128, 214 MB in 41.6 us, 5.1 TB/s and 62 % of the
// issue slots (a lane for each word, 8 bytes at a time, 94 us; two rows for each four lanes 86, where one took 70); 16 texts of 900 to 15900 read back, 705 MB in 116 us, 6.1 TB/s.
#include <algorithm>

#include "attn4.h"
#include "cache4.cuh"

namespace b200gptq {
namespace {

constexpr int kThreads = 256;

struct WriteDivisors { Divisor rows, tokens; };

template <typename T> __device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = Half<T>::unpack(w[i]);
        x[2 * i] = f.x; x[2 * i + 1] = f.y;
    }
}
template <typename T> __device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    return make_uint4(Half<T>::pack(x[0], x[1]), Half<T>::pack(x[2], x[3]), Half<T>::pack(x[4], x[5]), Half<T>::pack(x[6], x[7]));
}
template <int N> struct Words { uint32_t w[N]; };                 // 4, 8 or 16 bytes
template <int N> __device__ __forceinline__ Words<N> load_words(const void* at) {
    Words<N> r;
    if constexpr (N == 4) { const uint4 v = __ldcg(static_cast<const uint4*>(at)); r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w; }
    else if constexpr (N == 2) { const uint2 v = __ldcg(static_cast<const uint2*>(at)); r.w[0] = v.x; r.w[1] = v.y; }
    else r.w[0] = __ldcg(static_cast<const unsigned*>(at));
    return r;
}
template <int N> __device__ __forceinline__ void store_words(void* at, const Words<N>& r) {
    if constexpr (N == 4) *static_cast<uint4*>(at) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
    else if constexpr (N == 2) *static_cast<uint2*>(at) = make_uint2(r.w[0], r.w[1]);
    else *static_cast<uint32_t*>(at) = r.w[0];
}
// The value of a code.  (-65504 + 15 scales is 65536 where the scale was rounded up: not an infinity in fp16.)
template <typename T> constexpr float kLargest = std::is_same<T, __half>::value ? 65504.f : 3.38953139e38f;
template <typename T> __device__ __forceinline__ float value_of(unsigned code, float scale, float zero) {
    const float x = fmaf((float)code, scale, zero);
    return x > kLargest<T> ? kLargest<T> : x;                     // (the sum of zero, which is no smaller than -top, and of something that is not negative)
}

// The smaller or larger of pairs of 16-bit numbers; a NaN where one of them is one.
template <typename T> struct Pair;
template <> struct Pair<__half> { typedef __half2 type; };
template <> struct Pair<__nv_bfloat16> { typedef __nv_bfloat162 type; };
template <typename T> __device__ __forceinline__ uint32_t lower2(uint32_t a, uint32_t b) {
    using P = typename Pair<T>::type;
    const P r = __hmin2_nan(*reinterpret_cast<const P*>(&a), *reinterpret_cast<const P*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename T> __device__ __forceinline__ uint32_t upper2(uint32_t a, uint32_t b) {
    using P = typename Pair<T>::type;
    const P r = __hmax2_nan(*reinterpret_cast<const P*>(&a), *reinterpret_cast<const P*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
constexpr float kRound = 12582912.f;          // 1.5 2^23: a number below 2^22 that is added to it is rounded to a whole one, ties to even

// A lane's part of a row.  Rows: for each token the key heads, the value heads and, where queries are rotated, the query heads.
template <typename T, int HD> struct WriteRow {
    static constexpr int Y = HD / 32, HH = HD / 64;
    unsigned b;
    int t, head, c, p;
    bool is_k, is_v, is_q, there, valid;
    uint4 raw[Y];
    uint2 cos_w[Y], sin_w[Y];

    __device__ __forceinline__ void place(const b200gptq_cache_write_args& a, unsigned row, unsigned rows, const WriteDivisors& by) {
        c = threadIdx.x & 3;
        there = row < rows;
        row = min(row, rows - 1);
        const unsigned token = over(row, by.rows);
        const int per = 2 * a.cache.kv_heads + (a.q ? a.heads : 0), j = (int)(row - token * per), kv = a.cache.kv_heads;
        b = over(token, by.tokens);
        t = (int)(token - b * a.tokens);
        is_k = j < kv; is_v = !is_k && j < 2 * kv; is_q = !is_k && !is_v;
        head = is_k ? j : is_v ? j - kv : j - 2 * kv;
    }
    __device__ __forceinline__ void fetch(const b200gptq_cache_write_args& a) {
        const long long start = __ldcg(reinterpret_cast<const long long*>(a.pos) + (a.pos_each ? b : 0));
        const long long count = a.counts ? __ldcg(reinterpret_cast<const long long*>(a.counts) + b) : a.tokens;
        const T* src = (is_k   ? static_cast<const T*>(a.k) + b * a.k_stride[0] + t * a.k_stride[1] + head * a.k_stride[2]
                        : is_v ? static_cast<const T*>(a.v) + b * a.v_stride[0] + t * a.v_stride[1] + head * a.v_stride[2]
                               : static_cast<const T*>(a.q) + b * a.q_stride[0] + t * a.q_stride[1] + head * a.q_stride[2]) + 8 * c;
#pragma unroll
        for (int y = 0; y < Y; ++y) raw[y] = *reinterpret_cast<const uint4*>(src + 32 * y);       // (a row of padding is read too: it is there)
        // (a position near the end of 64 bits must not wrap around to one in the cache)
        valid = there && t < count && start < a.cache.max_seq && start >= -(long long)t && start + t < a.cache.max_seq && (!a.cos_t || start + t < a.angles);
        p = valid ? (int)(start + t) : 0;
        if (a.cos_t && !is_v) {
            const T *cos_t = static_cast<const T*>(a.cos_t) + (long long)p * (HD / 2) + 4 * c, *sin_t = static_cast<const T*>(a.sin_t) + (long long)p * (HD / 2) + 4 * c;
#pragma unroll
            for (int y = 0; y < Y; ++y) { cos_w[y] = *reinterpret_cast<const uint2*>(cos_t + 16 * y); sin_w[y] = *reinterpret_cast<const uint2*>(sin_t + 16 * y); }
        }
    }
    __device__ __forceinline__ void turn() {
#pragma unroll
        for (int y = 0; y < Y; ++y) {
            const uint32_t cs[2] = {cos_w[y].x, cos_w[y].y}, sn[2] = {sin_w[y].x, sin_w[y].y};
            float x[8];
            unpack8<T>(raw[y], x);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float2 f = Half<T>::unpack(cs[i]), s = Half<T>::unpack(sn[i]);
                float* z = x + 4 * i;
                // (products of 16-bit numbers are exact in fp32, so it does not matter whether they are fused with the sum)
                const float z0 = z[0] * f.x - z[1] * s.x, z1 = z[0] * s.x + z[1] * f.x, z2 = z[2] * f.y - z[3] * s.y, z3 = z[2] * s.y + z[3] * f.y;
                z[0] = z0; z[1] = z1; z[2] = z2; z[3] = z3;
            }
            raw[y] = pack8<T>(x);
        }
    }
    template <int GS> __device__ __forceinline__ void store(const b200gptq_cache_write_args& a) {
        constexpr int NG = HD / GS;
        if (a.cos_t && !is_v) turn();
        if (valid && is_q) {
            T* dst = static_cast<T*>(a.q_out) + b * a.q_out_stride[0] + t * a.q_out_stride[1] + head * a.q_out_stride[2] + 8 * c;
#pragma unroll
            for (int y = 0; y < Y; ++y) *reinterpret_cast<uint4*>(dst + 32 * y) = raw[y];
        }
        const bool writes = valid && !is_q;
        if (!__any_sync(0xffffffffu, writes)) return;
        Words<2 * HH> word = {};                  // of words (HD / 64) (2 c + x) + h of the row: HH x + h
        Words<NG> constants;
        T* out = static_cast<T*>(is_k ? a.k_out : a.v_out);
        if (out && writes)
            out += (is_k ? b * a.k_out_stride[0] + t * a.k_out_stride[1] + head * a.k_out_stride[2] : b * a.v_out_stride[0] + t * a.v_out_stride[1] + head * a.v_out_stride[2]) + 8 * c;
#pragma unroll
        for (int n = 0; n < NG; ++n) {            // a group: 32 dims or 64
            constexpr int SPAN = GS / 32;
            uint32_t lo = raw[SPAN * n].x, hi = lo;
#pragma unroll
            for (int y = 0; y < SPAN; ++y) {
                const uint4 v = raw[SPAN * n + y];
                lo = lower2<T>(lower2<T>(lo, v.x), lower2<T>(lower2<T>(v.y, v.z), v.w));
                hi = upper2<T>(upper2<T>(hi, v.x), upper2<T>(upper2<T>(v.y, v.z), v.w));
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                lo = lower2<T>(lo, __shfl_xor_sync(0xffffffffu, lo, o));
                hi = upper2<T>(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            }
            const float2 lo2 = Half<T>::unpack(lower2<T>(lo, lo >> 16 | lo << 16)), hi2 = Half<T>::unpack(upper2<T>(hi, hi >> 16 | hi << 16));
            float scale = Half<T>::wide(Half<T>::round(__fdiv_rn(__fsub_rn(hi2.x, lo2.x), 15.f))), zero = lo2.x;
            if (!isfinite(scale)) scale = zero = __int_as_float(0x7fc00000);
            constants.w[n] = Half<T>::pack(scale, zero);
            // (a scale of zero: all codes are 0; one that is subnormal in fp32, bf16 below 2^-126, has no reciprocal there)
            const float inverse = scale > 0.f ? __frcp_rn(scale) : 0.f;
            const bool high = fmaf(15.f, scale, zero) > kLargest<T> || !(inverse < INFINITY);
#pragma unroll
            for (int y = 0; y < SPAN; ++y) {
                const int at = SPAN * n + y, h = at >> 1;
                float x[8], code[8], off = 0.f;
                unpack8<T>(raw[at], x);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float d = __fsub_rn(x[e], zero), q = fminf(d * inverse, 15.f);
                    code[e] = __fsub_rn(__fadd_rn(q, kRound), kRound);
                    off = fmaxf(off, fabsf(q - code[e]));
                }
                if (off > 0.5f - 0x1p-18f || high) {           // near the middle between two codes, or a range that is not ordinary: by the definition
#pragma unroll
                    for (int e = 0; e < 8; ++e) code[e] = scale > 0.f ? fminf(rintf(__fdiv_rn(__fsub_rn(x[e], zero), scale)), 15.f) : 0.f;
                }
                // fields of dims 0, 2 (of four), 1, 3: 0, 1, 4, 5; in the second half of 64 dims two further on
#pragma unroll
                for (int x4 = 0; x4 < 2; ++x4) {
                    const float *c4 = code + 4 * x4;
                    const unsigned two = __float_as_uint(__fadd_rn(fmaf(c4[2], 16.f, c4[0]), kRound)) & 0xffu, other = __float_as_uint(__fadd_rn(fmaf(c4[3], 16.f, c4[1]), kRound)) & 0xffu;
                    word.w[HH * x4 + h] |= (two | other << 16) << (at & 1) * 8;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = fmaf(code[e], scale, zero);
                if (high)
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = value_of<T>((unsigned)code[e], scale, zero);
                if (out && writes) *reinterpret_cast<uint4*>(out + 32 * at) = pack8<T>(x);
            }
        }
        if (!writes) return;
        const b200gptq_cache4& cache = a.cache;
        uint8_t* codes = static_cast<uint8_t*>(is_k ? cache.k : cache.v) + (is_k ? b * cache.k_stride[0] + head * cache.k_stride[1] + p * cache.k_stride[2]
                                                                                 : b * cache.v_stride[0] + head * cache.v_stride[1] + p * cache.v_stride[2]);
        store_words<2 * HH>(codes + 8 * HH * c, word);
        if (c == 0)
            store_words<NG>(static_cast<T*>(is_k ? cache.k_scales : cache.v_scales) + (is_k ? b * cache.k_scale_stride[0] + head * cache.k_scale_stride[1] + p * cache.k_scale_stride[2]
                                                                                            : b * cache.v_scale_stride[0] + head * cache.v_scale_stride[1] + p * cache.v_scale_stride[2]),
                            constants);
    }
};

template <typename T, int HD, int GS>
__global__ void __launch_bounds__(kThreads)
cache_write_kernel(const __grid_constant__ b200gptq_cache_write_args a, unsigned rows, const __grid_constant__ WriteDivisors by) {
    asm volatile("griddepcontrol.launch_dependents;");
    WriteRow<T, HD> row;
    row.place(a, blockIdx.x * (unsigned)(kThreads / 4) + threadIdx.x / 4, rows, by);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    row.fetch(a);
    row.template store<GS>(a);
}

// Lane c's part of a row back in 16 bits.
template <typename T, int HD, int GS> __device__ __forceinline__ void unpack_row(const Words<HD / 32>& word, const Words<HD / GS>& constants, T* out, int c) {
    constexpr int HH = HD / 64;
#pragma unroll
    for (int y = 0; y < HD / 32; ++y) {
        const float2 of = Half<T>::unpack(constants.w[GS == 32 ? y : y >> 1]);        // (scale, zero)
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = value_of<T>(word.w[HH * (e >> 2) + (y >> 1)] >> 4 * ((y & 1) * 2 + (e & 1) * 4 + (e & 3) / 2) & 15u, of.x, of.y);
        *reinterpret_cast<uint4*>(out + 32 * y + 8 * c) = pack8<T>(x);
    }
}

// A CTA takes kRowsPerCta rows of the keys or the values of one sequence and head; a lane kDeep of them, all asked for at once.
constexpr int kDeep = 4, kRowsPerCta = kThreads / 4 * kDeep;
template <typename T, int HD, int GS, typename From, typename Out>
__device__ __forceinline__ void read_rows(const b200gptq_cache4& cache, unsigned b, int head, bool is_k, int j0, From from, Out out) {
    const int c = threadIdx.x & 3;
    const uint8_t* codes = static_cast<const uint8_t*>(is_k ? cache.k : cache.v) + (is_k ? b * cache.k_stride[0] + head * cache.k_stride[1] : b * cache.v_stride[0] + head * cache.v_stride[1]);
    const T* constants = static_cast<const T*>(is_k ? cache.k_scales : cache.v_scales) +
                         (is_k ? b * cache.k_scale_stride[0] + head * cache.k_scale_stride[1] : b * cache.v_scale_stride[0] + head * cache.v_scale_stride[1]);
    const long long stride = is_k ? cache.k_stride[2] : cache.v_stride[2], scale_stride = is_k ? cache.k_scale_stride[2] : cache.v_scale_stride[2];
    Words<HD / 32> word[kDeep];
    Words<HD / GS> of[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
        const int j = j0 + i * (kThreads / 4);
        const int row = from(j);                  // of the cache; -1: none
        if (row < 0) continue;
        word[i] = load_words<HD / 32>(codes + row * stride + HD / 8 * c);
        of[i] = load_words<HD / GS>(constants + row * scale_stride);
    }
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
        const int j = j0 + i * (kThreads / 4);
        if (from(j) >= 0) unpack_row<T, HD, GS>(word[i], of[i], out(j), c);
    }
}

template <typename T, int HD, int GS>
__global__ void __launch_bounds__(kThreads)
cache_read_kernel(const __grid_constant__ b200gptq_cache_read_args a, unsigned chunks, const __grid_constant__ Divisor by_chunks, const __grid_constant__ Divisor by_heads) {
    asm volatile("griddepcontrol.launch_dependents;");
    const unsigned which = over(blockIdx.x, by_chunks), pair = which >> 1, b = over(pair, by_heads);
    const int head = (int)(pair - b * a.cache.kv_heads), j0 = (int)((blockIdx.x - which * chunks) * kRowsPerCta + threadIdx.x / 4);
    const bool is_k = !(which & 1);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long length = a.lengths ? min(__ldcg(reinterpret_cast<const long long*>(a.lengths) + b), (long long)a.cache.max_seq) : a.cache.max_seq;
    T* out = static_cast<T*>(is_k ? a.k_out : a.v_out) + (is_k ? b * a.k_out_stride[0] + head * a.k_out_stride[1] : b * a.v_out_stride[0] + head * a.v_out_stride[1]);
    const long long stride = is_k ? a.k_out_stride[2] : a.v_out_stride[2];
    read_rows<T, HD, GS>(a.cache, b, head, is_k, j0, [&](int j) { return j < length ? j : -1; }, [&](int j) { return out + j * stride; });
}

// For prompts: the rows that the tokens see between them, into k and v of `rows` rows (attn4_read_back).
template <typename T, int HD, int GS>
__global__ void __launch_bounds__(kThreads)
cache_read_seen_kernel(const __grid_constant__ Attn4Args a, T* __restrict__ k, T* __restrict__ v, int rows, long long* __restrict__ pos, unsigned chunks, const __grid_constant__ Divisor by_chunks,
                       const __grid_constant__ Divisor by_heads) {
    asm volatile("griddepcontrol.launch_dependents;");
    const unsigned which = over(blockIdx.x, by_chunks), pair = which >> 1, b = over(pair, by_heads);
    const int head = (int)(pair - b * a.cache.kv_heads), j0 = (int)((blockIdx.x - which * chunks) * kRowsPerCta + threadIdx.x / 4);
    const bool is_k = !(which & 1);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int p0 = attn_pos(a.attn, b), count = attn_count(a.attn, b);
    const AttnRange r = attn_range(p0, p0 + count - 1, a.attn.window ? a.attn.window : 1 << 30, a.attn.sinks, a.cache.max_seq);
    const int end = count ? min(r.w_end, a.cache.max_seq) : 0;
    // (There are as many rows as a window, the tokens behind its first one and the sinks make up, so the first row of the window does not come to lie before the sinks' end, and where
    // the two meet nothing has moved.)
    const int up = max(0, min(p0 + count, a.cache.max_seq) - rows);
    if (pos && threadIdx.x == 0 && head == 0 && is_k && blockIdx.x == which * chunks) pos[b] = p0 - up;
    T* out = (is_k ? k : v) + ((long long)b * a.cache.kv_heads + head) * rows * HD;
    read_rows<T, HD, GS>(
        a.cache, b, head, is_k, j0,
        [&](int j) {
            const int from = j < r.s_end ? j : j + up;
            return j < rows && from < end && (from < r.s_end || from >= r.w_start) ? from : -1;
        },
        [&](int j) { return out + (long long)j * HD; });
}

template <typename... KArgs, typename... Args>
int launch(void (*kernel)(KArgs...), dim3 grid, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = attn_pdl_enabled() ? 1 : 0;
    B200GPTQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...));
    return B200GPTQ_OK;
}

template <typename T, int HD, int GS>
int write(const b200gptq_cache_write_args& a, cudaStream_t stream) {
    const long long per = 2LL * a.cache.kv_heads + (a.q ? a.heads : 0), rows = per * a.cache.batch * a.tokens;
    const WriteDivisors by = {Divisor(per), Divisor(a.tokens)};
    return launch(cache_write_kernel<T, HD, GS>, dim3((unsigned)((rows * 4 + kThreads - 1) / kThreads)), stream, a, (unsigned)rows, by);
}

template <typename T, int HD, int GS>
int read(const b200gptq_cache_read_args& a, cudaStream_t stream) {
    const long long chunks = (a.cache.max_seq + kRowsPerCta - 1) / kRowsPerCta, ctas = 2LL * a.cache.batch * a.cache.kv_heads;
    if (ctas > 0x7fffffff / chunks) return B200GPTQ_ERR_TOO_LARGE;
    return launch(cache_read_kernel<T, HD, GS>, dim3((unsigned)(ctas * chunks)), stream, a, (unsigned)chunks, Divisor(chunks), Divisor(a.cache.kv_heads));
}

template <typename T, int HD, int GS>
int read_seen(const Attn4Args& a, void* k, void* v, int rows, int64_t* pos, cudaStream_t stream) {
    const long long chunks = (rows + kRowsPerCta - 1) / kRowsPerCta, ctas = 2LL * a.cache.batch * a.cache.kv_heads;
    if (ctas > 0x7fffffff / chunks) return B200GPTQ_ERR_TOO_LARGE;
    return launch(cache_read_seen_kernel<T, HD, GS>, dim3((unsigned)(ctas * chunks)), stream, a, static_cast<T*>(k), static_cast<T*>(v), rows, reinterpret_cast<long long*>(pos), (unsigned)chunks,
                  Divisor(chunks), Divisor(a.cache.kv_heads));
}

template <typename T, typename Args> int by_shape(const Args& a, cudaStream_t stream, int (*const (&run)[2][2])(const Args&, cudaStream_t)) {
    return run[a.cache.hd == 128][a.cache.group == 64](a, stream);
}

uintptr_t bits_of(const void* p, const int64_t (&stride)[3]) { return p ? reinterpret_cast<uintptr_t>(p) | (uintptr_t)(2 * (stride[0] | stride[1] | stride[2])) : 0; }

}  // namespace

int attn4_read_back(const Attn4Args& a, void* k, void* v, int rows, int64_t* pos, cudaStream_t s) {
    using F = int (*)(const Attn4Args&, void*, void*, int, int64_t*, cudaStream_t);
    static const F run[2][2][2] = {{{read_seen<__half, 64, 32>, read_seen<__half, 64, 64>}, {read_seen<__half, 128, 32>, read_seen<__half, 128, 64>}},
                                   {{read_seen<__nv_bfloat16, 64, 32>, read_seen<__nv_bfloat16, 64, 64>}, {read_seen<__nv_bfloat16, 128, 32>, read_seen<__nv_bfloat16, 128, 64>}}};
    return run[a.cache.dtype == B200GPTQ_BF16][a.cache.hd == 128][a.cache.group == 64](a, k, v, rows, pos, s);
}

}  // namespace b200gptq

using namespace b200gptq;

extern "C" {

B200GPTQ_API int b200gptq_cache_write(const b200gptq_cache_write_args* args, void* stream) {
    if (!args) return B200GPTQ_ERR_NULL_POINTER;
    const b200gptq_cache_write_args& a = *args;
    int st = cache4_check(a.cache);
    if (st != B200GPTQ_OK) return st;
    if (a.tokens < 1 || (a.q && a.heads < 1) || (a.cos_t && a.angles < 1)) return B200GPTQ_ERR_SHAPE;
    if (!a.k || !a.v || !a.pos || !a.q != !a.q_out || !a.cos_t != !a.sin_t || (a.q && !a.cos_t)) return B200GPTQ_ERR_NULL_POINTER;
    // (rows are numbered in 31 bits)
    if (a.tokens > kCacheMost || (a.q && a.heads > kCacheMost)) return B200GPTQ_ERR_TOO_LARGE;
    const double rows = (2.0 * a.cache.kv_heads + (a.q ? a.heads : 0)) * a.cache.batch * a.tokens;
    if (rows > 2147483647.0) return B200GPTQ_ERR_TOO_LARGE;
    st = cache4_check_memory(a.cache);
    if (st != B200GPTQ_OK) return st;
    if ((bits_of(a.k, a.k_stride) | bits_of(a.v, a.v_stride) | bits_of(a.q, a.q_stride) | bits_of(a.q_out, a.q_out_stride) | bits_of(a.k_out, a.k_out_stride) |
         bits_of(a.v_out, a.v_out_stride) | reinterpret_cast<uintptr_t>(a.cos_t) | reinterpret_cast<uintptr_t>(a.sin_t)) & 15u ||
        (reinterpret_cast<uintptr_t>(a.pos) | reinterpret_cast<uintptr_t>(a.counts)) & 7u)
        return B200GPTQ_ERR_ALIGNMENT;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a.cache.dtype == B200GPTQ_F16) return by_shape<__half>(a, s, {{write<__half, 64, 32>, write<__half, 64, 64>}, {write<__half, 128, 32>, write<__half, 128, 64>}});
    return by_shape<__nv_bfloat16>(a, s, {{write<__nv_bfloat16, 64, 32>, write<__nv_bfloat16, 64, 64>}, {write<__nv_bfloat16, 128, 32>, write<__nv_bfloat16, 128, 64>}});
}

B200GPTQ_API int b200gptq_cache_read(const b200gptq_cache_read_args* args, void* stream) {
    if (!args) return B200GPTQ_ERR_NULL_POINTER;
    const b200gptq_cache_read_args& a = *args;
    int st = cache4_check(a.cache);
    if (st != B200GPTQ_OK) return st;
    if (!a.k_out || !a.v_out) return B200GPTQ_ERR_NULL_POINTER;
    st = cache4_check_memory(a.cache);
    if (st != B200GPTQ_OK) return st;
    if ((bits_of(a.k_out, a.k_out_stride) | bits_of(a.v_out, a.v_out_stride)) & 15u || reinterpret_cast<uintptr_t>(a.lengths) & 7u) return B200GPTQ_ERR_ALIGNMENT;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a.cache.dtype == B200GPTQ_F16) return by_shape<__half>(a, s, {{read<__half, 64, 32>, read<__half, 64, 64>}, {read<__half, 128, 32>, read<__half, 128, 64>}});
    return by_shape<__nv_bfloat16>(a, s, {{read<__nv_bfloat16, 64, 32>, read<__nv_bfloat16, 64, 64>}, {read<__nv_bfloat16, 128, 32>, read<__nv_bfloat16, 128, 64>}});
}

}  // extern "C"
