// b200gptq_cache_write and b200gptq_cache_read: a KV cache held in 4 bits, see include/b200gptq.h.
//
//   zero = min x,  scale = (max x - min x) / 15,  code = round((x - zero) / scale);   value = zero + scale * code
//
// One word (eight codes) per lane: HD / 8 lanes share a row, and since a word's fields come from two runs of four dims (cache4.cuh) a lane reads two times 8
// bytes and the 8 lanes of a group meet in three shuffles for its minimum and maximum.  A row's words, constants and values leave in whole sectors.
// Bound by the bytes of long prompts and by the launch for a decode step.
#include <algorithm>

#include "attn4.h"
#include "cache4.cuh"

namespace b200gptq {
namespace {

constexpr int kThreads = 256;

struct WriteDivisors { Divisor rows, tokens; };

template <typename T> __device__ __forceinline__ void unpack4(uint2 v, float* x) {
    const float2 a = Half<T>::unpack(v.x), b = Half<T>::unpack(v.y);
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}
template <typename T> __device__ __forceinline__ uint2 pack4(const float* x) { return make_uint2(Half<T>::pack(x[0], x[1]), Half<T>::pack(x[2], x[3])); }
// The value of a code.  (-65504 + 15 scales is 65536 where the scale was rounded up: not an infinity in fp16.)
template <typename T> __device__ __forceinline__ float value_of(unsigned code, float scale, float zero) {
    constexpr float top = std::is_same<T, __half>::value ? 65504.f : 3.38953139e38f;
    const float x = fmaf((float)code, scale, zero);
    return x > top ? top : x;                     // (the sum of zero, which is no smaller than -top, and of something that is not negative)
}

// Rows: for each token the key heads, the value heads and, where queries are rotated, the query heads.
template <typename T, int HD, int GS>
__global__ void __launch_bounds__(kThreads)
cache_write_kernel(const __grid_constant__ b200gptq_cache_write_args a, unsigned rows, const __grid_constant__ WriteDivisors by) {
    constexpr int LANES = HD / 8;
    asm volatile("griddepcontrol.launch_dependents;");
    const unsigned row = (unsigned)((blockIdx.x * (unsigned long long)kThreads + threadIdx.x) / LANES);
    const int lane = threadIdx.x & 31, u = lane % LANES, g = u & 7, h = u >> 3, d = 64 * h + 4 * g;
    const unsigned token = over(min(row, rows - 1), by.rows), b = over(token, by.tokens);
    const int per = 2 * a.cache.kv_heads + (a.q ? a.heads : 0), j = (int)(min(row, rows - 1) - token * per), t = (int)(token - b * a.tokens), kv = a.cache.kv_heads;
    const bool is_k = j < kv, is_v = !is_k && j < 2 * kv, is_q = !is_k && !is_v;
    const int head = is_k ? j : is_v ? j - kv : j - 2 * kv;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long start = __ldcg(reinterpret_cast<const long long*>(a.pos) + (a.pos_each ? b : 0));
    const long long count = a.counts ? __ldcg(reinterpret_cast<const long long*>(a.counts) + b) : a.tokens;
    // (a position near the end of 64 bits must not wrap around to one in the cache)
    const bool valid = row < rows && t < count && start < a.cache.max_seq && start >= -(long long)t && start + t < a.cache.max_seq && (!a.cos_t || start + t < a.angles);
    const int p = valid ? (int)(start + t) : 0;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (valid) {
        const T* src = is_k   ? static_cast<const T*>(a.k) + b * a.k_stride[0] + t * a.k_stride[1] + head * a.k_stride[2]
                       : is_v ? static_cast<const T*>(a.v) + b * a.v_stride[0] + t * a.v_stride[1] + head * a.v_stride[2]
                              : static_cast<const T*>(a.q) + b * a.q_stride[0] + t * a.q_stride[1] + head * a.q_stride[2];
        unpack4<T>(*reinterpret_cast<const uint2*>(src + d), x);
        unpack4<T>(*reinterpret_cast<const uint2*>(src + d + 32), x + 4);
        if (a.cos_t && !is_v) {
            const T *cos_t = static_cast<const T*>(a.cos_t) + (long long)p * (HD / 2) + d / 2, *sin_t = static_cast<const T*>(a.sin_t) + (long long)p * (HD / 2) + d / 2;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float2 c = Half<T>::unpack(*reinterpret_cast<const uint32_t*>(cos_t + 16 * i)), s = Half<T>::unpack(*reinterpret_cast<const uint32_t*>(sin_t + 16 * i));
                float* y = x + 4 * i;
                // (products of 16-bit numbers are exact in fp32, so it does not matter whether they are fused with the sum)
                const float y0 = y[0] * c.x - y[1] * s.x, y1 = y[0] * s.x + y[1] * c.x, y2 = y[2] * c.y - y[3] * s.y, y3 = y[2] * s.y + y[3] * c.y;
                y[0] = y0; y[1] = y1; y[2] = y2; y[3] = y3;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = Half<T>::wide(Half<T>::round(x[i]));
        }
    }
    if (valid && is_q) {
        T* dst = static_cast<T*>(a.q_out) + b * a.q_out_stride[0] + t * a.q_out_stride[1] + head * a.q_out_stride[2] + d;
        *reinterpret_cast<uint2*>(dst) = pack4<T>(x);
        *reinterpret_cast<uint2*>(dst + 32) = pack4<T>(x + 4);
    }
    // ---- range of each group: the lane's four dims of it (eight, where both runs are in one group), then the 8 lanes ----
    float lo[2], hi[2], scale[2], zero[2];
    unsigned odd[2];                              // of the warp's lanes, those with a NaN or an infinity
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float* y = x + 4 * i;
        lo[i] = fminf(fminf(y[0], y[1]), fminf(y[2], y[3]));
        hi[i] = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
        bool finite = true;
#pragma unroll
        for (int e = 0; e < 4; ++e) finite = finite && isfinite(y[e]);
        odd[i] = __ballot_sync(0xffffffffu, !finite);
    }
    if constexpr (GS == 64) { lo[0] = fminf(lo[0], lo[1]); hi[0] = fmaxf(hi[0], hi[1]); odd[0] |= odd[1]; }
#pragma unroll
    for (int i = 0; i < (GS == 64 ? 1 : 2); ++i) {
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
            lo[i] = fminf(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], o));
            hi[i] = fmaxf(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], o));
        }
        scale[i] = Half<T>::wide(Half<T>::round(__fdiv_rn(__fsub_rn(hi[i], lo[i]), 15.f)));
        zero[i] = lo[i];
        if ((odd[i] >> (lane & ~7) & 0xffu) || !isfinite(scale[i])) scale[i] = zero[i] = __int_as_float(0x7fc00000);
    }
    if constexpr (GS == 64) { scale[1] = scale[0]; zero[1] = zero[0]; }
    if (!valid || is_q) return;
    unsigned code[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float s = scale[e / 4];
        code[e] = s > 0.f ? (unsigned)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[e], zero[e / 4]), s)), 0.f), 15.f) : 0u;
        x[e] = value_of<T>(code[e], s, zero[e / 4]);
    }
    const b200gptq_cache4& c = a.cache;
    uint8_t* codes = static_cast<uint8_t*>(is_k ? c.k : c.v) + (is_k ? b * c.k_stride[0] + head * c.k_stride[1] + p * c.k_stride[2]
                                                                     : b * c.v_stride[0] + head * c.v_stride[1] + p * c.v_stride[2]);
    reinterpret_cast<uint32_t*>(codes)[(HD / 64) * g + h] = cache4_word(code);
    if (g == 0) {
        T* constants = static_cast<T*>(is_k ? c.k_scales : c.v_scales) + (is_k ? b * c.k_scale_stride[0] + head * c.k_scale_stride[1] + p * c.k_scale_stride[2]
                                                                               : b * c.v_scale_stride[0] + head * c.v_scale_stride[1] + p * c.v_scale_stride[2]);
        if constexpr (GS == 64) reinterpret_cast<uint32_t*>(constants)[h] = Half<T>::pack(scale[0], zero[0]);
        else reinterpret_cast<uint2*>(constants)[h] = make_uint2(Half<T>::pack(scale[0], zero[0]), Half<T>::pack(scale[1], zero[1]));
    }
    T* out = static_cast<T*>(is_k ? a.k_out : a.v_out);
    if (out) {
        out += (is_k ? b * a.k_out_stride[0] + t * a.k_out_stride[1] + head * a.k_out_stride[2] : b * a.v_out_stride[0] + t * a.v_out_stride[1] + head * a.v_out_stride[2]) + d;
        *reinterpret_cast<uint2*>(out) = pack4<T>(x);
        *reinterpret_cast<uint2*>(out + 32) = pack4<T>(x + 4);
    }
}

// A row back in 16 bits, HD / 8 lanes (of which this is number u) a row.
template <typename T, int HD, int GS> __device__ __forceinline__ void read_row(const uint8_t* codes, const T* constants, T* out, int u) {
    constexpr int NG = HD / GS;
    const int g = u & 7, h = u >> 3;
    const uint32_t w = __ldcg(reinterpret_cast<const unsigned*>(codes) + (HD / 64) * g + h);
    float2 of[2];                                 // (scale, zero) of the two runs of dims
    of[0] = Half<T>::unpack(__ldcg(reinterpret_cast<const unsigned*>(constants) + h * NG / (HD / 64)));
    of[1] = GS == 64 ? of[0] : Half<T>::unpack(__ldcg(reinterpret_cast<const unsigned*>(constants) + 2 * h + 1));
    unsigned code[8];
    cache4_codes(w, code);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = value_of<T>(code[e], of[e / 4].x, of[e / 4].y);
    out += 64 * h + 4 * g;
    *reinterpret_cast<uint2*>(out) = pack4<T>(x);
    *reinterpret_cast<uint2*>(out + 32) = pack4<T>(x + 4);
}

// A CTA takes ROWS rows of the keys or the values of one sequence and head.
template <typename T, int HD, int GS>
__global__ void __launch_bounds__(kThreads)
cache_read_kernel(const __grid_constant__ b200gptq_cache_read_args a, unsigned chunks, const __grid_constant__ Divisor by_chunks, const __grid_constant__ Divisor by_heads) {
    constexpr int LANES = HD / 8, ROWS = kThreads / LANES;
    asm volatile("griddepcontrol.launch_dependents;");
    const b200gptq_cache4& c = a.cache;
    const unsigned which = over(blockIdx.x, by_chunks), pair = which >> 1, b = over(pair, by_heads);
    const int head = (int)(pair - b * c.kv_heads);
    const bool is_k = !(which & 1);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long length = a.lengths ? min(__ldcg(reinterpret_cast<const long long*>(a.lengths) + b), (long long)c.max_seq) : c.max_seq;
    const int j = (int)((blockIdx.x - which * chunks) * ROWS + threadIdx.x / LANES);
    if (j >= length) return;
    const uint8_t* codes = static_cast<const uint8_t*>(is_k ? c.k : c.v) + (is_k ? b * c.k_stride[0] + head * c.k_stride[1] + j * c.k_stride[2]
                                                                                 : b * c.v_stride[0] + head * c.v_stride[1] + j * c.v_stride[2]);
    const T* constants = static_cast<const T*>(is_k ? c.k_scales : c.v_scales) + (is_k ? b * c.k_scale_stride[0] + head * c.k_scale_stride[1] + j * c.k_scale_stride[2]
                                                                                       : b * c.v_scale_stride[0] + head * c.v_scale_stride[1] + j * c.v_scale_stride[2]);
    T* out = static_cast<T*>(is_k ? a.k_out : a.v_out) + (is_k ? b * a.k_out_stride[0] + head * a.k_out_stride[1] + j * a.k_out_stride[2]
                                                               : b * a.v_out_stride[0] + head * a.v_out_stride[1] + j * a.v_out_stride[2]);
    read_row<T, HD, GS>(codes, constants, out, threadIdx.x % LANES);
}

// For prompts: the rows that the tokens see between them, into dense k and v [batch, kv_heads, max_seq, hd].
template <typename T, int HD, int GS>
__global__ void __launch_bounds__(kThreads)
cache_read_seen_kernel(const __grid_constant__ Attn4Args a, T* __restrict__ k, T* __restrict__ v, unsigned chunks, const __grid_constant__ Divisor by_chunks,
                       const __grid_constant__ Divisor by_heads) {
    constexpr int LANES = HD / 8, ROWS = kThreads / LANES;
    asm volatile("griddepcontrol.launch_dependents;");
    const b200gptq_cache4& c = a.cache;
    const unsigned which = over(blockIdx.x, by_chunks), pair = which >> 1, b = over(pair, by_heads);
    const int head = (int)(pair - b * c.kv_heads);
    const bool is_k = !(which & 1);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int j = (int)((blockIdx.x - which * chunks) * ROWS + threadIdx.x / LANES);
    const int p0 = attn_pos(a.attn, b), count = attn_count(a.attn, b);
    const AttnRange r = attn_range(p0, p0 + count - 1, a.attn.window ? a.attn.window : 1 << 30, a.attn.sinks, c.max_seq);
    if (!count || j >= r.w_end || (j >= r.s_end && j < r.w_start) || j >= c.max_seq) return;
    const uint8_t* codes = static_cast<const uint8_t*>(is_k ? c.k : c.v) + (is_k ? b * c.k_stride[0] + head * c.k_stride[1] + j * c.k_stride[2]
                                                                                 : b * c.v_stride[0] + head * c.v_stride[1] + j * c.v_stride[2]);
    const T* constants = static_cast<const T*>(is_k ? c.k_scales : c.v_scales) + (is_k ? b * c.k_scale_stride[0] + head * c.k_scale_stride[1] + j * c.k_scale_stride[2]
                                                                                       : b * c.v_scale_stride[0] + head * c.v_scale_stride[1] + j * c.v_scale_stride[2]);
    read_row<T, HD, GS>(codes, constants, (is_k ? k : v) + ((long long)pair * c.max_seq + j) * HD, threadIdx.x % LANES);
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
    return launch(cache_write_kernel<T, HD, GS>, dim3((unsigned)((rows * (HD / 8) + kThreads - 1) / kThreads)), stream, a, (unsigned)rows, by);
}

template <typename T, int HD, int GS>
int read(const b200gptq_cache_read_args& a, cudaStream_t stream) {
    constexpr int ROWS = kThreads / (HD / 8);
    const long long chunks = (a.cache.max_seq + ROWS - 1) / ROWS, ctas = 2LL * a.cache.batch * a.cache.kv_heads;
    if (ctas > 0x7fffffff / chunks) return B200GPTQ_ERR_TOO_LARGE;
    return launch(cache_read_kernel<T, HD, GS>, dim3((unsigned)(ctas * chunks)), stream, a, (unsigned)chunks, Divisor(chunks), Divisor(a.cache.kv_heads));
}

template <typename T, int HD, int GS>
int read_seen(const Attn4Args& a, void* k, void* v, cudaStream_t stream) {
    constexpr int ROWS = kThreads / (HD / 8);
    const long long chunks = (a.cache.max_seq + ROWS - 1) / ROWS, ctas = 2LL * a.cache.batch * a.cache.kv_heads;
    if (ctas > 0x7fffffff / chunks) return B200GPTQ_ERR_TOO_LARGE;
    return launch(cache_read_seen_kernel<T, HD, GS>, dim3((unsigned)(ctas * chunks)), stream, a, static_cast<T*>(k), static_cast<T*>(v), (unsigned)chunks, Divisor(chunks),
                  Divisor(a.cache.kv_heads));
}

template <typename T, typename Args> int by_shape(const Args& a, cudaStream_t stream, int (*const (&run)[2][2])(const Args&, cudaStream_t)) {
    return run[a.cache.hd == 128][a.cache.group == 64](a, stream);
}

uintptr_t bits_of(const void* p, const int64_t (&stride)[3]) { return p ? reinterpret_cast<uintptr_t>(p) | (uintptr_t)(2 * (stride[0] | stride[1] | stride[2])) : 0; }

}  // namespace

int attn4_read_back(const Attn4Args& a, void* k, void* v, cudaStream_t s) {
    using F = int (*)(const Attn4Args&, void*, void*, cudaStream_t);
    static const F run[2][2][2] = {{{read_seen<__half, 64, 32>, read_seen<__half, 64, 64>}, {read_seen<__half, 128, 32>, read_seen<__half, 128, 64>}},
                                   {{read_seen<__nv_bfloat16, 64, 32>, read_seen<__nv_bfloat16, 64, 64>}, {read_seen<__nv_bfloat16, 128, 32>, read_seen<__nv_bfloat16, 128, 64>}}};
    return run[a.cache.dtype == B200GPTQ_BF16][a.cache.hd == 128][a.cache.group == 64](a, k, v, s);
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
    if (rows * (a.cache.hd / 8) > 2147483647.0) return B200GPTQ_ERR_TOO_LARGE;
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
