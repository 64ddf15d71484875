// b200gptq_adjust_logits: penalties for repeated tokens, biases and grammar masks on the logits of the next token, one pass.
//
// A CTA takes a slice of one row's vocabulary.  It goes through the row's whole history and counts the tokens of its slice in shared memory
// (integers: the order of the additions does not matter), notes for each token the last entry among the biases, and then streams its slice of the
// logits.  What bounds it: a few rows, the launch and the round trips history -> counts -> logits; many rows, the logits' bytes and the L2 reads
// of the history, 8 bytes per token and slice.
#include <cuda_bf16.h>

#include <cstdlib>

#include "common.cuh"

namespace b200gptq {
namespace {

constexpr int kThreads = 512;
constexpr unsigned kSeen = 0x80000000u;     // the token occurs; the other bits: how often behind the prompt

template <typename T> struct Conv;
template <> struct Conv<float> {
    __device__ static __forceinline__ float in(float x) { return x; }
    __device__ static __forceinline__ float out(float x) { return x; }
};
template <> struct Conv<__half> {
    __device__ static __forceinline__ float in(__half x) { return __half2float(x); }
    __device__ static __forceinline__ __half out(float x) { return __float2half_rn(x); }
};
template <> struct Conv<__nv_bfloat16> {
    __device__ static __forceinline__ float in(__nv_bfloat16 x) { return __bfloat162float(x); }
    __device__ static __forceinline__ __nv_bfloat16 out(float x) { return __float2bfloat16_rn(x); }
};

// Shared memory: a word per token of the slice (counts), the slice's mask words, and with biases another word per token (number of the last entry + 1).
template <typename T>
__global__ void __launch_bounds__(kThreads)
adjust_kernel(const __grid_constant__ b200gptq_logit_args a, int slice, int slices) {
    extern __shared__ __align__(16) unsigned smem[];
    unsigned *count = smem, *mask = count + slice, *entry = mask + slice / 32;
    const int tid = threadIdx.x, row = blockIdx.x / slices, base = (blockIdx.x - row * slices) * slice, n = min(slice, a.vocab - base);
    for (int i = tid; i < slice / 4; i += kThreads) {
        reinterpret_cast<uint4*>(count)[i] = make_uint4(0, 0, 0, 0);
        if (a.biases) reinterpret_cast<uint4*>(entry)[i] = make_uint4(0, 0, 0, 0);
    }
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __syncthreads();
    const int limit = a.history_len;
    auto held = [&](const int64_t* p, int otherwise) { return p ? (int)max(min((long long)p[row], (long long)limit), 0LL) : otherwise; };
    if (a.history) {
        const int length = held(a.lengths, limit), prompt = held(a.prompt_lens, 0);
        const int64_t* h = a.history + row * a.history_stride;
        for (int i0 = tid; i0 < length; i0 += 4 * kThreads) {
            unsigned long long t[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) t[u] = i0 + u * kThreads < length ? (unsigned long long)h[i0 + u * kThreads] - (unsigned long long)base : ~0ull;
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (t[u] < (unsigned long long)n) {
                    if (i0 + u * kThreads >= prompt) atomicAdd(count + t[u], 1u);
                    atomicOr(count + t[u], kSeen);
                }
        }
    }
    for (int i = tid; i < a.biases; i += kThreads) {
        const unsigned long long t = (unsigned long long)a.bias_tokens[(size_t)row * a.biases + i] - (unsigned long long)base;
        if (t < (unsigned long long)n) atomicMax(entry + t, (unsigned)i + 1u);
    }
    if (a.mask)
        for (int i = tid; i < (n + 31) / 32; i += kThreads) mask[i] = (unsigned)a.mask[row * a.mask_stride + base / 32 + i];
    __syncthreads();
    const float rep = a.repetition ? a.repetition[row] : 1.f, freq = a.frequency ? a.frequency[row] : 0.f, pres = a.presence ? a.presence[row] : 0.f;
    const float* values = a.bias_values + (size_t)row * a.biases;
    auto adjust = [&](float x, int i) {
        const unsigned c = count[i], times = c & ~kSeen;
        if (c) {
            x = x > 0.f ? __fdiv_rn(x, rep) : x * rep;
            if (times) x = x - freq * (float)times - pres;
        }
        if (a.biases) {
            const unsigned e = entry[i];
            if (e) x += values[e - 1];
        }
        if (a.mask && !(mask[i >> 5] >> (i & 31) & 1u)) x = -INFINITY;
        return x;
    };
    const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride + base;
    T* out = static_cast<T*>(a.out) + row * a.out_stride + base;
    // 16 bytes at a time from the first aligned element on, where input and output are aligned alike
    constexpr int V = 16 / sizeof(T);
    const int skew = (int)(reinterpret_cast<uintptr_t>(in) & 15u) / (int)sizeof(T);
    const bool alike = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
    const int head = alike ? min(n, (V - skew) % V) : n, vecs = (n - head) / V;
    for (int i = tid; i < head; i += kThreads) out[i] = Conv<T>::out(adjust(Conv<T>::in(in[i]), i));
    for (int v = tid; v < vecs; v += kThreads) {
        const int i = head + v * V;
        uint4 raw = *reinterpret_cast<const uint4*>(in + i);
        T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
        for (int u = 0; u < V; ++u) e[u] = Conv<T>::out(adjust(Conv<T>::in(e[u]), i + u));
        *reinterpret_cast<uint4*>(out + i) = raw;
    }
    for (int i = head + vecs * V + tid; i < n; i += kThreads) out[i] = Conv<T>::out(adjust(Conv<T>::in(in[i]), i));
}

template <typename T>
int launch(const b200gptq_logit_args& a, int slice, cudaStream_t stream) {
    const int slices = (a.vocab + slice - 1) / slice;
    if ((long long)a.rows * slices > 0x7fffffff) return B200GPTQ_ERR_TOO_LARGE;
    static const bool pdl = [] {
        const char* e = std::getenv("B200GPTQ_PDL");
        return !(e && e[0] == '0');
    }();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * slices));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)slice * 4 + slice / 8 + (a.biases ? (size_t)slice * 4 : 0);
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = pdl ? 1 : 0;
    B200GPTQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, adjust_kernel<T>, a, slice, slices));
    return B200GPTQ_OK;
}

}  // namespace
}  // namespace b200gptq

using namespace b200gptq;

extern "C" B200GPTQ_API int b200gptq_adjust_logits(const b200gptq_logit_args* args, void* stream) {
    if (!args) return B200GPTQ_ERR_NULL_POINTER;
    const b200gptq_logit_args& a = *args;
    if (!a.logits || !a.out || (a.history && !a.lengths) || (a.biases && (!a.bias_tokens || !a.bias_values))) return B200GPTQ_ERR_NULL_POINTER;
    if (a.rows < 1 || a.vocab < 1 || a.history_len < 0 || a.biases < 0 || a.logits_stride < 0 || a.out_stride < 0) return B200GPTQ_ERR_SHAPE;
    const int size = a.dtype == B200GPTQ_F32 ? 4 : 2;
    if (a.dtype != B200GPTQ_F16 && a.dtype != B200GPTQ_BF16 && a.dtype != B200GPTQ_F32) return B200GPTQ_ERR_SHAPE;
    if ((reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.out)) & (size - 1) ||
        (reinterpret_cast<uintptr_t>(a.history) | reinterpret_cast<uintptr_t>(a.bias_tokens) | reinterpret_cast<uintptr_t>(a.lengths) |
         reinterpret_cast<uintptr_t>(a.prompt_lens)) & 7u)
        return B200GPTQ_ERR_ALIGNMENT;
    // Slices: as small as leaves four CTAs per SM, since every CTA goes through the history.
    const long long ctas = 4LL * sm_count();
    int slice = 1024;
    while (slice < 4096 && (long long)a.rows * ((a.vocab + slice - 1) / slice) > ctas) slice *= 2;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return a.dtype == B200GPTQ_F16 ? launch<__half>(a, slice, s) : a.dtype == B200GPTQ_BF16 ? launch<__nv_bfloat16>(a, slice, s) : launch<float>(a, slice, s);
}
