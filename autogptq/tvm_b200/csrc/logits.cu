// b200gptq_adjust_logits: penalties for repeated tokens, biases and grammar masks on the logits of the next token, one pass.
//
// A CTA takes a slice of one row's vocabulary.  It goes through the row's whole history and counts the tokens of its slice in shared memory
// (integers: the order of the additions does not matter), notes for each token the last entry among the biases, and lists the tokens that occur at all.  It
// copies its slice of the logits, with what the mask forbids, and then does the listed tokens: there are few, and in the loop over all tokens nearly every
// warp had one and went through all the branches (128 rows of 100003: 41 us and bound by instructions, now LLL).
// What bounds it: a few rows, the launch and one round trip to memory (the logits, the history, the lengths and the parameters are asked for at
// once); many rows, the logits' bytes and the L2 reads of the history, 8 bytes per token and slice.
#include <cuda_bf16.h>

#include <cstdlib>
#include <mutex>

#include "common.cuh"

namespace b200gptq {
namespace {

constexpr int kThreads = 256, kMaxSlice = 4096;
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

// Shared memory: a word per token of the slice (counts), the list of tokens (16 bits each) and its length, the slice's mask words, and with biases another
// word per token (number of the last entry + 1).
size_t shared_bytes(int slice, bool biases) { return (size_t)slice * 4 + (size_t)slice * 2 + 16 + slice / 8 + (biases ? (size_t)slice * 4 : 0); }

template <typename T>
__global__ void __launch_bounds__(kThreads)
adjust_kernel(const __grid_constant__ b200gptq_logit_args a, int slice, int slices) {
    extern __shared__ __align__(16) unsigned smem[];
    constexpr int V = 16 / sizeof(T), VECS = kMaxSlice / V / kThreads, H = 4;
    unsigned *count = smem, *listed = count + slice + slice / 2, *mask = listed + 4, *entry = mask + slice / 32;
    unsigned short* list = reinterpret_cast<unsigned short*>(count + slice);
    const int tid = threadIdx.x, row = blockIdx.x / slices, base = (blockIdx.x - row * slices) * slice, n = min(slice, a.vocab - base);
    for (int i = tid; i < slice / 4; i += kThreads) {
        reinterpret_cast<uint4*>(count)[i] = make_uint4(0, 0, 0, 0);
        if (a.biases) reinterpret_cast<uint4*>(entry)[i] = make_uint4(0, 0, 0, 0);
    }
    if (tid == 0) *listed = 0;
    const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride + base;
    T* out = static_cast<T*>(a.out) + row * a.out_stride + base;
    // 16 bytes at a time from the first aligned element on, where input and output are aligned alike
    const int skew = (int)(reinterpret_cast<uintptr_t>(in) & 15u) / (int)sizeof(T);
    const bool alike = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
    const int head = alike ? min(n, (V - skew) % V) : n, vecs = (n - head) / V;
    const int64_t* history = a.history + row * a.history_stride;
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    uint4 raw[VECS];
#pragma unroll
    for (int k = 0; k < VECS; ++k)
        if (tid + k * kThreads < vecs) raw[k] = *reinterpret_cast<const uint4*>(in + head + (tid + k * kThreads) * V);
    const int limit = a.history ? a.history_len : 0;
    unsigned long long t[H];                  // the first tokens, before it is known how many there are
#pragma unroll
    for (int u = 0; u < H; ++u) t[u] = tid + u * kThreads < limit ? (unsigned long long)history[tid + u * kThreads] : ~0ull;
    auto held = [&](const int64_t* p, int otherwise) { return p ? (int)max(min((long long)p[row], (long long)limit), 0LL) : otherwise; };
    const int length = held(a.history ? a.lengths : nullptr, limit), prompt = held(a.prompt_lens, 0);
    const float rep = a.repetition ? a.repetition[row] : 1.f, freq = a.frequency ? a.frequency[row] : 0.f, pres = a.presence ? a.presence[row] : 0.f;
    if (a.mask)
        for (int i = tid; i < (n + 31) / 32; i += kThreads) mask[i] = (unsigned)a.mask[row * a.mask_stride + base / 32 + i];
    __syncthreads();
    for (int i0 = tid; i0 < length; i0 += H * kThreads) {
        unsigned long long more[H];
#pragma unroll
        for (int u = 0; u < H; ++u) more[u] = i0 + (u + H) * kThreads < length ? (unsigned long long)history[i0 + (u + H) * kThreads] : ~0ull;
#pragma unroll
        for (int u = 0; u < H; ++u) {
            const int i = i0 + u * kThreads;
            const unsigned long long at = t[u] - (unsigned long long)base;
            if (i < length && at < (unsigned long long)n) {
                const unsigned before = i >= prompt ? atomicAdd(count + at, 1u) : atomicOr(count + at, kSeen);
                if (before == 0) list[atomicAdd(listed, 1u)] = (unsigned short)at;
            }
            t[u] = more[u];
        }
    }
    if (a.biases) {
        __syncthreads();                      // (which tokens the history has listed is known)
        for (int i = tid; i < a.biases; i += kThreads) {
            const unsigned long long at = (unsigned long long)a.bias_tokens[(size_t)row * a.biases + i] - (unsigned long long)base;
            if (at < (unsigned long long)n && atomicMax(entry + at, (unsigned)i + 1u) == 0 && count[at] == 0) list[atomicAdd(listed, 1u)] = (unsigned short)at;
        }
    }
    // ---- the slice as it is, minus infinity where the mask says so ----
    auto allowed = [&](int i) { return !a.mask || (mask[i >> 5] >> (i & 31) & 1u); };
    auto single = [&](int i) { out[i] = allowed(i) ? in[i] : Conv<T>::out(-INFINITY); };
    for (int i = tid; i < head; i += kThreads) single(i);
#pragma unroll
    for (int k = 0; k < VECS; ++k)
        if (tid + k * kThreads < vecs) {
            const int i = head + (tid + k * kThreads) * V;
            T* x = reinterpret_cast<T*>(&raw[k]);
            if (a.mask) {
                const unsigned bits = __funnelshift_r(mask[i >> 5], mask[(i + V - 1) >> 5], i & 31);
#pragma unroll
                for (int u = 0; u < V; ++u)
                    if (!(bits >> u & 1u)) x[u] = Conv<T>::out(-INFINITY);
            }
            *reinterpret_cast<uint4*>(out + i) = raw[k];
        }
    for (int i = head + vecs * V + tid; i < n; i += kThreads) single(i);
    __syncthreads();
    // ---- the listed tokens.  What stands in the output is the logit as it was, except where the mask forbids it. ----
    const int many = (int)*listed;
    for (int k = tid; k < many; k += kThreads) {
        const int i = list[k];
        if (!allowed(i)) continue;
        float x = Conv<T>::in(out[i]);
        const unsigned c = count[i], times = c & ~kSeen;
        if (c) {
            x = x > 0.f ? __fdiv_rn(x, rep) : x * rep;
            if (times) x = x - freq * (float)times - pres;
        }
        if (a.biases) {
            const unsigned e = entry[i];
            if (e) x += a.bias_values[(size_t)row * a.biases + e - 1];
        }
        out[i] = Conv<T>::out(x);
    }
}

template <typename T>
int launch(const b200gptq_logit_args& a, int slice, cudaStream_t stream) {
    const int slices = (a.vocab + slice - 1) / slice;
    if ((long long)a.rows * slices > 0x7fffffff) return B200GPTQ_ERR_TOO_LARGE;
    static const bool pdl = [] {
        const char* e = std::getenv("B200GPTQ_PDL");
        return !(e && e[0] == '0');
    }();
    static std::once_flag once[64];
    static cudaError_t result[64];
    int dev = 0;
    B200GPTQ_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return B200GPTQ_ERR_TOO_LARGE;
    std::call_once(once[dev], [&] { result[dev] = cudaFuncSetAttribute(adjust_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared_bytes(kMaxSlice, true)); });
    B200GPTQ_CUDA_TRY(result[dev]);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * slices));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = shared_bytes(slice, a.biases > 0);
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
    // Slices: as small as leaves five CTAs per SM, since every CTA goes through the history.
    const long long ctas = 5LL * sm_count();
    int slice = 1024;
    while (slice < kMaxSlice && (long long)a.rows * ((a.vocab + slice - 1) / slice) > ctas) slice *= 2;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return a.dtype == B200GPTQ_F16 ? launch<__half>(a, slice, s) : a.dtype == B200GPTQ_BF16 ? launch<__nv_bfloat16>(a, slice, s) : launch<float>(a, slice, s);
}
