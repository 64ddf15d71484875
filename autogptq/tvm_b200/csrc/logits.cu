// b200gptq_adjust_logits: penalties for repeated tokens, biases and grammar masks on the logits of the next token, one pass.
//
// A CTA takes a slice of one row's vocabulary.  It goes through the row's whole history and counts the tokens of its slice in shared memory
// (integers: the order of the additions does not matter), notes for each token the last entry among the biases, and lists the tokens that occur at all.  It
// copies its slice of the logits, with what the mask forbids, and then does the listed tokens: there are few, and in the loop over all tokens nearly every
// warp had one and went through all the branches (128 rows of 100003: 41 us and bound by instructions, now 32).
// What bounds it: a few rows, the launch and the round trips to memory, of which there are two, everything else is asked for at once in front
// of them (64 rows of 50272: lengths, history, biases and logits one after the other 14.7 us, now 7.7); many rows, the logits' bytes and the L2 reads of the
// history, 8 bytes per token and slice.  (A cluster of eight CTAs that shares the work on the history: 3 to 18 us slower.)
#include <cuda_bf16.h>

#include <cstdlib>
#include <mutex>

#include "common.cuh"

namespace b200gptq {
namespace {

constexpr int kThreads = 512, kMaxSlice = 8192, kPerSm = 3;
// A token's word: bit 31, it stands in the prompt; bits 0 .. 15, how often behind it; bits 16 .. 30, number of its last entry among the biases + 1.  With texts or
// lists too long for that (WIDE) bits 0 .. 29 count, bit 30 says that there is an entry, and the entries have words of their own.
constexpr unsigned kSeen = 0x80000000u, kBiased = 0x40000000u;
constexpr int kMostCounted = 0xffff, kMostEntries = 0x7fff;

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

// Shared memory: a word per token of the slice, the list of tokens (16 bits each) and its length, the slice's mask words, WIDE: another word per token (number
// of the last entry + 1).
size_t shared_bytes(int slice, bool wide) { return (size_t)slice * 4 + (size_t)slice * 2 + 16 + slice / 8 + (wide ? (size_t)slice * 4 : 0); }

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads, kPerSm)
adjust_kernel(const __grid_constant__ b200gptq_logit_args a, int slice, int slices) {
    extern __shared__ __align__(16) unsigned smem[];
    constexpr int V = 16 / sizeof(T), VECS = kMaxSlice / V / kThreads, H = 2, L = 1;
    unsigned *count = smem, *listed = count + slice + slice / 2, *mask = listed + 4, *entry = mask + slice / 32;
    unsigned short* list = reinterpret_cast<unsigned short*>(count + slice);
    const int tid = threadIdx.x, row = blockIdx.x / slices, base = (blockIdx.x - row * slices) * slice, n = min(slice, a.vocab - base);
    for (int i = tid; i < slice / 4; i += kThreads) {
        reinterpret_cast<uint4*>(count)[i] = make_uint4(0, 0, 0, 0);
        if (WIDE) reinterpret_cast<uint4*>(entry)[i] = make_uint4(0, 0, 0, 0);
    }
    if (tid == 0) *listed = 0;
    const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride + base;
    T* out = static_cast<T*>(a.out) + row * a.out_stride + base;
    // 16 bytes at a time from the first aligned element on, where input and output are aligned alike
    const int skew = (int)(reinterpret_cast<uintptr_t>(in) & 15u) / (int)sizeof(T);
    const bool alike = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
    const int head = alike ? min(n, (V - skew) % V) : n, vecs = (n - head) / V;
    const int64_t *history = a.history + row * a.history_stride, *bias_tokens = a.bias_tokens + (size_t)row * a.biases;
    const float* bias_values = a.bias_values + (size_t)row * a.biases;
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // ---- all that can be asked for at once, what is waited for first in front (the logits first: 128 rows of 100003 40 us, now 32) ----
    const int limit = a.history ? a.history_len : 0;
    // The history, two tokens at a time where it lies on 16 bytes; the first of them before it is known how many there are.
    const bool paired = (reinterpret_cast<uintptr_t>(history) & 15u) == 0;
    auto fetch = [&](int i, int end, unsigned long long (&t)[2]) {         // tokens i and i + 1
        t[0] = t[1] = ~0ull;
        if (paired && i + 1 < end) {
            const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(history + i);
            t[0] = two.x;
            t[1] = two.y;
        } else {
            if (i < end) t[0] = (unsigned long long)history[i];
            if (i + 1 < end) t[1] = (unsigned long long)history[i + 1];
        }
    };
    unsigned long long t[H][2], biased = ~0ull;
#pragma unroll
    for (int u = 0; u < H; ++u) fetch(2 * (tid + u * kThreads), limit, t[u]);
    if (tid < a.biases) biased = (unsigned long long)bias_tokens[tid];
    auto held = [&](const int64_t* p, int otherwise) { return p ? (int)max(min((long long)p[row], (long long)limit), 0LL) : otherwise; };
    const int length = held(a.history ? a.lengths : nullptr, limit), prompt = held(a.prompt_lens, 0);
    const float rep = a.repetition ? a.repetition[row] : 1.f, freq = a.frequency ? a.frequency[row] : 0.f, pres = a.presence ? a.presence[row] : 0.f;
    uint4 raw[VECS];
#pragma unroll
    for (int k = 0; k < VECS; ++k)
        if (tid + k * kThreads < vecs) raw[k] = *reinterpret_cast<const uint4*>(in + head + (tid + k * kThreads) * V);
    if (a.mask)
        for (int i = tid; i < (n + 31) / 32; i += kThreads) mask[i] = (unsigned)a.mask[row * a.mask_stride + base / 32 + i];
    __syncthreads();
    // ---- the words, and the list of those that are no longer zero ----
    for (int i0 = 2 * tid; i0 < length; i0 += 2 * H * kThreads) {
        if (i0 >= 2 * H * kThreads)
#pragma unroll
            for (int u = 0; u < H; ++u) fetch(i0 + 2 * u * kThreads, length, t[u]);
#pragma unroll
        for (int u = 0; u < H; ++u)
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const int i = i0 + 2 * u * kThreads + v;
                const unsigned at = (unsigned)t[u][v] - (unsigned)base;          // (the vocabulary has below 2^31 tokens)
                if (i < length && at < (unsigned)n && !(unsigned)(t[u][v] >> 32)) {
                    const unsigned before = i >= prompt ? atomicAdd(count + at, 1u) : atomicOr(count + at, kSeen);
                    if (before == 0) list[atomicAdd(listed, 1u)] = (unsigned short)at;
                }
            }
    }
    for (int i = tid; i < a.biases; i += kThreads) {
        if (i >= kThreads) biased = (unsigned long long)bias_tokens[i];
        const unsigned long long at = biased - (unsigned long long)base;
        if (at >= (unsigned long long)n) continue;
        unsigned before;
        if constexpr (WIDE) {
            before = atomicOr(count + at, kBiased);
            atomicMax(entry + at, (unsigned)i + 1u);
        } else {
            unsigned now = count[at];
            do {
                before = now;
                if ((before >> 16 & (unsigned)kMostEntries) > (unsigned)i) break;
                now = atomicCAS(count + at, before, (before & (kSeen | (unsigned)kMostCounted)) | ((unsigned)i + 1u) << 16);
            } while (now != before);
        }
        if (before == 0) list[atomicAdd(listed, 1u)] = (unsigned short)at;
    }
    __syncthreads();
    // ---- the logits and biases of the thread's first listed tokens (a token that another thread overwrites meanwhile, in place, keeps its value, or is one
    //      that the mask forbids) ----
    const int many = (int)*listed;
    auto allowed = [&](int i) { return !a.mask || (mask[i >> 5] >> (i & 31) & 1u); };
    auto number = [&](unsigned w, int i) { return WIDE ? (w & kBiased ? entry[i] : 0u) : w >> 16 & (unsigned)kMostEntries; };
    auto bias_of = [&](unsigned w, int i) { const unsigned e = a.biases ? number(w, i) : 0u; return e ? bias_values[e - 1] : 0.f; };
    float x[L], y[L];
#pragma unroll
    for (int k = 0; k < L; ++k)
        if (tid + k * kThreads < many) {
            const int i = list[tid + k * kThreads];
            x[k] = Conv<T>::in(in[i]);
            y[k] = bias_of(count[i], i);
        }
    // ---- the slice as it is, minus infinity where the mask says so ----
    auto single = [&](int i) { out[i] = allowed(i) ? in[i] : Conv<T>::out(-INFINITY); };
    for (int i = tid; i < head; i += kThreads) single(i);
#pragma unroll
    for (int k = 0; k < VECS; ++k)
        if (tid + k * kThreads < vecs) {
            const int i = head + (tid + k * kThreads) * V;
            T* v = reinterpret_cast<T*>(&raw[k]);
            if (a.mask) {
                const unsigned bits = __funnelshift_r(mask[i >> 5], mask[(i + V - 1) >> 5], i & 31);
#pragma unroll
                for (int u = 0; u < V; ++u)
                    if (!(bits >> u & 1u)) v[u] = Conv<T>::out(-INFINITY);
            }
            *reinterpret_cast<uint4*>(out + i) = raw[k];
        }
    for (int i = head + vecs * V + tid; i < n; i += kThreads) single(i);
    __syncthreads();
    // ---- the listed tokens.  What stands in the output is the logit as it was, except where the mask forbids it. ----
    auto adjust = [&](int i, float x, float bias) {
        const unsigned w = count[i], times = w & (WIDE ? kBiased - 1u : (unsigned)kMostCounted);
        if (w & kSeen || times) {
            x = x > 0.f ? __fdiv_rn(x, rep) : x * rep;
            if (times) x = x - freq * (float)times - pres;
        }
        if (a.biases && number(w, i)) x += bias;
        if (allowed(i)) out[i] = Conv<T>::out(x);
    };
#pragma unroll
    for (int k = 0; k < L; ++k)
        if (tid + k * kThreads < many) adjust(list[tid + k * kThreads], x[k], y[k]);
    for (int k = tid + L * kThreads; k < many; k += kThreads) {
        const int i = list[k];
        adjust(i, Conv<T>::in(out[i]), bias_of(count[i], i));
    }
}

template <typename T, bool WIDE>
int launch(const b200gptq_logit_args& a, cudaStream_t stream) {
    // Slices: the first of 1024, 2048, 4096 and 8192 whose grid is at most kPerSm CTAs per SM, else the last, since every CTA goes through the history.  (Where words
    // are WIDE, 83 KB for 8192, two of the last are on an SM at once.)  Not all grids are whole waves: 64 rows of 50272 are 448 CTAs for 444 places, 128 of 32000 are 512 (7.3 and 6.5 us with penalties alone).
    int slice = 1024;
    while (slice < kMaxSlice && (long long)a.rows * ((a.vocab + slice - 1) / slice) > (long long)kPerSm * sm_count()) slice *= 2;
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
    auto* kernel = adjust_kernel<T, WIDE>;
    std::call_once(once[dev], [&] { result[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared_bytes(kMaxSlice, WIDE)); });
    B200GPTQ_CUDA_TRY(result[dev]);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * slices));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = shared_bytes(slice, WIDE);
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = pdl ? 1 : 0;
    B200GPTQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a, slice, slices));
    return B200GPTQ_OK;
}

template <typename T>
int launch(const b200gptq_logit_args& a, cudaStream_t stream) {
    return (a.history && a.history_len > kMostCounted) || a.biases > kMostEntries ? launch<T, true>(a, stream) : launch<T, false>(a, stream);
}

}  // namespace
}  // namespace b200gptq

using namespace b200gptq;

extern "C" B200GPTQ_API int b200gptq_adjust_logits(const b200gptq_logit_args* args, void* stream) {
    if (!args) return B200GPTQ_ERR_NULL_POINTER;
    const b200gptq_logit_args& a = *args;
    if (!a.logits || !a.out || (a.history && !a.lengths) || (a.biases && (!a.bias_tokens || !a.bias_values))) return B200GPTQ_ERR_NULL_POINTER;
    if (a.rows < 1 || a.vocab < 1 || a.vocab > 1 << 30 || a.history_len < 0 || a.history_len >= 1 << 30 || a.biases < 0 || a.biases >= 1 << 30 ||
        a.logits_stride < 0 || a.out_stride < 0)
        return B200GPTQ_ERR_SHAPE;
    const int size = a.dtype == B200GPTQ_F32 ? 4 : 2;
    if (a.dtype != B200GPTQ_F16 && a.dtype != B200GPTQ_BF16 && a.dtype != B200GPTQ_F32) return B200GPTQ_ERR_SHAPE;
    if ((reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.out)) & (size - 1) ||
        (reinterpret_cast<uintptr_t>(a.history) | reinterpret_cast<uintptr_t>(a.bias_tokens) | reinterpret_cast<uintptr_t>(a.lengths) |
         reinterpret_cast<uintptr_t>(a.prompt_lens)) & 7u ||
        (reinterpret_cast<uintptr_t>(a.repetition) | reinterpret_cast<uintptr_t>(a.frequency) | reinterpret_cast<uintptr_t>(a.presence) |
         reinterpret_cast<uintptr_t>(a.bias_values) | reinterpret_cast<uintptr_t>(a.mask)) & 3u)
        return B200GPTQ_ERR_ALIGNMENT;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return a.dtype == B200GPTQ_F16 ? launch<__half>(a, s) : a.dtype == B200GPTQ_BF16 ? launch<__nv_bfloat16>(a, s) : launch<float>(a, s);
}
