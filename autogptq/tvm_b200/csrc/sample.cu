// b200gptq_sample: the next token under temperature, top-k, top-p and min-p, from a given random number; see include/b200gptq.h.
//
//   w_v = exp((x_v - max x) / T),  kept: a beginning of the order "larger x, then lower v",  token: the first v whose kept sum passes u * (sum of all kept)
//
// What decides are sums over the vocabulary, and a random number may fall anywhere between two tokens: sums in fp32 put borders off by more than what lies
// between neighbours.  Weights are integers here (units of 2^-F of the largest, F so that the vocabulary's sum fits 62 bits; off by 2^-32 relative at most: the logarithm in fixed
// point of 32 fractional bits, by one FMA in 64 bits, a table of 256 powers and a Taylor polynomial of degree 3, after P. T. P. Tang, "Table-driven implementation of the
// exponential function", 1989; the table has 52 bits and the products with it 40, so that the logarithm's last one is what counts, 2^-33.5), their sums have
// neither order nor rounding, and the products p * S and u * S are taken in 128 bits.
//
// A cluster of CTAs shares a row, each keeps a slice of the logits in shared memory.  Where top-k or top-p ends follows from histograms: 1024 bins, linear in
// the logarithm of the weight, of the tokens' number (top-k) or weight (top-p; the order of x and of the bins is the same), then the bin in which the search ends
// again by the bits of x until one value is left.  Tokens of that value are kept from the lowest on.  After the first bins only the tokens down to where the
// search ended are looked at again: each warp moves its own together.  The CTAs of the cluster read each other's sums through distributed shared memory and all come
// to the same results.
// Bound by the chain of searches (2 to 5 after one another, some 5000 clk each: bins, a meeting, sums from the other CTAs, a decision) and, with many rows, by the
// instructions of the pass over all weights.  Measured: 1 row of 32000 17.7 us, 64 rows of 50272 30.9, 128 of 100003 in fp32 130 (half of
// the issue slots in use).
#include <cuda_bf16.h>

#include <cstddef>
#include <cstdlib>
#include <mutex>

#include "common.cuh"

namespace b200gptq {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 1024, kBinBits = 10, kMostCtas = 8, kTableBits = 8, kTable = 1 << kTableBits;
constexpr float kColdest = 1e-18f;       // temperatures below count as 0, so that no scale leaves fp32
typedef unsigned long long u64;

template <typename T> __device__ __forceinline__ float wide(T x);
template <> __device__ __forceinline__ float wide(float x) { return x; }
template <> __device__ __forceinline__ float wide(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float wide(__nv_bfloat16 x) { return __bfloat162float(x); }

// Larger x, larger key; a NaN counts as minus infinity.  (The last 13 or 16 bits of a number of 16 bits say nothing in fp32.)
template <typename T> struct Key { static constexpr int shift = 0; };
template <> struct Key<__half> { static constexpr int shift = 13; };
template <> struct Key<__nv_bfloat16> { static constexpr int shift = 16; };
template <typename T> __device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __float_as_uint(x == 0.f ? 0.f : x);
    return x != x ? 0u : (b & 0x80000000u ? ~b : b | 0x80000000u) >> Key<T>::shift;
}
template <typename T> __device__ __forceinline__ float of_key(unsigned k) {
    const unsigned b = k << Key<T>::shift;
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~(b | ((1u << Key<T>::shift) - 1)));
}

__device__ __forceinline__ uint32_t remote_of(const void* local, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    return r;
}
__device__ __forceinline__ unsigned ld_remote(uint32_t at) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void st_remote(uint32_t at, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory"); }
__device__ __forceinline__ void st_remote(uint32_t at, unsigned long long v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }
__device__ __forceinline__ void st_remote(uint32_t at, const uint4& v) {
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <typename V> __device__ __forceinline__ V warp_total(V v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <typename V> __device__ __forceinline__ V warp_prefix(V v, int lane) {      // with the lane's own
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}

// f * s for f >= 0, rounded down or up; 2^62 at most.
__device__ __forceinline__ u64 share(float f, u64 s, bool up) {
    if (!(f > 0.f)) return 0;
    if (f >= 1.f) return s;
    int e;
    const unsigned m = (unsigned)ldexpf(frexpf(f, &e), 24);       // f = m 2^(e - 24), e <= 0
    const int down = 24 - e;
    const u64 hi = __umul64hi(m, s), lo = m * s;
    u64 q, rest;
    if (down < 64) { q = hi << (64 - down) | lo >> down; rest = lo & ((1ull << down) - 1); }
    else if (down < 128) { q = down == 64 ? hi : hi >> (down - 64); rest = lo | (down == 64 ? 0 : hi & ((1ull << (down - 64)) - 1)); }
    else { q = 0; rest = 1; }
    return q + (up && rest ? 1 : 0);
}

// A bin's weight in three words of 17 bits and what they pass over, so that adding takes no carry (a slice has below 2^15 tokens); its number of tokens is in the first.
struct Bins { unsigned part[3][kBins]; };
constexpr int kPart = 17;
struct __align__(16) Warp { u64 mass; unsigned ties, unused; };       // of a warp's tokens: sum above the border, how many are at it
// (What all CTAs want of each other they push before they meet: reading it after that cost a round trip of some 700 clk more.)
struct Shared {
    Bins bins[2];                         // in turn: this pass's, and the last one's, which become the next one's
    u64 groups[2][kMostCtas][kBins / 32]; // sums of 32 bins of each CTA
    u64 table[kTable];                    // 2^(52 + j / kTable)
    Warp warps[kMostCtas * kWarps];       // of all CTAs
    u64 found_above, all, target, before;
    unsigned ties_before;
    float tops[kMostCtas], warp_top[kWarps];
    int found, owner;
};

// Everything of a row that the CTAs of its cluster agree on.
struct Row {
    float top, half_scale;               // largest logit; bins per half a unit of x
    double step;                         // log2(e) / T
    int bits;                            // F
};
__device__ __forceinline__ u64 weight(float x, const Row& r, const u64* table) {        // (no branches: several at once hide each other's latency)
    // 1.5 2^20 + log2 of the weight: the number's last word is the fraction of the logarithm, the first its whole part
    const long long y = __double_as_longlong(fma((double)x - (double)r.top, r.step, 1572864.0));
    const unsigned down = 0x41380000u - (unsigned)(y >> 32);                             // (a NaN, minus infinity: far outside)
    const unsigned f = (unsigned)y;
    const u64 p = table[f >> (32 - kTableBits)];
    // 2^rest - 1 in units of 2^-40, below 2^31.5: z + z^2 / 2 + z^3 / 6 with z = ln 2 times the rest, the first of these as a whole number
    constexpr double ln2 = 0.69314718055994531;
    const float z = (float)(f & ((1u << (32 - kTableBits)) - 1));                        // (units of 2^-32)
    const unsigned e = __umulhi(f << kTableBits, (unsigned)(ln2 * 0x1p32 + 0.5)) + __float2uint_rn(z * z * fmaf(z, (float)(ln2 * ln2 * ln2 / 6 * 0x1p-56), (float)(ln2 * ln2 / 2 * 0x1p-24)));
    const u64 m = p + ((u64)(unsigned)(p >> 21) * e >> 19);                              // the weight in units of 2^-52, before it is shifted down
    const u64 w = ((m >> min(51 - r.bits + down, 63u)) + 1) >> 1;
    return x == r.top ? 1ull << r.bits : down < 64u ? w : 0;
}
// The same where it is not worth its code.
__device__ __noinline__ u64 weight_apart(float x, const Row& r, const u64* table) { return weight(x, r, table); }
// Bin of x, kBins or more where its weight is zero.
__device__ __forceinline__ int bin_of(float x, const Row& r) {
    if (x == r.top) return 0;
    const float f = (0.5f * r.top - 0.5f * x) * r.half_scale;
    return f < (float)kBins ? (int)f : kBins;                                                // (a NaN: kBins)
}

__device__ __forceinline__ u64 sum_of(unsigned a, unsigned b, unsigned c) { return a + ((u64)b << kPart) + ((u64)c << 2 * kPart); }
__device__ __forceinline__ void put(Bins& h, unsigned at, u64 w) {
    const unsigned a = (unsigned)w & ((1u << kPart) - 1), b = (unsigned)(w >> kPart) & ((1u << kPart) - 1), c = (unsigned)(w >> 2 * kPart);
    if (a) atomicAdd(h.part[0] + at, a);
    if (b) atomicAdd(h.part[1] + at, b);
    if (c) atomicAdd(h.part[2] + at, c);
}

// The sums of 32 bins each, by all warps, to all CTAs; a bin's sum into its first two words.
__device__ __forceinline__ void add_groups(Bins& h, u64* groups, int rank, int ctas) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int g = threadIdx.x >> 5; g < kBins / 32; g += kWarps) {
        const u64 bin = sum_of(h.part[0][32 * g + lane], h.part[1][32 * g + lane], h.part[2][32 * g + lane]), sum = warp_total(bin);
        h.part[0][32 * g + lane] = (unsigned)bin;
        h.part[1][32 * g + lane] = (unsigned)(bin >> 32);
        if (lane < ctas) st_remote(remote_of(groups + rank * (kBins / 32) + g, lane), sum);
    }
}

// One warp of each CTA, when the CTAs have met: the first bin of all of them added up, from the top on, with which the sum (and what lies `above` all bins)
// reaches its target, which may be a share of all, and the sum above it; -1 where it does not.  (Reading all bins of all CTAs instead, 96 KB each through the cluster's network, took 2.7 us.)
template <typename Target> __device__ __forceinline__ void find(Shared& s, const Bins& h, const u64* groups, int ctas, u64 above, Target target_of) {
    static_assert(kBins == 32 * 32, "");
    const int lane = threadIdx.x & 31;
    u64 sum = 0;
#pragma unroll
    for (int r = 0; r < kMostCtas; ++r) sum += r < ctas ? groups[r * (kBins / 32) + lane] : 0;
    u64 to = above + warp_prefix(sum, lane);
    const u64 all = __shfl_sync(0xffffffffu, to, 31), target = target_of(all);
    if (lane == 0) { s.all = all; s.target = target; }
    const unsigned hit = __ballot_sync(0xffffffffu, to >= target);
    if (lane == 0) s.found = -1;
    if (!hit) return;
    const int g = __ffs(hit) - 1;
    above = __shfl_sync(0xffffffffu, to - sum, g);
    unsigned n[kMostCtas][2];
#pragma unroll
    for (int r = 0; r < kMostCtas; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i) n[r][i] = r < ctas ? ld_remote(remote_of(h.part[i] + 32 * g + lane, r)) : 0;
    sum = 0;
#pragma unroll
    for (int r = 0; r < kMostCtas; ++r) sum += ((u64)n[r][1] << 32) + n[r][0];
    to = above + warp_prefix(sum, lane);
    const unsigned in = __ballot_sync(0xffffffffu, to >= target);
    if (lane == __ffs(in) - 1) {
        s.found = 32 * g + lane;
        s.found_above = to - sum;
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
sample_kernel(const __grid_constant__ b200gptq_sample_args a, int slice, int cluster_bits, int bits) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem);
    T* x = reinterpret_cast<T*>(smem + (sizeof(Shared) + 15) / 16 * 16);                  // the slice, later what each warp has kept of its run of it
    unsigned short* places = reinterpret_cast<unsigned short*>(x + slice);                // and where that stood in the run
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ctas = 1 << cluster_bits, row = blockIdx.x >> cluster_bits, rank = blockIdx.x & (ctas - 1);
    const int base = min(rank * slice, a.vocab), n = min(slice, a.vocab - base);
    // A warp's tokens: a run of the slice
    const int run = (slice + kWarps - 1) / kWarps, first = min(warp * run, n), last = min(first + run, n);
    for (int i = tid; i < (int)sizeof(s.bins) / 16; i += kThreads) reinterpret_cast<uint4*>(s.bins)[i] = make_uint4(0, 0, 0, 0);
    if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    auto meet = [&] {
        if (ctas > 1) cluster_sync();
        else __syncthreads();
    };
    if (tid < kTable) s.table[tid] = __double2ull_rn(exp2(52 + (double)tid / kTable));
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride + base;
    const float temperature = a.temperature ? a.temperature[row] : 1.f, top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f, u = a.uniform[row];
    const long long top_k = a.top_k ? a.top_k[row] : 0;
    const double step = 1.4426950408889634074 / (double)temperature;                     // (of no use where the temperature is 0)
    // ---- the slice, and the row's largest logit ----
    float top = -INFINITY;
    if ((reinterpret_cast<uintptr_t>(in) & 15u) == 0) {
        constexpr int V = 16 / sizeof(T);
        for (int i = tid; i < n / V; i += kThreads) {
            const uint4 raw = *reinterpret_cast<const uint4*>(in + i * V);
            reinterpret_cast<uint4*>(x)[i] = raw;
            const T* v = reinterpret_cast<const T*>(&raw);
#pragma unroll
            for (int e = 0; e < V; ++e) top = fmaxf(top, wide(v[e]));
        }
        for (int i = n / V * V + tid; i < n; i += kThreads) { x[i] = in[i]; top = fmaxf(top, wide(x[i])); }
    } else {
#pragma unroll 8
        for (int i = tid; i < n; i += kThreads) { const T v = in[i]; x[i] = v; top = fmaxf(top, wide(v)); }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) s.warp_top[warp] = top;
    __syncthreads();
    if (tid < 32) {
        top = tid < kWarps ? s.warp_top[tid] : -INFINITY;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");      // (all CTAs of the cluster run)
    if (tid < ctas) st_remote(remote_of(s.tops + rank, tid), top);
    meet();
    Row r;
    r.top = s.tops[0];
#pragma unroll
    for (int c = 1; c < kMostCtas; ++c) r.top = c < ctas ? fmaxf(r.top, s.tops[c]) : r.top;
    r.bits = bits;
    const bool greedy = !(temperature >= kColdest) || top_k == 1 || min_p > 1.f || r.top == -INFINITY;
    r.step = greedy ? 0.0 : step;
    r.half_scale = (float)(r.step * (2.0 * kBins) / (bits + 1) * (1 - 0x1p-20));          // (less than roundings in fp32 may add: no weight that is not zero lies behind the bins)
    // ---- the border: tokens of larger keys are kept, and of those at it the first `ties` ----
    enum { kNumber, kWeight, kKept };            // tokens into bins, for top-k; weights into bins, for top-p; sums of what is kept
    unsigned border = greedy ? key_of<T>(r.top) : 0, ties = greedy ? 1 : 0xffffffffu, lo = 0, hi = 0xffffffffu;
    int mode = greedy ? kKept : top_k > 0 ? kNumber : top_p < 1.f ? kWeight : kKept, bin = -1, shift = 0, turn = 0;        // bin -1: by the logarithm
    u64 above = 0, target = (u64)top_k;
    bool cut = false, moved = false;
    const u64 least = share(min_p, 1ull << bits, true);
    // (what min-p leaves out has a smaller key than all that it keeps)
    auto keeps = [&](float v, u64 w) { return w >= least || v == r.top ? w : 0; };
    Warp mine = {0, 0, 0};
    const T* run_x = x + first;
    int many = last - first;                     // of the warp's run
    while (mode != kKept) {
        Bins& h = s.bins[turn];
        if (bin < 0 && mode == kNumber) {
#pragma unroll 4
            for (int i = lane; i < many; i += 32) {
                const int at = bin_of(wide(run_x[i]), r);
                if (at < kBins) atomicAdd(h.part[0] + at, 1u);
            }
        } else if (bin < 0) {
#pragma unroll 4
            for (int i = lane; i < many; i += 32) {
                const float v = wide(run_x[i]);
                const int at = bin_of(v, r);
                put(h, min(at, kBins - 1), at < kBins && key_of<T>(v) > border ? weight(v, r, s.table) : 0);
            }
        } else {
            for (int i = lane; i < many; i += 32) {
                const float v = wide(run_x[i]);
                const unsigned k = key_of<T>(v);
                if (k > border && k >= lo && k <= hi && bin_of(v, r) == bin) put(h, (hi - k) >> shift, mode == kNumber ? 1 : weight_apart(v, r, s.table));
            }
        }
        __syncthreads();
        add_groups(h, s.groups[turn][0], rank, ctas);
        meet();
        // (the last turn's bins have been read by all: before they met; so have its groups)
        if (warp == 0) {
            find(s, h, s.groups[turn][0], ctas, bin < 0 ? 0 : above, [&](u64 sum) {
                if (mode != kWeight || bin >= 0) return target;
                // (of all, or of what top-k keeps; one token at least)
                return max(share(top_p, cut ? sum + ties * weight_apart(of_key<T>(border), r, s.table) : sum, true), (u64)1);
            });
        } else {
            for (int i = tid - 32; i < (int)sizeof(Bins) / 16; i += kThreads - 32) reinterpret_cast<uint4*>(s.bins + (turn ^ 1))[i] = make_uint4(0, 0, 0, 0);
        }
        turn ^= 1;
        __syncthreads();
        const int found = s.found;
        const u64 all = s.all;
        target = s.target;
        if (found >= 0) above = s.found_above;
        __syncthreads();                         // (what was found has been read)
        if (found >= 0) {
            if (bin < 0) {
                // The keys of that bin lie between those of its ends, a little further out (rounding of bin_of)
                bin = found;
                const double unit = (double)(bits + 1) / kBins / r.step;
                const float far = fmaxf((float)((double)r.top - (bin + 1.01) * unit), -3.4028235e38f), near = bin == 0 ? r.top : (float)((double)r.top - (bin - 0.01) * unit);
                lo = key_of<T>(far) > 2 ? key_of<T>(far) - 2 : 0;
                hi = max(key_of<T>(fminf(near, r.top)), 3u) + (bin == 0 ? 0 : 2);
                shift = max(0, 32 - __clz(hi - lo) - kBinBits);
                if (!moved) {            // nothing below the keys of this bin will be kept: the others move to the front of the run
                    int held = 0;
                    constexpr int DEEP = 4;
                    const float least_x = lo <= key_of<T>(-INFINITY) ? -INFINITY : of_key<T>(lo);       // (not a NaN)
                    for (int i0 = 0; i0 < many; i0 += 32 * DEEP) {
                        T v[DEEP];
#pragma unroll
                        for (int e = 0; e < DEEP; ++e) v[e] = i0 + 32 * e + lane < many ? run_x[i0 + 32 * e + lane] : T(0.f);
                        __syncwarp();            // (read, by all lanes, before anything is put there)
#pragma unroll
                        for (int e = 0; e < DEEP; ++e) {
                            const int i = i0 + 32 * e + lane;
                            const bool in = i < many && wide(v[e]) >= least_x;
                            const unsigned whom = __ballot_sync(0xffffffffu, in);
                            const int to = held + __popc(whom & ((1u << lane) - 1));
                            if (in) { x[first + to] = v[e]; places[first + to] = (unsigned short)i; }
                            held += __popc(whom);
                        }
                    }
                    __syncwarp();
                    many = held;
                    moved = true;
                }
                continue;
            }
            hi -= (unsigned)found << shift;
            lo = max(lo, hi - ((1u << shift) - 1));
            if (shift > 0) {
                shift = max(0, 32 - __clz(hi - lo) - kBinBits);
                continue;
            }
        }
        // ---- a search has ended, at the value of key hi ----
        if (mode == kNumber) {
            if (found >= 0) {                    // (else top-k keeps all that have a weight)
                cut = true;
                border = hi;
                ties = (unsigned)(top_k - above);
            }
            mode = top_p < 1.f ? kWeight : kKept;
            bin = -1;
        } else {
            if (found >= 0) {
                const u64 w = weight_apart(of_key<T>(hi), r, s.table);
                border = hi;
                ties = (unsigned)((target - above + w - 1) / w);
            } else {                             // among those at top-k's border
                const u64 w = weight_apart(of_key<T>(border), r, s.table);
                ties = min(ties, (unsigned)((target - all + w - 1) / w));
            }
            mode = kKept;
        }
    }
    // ---- sums of the kept tokens by warp, in the vocabulary's order ----
#pragma unroll 2
    for (int i = lane; i < many; i += 32) {
        const float v = wide(run_x[i]);
        const unsigned k = key_of<T>(v);
        const u64 w = greedy ? 1 : weight(v, r, s.table);
        if (k > border) mine.mass += keeps(v, w);
        if (k == border) ++mine.ties;
    }
    mine.mass = warp_total(mine.mass);
    mine.ties = warp_total(mine.ties);
    if (lane < ctas) st_remote(remote_of(s.warps + rank * kWarps + warp, lane), make_uint4((unsigned)mine.mass, (unsigned)(mine.mass >> 32), mine.ties, 0));
    meet();
    auto kept_weight = [&](float v) { return keeps(v, greedy ? 1 : weight_apart(v, r, s.table)); };
    const u64 border_w = border ? kept_weight(of_key<T>(border)) : 0;
    // ---- warp 0 of each CTA looks for the warp of the cluster that has the token; lane l has kPer warps in their order ----
    constexpr int kPer = kMostCtas * kWarps / 32;
    if (warp == 0) {
        uint4 v[kPer];
        unsigned lane_ties = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int w = kPer * lane + i;
            v[i] = make_uint4(0, 0, 0, 0);
            if (w < ctas * kWarps) v[i] = reinterpret_cast<const uint4*>(s.warps)[w];
            lane_ties += v[i].z;
        }
        unsigned to = warp_prefix(lane_ties, lane) - lane_ties;          // (equal tokens before)
        u64 mass[kPer], sum = 0;
        unsigned ties_to[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            ties_to[i] = to;
            to += v[i].z;
            mass[i] = ((u64)v[i].y << 32) + v[i].x + (u64)(min(to, ties) - min(ties_to[i], ties)) * border_w;
            sum += mass[i];
        }
        u64 before = warp_prefix(sum, lane);
        const u64 total = __shfl_sync(0xffffffffu, before, 31);
        before -= sum;
        u64 target = share(u, total, false);
        if (total > 0 && target >= total) target = total - 1;
        if (lane == 0) s.owner = -1;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (target >= before && target < before + mass[i]) {
                s.owner = kPer * lane + i;
                s.before = before;
                s.ties_before = ties_to[i];
                s.found_above = target;
            }
            before += mass[i];
        }
    }
    __syncthreads();                              // (what the CTAs push has arrived before they met: each may leave)
    if (s.owner < 0) {                            // nothing to choose from
        if (rank == 0 && tid == 0) a.out[row] = 0;
        return;
    }
    if (s.owner != rank * kWarps + warp) return;
    // ---- this warp's run has the token: what is kept, 32 at a time, in order ----
    u64 before = s.before;
    target = s.found_above;
    unsigned at_border = s.ties_before;
    int* next = reinterpret_cast<int*>(s.bins) + warp * 64;                   // (the bins are done with)
    int held = 0;
    for (int i0 = 0; i0 < many || held > 0; i0 += 32) {
        const int i = i0 + lane;
        const unsigned k = i < many ? key_of<T>(wide(run_x[i])) : 0;
        const unsigned tie = __ballot_sync(0xffffffffu, i < many && k == border), earlier = (1u << lane) - 1;
        const bool in = i < many && (k > border || (k == border && at_border + __popc(tie & earlier) < ties));
        at_border += __popc(tie);
        const unsigned whom = __ballot_sync(0xffffffffu, in);
        if (in) next[held + __popc(whom & earlier)] = i;
        held += __popc(whom);
        __syncwarp();
        if (held < 32 && i0 + 32 < many) continue;
        const int now = min(held, 32), place = lane < now ? next[lane] : -1, rest = next[32 + lane];
        __syncwarp();
        const u64 to = before + warp_prefix(place >= 0 ? kept_weight(wide(run_x[place])) : 0, lane);
        const unsigned hit = __ballot_sync(0xffffffffu, target < to);
        if (hit) {
            if (lane == __ffs(hit) - 1) a.out[row] = base + first + (moved ? (int)places[first + place] : place);
            return;
        }
        before = __shfl_sync(0xffffffffu, to, 31);
        held -= now;
        if (lane < held) next[lane] = rest;
        __syncwarp();
    }
}

constexpr size_t kMostShared = 227 * 1024;
constexpr int kMostVocab = 1 << 18;
// Of a slice: logits and 16 bits of place for each.
constexpr size_t shared_bytes(int slice, size_t size) { return (sizeof(Shared) + 15) / 16 * 16 + slice * (size + sizeof(unsigned short)); }
static_assert(shared_bytes(kMostVocab / kMostCtas, sizeof(float)) <= kMostShared, "");

template <typename T>
int launch(const b200gptq_sample_args& a, cudaStream_t stream) {
    // CTAs per row: as many as the SMs hold two of, a slice of 1024 tokens or more, and enough that a slice leaves an SM room for two (what eight cannot hold so
    // takes more).  Measured, us, with this and with other numbers of CTAs per row, temperatures of 0.6 to 1.2.  Top-k 50, then top-p 0.95: 1 row of 32000, 8 CTAs 17.6, 4 18.2, 1
    // 21.9; 64 rows of 32000, 4 21.8, 2 25.4, 8 41.7; 64 of 50272, 4 24.9, 2 23.8, 8 43.8; 300 of 4099, 1 29.6, 2 52; 20 of 100003 in fp32, 8 31.9, 4 29.0; 128 of them, 8 133, 4, which
    // leave an SM one CTA, 124.  Top-p 0.95 alone, where more is searched: 64 of 50272, 4 35.8, 2 40.4, 8 46.6; 300 of 4099, 1 28.2, 2 42; 20 of 100003, 8 38.9, 4 42.6; 128, 8 146, 4 159.
    int cluster_bits = 0;
    while (cluster_bits < 3 && ((long long)a.rows << (cluster_bits + 1) <= 2LL * sm_count() || shared_bytes((a.vocab >> cluster_bits) + 8, sizeof(T)) > 113 * 1024) &&
           a.vocab >> (cluster_bits + 1) >= 1024)
        ++cluster_bits;
    // (slices begin at multiples of 16 bytes)
    const int slice = (((a.vocab + (1 << cluster_bits) - 1) >> cluster_bits) + 7) / 8 * 8;
    int log2v = 0;
    while (1 << log2v < a.vocab) ++log2v;
    const int bits = 62 - log2v < 49 ? 62 - log2v : 49;
    const size_t smem = shared_bytes(slice, sizeof(T));
    static const bool pdl = [] {
        const char* e = std::getenv("B200GPTQ_PDL");
        return !(e && e[0] == '0');
    }();
    static std::once_flag once[64];
    static cudaError_t result[64];
    int dev = 0;
    B200GPTQ_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return B200GPTQ_ERR_TOO_LARGE;
    auto* kernel = sample_kernel<T>;
    std::call_once(once[dev], [&] { result[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostShared); });
    B200GPTQ_CUDA_TRY(result[dev]);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.rows << cluster_bits);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    if (cluster_bits) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = 1 << cluster_bits;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    B200GPTQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a, slice, cluster_bits, bits));
    return B200GPTQ_OK;
}

}  // namespace
}  // namespace b200gptq

using namespace b200gptq;

extern "C" B200GPTQ_API int b200gptq_sample(const b200gptq_sample_args* args, void* stream) {
    if (!args) return B200GPTQ_ERR_NULL_POINTER;
    const b200gptq_sample_args& a = *args;
    if (!a.logits || !a.uniform || !a.out) return B200GPTQ_ERR_NULL_POINTER;
    if (a.dtype != B200GPTQ_F16 && a.dtype != B200GPTQ_BF16 && a.dtype != B200GPTQ_F32) return B200GPTQ_ERR_SHAPE;
    if (a.rows < 1 || a.vocab < 1 || a.logits_stride < 0) return B200GPTQ_ERR_SHAPE;
    if (a.vocab > kMostVocab || a.rows > 1 << 27) return B200GPTQ_ERR_TOO_LARGE;
    const int size = a.dtype == B200GPTQ_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(a.logits) & (size - 1) || (reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.top_k)) & 7u ||
        (reinterpret_cast<uintptr_t>(a.uniform) | reinterpret_cast<uintptr_t>(a.temperature) | reinterpret_cast<uintptr_t>(a.top_p) | reinterpret_cast<uintptr_t>(a.min_p)) & 3u)
        return B200GPTQ_ERR_ALIGNMENT;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return a.dtype == B200GPTQ_F16 ? launch<__half>(a, s) : a.dtype == B200GPTQ_BF16 ? launch<__nv_bfloat16>(a, s) : launch<float>(a, s);
}
