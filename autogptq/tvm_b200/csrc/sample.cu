// b200gptq_sample: the next token under temperature, top-k, top-p and min-p, from a given random number; see include/b200gptq.h.
//
//   w_v = exp((x_v - max x) / T),  kept: a beginning of the order "larger x, then lower v",  token: the first v whose kept sum passes u * (sum of all kept)
//
// All that decides is exact: weights are integers (units of 2^-F of the largest, F so that the vocabulary's sum fits 62 bits; exp2 in 64 bits from a table of 64 powers
// and a Taylor polynomial of degree 5, after P. T. P. Tang, "Table-driven implementation of the exponential function", 1989), their sums have no order, and the
// products p * S and u * S are taken in 128 bits. Sums in fp32 would put the border off by more than what lies between two tokens of a large vocabulary.
//
// A cluster of CTAs shares a row, each keeps a slice of the logits in shared memory. The number of kept tokens follows from histograms: 1024 bins, linear in
// the logarithm of the weight, with the number and the sum of the tokens in each (the order of x and of the bins is the same), then the bin in which top-k or top-p ends
// again by the bits of x until one value is left. Tokens of that value are kept from the lowest on. The CTAs of a cluster read each other's bins
// through distributed shared memory and all come to the same results.
#include <cuda_bf16.h>

#include <cstddef>
#include <cstdlib>
#include <mutex>

#include "common.cuh"

namespace b200gptq {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 1024, kFine = 512, kFineBits = 9, kMostCtas = 8, kTable = 64;
constexpr float kColdest = 1e-18f;       // temperatures below count as 0, so that no scale leaves fp32
typedef unsigned long long u64;

template <typename T> __device__ __forceinline__ float wide(T x);
template <> __device__ __forceinline__ float wide(float x) { return x; }
template <> __device__ __forceinline__ float wide(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float wide(__nv_bfloat16 x) { return __bfloat162float(x); }

// Larger x, larger key; a NaN counts as minus infinity.
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __float_as_uint(x == 0.f ? 0.f : x);
    return x != x ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

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
__device__ __forceinline__ uint2 ld_remote2(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
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

template <int N> struct Bins { unsigned count[N], low[N], high[N]; };
struct Warp { u64 mass; unsigned ties, unused; };       // of a warp's tokens: sum above the border, how many are at it
struct Shared {
    Bins<kBins> bins;
    Bins<kFine> fine[2];
    double table[kTable];
    Warp warps[kWarps];
    u64 scan_mass[kWarps], found_mass;
    unsigned scan_count[kWarps], found_count;
    float top, warp_top[kWarps];
    int found;
};

// Everything of a row that the CTAs of its cluster agree on.
struct Row {
    float top, half_scale;               // largest logit; bins per half a unit of x
    double step;                         // 64 log2(e) / T
    int bits;                            // F
};
__device__ __forceinline__ u64 weight(float x, const Row& r, const double* table) {
    if (x == r.top) return 1ull << r.bits;
    const double z = ((double)x - (double)r.top) * r.step;
    if (!(z > -64.0 * 64)) return 0;
    const double magic = 6755399441055744.0, y = z + magic, f = z - (y - magic);             // z = i + f, |f| <= 1/2
    const int i = (int)(unsigned)__double_as_longlong(y);
    constexpr double l = 0.69314718055994530942 / kTable;
    double p = fma(f, l * l * l * l * l / 120, l * l * l * l / 24);
    p = fma(f, p, l * l * l / 6);
    p = fma(f, p, l * l / 2);
    p = fma(f, p, l);
    p = fma(f, p, 1.0);
    const u64 b = (u64)__double_as_longlong(p * table[i & (kTable - 1)]);                    // [1/2, 2): near 1 the polynomial may be below it
    const int e = (int)(b >> 52) - 1023 + (i >> 6) + r.bits, down = 52 - e;
    const u64 m = (b & ((1ull << 52) - 1)) | 1ull << 52;
    return down > 54 ? 0 : ((m >> (down - 1)) + 1) >> 1;                                     // (down is 3 at least: F is 49 at most)
}
// Bin of x, kBins or more where its weight is zero.
__device__ __forceinline__ int bin_of(float x, const Row& r) {
    if (x == r.top) return 0;
    const float f = (0.5f * r.top - 0.5f * x) * r.half_scale;
    return f < (float)kBins ? (int)f : kBins;                                                // (a NaN: kBins)
}

template <int N> __device__ __forceinline__ void put(Bins<N>& h, unsigned at, u64 w, bool counts) {
    if (counts) atomicAdd(h.count + at, 1u);
    const unsigned low = (unsigned)w, old = atomicAdd(h.low + at, low), high = (unsigned)(w >> 32) + (old + low < low ? 1u : 0u);
    if (high) atomicAdd(h.high + at, high);
}

// The thread's bins (PER adjacent ones) of all CTAs of the cluster added up, and what lies above them.  The CTAs have met before.
template <int PER> struct Sums {
    unsigned n[PER];
    u64 m[PER], count_before, mass_before, mass_all;

    template <int N> __device__ __forceinline__ void add_up(Shared& s, const Bins<N>& mine, int ctas, bool counts) {
        static_assert(N == PER * kThreads, "");
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
#pragma unroll
        for (int i = 0; i < PER; ++i) n[i] = 0, m[i] = 0;
        if (ctas == 1) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                n[i] = mine.count[tid * PER + i];
                m[i] = ((u64)mine.high[tid * PER + i] << 32) + mine.low[tid * PER + i];
            }
        } else {
            const int bin = tid * PER;
#pragma unroll
            for (int half = 0; half < 2; ++half) {        // (all loads of four CTAs on their way at once)
                uint2 c[4], l[4], h[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    c[r] = l[r] = h[r] = make_uint2(0, 0);
                    if (4 * half + r >= ctas) continue;
                    if constexpr (PER == 2) {
                        if (counts) c[r] = ld_remote2(remote_of(mine.count + bin, 4 * half + r));
                        l[r] = ld_remote2(remote_of(mine.low + bin, 4 * half + r));
                        h[r] = ld_remote2(remote_of(mine.high + bin, 4 * half + r));
                    } else {
                        if (counts) c[r].x = ld_remote(remote_of(mine.count + bin, 4 * half + r));
                        l[r].x = ld_remote(remote_of(mine.low + bin, 4 * half + r));
                        h[r].x = ld_remote(remote_of(mine.high + bin, 4 * half + r));
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    n[0] += c[r].x;
                    m[0] += ((u64)h[r].x << 32) + l[r].x;
                    if constexpr (PER == 2) { n[1] += c[r].y; m[1] += ((u64)h[r].y << 32) + l[r].y; }
                }
            }
        }
        u64 count = 0, mass = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) { count += n[i]; mass += m[i]; }
        const u64 count_to = counts ? warp_prefix(count, lane) : 0, mass_to = warp_prefix(mass, lane);
        if (lane == 31) { s.scan_count[warp] = (unsigned)count_to; s.scan_mass[warp] = mass_to; }
        if (tid == 0) s.found = -1;
        __syncthreads();
        count_before = count_to - count;
        mass_before = mass_to - mass;
        mass_all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) { count_before += s.scan_count[w]; mass_before += s.scan_mass[w]; }
            mass_all += s.scan_mass[w];
        }
    }
    // The first bin, from the top on, with which count or mass (and what lies `above` all of them) reaches its target, with what lies above it among
    // the bins, in `s`; s.found is -1 on entry and where there is none.
    __device__ __forceinline__ void find(Shared& s, bool by_count, u64 target, u64 above) const {
        u64 count_to = count_before, mass_to = mass_before;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const u64 before = above + (by_count ? count_to : mass_to), after = before + (by_count ? n[i] : m[i]);
            if (before < target && after >= target) {
                s.found = threadIdx.x * PER + i;
                s.found_count = (unsigned)count_to;
                s.found_mass = mass_to;
            }
            count_to += n[i];
            mass_to += m[i];
        }
        __syncthreads();
    }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
sample_kernel(const __grid_constant__ b200gptq_sample_args a, int slice, int cluster_bits, int bits) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem);
    T* x = reinterpret_cast<T*>(smem + (sizeof(Shared) + 15) / 16 * 16);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ctas = 1 << cluster_bits, row = blockIdx.x >> cluster_bits, rank = blockIdx.x & (ctas - 1);
    const int base = min(rank * slice, a.vocab), n = min(slice, a.vocab - base);
    // A warp's tokens: a run of the slice
    const int run = (slice + kWarps - 1) / kWarps, first = min(warp * run, n), last = min(first + run, n);
    static_assert(offsetof(Shared, fine) == sizeof(Bins<kBins>), "");
    for (int i = tid; i < kBins * 3 + 2 * kFine * 3; i += kThreads) reinterpret_cast<unsigned*>(&s.bins)[i] = 0;
    auto meet = [&] {
        if (ctas > 1) cluster_sync();
        else __syncthreads();
    };
    if (tid < kTable) s.table[tid] = exp2((double)tid / kTable);
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride + base;
    const float temperature = a.temperature ? a.temperature[row] : 1.f, top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f, u = a.uniform[row];
    const long long top_k = a.top_k ? a.top_k[row] : 0;
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
        if (tid == 0) s.top = top;
    }
    meet();
    Row r;
    r.top = s.top;
    if (ctas > 1) {
        float others[kMostCtas];
#pragma unroll
        for (int c = 0; c < kMostCtas; ++c) others[c] = c < ctas ? __uint_as_float(ld_remote(remote_of(&s.top, c))) : -INFINITY;
#pragma unroll
        for (int c = 0; c < kMostCtas; ++c) r.top = fmaxf(r.top, others[c]);
    }
    r.bits = bits;
    const bool greedy = !(temperature >= kColdest) || top_k == 1 || min_p > 1.f || r.top == -INFINITY;
    r.step = greedy ? 0.0 : 64 * 1.4426950408889634074 / (double)temperature;
    r.half_scale = (float)(r.step * (2.0 * kBins / 64) / (bits + 1));
    // ---- the border: tokens of larger keys are kept, and of those at it the first `ties` ----
    unsigned border = 0, ties = 0xffffffffu;
    if (greedy) {
        border = key_of(r.top);
        ties = 1;
    } else if (top_k > 0 || top_p < 1.f) {
        const bool counts = top_k > 0;
#pragma unroll 4
        for (int i = first + lane; i < last; i += 32) {
            const float v = wide(x[i]);
            const int bin = bin_of(v, r);
            if (bin < kBins) put(s.bins, bin, weight(v, r, s.table), counts);
        }
        meet();
        Sums<kBins / kThreads> whole;
        whole.add_up(s, s.bins, ctas, counts);
        int level = 0;
        u64 above_count = 0, above_mass = 0;
        // The value of x at which the first `target` tokens (by_count), or the shortest beginning that weighs `target`, end, and what lies above it
        auto search = [&](bool by_count, u64 target, unsigned& key) {
            whole.find(s, by_count, target, 0);
            const int bin = s.found;
            if (bin < 0) return false;
            above_count = s.found_count;
            above_mass = s.found_mass;
            // The keys of that bin lie between those of its ends, a little further out (rounding of bin_of)
            const double unit = 64.0 * (bits + 1) / kBins / r.step;
            const float far = fmaxf((float)((double)r.top - (bin + 1.01) * unit), -3.4028235e38f), near = bin == 0 ? r.top : (float)((double)r.top - (bin - 0.01) * unit);
            unsigned lo = key_of(far) > 2 ? key_of(far) - 2 : 0, hi = max(key_of(fminf(near, r.top)), 3u) + (bin == 0 ? 0 : 2);
            int shift;
            do {
                shift = max(0, 32 - __clz(hi - lo) - kFineBits);
                Bins<kFine>& h = s.fine[level & 1];
#pragma unroll 4
                for (int i = first + lane; i < last; i += 32) {
                    const float v = wide(x[i]);
                    const unsigned k = key_of(v);
                    if (k >= lo && k <= hi && bin_of(v, r) == bin) put(h, (hi - k) >> shift, weight(v, r, s.table), counts);
                }
                meet();
                // (the other one has been read by all: it was added up before they met)
                ++level;
                for (int i = tid; i < kFine * 3; i += kThreads) reinterpret_cast<unsigned*>(s.fine + (level & 1))[i] = 0;
                Sums<kFine / kThreads> part;
                part.add_up(s, h, ctas, counts);
                part.find(s, by_count, target, by_count ? above_count : above_mass);
                above_count += s.found_count;
                above_mass += s.found_mass;
                hi -= (unsigned)s.found << shift;
                lo = max(lo, hi - ((1u << shift) - 1));
                __syncthreads();         // (what was found has been read)
                if (tid == 0) s.found = -1;
            } while (shift > 0);
            __syncthreads();
            key = hi;
            return true;
        };
        u64 sum = whole.mass_all;        // of what top-k keeps
        const bool cut = top_k > 0 && search(true, (u64)top_k, border);
        if (cut) {
            ties = (unsigned)(top_k - above_count);
            sum = above_mass + ties * weight(of_key(border), r, s.table);
        }
        if (top_p < 1.f) {
            u64 target = share(top_p, sum, true);
            if (target == 0) target = 1;
            unsigned key = 0;
            if (search(false, target, key)) {
                const u64 w = weight(of_key(key), r, s.table), need = (target - above_mass + w - 1) / w;
                ties = key == border && cut ? min(ties, (unsigned)need) : (unsigned)need;
                border = key;
            }
        }
    }
    // ---- sums of the kept tokens by warp, in the vocabulary's order ----
    const u64 least = share(min_p, 1ull << bits, true);
    // (what min-p leaves out has a smaller key than all that it keeps)
    auto kept_weight = [&](float v) { const u64 w = greedy ? 1 : weight(v, r, s.table); return w >= least || v == r.top ? w : 0; };
    Warp mine = {0, 0, 0};
#pragma unroll 4
    for (int i = first + lane; i < last; i += 32) {
        const float v = wide(x[i]);
        const unsigned k = key_of(v);
        if (k > border) mine.mass += kept_weight(v);
        else if (k == border) ++mine.ties;
    }
    mine.mass = warp_total(mine.mass);
    mine.ties = warp_total(mine.ties);
    if (lane == 0) s.warps[warp] = mine;
    meet();
    const u64 border_w = border ? kept_weight(of_key(border)) : 0;
    // every warp looks at all warps of the cluster, 32 at a time: those before it, and all
    u64 before = 0, total = 0;
    unsigned ties_before = 0, ties_all = 0;
    for (int w0 = 0; w0 < ctas * kWarps; w0 += 32) {
        const int w = w0 + lane;
        Warp other = {0, 0, 0};
        if (w < ctas * kWarps) {
            if (ctas > 1) {
                const uint32_t at = remote_of(s.warps + (w % kWarps), w / kWarps);
                const uint2 mass = ld_remote2(at);
                other.mass = (u64)mass.y << 32 | mass.x;
                other.ties = ld_remote(at + 8);
            } else {
                other = s.warps[w];
            }
        }
        const u64 to = ties_all + warp_prefix((u64)other.ties, lane);
        const u64 taken = min(to, (u64)ties) - min(to - other.ties, (u64)ties);
        const u64 mass = other.mass + taken * border_w;
        const bool earlier = w < rank * kWarps + warp;
        before += warp_total(earlier ? mass : 0);
        total += warp_total(mass);
        ties_before += warp_total(earlier ? other.ties : 0u);
        ties_all += warp_total(other.ties);
    }
    if (ctas > 1) cluster_sync();                 // (nobody leaves while others read)
    u64 target = share(u, total, false);
    if (total > 0 && target >= total) target = total - 1;
    if (total == 0) {                             // nothing to choose from
        if (rank == 0 && tid == 0) a.out[row] = 0;
        return;
    }
    const u64 own = mine.mass + (min((u64)ties_before + mine.ties, (u64)ties) - min((u64)ties_before, (u64)ties)) * border_w;
    if (target < before || target >= before + own) return;
    // ---- this warp's run has the token: a run of it per lane, then that one again, a token per lane ----
    int begin = first, end = last;
    unsigned at_border = ties_before;
    while (true) {
        const int each = (end - begin + 31) / 32, from = min(begin + lane * each, end), to = min(from + each, end);
        u64 mass = 0;
        unsigned mine_ties = 0;
        for (int i = from; i < to; ++i) {
            const float v = wide(x[i]);
            const unsigned k = key_of(v);
            if (k > border) mass += kept_weight(v);
            else if (k == border) ++mine_ties;
        }
        const unsigned ties_to = at_border + warp_prefix(mine_ties, lane);
        mass += (u64)(min(ties_to, ties) - min(ties_to - mine_ties, ties)) * border_w;
        const u64 to_here = before + warp_prefix(mass, lane);
        const unsigned hit = __ballot_sync(0xffffffffu, target < to_here);
        const int who = __ffs(hit) - 1;
        begin = __shfl_sync(0xffffffffu, from, who);
        end = __shfl_sync(0xffffffffu, to, who);
        before = __shfl_sync(0xffffffffu, to_here - mass, who);
        at_border = __shfl_sync(0xffffffffu, ties_to - mine_ties, who);
        if (end - begin <= 1) break;
    }
    if (lane == 0) a.out[row] = base + begin;
}

template <typename T>
int launch(const b200gptq_sample_args& a, cudaStream_t stream) {
    // CTAs per row: as many as the SMs hold three of, a slice of 1024 tokens or more, and enough that a slice leaves an SM room for three (51 KB; what eight cannot
    // hold so takes more).
    int cluster_bits = 0;
    while (cluster_bits < 3 && ((long long)a.rows << (cluster_bits + 1) <= 3LL * sm_count() || (long long)a.vocab * sizeof(T) > 51200LL << cluster_bits) &&
           a.vocab >> (cluster_bits + 1) >= 1024)
        ++cluster_bits;
    // (slices begin at multiples of 16 bytes)
    const int slice = (((a.vocab + (1 << cluster_bits) - 1) >> cluster_bits) + 7) / 8 * 8;
    int log2v = 0;
    while (1 << log2v < a.vocab) ++log2v;
    const int bits = 62 - log2v < 49 ? 62 - log2v : 49;
    const size_t smem = (sizeof(Shared) + 15) / 16 * 16 + (size_t)slice * sizeof(T);
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
    std::call_once(once[dev], [&] { result[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)((sizeof(Shared) + 15) / 16 * 16 + 128 * 1024 + 64)); });
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
    if (a.vocab > 1 << 18 || a.rows > 1 << 27) return B200GPTQ_ERR_TOO_LARGE;
    const int size = a.dtype == B200GPTQ_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(a.logits) & (size - 1) || (reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.top_k)) & 7u ||
        (reinterpret_cast<uintptr_t>(a.uniform) | reinterpret_cast<uintptr_t>(a.temperature) | reinterpret_cast<uintptr_t>(a.top_p) | reinterpret_cast<uintptr_t>(a.min_p)) & 3u)
        return B200GPTQ_ERR_ALIGNMENT;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return a.dtype == B200GPTQ_F16 ? launch<__half>(a, s) : a.dtype == B200GPTQ_BF16 ? launch<__nv_bfloat16>(a, s) : launch<float>(a, s);
}
