// b200gptq_attn for few query rows per key head: the single tokens of a decode step (and short runs of them), over a windowed cache or behind
// a shared prefix.
//
//   S = Q K^T,  w = softmax(scale S) over the visible keys,  O = w V
//
// The bytes of K and V bound it (4 flop per byte and row of Q), so a CTA holds up to 16 or 32 rows of Q (all that share a key head: the heads
// of its group, the tokens of a short run, and with a prefix all sequences of the batch) and streams the keys once.  Every warp takes blocks of 16
// keys on its own and goes from global memory to mma.sync fragments without shared memory:
//   * Q K^T: operand B of m16n8k16 wants, from lane (g, c) = (lane / 4, lane % 4), the pairs 2c and 2c + 8 of key g.  Any order of the 16 dims
//     serves as long as Q has the same, so a lane loads 16 bytes = 8 adjacent dims of key g, which are the operand of two products;
//   * w V: operand B wants pairs of keys of one dim.  A lane loads 8 adjacent dims of keys 2c, 2c + 1, 2c + 8, 2c + 9 and pairs them with byte
//     permutations; column g of product (h, i) is dim 64 h + 8 g + i;
//   * the accumulators of S are operand A of the second product as they lie.
// The next block's keys are requested when this block's have been multiplied, its values likewise, so that 6 to 8 KB per warp are on their way.
//
// The key range is split over a cluster of up to 8 CTAs, which add up through distributed shared memory, each a slice of the dims.  With a prefix
// there are two launches: the first takes the prefix, split over CTAs whose sums (fp32) go to scratch; the second takes each sequence's own rows
// meanwhile, waits for the first (griddepcontrol.wait) and adds everything up.  All sums are in a fixed order.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "attn.cuh"
#include "attn.h"

namespace b200gptq {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32, kBlock = 16, kMaxSplit = kAttnMaxSplit;
static_assert(kWarps * kBlock == kAttnRowsKeys, "");

template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ void st_cluster(const float* local, int rank, float v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote), "f"(v) : "memory");
}

// Shared memory, in floats: the warps' sums [warp][row][HD + 4], their maxima and denominators, the slices that the CTAs of the cluster push
// [split][row][HD / splits] with maxima and denominators, a flag per row; the queries (padded rows).
template <int HD, int MT> struct Lay {
    static constexpr int R = 16 * MT, LD = HD + 4, QLD = HD + 8;
    static constexpr int acc = 0, ml = acc + kWarps * R * LD, slice = ml + 2 * kWarps * R, slice_ml = slice + R * HD,
                         flags = slice_ml + 2 * kMaxSplit * R, q = flags + R, total = q + R * QLD / 2;
};

// PREFIX: rows (b, t, g) of one key head against the prefix, sums to `part`.  Otherwise: rows (t, g) of one sequence and key head against its cache
// (and the sums of the prefix).  A row tile is blockIdx.x / splits % row_tiles.
template <typename T, int HD, int MT, bool PREFIX>
__global__ void __launch_bounds__(kThreads, 1)
attn_rows_kernel(const __grid_constant__ b200gptq_attn_args a, float* __restrict__ part, int splits, int row_tiles, int parts) {
    using L = Lay<HD, MT>;
    constexpr int R = L::R, SEG = HD / 32, HH = HD / 64;
    extern __shared__ __align__(16) float sm[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int G = a.heads / a.kv_heads, window = a.window ? a.window : 1 << 30;
    const int split = blockIdx.x % splits, unit = blockIdx.x / splits, tile = unit % row_tiles;
    const int kh = unit / row_tiles % a.kv_heads, b0 = unit / row_tiles / a.kv_heads;        // (PREFIX: b0 = 0)
    // What is read below was written before the launch in front of this one ended (window) or began (behind the prefix launch, which lets this one
    // start only after it has itself waited; the loads by-pass L1).
    if (!PREFIX && splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    if (PREFIX || !a.prefix) asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");

    const int row0 = tile * R, rows_all = (PREFIX ? a.batch : 1) * a.tokens * G;
    int p0 = 0, count = a.tokens;
    if constexpr (!PREFIX) { p0 = attn_pos(a, b0); count = attn_count(a, b0); }
    const int nrows = min(R, (PREFIX ? rows_all : count * G) - row0);
    if (nrows <= 0) {                         // padding: every CTA of the cluster leaves
        if (!PREFIX && a.prefix) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    // ---- queries ----
    T* qs = reinterpret_cast<T*>(sm + L::q);
    for (int i = threadIdx.x; i < R * HD / 8; i += kThreads) {
        const int r = i / (HD / 8), d = i % (HD / 8) * 8, idx = row0 + min(r, nrows - 1), head = kh * G + idx % G, tok = idx / G;
        const int bb = PREFIX ? tok / a.tokens : b0, t = PREFIX ? tok - bb * a.tokens : tok;
        *reinterpret_cast<uint4*>(qs + r * L::QLD + d) = __ldcg(reinterpret_cast<const uint4*>(
            static_cast<const T*>(a.q) + bb * a.q_stride[0] + t * a.q_stride[1] + head * a.q_stride[2] + d));
    }
    // ---- keys ----
    AttnRange range = {0, 0, a.prefix};
    const int p_lo = p0 + row0 / G, p_hi = p0 + (row0 + nrows - 1) / G;
    if constexpr (!PREFIX) range = attn_range(p_lo, p_hi, window, a.sinks, a.max_seq);
    const int nb_s = (range.s_end + kBlock - 1) / kBlock, nb = nb_s + (range.w_end - range.w_start + kBlock - 1) / kBlock;
    const int first = (int)((long long)nb * split / splits), last = (int)((long long)nb * (split + 1) / splits);
    const T *kb, *vb;
    long long ks, vs;
    if constexpr (PREFIX) {
        kb = static_cast<const T*>(a.k_prefix) + kh * a.k_prefix_stride[0]; ks = a.k_prefix_stride[1];
        vb = static_cast<const T*>(a.v_prefix) + kh * a.v_prefix_stride[0]; vs = a.v_prefix_stride[1];
    } else {
        kb = static_cast<const T*>(a.k_cache) + b0 * a.k_stride[0] + kh * a.k_stride[1]; ks = a.k_stride[2];
        vb = static_cast<const T*>(a.v_cache) + b0 * a.v_stride[0] + kh * a.v_stride[1]; vs = a.v_stride[2];
    }
    uint4 kr[2][SEG], vr[4][HH];
    auto block = [&](int i, int& j0, int& end) {
        const bool s = i < nb_s;
        j0 = s ? kBlock * i : range.w_start + kBlock * (i - nb_s);
        end = s ? range.s_end : range.w_end;
    };
    // (rows behind the end of the range: its last row again, with weight zero)
    auto load_k = [&](int i) {
        int j0, end;
        block(i, j0, end);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const T* src = kb + min(j0 + 8 * n + g, end - 1) * ks + 8 * c;
#pragma unroll
            for (int s = 0; s < SEG; ++s) kr[n][s] = __ldcg(reinterpret_cast<const uint4*>(src + 32 * s));
        }
    };
    auto load_v = [&](int i) {
        int j0, end;
        block(i, j0, end);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const T* src = vb + min(j0 + 2 * c + (n & 1) + 4 * (n & 2), end - 1) * vs + 8 * g;
#pragma unroll
            for (int h = 0; h < HH; ++h) vr[n][h] = __ldcg(reinterpret_cast<const uint4*>(src + 64 * h));
        }
    };
    int i = first + warp;
    if (i < last) { load_k(i); load_v(i); }
    __syncthreads();

    const float scale = a.scale * kLog2e;
    float acc[MT][8 * HH][4], m[MT][2], l[MT][2];
    int pr[MT][2];                            // positions of the lane's rows
    uint4 qf[MT == 1 ? MT : 1][SEG][2];       // (two row tiles read theirs from shared memory each time: registers)
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int n = 0; n < 8 * HH; ++n) acc[t][n][0] = acc[t][n][1] = acc[t][n][2] = acc[t][n][3] = 0.f;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            m[t][r] = -INFINITY; l[t][r] = 0.f;
            pr[t][r] = p0 + (row0 + min(16 * t + 8 * r + g, nrows - 1)) / G;
            if constexpr (MT == 1)
#pragma unroll
                for (int s = 0; s < SEG; ++s) qf[t][s][r] = *reinterpret_cast<const uint4*>(qs + (8 * r + g) * L::QLD + 32 * s + 8 * c);
        }
    }
    for (; i < last; i += kWarps) {
        int j0, end;
        block(i, j0, end);
        float s[MT][2][4];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
#pragma unroll
            for (int n = 0; n < 2; ++n) s[t][n][0] = s[t][n][1] = s[t][n][2] = s[t][n][3] = 0.f;
#pragma unroll
            for (int e = 0; e < SEG; ++e) {
                uint4 x, y;
                if constexpr (MT == 1) { x = qf[t][e][0]; y = qf[t][e][1]; }
                else {
                    x = *reinterpret_cast<const uint4*>(qs + (16 * t + g) * L::QLD + 32 * e + 8 * c);
                    y = *reinterpret_cast<const uint4*>(qs + (16 * t + 8 + g) * L::QLD + 32 * e + 8 * c);
                }
                const uint32_t a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w};
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    mma16<T>(s[t][n], a0, kr[n][e].x, kr[n][e].y);
                    mma16<T>(s[t][n], a1, kr[n][e].z, kr[n][e].w);
                }
            }
        }
        if (i + kWarps < last) load_k(i + kWarps);
        bool whole = j0 + kBlock <= end;      // every row of the tile sees the whole block
        if constexpr (!PREFIX) whole = whole && j0 + kBlock - 1 <= p_lo && (j0 > p_hi - window || j0 + kBlock <= a.sinks);
        uint32_t w[MT][4];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = s[t][e >> 1][2 * r + (e & 1)] * scale;
                    if (!whole) {
                        const int j = j0 + 8 * (e >> 1) + 2 * c + (e & 1);
                        bool see = j < end;
                        if constexpr (!PREFIX) see = see && attn_sees(pr[t][r], j, window, a.sinks);
                        x[e] = see ? x[e] : -INFINITY;
                    }
                }
                float up = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, 1));
                up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, 2));
                up = fmaxf(up, m[t][r]);
                const float safe = up == -INFINITY ? 0.f : up, corr = exp2_fast(m[t][r] - safe);
                m[t][r] = up;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = exp2_fast(x[e] - safe);
                l[t][r] = l[t][r] * corr + ((x[0] + x[1]) + (x[2] + x[3]));
#pragma unroll
                for (int n = 0; n < 8 * HH; ++n) { acc[t][n][2 * r] *= corr; acc[t][n][2 * r + 1] *= corr; }
                w[t][r] = Half<T>::pack(x[0], x[1]);
                w[t][2 + r] = Half<T>::pack(x[2], x[3]);
            }
#pragma unroll
        for (int h = 0; h < HH; ++h)
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const uint32_t pick = (n & 1) ? 0x7632u : 0x5410u;
                const uint32_t y0 = __byte_perm(word(vr[0][h], n / 2), word(vr[1][h], n / 2), pick);
                const uint32_t y1 = __byte_perm(word(vr[2][h], n / 2), word(vr[3][h], n / 2), pick);
#pragma unroll
                for (int t = 0; t < MT; ++t) mma16<T>(acc[t][8 * h + n], w[t], y0, y1);
            }
        if (i + kWarps < last) load_v(i + kWarps);
    }
    // ---- the warps' sums ----
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float sum = l[t][r];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const int row = 16 * t + 8 * r + g;
            if (row < nrows) {
                if (c == 0) { sm[L::ml + 2 * (warp * R + row)] = m[t][r]; sm[L::ml + 2 * (warp * R + row) + 1] = sum; }
                float* dst = sm + L::acc + (warp * R + row) * L::LD;
#pragma unroll
                for (int h = 0; h < HH; ++h)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {         // columns 2 c + e: dims 64 h + 8 (2 c + e) ..
                        float4* to = reinterpret_cast<float4*>(dst + 64 * h + 8 * (2 * c + e));
#pragma unroll
                        for (int x = 0; x < 2; ++x)
                            to[x] = make_float4(acc[t][8 * h + 4 * x][2 * r + e], acc[t][8 * h + 4 * x + 1][2 * r + e],
                                                acc[t][8 * h + 4 * x + 2][2 * r + e], acc[t][8 * h + 4 * x + 3][2 * r + e]);
                    }
            }
        }
    if (threadIdx.x < R) reinterpret_cast<int*>(sm + L::flags)[threadIdx.x] = 0;
    __syncthreads();
    if (!PREFIX && splits > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");      // (all CTAs of the cluster run)
    // ---- the CTA's sums: to the scratch, or slice by slice to the CTAs of the cluster ----
    const int slice = PREFIX ? HD : HD / splits;
    const long long rows_total = (long long)a.batch * a.tokens * a.heads;
    for (int x = threadIdx.x; x < nrows * HD; x += kThreads) {
        const int row = x / HD, d = x % HD;
        float cm = -INFINITY, cl = 0.f, ca = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) cm = fmaxf(cm, sm[L::ml + 2 * (w * R + row)]);
        const float safe = cm == -INFINITY ? 0.f : cm;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float e = exp2_fast(sm[L::ml + 2 * (w * R + row)] - safe);
            cl += sm[L::ml + 2 * (w * R + row) + 1] * e;
            ca += sm[L::acc + (w * R + row) * L::LD + d] * e;
        }
        if constexpr (PREFIX) {
            const int idx = row0 + row;
            const long long at = split * rows_total + (long long)(idx / G) * a.heads + kh * G + idx % G;
            part[at * HD + d] = ca;
            if (d == 0) {
                float* ml = part + splits * rows_total * HD + 2 * at;
                ml[0] = cm; ml[1] = cl;
            }
        } else {
            const int to = d / slice;
            st_cluster(sm + L::slice + (split * R + row) * slice + d - to * slice, to, ca);
            if (d - to * slice == 0) {
                st_cluster(sm + L::slice_ml + 2 * (split * R + row), to, cm);
                st_cluster(sm + L::slice_ml + 2 * (split * R + row) + 1, to, cl);
            }
        }
    }
    if constexpr (PREFIX) return;
    if (splits > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
    if (a.prefix) asm volatile("griddepcontrol.wait;" ::: "memory");                        // the prefix's sums
    // ---- this CTA's slice of the dims ----
    int* flags = reinterpret_cast<int*>(sm + L::flags);
    const float* part_ml = part + parts * rows_total * HD;
    for (int x = threadIdx.x; x < nrows * slice; x += kThreads) {
        const int row = x / slice, d = x - row * slice, idx = row0 + row, t = idx / G, head = kh * G + idx % G;
        const long long at = ((long long)b0 * a.tokens + t) * a.heads + head;
        float tm = -INFINITY, tl = 0.f, ta = 0.f;
        for (int r = 0; r < splits; ++r) tm = fmaxf(tm, sm[L::slice_ml + 2 * (r * R + row)]);
        for (int r = 0; r < parts; ++r) tm = fmaxf(tm, __ldcg(part_ml + 2 * (r * rows_total + at)));
        const float safe = tm == -INFINITY ? 0.f : tm;
        for (int r = 0; r < splits; ++r) {
            const float e = exp2_fast(sm[L::slice_ml + 2 * (r * R + row)] - safe);
            tl += sm[L::slice_ml + 2 * (r * R + row) + 1] * e;
            ta += sm[L::slice + (r * R + row) * slice + d] * e;
        }
        for (int r = 0; r < parts; ++r) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(part_ml + 2 * (r * rows_total + at)));
            const float e = exp2_fast(ml.x - safe);
            tl += ml.y * e;
            ta += __ldcg(part + (r * rows_total + at) * HD + split * slice + d) * e;
        }
        const float o = tl != 0.f ? ta / tl : 0.f;
        static_cast<T*>(a.out)[b0 * a.out_stride[0] + t * a.out_stride[1] + head * a.out_stride[2] + split * slice + d] = Half<T>::round(o);
        if (!isfinite(o)) flags[row] = 1;
    }
    // rows of several tokens in one tile: a NaN may come from a row of the cache that this one does not see
    if (p_hi > p_lo) {
        __syncthreads();
        for (int row = warp; row < nrows; row += kWarps)
            if (flags[row]) {
                const int idx = row0 + row;
                attn_row_again<T, HD>(a, b0, idx / G, kh * G + idx % G, p0 + idx / G, split * slice, (split + 1) * slice);
            }
    }
}

template <typename K>
int launch(K* kernel, const b200gptq_attn_args& a, int smem, long long ctas, int cluster, bool pdl, float* part, int splits, int row_tiles,
           int parts, cudaStream_t stream) {
    if (ctas > 0x7fffffff) return B200GPTQ_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    B200GPTQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a, part, splits, row_tiles, parts));
    return B200GPTQ_OK;
}

template <typename T, int HD, int MT, bool PREFIX>
int run(const b200gptq_attn_args& a, float* part, const AttnPlan& s, cudaStream_t stream) {
    static std::once_flag once[64];
    static cudaError_t result[64];
    auto* kernel = attn_rows_kernel<T, HD, MT, PREFIX>;
    constexpr int smem = Lay<HD, MT>::total * 4;
    int dev = 0;
    B200GPTQ_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return B200GPTQ_ERR_TOO_LARGE;
    std::call_once(once[dev], [&] { result[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    B200GPTQ_CUDA_TRY(result[dev]);
    const long long rows = (long long)a.tokens * (a.heads / a.kv_heads) * (PREFIX ? a.batch : 1);
    const int tiles = (int)((rows + 16 * MT - 1) / (16 * MT));
    const long long units = (long long)tiles * a.kv_heads * (PREFIX ? 1 : a.batch);
    const int splits = PREFIX ? s.parts : s.own;
    return launch(kernel, a, smem, units * splits, PREFIX ? 1 : splits, attn_pdl_enabled(), part, splits, tiles, s.parts, stream);
}

template <typename T, int HD>
int run_all(const b200gptq_attn_args& a, float* part, const AttnPlan& s, cudaStream_t stream) {
    const long long per_sequence = (long long)a.tokens * (a.heads / a.kv_heads);
    if (a.prefix && !s.prefix_tiles) {
        const int st = per_sequence * a.batch <= 16 ? run<T, HD, 1, true>(a, part, s, stream) : run<T, HD, 2, true>(a, part, s, stream);
        if (st != B200GPTQ_OK) return st;
    }
    return per_sequence <= 16 ? run<T, HD, 1, false>(a, part, s, stream) : run<T, HD, 2, false>(a, part, s, stream);
}

}  // namespace

int attn_rows_dispatch(const b200gptq_attn_args& a, float* part, const AttnPlan& s, cudaStream_t stream) {
    if (a.dtype == B200GPTQ_F16) return a.hd == 128 ? run_all<__half, 128>(a, part, s, stream) : run_all<__half, 64>(a, part, s, stream);
    return a.hd == 128 ? run_all<__nv_bfloat16, 128>(a, part, s, stream) : run_all<__nv_bfloat16, 64>(a, part, s, stream);
}

}  // namespace b200gptq
