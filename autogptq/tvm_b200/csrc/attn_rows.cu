// b200gptq_attn for few query rows per key head: the single tokens of a decode step (and short runs of them), over a windowed cache or behind
// a shared prefix.
//
//   S = Q K^T,  w = softmax(scale S) over the visible keys,  O = w V
//
// The bytes of K and V bound it (4 flop per byte and row of Q), so a CTA holds up to 8, 16 or 32 rows of Q (all that share a key head: the heads
// of its group, the tokens of a short run, and with a prefix all sequences of the batch) and streams the keys once.  Every warp takes blocks of 16
// keys on its own and goes from global memory to mma.sync fragments without shared memory:
//   * Q K^T: an operand of m16n8k16 wants, from lane (g, c) = (lane / 4, lane % 4), the pairs 2c and 2c + 8 of key g.  Any order of the 16 dims
//     serves as long as Q has the same, so a lane loads 16 bytes = 8 adjacent dims of key g, which are the operand of two products;
//   * w V: an operand wants pairs of keys of one dim.  A lane loads 8 adjacent dims of keys 2c, 2c + 1, 2c + 8, 2c + 9 and pairs them with byte
//     permutations; index g of product (h, i) is dim 64 h + 8 g + i;
//   * up to 8 rows: keys are the 16, rows the 8 (half the accumulators: two CTAs per SM); the weights change hands by movmatrix.  More: rows are the 16, and the
//     accumulators of S are operand A of the second product as they lie.
// The next block's keys are requested when this block's have been multiplied, its values likewise, so that 6 to 8 KB per warp are on their way.  Rows are
// only rescaled when a score is more than 2^8 above the maximum in use (no weight is above 2^8; fp32 sums).
//
// The key range is split over the warps of a CTA and a cluster of up to 8 CTAs, which add up through distributed shared memory, each a slice of the dims.
// A prefix is part of every sequence's keys where reading it again from L2 takes less time than more launches; else there are three: the first
// takes the prefix, split over CTAs, the second each sequence's own rows, beside it, on what registers and shared memory it leaves, and both leave their
// sums (fp32) in scratch; the third adds them up.  All sums are in a fixed order.  (Two launches, the second of which adds up: its CTAs wait for the first
// one's sums where they are, so that few ran beside it: 32 sequences behind 8192 positions 34 us, now 24; 64 behind 16384 98, now 81.)
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "attn.cuh"
#include "attn.h"

namespace b200gptq {
namespace {

constexpr int kBlock = 16, kMaxSplit = kAttnMaxSplit;
constexpr float kGrow = 8.f;             // log2 of what a score may be above the maximum in use

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

__device__ __forceinline__ uint32_t transposed(uint32_t v) {      // of an 8 x 8 matrix of 16-bit values, a pair of a row per lane
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Shared memory, in floats: the warps' sums [warp][row][HD + 4], their maxima and denominators, the slices that the CTAs of the cluster push
// [split][row][HD / splits] with maxima and denominators, a flag per row; the queries (padded rows).
template <int HD, int R, int W> struct Lay {
    static constexpr int LD = HD + 4, QLD = HD + 8, acc = 0, ml = acc + W * R * LD, slice = ml + 2 * W * R, slice_ml = slice + R * HD,
                         flags = slice_ml + 2 * kMaxSplit * R, places = flags + (R < 16 ? 16 : R), q = places + 6 * R, total = q + R * QLD / 2;
};

struct RowDivisors { Divisor parts, row_tiles, kv_heads, group, tokens; };

// PREFIX: rows (b, t, g) of one key head against the prefix, sums to runs 0 .. parts - 1 of `part`.  Otherwise: rows (t, g) of one sequence and key head against
// its cache (and the prefix, where with_prefix); with parts, sums to run `parts`.  A tile of R rows is blockIdx.x / splits % row_tiles.
template <typename T, int HD, int R, int W, bool PREFIX>
__global__ void __launch_bounds__(W * 32, R == 8 ? 16 / W : 1)
attn_rows_kernel(const __grid_constant__ b200gptq_attn_args a, float* __restrict__ part, int split_bits, int row_tiles, int parts, int with_prefix, int G,
                 const __grid_constant__ RowDivisors by) {
    using L = Lay<HD, R, W>;
    constexpr int MT = R == 8 ? 1 : R / 16, SEG = HD / 32, HH = HD / 64, kThreads = W * 32;
    extern __shared__ __align__(16) float sm[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int window = a.window ? a.window : 1 << 30, splits = PREFIX ? parts : 1 << split_bits;
    const unsigned per_unit = PREFIX ? over(blockIdx.x, by.parts) : blockIdx.x >> split_bits, unit = over(per_unit, by.row_tiles);
    const int split = blockIdx.x - per_unit * splits, tile = per_unit - unit * row_tiles;
    const int b0 = PREFIX ? 0 : over(unit, by.kv_heads), kh = unit - b0 * a.kv_heads;
    auto token_of = [&](int idx) { return (int)over((unsigned)idx, by.group); };       // of row idx
    // What is read below was written before the launch in front of this one ended, or began (beside the prefix launch, which lets this one
    // start only after it has itself waited; the loads by-pass L1).  One CTA waits for the prefix launch at its end, so that this launch does not end before it.
    if (!PREFIX && splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    if (PREFIX || !parts) asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");

    const int row0 = tile * R, rows_all = (PREFIX ? a.batch : 1) * a.tokens * G;
    int p0 = 0, count = a.tokens;
    if constexpr (!PREFIX) { p0 = attn_pos(a, b0); count = attn_count(a, b0); }
    const int nrows = min(R, (PREFIX ? rows_all : count * G) - row0);
    if (nrows <= 0) {                         // padding: every CTA of the cluster leaves
        if (!PREFIX && parts && blockIdx.x == gridDim.x - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    // ---- keys: the prefix, the sinks, the window ----
    AttnRange range = {0, 0, 0};
    const int p_lo = PREFIX ? 0 : p0 + token_of(row0), p_hi = PREFIX ? 0 : p0 + token_of(row0 + nrows - 1);
    if constexpr (!PREFIX) range = attn_range(p_lo, p_hi, window, a.sinks, a.max_seq);
    const int n_p = PREFIX || with_prefix ? (a.prefix + kBlock - 1) / kBlock : 0, n_s = n_p + (range.s_end + kBlock - 1) / kBlock,
              nb = n_s + (range.w_end - range.w_start + kBlock - 1) / kBlock;
    int first, last;
    if constexpr (PREFIX) {
        const int each = over(nb, by.parts), more = nb - each * splits;
        first = split * each + min(split, more);
        last = first + each + (split < more ? 1 : 0);
    } else {
        first = (int)((long long)nb * split >> split_bits);
        last = (int)((long long)nb * (split + 1) >> split_bits);
    }
    const T *k_own = nullptr, *v_own = nullptr, *k_front = nullptr, *v_front = nullptr;
    if constexpr (!PREFIX) {
        k_own = static_cast<const T*>(a.k_cache) + b0 * a.k_stride[0] + kh * a.k_stride[1];
        v_own = static_cast<const T*>(a.v_cache) + b0 * a.v_stride[0] + kh * a.v_stride[1];
    }
    if (n_p) {
        k_front = static_cast<const T*>(a.k_prefix) + kh * a.k_prefix_stride[0];
        v_front = static_cast<const T*>(a.v_prefix) + kh * a.v_prefix_stride[0];
    }
    uint4 kr[2][SEG], vr[4][HH];
    auto block = [&](int i, int& j0, int& end) {
        j0 = i < n_p ? kBlock * i : i < n_s ? kBlock * (i - n_p) : range.w_start + kBlock * (i - n_s);
        end = i < n_p ? a.prefix : i < n_s ? range.s_end : range.w_end;
    };
    // (rows behind the end of the range: its last row again, with weight zero)
    auto load_k = [&](int i) {
        int j0, end;
        block(i, j0, end);
        const bool front = PREFIX || i < n_p;
        const T* base = (front ? k_front : k_own) + 8 * c;
        const long long stride = front ? a.k_prefix_stride[1] : a.k_stride[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const T* src = base + min(j0 + 8 * n + g, end - 1) * stride;
#pragma unroll
            for (int s = 0; s < SEG; ++s) kr[n][s] = __ldcg(reinterpret_cast<const uint4*>(src + 32 * s));
        }
    };
    auto load_v = [&](int i) {
        int j0, end;
        block(i, j0, end);
        const bool front = PREFIX || i < n_p;
        const T* base = (front ? v_front : v_own) + 8 * g;
        const long long stride = front ? a.v_prefix_stride[1] : a.v_stride[2];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const T* src = base + min(j0 + 2 * c + (n & 1) + 4 * (n & 2), end - 1) * stride;
#pragma unroll
            for (int h = 0; h < HH; ++h) vr[n][h] = __ldcg(reinterpret_cast<const uint4*>(src + 64 * h));
        }
    };
    int i = first + warp;
    if (i < last) { load_k(i); load_v(i); }
    // ---- the rows' places in q, out and the scratch (divisions once per row), queries ----
    long long* places = reinterpret_cast<long long*>(sm + L::places);
    if (threadIdx.x < R) {
        const int idx = row0 + min((int)threadIdx.x, nrows - 1), tok = token_of(idx), head = kh * G + idx - tok * G;
        const int bb = PREFIX ? (int)over((unsigned)tok, by.tokens) : b0, t = PREFIX ? tok - bb * a.tokens : tok;
        places[threadIdx.x] = bb * a.q_stride[0] + t * a.q_stride[1] + head * a.q_stride[2];
        places[R + threadIdx.x] = bb * a.out_stride[0] + t * a.out_stride[1] + head * a.out_stride[2];
        places[2 * R + threadIdx.x] = ((long long)bb * a.tokens + t) * a.heads + head;
        reinterpret_cast<int*>(sm + L::flags)[threadIdx.x] = 0;
    }
    __syncthreads();
    T* qs = reinterpret_cast<T*>(sm + L::q);
    for (int x = threadIdx.x; x < R * HD / 8; x += kThreads) {
        const int r = x / (HD / 8), d = x % (HD / 8) * 8;
        *reinterpret_cast<uint4*>(qs + r * L::QLD + d) = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + places[r] + d));
    }
    __syncthreads();

    const float scale = a.scale * kLog2e;
    float acc[MT][R == 8 ? 4 * HH : 8 * HH][4], m[MT][2], l[MT][2];
    // Rows of the lane: 2 c, 2 c + 1 (up to 8 rows), else g, g + 8 of each 16; pr: their positions
    int pr[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int n = 0; n < (R == 8 ? 4 * HH : 8 * HH); ++n) acc[t][n][0] = acc[t][n][1] = acc[t][n][2] = acc[t][n][3] = 0.f;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            m[t][r] = -INFINITY; l[t][r] = 0.f;
            pr[t][r] = PREFIX ? 0 : p0 + token_of(row0 + min(R == 8 ? 2 * c + r : 16 * t + 8 * r + g, nrows - 1));
        }
    }
    for (; i < last; i += W) {
        int j0, end;
        block(i, j0, end);
        const bool front = PREFIX || i < n_p;
        bool whole = j0 + kBlock <= end;      // every row of the tile sees the whole block
        if constexpr (!PREFIX) whole = whole && (front || (j0 + kBlock - 1 <= p_lo && (j0 > p_hi - window || j0 + kBlock <= a.sinks)));
        auto sees = [&](int j, int p) { return j < end && (front || attn_sees(p, j, window, a.sinks)); };
        if constexpr (R == 8) {
            float s[4] = {0.f, 0.f, 0.f, 0.f};        // keys g (0, 1) and g + 8 (2, 3), rows 2 c and 2 c + 1
#pragma unroll
            for (int e = 0; e < SEG; ++e) {
                const uint4 x = *reinterpret_cast<const uint4*>(qs + g * L::QLD + 32 * e + 8 * c);
                const uint32_t a0[4] = {kr[0][e].x, kr[1][e].x, kr[0][e].y, kr[1][e].y}, a1[4] = {kr[0][e].z, kr[1][e].z, kr[0][e].w, kr[1][e].w};
                mma16<T>(s, a0, x.x, x.y);
                mma16<T>(s, a1, x.z, x.w);
            }
            if (i + W < last) load_k(i + W);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[e] *= scale;
                if (!whole) s[e] = sees(j0 + g + 8 * (e >> 1), pr[0][e & 1]) ? s[e] : -INFINITY;
            }
            if (__any_sync(0xffffffffu, fmaxf(s[0], s[2]) - m[0][0] > kGrow || fmaxf(s[1], s[3]) - m[0][1] > kGrow)) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float up = fmaxf(fmaxf(s[r], s[2 + r]), m[0][r]);
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, o));
                    const float corr = up == -INFINITY ? 1.f : exp2_fast(m[0][r] - up);
                    m[0][r] = up;
                    l[0][r] *= corr;
#pragma unroll
                    for (int n = 0; n < 4 * HH; ++n) { acc[0][n][r] *= corr; acc[0][n][2 + r] *= corr; }
                }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float safe = m[0][r] == -INFINITY ? 0.f : m[0][r];
                s[r] = exp2_fast(s[r] - safe);
                s[2 + r] = exp2_fast(s[2 + r] - safe);
                l[0][r] += s[r] + s[2 + r];
            }
            const uint32_t w0 = transposed(Half<T>::pack(s[0], s[1])), w1 = transposed(Half<T>::pack(s[2], s[3]));
#pragma unroll
            for (int h = 0; h < HH; ++h)
#pragma unroll
                for (int n = 0; n < 4; ++n) {         // dims 64 h + 8 g + 2 n (rows 0 .. 7 of the product) and + 1 (8 .. 15)
                    const uint32_t x[4] = {__byte_perm(word(vr[0][h], n), word(vr[1][h], n), 0x5410u), __byte_perm(word(vr[0][h], n), word(vr[1][h], n), 0x7632u),
                                           __byte_perm(word(vr[2][h], n), word(vr[3][h], n), 0x5410u), __byte_perm(word(vr[2][h], n), word(vr[3][h], n), 0x7632u)};
                    mma16<T>(acc[0][4 * h + n], x, w0, w1);
                }
            if (i + W < last) load_v(i + W);
        } else {
            float s[MT][2][4];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
#pragma unroll
                for (int n = 0; n < 2; ++n) s[t][n][0] = s[t][n][1] = s[t][n][2] = s[t][n][3] = 0.f;
#pragma unroll
                for (int e = 0; e < SEG; ++e) {
                    const uint4 x = *reinterpret_cast<const uint4*>(qs + (16 * t + g) * L::QLD + 32 * e + 8 * c);
                    const uint4 y = *reinterpret_cast<const uint4*>(qs + (16 * t + 8 + g) * L::QLD + 32 * e + 8 * c);
                    const uint32_t a0[4] = {x.x, y.x, x.y, y.y}, a1[4] = {x.z, y.z, x.w, y.w};
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        mma16<T>(s[t][n], a0, kr[n][e].x, kr[n][e].y);
                        mma16<T>(s[t][n], a1, kr[n][e].z, kr[n][e].w);
                    }
                }
            }
            if (i + W < last) load_k(i + W);
            bool grow = false;
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float& x = s[t][e >> 1][2 * r + (e & 1)];
                        x *= scale;
                        if (!whole) x = sees(j0 + 8 * (e >> 1) + 2 * c + (e & 1), pr[t][r]) ? x : -INFINITY;
                    }
                    grow = grow || fmaxf(fmaxf(s[t][0][2 * r], s[t][0][2 * r + 1]), fmaxf(s[t][1][2 * r], s[t][1][2 * r + 1])) - m[t][r] > kGrow;
                }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float up = fmaxf(fmaxf(s[t][0][2 * r], s[t][0][2 * r + 1]), fmaxf(s[t][1][2 * r], s[t][1][2 * r + 1]));
                        up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, 1));
                        up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, 2));
                        up = fmaxf(up, m[t][r]);
                        const float corr = up == -INFINITY ? 1.f : exp2_fast(m[t][r] - up);
                        m[t][r] = up;
                        l[t][r] *= corr;
#pragma unroll
                        for (int n = 0; n < 8 * HH; ++n) { acc[t][n][2 * r] *= corr; acc[t][n][2 * r + 1] *= corr; }
                    }
            }
            uint32_t w[MT][4];
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float safe = m[t][r] == -INFINITY ? 0.f : m[t][r];
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = exp2_fast(s[t][e >> 1][2 * r + (e & 1)] - safe);
                    l[t][r] += (x[0] + x[1]) + (x[2] + x[3]);
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
            if (i + W < last) load_v(i + W);
        }
    }
    // ---- the warps' sums: rows, 8 adjacent dims each ----
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float sum = l[t][r];
#pragma unroll
            for (int o = R == 8 ? 4 : 1; o < (R == 8 ? 32 : 4); o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const int row = R == 8 ? 2 * c + r : 16 * t + 8 * r + g;
            if (row < nrows) {
                if (R == 8 ? g == 0 : c == 0) { sm[L::ml + 2 * (warp * R + row)] = m[t][r]; sm[L::ml + 2 * (warp * R + row) + 1] = sum; }
                float* dst = sm + L::acc + (warp * R + row) * L::LD;
#pragma unroll
                for (int h = 0; h < HH; ++h) {
                    if constexpr (R == 8) {
                        float4* to = reinterpret_cast<float4*>(dst + 64 * h + 8 * g);
#pragma unroll
                        for (int x = 0; x < 2; ++x)
                            to[x] = make_float4(acc[t][4 * h + 2 * x][r], acc[t][4 * h + 2 * x][2 + r], acc[t][4 * h + 2 * x + 1][r], acc[t][4 * h + 2 * x + 1][2 + r]);
                    } else {
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
            }
        }
    __syncthreads();
    if (!PREFIX && splits > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");      // (all CTAs of the cluster run)
    // ---- the CTA's sums: to the scratch, or slice by slice to the CTAs of the cluster ----
    const int slice = PREFIX ? HD : HD >> split_bits;
    constexpr int HD_BITS = HD == 128 ? 7 : 6;
    const long long rows_total = (long long)a.batch * a.tokens * a.heads;
    for (int x = threadIdx.x; x < nrows * HD; x += kThreads) {
        const int row = x / HD, d = x % HD;
        float cm = -INFINITY, cl = 0.f, ca = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) cm = fmaxf(cm, sm[L::ml + 2 * (w * R + row)]);
        const float safe = cm == -INFINITY ? 0.f : cm;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float e = exp2_fast(sm[L::ml + 2 * (w * R + row)] - safe);
            cl += sm[L::ml + 2 * (w * R + row) + 1] * e;
            ca += sm[L::acc + (w * R + row) * L::LD + d] * e;
        }
        if constexpr (PREFIX) {
            const long long at = split * rows_total + places[2 * R + row];
            part[at * HD + d] = ca;
            if (d == 0) *reinterpret_cast<float2*>(part + (parts + 1) * rows_total * HD + 2 * at) = make_float2(cm, cl);
        } else {
            const int to = d >> (HD_BITS - split_bits);
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
    // ---- this CTA's slice of the dims ----
    int* flags = reinterpret_cast<int*>(sm + L::flags);
    for (int x = threadIdx.x; x < nrows * (slice / 4); x += kThreads) {
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
        if (parts) {
            const long long at = parts * rows_total + places[2 * R + row];
            *reinterpret_cast<float4*>(part + at * HD + split * slice + d) = o;
            if (split * slice + d == 0) *reinterpret_cast<float2*>(part + (parts + 1) * rows_total * HD + 2 * at) = make_float2(tm, tl);
            continue;
        }
        const bool none = tl == 0.f;
        float f[4] = {none ? 0.f : o.x / tl, none ? 0.f : o.y / tl, none ? 0.f : o.z / tl, none ? 0.f : o.w / tl};
        if (settle<T>(f) && isfinite(tl)) flags[row] = 1;
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + places[R + row] + split * slice + d) =
            make_uint2(Half<T>::pack(f[0], f[1]), Half<T>::pack(f[2], f[3]));
    }
    if (parts) {
        if (blockIdx.x == gridDim.x - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    // A weight of zero times a NaN or an infinity, of a key that the row does not see or that stands in for one behind the end: the row is done again.  (Not
    // where the denominator is not finite: then a score that the row sees is a NaN.)
    __syncthreads();
    for (int row = warp; row < nrows; row += W)
        if (flags[row]) {
            const int idx = row0 + row, t = token_of(idx);
            attn_row_again<T, HD>(a, b0, t, kh * G + idx - t * G, p0 + t, split * slice, (split + 1) * slice);
        }
}

// The sums of all runs of a row, a warp per row: lane l knows runs l, l + 32 .. and, later, adds 4 dims.
template <typename T, int HD>
__global__ void __launch_bounds__(256)
attn_sum_kernel(const __grid_constant__ b200gptq_attn_args a, const float* __restrict__ part, int runs, const Divisor by_heads, const Divisor by_tokens) {
    constexpr int LANES = HD / 4, MOST = (kAttnMaxParts + 1 + 31) / 32;
    const int lane = threadIdx.x & 31;
    const long long rows_total = (long long)a.batch * a.tokens * a.heads, at = blockIdx.x * 8LL + (threadIdx.x >> 5);       // (below 2^31)
    const unsigned token = over((unsigned)at, by_heads);
    const int head = (int)at - (int)token * a.heads, b = over(token, by_tokens), t = token - b * a.tokens;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    if (at >= rows_total) return;
    if (t >= attn_count(a, b)) return;
    float m[MOST], l[MOST], tm = -INFINITY, tl = 0.f;
#pragma unroll
    for (int k = 0; k < MOST; ++k) {
        const int r = lane + 32 * k;
        const float2 v = r < runs ? __ldcg(reinterpret_cast<const float2*>(part + runs * rows_total * HD + 2 * (r * rows_total + at))) : make_float2(-INFINITY, 0.f);
        m[k] = v.x;
        l[k] = v.y;
        tm = fmaxf(tm, v.x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, o));
    const float safe = tm == -INFINITY ? 0.f : tm;
#pragma unroll
    for (int k = 0; k < MOST; ++k) {
        m[k] = exp2_fast(m[k] - safe);
        tl += l[k] * m[k];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) tl += __shfl_xor_sync(0xffffffffu, tl, o);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    const float* src = part + at * HD + 4 * (lane % LANES);
    // (64 dims: the halves of the warp take every other run)
    constexpr int STEP = 32 / LANES;
#pragma unroll
    for (int k = 0; k < MOST; ++k)
#pragma unroll 8
        for (int r = 32 * k; r < min(runs, 32 * k + 32); r += STEP) {
            const int mine = r + lane / LANES;
            const float w = __shfl_sync(0xffffffffu, m[k], mine & 31);
            if (mine < runs) {
                const float4 f = __ldcg(reinterpret_cast<const float4*>(src + mine * rows_total * HD));
                sum.x += f.x * w; sum.y += f.y * w; sum.z += f.z * w; sum.w += f.w * w;
            }
        }
    if constexpr (STEP == 2) {
        sum.x += __shfl_xor_sync(0xffffffffu, sum.x, 16); sum.y += __shfl_xor_sync(0xffffffffu, sum.y, 16);
        sum.z += __shfl_xor_sync(0xffffffffu, sum.z, 16); sum.w += __shfl_xor_sync(0xffffffffu, sum.w, 16);
    }
    const bool none = tl == 0.f;
    float mean[4] = {none ? 0.f : sum.x / tl, none ? 0.f : sum.y / tl, none ? 0.f : sum.z / tl, none ? 0.f : sum.w / tl};
    const bool bad = settle<T>(mean);
    if (lane < LANES)
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + b * a.out_stride[0] + t * a.out_stride[1] + head * a.out_stride[2] + 4 * lane) =
            make_uint2(Half<T>::pack(mean[0], mean[1]), Half<T>::pack(mean[2], mean[3]));
    __syncwarp();
    // (as in attn_rows_kernel)
    if (__any_sync(0xffffffffu, isfinite(tl) && bad))
        attn_row_again<T, HD>(a, b, t, head, attn_pos(a, b) + t, 0, HD);
}

template <typename T, int HD, int R, int W, bool PREFIX>
int run(const b200gptq_attn_args& a, float* part, const AttnPlan& s, cudaStream_t stream) {
    static std::once_flag once[64];
    static cudaError_t result[64];
    auto* kernel = attn_rows_kernel<T, HD, R, W, PREFIX>;
    constexpr int smem = Lay<HD, R, W>::total * 4;
    int dev = 0;
    B200GPTQ_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return B200GPTQ_ERR_TOO_LARGE;
    std::call_once(once[dev], [&] { result[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    B200GPTQ_CUDA_TRY(result[dev]);
    const long long rows = (long long)a.tokens * (a.heads / a.kv_heads) * (PREFIX ? a.batch : 1);
    const int tiles = (int)((rows + R - 1) / R), splits = PREFIX ? s.parts : s.own;
    const long long ctas = (long long)tiles * a.kv_heads * (PREFIX ? 1 : a.batch) * splits;
    if (ctas > 0x7fffffff) return B200GPTQ_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(W * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (!PREFIX && splits > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = splits;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (attn_pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    int bits = 0;
    while ((1 << bits) < splits) ++bits;      // (a cluster has 1, 2, 4 or 8 CTAs)
    B200GPTQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a, part, bits, tiles, s.parts, a.prefix && !s.parts ? 1 : 0, a.heads / a.kv_heads,
                                         RowDivisors{Divisor(std::max(s.parts, 1)), Divisor(tiles), Divisor(a.kv_heads), Divisor(a.heads / a.kv_heads), Divisor(a.tokens)}));
    return B200GPTQ_OK;
}

template <typename T, int HD>
int run_all(const b200gptq_attn_args& a, float* part, const AttnPlan& s, cudaStream_t stream) {
    const long long rows = (long long)a.tokens * (a.heads / a.kv_heads), all = rows * a.batch;
    if (s.parts && !s.prefix_tiles) {
        const int st = all <= 8    ? run<T, HD, 8, 8, true>(a, part, s, stream)
                       : all <= 16 ? run<T, HD, 16, 8, true>(a, part, s, stream)
                                   : run<T, HD, 32, 8, true>(a, part, s, stream);
        if (st != B200GPTQ_OK) return st;
    }
    if (rows <= 8) {
        if (s.warps == 1) return run<T, HD, 8, 1, false>(a, part, s, stream);
        if (s.warps == 2) return run<T, HD, 8, 2, false>(a, part, s, stream);
        return s.warps == 4 ? run<T, HD, 8, 4, false>(a, part, s, stream) : run<T, HD, 8, 8, false>(a, part, s, stream);
    }
    return rows <= 16 ? run<T, HD, 16, 8, false>(a, part, s, stream) : run<T, HD, 32, 8, false>(a, part, s, stream);
}

template <typename T, int HD>
int run_sum(const b200gptq_attn_args& a, const float* part, int runs, cudaStream_t stream) {
    const long long ctas = ((long long)a.batch * a.tokens * a.heads + 7) / 8;
    if (ctas > 0x7fffffff) return B200GPTQ_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = attn_pdl_enabled() ? 1 : 0;
    B200GPTQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, attn_sum_kernel<T, HD>, a, part, runs, Divisor(a.heads), Divisor(a.tokens)));
    return B200GPTQ_OK;
}

template <typename T, int HD>
int run_both(const b200gptq_attn_args& a, float* part, const AttnPlan& s, cudaStream_t stream) {
    const int st = run_all<T, HD>(a, part, s, stream);
    return st != B200GPTQ_OK || !s.parts ? st : run_sum<T, HD>(a, part, s.parts + 1, stream);
}

}  // namespace

int attn_rows_dispatch(const b200gptq_attn_args& a, float* part, const AttnPlan& s, cudaStream_t stream) {
    if (a.dtype == B200GPTQ_F16) return a.hd == 128 ? run_both<__half, 128>(a, part, s, stream) : run_both<__half, 64>(a, part, s, stream);
    return a.hd == 128 ? run_both<__nv_bfloat16, 128>(a, part, s, stream) : run_both<__nv_bfloat16, 64>(a, part, s, stream);
}

}  // namespace b200gptq
