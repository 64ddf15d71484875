// b200gptq_attn for many query rows per key head: prompts and chunks of them, and the prefix part of a large batch.
//
//   S = Q K^T,  w = softmax(scale S) over the visible keys,  O = w V
//
// A CTA takes two tiles of 128 rows of Q that share a key head (rows are (token, head of the group), so that shared key heads fill a tile) and streams units
// of 64 keys that either of them sees: 2 hd multiplications and one exponential per row and key, and of the latter an SM makes 16 per clock where the
// tensor cores make 4096 of the former, so for 128 dims both take as long (512 clk per unit and tile of Q) and have to run at once:
//
//   warps 0..3, 4..7  softmax of one tile of Q each, a thread per row: S from tensor memory into registers, the weights (16 bits) back over it.  O is
//                     only rescaled when a row's maximum grows by more than 2^8 over the one in use (no weight is above 2^8; fp32 sums)
//   warp 8            TMA: K and V of the units into a ring, in the order in which they are multiplied: K0 and K1, V0 and K2, V1 and K3 ..
//   warps 9, 10       tcgen05.mma for one tile of Q each: S of the unit after next as soon as the weights of this one have been multiplied, so that the
//                     softmax always finds the next S there and waits for no product
//
// Measured per unit and both tiles, 128 dims: 1 570 clk; the products alone 1 280 (Q and K are 48 KB of shared memory, 384 clk, for 256 of arithmetic), the
// exponentials, which both tiles do at the same time, 1 030 of a softmax warp's turn.  One prompt of 8192, 32 / 8 heads, window 4096: 357 us, 1 150 TFLOP/s;
// 411 when it runs for seconds and the power limit holds the clock at 1.6 GHz.
// Units of 128 keys with one S per tile of Q, so that softmax and products of a tile took turns, took 3900 to 4600 clk per 128 keys, with two threads per
// row (which exchange its maximum) 4100: 1550 of them the products, 2500 the softmax.
//
// Tensor memory: two S per tile of Q (64 columns each; the weights lie over the first 32), O of both (2 x hd).  The weights are the A operand from
// tensor memory, V is the B operand as it lies (MN-major, keys along K).
//
// Rows of V that no row of the tiles sees are zeroed in shared memory before they are multiplied (a weight of zero times a NaN is one).  Where rows of the
// tiles see different keys and one of these holds a NaN or an infinity, the rows that come out not finite are done again (attn_row_again).
//
// PACKED: the rows are (sequence, token, head of the group) of the whole batch against the shared prefix, split over CTAs, sums to scratch.
// ALT (few rows): both tiles of Q are the same rows, one takes the even units of keys and the other the odd ones; they add up at the end.
#include <cuda.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "attn.cuh"
#include "attn.h"

namespace b200gptq {
namespace {

constexpr int kRows = 128, kKeys = kAttnTilesKeys, kSoftmaxWarps = 8, kLoadWarp = 8, kMmaWarp = 9, kThreads = 384;
constexpr int kTmemCols = 512, kColO = 256;          // S of tile q, buffer b at 128 q + 64 b, O at 256 + 128 q
constexpr float kGrow = 8.f;                         // log2 of what a maximum may grow before O is rescaled

template <int HD> struct Smem {
    static constexpr int q_tile = kRows * HD * 2, unit = kKeys * HD * 2, stages = HD == 128 ? 5 : 8, total = 2 * q_tile + stages * 2 * unit + 1024;
    static_assert(stages * 2 * unit >= 2 * kRows * HD * 4, "");
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity), "r"(4000u) : "memory");
    return ok != 0;
}
// Bounded wait: gives up after ~2e9 clocks or as soon as another warp of the CTA has.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    if (mbar_try(bar, parity)) return true;
    const long long t0 = clock64();
    while (true) {
        for (int i = 0; i < 8; ++i)
            if (mbar_try(bar, parity)) return true;
        if (*abort_flag) return false;
        if (clock64() - t0 > 2000000000LL) { *abort_flag = 1; return false; }
    }
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
}
// Issued by the one thread for which `lead` is set.  The others come along, so that addresses and descriptors are the warp's (uniform registers): inside
// a branch of one thread an mma took 69 clk to issue, whatever its size.
__device__ __forceinline__ void mma_commit(uint32_t bar, uint32_t lead) {       // arrives when all products issued so far have retired
    asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
                 "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(lead) : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(lead) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(lead) : "memory");
}
#define B200GPTQ_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define B200GPTQ_RW8(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7])
#define B200GPTQ_I8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : B200GPTQ_R8(r, 0), B200GPTQ_R8(r, 8), B200GPTQ_R8(r, 16), B200GPTQ_R8(r, 24) : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// (registers that a load has filled pass through here after the wait, so that nothing reads them before it)
__device__ __forceinline__ void after_wait(uint32_t (&r)[32]) {
    asm volatile("" : B200GPTQ_RW8(r, 0), B200GPTQ_RW8(r, 8), B200GPTQ_RW8(r, 16), B200GPTQ_RW8(r, 24) :: "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(taddr), B200GPTQ_I8(r, 0), B200GPTQ_I8(r, 8), B200GPTQ_I8(r, 16), B200GPTQ_I8(r, 24) : "memory");
}
// Pairs of fp32 in one instruction.
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b, float m, float c) {
    asm("{\n\t.reg .b64 u, v, w;\n\tmov.b64 u, {%2, %3};\n\tmov.b64 v, {%4, %4};\n\tmov.b64 w, {%5, %5};\n\t"
        "fma.rn.f32x2 u, u, v, w;\n\tmov.b64 {%0, %1}, u;\n\t}" : "=f"(x), "=f"(y) : "f"(a), "f"(b), "f"(m), "f"(c));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float m;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {
    asm("{\n\t.reg .b64 u, v;\n\tmov.b64 u, {%0, %1};\n\tmov.b64 v, {%2, %3};\n\tadd.rn.f32x2 u, u, v;\n\tmov.b64 {%0, %1}, u;\n\t}"
        : "+f"(x), "+f"(y) : "f"(a), "f"(b));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Operand tiles are boxes of 64 dims (128 bytes, swizzled) by 128 rows of Q or 64 keys, one after the other.  Q and K: K-major, 8-row groups 1024 bytes apart.  V: MN-major,
// groups of 8 keys 1024 bytes apart, the next 64 dims a box further on.
__device__ __forceinline__ uint64_t smem_desc(uint32_t saddr, uint32_t leading) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3FFF);   // start address, 16-byte units
    d |= (uint64_t)(leading >> 4) << 16;       // leading byte offset (not used K-major)
    d |= (uint64_t)(1024 >> 4) << 32;          // stride byte offset
    d |= (uint64_t)1 << 46;                    // descriptor version of sm_100
    d |= (uint64_t)2 << 61;                    // SWIZZLE_128B
    return d;
}

struct TileArgs {
    b200gptq_attn_args a;
    float* part;
    float sl2;                // |scale| log2 e, and Q is negated where the scale is negative
    int negate, tiles, splits, prefix_units, group, alt;
    int units_each, units_more;             // of a run of the prefix; the first units_more runs have one more
    Divisor by_splits, by_kv_heads, by_batch, by_group, by_tokens;
};

template <typename T, int HD, bool PACKED>
__global__ void __launch_bounds__(kThreads, 1)
attn_tiles_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_kp,
                  const __grid_constant__ CUtensorMap map_vp, const __grid_constant__ TileArgs p) {
    using SM = Smem<HD>;
    constexpr int ST = SM::stages, QBOX = kRows * 128, BOX = kKeys * 128, HALVES = HD / 64;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - raw);
    __shared__ __align__(8) uint64_t bars[2 * ST + 15];
    __shared__ uint32_t tmem_base_holder;
    __shared__ volatile int abort_flag;

    const b200gptq_attn_args& a = p.a;
    const bool alt = p.alt;                   // both tiles are the same rows
    const uint32_t ring = alt ? SM::q_tile : 2 * SM::q_tile;       // where it begins, behind one or two tiles of Q
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t bar_base = smem_u32(bars);
    auto full = [&](int s) { return bar_base + 8u * s; };
    auto empty = [&](int s) { return bar_base + 8u * (ST + s); };
    auto s_full = [&](int q, int b) { return bar_base + 8u * (2 * ST + 2 * q + b); };
    auto p_full = [&](int q, int b) { return bar_base + 8u * (2 * ST + 4 + 2 * q + b); };
    auto q_full = [&](int q) { return bar_base + 8u * (2 * ST + 8 + q); };
    auto o_done = [&](int q) { return bar_base + 8u * (2 * ST + 10 + q); };     // O has the unit's products
    auto retired = [&](int q) { return bar_base + 8u * (2 * ST + 12 + q); };    // all products of the tile
    const uint32_t all_met = bar_base + 8u * (2 * ST + 14);

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < ST; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 2); }
        for (int q = 0; q < 2; ++q) {
            for (int b = 0; b < 2; ++b) { mbar_init(s_full(q, b), 1); mbar_init(p_full(q, b), 4); }
            mbar_init(q_full(q), 4);
            mbar_init(o_done(q), 1);
            mbar_init(retired(q), 1);
        }
        mbar_init(all_met, kSoftmaxWarps);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_holder)), "r"((uint32_t)kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base_holder, 0);
    // ---- which rows, which keys.  The last rows of a prompt see most, and come first (the tiles of one head one after the other read two chunks of 512 of 72
    //      heads once instead of 1.4 times, which took as long; one prompt of 4096, 32 heads, without a window 158 us, now 137). ----
    const int G = p.group, window = a.window ? a.window : 1 << 30;
    const unsigned part_unit = PACKED ? over(blockIdx.x, p.by_splits) : blockIdx.x, over_heads = over(part_unit, p.by_kv_heads);
    const unsigned row_tile = PACKED ? over_heads : over(over_heads, p.by_batch);
    const int split = PACKED ? blockIdx.x - part_unit * p.splits : 0, kh = part_unit - over_heads * a.kv_heads, b0 = PACKED ? 0 : over_heads - row_tile * a.batch;
    const int row0 = (p.tiles - 1 - (int)row_tile) * (alt ? kRows : 2 * kRows);
    // (nothing that another launch has written is read before this)
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");

    const int pos0 = PACKED ? 0 : attn_pos(a, b0);
    const int rows_all = PACKED ? a.batch * a.tokens * G : attn_count(a, b0) * G;
    int nrows[2], p_lo[2], p_hi[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int r = row0 + (alt ? 0 : q * kRows);
        nrows[q] = max(0, min(kRows, rows_all - r));
        p_lo[q] = PACKED ? 0 : pos0 + (int)over((unsigned)r, p.by_group);
        p_hi[q] = PACKED ? 0 : pos0 + (int)over((unsigned)(r + max(nrows[q], 1) - 1), p.by_group);
    }
    auto of = [](const int (&v)[2], int q) { return q ? v[1] : v[0]; };       // (registers, not an array that is indexed)
    // Units of three regions, one after the other: the prefix, the sinks, the window (which begin where the keys begin; where sinks and window meet, they
    // are one run of keys, cut at a multiple of 64).
    int n_units = 0, n_p = 0, n_s = 0, first = 0, s_end = 0, w_base = 0, w_end = 0;
    if (nrows[0] > 0) {
        if constexpr (PACKED) {
            first = split * p.units_each + min(split, p.units_more);
            n_units = n_p = p.units_each + (split < p.units_more ? 1 : 0);
        } else {
            const AttnRange range = attn_range(p_lo[0], nrows[1] > 0 ? p_hi[1] : p_hi[0], window, a.sinks, a.max_seq);
            const bool one = range.w_start == 0;
            w_end = range.w_end;
            s_end = one ? w_end : range.s_end;
            n_p = p.prefix_units;
            n_s = (min(a.sinks, s_end) + kKeys - 1) / kKeys;
            w_base = one ? n_s * kKeys : range.w_start;
            n_units = n_p + n_s + max(0, w_end - w_base + kKeys - 1) / kKeys;
        }
    }
    struct Region { int begin, end, j_first, j_end; };           // units, key of unit `begin`, end of the keys
    // What rows of tile q see of region g
    auto region = [&](int q, int g) {
        Region v = {0, 0, 0, 0};
        if (of(nrows, q) <= 0) return v;
        if (g == 0) return Region{0, n_p, first * kKeys, a.prefix};
        if (PACKED) return v;
        const int hi = of(p_hi, q);
        if (g == 1) return Region{n_p, n_p + (hi < 0 ? 0 : min(n_s, hi / kKeys + 1)), 0, s_end};
        const int n_w = n_units - n_p - n_s, from = max(0, (of(p_lo, q) - window + 1 - w_base) >> 6), to = max(from, min(n_w, ((hi - w_base) >> 6) + 1));
        return Region{n_p + n_s + from, n_p + n_s + to, w_base + from * kKeys, w_end};
    };
    static_assert(kKeys == 64, "");
    bool ok = true;
    if (warp == kLoadWarp) {
        // ===== keys and values =====
        if (elect_one()) {
            auto load = [&](int i, uint32_t dst, uint32_t bar, bool value) {
                const bool prefix = i < n_p;
                const int j0 = prefix ? (first + i) * kKeys : i < n_p + n_s ? (i - n_p) * kKeys : w_base + (i - n_p - n_s) * kKeys;
#pragma unroll
                for (int h = 0; h < HALVES; ++h) {
                    if (prefix) tma_3d(dst + h * BOX, value ? &map_vp : &map_kp, 64 * h, j0, kh, bar);
                    else tma_4d(dst + h * BOX, value ? &map_v : &map_k, 64 * h, j0, kh, b0, bar);
                }
            };
            int n = 0;                        // slots: K0 and K1, then V i and K i + 2
            for (int s = 0, round = 0; n_units > 0 && n <= n_units; ++n) {
                if (round > 0) ok = mbar_wait(empty(s), (round - 1) & 1, &abort_flag);
                if (!ok) break;
                const uint32_t dst = base + ring + s * 2 * SM::unit, bar = full(s);
                mbar_expect(bar, n < 1 ? min(2, n_units) * SM::unit : n + 1 < n_units ? 2 * SM::unit : SM::unit);
                if (n == 0) load(0, dst, bar, false);
                else load(n - 1, dst, bar, true);
                if (n + 1 < n_units) load(n + 1, dst + SM::unit, bar, false);
                if (++s == ST) { s = 0; ++round; }
            }
            if (!ok) {                        // what is on its way lands before the CTA ends
                int never = 0;
                for (int i = max(0, n - ST); i < n; ++i) mbar_wait(full(i % ST), (i / ST) & 1, &never);
            }
        }
        __syncwarp();
    } else if (warp == kMmaWarp || warp == kMmaWarp + 1) {
        // ===== products of tile q, load by load =====
        const uint32_t lead = elect_one();
        constexpr uint32_t type = std::is_same<T, __half>::value ? 0u : 1u;
        constexpr uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)(kRows >> 4) << 24);
        constexpr uint32_t idesc_qk = idesc | ((uint32_t)(kKeys >> 3) << 17), idesc_pv = idesc | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
        const int q = warp - kMmaWarp;
        const uint64_t qd = smem_desc(base + (alt ? 0 : q) * SM::q_tile, 0);
        const uint32_t ts = tmem + 128u * q, to = tmem + kColO + 128u * q;
        const Region r0 = region(q, 0), r1 = region(q, 1), r2 = region(q, 2);
        auto needs = [&](int i) {
            return (!alt || (i & 1) == q) && ((i >= r0.begin && i < r0.end) || (i >= r1.begin && i < r1.end) || (i >= r2.begin && i < r2.end));
        };
        int started = 0, mixed = 0;           // S begun, weights multiplied
        auto qk = [&](uint32_t at) {
            const uint64_t kd = smem_desc(at, 0);
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
                mma_ss(ts + 64u * (started & 1), qd + ((k / 4 * QBOX + k % 4 * 32) >> 4), kd + ((k / 4 * BOX + k % 4 * 32) >> 4), idesc_qk, k > 0 ? 1u : 0u, lead);
            mma_commit(s_full(q, started & 1), lead);
        };
        // One barrier for both loads of a turn: what a turn costs here besides the products (each wait 150 to 250 clk, also one that is over already) is
        // time in which the tensor cores idle.  (A wait that runs out is not looked at: those after it give up at once, and the results are not defined then.)
        if (n_units > 0) {
            if (of(nrows, q) > 0) mbar_wait(q_full(alt ? 0 : q), 0, &abort_flag);
            mbar_wait(full(0), 0, &abort_flag);
            tc_after();
            for (int i = 0; i < min(2, n_units); ++i)
                if (needs(i)) {
                    qk(base + ring + i * SM::unit);
                    ++started;
                }
            if (started) mma_commit(empty(0), lead);
            else if (lead) mbar_arrive(empty(0));
        }
        for (int i = 0, s = 1, round = 0; i < n_units; ++i) {
            const bool mine = needs(i), mine2 = i + 2 < n_units && needs(i + 2);
            const uint32_t at = base + ring + s * 2 * SM::unit;
            const int seen = i < n_p ? r0.j_end - r0.j_first - i * kKeys : i < n_p + n_s ? r1.j_end - (i - n_p) * kKeys : r2.j_end - r2.j_first - (i - r2.begin) * kKeys;
            if (mine && seen < kKeys) {       // rows that nobody sees (both warps write the same zeros)
                mbar_wait(full(s), round & 1, &abort_flag);
                __syncwarp();
                for (int x = lane; x < (kKeys - seen) * HALVES * 8; x += 32) {
                    const int r = seen + x / (HALVES * 8), c = x % (HALVES * 8);
                    *reinterpret_cast<uint4*>(base_ptr + (at - base) + (c / 8) * BOX + r * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            mbar_wait(full(s), round & 1, &abort_flag);
            __syncwarp();
            // (an S that is free already, as where the tile takes every other unit, is filled at once, the softmax need not wait for it)
            bool next = mine2;
            if (next && started - mixed < 2) {
                tc_after();
                qk(at + SM::unit);
                ++started;
                next = false;
            }
            if (mine) {
                mbar_wait(p_full(q, mixed & 1), (mixed >> 1) & 1, &abort_flag);
                __syncwarp();
                tc_after();
                const uint64_t vd = smem_desc(at, BOX);
#pragma unroll
                for (int k = 0; k < kKeys / 16; ++k)
                    mma_ts(to, ts + 64u * (mixed & 1) + 8u * k, vd + k * (2048 >> 4), idesc_pv, (mixed > 0 || k > 0) ? 1u : 0u, lead);
                mma_commit(o_done(q), lead);
                ++mixed;
            }
            if (next) {
                tc_after();
                qk(at + SM::unit);
                ++started;
            }
            if (mine || mine2) mma_commit(empty(s), lead);
            else if (lead) mbar_arrive(empty(s));
            __syncwarp();
            if (++s == ST) { s = 0; ++round; }
        }
        mma_commit(retired(q), lead);
        __syncwarp();
        int never = 0;                        // (also after a wait that ran out: nothing is in flight when tensor memory is freed)
        mbar_wait(retired(q), 0, &never);
    } else if (warp < kSoftmaxWarps) {
        // ===== softmax of tile q, one row per thread =====
        const int q = warp >> 2, quarter = warp & 3, r = 32 * quarter + lane, rows = of(nrows, q), row_first = row0 + (alt ? 0 : q * kRows);
        const uint32_t lane_off = (uint32_t)(32 * quarter) << 16, ts = tmem + 128u * q + lane_off, to = tmem + kColO + 128u * q + lane_off;
        const bool mine = 32 * quarter < rows;          // the warp has rows at all
        // The thread's row.  (Once per row; where other threads need its place they ask for it.)
        const int idx = row_first + min(r, max(rows, 1) - 1), token = (int)over((unsigned)idx, p.by_group), head = kh * G + idx - token * G;
        const int b = PACKED ? (int)over((unsigned)token, p.by_tokens) : b0, t = PACKED ? token - b * a.tokens : token, pr = pos0 + token;
        const long long q_at = b * a.q_stride[0] + t * a.q_stride[1] + head * a.q_stride[2];
        // Q, in the swizzled layout of the tiles: 16 bytes per thread and load, all of them on their way at once
        if (!(alt && q == 1)) {
            uint8_t* dst = base_ptr + q * SM::q_tile;
            const int c = lane % (HD / 8);
            uint4 val[HD / 8];
#pragma unroll
            for (int x = 0; x < HD / 8; ++x) {
                const int rw = (x * 32 + lane) / (HD / 8);
                const long long from = __shfl_sync(0xffffffffu, q_at, rw);
                val[x] = make_uint4(0, 0, 0, 0);
                if (32 * quarter + rw < rows) val[x] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + from + 8 * c));
            }
#pragma unroll
            for (int x = 0; x < HD / 8; ++x) {
                const int rr = 32 * quarter + (x * 32 + lane) / (HD / 8);
                if (p.negate) { val[x].x ^= 0x80008000u; val[x].y ^= 0x80008000u; val[x].z ^= 0x80008000u; val[x].w ^= 0x80008000u; }
                *reinterpret_cast<uint4*>(dst + (c / 8) * QBOX + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = val[x];
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full(q));
        }
        float m = -INFINITY, l = 0.f;           // the maximum in use (of scores, not scaled), the denominator
        float off = 0.f;                        // -m, scaled (m = -infinity: 0, every weight is then 0)
        int turn = 0;
#pragma unroll 1
        for (int g = 0; g < 3; ++g) {
            const Region v = region(q, g);
            // A unit whose keys all rows of the tile see: from key `least` to key `most`
            const int most = min(g == 1 ? min(v.j_end, a.sinks) : v.j_end, g == 0 ? v.j_end : of(p_lo, q) + 1) - kKeys, least = g == 2 ? of(p_hi, q) - window + 1 : 0;
            const int skip = alt ? (v.begin ^ q) & 1 : 0, step = alt ? 2 : 1;
            int j0 = v.j_first + skip * kKeys;
#pragma unroll 1
            for (int i = v.begin + skip; i < v.end; i += step, j0 += step * kKeys) {
                const uint32_t tb = ts + 64u * (turn & 1);
                // (A wait that runs out is not looked at before the end: those after it give up at once, and the results are not defined then.)
                mbar_wait(s_full(q, turn & 1), (turn >> 1) & 1, &abort_flag);
                __syncwarp();
                tc_after();
                if (mine) {
                    uint32_t s[2][32];
                    tmem_ld32(tb, s[0]);
                    tmem_ld32(tb + 32u, s[1]);
                    tmem_wait_ld();
                    after_wait(s[0]);
                    after_wait(s[1]);
                    if (j0 > most || j0 < least) {
                        // columns [0, front) and [lo, hi) are seen
                        int front = v.j_end - j0, lo = 0, hi = 0;
                        if (g != 0) {
                            front = min(min(a.sinks, pr + 1), v.j_end) - j0;
                            lo = pr - window + 1 - j0;
                            hi = min(pr + 1, v.j_end) - j0;
                        }
#pragma unroll
                        for (int x = 0; x < kKeys; ++x)
                            if (!(x < front || (x >= lo && x < hi))) s[x / 32][x % 32] = 0xff800000u;       // -infinity
                    }
                    float top[4];
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        top[g] = __uint_as_float(s[g / 2][g % 2 * 16]);
#pragma unroll
                        for (int e = 1; e < 15; e += 2)
                            top[g] = max3(top[g], __uint_as_float(s[g / 2][g % 2 * 16 + e]), __uint_as_float(s[g / 2][g % 2 * 16 + e + 1]));
                        top[g] = fmaxf(top[g], __uint_as_float(s[g / 2][g % 2 * 16 + 15]));
                    }
                    const float up = fmaxf(max3(top[0], top[1], top[2]), top[3]);
                    const bool grow = (up - m) * p.sl2 > kGrow;         // (from -infinity too, but not where both are)
                    if (__any_sync(0xffffffffu, grow)) {
                        const float corr = grow ? exp2_fast((m - up) * p.sl2) : 1.f;
                        if (grow) { m = up; l *= corr; off = -m * p.sl2; }
                        if (turn > 0) {             // (the first products overwrite O)
                            mbar_wait(o_done(q), (turn - 1) & 1, &abort_flag);
                            __syncwarp();
                            tc_after();
                            uint32_t o[32];
#pragma unroll 1
                            for (int c = 0; c < HD / 32; ++c) {
                                tmem_ld32(to + 32u * c, o);
                                tmem_wait_ld();
                                after_wait(o);
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                                tmem_st32(to + 32u * c, o);
                            }
                        }
                    }
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
                    uint32_t w[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        float x0, x1;
                        fma2(x0, x1, __uint_as_float(s[e / 16][e % 16 * 2]), __uint_as_float(s[e / 16][e % 16 * 2 + 1]), p.sl2, off);
                        x0 = exp2_fast(x0);
                        x1 = exp2_fast(x1);
                        add2(sum[2 * (e & 1)], sum[2 * (e & 1) + 1], x0, x1);
                        w[e] = Half<T>::pack(x0, x1);
                    }
                    tmem_st32(tb, w);
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tmem_wait_st();
                }
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(q, turn & 1));
                ++turn;
            }
        }
        // ---- O ----
        if (turn > 0) mbar_wait(retired(q), 0, &abort_flag);
        ok = __all_sync(0xffffffffu, !abort_flag);
        tc_after();
        const long long rows_total = (long long)a.batch * a.tokens * a.heads;
        if (PACKED || alt) {
            // Sums in fp32, through shared memory: so that rows are written whole (with one thread per row 4 us more), and that two tiles which are the same rows
            // add up.  For 128 dims they lie where the ring was, for 64 over Q too: what each tile multiplies has been multiplied when both have met here.
            constexpr int CH = HD / 4;          // 16-byte pieces of a row
            float4* stage = reinterpret_cast<float4*>(base_ptr + (HD == 128 ? ring : 0));
            float (*stats)[2][kRows] = reinterpret_cast<float (*)[2][kRows]>(stage + 2 * kRows * CH);              // behind them: [tile][maximum, denominator][row]
            long long (*places)[kRows] = reinterpret_cast<long long (*)[kRows]>(stats + 2);                         // the rows' places among the sums, or in out
            int* flags = reinterpret_cast<int*>(places + 2);                                                        // rows that are done again
            static_assert((HD == 128 ? SM::q_tile : 0) + 2 * kRows * HD * 4 + 2 * kRows * 16 + kRows * 4 <= SM::total - SM::q_tile - 1024, "");
            auto meet = [&](int phase) {
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(all_met);
                if (ok) ok = mbar_wait(all_met, phase & 1, &abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                tc_after();
            };
            meet(0);
            if (ok && mine) {
                places[q][r] = PACKED ? split * rows_total + (long long)token * a.heads + head : b * a.out_stride[0] + t * a.out_stride[1] + head * a.out_stride[2];
                stats[q][0][r] = m * p.sl2;
                stats[q][1][r] = l;
                if (q == 0) flags[r] = 0;
#pragma unroll 1
                for (int c = 0; c < HD / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld32(to + 32u * c, o);
                    tmem_wait_ld();
                    after_wait(o);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float4 f = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
                        if (turn == 0) f = make_float4(0.f, 0.f, 0.f, 0.f);       // (no keys)
                        stage[(q * kRows + r) * CH + ((8 * c + e) ^ (r & 7))] = f;
                    }
                }
            }
            meet(1);
            // A warp takes whole rows; a lane knows one of them: what its tiles' sums count, and where it goes.
            const int all = alt ? nrows[0] : nrows[0] + nrows[1], per_warp = alt ? kRows / kSoftmaxWarps : 2 * kRows / kSoftmaxWarps, row_0 = warp * per_warp;
            float w0 = 1.f, w1 = 0.f;
            long long place = 0;
            if (ok && lane < per_warp && row_0 + lane < all) {
                const int row = row_0 + lane, tile = row / kRows, at = row % kRows;
                place = places[tile][at];
                float tm = stats[tile][0][at], tl = stats[tile][1][at];
                if (alt) {
                    const float um = stats[1][0][at], both = fmaxf(tm, um), safe = both == -INFINITY ? 0.f : both;
                    w0 = exp2_fast(tm - safe);
                    w1 = exp2_fast(um - safe);
                    tl = tl * w0 + stats[1][1][at] * w1;
                    tm = both;
                }
                if constexpr (PACKED) {
                    *reinterpret_cast<float2*>(p.part + (p.splits + 1) * rows_total * HD + 2 * place) = make_float2(tm, tl);
                } else {
                    const float inv = tl != 0.f ? 1.f / tl : 0.f;         // (nothing seen: zero)
                    if (!isfinite(tl)) flags[at] = -1;                    // (a score that the row sees is a NaN)
                    w0 *= inv;
                    w1 *= inv;
                }
            }
            if (ok)
#pragma unroll 4
                for (int x = 0; x < per_warp * CH / 32; ++x) {
                    const int rw = (x * 32 + lane) / CH, row = row_0 + rw, chunk = lane % CH;
                    const float e0 = __shfl_sync(0xffffffffu, w0, rw), e1 = __shfl_sync(0xffffffffu, w1, rw);
                    const long long at = __shfl_sync(0xffffffffu, place, rw);
                    if (row >= all) continue;
                    float4 f = stage[row * CH + (chunk ^ (row & 7))];
                    if (alt) {
                        const float4 g = stage[(kRows + row) * CH + (chunk ^ (row & 7))];
                        f = make_float4(f.x * e0 + g.x * e1, f.y * e0 + g.y * e1, f.z * e0 + g.z * e1, f.w * e0 + g.w * e1);
                        if (e0 == 0.f && e1 == 0.f) f = make_float4(0.f, 0.f, 0.f, 0.f);       // (nothing seen, as above: not zero times a NaN)
                    }
                    if constexpr (PACKED) {
                        *reinterpret_cast<float4*>(p.part + at * HD + 4 * chunk) = f;
                    } else {
                        float mean[4] = {f.x, f.y, f.z, f.w};
                        // (a NaN or an infinity in V that the row does not see: done again below)
                        if (settle<T>(mean)) atomicOr(flags + row, 1);
                        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at + 4 * chunk) = make_uint2(Half<T>::pack(mean[0], mean[1]), Half<T>::pack(mean[2], mean[3]));
                    }
                }
            if constexpr (!PACKED) {
                meet(2);
                unsigned again = __ballot_sync(0xffffffffu, ok && q == 0 && r < rows && flags[r] > 0);
                while (again) {
                    const int from = __ffs(again) - 1, t2 = __shfl_sync(0xffffffffu, t, from);
                    again &= again - 1;
                    attn_row_again<T, HD>(a, b0, t2, __shfl_sync(0xffffffffu, head, from), pos0 + t2, 0, HD);
                }
            }
        } else if (ok && mine) {
            const float inv = l != 0.f ? 1.f / l : 0.f;
            const long long out_at = b * a.out_stride[0] + t * a.out_stride[1] + head * a.out_stride[2];
            bool bad = false;
            // A warp stores what it has staged, where other warps have written Q: the products with Q are done, or, in a tile that sees no keys and has
            // waited for none, Q is there (else it came down on rows that were staged already).
            uint8_t* stage = base_ptr + q * SM::q_tile;
            if (turn == 0) mbar_wait(q_full(q), 0, &abort_flag);
            __syncwarp();
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
                uint32_t o[32];
                if (turn > 0) {
                    tmem_ld32(to + 32u * c, o);
                    tmem_wait_ld();
                    after_wait(o);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float f[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) f[x] = turn == 0 || l == 0.f ? 0.f : __uint_as_float(o[8 * e + x]) * inv;       // (nothing seen: zero)
                    if (settle<T>(f)) bad = true;              // (a NaN or an infinity in V that the row does not see: done again below)
                    const uint4 h = make_uint4(Half<T>::pack(f[0], f[1]), Half<T>::pack(f[2], f[3]), Half<T>::pack(f[4], f[5]), Half<T>::pack(f[6], f[7]));
                    *reinterpret_cast<uint4*>(stage + r * HD * 2 + (((4 * c + e) ^ (r & 7)) << 4)) = h;
                }
            }
            __syncwarp();
            const int last = min(32, rows - 32 * quarter);
#pragma unroll 4
            for (int x = 0; x < HD / 8; ++x) {
                const int rw = (x * 32 + lane) / (HD / 8), rr = 32 * quarter + rw, c = lane % (HD / 8);
                const long long to_row = __shfl_sync(0xffffffffu, out_at, rw);
                if (rw < last)
                    *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + to_row + 8 * c) = *reinterpret_cast<const uint4*>(stage + rr * HD * 2 + ((c ^ (rr & 7)) << 4));
            }
            __syncwarp();
            unsigned again = __ballot_sync(0xffffffffu, bad && isfinite(l) && r < rows);     // (no finite denominator: a score that the row sees is a NaN)
            while (again) {
                const int from = __ffs(again) - 1, t2 = __shfl_sync(0xffffffffu, t, from);
                again &= again - 1;
                attn_row_again<T, HD>(a, b0, t2, __shfl_sync(0xffffffffu, head, from), pos0 + t2, 0, HD);
            }
        }
    }
    // ===== teardown: every role arrives here, also after a wait that ran out =====
    tc_before();
    __syncthreads();
    if (threadIdx.x == 0 && abort_flag && a.status) atomicExch(a.status, 1u);
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)kTmemCols) : "memory");
}

// One tensor map: boxes of 64 dims by 64 keys.  Strides of dimensions of size one are any that the encoder takes.
bool encode(CUtensorMap* m, bool bf16, int hd, const void* ptr, int rank, const int* sizes, const int64_t* strides) {
    const EncodeTiledFn fn = encode_tiled_fn();
    cuuint64_t dims[4] = {(cuuint64_t)hd}, st[3] = {};
    cuuint32_t box[4] = {64, kKeys, 1, 1}, est[4] = {1, 1, 1, 1};
    for (int i = 1; i < rank; ++i) {
        dims[i] = (cuuint64_t)sizes[i - 1];
        st[i - 1] = (cuuint64_t)(sizes[i - 1] == 1 ? hd : strides[i - 1]) * 2;
    }
    return fn && fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(ptr), dims, st, box, est,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD, bool PACKED>
int run(const b200gptq_attn_args& a, float* part, int splits, bool alt, cudaStream_t stream) {
    static std::once_flag once[64];
    static cudaError_t result[64];
    auto* kernel = attn_tiles_kernel<T, HD, PACKED>;
    int dev = 0;
    B200GPTQ_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return B200GPTQ_ERR_TOO_LARGE;
    std::call_once(once[dev], [&] { result[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<HD>::total); });
    B200GPTQ_CUDA_TRY(result[dev]);
    CUtensorMap mk = {}, mv = {}, mkp = {}, mvp = {};
    const int cache[3] = {a.max_seq, a.kv_heads, a.batch}, front[2] = {a.prefix, a.kv_heads};
    const int64_t ks[3] = {a.k_stride[2], a.k_stride[1], a.k_stride[0]}, vs[3] = {a.v_stride[2], a.v_stride[1], a.v_stride[0]};
    const int64_t kps[2] = {a.k_prefix_stride[1], a.k_prefix_stride[0]}, vps[2] = {a.v_prefix_stride[1], a.v_prefix_stride[0]};
    const bool bf16 = a.dtype == B200GPTQ_BF16;
    if ((!PACKED && !(encode(&mk, bf16, HD, a.k_cache, 4, cache, ks) && encode(&mv, bf16, HD, a.v_cache, 4, cache, vs))) ||
        (a.prefix && !(encode(&mkp, bf16, HD, a.k_prefix, 3, front, kps) && encode(&mvp, bf16, HD, a.v_prefix, 3, front, vps)))) {
        set_last_cuda_error((int)cudaErrorInvalidValue);
        return B200GPTQ_ERR_CUDA;
    }
    TileArgs t = {};
    t.a = a;
    t.part = part;
    t.sl2 = std::max(std::fabs(a.scale) * kLog2e, 1e-30f);        // (a scale of zero: all weights alike, and no infinity times zero)
    t.negate = a.scale < 0.f;
    t.splits = splits;
    t.group = a.heads / a.kv_heads;
    t.alt = alt;
    t.prefix_units = (int)((a.prefix + kKeys - 1) / kKeys);
    t.units_each = t.prefix_units / splits;
    t.units_more = t.prefix_units % splits;
    t.by_splits = Divisor(splits);
    t.by_kv_heads = Divisor(a.kv_heads);
    t.by_batch = Divisor(a.batch);
    t.by_group = Divisor(t.group);
    t.by_tokens = Divisor(a.tokens);
    const long long rows = (long long)a.tokens * (a.heads / a.kv_heads) * (PACKED ? a.batch : 1);
    const int per_cta = alt ? kRows : 2 * kRows;
    t.tiles = (int)((rows + per_cta - 1) / per_cta);
    const long long ctas = (long long)t.tiles * a.kv_heads * (PACKED ? splits : a.batch);
    if (ctas > 0x7fffffff) return B200GPTQ_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Smem<HD>::total - (alt ? Smem<HD>::q_tile : 0);
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = attn_pdl_enabled() ? 1 : 0;
    B200GPTQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, mk, mv, mkp, mvp, t));
    return B200GPTQ_OK;
}

template <bool PACKED>
int run_any(const b200gptq_attn_args& a, float* part, int splits, bool alt, cudaStream_t stream) {
    if (a.dtype == B200GPTQ_F16)
        return a.hd == 128 ? run<__half, 128, PACKED>(a, part, splits, alt, stream) : run<__half, 64, PACKED>(a, part, splits, alt, stream);
    return a.hd == 128 ? run<__nv_bfloat16, 128, PACKED>(a, part, splits, alt, stream) : run<__nv_bfloat16, 64, PACKED>(a, part, splits, alt, stream);
}

}  // namespace

// Whether tensor maps can describe the keys and values: no dimension that repeats (stride 0), strides below 2^40 bytes.
bool attn_tiles_maps(const b200gptq_attn_args& a, bool prefix) {
    auto fits = [](int size, int64_t stride) { return size == 1 || (stride > 0 && stride < (1LL << 39)); };
    if (prefix)
        for (const int64_t* s : {a.k_prefix_stride, a.v_prefix_stride})
            if (!fits(a.kv_heads, s[0]) || !fits(a.prefix, s[1])) return false;
    if (!prefix)
        for (const int64_t* s : {a.k_stride, a.v_stride})
            if (!fits(a.batch, s[0]) || !fits(a.kv_heads, s[1]) || !fits(a.max_seq, s[2])) return false;
    return true;
}

// One tile of rows per CTA, its units shared by both halves, where all tiles then run at once; else two.
int attn_tiles_dispatch(const b200gptq_attn_args& a, cudaStream_t stream) {
    const long long tiles = ((long long)a.tokens * (a.heads / a.kv_heads) + kRows - 1) / kRows * a.kv_heads * a.batch;
    return run_any<false>(a, nullptr, 1, tiles <= sm_count(), stream);
}

int attn_tiles_prefix(const b200gptq_attn_args& a, float* part, int parts, cudaStream_t stream) {
    return run_any<true>(a, part, parts, (long long)a.batch * a.tokens * (a.heads / a.kv_heads) <= kRows, stream);
}

}  // namespace b200gptq
