// b200gptq_attn for many query rows per key head: prompts and chunks of them, and the prefix part of a large batch.
//
//   S = Q K^T,  w = softmax(scale S) over the visible keys,  O = w V
//
// A CTA takes two tiles of 128 rows of Q that share a key head (rows are (token, head of the group), so that shared key heads fill a tile) and streams tiles
// of 128 keys that either of them sees: 2 hd multiplications and one exponential per row and key, and of the latter an SM makes 16 per clock where the
// tensor cores make 4096 of the former, so for 128 dims both take as long and have to run at once:
//
//   warps 0..3, 4..7  softmax of one tile of Q each, a thread per row: S from tensor memory into registers, the weights (16 bits) back over it.  O is
//                     only rescaled when a row's maximum grows by more than 2^8 over the one in use (no weight is above 2^8; fp32 sums)
//   warp 8            TMA: K and V tiles into a ring, in the order K0 V0 K1 V1 ..
//   warp 9            tcgen05.mma: PV of one tile of Q and QK of its next keys while the other tile's softmax runs.  Products are retired in order, so
//                     that S of the next keys may overwrite the weights, and the arrival of S says that O is complete up to the keys before
//
// Tensor memory: S of both tiles (2 x 128 columns; the weights lie over the first 64), O of both (2 x hd).  The weights are the A operand from
// tensor memory, V is the B operand as it lies (MN-major, keys along K).
//
// Rows of V that no row of the tiles sees are zeroed in shared memory before they are multiplied (a weight of zero times a NaN is one).  Where rows of the
// tiles see different keys and one of these holds a NaN or an infinity, the rows that come out not finite are done again, key by key.
//
// PACKED: the rows are (sequence, token, head of the group) of the whole batch against the shared prefix, split over CTAs, sums to scratch.  Up to 128 rows: both
// tiles of Q are the same rows, one takes the even tiles of keys and the other the odd ones.
#include <cuda.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "attn.cuh"
#include "attn.h"

namespace b200gptq {
namespace {

constexpr int kRows = 128, kKeys = 128, kLoadWarp = 8, kMmaWarp = 9, kThreads = 320;
constexpr int kTmemCols = 512, kColO = 256;          // S of tile q at 128 q, O at 256 + 128 q
constexpr float kGrow = 8.f;                         // log2 of what a maximum may grow before O is rescaled

template <int HD> struct Smem {
    static constexpr int tile = kKeys * HD * 2, stages = HD == 128 ? 4 : 6, q = 0, ring = 2 * tile, total = ring + stages * tile + 1024;
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
__device__ __forceinline__ void mma_commit(uint32_t bar) {       // arrives when all products issued so far have retired
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
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
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Operand tiles are boxes of 64 dims (128 bytes, swizzled) by 128 rows, one after the other.  Q and K: K-major, 8-row groups 1024 bytes apart.  V: MN-major,
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
    int negate, pairs, splits, part_splits, prefix_tiles;
};

template <typename T, int HD, bool PACKED>
__global__ void __launch_bounds__(kThreads, 1)
attn_tiles_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_kp,
                  const __grid_constant__ CUtensorMap map_vp, const __grid_constant__ TileArgs p) {
    using SM = Smem<HD>;
    constexpr int ST = SM::stages, BOX = kKeys * 128, HALVES = HD / 64;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - raw);
    __shared__ __align__(8) uint64_t bars[2 * ST + 8];
    __shared__ uint32_t tmem_base_holder;
    __shared__ volatile int abort_flag;

    const b200gptq_attn_args& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t bar_base = smem_u32(bars);
    auto full = [&](int s) { return bar_base + 8u * s; };
    auto empty = [&](int s) { return bar_base + 8u * (ST + s); };
    auto q_full = [&](int q) { return bar_base + 8u * (2 * ST + q); };
    auto s_full = [&](int q) { return bar_base + 8u * (2 * ST + 2 + q); };
    auto p_full = [&](int q) { return bar_base + 8u * (2 * ST + 4 + q); };
    auto o_full = [&](int q) { return bar_base + 8u * (2 * ST + 6 + q); };

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < ST; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int q = 0; q < 2; ++q) { mbar_init(q_full(q), 4); mbar_init(s_full(q), 1); mbar_init(p_full(q), 4); mbar_init(o_full(q), 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_holder)), "r"((uint32_t)kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = tmem_base_holder;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");

    // ---- which rows, which keys.  The last rows of a prompt see most, and come first. ----
    const int G = a.heads / a.kv_heads, window = a.window ? a.window : 1 << 30;
    const int split = PACKED ? blockIdx.x % p.splits : 0, unit = PACKED ? blockIdx.x / p.splits : blockIdx.x;
    const int kh = unit % a.kv_heads, b0 = PACKED ? 0 : unit / a.kv_heads % a.batch;
    const int pair = p.pairs - 1 - unit / a.kv_heads / (PACKED ? 1 : a.batch), row0 = pair * 2 * kRows;
    const int pos0 = PACKED ? 0 : attn_pos(a, b0);
    const int rows_all = PACKED ? a.batch * a.tokens * G : attn_count(a, b0) * G;
    const bool alt = PACKED && rows_all <= kRows;       // both tiles are the same rows
    int nrows[2], p_lo[2], p_hi[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int r = row0 + (alt ? 0 : q * kRows);
        nrows[q] = max(0, min(kRows, rows_all - r));
        p_lo[q] = pos0 + r / G;
        p_hi[q] = pos0 + (r + max(nrows[q], 1) - 1) / G;
    }
    int n_tiles = 0, n_s = 0, first = 0;
    AttnRange range = {0, 0, 0};
    if (nrows[0] > 0) {
        if constexpr (PACKED) {
            first = (int)((long long)p.prefix_tiles * split / p.splits);
            n_tiles = (int)((long long)p.prefix_tiles * (split + 1) / p.splits) - first;
        } else {
            range = attn_range(p_lo[0], nrows[1] > 0 ? p_hi[1] : p_hi[0], window, a.sinks, a.max_seq);
            n_s = (range.s_end + kKeys - 1) / kKeys;
            n_tiles = p.prefix_tiles + n_s + (range.w_end - range.w_start + kKeys - 1) / kKeys;
        }
    }
    struct Keys { int j0, end; bool prefix; };
    auto keys_at = [&](int i) {
        Keys k;
        if constexpr (PACKED) { k.prefix = true; k.j0 = (first + i) * kKeys; k.end = a.prefix; return k; }
        k.prefix = i < p.prefix_tiles;
        i -= p.prefix_tiles;
        k.j0 = k.prefix ? (i + p.prefix_tiles) * kKeys : i < n_s ? i * kKeys : range.w_start + (i - n_s) * kKeys;
        k.end = k.prefix ? a.prefix : i < n_s ? range.s_end : range.w_end;
        return k;
    };
    auto needs = [&](int q, int i) {          // whether any row of tile q sees any of the keys
        if (nrows[q] <= 0) return false;
        if (alt) return (i & 1) == q;
        if (PACKED) return true;
        const Keys k = keys_at(i);
        return k.prefix || (k.j0 <= p_hi[q] && (k.j0 + kKeys - 1 > p_lo[q] - window || k.j0 < a.sinks));
    };

    bool ok = true;
    if (warp == kLoadWarp) {
        // ===== keys and values =====
        if (elect_one()) {
            int n = 0;                        // loads issued: K i is number 2 i, V i number 2 i + 1
            for (; n < 2 * n_tiles && ok; ++n) {
                const int s = n % ST;
                if (n >= ST) ok = mbar_wait(empty(s), (n / ST - 1) & 1, &abort_flag);
                if (!ok) break;
                const Keys k = keys_at(n / 2);
                const uint32_t dst = base + SM::ring + s * SM::tile, bar = full(s);
                mbar_expect(bar, SM::tile);
#pragma unroll
                for (int h = 0; h < HALVES; ++h) {
                    if (k.prefix) tma_3d(dst + h * BOX, (n & 1) ? &map_vp : &map_kp, 64 * h, k.j0, kh, bar);
                    else tma_4d(dst + h * BOX, (n & 1) ? &map_v : &map_k, 64 * h, k.j0, kh, b0, bar);
                }
            }
            if (!ok) {                        // what is on its way lands before the CTA ends
                int never = 0;
                for (int i = max(0, n - ST); i < n; ++i) mbar_wait(full(i % ST), (i / ST) & 1, &never);
            }
        }
        __syncwarp();
    } else if (warp == kMmaWarp) {
        // ===== products =====
        constexpr uint32_t type = std::is_same<T, __half>::value ? 0u : 1u;
        constexpr uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)(kRows >> 4) << 24);
        constexpr uint32_t idesc_qk = idesc | ((uint32_t)(kKeys >> 3) << 17), idesc_pv = idesc | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
        int started[2] = {0, 0}, mixed[2] = {0, 0};      // QK and PV issued
        auto wait_load = [&](int n) { if (ok) ok = mbar_wait(full(n % ST), (n / ST) & 1, &abort_flag); ok = __all_sync(0xffffffffu, ok); };
        auto release = [&](int n) { if (elect_one()) mma_commit(empty(n % ST)); __syncwarp(); };
        auto qk = [&](int q, int i) {
            if (started[q]++ == 0) {
                ok = mbar_wait(q_full(alt ? 0 : q), 0, &abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return;
            }
            tc_after();
            if (elect_one()) {
                const uint64_t ad = smem_desc(base + SM::q + (alt ? 0 : q) * SM::tile, 0), bd = smem_desc(base + SM::ring + (2 * i) % ST * SM::tile, 0);
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {
                    const uint32_t off = (k / 4 * BOX + k % 4 * 32) >> 4;
                    mma_ss(tmem + 128u * q, ad + off, bd + off, idesc_qk, k > 0 ? 1u : 0u);
                }
                mma_commit(s_full(q));
            }
            __syncwarp();
        };
        if (n_tiles > 0) {
            wait_load(0);
            for (int q = 0; q < 2 && ok; ++q)
                if (needs(q, 0)) qk(q, 0);
            release(0);
        }
        for (int i = 0; i < n_tiles && ok; ++i) {
            const int v = 2 * i + 1, s = v % ST;
            const uint32_t vt = base + SM::ring + s * SM::tile;
            wait_load(v);
            if (!ok) break;
            const Keys k = keys_at(i);
            if (k.j0 + kKeys > k.end) {       // rows that nobody sees
                for (int x = lane; x < (k.j0 + kKeys - k.end) * HALVES * 8; x += 32) {
                    const int r = k.end - k.j0 + x / (HALVES * 8), c = x % (HALVES * 8);
                    *reinterpret_cast<uint4*>(base_ptr + (vt - base) + (c / 8) * BOX + r * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            for (int q = 0; q < 2 && ok; ++q) {
                if (needs(q, i)) {
                    ok = mbar_wait(p_full(q), mixed[q] & 1, &abort_flag);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_after();
                    if (elect_one()) {
                        const uint64_t bd = smem_desc(vt, BOX);
#pragma unroll
                        for (int k16 = 0; k16 < kKeys / 16; ++k16)
                            mma_ts(tmem + kColO + 128u * q, tmem + 128u * q + 8u * k16, bd + k16 * (2048 >> 4), idesc_pv, (mixed[q] > 0 || k16 > 0) ? 1u : 0u);
                    }
                    __syncwarp();
                    ++mixed[q];
                }
                if (i + 1 < n_tiles) {
                    wait_load(v + 1);
                    if (ok && needs(q, i + 1)) qk(q, i + 1);
                }
            }
            if (!ok) break;
            release(v);
            if (i + 1 < n_tiles) release(v + 1);
        }
        if (elect_one()) { mma_commit(o_full(0)); mma_commit(o_full(1)); }
        __syncwarp();
        int never = 0;                        // (also after a wait that ran out: nothing is in flight when tensor memory is freed)
        mbar_wait(o_full(1), 0, &never);
    } else {
        // ===== softmax of tile q, one row per thread =====
        const int q = warp >> 2, r = threadIdx.x & 127, rows = nrows[q], row_first = row0 + (alt ? 0 : q * kRows);
        const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16, ts = tmem + 128u * q + lane_off, to = tmem + kColO + 128u * q + lane_off;
        const bool mine = 32 * (warp & 3) < rows;       // the warp has rows at all
        // Q, in the swizzled layout of the tiles
        if (!(alt && q == 1)) {
            uint8_t* dst = base_ptr + SM::q + q * SM::tile;
            for (int x = lane; x < 32 * HD / 8; x += 32) {
                const int rr = 32 * (warp & 3) + x / (HD / 8), c = x % (HD / 8);
                uint4 val = make_uint4(0, 0, 0, 0);
                if (rr < rows) {
                    const int idx = row_first + rr, tok = idx / G, head = kh * G + idx - tok * G;
                    const int b = PACKED ? tok / a.tokens : b0, t = PACKED ? tok - b * a.tokens : tok;
                    val = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.q_stride[0] + t * a.q_stride[1] + head * a.q_stride[2] + 8 * c));
                    if (p.negate) { val.x ^= 0x80008000u; val.y ^= 0x80008000u; val.z ^= 0x80008000u; val.w ^= 0x80008000u; }
                }
                *reinterpret_cast<uint4*>(dst + (c / 8) * BOX + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = val;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full(q));
        }
        const int pr = pos0 + (row_first + min(r, max(rows, 1) - 1)) / G;
        float m = -INFINITY, l = 0.f;           // the maximum in use (of scores, not scaled), the denominator
        int turn = 0;
        for (int i = 0; i < n_tiles; ++i) {
            if (!needs(q, i)) continue;
            ok = mbar_wait(s_full(q), turn & 1, &abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_after();
            if (mine) {
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32u * c, s[c]);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 4; ++c) after_wait(s[c]);
                const Keys k = keys_at(i);
                bool whole = k.j0 + kKeys <= k.end;
                if (!k.prefix) whole = whole && k.j0 + kKeys - 1 <= p_lo[q] && (k.j0 > p_hi[q] - window || k.j0 + kKeys <= a.sinks);
                if (!whole) {
                    // columns [0, front) and [lo, hi) are seen
                    int front = k.end - k.j0, lo = 0, hi = 0;
                    if (!k.prefix) {
                        front = min(min(a.sinks, pr + 1), k.end) - k.j0;
                        lo = pr - window + 1 - k.j0;
                        hi = min(pr + 1, k.end) - k.j0;
                    }
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const int x = 32 * c + e;
                            if (!(x < front || (x >= lo && x < hi))) s[c][e] = 0xff800000u;       // -infinity
                        }
                }
                float top[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    top[c] = __uint_as_float(s[c][0]);
#pragma unroll
                    for (int e = 1; e < 32; ++e) top[c] = fmaxf(top[c], __uint_as_float(s[c][e]));
                }
                const float up = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                const bool grow = up > m && (m == -INFINITY || (up - m) * p.sl2 > kGrow);
                if (__any_sync(0xffffffffu, grow)) {
                    const float corr = grow ? exp2_fast((m - up) * p.sl2) : 1.f;
                    if (grow) { m = up; l *= corr; }
                    if (turn > 0) {             // (the first products overwrite O)
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
                const float off = m == -INFINITY ? 0.f : -m * p.sl2;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t w[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const int c = 2 * half + e / 16;
                        const float x0 = exp2_fast(fmaf(__uint_as_float(s[c][e % 16 * 2]), p.sl2, off));
                        const float x1 = exp2_fast(fmaf(__uint_as_float(s[c][e % 16 * 2 + 1]), p.sl2, off));
                        sum[e & 1] += x0;
                        sum[2 + (e & 1)] += x1;
                        w[e] = Half<T>::pack(x0, x1);
                    }
                    tmem_st32(ts + 32u * half, w);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_wait_st();
            }
            tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(q));
            ++turn;
        }
        // ---- O ----
        if (ok && rows > 0) {
            if (turn > 0) {
                ok = mbar_wait(o_full(q), 0, &abort_flag);
                ok = __all_sync(0xffffffffu, ok);
            }
            tc_after();
            const long long rows_total = (long long)a.batch * a.tokens * a.heads;
            const float inv = l != 0.f ? 1.f / l : 0.f;
            bool bad = false;
            uint8_t* stage = base_ptr + SM::q + q * SM::tile;            // (the products with Q are done)
            const int idx = row_first + min(r, rows - 1);
            const long long at = (PACKED ? (alt ? 2 * split + q : split) * rows_total : 0LL) + (long long)(idx / G) * a.heads + kh * G + idx % G;
            if (ok && mine)
#pragma unroll 1
                for (int c = 0; c < HD / 32; ++c) {
                    uint32_t o[32];
                    if (turn > 0) {
                        tmem_ld32(to + 32u * c, o);
                        tmem_wait_ld();
                        after_wait(o);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0u;
                    }
                    if constexpr (PACKED) {
                        if (r < rows) {
                            float4* dst = reinterpret_cast<float4*>(p.part + at * HD + 32 * c);
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                dst[e] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float f[8];
#pragma unroll
                            for (int x = 0; x < 8; ++x) {
                                // (nothing seen: zero; a NaN or an infinity in V that the row does not see: done again below)
                                f[x] = l == 0.f ? 0.f : __uint_as_float(o[8 * e + x]) * inv;
                                bad = bad || !isfinite(f[x]);
                            }
                            const uint4 h = make_uint4(Half<T>::pack(f[0], f[1]), Half<T>::pack(f[2], f[3]), Half<T>::pack(f[4], f[5]), Half<T>::pack(f[6], f[7]));
                            const int chunk = 4 * c + e;
                            *reinterpret_cast<uint4*>(stage + r * HD * 2 + ((chunk ^ (r & 7)) << 4)) = h;
                        }
                    }
                }
            if constexpr (PACKED) {
                if (ok && r < rows) {
                    float* ml = p.part + p.part_splits * rows_total * HD + 2 * at;
                    ml[0] = m * p.sl2;
                    ml[1] = l;
                }
            } else {
                __syncwarp();                   // (a warp stores its own rows)
                const int last = min(32, rows - 32 * (warp & 3));
                for (int x = lane; ok && x < last * (HD / 8); x += 32) {
                    const int rr = 32 * (warp & 3) + x / (HD / 8), c = x % (HD / 8), id = row_first + rr, t = id / G, head = kh * G + id - t * G;
                    *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + b0 * a.out_stride[0] + t * a.out_stride[1] + head * a.out_stride[2] + 8 * c) =
                        *reinterpret_cast<const uint4*>(stage + rr * HD * 2 + ((c ^ (rr & 7)) << 4));
                }
                __syncwarp();
                unsigned again = __ballot_sync(0xffffffffu, bad && r < rows && ok);
                while (again) {
                    const int rr = 32 * (warp & 3) + __ffs(again) - 1, id = row_first + rr, t = id / G;
                    again &= again - 1;
                    attn_row_again<T, HD>(a, b0, t, kh * G + id - t * G, pos0 + t, 0, HD);
                }
            }
        }
    }
    // ===== teardown: every role arrives here, also after a wait that ran out =====
    tc_before();
    __syncthreads();
    if (threadIdx.x == 0 && abort_flag && a.status) atomicExch(a.status, 1u);
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)kTmemCols) : "memory");
}

// One tensor map: boxes of 64 dims by 128 rows.  Strides of dimensions of size one are any that the encoder takes.
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
int run(const b200gptq_attn_args& a, float* part, int splits, int part_splits, cudaStream_t stream) {
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
    t.part_splits = part_splits;
    t.prefix_tiles = (int)((a.prefix + kKeys - 1) / kKeys);
    const long long rows = (long long)a.tokens * (a.heads / a.kv_heads) * (PACKED ? a.batch : 1);
    t.pairs = (int)((rows + 2 * kRows - 1) / (2 * kRows));
    const long long ctas = (long long)t.pairs * a.kv_heads * (PACKED ? splits : a.batch);
    if (ctas > 0x7fffffff) return B200GPTQ_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Smem<HD>::total;
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
int run_any(const b200gptq_attn_args& a, float* part, int splits, int part_splits, cudaStream_t stream) {
    if (a.dtype == B200GPTQ_F16)
        return a.hd == 128 ? run<__half, 128, PACKED>(a, part, splits, part_splits, stream) : run<__half, 64, PACKED>(a, part, splits, part_splits, stream);
    return a.hd == 128 ? run<__nv_bfloat16, 128, PACKED>(a, part, splits, part_splits, stream) : run<__nv_bfloat16, 64, PACKED>(a, part, splits, part_splits, stream);
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

int attn_tiles_dispatch(const b200gptq_attn_args& a, cudaStream_t stream) { return run_any<false>(a, nullptr, 1, 0, stream); }

// `parts` sums per row: runs of the prefix, or two of each (up to 128 rows).
int attn_tiles_prefix(const b200gptq_attn_args& a, float* part, int parts, cudaStream_t stream) {
    const bool alt = (long long)a.batch * a.tokens * (a.heads / a.kv_heads) <= kRows;
    return run_any<true>(a, part, alt ? parts / 2 : parts, parts, stream);
}

}  // namespace b200gptq
