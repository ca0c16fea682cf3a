// ec_tree_tc.cu -- the tree attention of ec_tree.cu on the 5th-generation
// tensor cores, for tiles of 128 rows: large drafts, or many query heads on a
// KV head.
//
// A CTA (two per SM) takes its piece of the line of pages, tile by tile:
//   warp 5     TMA producer: K and V of a page, [64 positions][hd] each in
//              columns of 128 bytes with the 128-byte swizzle, into a ring
//   warp 4     one thread issues the MMAs: S = Q K^T (128 x 64, both operands
//              K-major in shared memory) into one of two S buffers, and
//              O += P V with P from tensor memory and V as it lies (rows of hd,
//              "MN-major")
//   warps 0-3  one row per thread: S from tensor memory, the positions that
//              the row sees, running maximum and sum, P back over S as 16-bit
//              pairs; O is rescaled in tensor memory only when the maximum has
//              grown by more than 2^8 (the reference of a row is any earlier
//              maximum, and p stays below 2^14)
// so that the products of one page run under the exponentials of the next,
// and one CTA's under the other's.  Per page and SM: 128 x 64 exponentials, 512
// cycles of the special function units, and 2 x 128 x 64 x hd products, 350
// (hd 64) to 700 (hd 128) cycles at the rate that cuBLAS reaches.  Every wait is
// bounded; loads use no multicast.
#include "ec_tree.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>
#include <pthread.h>
#include <string.h>

namespace {

constexpr int TT_THREADS = 192, TT_ROWS = 128;
constexpr float TT_GROWTH = 8.0f;                      // log2 growth of a maximum that is let be

template <int QT, int KT, int HD> struct TtCfg {
    static constexpr bool BF = KT == EC_T_BF16;
    static constexpr int COLS = HD / 64;               // 128-byte columns of a row
    static constexpr int TILE = 64 * HD * 2;           // K or V of a page
    static constexpr int KS = HD == 64 ? 5 : 3, VS = HD == 64 ? 4 : 2;   // pages of K and of V in flight: K is free once S is done
    static constexpr int Q_BYTES = TT_ROWS * HD * 2;
    static constexpr int SMEM = Q_BYTES + (KS + VS) * TILE + 256;
    static constexpr int TMEM = 256;                   // S 2 x 64, O up to 128 columns: two CTAs share an SM's 512
    static constexpr float LIFT = BF ? 0.0f : 6.0f;
    static constexpr uint32_t TYPES = (1u << 4) | ((BF ? 1u : 0u) << 7) | ((BF ? 1u : 0u) << 10) | ((uint32_t)(TT_ROWS >> 4) << 24);
    static constexpr uint32_t IDESC_S = TYPES | ((64u >> 3) << 17);
    static constexpr uint32_t IDESC_O = TYPES | (1u << 16) | ((uint32_t)(HD >> 3) << 17);   // B is MN-major
};

// Shared-memory descriptors, 128-byte swizzle: start, leading and stride byte
// offsets (>> 4), version 1, mode 2.  K-major: 8-row groups 1024 bytes apart.
// MN-major: 8-row (K) groups 1024 bytes apart, 64-element columns `lead` apart.
EC_DEV uint64_t tt_desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
EC_DEV void tt_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t more) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(more), "r"(0u));
}
EC_DEV void tt_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t more) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(more), "r"(0u));
}
EC_DEV void tt_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(ec_smem_u32(bar)) : "memory");
}
EC_DEV void tt_arrive(uint64_t *bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(ec_smem_u32(bar)) : "memory"); }
EC_DEV void tt_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
EC_DEV void tt_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
EC_DEV void tt_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
EC_DEV void tt_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 64 or 32 columns of this thread's row, arrived (the wait is part of the
// statement: nothing may use the registers before it)
EC_DEV void tt_ld64(uint32_t taddr, float *f) {
    __syncwarp();   // a whole warp executes these as one
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
                 "%30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, "
                 "%58, %59, %60, %61, %62, %63}, [%64];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]), "=f"(f[8]), "=f"(f[9]), "=f"(f[10]),
                   "=f"(f[11]), "=f"(f[12]), "=f"(f[13]), "=f"(f[14]), "=f"(f[15]), "=f"(f[16]), "=f"(f[17]), "=f"(f[18]), "=f"(f[19]), "=f"(f[20]),
                   "=f"(f[21]), "=f"(f[22]), "=f"(f[23]), "=f"(f[24]), "=f"(f[25]), "=f"(f[26]), "=f"(f[27]), "=f"(f[28]), "=f"(f[29]), "=f"(f[30]),
                   "=f"(f[31]), "=f"(f[32]), "=f"(f[33]), "=f"(f[34]), "=f"(f[35]), "=f"(f[36]), "=f"(f[37]), "=f"(f[38]), "=f"(f[39]), "=f"(f[40]),
                   "=f"(f[41]), "=f"(f[42]), "=f"(f[43]), "=f"(f[44]), "=f"(f[45]), "=f"(f[46]), "=f"(f[47]), "=f"(f[48]), "=f"(f[49]), "=f"(f[50]),
                   "=f"(f[51]), "=f"(f[52]), "=f"(f[53]), "=f"(f[54]), "=f"(f[55]), "=f"(f[56]), "=f"(f[57]), "=f"(f[58]), "=f"(f[59]), "=f"(f[60]),
                   "=f"(f[61]), "=f"(f[62]), "=f"(f[63])
                 : "r"(taddr) : "memory");
}
EC_DEV void tt_ld32(uint32_t taddr, float *f) {
    __syncwarp();
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
                 "%30, %31}, [%32];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]), "=f"(f[8]), "=f"(f[9]), "=f"(f[10]),
                   "=f"(f[11]), "=f"(f[12]), "=f"(f[13]), "=f"(f[14]), "=f"(f[15]), "=f"(f[16]), "=f"(f[17]), "=f"(f[18]), "=f"(f[19]), "=f"(f[20]),
                   "=f"(f[21]), "=f"(f[22]), "=f"(f[23]), "=f"(f[24]), "=f"(f[25]), "=f"(f[26]), "=f"(f[27]), "=f"(f[28]), "=f"(f[29]), "=f"(f[30]),
                   "=f"(f[31])
                 : "r"(taddr) : "memory");
}
EC_DEV void tt_st32(uint32_t taddr, const uint32_t *r) {
    __syncwarp();
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, "
                 "%26, %27, %28, %29, %30, %31, %32};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                   "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
                   "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
                 : "memory");
}

EC_DEV void tt_load(uint32_t dst, const CUtensorMap *map, uint64_t *bar, int x, int page) {   // 64 positions of 128 bytes
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(map), "r"(ec_smem_u32(bar)), "r"(x), "r"(0), "r"(page) : "memory");
}

// Bounded wait; false (and the error word set) if the phase never completes
// or another role has given up.
EC_DEV bool tt_wait(uint64_t *bar, uint32_t parity, volatile int *stop, int *err) {
    for (uint32_t i = 0; i < EC_WAIT_LIMIT; ++i) {
        if (ec_mbar_try_wait(bar, parity)) return true;
        if (*stop) return false;
    }
    *stop = 1;
    atomicCAS(err, 0, EC_KERR_WAIT_TIMEOUT);
    return false;
}

// The same for a whole warp, which goes on together: lane 0 waits.
EC_DEV bool tt_wait_warp(uint64_t *bar, uint32_t parity, volatile int *stop, int *err) {
    int ok = 0;
    if ((threadIdx.x & 31) == 0) ok = tt_wait(bar, parity, stop, err);
    ok = __shfl_sync(0xffffffffu, ok, 0);
    __syncwarp();
    return ok != 0;
}

// OR over the 128 threads of the row warps.  A warp whose wait gave up goes on
// to take part in every one of these, so that no other waits for it.
EC_DEV bool tt_any(bool v) {
    int r;
    __syncwarp();
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %1, 0;\n\tbar.red.or.pred p, 1, 128, p;\n\tselp.s32 %0, 1, 0, p;\n\t}" : "=r"(r) : "r"((int)v) : "memory");
    return r != 0;
}

struct TtMaps { CUtensorMap k, v; };

template <int QT, int KT, int HD>
__global__ void __launch_bounds__(TT_THREADS, 2)
k_tree_tc(const __grid_constant__ TtMaps maps, const ec_kv_pages kv, const ec_tree_attn a, const TaGeo g, int *err) {
    typedef TtCfg<QT, KT, HD> C;
    constexpr int KS = C::KS, VS = C::VS, TILE = C::TILE;
    extern __shared__ __align__(1024) unsigned char smem[];
    const uint32_t base = ec_smem_u32(smem);              // 1024-byte aligned: the kernel has no other shared memory
    const uint32_t k_ring = base + C::Q_BYTES, v_ring = k_ring + KS * TILE;
    uint64_t *k_full = reinterpret_cast<uint64_t *>(smem + C::Q_BYTES + (KS + VS) * TILE), *k_empty = k_full + KS;
    uint64_t *v_full = k_empty + KS, *v_empty = v_full + VS, *s_full = v_empty + VS, *p_ready = s_full + 2, *o_done = p_ready + 2, *drain = o_done + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *stop_word = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < KS; ++i) {
            ec_mbar_init(&k_full[i], 1);
            ec_mbar_init(&k_empty[i], 1);
        }
        for (int i = 0; i < VS; ++i) {
            ec_mbar_init(&v_full[i], 1);
            ec_mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            ec_mbar_init(&s_full[i], 1);
            ec_mbar_init(&p_ready[i], 4);   // an arrival per row warp
        }
        ec_mbar_init(o_done, 1);
        ec_mbar_init(drain, 1);
        *stop_word = (base & 1023) != 0;
        if (base & 1023) atomicCAS(err, 0, EC_KERR_BAD_INDEX);
        ec_fence_mbar_init();
    }
    if (warp == 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ec_smem_u32(tmem_slot)), "r"(C::TMEM));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tt_before();
    __syncthreads();
    tt_after();
    const uint32_t tmem = *tmem_slot, tmem_o = tmem + 128;
    EC_PDL_ENTER();

    TaLine line;
    line.init(kv, a, g, TT_ROWS, gridDim.x, err);
    int at = (int)blockIdx.x < line.n ? line.start(blockIdx.x) : 0;
    const int stop_at = (int)blockIdx.x < line.n ? line.start(blockIdx.x + 1) : 0;
    int count = 0;        // pages of this CTA so far: stages count % KS and % VS, S buffer count % 2
    int k_issued = 0, v_issued = 0, next = 0;   // producer: loads issued, arena page of the next one
    while (at < stop_at) {
        int begin;
        const TaTile s = line.tile(kv, a, g, TT_ROWS, at, begin, err);
        const int p_begin = s.page0 + (at - begin), p_end = min(s.page1, p_begin + (stop_at - at)), pages = p_end - p_begin;
        const int kh = s.kh, end = s.base + s.t;

        // The producer: what the rings hold before the row warps are met below
        // (they are empty: the last tile is done), the rest after.
        auto produce = [&](int i0, int i1) {
            for (int i = i0; i < i1; ++i) {
                const int n = count + i, ks = n % KS, vs = n % VS, page = next;
                if (i + 1 < pages) next = ta_page(kv, s.slot, p_begin + i + 1, err);
                if (n >= KS && !tt_wait(&k_empty[ks], (uint32_t)((n / KS - 1) & 1), stop_word, err)) break;
                ec_mbar_expect_tx(&k_full[ks], TILE);
#pragma unroll
                for (int c = 0; c < C::COLS; ++c) tt_load(k_ring + ks * TILE + c * 8192, &maps.k, &k_full[ks], kh * HD + c * 64, page);
                k_issued = n + 1;
                if (n >= VS && !tt_wait(&v_empty[vs], (uint32_t)((n / VS - 1) & 1), stop_word, err)) break;
                ec_mbar_expect_tx(&v_full[vs], TILE);
#pragma unroll
                for (int c = 0; c < C::COLS; ++c) tt_load(v_ring + vs * TILE + c * 8192, &maps.v, &v_full[vs], kh * HD + c * 64, page);
                v_issued = n + 1;
            }
        };
        if (warp == 5) {
            if (lane == 0) {
                next = ta_page(kv, s.slot, p_begin, err);
                produce(0, min(pages, VS));
            }
        } else if (warp < 4) {
            // the queries: rows behind the sequence are zero
            const bool wide = (a.ldq & 7) == 0 && (reinterpret_cast<uintptr_t>(a.q) & 15) == 0;
#pragma unroll 4
            for (int i = threadIdx.x; i < TT_ROWS * HD / 8; i += 128) {
                const int r = i / (HD / 8), c = i % (HD / 8), rr = s.first + r, node = ta_node(g, rr);
                uint4 u = make_uint4(0u, 0u, 0u, 0u);
                if (node < s.t) {
                    const uint16_t *q = static_cast<const uint16_t *>(a.q) + (size_t)(s.r0 + node) * a.ldq + (size_t)(kh * g.group + rr - node * g.group) * HD + c * 8;
                    if (wide) u = *reinterpret_cast<const uint4 *>(q);
                    else u = make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16, q[6] | (uint32_t)q[7] << 16);
                }
                *reinterpret_cast<uint4 *>(smem + (c / 8) * (TT_ROWS * 128) + r * 128 + (((c % 8) ^ (r & 7)) << 4)) = u;
            }
            // O starts from zero
            uint32_t zero[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) zero[i] = 0u;
#pragma unroll
            for (int c = 0; c < HD; c += 32) tt_st32(tmem_o + ((uint32_t)(warp * 32) << 16) + c, zero);
            tt_wait_st();
            tt_proxy();
            tt_before();
        }
        __syncthreads();
        tt_after();

        if (warp == 5) {
            if (lane == 0) produce(min(pages, VS), pages);
        } else if (warp == 4) {
            if (lane == 0) {
                const uint64_t dq = tt_desc(base, 16);
                for (int i = 0; i <= pages; ++i) {
                    if (i < pages) {   // S of page i
                        const int n = count + i, ks = n % KS;
                        if (!tt_wait(&k_full[ks], (uint32_t)((n / KS) & 1), stop_word, err)) break;
                        tt_after();
                        const uint64_t dk = tt_desc(k_ring + ks * TILE, 16);
#pragma unroll
                        for (int k = 0; k < HD / 16; ++k)
                            tt_mma_ss(tmem + (n & 1) * 64, dq + (k / 4) * (TT_ROWS * 128 >> 4) + (k % 4) * 2, dk + (k / 4) * (8192 >> 4) + (k % 4) * 2, C::IDESC_S, k > 0);
                        tt_commit(&s_full[n & 1]);
                        tt_commit(&k_empty[ks]);
                    }
                    if (i > 0) {       // P V of page i - 1
                        const int n = count + i - 1, vs = n % VS;
                        if (!tt_wait(&v_full[vs], (uint32_t)((n / VS) & 1), stop_word, err)) break;
                        if (!tt_wait(&p_ready[n & 1], (uint32_t)((n / 2) & 1), stop_word, err)) break;
                        tt_after();
                        const uint64_t dv = tt_desc(v_ring + vs * TILE, 8192);
#pragma unroll
                        for (int k = 0; k < 4; ++k) tt_mma_ts(tmem_o, tmem + (n & 1) * 64 + k * 8, dv + k * (2048 >> 4), C::IDESC_O, 1);
                        tt_commit(&v_empty[vs]);
                        tt_commit(o_done);
                    }
                }
            }
        } else if (warp < 4) {
            const int row = threadIdx.x, rr = s.first + row, node = ta_node(g, rr);
            const uint32_t lane_at = (uint32_t)(warp * 32) << 16;
            const float f = g.scale2;
            float m = -INFINITY, l = 0.0f;
            bool ok = true;
            for (int i = 0; i < pages; ++i) {
                const int n = count + i, vs = n % VS, p0 = (p_begin + i) * PAGE;
                const bool part = p0 + PAGE > s.base || (a.window > 0 && p0 < (long long)s.base + 64 * a.mask_words - a.window);
                ok = ok && tt_wait_warp(&s_full[n & 1], (uint32_t)((n / 2) & 1), stop_word, err);
                if (!ok) {
                    if (part && tt_any(false)) {
                        tt_any(false);
                        tt_any(false);
                    }
                    continue;
                }
                tt_after();
                float x[64];
                tt_ld64(tmem + lane_at + (n & 1) * 64, x);
                unsigned long long see = ~0ull;
                if (part) {
                    see = ta_allow(a, s, node, p0);
#pragma unroll
                    for (int j = 0; j < 64; ++j)
                        if (!((j < 32 ? (uint32_t)see >> j : (uint32_t)(see >> 32) >> (j - 32)) & 1u)) x[j] = -INFINITY;
                }
                float hi[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                for (int j = 4; j < 64; ++j) hi[j & 3] = fmaxf(hi[j & 3], x[j]);
                const float top = fmaxf(fmaxf(hi[0], hi[1]), fmaxf(hi[2], hi[3])) * f;
                const bool grow = top > m + TT_GROWTH || (m == -INFINITY && top > m);
                float scale = 1.0f;
                if (grow) {
                    scale = ex2(m - top);   // 0 at first
                    m = top;
                    l *= scale;
                }
                bool odd = false;
                if (part) {
                    // V of positions that are not there is zero, and infinities
                    // and NaN (0 times them is NaN) are taken out and added by
                    // the rows that see them
                    unsigned char *v = smem + (v_ring - base) + vs * TILE;
                    constexpr uint32_t E = C::BF ? 0x7f80u : 0x7c00u;
                    ok = tt_wait_warp(&v_full[vs], (uint32_t)((n / VS) & 1), stop_word, err);
                    for (int b = row; b < TILE / 16; b += 128) {
                        const int pos = (b * 16 % 8192) / 128;
                        uint4 *u = reinterpret_cast<uint4 *>(v + b * 16);
                        if (p0 + pos >= end) {
                            *u = make_uint4(0u, 0u, 0u, 0u);
                        } else {
                            const uint4 w = *u;
                            const uint32_t w4[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) odd |= (w4[j] & E) == E || (w4[j] >> 16 & E) == E;
                        }
                    }
                    tt_proxy();
                    odd = tt_any(odd);
                }
                if (__any_sync(0xffffffffu, grow) || odd) {
                    // all earlier products are in O
                    if (n > 0) ok = tt_wait_warp(o_done, (uint32_t)((n - 1) & 1), stop_word, err) && ok;
                    tt_after();
#pragma unroll
                    for (int c = 0; c < HD; c += 32) {
                        float o[32];
                        tt_ld32(tmem_o + lane_at + c, o);
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] *= scale;
                        if (odd) {
                            const unsigned char *v = smem + (v_ring - base) + vs * TILE + (c / 64) * 8192;
                            for (int k = 0; k < 64; ++k) {
                                if (!(see >> k & 1)) continue;
#pragma unroll
                                for (int j = 0; j < 32; j += 2) {
                                    const int ch = (c % 64 + j) / 8;
                                    const float2 y = unpack2<C::BF>(*reinterpret_cast<const uint32_t *>(v + k * 128 + ((ch ^ (k & 7)) << 4) + (j % 8) * 2));
                                    if (!(fabsf(y.x) < INFINITY)) o[j] += y.x;
                                    if (!(fabsf(y.y) < INFINITY)) o[j + 1] += y.y;
                                }
                            }
                        }
                        uint32_t r[32];
#pragma unroll
                        for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(o[j]);
                        tt_st32(tmem_o + lane_at + c, r);
                    }
                    tt_wait_st();
                    if (odd) {
                        tt_any(false);   // every row has added them
                        uint16_t *v = reinterpret_cast<uint16_t *>(smem + (v_ring - base) + vs * TILE);
                        constexpr uint16_t E = C::BF ? 0x7f80u : 0x7c00u;
                        for (int b = row; b < TILE / 2; b += 128)
                            if ((v[b] & E) == E) v[b] = 0;
                        tt_proxy();
                        tt_any(false);
                    }
                }
                const float shift = C::LIFT - (m == -INFINITY ? 0.0f : m);
                uint32_t p[32];
                float sum[2] = {0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    const float y0 = ex2(fmaf(x[2 * j], f, shift)), y1 = ex2(fmaf(x[2 * j + 1], f, shift));
                    sum[0] += y0;
                    sum[1] += y1;
                    p[j] = pack2<C::BF>(y0, y1);
                }
                l += sum[0] + sum[1];
                tt_st32(tmem + lane_at + (n & 1) * 64, p);
                tt_wait_st();
                // The product of the last page is done before this one may
                // begin: a phase of o_done can be waited for by its parity only
                // while it is the last or the next to complete, and S of a page
                // says no more than that the product two pages back is done.
                if (n > 0) ok = tt_wait_warp(o_done, (uint32_t)((n - 1) & 1), stop_word, err) && ok;
                tt_before();
                __syncwarp();
                if (lane == 0) tt_arrive(&p_ready[n & 1]);
            }
            // the tile's O once its last product is done
            if (ok && tt_wait_warp(o_done, (uint32_t)((count + pages - 1) & 1), stop_word, err)) {
                tt_after();
                const bool whole = p_begin == s.page0 && p_end == s.page1;
                const size_t part_at = ((size_t)blockIdx.x * 2 + (p_begin == s.page0)) * TT_ROWS + row;
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const bool real = node < s.t;
                uint16_t *to = static_cast<uint16_t *>(a.out) + (real ? (size_t)(s.r0 + node) * a.ldo + (size_t)(kh * g.group + rr - node * g.group) * HD : 0);
                const bool vec = (a.ldo & 7) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
                float *po = g.part + part_at * HD;
                if (real && !whole) *reinterpret_cast<float2 *>(g.part + (size_t)gridDim.x * 2 * TT_ROWS * HD + part_at * 2) = make_float2(m, l);
#pragma unroll
                for (int c = 0; c < HD; c += 32) {
                    float o[32];
                    tt_ld32(tmem_o + lane_at + c, o);
                    if (!real) continue;
                    if (!whole) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4 *>(po + c + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j += 8) {
                            const uint4 u = make_uint4(pack2<C::BF>(o[j] * inv, o[j + 1] * inv), pack2<C::BF>(o[j + 2] * inv, o[j + 3] * inv),
                                                       pack2<C::BF>(o[j + 4] * inv, o[j + 5] * inv), pack2<C::BF>(o[j + 6] * inv, o[j + 7] * inv));
                            if (vec) {
                                *reinterpret_cast<uint4 *>(to + c + j) = u;
                            } else {
                                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                                for (int e = 0; e < 8; ++e) to[c + j + e] = (uint16_t)(w[e / 2] >> (16 * (e % 2)));
                            }
                        }
                    }
                }
            }
            tt_before();
        }
        count += pages;
        at += pages;
        // Q, O and the line are free for the next tile, or a role gave up
        if (__syncthreads_or(*stop_word)) break;
        tt_after();
    }
    // Loads that nobody waited for (after a wait that gave up) land before the
    // shared memory goes away, bounded; then the columns are freed.
    if (warp == 5 && lane == 0 && *stop_word)
        for (int j = 0; j < KS + VS; ++j) {
            const int n = j < KS ? k_issued - 1 - j : v_issued - 1 - (j - KS);
            for (uint32_t i = 0; n >= 0 && i < (1u << 20); ++i)
                if (j < KS ? ec_mbar_try_wait(&k_full[n % KS], (uint32_t)((n / KS) & 1)) : ec_mbar_try_wait(&v_full[n % VS], (uint32_t)((n / VS) & 1))) break;
        }
    if (warp == 4 && lane == 0) {
        tt_commit(drain);     // every MMA that was issued is complete once this fires
        for (uint32_t i = 0; i < (1u << 24); ++i)
            if (ec_mbar_try_wait(drain, 0)) break;
    }
    tt_before();
    __syncthreads();
    if (warp == 4) {
        __syncwarp();
        tt_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM));
    }
}

PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
pthread_once_t g_once = PTHREAD_ONCE_INIT;
int g_attr[4][64];

void resolve() {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
        g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
}

// A layer's K or V cache as [pages][64][dim], boxes of a page by 64 elements.
int map_of(CUtensorMap *map, const void *p, const ec_kv_pages &kv) {
    const cuuint64_t dims[3] = {(cuuint64_t)kv.dim, (cuuint64_t)PAGE, (cuuint64_t)kv.n_pages};
    const cuuint64_t strides[2] = {(cuuint64_t)kv.ld_pos * 2, (cuuint64_t)kv.ld_page * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)PAGE, 1}, es[3] = {1, 1, 1};
    return g_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void *>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? 0 : (int)cudaErrorInvalidValue;
}

template <int QT, int KT, int HD>
int launch(const ec_kv_pages &kv, const ec_tree_attn &a, const TaGeo &g, int pieces, int id, int *err, cudaStream_t stream) {
    typedef TtCfg<QT, KT, HD> C;
    static_assert(C::SMEM <= 114 * 1024 - 1024, "two CTAs per SM");
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (!g_attr[id][dev]) {
        e = cudaFuncSetAttribute(k_tree_tc<QT, KT, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return (int)e;
        g_attr[id][dev] = 1;
    }
    TtMaps maps;
    memset(&maps, 0, sizeof maps);
    int rc = map_of(&maps.k, kv.k, kv);
    if (!rc) rc = map_of(&maps.v, kv.v, kv);
    if (rc) return rc;
    return (int)ec_launch_k(k_tree_tc<QT, KT, HD>, dim3(pieces), dim3(TT_THREADS), C::SMEM, stream, maps, kv, a, g, err);
}

}  // namespace

bool ec_tree::ta_tc_takes(int q_type, int kv_type, int hd) {
    if (q_type != kv_type || (hd != 64 && hd != 128)) return false;
    pthread_once(&g_once, resolve);
    return g_encode != nullptr;
}

int ec_tree::ta_tc_launch(const ec_kv_pages &kv, const ec_tree_attn &a, const TaGeo &g, int pieces, int *err, cudaStream_t stream) {
    const bool bf = kv.type == EC_T_BF16;
    if (a.head_dim == 64) return bf ? launch<EC_T_BF16, EC_T_BF16, 64>(kv, a, g, pieces, 0, err, stream) : launch<EC_T_F16, EC_T_F16, 64>(kv, a, g, pieces, 1, err, stream);
    return bf ? launch<EC_T_BF16, EC_T_BF16, 128>(kv, a, g, pieces, 2, err, stream) : launch<EC_T_F16, EC_T_F16, 128>(kv, a, g, pieces, 3, err, stream);
}
