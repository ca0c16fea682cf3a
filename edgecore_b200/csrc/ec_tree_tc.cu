// ec_tree_tc.cu -- the tree attention of ec_tree.cu on the 5th-generation
// tensor cores, for tiles of two halves of 128 rows: large drafts, or many
// query heads on a KV head.
//
// A CTA (one per SM) takes its piece of the line of pages, tile by tile.  A
// step is 128 rows against two pages (128 positions); the steps of the two
// halves alternate, so that the products of one run under the exponentials of
// the other.  A tile with rows for one half only gives its even steps to half 0
// and its odd ones to half 1, whose sums are added at the end.
//   warp 9      TMA producer: K and V of two pages, [64 positions][hd] each in
//               columns of 128 bytes with the 128-byte swizzle, into rings
//   warp 8      one thread issues the MMAs: S = Q K^T (128 x 128, both operands
//               K-major in shared memory) of a step, then O += P V of the step
//               before, a page at a time, with P from tensor memory and V as it
//               lies (rows of hd, "MN-major")
//   warps 0-3   half 0, warps 4-7 half 1, a row per thread: S from tensor memory,
//               the positions that the row sees, running maximum and sum, P back
//               over S as 16-bit pairs; O is rescaled in tensor memory only when
//               the maximum has grown by more than 2^8 (the reference of a row is
//               any earlier maximum, and p stays below 2^14)
// Per step: 128 x 128 exponentials, 1024 cycles of an SM's special function
// units, and 2 x 128 x 128 x hd products, 700 (hd 64) to 1400 (hd 128) cycles at
// the rate that cuBLAS reaches.  Two CTAs per SM of 128 rows each, which nothing
// kept out of step, took 3400 cycles a page instead.  Every wait is bounded;
// loads use no multicast.
// Measured: 16 trees of 48 to 64 nodes at 6000 to 10000 positions, 12 heads of
// 128 on 2 (43.7 GFLOP), 99 us or 440 TFLOP/s, join included; the register
// tiles of ec_tree.cu take 192.  A round of two steps takes 2.3 to 2.9 us where its exponentials and
// products need 1.5: the rows' own instructions (scale, mask, maximum, pack)
// are the longest link, with 282 bytes of a row's 128 scores spilled at 168
// registers (ten warps put three on one scheduler); the tensor cores are busy in
// 34 % of the cycles.  The join and its launch are 20 us, the ends of two tiles
// in a piece 10.
#include "ec_tree.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>
#include <pthread.h>
#include <string.h>

namespace {

constexpr int TT_THREADS = 320, TT_ROWS = 128;
constexpr float TT_GROWTH = 8.0f;                      // log2 growth of a maximum that is let be

template <int QT, int KT, int HD> struct TtCfg {
    static constexpr bool BF = KT == EC_T_BF16;
    static constexpr int COLS = HD / 64;               // 128-byte columns of a row
    static constexpr int TILE = 64 * HD * 2;           // K or V of a page
    static constexpr int ROUND = 2 * TILE;             // two pages of K or V: [column][page][64][128 bytes]
    static constexpr int KS = HD == 64 ? 5 : 2, VS = HD == 64 ? 5 : 3;   // in flight; K is free once its S are done
    static constexpr int Q_BYTES = TT_ROWS * HD * 2;   // of one half
    static constexpr int SMEM = 2 * Q_BYTES + (KS + VS) * ROUND + 2048;
    static constexpr int TMEM = 512;                   // S of the halves at 0 and 128, O at 256 and 384
    static constexpr float LIFT = BF ? 0.0f : 6.0f;
    static constexpr uint32_t TYPES = (1u << 4) | ((BF ? 1u : 0u) << 7) | ((BF ? 1u : 0u) << 10) | ((uint32_t)(TT_ROWS >> 4) << 24);
    static constexpr uint32_t IDESC_S = TYPES | ((64u >> 3) << 17), IDESC_S2 = TYPES | ((128u >> 3) << 17);   // one page, two
    static constexpr uint32_t IDESC_O = TYPES | (1u << 16) | ((uint32_t)(HD >> 3) << 17);   // B is MN-major
};

// Shared-memory descriptors, 128-byte swizzle: start, leading and stride byte
// offsets (>> 4), version 1, mode 2.  K-major: 8-row groups 1024 bytes apart.
// MN-major: 8-row (K) groups 1024 bytes apart, 64-element columns `lead` apart.
EC_DEV uint64_t tt_desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// The MMA warp runs as one: every lane computes the operands, which then stay
// in uniform registers, and an elected lane issues.  (From a branch of one lane
// each product took 110 cycles to issue, twice what it takes to run.)
EC_DEV void tt_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t more) {
    asm volatile("{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(more), "r"(0u));
}
EC_DEV void tt_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t more) {
    asm volatile("{\n\t.reg .pred p, q;\n\telect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(more), "r"(0u));
}
EC_DEV void tt_commit(uint32_t bar) {
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar) : "memory");
}
EC_DEV void tt_arrive(uint64_t *bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(ec_smem_u32(bar)) : "memory"); }
EC_DEV void tt_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
EC_DEV void tt_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
EC_DEV void tt_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
EC_DEV void tt_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 128 or 32 columns of this thread's row, arrived (the wait is part of the
// statement: nothing may use the registers before it)
EC_DEV void tt_ld128(uint32_t taddr, float *f) {
    __syncwarp();   // a whole warp executes these as one
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
                 "%30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, "
                 "%58, %59, %60, %61, %62, %63}, [%128];\n\t"
                 "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%64, %65, %66, %67, %68, %69, %70, %71, %72, %73, %74, %75, %76, %77, %78, %79, %80, %81, %82, %83, %84, %85, %86, %87, %88, %89, %90, %91, "
                 "%92, %93, %94, %95, %96, %97, %98, %99, %100, %101, %102, %103, %104, %105, %106, %107, %108, %109, %110, %111, %112, %113, %114, %115, %116, "
                 "%117, %118, %119, %120, %121, %122, %123, %124, %125, %126, %127}, [%129];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]), "=f"(f[8]), "=f"(f[9]), "=f"(f[10]),
                   "=f"(f[11]), "=f"(f[12]), "=f"(f[13]), "=f"(f[14]), "=f"(f[15]), "=f"(f[16]), "=f"(f[17]), "=f"(f[18]), "=f"(f[19]), "=f"(f[20]),
                   "=f"(f[21]), "=f"(f[22]), "=f"(f[23]), "=f"(f[24]), "=f"(f[25]), "=f"(f[26]), "=f"(f[27]), "=f"(f[28]), "=f"(f[29]), "=f"(f[30]),
                   "=f"(f[31]), "=f"(f[32]), "=f"(f[33]), "=f"(f[34]), "=f"(f[35]), "=f"(f[36]), "=f"(f[37]), "=f"(f[38]), "=f"(f[39]), "=f"(f[40]),
                   "=f"(f[41]), "=f"(f[42]), "=f"(f[43]), "=f"(f[44]), "=f"(f[45]), "=f"(f[46]), "=f"(f[47]), "=f"(f[48]), "=f"(f[49]), "=f"(f[50]),
                   "=f"(f[51]), "=f"(f[52]), "=f"(f[53]), "=f"(f[54]), "=f"(f[55]), "=f"(f[56]), "=f"(f[57]), "=f"(f[58]), "=f"(f[59]), "=f"(f[60]),
                   "=f"(f[61]), "=f"(f[62]), "=f"(f[63]), "=f"(f[64]), "=f"(f[65]), "=f"(f[66]), "=f"(f[67]), "=f"(f[68]), "=f"(f[69]), "=f"(f[70]),
                   "=f"(f[71]), "=f"(f[72]), "=f"(f[73]), "=f"(f[74]), "=f"(f[75]), "=f"(f[76]), "=f"(f[77]), "=f"(f[78]), "=f"(f[79]), "=f"(f[80]),
                   "=f"(f[81]), "=f"(f[82]), "=f"(f[83]), "=f"(f[84]), "=f"(f[85]), "=f"(f[86]), "=f"(f[87]), "=f"(f[88]), "=f"(f[89]), "=f"(f[90]),
                   "=f"(f[91]), "=f"(f[92]), "=f"(f[93]), "=f"(f[94]), "=f"(f[95]), "=f"(f[96]), "=f"(f[97]), "=f"(f[98]), "=f"(f[99]), "=f"(f[100]),
                   "=f"(f[101]), "=f"(f[102]), "=f"(f[103]), "=f"(f[104]), "=f"(f[105]), "=f"(f[106]), "=f"(f[107]), "=f"(f[108]), "=f"(f[109]), "=f"(f[110]),
                   "=f"(f[111]), "=f"(f[112]), "=f"(f[113]), "=f"(f[114]), "=f"(f[115]), "=f"(f[116]), "=f"(f[117]), "=f"(f[118]), "=f"(f[119]), "=f"(f[120]),
                   "=f"(f[121]), "=f"(f[122]), "=f"(f[123]), "=f"(f[124]), "=f"(f[125]), "=f"(f[126]), "=f"(f[127])
                 : "r"(taddr), "r"(taddr + 64) : "memory");
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

// two fp32 at a time
EC_DEV float2 tt_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
EC_DEV float2 tt_add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
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

// The same for a whole warp, which goes on together.
EC_DEV bool tt_wait_warp(uint64_t *bar, uint32_t parity, volatile int *stop, int *err) {
    if (__all_sync(0xffffffffu, ec_mbar_try_wait(bar, parity))) return true;
    int ok = 0;
    if ((threadIdx.x & 31) == 0) ok = tt_wait(bar, parity, stop, err);
    ok = __shfl_sync(0xffffffffu, ok, 0);
    // every lane sees the phase complete for itself: what it guards is visible to it
    return ok && __all_sync(0xffffffffu, ec_mbar_try_wait(bar, parity));
}

// OR over the row warps that share V: all 256 threads, or the 128 of one half.
// A warp whose wait gave up goes on to take part in every one of these, so that
// no other waits for it.
EC_DEV bool tt_any(bool v, int bar, int threads) {
    int r;
    __syncwarp();
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %1, 0;\n\tbar.red.or.pred p, %2, %3, p;\n\tselp.s32 %0, 1, 0, p;\n\t}"
                 : "=r"(r) : "r"((int)v), "r"(bar), "r"(threads) : "memory");
    return r != 0;
}

// O of this thread's row plus the infinities and NaN of the positions of a
// round that it sees (a page's mask each).  Out of line: hardly ever called.
template <bool BF> __noinline__ __device__ void tt_add_odd(uint32_t tmem_o, int hd, const unsigned char *v, unsigned long long see0, unsigned long long see1) {
#pragma unroll 1
    for (int c = 0; c < hd; c += 32) {
        float o[32];
        tt_ld32(tmem_o + c, o);
#pragma unroll 1
        for (int k = 0; k < 128; ++k) {
            if (!((k < 64 ? see0 : see1) >> (k & 63) & 1)) continue;
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
                const int ch = (c % 64 + j) / 8;
                const float2 y = unpack2<BF>(*reinterpret_cast<const uint32_t *>(v + (c / 64) * 16384 + k * 128 + ((ch ^ (k & 7)) << 4) + (j % 8) * 2));
                if (!(fabsf(y.x) < INFINITY)) o[j] += y.x;
                if (!(fabsf(y.y) < INFINITY)) o[j + 1] += y.y;
            }
        }
        tt_st32(tmem_o + c, reinterpret_cast<const uint32_t *>(o));
    }
    tt_wait_st();
}

struct TtMaps { CUtensorMap k, v; };

template <int QT, int KT, int HD>
__global__ void __launch_bounds__(TT_THREADS, 1)
k_tree_tc(const __grid_constant__ TtMaps maps, const ec_kv_pages kv, const ec_tree_attn a, const TaGeo g, int *err) {
    typedef TtCfg<QT, KT, HD> C;
    constexpr int KS = C::KS, VS = C::VS, ROUND = C::ROUND;
    extern __shared__ __align__(1024) unsigned char smem[];
    const uint32_t base = ec_smem_u32(smem);              // 1024-byte aligned: the kernel has no other shared memory
    const uint32_t k_ring = base + 2 * C::Q_BYTES, v_ring = k_ring + KS * ROUND;
    float2 *other = reinterpret_cast<float2 *>(smem + 2 * C::Q_BYTES + (KS + VS) * ROUND);   // (m, l) of half 1, [128]
    uint64_t *k_full = reinterpret_cast<uint64_t *>(other + TT_ROWS), *k_empty = k_full + KS;
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
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ec_smem_u32(tmem_slot)), "r"(C::TMEM));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tt_before();
    __syncthreads();
    tt_after();
    const uint32_t tmem = *tmem_slot;
    EC_PDL_ENTER();

    TaLine line;
    line.init(kv, a, g, TC_ROWS, gridDim.x, err);
    int at = (int)blockIdx.x < line.n ? line.start(blockIdx.x) : 0;
    const int stop_at = (int)blockIdx.x < line.n ? line.start(blockIdx.x + 1) : 0;
    int count = 0, tiles = 0;         // loads of K (and of V) and tiles of this CTA so far
    int steps_of[2] = {0, 0};         // steps of each half so far
    int k_issued = 0, v_issued = 0;   // producer: loads issued
    int k_at = 0, v_at = 0;           // MMA warp: stages of the rings, and the phases to wait for
    uint32_t k_phase = 0, v_phase = 0, p_phase = 0;
    while (at < stop_at) {
        int begin;
        const TaTile s = line.tile(kv, a, g, TC_ROWS, at, begin, err);
        const int places = min(begin + s.len, stop_at) - at;
        const int p_begin = s.page0 + (at - begin) * s.step, p_end = min(s.page1, p_begin + places * s.step), pages = p_end - p_begin, rounds = (pages + 1) / 2;
        const int kh = s.kh, end = s.base + s.t;
        const bool split = s.step == 2;   // one half's rows, the rounds shared out over both
        const int steps = split ? rounds : 2 * rounds;

        // The producer: what the rings hold before the row warps are met below
        // (they are empty: the last tile is done), the rest after.
        auto produce = [&](int i0, int i1) {
            for (int i = i0; i < i1; ++i) {
                const int n = count + i, ks = n % KS, vs = n % VS, two = 2 * i + 1 < pages;
                const int pg[2] = {ta_page(kv, s.slot, p_begin + 2 * i, err), two ? ta_page(kv, s.slot, p_begin + 2 * i + 1, err) : 0};
                auto load = [&](uint32_t to, const CUtensorMap *map, uint64_t *bar) {
                    ec_mbar_expect_tx(bar, (1 + two) * C::TILE);
                    for (int h = 0; h <= two; ++h)
#pragma unroll
                        for (int c = 0; c < C::COLS; ++c) tt_load(to + c * 16384 + h * 8192, map, bar, kh * HD + c * 64, pg[h]);
                };
                if (n >= KS && !tt_wait(&k_empty[ks], (uint32_t)((n / KS - 1) & 1), stop_word, err)) break;
                load(k_ring + ks * ROUND, &maps.k, &k_full[ks]);
                k_issued = n + 1;
                if (n >= VS && !tt_wait(&v_empty[vs], (uint32_t)((n / VS - 1) & 1), stop_word, err)) break;
                load(v_ring + vs * ROUND, &maps.v, &v_full[vs]);
                v_issued = n + 1;
            }
        };
        constexpr int AHEAD = KS < VS ? KS : VS;
        if (warp == 9) {
            if (lane == 0) produce(0, min(rounds, AHEAD));
        } else if (warp < 8) {
            // the queries, all in flight at once; rows behind the sequence are zero
            const bool wide = (a.ldq & 7) == 0 && (reinterpret_cast<uintptr_t>(a.q) & 15) == 0;
            constexpr int CH = HD / 8, AT_ONCE = 256 / CH;   // 16-byte chunks of a row, rows at a time
            const int c = threadIdx.x % CH;
#pragma unroll 4
            for (int r = threadIdx.x / CH; r < (split ? 1 : 2) * TT_ROWS; r += AT_ONCE) {
                const int rr = s.first + r, node = ta_node(g, rr);
                const bool real = node < s.t;
                const uint16_t *q = static_cast<const uint16_t *>(a.q) + (real ? (size_t)(s.r0 + node) * a.ldq + (size_t)(kh * g.group + rr - node * g.group) * HD + c * 8 : 0);
                const uint32_t to = (r / TT_ROWS) * C::Q_BYTES + (c / 8) * (TT_ROWS * 128) + (r % TT_ROWS) * 128 + (((c % 8) ^ (r & 7)) << 4);
                if (wide) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(base + to), "l"(q), "r"(real ? 16 : 0) : "memory");
                } else {
                    uint4 u = make_uint4(0u, 0u, 0u, 0u);
                    if (real) u = make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16, q[6] | (uint32_t)q[7] << 16);
                    *reinterpret_cast<uint4 *>(smem + to) = u;
                }
            }
            // O starts from zero
            uint32_t zero[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) zero[i] = 0u;
#pragma unroll 1
            for (int i = 0; i < HD; i += 32) tt_st32(tmem + 256 + (warp / 4) * 128 + ((uint32_t)((warp & 3) * 32) << 16) + i, zero);
            tt_wait_st();
            asm volatile("cp.async.wait_all;" ::: "memory");
            tt_proxy();
            tt_before();
        }
        __syncthreads();
        tt_after();

        if (warp == 9) {
            if (lane == 0) produce(min(rounds, AHEAD), rounds);
        } else if (warp == 8) {
            const int all = __shfl_sync(0xffffffffu, steps, 0), pages_u = __shfl_sync(0xffffffffu, pages, 0);
            const bool split_u = __shfl_sync(0xffffffffu, split, 0);
            int i_s = 0, i_o = 0;   // rounds of the next S and of the next product with V
            for (int t = 0; t <= all; ++t) {
                if (t < all) {   // S of step t, over the P of the half's last step, which its products have read
                    const int half = t & 1;
                    if ((split_u || !half) && !tt_wait_warp(&k_full[k_at], k_phase, stop_word, err)) break;
                    tt_after();
                    const uint64_t dq = tt_desc(base + (split_u ? 0 : half * C::Q_BYTES), 16), dk = tt_desc(k_ring + k_at * ROUND, 16);
                    const uint32_t idesc = 2 * i_s + 1 < pages_u ? C::IDESC_S2 : C::IDESC_S;
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k)
                        tt_mma_ss(tmem + half * 128, dq + (k / 4) * (TT_ROWS * 128 >> 4) + (k % 4) * 2, dk + (k / 4) * (16384 >> 4) + (k % 4) * 2, idesc, k > 0);
                    tt_commit(ec_smem_u32(&s_full[half]));
                    if (split_u || half) {
                        tt_commit(ec_smem_u32(&k_empty[k_at]));
                        if (++k_at == KS) { k_at = 0; k_phase ^= 1; }
                        ++i_s;
                    }
                }
                if (t > 0) {       // P V of step t - 1
                    const int half = (t - 1) & 1;
                    const bool two = 2 * i_o + 1 < pages_u;
                    const uint64_t dv = tt_desc(v_ring + v_at * ROUND, 16384);
                    const uint32_t d = tmem + 256 + half * 128, pt = tmem + half * 128;
                    if ((split_u || !half) && !tt_wait_warp(&v_full[v_at], v_phase, stop_word, err)) break;
                    if (!tt_wait_warp(&p_ready[half], p_phase >> half & 1, stop_word, err)) break;
                    p_phase ^= 1u << half;
                    tt_after();
#pragma unroll
                    for (int k = 0; k < 4; ++k) tt_mma_ts(d, pt + k * 8, dv + k * (2048 >> 4), C::IDESC_O, 1);
                    if (two)
#pragma unroll
                        for (int k = 0; k < 4; ++k) tt_mma_ts(d, pt + 32 + k * 8, dv + (8192 >> 4) + k * (2048 >> 4), C::IDESC_O, 1);
                    if (split_u || half) {
                        tt_commit(ec_smem_u32(&v_empty[v_at]));
                        if (++v_at == VS) { v_at = 0; v_phase ^= 1; }
                        ++i_o;
                    }
                }
            }
            tt_commit(ec_smem_u32(o_done));
        } else {
            const int half = warp / 4, row = threadIdx.x & 127, rr = s.first + (split ? 0 : half * TT_ROWS) + row, node = ta_node(g, rr);
            const uint32_t lane_at = (uint32_t)((warp & 3) * 32) << 16, tmem_s = tmem + half * 128 + lane_at, tmem_o = tmem + 256 + half * 128 + lane_at;
            const int bar = split ? 1 + half : 1, voters = split ? 128 : 256;   // who shares a round's V
            const float f = g.scale2;
            float m = -INFINITY, l = 0.0f;
            bool ok = true;
            int step = steps_of[half];
            for (int i = split ? half : 0; i < rounds; i += split ? 2 : 1, ++step) {
                const int n = count + i, vs = n % VS, two = 2 * i + 1 < pages, p0 = (p_begin + 2 * i) * PAGE;
                const bool part = !two || p0 + 2 * PAGE > s.base || (a.window > 0 && p0 < (long long)s.base + 64 * a.mask_words - a.window);
                ok = ok && tt_wait_warp(&s_full[half], (uint32_t)(step & 1), stop_word, err);
                if (!ok) {
                    if (part && tt_any(false, bar, voters)) {
                        tt_any(false, bar, voters);
                        tt_any(false, bar, voters);
                    }
                    continue;
                }
                tt_after();
                // S is done, and with it every product of this half before it: O may be changed
                float x[128];
                tt_ld128(tmem_s, x);
                unsigned long long see[2] = {~0ull, ~0ull};
                if (part) {
                    see[0] = ta_allow(a, s, node, p0);
                    see[1] = two ? ta_allow(a, s, node, p0 + PAGE) : 0ull;
                    const uint32_t w[4] = {(uint32_t)see[0], (uint32_t)(see[0] >> 32), (uint32_t)see[1], (uint32_t)(see[1] >> 32)};
#pragma unroll
                    for (int j = 0; j < 128; ++j)
                        if (!(w[j / 32] >> (j % 32) & 1u)) x[j] = -INFINITY;
                }
                float hi[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) hi[e] = fmaxf(x[e], x[8 + e]);
#pragma unroll
                for (int j = 16; j < 128; j += 16)
#pragma unroll
                    for (int e = 0; e < 8; ++e) hi[e] = fmaxf(fmaxf(hi[e], x[j + e]), x[j + 8 + e]);
                const float top = fmaxf(fmaxf(fmaxf(hi[0], hi[1]), fmaxf(hi[2], hi[3])), fmaxf(fmaxf(hi[4], hi[5]), fmaxf(hi[6], hi[7]))) * f;
                const bool grow = top > m + TT_GROWTH || (m == -INFINITY && top > m);
                float scale = 1.0f;
                if (grow) {
                    scale = ex2(m - top);   // 0 at first
                    m = top;
                    l *= scale;
                }
                unsigned char *v = smem + (v_ring - base) + vs * ROUND;   // position k of the round: page k / 64, row k % 64 of each column
                auto v_row = [&](int c, int k) { return v + c * 16384 + k * 128; };
                constexpr uint32_t E = C::BF ? 0x7f80u : 0x7c00u;
                bool odd = false;
                const bool keeper = split || half == 0;   // changes V where it has to be
                if (part) {
                    // V of positions that are not there is zero, and infinities
                    // and NaN (0 times them is NaN) are taken out and added by
                    // the rows that see them.  The halves that share a round
                    // meet here; the first product of the round comes after.
                    ok = tt_wait_warp(&v_full[vs], (uint32_t)((n / VS) & 1), stop_word, err);
                    const int k = row;   // a position of the round per thread
                    if (keeper && k < (1 + two) * 64)
                        for (int c = 0; c < C::COLS; ++c)
                            for (int b = 0; b < 8; ++b) {
                                uint4 *u = reinterpret_cast<uint4 *>(v_row(c, k) + ((b + k) % 8) * 16);
                                if (p0 + k >= end) {
                                    *u = make_uint4(0u, 0u, 0u, 0u);
                                } else {
                                    const uint4 w = *u;
                                    const uint32_t w4[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                                    for (int j = 0; j < 4; ++j) odd |= (w4[j] & E) == E || (w4[j] >> 16 & E) == E;
                                }
                            }
                    tt_proxy();
                    odd = tt_any(odd, bar, voters);
                }
                if (__any_sync(0xffffffffu, grow)) {
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        float o[32];
                        tt_ld32(tmem_o + c, o);
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] *= scale;
                        tt_st32(tmem_o + c, reinterpret_cast<const uint32_t *>(o));
                    }
                    tt_wait_st();
                }
                if (odd) {
                    tt_add_odd<C::BF>(tmem_o, HD, v, see[0], see[1]);
                    tt_any(false, bar, voters);   // every row has added them
                    const int k = row;
                    if (keeper && k < (1 + two) * 64)
                        for (int c = 0; c < C::COLS; ++c)
                            for (int b = 0; b < 64; ++b) {
                                uint16_t *u = reinterpret_cast<uint16_t *>(v_row(c, k)) + b;
                                if ((*u & E) == E) *u = 0;
                            }
                    tt_proxy();
                    tt_any(false, bar, voters);
                }
                const float shift = C::LIFT - (m == -INFINITY ? 0.0f : m);
                const float2 f2 = make_float2(f, f), shift2 = make_float2(shift, shift);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h && !two) break;
                    uint32_t p[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        float2 y = tt_fma2(make_float2(x[h * 64 + 2 * j], x[h * 64 + 2 * j + 1]), f2, shift2);
                        y = make_float2(ex2(y.x), ex2(y.y));
                        sum[j & 1] = tt_add2(sum[j & 1], y);
                        p[j] = pack2<C::BF>(y.x, y.y);
                    }
                    tt_st32(tmem_s + h * 32, p);
                }
                tt_wait_st();
                tt_before();
                __syncwarp();
                if (lane == 0) tt_arrive(&p_ready[half]);
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            }
            // the tile's O once its last product is done
            ok = ok && tt_wait_warp(o_done, (uint32_t)(tiles & 1), stop_word, err);
            tt_after();
            float mine = 1.0f, theirs = 0.0f;   // weights of the halves' sums
            if (split) {
                if (half == 1) other[row] = make_float2(m, l);
                tt_any(false, 3, 256);
                if (half == 0) {
                    const float2 o = other[row];
                    const float top = fmaxf(m, o.x), u = top == -INFINITY ? 0.0f : top;
                    mine = ex2(m - u);
                    theirs = ex2(o.x - u);
                    m = top;
                    l = l * mine + o.y * theirs;
                }
            }
            // O as rows of shared memory (Q, K and V are done with), from where
            // a warp writes a row at a time; a row is 16 bytes longer than hd
            // floats, so that eight of them fall into different banks.
            constexpr int LD = HD + 4;
            static_assert(2 * TT_ROWS * LD * 4 <= 2 * C::Q_BYTES + (KS + VS) * ROUND, "staging of O");
            float *stage = reinterpret_cast<float *>(smem) + (size_t)half * TT_ROWS * LD;
            const bool whole = p_begin == s.page0 && p_end == s.page1, active = ok && (!split || half == 0);
            if (active) {
                const float inv = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
                mine *= inv;
                theirs *= inv;
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    float o[32];
                    tt_ld32(tmem_o + c, o);
                    if (split) {
                        float y[32];
                        tt_ld32(tmem_o + 128 + c, y);
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = o[j] * mine + y[j] * theirs;
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] *= mine;
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4 *>(stage + row * LD + c + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                }
                const size_t part_at = ((size_t)blockIdx.x * 2 + (p_begin == s.page0)) * TC_ROWS + half * TT_ROWS;
                if (!whole && node < s.t) *reinterpret_cast<float2 *>(g.part + (size_t)gridDim.x * 2 * TC_ROWS * HD + (part_at + row) * 2) = make_float2(m, l);
                __syncwarp();
                const int r0 = (warp & 3) * 32;   // the warp's own rows
                if (!whole) {
                    constexpr int LANES = HD / 4, ROWS = 32 / LANES;   // lanes of a row, rows at a time
#pragma unroll 4
                    for (int i = 0; i < 32; i += ROWS) {
                        const int r = r0 + i + lane / LANES, d = lane % LANES * 4;
                        *reinterpret_cast<float4 *>(g.part + (part_at + r) * HD + d) = *reinterpret_cast<const float4 *>(stage + r * LD + d);
                    }
                } else {
                    constexpr int LANES = HD / 4, ROWS = 32 / LANES;
                    const bool vec = (a.ldo & 3) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 7) == 0;
#pragma unroll 4
                    for (int i = 0; i < 32; i += ROWS) {
                        const int r = r0 + i + lane / LANES, d = lane % LANES * 4, to_rr = s.first + (split ? 0 : half * TT_ROWS) + r, to_node = ta_node(g, to_rr);
                        if (to_node >= s.t) continue;
                        const float4 o = *reinterpret_cast<const float4 *>(stage + r * LD + d);
                        uint16_t *to = static_cast<uint16_t *>(a.out) + (size_t)(s.r0 + to_node) * a.ldo + (size_t)(kh * g.group + to_rr - to_node * g.group) * HD + d;
                        const uint2 u = make_uint2(pack2<C::BF>(o.x, o.y), pack2<C::BF>(o.z, o.w));
                        if (vec) {
                            *reinterpret_cast<uint2 *>(to) = u;
                        } else {
                            to[0] = (uint16_t)u.x;
                            to[1] = (uint16_t)(u.x >> 16);
                            to[2] = (uint16_t)u.y;
                            to[3] = (uint16_t)(u.y >> 16);
                        }
                    }
                }
            }
            tt_proxy();   // before the next tile's loads into the same memory
            tt_before();
        }
        count += rounds;
        steps_of[0] += split ? (steps + 1) / 2 : rounds;
        steps_of[1] += split ? steps / 2 : rounds;
        ++tiles;
        at += places;
        // Q, O and the rings are free for the next tile, or a role gave up
        if (__syncthreads_or(*stop_word)) break;
        tt_after();
    }
    // Loads that nobody waited for (after a wait that gave up) land before the
    // shared memory goes away, bounded; then the columns are freed.
    if (warp == 9 && lane == 0 && *stop_word)
        for (int j = 0; j < KS + VS; ++j) {
            const int n = j < KS ? k_issued - 1 - j : v_issued - 1 - (j - KS);
            for (uint32_t i = 0; n >= 0 && i < (1u << 20); ++i)
                if (j < KS ? ec_mbar_try_wait(&k_full[n % KS], (uint32_t)((n / KS) & 1)) : ec_mbar_try_wait(&v_full[n % VS], (uint32_t)((n / VS) & 1))) break;
        }
    if (warp == 8) {
        tt_commit(ec_smem_u32(drain));   // every MMA that was issued is complete once this fires
        for (uint32_t i = 0; i < (1u << 24); ++i)
            if (ec_mbar_try_wait(drain, 0)) break;
    }
    tt_before();
    __syncthreads();
    if (warp == 8) {
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
    static_assert(C::SMEM <= 232448, "shared memory per CTA");
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
