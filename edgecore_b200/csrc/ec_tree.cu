// ec_tree.cu -- attention of drafted-token trees over a paged KV arena
// (ec_tree_attention).
//
// The rows of one KV head and sequence -- its T nodes times the G query heads
// that read the KV head -- share every K and V row, so they are one tile: row
// r is node r / G, query head r % G.  A page of 64 positions is one key tile.
// One pass over the pages with a running maximum m and sum l per row:
//   s = scale * q.k (masked: -inf), m' = max(m, s), p = 2^((s - m') log2 e),
//   l = l 2^((m - m') log2 e) + sum p,  o = o 2^((m - m') log2 e) + p V
// and out = o / l (0 where nothing was seen).  The pages are the work: short
// contexts give every row tile to the CTAs of a cluster, which join their (m,
// l, o) through each other's shared memory; longer ones cut the pages of all
// tiles, one after the other, into equal pieces, one per resident CTA, so that
// ragged sequences keep every SM busy to the end, and k_tree_join adds up the
// tiles that a border cuts, in the order of their pages.
// Measured: one token of one stream, 7 us; a tree of 9 nodes at 30011 positions,
// 12 heads of 128 on 2 (31 MB, 1.7 GFLOP), 26 us or 1.2 TB/s, 7 us of it the
// second launch with its wait for the first; 32 sequences of 1
// to 17 nodes with fp32 q at 65 to 1900 positions 35 us; 24 windowed ones 20 us
// or 1.6 TB/s.  All are bound by latency, not by a pipe or by memory: a CTA of
// the long and of the fp32 call has three to five pages, an SM is busy for 64 %
// of the first kernel's cycles (its chain of lengths, page table, queries and
// first pages, gone through again at every change of tile, is the rest), and
// while it is, its schedulers issue in a third of the cycles, the tensor cores
// run in a quarter to a third and DRAM gives 8 to 17 % of its rate.
#include "ec_tree.cuh"

#include <cooperative_groups.h>
#include <limits.h>

namespace cg = cooperative_groups;

namespace {

// ---- register tiles ------------------------------------------------------------

EC_DEV void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
EC_DEV void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool BF> EC_DEV void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
EC_DEV void cp16(uint32_t dst, const void *src, bool real) {   // 16 bytes, or zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
EC_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> EC_DEV void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Byte address of 16-byte chunk c of row r in a tile of rows of HDP 16-bit
// elements: chunks are exchanged within groups of eight so that the eight
// rows of an ldmatrix fall into different banks.
template <int HDP> EC_DEV uint32_t ta_at(int r, int c) { return (uint32_t)(r * HDP * 2 + ((c ^ (r & 7)) << 4)); }

// fp32 queries are written as NP 16-bit parts whose sum is the row times a
// power of two (fp16: two parts, 2^-22 of the largest element, scaled so that
// it lies in [2^13, 2^14); bf16: three parts, 2^-26), and so are the weights
// p for the product with V.  Every part is one more product with the same
// tile.  16-bit queries are taken as they are and p is rounded to the cache's
// type, half a step of 2^-11 or 2^-8 of each p: the product with V has no
// wider operand, and the roundings of a row's weights are independent.  fp16
// p carry 2^14 (in o and l alike), so that the smallest keep their bits.
template <int QT, int KT> struct TaType {
    static constexpr bool BF = KT == EC_T_BF16, F32 = QT == EC_T_F32;
    static constexpr int NP = !F32 ? 1 : BF ? 3 : 2;
    // fp32 q: p itself is exact to its last bit, and 2^14 multiplies its parts;
    // 16-bit q: 14 is added to the exponent
    static constexpr float LIFT = BF || F32 ? 0.0f : 14.0f, PARTS = F32 && !BF ? 16384.0f : 1.0f;
};

// WM x WN warps: WM groups of 16 rows, the 64 positions of a page shared out
// over WN warps (few rows: more warps for the page, each with its own running
// maximum, joined at the end).
template <int QT, int KT, int HDP, int WM, int WN, int STAGES> struct TaMma {
    typedef TaType<QT, KT> Ty;
    static constexpr int THREADS = 32 * WM * WN, MT = 16 * WM, KN = PAGE / WN, NP = Ty::NP;
    static constexpr int TILE = PAGE * HDP * 2;                 // bytes of a K or V tile
    static constexpr int Q_BYTES = NP * MT * HDP * 2;
    static constexpr int RING = STAGES * 2 * TILE;
    static constexpr int JOIN = WN * MT * (HDP + 2) * 4;       // overlays the ring
    static constexpr int SMEM = Q_BYTES + (RING > JOIN ? RING : JOIN) + MT * 4 + 128;
};

// Bounded by the bytes of K and V for few rows, and there by how many of them
// are in flight: STAGES pages of K and V per CTA and two or three CTAs per SM
// (hd 64: 16 KB a stage, hd 128: 32 KB).
// PIECES: a CTA takes its piece of the line of pages, else (grid: tiles,
// cluster, KV heads) its share of one tile.
template <int QT, int KT, int HDP, int WM, int WN, int STAGES, bool PIECES>
__global__ void __launch_bounds__(32 * WM * WN, HDP == 64 && QT != EC_T_F32 ? 3 : HDP <= 128 ? 2 : 1) k_tree_mma(const ec_kv_pages kv, const ec_tree_attn a, const TaGeo g, int *err) {
    EC_PDL_ENTER();
    typedef TaMma<QT, KT, HDP, WM, WN, STAGES> C;
    typedef typename C::Ty Ty;
    constexpr bool BF = Ty::BF;
    constexpr int NP = C::NP, KN = C::KN, NK = KN / 8, ND = HDP / 8;
    extern __shared__ __align__(1024) unsigned char smem[];
    const uint32_t sq = ec_smem_u32(smem), ring = sq + C::Q_BYTES;
    float *row_scale = reinterpret_cast<float *>(smem + C::SMEM - 128 - C::MT * 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wm = warp % WM, wn = warp / WM;
    const int hd = a.head_dim;
    TaTile s;
    int p_begin, p_end;
    int at = 0, stop = 0, tile_begin = 0;   // PIECES: places on the line
    TaLine line;
    if constexpr (PIECES) {
        line.init(kv, a, g, C::MT, gridDim.x, err);
        if ((int)blockIdx.x >= line.n) return;
        at = line.start(blockIdx.x);
        stop = line.start(blockIdx.x + 1);
    } else {
        if (!ta_find(kv, a, g, blockIdx.x, blockIdx.z, C::MT, s, err)) return;   // all CTAs of the cluster alike
        const int chunk = (s.page1 - s.page0 + g.cluster - 1) / g.cluster;
        p_begin = min(s.page1, s.page0 + (int)blockIdx.y * chunk);
        p_end = min(s.page1, p_begin + chunk);
    }
    do {
    if constexpr (PIECES) {
        if (at >= stop) return;
        s = line.tile(kv, a, g, C::MT, at, tile_begin, err);
        p_begin = s.page0 + (at - tile_begin);
        p_end = min(s.page1, p_begin + (stop - at));
    }
    const int kh = s.kh, end = s.base + s.t;

    // the numbers of the first pages, the queries, then the pages themselves
    int pg[STAGES];
#pragma unroll
    for (int i = 0; i < STAGES; ++i) pg[i] = p_begin + i < p_end ? ta_page(kv, s.slot, p_begin + i, err) : 0;
    const bool wide = Ty::F32 ? (a.ldq & 3) == 0 && (reinterpret_cast<uintptr_t>(a.q) & 15) == 0
                              : (a.ldq & 7) == 0 && (reinterpret_cast<uintptr_t>(a.q) & 15) == 0;   // 16-byte reads of q
    auto q_at = [&](int r, bool &real) {   // offset in q of the tile's row r; rows behind the sequence are zero
        const int rr = s.first + r, node = ta_node(g, rr);
        real = node < s.t;
        return real ? (size_t)(s.r0 + node) * a.ldq + (size_t)(kh * g.group + rr - node * g.group) * hd : 0;
    };
    auto fetch = [&](int page, int stage, int pg) {   // page: index in the slot; pg: in the arena
        const uint32_t dk = ring + stage * 2 * C::TILE, dv = dk + C::TILE;
        const size_t off = (size_t)pg * kv.ld_page + (size_t)kh * hd;
        const uint16_t *k = static_cast<const uint16_t *>(kv.k) + off, *v = static_cast<const uint16_t *>(kv.v) + off;
        constexpr int CH = HDP / 8;   // 16-byte chunks of a row
#pragma unroll 4
        for (int i = threadIdx.x; i < PAGE * CH; i += C::THREADS) {
            const int r = i / CH, c = i % CH;
            const bool real = c * 8 < hd && page * PAGE + r < end;   // what is not there reads as 0
            const size_t at = real ? (size_t)r * kv.ld_pos + c * 8 : 0;
            cp16(dk + ta_at<HDP>(r, c), k + at, real);
            cp16(dv + ta_at<HDP>(r, c), v + at, real);
        }
    };
    auto fetch_first = [&]() {
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) {
            if (p_begin + i < p_end) fetch(p_begin + i, i, pg[i]);
            cp_commit();
        }
    };
    if constexpr (!Ty::F32) {
        constexpr int CH = HDP / 8;
        if (wide) {
#pragma unroll 4
            for (int i = threadIdx.x; i < C::MT * CH; i += C::THREADS) {
                const int r = i / CH, c = i % CH;
                bool real;
                const size_t at = q_at(r, real);
                real = real && c * 8 < hd;
                cp16(sq + ta_at<HDP>(r, c), static_cast<const uint16_t *>(a.q) + (real ? at + c * 8 : 0), real);
            }
        } else {
            for (int i = threadIdx.x; i < C::MT * HDP; i += C::THREADS) {
                const int r = i / HDP, d = i % HDP;
                bool real;
                const size_t at = q_at(r, real);
                *reinterpret_cast<uint16_t *>(smem + ta_at<HDP>(r, d / 8) + (d % 8) * 2) = real && d < hd ? static_cast<const uint16_t *>(a.q)[at + d] : (uint16_t)0;
            }
        }
        fetch_first();   // q is part of the first group
        cp_wait<STAGES - 2>();
    } else {
        // four elements a lane, BATCH rows' loads in flight
        constexpr int LANES = HDP / 4 < 32 ? HDP / 4 : 32, EACH = HDP / 4 / LANES, ROWS = 32 / LANES, PASSES = C::MT / (WM * WN * ROWS);
        constexpr int BATCH = PASSES < 8 / EACH ? PASSES : 8 / EACH;
        bool fetched = false;
        for (int b0 = 0; b0 < PASSES; b0 += BATCH) {
            float4 x[BATCH][EACH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                bool real;
                const size_t at = q_at(((b0 + i) * WM * WN + warp) * ROWS + lane / LANES, real);
#pragma unroll
                for (int e = 0; e < EACH; ++e) {
                    const int d = (lane % LANES + e * LANES) * 4;
                    const float *q = static_cast<const float *>(a.q) + at + d;
                    x[i][e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (real && d < hd) x[i][e] = wide ? *reinterpret_cast<const float4 *>(q) : make_float4(q[0], q[1], q[2], q[3]);
                }
            }
            if (!fetched) fetch_first();
            fetched = true;
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int r = ((b0 + i) * WM * WN + warp) * ROWS + lane / LANES;
                float scale = 1.0f, back = 1.0f, mx = 0.0f;
#pragma unroll
                for (int e = 0; e < EACH; ++e)
                    mx = fmaxf(fmaxf(fmaxf(mx, fabsf(x[i][e].x)), fmaxf(fabsf(x[i][e].y), fabsf(x[i][e].z))), fabsf(x[i][e].w));
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                if (!BF && mx > 0.0f && mx < INFINITY) {
                    int e;
                    frexpf(mx, &e);
                    e = max(e, -100);   // 2^(14 - e) and its inverse stay normal
                    scale = __int_as_float((127 + 14 - e) << 23);
                    back = __int_as_float((127 + e - 14) << 23);
                }
                if (lane % LANES == 0) row_scale[r] = back;
#pragma unroll
                for (int e = 0; e < EACH; ++e) {
                    const int d = (lane % LANES + e * LANES) * 4;
                    float4 y = make_float4(x[i][e].x * scale, x[i][e].y * scale, x[i][e].z * scale, x[i][e].w * scale);
                    unsigned char *to = smem + ta_at<HDP>(r, d / 8) + (d % 8) * 2;
#pragma unroll
                    for (int p = 0; p < NP; ++p) {
                        const uint2 u = make_uint2(pack2<BF>(y.x, y.y), pack2<BF>(y.z, y.w));
                        *reinterpret_cast<uint2 *>(to + p * C::MT * HDP * 2) = u;
                        const float2 lo = unpack2<BF>(u.x), hi = unpack2<BF>(u.y);
                        y = make_float4(y.x - lo.x, y.y - lo.y, y.z - hi.x, y.w - hi.y);
                    }
                }
            }
        }
    }
    int next_pg = pg[STAGES - 1];
    __syncthreads();

    const int row_lo = wm * 16 + lane / 4;                 // this thread's rows: row_lo and row_lo + 8
    const int node_lo = ta_node(g, s.first + row_lo), node_hi = ta_node(g, s.first + row_lo + 8);
    const float f_lo = Ty::F32 ? fmaxf(g.scale2 * row_scale[row_lo], 1e-37f) : g.scale2;   // above 0: masked scores stay -inf
    const float f_hi = Ty::F32 ? fmaxf(g.scale2 * row_scale[row_lo + 8], 1e-37f) : g.scale2;
    const int depth_lo = a.window > 0 && node_lo < s.t ? ta_depth(a, s.r0 + node_lo) : 0;
    const int depth_hi = a.window > 0 && node_hi < s.t ? ta_depth(a, s.r0 + node_hi) : 0;
    float o[ND][4], m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.0f, l_hi = 0.0f;
#pragma unroll
    for (int i = 0; i < ND; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    constexpr bool Q_REGS = HDP * NP <= 128;
    uint32_t qr[Q_REGS ? NP : 1][Q_REGS ? HDP / 16 : 1][4];
    const uint32_t q_row = (uint32_t)(wm * 16 + lane % 16);
    if (Q_REGS)
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int ks = 0; ks < HDP / 16; ++ks) ldsm4(qr[p][ks], sq + p * C::MT * HDP * 2 + ta_at<HDP>(q_row, ks * 2 + lane / 16));

    for (int page = p_begin; page < p_end; ++page) {
        cp_wait<STAGES - 2>();
        __syncthreads();
        const int it = page - p_begin;
        {   // the stage that was read in the last round takes the next page
            const int ahead = page + STAGES - 1;
            if (ahead < p_end) {
                fetch(ahead, (it + STAGES - 1) % STAGES, next_pg);
                if (ahead + 1 < p_end) next_pg = ta_page(kv, s.slot, ahead + 1, err);
            }
            cp_commit();
        }
        const uint32_t sk = ring + (it % STAGES) * 2 * C::TILE, sv = sk + C::TILE;
        float sc[NK][4];
#pragma unroll
        for (int i = 0; i < NK; ++i) sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < HDP / 16; ++ks) {
            uint32_t qa[NP][4];
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                if (Q_REGS) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) qa[p][e] = qr[Q_REGS ? p : 0][Q_REGS ? ks : 0][e];
                } else {
                    ldsm4(qa[p], sq + p * C::MT * HDP * 2 + ta_at<HDP>(q_row, ks * 2 + lane / 16));
                }
            }
#pragma unroll
            for (int i = 0; i < NK / 2; ++i) {
                uint32_t kb[4];   // positions 16 i .. + 7 (words 0, 1) and + 8 .. 15 (2, 3)
                ldsm4(kb, sk + ta_at<HDP>(wn * KN + i * 16 + (lane / 16) * 8 + lane % 8, ks * 2 + (lane / 8) % 2));
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    mma16816<BF>(sc[2 * i], qa[p], kb[0], kb[1]);
                    mma16816<BF>(sc[2 * i + 1], qa[p], kb[2], kb[3]);
                }
            }
        }
        const int p0 = page * PAGE;
        const bool part = p0 + PAGE > s.base || (a.window > 0 && p0 < (long long)s.base + 64 * a.mask_words - a.window);
        unsigned long long see_lo = ~0ull, see_hi = ~0ull;
        if (part) {
            see_lo = ta_see(a, s, node_lo, p0, depth_lo);
            see_hi = ta_see(a, s, node_hi, p0, depth_hi);
            if (ta_short_window(a) && p0 + PAGE > s.base) {
                // the depths of the page's nodes, two a lane, against each of
                // the warp's rows in turn (reading them per ancestor of a row:
                // 53 trees of 130 nodes, window 4, 12 heads of 64, fp32: 176 us
                // instead of 105)
                const int j = p0 - s.base + lane;
                const int d0 = j >= 0 && j < s.t ? ta_depth(a, s.r0 + j) : INT_MAX, d1 = j + 32 >= 0 && j + 32 < s.t ? ta_depth(a, s.r0 + j + 32) : INT_MAX;
                const int least_lo = depth_lo - a.window + 1, least_hi = depth_hi - a.window + 1;
                unsigned long long keep_lo = 0, keep_hi = 0;
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const int t_lo = __shfl_sync(0xffffffffu, least_lo, 4 * r), t_hi = __shfl_sync(0xffffffffu, least_hi, 4 * r);
                    const unsigned long long b_lo = __ballot_sync(0xffffffffu, d0 >= t_lo) | (unsigned long long)__ballot_sync(0xffffffffu, d1 >= t_lo) << 32;
                    const unsigned long long b_hi = __ballot_sync(0xffffffffu, d0 >= t_hi) | (unsigned long long)__ballot_sync(0xffffffffu, d1 >= t_hi) << 32;
                    if (lane / 4 == r) { keep_lo = b_lo; keep_hi = b_hi; }
                }
                see_lo &= keep_lo;   // committed positions: INT_MAX above, kept
                see_hi &= keep_hi;
            }
        }
        float x_lo = -INFINITY, x_hi = -INFINITY;
        const unsigned w_lo = (unsigned)(see_lo >> (wn * KN + (lane % 4) * 2)), w_hi = (unsigned)(see_hi >> (wn * KN + (lane % 4) * 2));
        const unsigned z_lo = (unsigned)(see_lo >> 32 >> ((lane % 4) * 2)), z_hi = (unsigned)(see_hi >> 32 >> ((lane % 4) * 2));
#pragma unroll
        for (int i = 0; i < NK; ++i) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (part) {
                    const unsigned b_lo = i < 4 ? w_lo >> (8 * i + e) : z_lo >> (8 * (i - 4) + e), b_hi = i < 4 ? w_hi >> (8 * i + e) : z_hi >> (8 * (i - 4) + e);
                    if (!(b_lo & 1u)) sc[i][e] = -INFINITY;
                    if (!(b_hi & 1u)) sc[i][2 + e] = -INFINITY;
                }
                x_lo = fmaxf(x_lo, sc[i][e]);
                x_hi = fmaxf(x_hi, sc[i][2 + e]);
            }
        }
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
            x_lo = fmaxf(x_lo, __shfl_xor_sync(0xffffffffu, x_lo, d));
            x_hi = fmaxf(x_hi, __shfl_xor_sync(0xffffffffu, x_hi, d));
        }
        x_lo = fmaxf(x_lo * f_lo, m_lo);
        x_hi = fmaxf(x_hi * f_hi, m_hi);
        const float u_lo = x_lo == -INFINITY ? 0.0f : x_lo, u_hi = x_hi == -INFINITY ? 0.0f : x_hi;   // nothing seen yet: weights 0
        float c_lo = ex2(m_lo - u_lo), c_hi = ex2(m_hi - u_hi);
        m_lo = x_lo;
        m_hi = x_hi;
        l_lo *= c_lo;
        l_hi *= c_hi;
        uint32_t pa[NP][KN / 16][4];
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            float p[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                p[e] = ex2(fmaf(sc[i][e], f_lo, Ty::LIFT - u_lo));
                p[2 + e] = ex2(fmaf(sc[i][2 + e], f_hi, Ty::LIFT - u_hi));
                l_lo += p[e];
                l_hi += p[2 + e];
            }
            if (Ty::PARTS != 1.0f)
#pragma unroll
                for (int e = 0; e < 4; ++e) p[e] *= Ty::PARTS;
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                const uint32_t lo = pack2<BF>(p[0], p[1]), hi = pack2<BF>(p[2], p[3]);
                pa[q][i / 2][(i % 2) * 2] = lo;
                pa[q][i / 2][(i % 2) * 2 + 1] = hi;
                if (q + 1 < NP) {
                    const float2 a0 = unpack2<BF>(lo), a1 = unpack2<BF>(hi);
                    p[0] -= a0.x; p[1] -= a0.y; p[2] -= a1.x; p[3] -= a1.y;
                }
            }
        }
        // A weight 0 times an infinity or NaN in V is NaN: in a page that not
        // every row sees whole, such elements are taken out of the tile and
        // added by the rows that do see them.
        bool odd = false;
        if (part) {
            for (int i = threadIdx.x; i < C::TILE / 16; i += C::THREADS) {
                const uint4 u = *reinterpret_cast<const uint4 *>(smem + (sv - sq) + i * 16);
                const uint32_t e = BF ? 0x7f807f80u : 0x7c007c00u;
                const uint32_t w4[4] = {u.x, u.y, u.z, u.w};
                for (int j = 0; j < 4; ++j) odd |= (w4[j] & e & 0xffffu) == (e & 0xffffu) || (w4[j] & e & 0xffff0000u) == (e & 0xffff0000u);
            }
            odd = __syncthreads_or(odd);
        }
        if (part && odd) {
#pragma unroll
            for (int n = 0; n < ND; ++n) {
                float add[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                for (int j = wn * KN; j < wn * KN + KN; ++j) {
                    const uint32_t u = *reinterpret_cast<const uint32_t *>(smem + (sv - sq) + ta_at<HDP>(j, n) + (lane % 4) * 4);
                    const float2 v = unpack2<BF>(u);
                    const float vx = fabsf(v.x) < INFINITY ? 0.0f : v.x, vy = fabsf(v.y) < INFINITY ? 0.0f : v.y;
                    if (see_lo >> j & 1) { add[0] += vx; add[1] += vy; }
                    if (see_hi >> j & 1) { add[2] += vx; add[3] += vy; }
                }
                o[n][0] = fmaf(o[n][0], c_lo, add[0]); o[n][1] = fmaf(o[n][1], c_lo, add[1]);
                o[n][2] = fmaf(o[n][2], c_hi, add[2]); o[n][3] = fmaf(o[n][3], c_hi, add[3]);
            }
            c_lo = c_hi = 1.0f;
            __syncthreads();
            for (int i = threadIdx.x; i < PAGE * HDP; i += C::THREADS) {
                uint16_t *p = reinterpret_cast<uint16_t *>(smem + (sv - sq)) + i;
                const uint16_t e = BF ? 0x7f80u : 0x7c00u;
                if ((*p & e) == e) *p = 0;
            }
            __syncthreads();
        }
#pragma unroll
        for (int n = 0; n < ND / 2; ++n) {   // 16 columns at a time
            float add[2][4];
            if (Ty::F32) {
#pragma unroll
                for (int e = 0; e < 4; ++e) add[0][e] = add[1][e] = 0.0f;
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    add[h][0] = o[2 * n + h][0] * c_lo; add[h][1] = o[2 * n + h][1] * c_lo;
                    add[h][2] = o[2 * n + h][2] * c_hi; add[h][3] = o[2 * n + h][3] * c_hi;
                }
            }
#pragma unroll
            for (int ks = 0; ks < KN / 16; ++ks) {
                uint32_t vb[4];   // positions 16 ks .. + 15, columns 16 n .. + 7 (words 0, 1) and + 8 .. 15 (2, 3)
                ldsm4t(vb, sv + ta_at<HDP>(wn * KN + ks * 16 + lane % 16, n * 2 + lane / 16));
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    mma16816<BF>(add[0], pa[q][ks], vb[0], vb[1]);
                    mma16816<BF>(add[1], pa[q][ks], vb[2], vb[3]);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (Ty::F32) {   // the page's sum, added in fp32: long sums do not stay in the tensor cores' accumulators
                    o[2 * n + h][0] = fmaf(o[2 * n + h][0], c_lo, add[h][0]); o[2 * n + h][1] = fmaf(o[2 * n + h][1], c_lo, add[h][1]);
                    o[2 * n + h][2] = fmaf(o[2 * n + h][2], c_hi, add[h][2]); o[2 * n + h][3] = fmaf(o[2 * n + h][3], c_hi, add[h][3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[2 * n + h][e] = add[h][e];
                }
        }
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
        l_lo += __shfl_xor_sync(0xffffffffu, l_lo, d);
        l_hi += __shfl_xor_sync(0xffffffffu, l_hi, d);
    }
    // Where this CTA has all of the tile's pages it writes out, else (m, l, o).
    const bool pair = (a.ldo & 1) == 0 && (reinterpret_cast<uintptr_t>(a.out) & (QT == EC_T_F32 ? 7 : 3)) == 0;
    const bool whole = !PIECES || (p_begin == s.page0 && p_end == s.page1);
    const size_t part_at = ((size_t)blockIdx.x * 2 + (p_begin == s.page0)) * C::MT;   // PIECES: a CTA has at most one tile begun before, one left open
    float *po = g.part + part_at * HDP, *pm = g.part + (size_t)gridDim.x * 2 * C::MT * HDP + part_at * 2;
    // Join the warps that share rows and the CTAs of the cluster: every one
    // leaves its (m, l, o) in its shared memory, each CTA takes a share of the
    // rows, a warp a row, and lane i the weight of source i.
    const int ctas = PIECES ? 1 : g.cluster, me = PIECES ? 0 : (int)blockIdx.y, sources = ctas * WN;
    if (sources > 1) {
        cg::cluster_group cl = cg::this_cluster();
        cp_wait<0>();
        __syncthreads();
        float *jo = reinterpret_cast<float *>(smem + C::Q_BYTES), *jm = jo + WN * C::MT * HDP;   // [WN][MT][HDP], [WN][MT][2]
#pragma unroll
        for (int n = 0; n < ND; ++n) {
            float *p = jo + (size_t)(wn * C::MT + row_lo) * HDP + ((n * 8 + (lane % 4) * 2) ^ ((row_lo & 7) * 4));   // rows shifted against bank conflicts
            *reinterpret_cast<float2 *>(p) = make_float2(o[n][0], o[n][1]);
            *reinterpret_cast<float2 *>(p + 8 * HDP) = make_float2(o[n][2], o[n][3]);
        }
        if (lane % 4 == 0) {
            *reinterpret_cast<float2 *>(jm + (wn * C::MT + row_lo) * 2) = make_float2(m_lo, l_lo);
            *reinterpret_cast<float2 *>(jm + (wn * C::MT + row_lo + 8) * 2) = make_float2(m_hi, l_hi);
        }
        if (ctas > 1) cl.sync();
        else __syncthreads();
        for (int r = me + warp * ctas; r < C::MT; r += ctas * WM * WN) {
            const int rr = s.first + r, node = ta_node(g, rr);
            if (node >= s.t) continue;
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (lane < sources) {
                const float *p = jm + ((lane / ctas) * C::MT + r) * 2;
                ml = *reinterpret_cast<const float2 *>(ctas > 1 ? cl.map_shared_rank(p, lane % ctas) : p);
            }
            float m = ml.x;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            const float f = ex2(ml.x - (m == -INFINITY ? 0.0f : m));
            const float l = ec_warp_sum(ml.y * f);
            constexpr int EACH = HDP >= 128 ? HDP / 128 : 1, VEC = HDP >= 128 ? 4 : 2;
            float acc[EACH][VEC] = {};
#pragma unroll 4
            for (int i = 0; i < sources; ++i) {
                const float w = __shfl_sync(0xffffffffu, f, i);
                const float *p = jo + (size_t)((i / ctas) * C::MT + r) * HDP;
                if (ctas > 1) p = cl.map_shared_rank(p, i % ctas);
#pragma unroll
                for (int e = 0; e < EACH; ++e) {
                    const int d = (lane * VEC + e * 128) ^ ((r & 7) * 4);
                    if constexpr (VEC == 4) {
                        const float4 v = *reinterpret_cast<const float4 *>(p + d);
                        acc[e][0] = fmaf(v.x, w, acc[e][0]); acc[e][1] = fmaf(v.y, w, acc[e][1]);
                        acc[e][2] = fmaf(v.z, w, acc[e][2]); acc[e][3] = fmaf(v.w, w, acc[e][3]);
                    } else {
                        const float2 v = *reinterpret_cast<const float2 *>(p + d);
                        acc[e][0] = fmaf(v.x, w, acc[e][0]); acc[e][1] = fmaf(v.y, w, acc[e][1]);
                    }
                }
            }
            const float inv = l == 0.0f ? 0.0f : (1.0f / Ty::PARTS) / l;
            const size_t to = (size_t)(s.r0 + node) * a.ldo + (size_t)(kh * g.group + rr - node * g.group) * hd;
            if (!whole && lane == 0) *reinterpret_cast<float2 *>(pm + r * 2) = make_float2(m, l);
#pragma unroll
            for (int e = 0; e < EACH; ++e)
#pragma unroll
                for (int h = 0; h < VEC; h += 2) {
                    const int d = lane * VEC + e * 128 + h;
                    if (d >= hd) continue;
                    if (!whole) *reinterpret_cast<float2 *>(po + (size_t)r * HDP + d) = make_float2(acc[e][h], acc[e][h + 1]);
                    else ta_store2<QT>(a.out, to + d, acc[e][h] * inv, acc[e][h + 1] * inv, pair);
                }
        }
        if (ctas > 1) cl.sync();   // the others have read this CTA's part
    } else {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = row_lo + 8 * half, rr = s.first + r, node = half ? node_hi : node_lo;
            if (node >= s.t) continue;
            const float m = half ? m_hi : m_lo, l = half ? l_hi : l_lo, inv = l == 0.0f ? 0.0f : (1.0f / Ty::PARTS) / l;
            const size_t to = (size_t)(s.r0 + node) * a.ldo + (size_t)(kh * g.group + rr - node * g.group) * hd;
            if (!whole && lane % 4 == 0) *reinterpret_cast<float2 *>(pm + r * 2) = make_float2(m, l);
#pragma unroll
            for (int n = 0; n < ND; ++n) {
                const int d = n * 8 + (lane % 4) * 2;
                if (d >= hd) continue;
                const float x = o[n][2 * half], y = o[n][2 * half + 1];
                if (!whole) *reinterpret_cast<float2 *>(po + (size_t)r * HDP + d) = make_float2(x, y);
                else ta_store2<QT>(a.out, to + d, x * inv, y * inv, pair);
            }
        }
    }
    if constexpr (PIECES) {
        at += p_end - p_begin;
        cp_wait<0>();
        __syncthreads();   // shared memory is free for the next tile
    }
    } while (PIECES);
}

// A lane's part of a row of partial sums: VEC floats, EACH times.
template <int HDP> struct TaLane {
    static constexpr int VEC = HDP >= 128 ? 4 : 2, EACH = HDP / 32 / VEC;
    float v[EACH][VEC];
    EC_DEV void zero() {
#pragma unroll
        for (int e = 0; e < EACH; ++e)
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[e][i] = 0.0f;
    }
    EC_DEV void load(const float *row) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const float *p = row + (threadIdx.x & 31) * VEC + e * 128;
            if constexpr (VEC == 4) {
                const float4 x = *reinterpret_cast<const float4 *>(p);
                v[e][0] = x.x; v[e][1] = x.y; v[e][2] = x.z; v[e][3] = x.w;
            } else {
                const float2 x = *reinterpret_cast<const float2 *>(p);
                v[e][0] = x.x; v[e][1] = x.y;
            }
        }
    }
    EC_DEV void add(const TaLane &o, float w) {
#pragma unroll
        for (int e = 0; e < EACH; ++e)
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[e][i] = fmaf(o.v[e][i], w, v[e][i]);
    }
    template <int QT> EC_DEV void store(void *out, size_t to, int hd, float inv) const {
#pragma unroll
        for (int e = 0; e < EACH; ++e)
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
                const int d = (threadIdx.x & 31) * VEC + e * 128 + i;
                if (d < hd) ta_store2<QT>(out, to + d, v[e][i] * inv, v[e][i + 1] * inv, false);
            }
    }
};

// Joins the tiles that borders between pieces cut, in the order of their
// pages.  SHARED (few tiles, cut into many pieces): CTA (tile, r) joins row r,
// its warps sharing out the pieces.  Otherwise CTA (i, y) joins half of the
// rows, up to four a warp, of the tile that the border behind piece i is the
// first to cut.
constexpr int TJ_THREADS = 256, TJ_WARPS = TJ_THREADS / 32, TJ_PIECES = 1024;

template <int QT, int HDP, bool SHARED>
__global__ void __launch_bounds__(TJ_THREADS) k_tree_join(const ec_kv_pages kv, const ec_tree_attn a, const TaGeo g, int mt, int pieces, float unit, int *err) {
    EC_PDL_ENTER();
    typedef TaLane<HDP> Lane;
    __shared__ float weight[SHARED ? TJ_PIECES : 1], red[TJ_WARPS], acc_of[SHARED ? TJ_WARPS : 1][HDP];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hd = a.head_dim;
    TaLine line;
    line.init(kv, a, g, mt, pieces, err);
    TaTile s;
    int begin, i0 = blockIdx.x;
    if (line.n == 0) return;
    if (SHARED) {
        if (!line.by_index(kv, a, g, mt, blockIdx.x, s, begin, err)) return;
        i0 = line.piece(begin);
    } else {
        if (i0 + 1 >= line.n) return;
        const int border = line.start(i0 + 1);
        s = line.tile(kv, a, g, mt, border, begin, err);
        if (begin == border || line.start(i0) > begin) return;   // cuts nothing, or not the first
    }
    const int n = line.piece(begin + s.len - 1) - i0 + 1;   // pieces of the tile
    if (n == 1) return;
    auto place = [&](int i, int r) { return ((size_t)(i0 + i) * 2 + (i == 0)) * mt + r; };   // begun in piece i0, goes on in the others
    auto out_at = [&](int r) {
        const int rr = s.first + r, node = ta_node(g, rr);
        return (size_t)(s.r0 + node) * a.ldo + (size_t)(s.kh * g.group + rr - node * g.group) * hd;
    };
    const float *po = g.part, *pm = g.part + (size_t)pieces * 2 * mt * HDP;
    if constexpr (SHARED) {
        const int r = blockIdx.y;
        if (ta_node(g, s.first + r) >= s.t) return;
        auto join = [&](float v, bool max) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float u = __shfl_xor_sync(0xffffffffu, v, o);
                v = max ? fmaxf(v, u) : v + u;
            }
            __syncthreads();
            if (lane == 0) red[warp] = v;
            __syncthreads();
            v = red[0];
#pragma unroll
            for (int w = 1; w < TJ_WARPS; ++w) v = max ? fmaxf(v, red[w]) : v + red[w];
            return v;
        };
        float m = -INFINITY, l = 0.0f;
        for (int i = threadIdx.x; i < n; i += TJ_THREADS) m = fmaxf(m, pm[place(i, r) * 2]);
        m = join(m, true);
        if (m == -INFINITY) m = 0.0f;
        for (int i = threadIdx.x; i < n; i += TJ_THREADS) {
            const float2 ml = *reinterpret_cast<const float2 *>(pm + place(i, r) * 2);
            const float f = ex2(ml.x - m);
            l = fmaf(ml.y, f, l);
            weight[i] = f;
        }
        l = join(l, false);
        Lane acc;
        acc.zero();
        for (int b = warp; b < n; b += 8 * TJ_WARPS) {
            Lane x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j].load(po + place(min(b + j * TJ_WARPS, n - 1), r) * HDP);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (b + j * TJ_WARPS < n) acc.add(x[j], weight[b + j * TJ_WARPS]);
        }
#pragma unroll
        for (int e = 0; e < Lane::EACH; ++e)
#pragma unroll
            for (int i = 0; i < Lane::VEC; ++i) acc_of[warp][lane * Lane::VEC + e * 128 + i] = acc.v[e][i];
        __syncthreads();
        const float inv = l == 0.0f ? 0.0f : unit / l;
        for (int d = threadIdx.x * 2; d < hd; d += 2 * TJ_THREADS) {
            float x = 0.0f, y = 0.0f;
#pragma unroll
            for (int w = 0; w < TJ_WARPS; ++w) { x += acc_of[w][d]; y += acc_of[w][d + 1]; }
            ta_store2<QT>(a.out, out_at(r) + d, x * inv, y * inv, false);
        }
    } else {
        constexpr int ROWS = HDP == 256 ? 2 : 4;
        const int stride = gridDim.y * TJ_WARPS;
        for (int r0 = blockIdx.y * TJ_WARPS + warp; r0 < mt; r0 += ROWS * stride) {
            Lane acc[ROWS];
            float m[ROWS], l[ROWS];
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
                acc[k].zero();
                m[k] = -INFINITY;
                l[k] = 0.0f;
            }
            for (int i = 0; i < n; ++i) {   // one pass with a running maximum: the rows' loads go together
                Lane x[ROWS];
                float2 ml[ROWS];
#pragma unroll
                for (int k = 0; k < ROWS; ++k) {
                    const int r = min(r0 + k * stride, mt - 1);
                    ml[k] = *reinterpret_cast<const float2 *>(pm + place(i, r) * 2);
                    x[k].load(po + place(i, r) * HDP);
                }
#pragma unroll
                for (int k = 0; k < ROWS; ++k) {
                    const float mn = fmaxf(m[k], ml[k].x), u = mn == -INFINITY ? 0.0f : mn;
                    const float c = ex2(m[k] - u), f = ex2(ml[k].x - u);
                    m[k] = mn;
                    l[k] = fmaf(ml[k].y, f, l[k] * c);
#pragma unroll
                    for (int e = 0; e < Lane::EACH; ++e)
#pragma unroll
                        for (int j = 0; j < Lane::VEC; ++j) acc[k].v[e][j] = fmaf(x[k].v[e][j], f, acc[k].v[e][j] * c);
                }
            }
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
                const int r = r0 + k * stride;
                if (r < mt && ta_node(g, s.first + r) < s.t) acc[k].template store<QT>(a.out, out_at(r), hd, l[k] == 0.0f ? 0.0f : unit / l[k]);
            }
        }
    }
}

// ---- launch --------------------------------------------------------------------

struct TaPlan {
    int hdp, mt, tiles;   // tiles: upper bound over all sequences
    int pieces;           // 0: clusters
    TaGeo g;
};

constexpr int TA_MOST = 0x7fffffff - PAGE;   // positions that a plan counts with, at most

int ta_up(int a, int b) { return (a + b - 1) / b; }

size_t ta_piece_bytes(const TaPlan &p) { return (size_t)2 * p.mt * (p.hdp + 2) * 4; }

// Clusters where they alone give every SM something to do or a tile has few
// pages: one launch (one token over 300 positions: 7.2 us, in pieces 9.5).
// Otherwise as many pieces as CTAs are resident.
TaPlan ta_plan(int n_seq, int rows, int n_head, int n_kv_head, int hd, int max_len, int slot_pages, int window, bool f32, bool tc, int sms) {
    TaPlan p;
    p.hdp = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
    p.g.group = n_head / n_kv_head;
    int up = 0;
    while ((1 << up) < p.g.group) ++up;
    p.g.div_shift = 30 + up;   // rounded up: exact for rows below 2^30
    p.g.div_mul = (unsigned)(((1ull << p.g.div_shift) + p.g.group - 1) / p.g.group);
    const int mean = (int)(((long long)rows * p.g.group + n_seq - 1) / n_seq);
    // from 65 rows on, tiles of twice 128 on the tensor cores of tcgen05
    p.mt = mean <= 16 ? 16 : mean <= 32 ? 32 : mean <= 64 || !tc ? 64 : TC_ROWS;
    p.tiles = (int)(((long long)rows * p.g.group) / p.mt + n_seq);   // every sequence rounds up once; rows * group fits 31 bits
    int pages = ta_up(max_len > 0 ? max_len : 1, PAGE);
    if (window > 0 && pages > window / PAGE + 2) pages = window / PAGE + 2;
    // Up to 16 pages a tile is one cluster's, of as many CTAs as two rounds of
    // the SMs hold: 24 windowed sequences of 10 pages, 12 heads of 64, take 20
    // us so and 31 us as equal pieces with a second launch; 64 sequences of one
    // token up to 900 positions, 14 heads of 64 on 2, 16 and 22 us.  Beyond,
    // ragged lengths leave clusters waiting: 32 sequences of 65 to 1900
    // positions take 35 us as pieces, 41 us as clusters.  fp32 rows wider
    // than 64, with two or three products for each of the others', are better
    // cut from 9 pages on unless the clusters leave SMs idle: 32 trees of 24
    // nodes at 450 to 900 positions 50 us, 57 as clusters.
    const long long tiles = (long long)p.tiles * n_kv_head;
    p.g.cluster = pages >= 8 ? 8 : pages >= 4 ? 4 : pages >= 2 ? 2 : 1;
    while (p.g.cluster > 1 && tiles * p.g.cluster > 2 * sms) p.g.cluster /= 2;
    p.pieces = 0;
    const bool cut = pages > 16 || (pages > 8 && f32 && p.hdp > 64 && tiles * p.g.cluster > sms);
    if (cut && tiles * slot_pages < TA_LINE)
        p.pieces = (p.mt == TC_ROWS ? 1 : p.hdp == 64 && !f32 ? 3 : p.hdp <= 128 ? 2 : 1) * sms;
    if (!p.pieces && p.mt == TC_ROWS) {   // clusters: the register tiles only
        p.mt = 64;
        p.tiles = (int)(((long long)rows * p.g.group) / p.mt + n_seq);
    }
    return p;
}

// A workspace of only `fit` pieces.  A CTA walks its piece alone, so fewer
// pieces than clusters would keep CTAs busy take longer than those: one tree of
// 9 nodes at 30011 positions, 12 heads of 128 on 2, 103 us in clusters (16
// CTAs), 753 in 2 pieces, 106 in 16; 32 fp32 sequences at 65 to 1900 positions
// 41 us in clusters, 61 in 74 pieces, 41 in 147.  A tcgen05 piece does the work
// of two CTAs of a cluster or more: 16 trees of 48 to 64 nodes at 6000 to 10000
// positions 234 us in clusters, 3607 in 2 pieces, 266 in 32, 146 in 74 (heads of
// 64: 159 in clusters, 148 in 74); one such tree 41 in clusters of 112 CTAs, 44
// in 48 pieces, 41 in 64.
void ta_fit(TaPlan &p, size_t fit, long long rows, int n_seq, int n_kv_head, int sms) {
    const bool tc = p.mt == TC_ROWS;
    TaPlan c = p;
    if (tc) {   // clusters: the register tiles only
        c.mt = 64;
        c.tiles = (int)(rows * c.g.group / c.mt + n_seq);
    }
    long long busy = (long long)c.tiles * n_kv_head * c.g.cluster;
    if (busy > sms) busy = sms;
    if (fit > 1 && (long long)fit * (tc ? 2 : 1) >= busy) {
        p.pieces = (int)fit;
        return;
    }
    p = c;
    p.pieces = 0;
}

int g_attr[64][64];

template <int QT, int HDP>
int ta_join(const ec_kv_pages &kv, const ec_tree_attn &a, const TaPlan &p, float unit, int *err, cudaStream_t stream) {
    const long long tiles = (long long)p.tiles * a.n_kv_head;
    if (4 * tiles <= p.pieces && p.pieces <= TJ_PIECES)
        return (int)ec_launch_k(k_tree_join<QT, HDP, true>, dim3((unsigned)tiles, p.mt), dim3(TJ_THREADS), 0, stream, kv, a, p.g, p.mt, p.pieces, unit, err);
    return (int)ec_launch_k(k_tree_join<QT, HDP, false>, dim3(p.pieces - 1, 2), dim3(TJ_THREADS), 0, stream, kv, a, p.g, p.mt, p.pieces, unit, err);
}

template <int QT, int KT, int HDP, int WM, int WN, int STAGES>
int ta_run(const ec_kv_pages &kv, const ec_tree_attn &a, const TaPlan &p, int id, int *err, cudaStream_t stream) {
    typedef TaMma<QT, KT, HDP, WM, WN, STAGES> C;
    static_assert(C::SMEM <= 232448, "shared memory per CTA");
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    auto pieces = k_tree_mma<QT, KT, HDP, WM, WN, STAGES, true>;
    auto shared = k_tree_mma<QT, KT, HDP, WM, WN, STAGES, false>;
    if (!g_attr[id][dev]) {
        e = cudaFuncSetAttribute(pieces, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(shared, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return (int)e;
        g_attr[id][dev] = 1;
    }
    if (p.pieces) {
        pieces<<<p.pieces, C::THREADS, C::SMEM, stream>>>(kv, a, p.g, err);
        e = cudaGetLastError();
        if (e != cudaSuccess || p.pieces == 1) return (int)e;
        return ta_join<QT, HDP>(kv, a, p, 1.0f / C::Ty::PARTS, err, stream);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.tiles, p.g.cluster, a.n_kv_head);
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = at[0].val.clusterDim.z = 1;
    at[0].val.clusterDim.y = (unsigned)p.g.cluster;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, shared, kv, a, p.g, err);
}

template <int QT, int KT, int HDP, int STAGES>
int ta_rows(const ec_kv_pages &kv, const ec_tree_attn &a, const TaPlan &p, int id, int *err, cudaStream_t stream) {
    if (p.mt == 16) return ta_run<QT, KT, HDP, 1, 4, STAGES>(kv, a, p, id, err, stream);
    if (p.mt == 32) return ta_run<QT, KT, HDP, 2, 2, STAGES>(kv, a, p, id + 1, err, stream);
    return ta_run<QT, KT, HDP, 4, 1, STAGES>(kv, a, p, id + 2, err, stream);
}

template <int QT, int KT>
int ta_dims(const ec_kv_pages &kv, const ec_tree_attn &a, const TaPlan &p, int id, int *err, cudaStream_t stream) {
    if (p.hdp == 64) return ta_rows<QT, KT, 64, 4>(kv, a, p, id, err, stream);
    if (p.hdp == 128) return ta_rows<QT, KT, 128, QT == EC_T_F32 ? 2 : 3>(kv, a, p, id + 3, err, stream);
    return ta_rows<QT, KT, 256, 2>(kv, a, p, id + 6, err, stream);
}

}  // namespace

// The larger of what 16-bit and fp32 queries take; a window only ever takes less.
extern "C" size_t ec_tree_attention_bytes(int n_seq, int rows, int n_head, int n_kv_head, int head_dim, int max_len, int num_sms) {
    size_t bytes = 0;
    for (int f32 = 0; f32 < 2; ++f32) {
        const TaPlan p = ta_plan(n_seq, rows, n_head, n_kv_head, head_dim, max_len > 0 && max_len < TA_MOST ? max_len : TA_MOST, 1, 0, f32,
                                 !f32 && (head_dim == 64 || head_dim == 128), num_sms);
        const size_t need = p.pieces * ta_piece_bytes(p);
        if (need > bytes) bytes = need;
    }
    return bytes;
}

extern "C" int ec_launch_tree_attention(const ec_kv_pages *kv, const ec_tree_attn *a, int num_sms, int *err, cudaStream_t stream) {
    long long len = a->max_len > 0 ? a->max_len : (long long)kv->pages_per_slot * PAGE;
    TaPlan p = ta_plan(a->n_seq, a->rows, a->n_head, a->n_kv_head, a->head_dim, (int)(len < TA_MOST ? len : TA_MOST), kv->pages_per_slot, a->window, a->type == EC_T_F32,
                       ta_tc_takes(a->type, kv->type, a->head_dim), num_sms);
    if (p.pieces) {
        const size_t fit = a->work ? a->work_bytes / ta_piece_bytes(p) : 0;
        if (fit < (size_t)p.pieces) ta_fit(p, fit, (long long)a->rows, a->n_seq, a->n_kv_head, num_sms);
    }
    p.g.scale2 = (a->scale > 0.0f ? a->scale : 1.0f / sqrtf((float)a->head_dim)) * LOG2E;
    p.g.part = static_cast<float *>(a->work);
    const bool bf = kv->type == EC_T_BF16;
    if (p.mt == TC_ROWS) {
        const int e = ta_tc_launch(*kv, *a, p.g, p.pieces, err, stream);
        if (e) return e;
        if (p.hdp == 64) return bf ? ta_join<EC_T_BF16, 64>(*kv, *a, p, 1.0f, err, stream) : ta_join<EC_T_F16, 64>(*kv, *a, p, 1.0f, err, stream);
        return bf ? ta_join<EC_T_BF16, 128>(*kv, *a, p, 1.0f, err, stream) : ta_join<EC_T_F16, 128>(*kv, *a, p, 1.0f, err, stream);
    }
    if (a->type == EC_T_F32) return bf ? ta_dims<EC_T_F32, EC_T_BF16>(*kv, *a, p, 0, err, stream) : ta_dims<EC_T_F32, EC_T_F16>(*kv, *a, p, 9, err, stream);
    return bf ? ta_dims<EC_T_BF16, EC_T_BF16>(*kv, *a, p, 18, err, stream) : ta_dims<EC_T_F16, EC_T_F16>(*kv, *a, p, 27, err, stream);
}
