// ec_tree.cu -- attention of drafted-token trees over a paged KV arena
// (ec_tree_attention).
//
// The rows of one KV head and sequence -- its T nodes times the G query heads
// that read the KV head -- share every K and V row, so they are one tile: row
// r is node r / G, query head r % G.  A page of 64 positions is one key tile.
// One pass over the pages with a running maximum m and sum l per row:
//   s = scale * q.k (masked: -inf), m' = max(m, s), p = 2^((s - m') log2 e),
//   l = l 2^((m - m') log2 e) + sum p,  o = o 2^((m - m') log2 e) + p V
// and out = o / l (0 where nothing was seen).  Positions of a sequence can be
// split over CTAs: each writes (m, l, o) of its pages and k_tree_join adds
// them up in the order of the pages.
#include "ec_common.cuh"
#include "ec_serve.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int PAGE = EC_KV_PAGE;

// ---- the work of a call ------------------------------------------------------

struct TaGeo {            // chosen by the launcher
    int group;            // query heads per KV head
    int nsplit, chunk;    // CTAs a sequence's pages are split over at most, pages per CTA at least
    int tiles;            // upper bound on row tiles of all sequences
    float scale2;         // scale * log2 e
    float *part;          // [tiles][n_kv_head][nsplit][MT][hdp] o, then [...][MT] (m, l)
};

struct TaTile {           // one row tile
    int b, first;         // sequence, its first row in the tile's (node, head) numbering
    int r0, t, base, slot;
    int page0, page1;     // pages that hold visible positions
};

EC_DEV int ta_splits(const TaTile &s, const TaGeo &g, int &chunk) {
    const int n = s.page1 - s.page0;
    chunk = max(g.chunk, (n + g.nsplit - 1) / g.nsplit);
    return n > 0 ? (n + chunk - 1) / chunk : 1;
}

// The row tile `ti` of `mt` rows in the sequences' order; false when there is
// none, or its sequence has a bad index (recorded).  Called by whole warps.
EC_DEV bool ta_find(const ec_kv_pages &kv, const ec_tree_attn &a, const TaGeo &g, int ti, int mt, TaTile &s, int *err) {
    const int lane = threadIdx.x & 31;
    int before = 0, b = -1, local = 0;
    for (int b0 = 0; b0 < a.n_seq && b < 0; b0 += 32) {
        const int i = b0 + lane;
        int n = 0;
        if (i < a.n_seq) {
            const long long t = (long long)a.row_start[i + 1] - a.row_start[i];
            const bool bad = t < 0 || t > a.rows;
            if (bad) atomicCAS(err, 0, EC_KERR_BAD_INDEX);
            n = bad ? 0 : (int)((t * g.group + mt - 1) / mt);
        }
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + sum > ti);
        if (hit) {
            const int l = __ffs((int)hit) - 1;
            b = b0 + l;
            local = ti - before - (__shfl_sync(0xffffffffu, sum, l) - __shfl_sync(0xffffffffu, n, l));
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (b < 0) return false;
    s.b = b;
    s.first = local * mt;
    s.r0 = a.row_start[b];
    s.t = a.row_start[b + 1] - s.r0;
    s.base = a.base[b];
    s.slot = a.slots ? a.slots[b] : b;
    if (s.r0 < 0 || s.r0 + s.t > a.rows || s.base < 0 || s.slot < 0 || s.slot >= kv.n_slots ||
        (long long)s.base + s.t > (long long)kv.pages_per_slot * PAGE) {
        if (threadIdx.x == 0) atomicCAS(err, 0, EC_KERR_BAD_INDEX);
        return false;
    }
    const int lo = a.window > 0 && s.base > a.window ? s.base - a.window : 0;   // no row sees a position below it
    s.page0 = lo / PAGE;
    s.page1 = (s.base + s.t + PAGE - 1) / PAGE;
    return true;
}

EC_DEV int ta_page(const ec_kv_pages &kv, int slot, int i, int *err) {
    int page = __ldg(kv.page_table + (size_t)slot * kv.pages_per_slot + i);
    if (page < 0 || page >= kv.n_pages) {
        if ((threadIdx.x & 31) == 0) atomicCAS(err, 0, EC_KERR_BAD_INDEX);
        page = 0;
    }
    return page;
}

EC_DEV int ta_depth(const ec_tree_attn &a, int row) {
    int d = -1;
    for (int w = 0; w < a.mask_words; ++w) d += __popcll(a.mask[(size_t)row * a.mask_words + w]);
    return d;
}

EC_DEV unsigned long long ta_low(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }

// Which of the 64 positions from p0 on the node `i` of the tile's sequence
// sees, one bit each.
EC_DEV unsigned long long ta_allow(const ec_tree_attn &a, const TaTile &s, int i, int p0) {
    if (i >= s.t) return 0ull;
    const int row = s.r0 + i, j0 = p0 - s.base;
    const unsigned long long *m = a.mask + (size_t)row * a.mask_words;
    unsigned long long tree = 0;
    if (j0 < 0) {
        if (j0 > -64) tree = m[0] << -j0;
    } else {
        const int w = j0 / 64, sh = j0 % 64;
        if (w < a.mask_words) tree = m[w] >> sh;
        if (sh && w + 1 < a.mask_words) tree |= m[w + 1] << (64 - sh);
    }
    const unsigned long long prefix = ta_low(s.base - p0);
    tree &= ta_low(s.base + s.t - p0) & ~prefix;
    if (a.window <= 0) return prefix | tree;
    const int depth = ta_depth(a, row);
    const int from = s.base + depth - a.window + 1;
    if (a.window < 64 * a.mask_words)   // nodes of one tree are fewer levels apart than that
        for (unsigned long long left = tree; left; left &= left - 1) {
            const int bit = __ffsll((long long)left) - 1;
            if (s.base + ta_depth(a, s.r0 + j0 + bit) < from) tree &= ~(1ull << bit);
        }
    return (prefix & ~ta_low(from - p0)) | tree;
}

template <int T> EC_DEV void ta_store2(void *p, size_t i, float x, float y, bool pair) {   // pair: i even and aligned
    if (T == EC_T_F32) {
        float *o = static_cast<float *>(p) + i;
        if (pair) *reinterpret_cast<float2 *>(o) = make_float2(x, y);
        else { o[0] = x; o[1] = y; }
    } else {
        uint16_t *o = static_cast<uint16_t *>(p) + i;
        const uint16_t a = T == EC_T_F16 ? __half_as_ushort(__float2half_rn(x)) : __bfloat16_as_ushort(__float2bfloat16_rn(x));
        const uint16_t b = T == EC_T_F16 ? __half_as_ushort(__float2half_rn(y)) : __bfloat16_as_ushort(__float2bfloat16_rn(y));
        if (pair) *reinterpret_cast<uint32_t *>(o) = (uint32_t)a | (uint32_t)b << 16;
        else { o[0] = a; o[1] = b; }
    }
}

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
EC_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
EC_DEV void cp16(uint32_t dst, const void *src, bool real) {   // 16 bytes, or zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
EC_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> EC_DEV void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <bool BF> EC_DEV uint32_t pack2(float x, float y) {
    if (BF) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <bool BF> EC_DEV float2 unpack2(uint32_t u) {
    if (BF) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}

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
    static constexpr float LIFT = BF ? 0.0f : 14.0f;
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
    static constexpr int JOIN = WN > 1 ? WN * MT * (HDP + 2) * 4 : 0;   // overlays the ring
    static constexpr int SMEM = Q_BYTES + (RING > JOIN ? RING : JOIN) + MT * 4 + 128;
};

// Bounded by the bytes of K and V for few rows, and there by how many of them
// are in flight: STAGES pages of K and V per CTA and two or three CTAs per SM
// (hd 64: 16 KB a stage, hd 128: 32 KB).
template <int QT, int KT, int HDP, int WM, int WN, int STAGES>
__global__ void __launch_bounds__(32 * WM * WN) k_tree_mma(const ec_kv_pages kv, const ec_tree_attn a, const TaGeo g, int *err) {
    EC_PDL_ENTER();
    typedef TaMma<QT, KT, HDP, WM, WN, STAGES> C;
    typedef typename C::Ty Ty;
    constexpr bool BF = Ty::BF;
    constexpr int NP = C::NP, KN = C::KN, NK = KN / 8, ND = HDP / 8;
    extern __shared__ __align__(1024) unsigned char smem[];
    const uint32_t sq = ec_smem_u32(smem), ring = sq + C::Q_BYTES;
    float *row_scale = reinterpret_cast<float *>(smem + C::SMEM - 128 - C::MT * 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wm = warp % WM, wn = warp / WM;
    const int kh = blockIdx.z, hd = a.head_dim;
    TaTile s;
    if (!ta_find(kv, a, g, blockIdx.x, C::MT, s, err)) return;
    int chunk;
    const int splits = ta_splits(s, g, chunk), split = blockIdx.y;
    if (split >= splits) return;
    const int p_begin = s.page0 + split * chunk, p_end = min(s.page1, p_begin + chunk), end = s.base + s.t;

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
    int next_pg = 0;
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
        if (p_begin + i < p_end) fetch(p_begin + i, i, ta_page(kv, s.slot, p_begin + i, err));
        cp_commit();
    }
    if (p_begin + STAGES - 1 < p_end) next_pg = ta_page(kv, s.slot, p_begin + STAGES - 1, err);

    // the queries of the tile, in parts; rows behind the sequence are zero
    for (int r = warp; r < C::MT; r += WM * WN) {
        const int rr = s.first + r, node = rr / g.group;
        const bool real = node < s.t;
        const size_t at = real ? (size_t)(s.r0 + node) * a.ldq + ((size_t)kh * g.group + rr % g.group) * hd : 0;
        float x[HDP / 32], scale = 1.0f;
        if (Ty::F32) {
            float mx = 0.0f;
#pragma unroll
            for (int i = 0; i < HDP / 32; ++i) {
                const int d = lane + 32 * i;
                x[i] = real && d < hd ? static_cast<const float *>(a.q)[at + d] : 0.0f;
                mx = ec_max_keep(mx, fabsf(x[i]));
            }
            mx = ec_warp_max(mx);
            float back = 1.0f;
            if (!BF && mx > 0.0f && mx < INFINITY) {
                int e;
                frexpf(mx, &e);
                e = max(e, -100);   // 2^(14 - e) and its inverse stay normal
                scale = ldexpf(1.0f, 14 - e);
                back = ldexpf(1.0f, e - 14);
            }
            if (lane == 0) row_scale[r] = back;
        }
#pragma unroll
        for (int i = 0; i < HDP / 32; ++i) {
            const int d = lane + 32 * i;
            unsigned char *to = smem + ta_at<HDP>(r, d / 8) + (d % 8) * 2;
            if (Ty::F32) {
                float left = x[i] * scale;
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    const uint32_t u = pack2<BF>(left, 0.0f) & 0xffffu;
                    *reinterpret_cast<uint16_t *>(to + p * C::MT * HDP * 2) = (uint16_t)u;
                    left -= unpack2<BF>(u).x;
                }
            } else {
                *reinterpret_cast<uint16_t *>(to) = real && d < hd ? static_cast<const uint16_t *>(a.q)[at + d] : (uint16_t)0;
            }
        }
    }
    __syncthreads();

    const int row_lo = wm * 16 + lane / 4;                 // this thread's rows: row_lo and row_lo + 8
    const int node_lo = (s.first + row_lo) / g.group, node_hi = (s.first + row_lo + 8) / g.group;
    const float f_lo = Ty::F32 ? g.scale2 * row_scale[row_lo] : g.scale2, f_hi = Ty::F32 ? g.scale2 * row_scale[row_lo + 8] : g.scale2;
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
            see_lo = ta_allow(a, s, node_lo, p0);
            see_hi = ta_allow(a, s, node_hi, p0);
        }
        float x_lo = -INFINITY, x_hi = -INFINITY;
        const unsigned w_lo = (unsigned)(see_lo >> (wn * KN + (lane % 4) * 2)), w_hi = (unsigned)(see_hi >> (wn * KN + (lane % 4) * 2));
        const unsigned z_lo = (unsigned)(see_lo >> 32 >> ((lane % 4) * 2)), z_hi = (unsigned)(see_hi >> 32 >> ((lane % 4) * 2));
#pragma unroll
        for (int i = 0; i < NK; ++i) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                sc[i][e] *= f_lo;
                sc[i][2 + e] *= f_hi;
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
        x_lo = fmaxf(x_lo, m_lo);
        x_hi = fmaxf(x_hi, m_hi);
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
                p[e] = ex2(sc[i][e] - u_lo + Ty::LIFT);
                p[2 + e] = ex2(sc[i][2 + e] - u_hi + Ty::LIFT);
                l_lo += p[e];
                l_hi += p[2 + e];
            }
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
    if (WN > 1) {   // join the warps that share the rows, in shared memory
        cp_wait<0>();
        __syncthreads();
        float *jo = reinterpret_cast<float *>(smem + C::Q_BYTES), *jm = jo + WN * C::MT * HDP;   // [WN][MT][HDP], [WN][MT][2]
#pragma unroll
        for (int n = 0; n < ND; ++n) {
            float *p = jo + (size_t)(wn * C::MT + row_lo) * HDP + n * 8 + (lane % 4) * 2;
            *reinterpret_cast<float2 *>(p) = make_float2(o[n][0], o[n][1]);
            *reinterpret_cast<float2 *>(p + 8 * HDP) = make_float2(o[n][2], o[n][3]);
        }
        if (lane % 4 == 0) {
            jm[(wn * C::MT + row_lo) * 2] = m_lo; jm[(wn * C::MT + row_lo) * 2 + 1] = l_lo;
            jm[(wn * C::MT + row_lo + 8) * 2] = m_hi; jm[(wn * C::MT + row_lo + 8) * 2 + 1] = l_hi;
        }
        __syncthreads();
        const size_t part_at = (((size_t)blockIdx.x * a.n_kv_head + kh) * g.nsplit + split) * C::MT;
        float *po = g.part + part_at * HDP, *pm = g.part + (size_t)g.tiles * a.n_kv_head * g.nsplit * C::MT * HDP + part_at * 2;
        for (int r = warp; r < C::MT; r += WM * WN) {
            const int rr = s.first + r, node = rr / g.group;
            if (node >= s.t) continue;
            float m = -INFINITY, f[WN], l = 0.0f;
#pragma unroll
            for (int w = 0; w < WN; ++w) m = fmaxf(m, jm[(w * C::MT + r) * 2]);
            const float u = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int w = 0; w < WN; ++w) {
                f[w] = ex2(jm[(w * C::MT + r) * 2] - u);
                l += jm[(w * C::MT + r) * 2 + 1] * f[w];
            }
            const float inv = splits > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            const size_t at = (size_t)(s.r0 + node) * a.ldo + ((size_t)kh * g.group + rr % g.group) * hd;
            if (splits > 1 && lane == 0) { pm[r * 2] = m; pm[r * 2 + 1] = l; }
            for (int d = lane * 2; d < hd; d += 64) {
                float x = 0.0f, y = 0.0f;
#pragma unroll
                for (int w = 0; w < WN; ++w) {
                    const float2 v = *reinterpret_cast<const float2 *>(jo + (size_t)(w * C::MT + r) * HDP + d);
                    x = fmaf(v.x, f[w], x);
                    y = fmaf(v.y, f[w], y);
                }
                if (splits > 1) *reinterpret_cast<float2 *>(po + (size_t)r * HDP + d) = make_float2(x, y);
                else ta_store2<QT>(a.out, at + d, x * inv, y * inv, false);
            }
        }
        return;
    }
    const size_t part_at = (((size_t)blockIdx.x * a.n_kv_head + kh) * g.nsplit + split) * C::MT;
    float *po = g.part + part_at * HDP, *pm = g.part + (size_t)g.tiles * a.n_kv_head * g.nsplit * C::MT * HDP + part_at * 2;
    const bool pair = ((a.ldo & 1) == 0) && ((reinterpret_cast<uintptr_t>(a.out) & (QT == EC_T_F32 ? 7 : 3)) == 0);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int r = row_lo + 8 * half, rr = s.first + r, node = half ? node_hi : node_lo;
        if (node >= s.t) continue;
        const float m = half ? m_hi : m_lo, l = half ? l_hi : l_lo;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const size_t at = (size_t)(s.r0 + node) * a.ldo + ((size_t)kh * g.group + rr % g.group) * hd;
        if (splits > 1 && lane % 4 == 0) { pm[r * 2] = m; pm[r * 2 + 1] = l; }
#pragma unroll
        for (int n = 0; n < ND; ++n) {
            const int d = n * 8 + (lane % 4) * 2;
            if (d >= hd) continue;
            const float x = o[n][2 * half], y = o[n][2 * half + 1];
            if (splits > 1) *reinterpret_cast<float2 *>(po + (size_t)r * HDP + d) = make_float2(x, y);
            else ta_store2<QT>(a.out, at + d, x * inv, y * inv, pair);
        }
    }
}

// out of a row tile from its splits' (m, l, o), in their order: one warp a row
template <int QT>
__global__ void __launch_bounds__(128) k_tree_join(const ec_kv_pages kv, const ec_tree_attn a, const TaGeo g, int mt, int hdp, int *err) {
    EC_PDL_ENTER();
    TaTile s;
    if (!ta_find(kv, a, g, blockIdx.x, mt, s, err)) return;
    int chunk;
    const int splits = ta_splits(s, g, chunk);
    if (splits <= 1) return;
    const int kh = blockIdx.z, r = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, hd = a.head_dim;
    const int rr = s.first + r, node = rr / g.group;
    if (r >= mt || node >= s.t) return;
    const size_t at = ((size_t)blockIdx.x * a.n_kv_head + kh) * g.nsplit * mt + r;
    const float *po = g.part + at * hdp, *pm = g.part + (size_t)g.tiles * a.n_kv_head * g.nsplit * mt * hdp + at * 2;
    float m = -INFINITY;
    for (int i = lane; i < splits; i += 32) m = fmaxf(m, pm[(size_t)i * mt * 2]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (m == -INFINITY) m = 0.0f;
    float l = 0.0f, acc[8] = {};
    for (int i = 0; i < splits; ++i) {
        const float2 ml = *reinterpret_cast<const float2 *>(pm + (size_t)i * mt * 2);
        const float f = ex2(ml.x - m);
        l = fmaf(ml.y, f, l);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = lane * 2 + 64 * j;
            if (d >= hd) break;
            const float2 v = *reinterpret_cast<const float2 *>(po + (size_t)i * mt * hdp + d);
            acc[2 * j] = fmaf(v.x, f, acc[2 * j]);
            acc[2 * j + 1] = fmaf(v.y, f, acc[2 * j + 1]);
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const size_t to = (size_t)(s.r0 + node) * a.ldo + ((size_t)kh * g.group + rr % g.group) * hd;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int d = lane * 2 + 64 * j;
        if (d < hd) ta_store2<QT>(a.out, to + d, acc[2 * j] * inv, acc[2 * j + 1] * inv, false);
    }
}

// ---- launch --------------------------------------------------------------------

struct TaPlan { int hdp, mt; TaGeo g; size_t bytes; };

int ta_up(int a, int b) { return (a + b - 1) / b; }

// The split: enough CTAs for two per SM where the pages allow it.
TaPlan ta_plan(int n_seq, int rows, int n_head, int n_kv_head, int hd, int max_len, int window, int sms) {
    TaPlan p;
    p.hdp = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
    p.g.group = n_head / n_kv_head;
    const int mean = (int)(((long long)rows * p.g.group + n_seq - 1) / n_seq);
    p.mt = mean <= 16 ? 16 : mean <= 32 ? 32 : 64;
    const long long tiles = ((long long)rows * p.g.group) / p.mt + n_seq;   // every sequence rounds up once
    p.g.tiles = (int)tiles;   // rows * group fits 31 bits
    int pages = ta_up(max_len > 0 ? max_len : 1, PAGE);
    if (window > 0 && pages > window / PAGE + 2) pages = window / PAGE + 2;
    const long long real = (long long)ta_up(mean, p.mt) * n_seq * n_kv_head;
    long long want = (2LL * sms + real - 1) / real;
    if (want > pages) want = pages;
    if (want > 256) want = 256;
    if (want < 1) want = 1;
    p.g.chunk = ta_up(pages, (int)want);
    p.g.nsplit = ta_up(pages, p.g.chunk);
    p.bytes = p.g.nsplit > 1 ? (size_t)p.g.tiles * n_kv_head * p.g.nsplit * p.mt * (p.hdp + 2) * 4 : 0;
    return p;
}

int g_attr[64][64];

template <int QT, int KT, int HDP, int WM, int WN, int STAGES>
int ta_run(const ec_kv_pages &kv, const ec_tree_attn &a, const TaPlan &p, int id, int *err, cudaStream_t stream) {
    typedef TaMma<QT, KT, HDP, WM, WN, STAGES> C;
    static_assert(C::SMEM <= 232448, "shared memory per CTA");
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    auto kern = k_tree_mma<QT, KT, HDP, WM, WN, STAGES>;
    if (!g_attr[id][dev]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return (int)e;
        g_attr[id][dev] = 1;
    }
    kern<<<dim3(p.g.tiles, p.g.nsplit, a.n_kv_head), C::THREADS, C::SMEM, stream>>>(kv, a, p.g, err);
    e = cudaGetLastError();
    if (e != cudaSuccess || p.g.nsplit == 1) return (int)e;
    return (int)ec_launch_k(k_tree_join<QT>, dim3(p.g.tiles, ta_up(p.mt, 4), a.n_kv_head), dim3(128), 0, stream, kv, a, p.g, p.mt, p.hdp, err);
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
    if (p.hdp == 128) return ta_rows<QT, KT, 128, 3>(kv, a, p, id + 3, err, stream);
    return ta_rows<QT, KT, 256, 2>(kv, a, p, id + 6, err, stream);
}

}  // namespace

extern "C" size_t ec_tree_attention_bytes(int n_seq, int rows, int n_head, int n_kv_head, int head_dim, int max_len, int num_sms) {
    return ta_plan(n_seq, rows, n_head, n_kv_head, head_dim, max_len, 0, num_sms).bytes;
}

extern "C" int ec_launch_tree_attention(const ec_kv_pages *kv, const ec_tree_attn *a, int num_sms, int *err, cudaStream_t stream) {
    long long len = a->max_len > 0 ? a->max_len : (long long)kv->pages_per_slot * PAGE;
    TaPlan p = ta_plan(a->n_seq, a->rows, a->n_head, a->n_kv_head, a->head_dim, (int)(len < 0x7fffffff - PAGE ? len : 0x7fffffff - PAGE), a->window, num_sms);
    const size_t one = (size_t)p.g.tiles * a->n_kv_head * p.mt * (p.hdp + 2) * 4;   // partial sums of one split of everything
    if (p.g.nsplit > 1 && (!a->work || a->work_bytes < p.bytes)) {
        const size_t fit = a->work ? a->work_bytes / one : 0;
        const int pages = p.g.chunk * p.g.nsplit;
        p.g.nsplit = fit > 1 ? (int)fit : 1;
        p.g.chunk = ta_up(pages, p.g.nsplit);
    }
    p.g.scale2 = (a->scale > 0.0f ? a->scale : 1.0f / sqrtf((float)a->head_dim)) * LOG2E;
    p.g.part = static_cast<float *>(a->work);
    const bool bf = kv->type == EC_T_BF16;
    if (a->type == EC_T_F32) return bf ? ta_dims<EC_T_F32, EC_T_BF16>(*kv, *a, p, 0, err, stream) : ta_dims<EC_T_F32, EC_T_F16>(*kv, *a, p, 9, err, stream);
    return bf ? ta_dims<EC_T_BF16, EC_T_BF16>(*kv, *a, p, 18, err, stream) : ta_dims<EC_T_F16, EC_T_F16>(*kv, *a, p, 27, err, stream);
}
