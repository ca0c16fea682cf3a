// ec_tree.cuh -- what the kernels of the tree attention share (ec_tree.cu: mma
// tiles of up to 64 rows, ec_tree_tc.cu: tcgen05 tiles of twice 128 rows): how the
// rows and pages of a call are laid out as work, which positions a row sees,
// and small helpers.
#pragma once
#include "ec_common.cuh"
#include "ec_serve.h"

namespace ec_tree {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int PAGE = EC_KV_PAGE;
constexpr int TC_ROWS = 256;            // rows of a tile on tcgen05: two halves of 128

// ---- the work of a call ------------------------------------------------------

struct TaGeo {            // chosen by the launcher
    int group;            // query heads per KV head
    unsigned div_mul;     // row / group = (row * div_mul) >> div_shift for rows below 2^30 (group > 1)
    int div_shift;
    int cluster;          // CTAs of a cluster that share a tile's pages
    float scale2;         // scale * log2 e
    float *part;          // pieces: [CTA][2][MT][hdp] o, then [CTA][2][MT] (m, l)
};

EC_DEV int ta_node(const TaGeo &g, int row) {
    return g.group == 1 ? row : (int)(((unsigned long long)(unsigned)row * g.div_mul) >> g.div_shift);
}

struct TaTile {           // one row tile of one KV head
    int first;            // its first row in the sequence's (node, head) numbering
    int kh;
    int r0, t, base, slot;
    int page0, page1;     // pages that hold visible positions
    int len, step;        // places on the line of pages (TaLine), pages of a place
};

struct TaSeq {            // a sequence, in the lane that holds it
    int r0, t, base, slot, page0, pages, tiles;   // a bad one has no tiles
    int half;             // the last tile has no more than half of the rows (TC_ROWS tiles only)
};

EC_DEV TaSeq ta_seq(const ec_kv_pages &kv, const ec_tree_attn &a, const TaGeo &g, int mt, int i, int *err) {
    TaSeq q = {};
    if (i >= a.n_seq) return q;
    q.r0 = a.row_start[i];
    const long long t = (long long)a.row_start[i + 1] - q.r0;
    q.base = a.base[i];
    q.slot = a.slots ? a.slots[i] : i;
    if (q.r0 < 0 || t < 0 || q.r0 + t > a.rows || q.base < 0 || q.slot < 0 || q.slot >= kv.n_slots ||
        q.base + t > (long long)kv.pages_per_slot * PAGE) {
        atomicCAS(err, 0, EC_KERR_BAD_INDEX);
        return q;
    }
    q.t = (int)t;
    q.tiles = (int)((t * g.group + mt - 1) / mt);
    q.half = mt == TC_ROWS && (int)(t * g.group - (long long)(q.tiles - 1) * mt) <= mt / 2;
    const int lo = a.window > 0 && q.base > a.window ? q.base - a.window : 0;   // no row sees a position below it
    q.page0 = lo / PAGE;
    q.pages = (q.base + q.t + PAGE - 1) / PAGE - q.page0;
    return q;
}

EC_DEV TaTile ta_tile(const TaSeq &q, int l, int tile, int kh, int mt) {   // from the sequence that lane l holds
    TaTile s;
    s.first = tile * mt;
    s.kh = kh;
    s.r0 = __shfl_sync(0xffffffffu, q.r0, l);
    s.t = __shfl_sync(0xffffffffu, q.t, l);
    s.base = __shfl_sync(0xffffffffu, q.base, l);
    s.slot = __shfl_sync(0xffffffffu, q.slot, l);
    s.page0 = __shfl_sync(0xffffffffu, q.page0, l);
    s.page1 = s.page0 + __shfl_sync(0xffffffffu, q.pages, l);
    const bool half = tile == __shfl_sync(0xffffffffu, q.tiles, l) - 1 && __shfl_sync(0xffffffffu, q.half, l);
    s.step = half ? 2 : 1;
    s.len = half ? (s.page1 - s.page0 + 1) / 2 : s.page1 - s.page0;
    return s;
}

EC_DEV int ta_scan(int v) {   // inclusive, over the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if ((int)(threadIdx.x & 31) >= o) v += u;
    }
    return v;
}

// The row tile `ti` in the sequences' order; false when there is none.  Called
// by whole warps.
EC_DEV bool ta_find(const ec_kv_pages &kv, const ec_tree_attn &a, const TaGeo &g, int ti, int kh, int mt, TaTile &s, int *err) {
    int before = 0;
    for (int b0 = 0; b0 < a.n_seq; b0 += 32) {
        const TaSeq q = ta_seq(kv, a, g, mt, b0 + (threadIdx.x & 31), err);
        const int sum = before + ta_scan(q.tiles);
        const unsigned hit = __ballot_sync(0xffffffffu, sum > ti);
        if (hit) {
            const int l = __ffs((int)hit) - 1;
            s = ta_tile(q, l, ti - __shfl_sync(0xffffffffu, sum - q.tiles, l), kh, mt);
            return true;
        }
        before = __shfl_sync(0xffffffffu, sum, 31);
    }
    return false;
}

constexpr unsigned TA_LINE = 1u << 26;   // places of a line, fewer (ta_plan)

// The pages of all tiles in one line: sequence by sequence, KV head by KV head,
// tile by tile; a place on it is a page, or two of them in a tile whose rows are
// half as many.  CTA i of the first n takes [start(i), start(i + 1)), at least
// one place each.
struct TaLine {
    TaSeq head;           // sequence of this lane among the first 32
    int n, total, per, more;   // the first `more` pieces have per + 1 places

    EC_DEV static int head_work(const TaSeq &q) { return q.tiles * q.pages - (q.half ? q.pages / 2 : 0); }   // of one KV head
    EC_DEV static int work(const TaSeq &q, int kvh) { return head_work(q) * kvh; }
    EC_DEV void init(const ec_kv_pages &kv, const ec_tree_attn &a, const TaGeo &g, int mt, int pieces, int *err) {
        head = ta_seq(kv, a, g, mt, threadIdx.x & 31, err);
        unsigned all = __reduce_add_sync(0xffffffffu, (unsigned)work(head, a.n_kv_head));   // 32 of less than TA_LINE fit 32 bits
        for (int b0 = 32; b0 < a.n_seq; b0 += 32)
            all = min(all, (unsigned)TA_LINE) + __reduce_add_sync(0xffffffffu, (unsigned)work(ta_seq(kv, a, g, mt, b0 + (threadIdx.x & 31), err), a.n_kv_head));
        // row_start that falls (ta_seq reports it) and rises again counts rows more than once: a line that no plan allows is empty
        total = all < TA_LINE ? (int)all : 0;
        n = min(pieces, total);
        per = n ? total / n : 0;
        more = total - per * n;
    }
    EC_DEV int start(int i) const { return per * i + min(i, more); }
    EC_DEV int piece(int at) const {
        const int wide = (per + 1) * more;
        return at < wide ? at / (per + 1) : more + (at - wide) / per;
    }
    // the tile that holds place `at` (below total), and where it begins
    EC_DEV TaTile tile(const ec_kv_pages &kv, const ec_tree_attn &a, const TaGeo &g, int mt, int at, int &begin, int *err) const {
        int before = 0;
        TaSeq q = head;
        for (int b0 = 0;; b0 += 32) {
            if (b0) q = ta_seq(kv, a, g, mt, b0 + (threadIdx.x & 31), err);
            const int w = work(q, a.n_kv_head), sum = before + ta_scan(w);
            const unsigned hit = __ballot_sync(0xffffffffu, sum > at);
            if (hit || b0 + 32 >= a.n_seq) {
                const int l = hit ? __ffs((int)hit) - 1 : 0;
                const int from = __shfl_sync(0xffffffffu, sum - w, l);
                const int pages = max(1, __shfl_sync(0xffffffffu, q.pages, l)), tiles = max(1, __shfl_sync(0xffffffffu, q.tiles, l));
                const int each = max(1, __shfl_sync(0xffffffffu, head_work(q), l));
                const int kh = (at - from) / each, tile = min((at - from - kh * each) / pages, tiles - 1);
                begin = from + kh * each + tile * pages;
                return ta_tile(q, l, tile, kh, mt);
            }
            before = __shfl_sync(0xffffffffu, sum, 31);
        }
    }
    // the tile number `index` of all, in the order of the line; false: none
    EC_DEV bool by_index(const ec_kv_pages &kv, const ec_tree_attn &a, const TaGeo &g, int mt, int index, TaTile &s, int &begin, int *err) const {
        int units = 0, before = 0;
        TaSeq q = head;
        for (int b0 = 0; b0 < a.n_seq; b0 += 32) {
            if (b0) q = ta_seq(kv, a, g, mt, b0 + (threadIdx.x & 31), err);
            const int w = work(q, a.n_kv_head), u = q.tiles * a.n_kv_head, ws = before + ta_scan(w), us = units + ta_scan(u);
            const unsigned hit = __ballot_sync(0xffffffffu, us > index);
            if (hit) {
                const int l = __ffs((int)hit) - 1, unit = index - __shfl_sync(0xffffffffu, us - u, l);
                const int tiles = __shfl_sync(0xffffffffu, q.tiles, l), kh = unit / tiles;
                begin = __shfl_sync(0xffffffffu, ws - w, l) + kh * __shfl_sync(0xffffffffu, head_work(q), l) +
                        (unit - kh * tiles) * __shfl_sync(0xffffffffu, q.pages, l);
                s = ta_tile(q, l, unit - kh * tiles, kh, mt);
                return true;
            }
            before = __shfl_sync(0xffffffffu, ws, 31);
            units = __shfl_sync(0xffffffffu, us, 31);
        }
        return false;
    }
};

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
// sees, one bit each, but for what a window hides of the tree itself.
EC_DEV unsigned long long ta_see(const ec_tree_attn &a, const TaTile &s, int i, int p0, int depth) {
    if (i >= s.t) return 0ull;
    const int j0 = p0 - s.base;
    const unsigned long long *m = a.mask + (size_t)(s.r0 + i) * a.mask_words;
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
    return (a.window > 0 ? prefix & ~ta_low(s.base + depth - a.window + 1 - p0) : prefix) | tree;
}

// A window hides nodes from each other only if it is no longer than two depths
// can be apart: a row of all bits has 64 words - 1, one of none has -1.
EC_DEV bool ta_short_window(const ec_tree_attn &a) { return a.window > 0 && a.window <= 64ll * a.mask_words; }

// The same with the window applied to the tree too.
EC_DEV unsigned long long ta_allow(const ec_tree_attn &a, const TaTile &s, int i, int p0) {
    if (i >= s.t) return 0ull;
    const int depth = a.window > 0 ? ta_depth(a, s.r0 + i) : 0;
    unsigned long long see = ta_see(a, s, i, p0, depth);
    if (ta_short_window(a))
        for (unsigned long long left = see & ~ta_low(s.base - p0); left; left &= left - 1) {
            const int bit = __ffsll((long long)left) - 1;
            if (ta_depth(a, s.r0 + p0 - s.base + bit) < depth - a.window + 1) see &= ~(1ull << bit);
        }
    return see;
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

EC_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

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

// tcgen05 tiles (ec_tree_tc.cu): whether they take a call of this kind, and
// the launch of its pieces (one per resident CTA of `pieces`).
bool ta_tc_takes(int q_type, int kv_type, int hd);
int ta_tc_launch(const ec_kv_pages &kv, const ec_tree_attn &a, const TaGeo &g, int pieces, int *err, cudaStream_t stream);

}  // namespace ec_tree

using namespace ec_tree;
