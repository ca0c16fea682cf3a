// ec_sample.cu -- drawing one token per row of logits (ec_sample).
//
// Weights w = 2^((logit - max) log2(e) / T) are held as integers, w rounded to
// a multiple of 2^-shift, shift = min(50, 62 - ceil(log2 vocab)): every sum of
// a row's weights fits 64 bits and is exact, so it depends on neither the
// order of its terms (atomics included) nor on how a row is cut.
//
// Candidates are ordered by (logit, then lowest index).  Top-k and top-p are
// cuts in that order, found without sorting the row: a histogram over max -
// logit gives the bin in which the running count or weight crosses, and only
// the candidates of that bin are sorted; a bin of more than SA_LIST of them
// (equal logits) is first cut down by the bits of their order.  A top-k of up
// to SA_LIST candidates is gathered whole and handled from the sorted list.
#include "ec_common.cuh"
#include "ec_serve.h"

#include <cooperative_groups.h>
#include <float.h>

namespace cg = cooperative_groups;

namespace {

typedef unsigned long long u64;
constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / 32;
constexpr int SA_BINS = 1024, SA_LIST = 2048, SA_PER = SA_LIST / SA_THREADS;
constexpr int SA_TAB = 512;                       // entries of the 2^(j/512) table
constexpr int SA_MAX_CTAS = 16;

template <int T> struct SaElt { typedef float V; };
template <> struct SaElt<EC_T_F16> { typedef uint16_t V; };
template <> struct SaElt<EC_T_BF16> { typedef uint16_t V; };

template <int T> EC_DEV float sa_value(typename SaElt<T>::V v) {
    if constexpr (T == EC_T_F32) return v;
    else return ec_h2f(v, T == EC_T_BF16);
}

// Position of a candidate in the order, larger first: order-preserving bits of
// the logit (-0 as +0), then the lower index.
EC_DEV u64 sa_rank(float v, int i) {
    const uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);
    return (u64)((b & 0x80000000u) ? ~b : (b | 0x80000000u)) << 32 | (uint32_t)~i;
}
EC_DEV float sa_rank_value(u64 r) {
    const uint32_t k = (uint32_t)(r >> 32);
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
EC_DEV int sa_rank_index(u64 r) { return (int)~(uint32_t)r; }

struct SaCtl {                 // what the first CTA tells the others
    int bin, crowd;            // crossing bin (-1: none), candidates in it
    u64 above;                 // count or weight before it
    u64 want;                  // what has to be reached
    u64 cut;                   // rank of the last candidate kept
    int at[SA_MAX_CTAS];       // where each CTA's candidates go in the list
};

struct SaShared {
    double tab[SA_TAB];        // 2^(j / 512)
    u64 part[SA_WARPS + 1];
    u64 sums[SA_MAX_CTAS];     // each CTA's weight
    float high[SA_MAX_CTAS], low[SA_MAX_CTAS];
    int first[SA_MAX_CTAS];
    float red[2 * SA_WARPS];
    int count, found;
    SaCtl ctl;
    u64 bar;
    union {
        struct { uint32_t count[SA_BINS], limb[3][SA_BINS]; } h;   // weights in 16-bit limbs
        struct { u64 rank[SA_LIST], w[SA_LIST]; } l;
    };
};

// w(v) * 2^shift in double, not yet rounded to an integer.  With t = 512 (v -
// max) log2(e) / T = j + f, |f| <= 1/2: 2^(t/512) = 2^(j div 512) tab[j mod
// 512] e^(f ln 2 / 512), the last as its Taylor sum to the third power
// (0.00068^4 / 24 = 2^-46.7 of it is left out).  0 for v below `floor`, where
// it is less than 2^-(shift + 2), and for NaN.
struct SaWeight {
    double mx, c;              // c: 512 log2(e) / T
    float floor;
    int shift;
    const double *tab;
    EC_DEV double operator()(float v) const {
        if (!(v >= floor)) return 0.0;
        const double magic = 6755399441055744.0;      // 1.5 * 2^52
        const double d = (double)v - mx;
        const double kd = __fma_rn(d, c, magic);
        const int j = __double2loint(kd);
        const double f = __fma_rn(d, c, magic - kd);
        double p = __fma_rn(f, 4.1353783506767136e-10, 9.163913992275265e-7);   // (ln2 / 512)^n / n!
        p = __fma_rn(f, p, 1.3538030870311431e-3);
        p = __fma_rn(f, p, 1.0);
        const double s = p * tab[j & (SA_TAB - 1)];
        return __hiloint2double(__double2hiint(s) + (((j >> 9) + shift) << 20), __double2loint(s));
    }
    // A weight (below 2^52) rounded to nearest, plus RAW: sums of these wrap
    // and are put right by the number of terms.
    static constexpr u64 RAW = 0x4330000000000000ull;
    static EC_DEV u64 raw(double w) { return (u64)__double_as_longlong(w + 4503599627370496.0); }
    static EC_DEV u64 whole(double w) { return raw(w) - RAW; }
};

EC_DEV u64 sa_warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum of v over the threads before this one; `total` gets the CTA's sum.
EC_DEV u64 sa_scan(u64 v, SaShared &s, u64 &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 u = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += u;
    }
    __syncthreads();
    if (lane == 31) s.part[warp] = sum;
    __syncthreads();
    u64 before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < SA_WARPS; ++w) {
        if (w == warp) before = total;
        total += s.part[w];
    }
    return before + sum - v;
}

// Sort list[0, n) (n a power of two), largest first.
EC_DEV void sa_sort(u64 *list, int n) {
    for (int k = 2; k <= n; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int p = threadIdx.x; p < n / 2; p += SA_THREADS) {
                const int i = 2 * p - (p & (j - 1)), o = i + j;
                const u64 a = list[i], b = list[o];
                if ((a < b) == ((i & k) == 0)) { list[i] = b; list[o] = a; }
            }
        }
    __syncthreads();
}

EC_DEV int sa_pow2(int n) { return n <= 1 ? 1 : 1 << (32 - __clz(n - 1)); }

// A CTA's share of a row in shared memory, in whole 16-byte blocks; places
// that are not the row's hold -inf.
template <int T> struct SaRow {
    typedef typename SaElt<T>::V V;
    static constexpr int ELT = sizeof(V), PER = 16 / ELT;
    SaShared &s;
    const uint4 *blocks;
    int n, ibase;              // blocks; index in the row of place 0
    SaWeight weight;
    float mx, per_bin;
    float cut_v;               // kept: larger, or equal and up to index cut_i
    int cut_i;
    bool cut;

    EC_DEV float at(int place) const { return sa_value<T>(reinterpret_cast<const V *>(blocks)[place]); }
    EC_DEV bool kept(float v, int place) const { return v > cut_v || (v == cut_v && place + ibase <= cut_i); }
    EC_DEV int bin(float v) const { return min((int)(fminf(mx - v, FLT_MAX) * per_bin), SA_BINS - 1); }   // of v >= weight.floor

    // f(value, place) for blocks [b0, b1), taken by threads t of `threads`
    template <typename F> EC_DEV void each(int b0, int b1, int t, int threads, F f) const {
#pragma unroll 2
        for (int b = b0 + t; b < b1; b += threads) {
            const uint4 u = blocks[b];
            if constexpr (T == EC_T_F32) {
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) f(__uint_as_float(w[j]), b * 4 + j);
            } else {
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int j = 0; j < 8; ++j) f(ec_h2f((uint16_t)(w[j / 2] >> (16 * (j % 2))), T == EC_T_BF16), b * 8 + j);
            }
        }
    }
    // Raw weights (SaWeight::raw) of what is kept and weighs at least `least`,
    // summed; `terms` counts them.
    template <bool CUT, bool LEAST> EC_DEV u64 sum(int b0, int b1, int t, int threads, double least) const {
        u64 raw = 0;
        int terms = 0;
        each(b0, b1, t, threads, [&](float v, int p) {
            if (CUT && !kept(v, p)) return;
            const double w = weight(v);
            if (LEAST && !(w >= least)) return;
            raw += SaWeight::raw(w);
            ++terms;
        });
        return raw - (u64)terms * SaWeight::RAW;
    }
    EC_DEV u64 sum(int b0, int b1, int t, int threads, double least) const {
        return least > 0.0 ? (cut ? sum<true, true>(b0, b1, t, threads, least) : sum<false, true>(b0, b1, t, threads, least))
                           : (cut ? sum<true, false>(b0, b1, t, threads, least) : sum<false, false>(b0, b1, t, threads, least));
    }
};

// Finds the candidate at which the running count (MASS: weight, among those
// kept so far) over the order reaches what is wanted, and cuts there.  With
// `whole`, everything up to it may be left unsorted in the first CTA's list
// instead, each CTA's number in its `first`; returns true then.  All CTAs of
// the cluster call it alike.
template <bool MASS, int T>
EC_DEV bool sa_select(cg::cluster_group &cl, SaRow<T> &row, u64 want, float top_p, bool whole) {
    SaShared &s = row.s;
    const int ctas = (int)cl.num_blocks(), me = (int)cl.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    u64 above = 0, prefix = 0;
    int bits = 64, bin = -1;   // from the second round: candidates of `bin` whose rank's top 64 - bits bits are `prefix`
    const float floor = row.weight.floor;
    auto in_class = [&](float v, int p) {
        if (!(v >= floor) || row.bin(v) != bin || (MASS && row.cut && !row.kept(v, p))) return false;
        return bits == 64 || (sa_rank(v, p + row.ibase) >> bits) == prefix;
    };
    for (;;) {
        __syncthreads();
        for (int b = tid; b < SA_BINS; b += SA_THREADS) s.h.count[b] = s.h.limb[0][b] = s.h.limb[1][b] = s.h.limb[2][b] = 0;
        if (tid == 0) s.count = 0;
        __syncthreads();
        const int step = bits - 10 > 0 ? bits - 10 : 0;
        auto add = [&](float v, int b) {
            atomicAdd(&s.h.count[b], 1u);
            if (MASS) {
                const u64 w = SaWeight::whole(row.weight(v));
                if (w & 0xffff) atomicAdd(&s.h.limb[0][b], (uint32_t)(w & 0xffff));
                if (w >> 16 & 0xffff) atomicAdd(&s.h.limb[1][b], (uint32_t)(w >> 16 & 0xffff));
                if (w >> 32) atomicAdd(&s.h.limb[2][b], (uint32_t)(w >> 32));
            }
        };
        if (bin < 0)
            row.each(0, row.n, tid, SA_THREADS, [&](float v, int p) {
                if (v >= floor && (!MASS || !row.cut || row.kept(v, p))) add(v, row.bin(v));
            });
        else
            row.each(0, row.n, tid, SA_THREADS, [&](float v, int p) {
                if (in_class(v, p)) add(v, SA_BINS - 1 - (int)((sa_rank(v, p + row.ibase) >> step) & (SA_BINS - 1)));
            });
        cl.sync();
        if (me == 0) {   // join the histograms, find the crossing
            u64 cnt[2] = {0, 0}, sum[2] = {0, 0};
            for (int c = 0; c < ctas; ++c) {
                const SaShared *o = cl.map_shared_rank(&s, c);
                const uint2 q = reinterpret_cast<const uint2 *>(o->h.count)[tid];
                cnt[0] += q.x;
                cnt[1] += q.y;
                if (MASS)
#pragma unroll
                    for (int l = 0; l < 3; ++l) {
                        const uint2 m = reinterpret_cast<const uint2 *>(o->h.limb[l])[tid];
                        sum[0] += (u64)m.x << (16 * l);
                        sum[1] += (u64)m.y << (16 * l);
                    }
            }
            if (!MASS) { sum[0] = cnt[0]; sum[1] = cnt[1]; }
            u64 total;
            u64 before = above + sa_scan(sum[0] + sum[1], s, total);
            if (MASS && bin < 0) want = max(1ull, min(total, (u64)ceil((double)top_p * (double)total)));
            if (tid == 0) s.ctl.bin = -1;
            __syncthreads();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                if (before < want && before + sum[q] >= want) {
                    s.ctl.bin = 2 * tid + q;
                    s.ctl.crowd = (int)cnt[q];
                    s.ctl.above = before;
                    s.ctl.want = want;
                }
                before += sum[q];
            }
            __syncthreads();
            // all up to the crossing, where they fit the list and it is asked for
            const bool all = whole && bin < 0 && s.ctl.bin >= 0 && s.ctl.above + s.ctl.crowd <= SA_LIST;
            if (warp == 0) {
                int c = 0;
                if (lane < ctas && s.ctl.bin >= 0 && !all) c = (int)cl.map_shared_rank(&s, lane)->h.count[s.ctl.bin];
                int sum32 = c;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int u = __shfl_up_sync(0xffffffffu, sum32, o);
                    if (lane >= o) sum32 += u;
                }
                if (lane < ctas) s.ctl.at[lane] = all ? -1 : sum32 - c;
            }
            __syncthreads();
            if (tid < ctas) cl.map_shared_rank(&s, tid)->ctl = s.ctl;
        }
        cl.sync();
        const int crossing = s.ctl.bin, crowd = s.ctl.crowd, place = s.ctl.at[me];
        if (crossing < 0) return false;   // fewer than wanted have any weight: nothing to cut
        want = s.ctl.want;
        above = s.ctl.above;
        u64 *list = cl.map_shared_rank(&s, 0)->l.rank;
        if (place < 0) {                  // everything up to the crossing goes to the list
            int c = 0;
            for (int b = tid; b <= crossing; b += SA_THREADS) c += (int)s.h.count[b];
            u64 total;
            sa_scan((u64)c, s, total);
            if (tid == 0) cl.map_shared_rank(&s, 0)->first[me] = (int)total;
            cl.sync();
            int at = 0;
            for (int q = 0; q < me; ++q) at += cl.map_shared_rank(&s, 0)->first[q];
            row.each(0, row.n, tid, SA_THREADS, [&](float v, int p) {
                if (v >= floor && row.bin(v) <= crossing) list[at + atomicAdd(&s.count, 1)] = sa_rank(v, p + row.ibase);
            });
            cl.sync();
            return true;
        }
        if (bin < 0) {
            bin = crossing;
        } else {
            prefix = prefix << (bits - step) | ((u64)(SA_BINS - 1 - crossing) & ((1ull << (bits - step)) - 1));
            bits = step;
        }
        if (crowd > SA_LIST) continue;
        row.each(0, row.n, tid, SA_THREADS, [&](float v, int p) {
            if (in_class(v, p)) list[place + atomicAdd(&s.count, 1)] = sa_rank(v, p + row.ibase);
        });
        cl.sync();
        if (me == 0) {
            const int size = sa_pow2(crowd);
            for (int i = tid; i < size; i += SA_THREADS)
                if (i >= crowd) s.l.rank[i] = 0;
            sa_sort(s.l.rank, size);
            u64 w[SA_PER], sum = 0, total;
#pragma unroll
            for (int j = 0; j < SA_PER; ++j) {
                const int i = tid * SA_PER + j;
                w[j] = i >= crowd ? 0ull : MASS ? SaWeight::whole(row.weight(sa_rank_value(s.l.rank[i]))) : 1ull;
                sum += w[j];
            }
            u64 before = above + sa_scan(sum, s, total);
#pragma unroll
            for (int j = 0; j < SA_PER; ++j) {
                if (before < want && before + w[j] >= want) s.ctl.cut = s.l.rank[tid * SA_PER + j];
                before += w[j];
            }
            __syncthreads();
            if (tid < ctas) cl.map_shared_rank(&s, tid)->ctl.cut = s.ctl.cut;
        }
        cl.sync();
        row.cut = true;
        row.cut_v = sa_rank_value(s.ctl.cut);
        row.cut_i = sa_rank_index(s.ctl.cut);
        return false;
    }
}

// The point u of a sum of whole weights: the running sum has to exceed it.
EC_DEV u64 sa_point(float u, u64 total) {
    const double x = u > 0.0f ? (double)u * (double)total : 0.0;
    return x >= (double)total ? total - 1 : min((u64)x, total - 1);
}

// The draw from the first CTA's list of `size` candidates, of which the first
// top_k in the order count.
template <int T>
EC_DEV void sa_draw_list(const ec_sample_args &a, SaRow<T> &row, int r, int size, int top_k, float top_p, double least) {
    SaShared &s = row.s;
    const int tid = threadIdx.x, full = sa_pow2(size);
    for (int i = tid; i < full; i += SA_THREADS)
        if (i >= size) s.l.rank[i] = 0;
    sa_sort(s.l.rank, full);
    u64 w[SA_PER], sum = 0, total;
    double wd[SA_PER];
#pragma unroll
    for (int j = 0; j < SA_PER; ++j) {
        const int i = tid * SA_PER + j;
        wd[j] = i < top_k && i < size ? row.weight(sa_rank_value(s.l.rank[i])) : 0.0;
        w[j] = SaWeight::whole(wd[j]);
        sum += w[j];
    }
    u64 before = sa_scan(sum, s, total);
    const u64 want = top_p < 1.0f ? max(1ull, min(total, (u64)ceil((double)top_p * (double)total))) : total;
    u64 kept = 0;
#pragma unroll
    for (int j = 0; j < SA_PER; ++j) {   // kept: what comes before `want` is reached, and weighs enough
        const int i = tid * SA_PER + j;
        const bool keep = w[j] > 0 && before < want && (wd[j] >= least || i == 0);
        before += w[j];
        kept += keep ? w[j] : 0ull;
        s.l.w[i] = (u64)__double_as_longlong(wd[j]);
        s.l.rank[i] = keep ? (u64)(uint32_t)~sa_rank_index(s.l.rank[i]) << 32 | (uint32_t)i : 0ull;   // lowest index largest
    }
    sa_scan(kept, s, total);
    const int most = sa_pow2(min(size, top_k));
    sa_sort(s.l.rank, most);
    const u64 target = sa_point(a.u[r], total);
    sum = 0;
#pragma unroll
    for (int j = 0; j < SA_PER; ++j) {
        const int i = tid * SA_PER + j;
        const u64 k = i < most ? s.l.rank[i] : 0ull;
        wd[j] = k ? __longlong_as_double((long long)s.l.w[(uint32_t)k]) : 0.0;
        w[j] = SaWeight::whole(wd[j]);
        sum += w[j];
    }
    u64 all;
    before = sa_scan(sum, s, all);
#pragma unroll
    for (int j = 0; j < SA_PER; ++j) {
        if (before <= target && target < before + w[j]) {
            a.ids[r] = (int)~(uint32_t)(s.l.rank[tid * SA_PER + j] >> 32);
            if (a.prob) a.prob[r] = (float)(wd[j] / (double)total);
        }
        before += w[j];
    }
}

// One cluster of CTAs per row: each keeps its share of the row in shared
// memory, so that the logits are read from HBM once.
template <int T>
__global__ void __launch_bounds__(SA_THREADS, 2) k_sample(const ec_sample_args a, int shift, int share, int *err) {
    EC_PDL_ENTER();
    typedef SaRow<T> Row;
    typedef typename Row::V V;
    constexpr int ELT = Row::ELT, PER = Row::PER;
    extern __shared__ __align__(128) unsigned char smem[];
    SaShared &s = *reinterpret_cast<SaShared *>(smem);
    V *vals = reinterpret_cast<V *>(smem + (sizeof(SaShared) + 127) / 128 * 128);
    cg::cluster_group cl = cg::this_cluster();
    const int ctas = (int)cl.num_blocks(), me = (int)cl.block_rank();
    const int r = (int)blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float temperature = a.temperature ? a.temperature[r] : 1.0f, min_p = a.min_p ? a.min_p[r] : 0.0f, top_p = a.top_p ? a.top_p[r] : 1.0f;
    const int top_k = a.top_k ? a.top_k[r] : 0;

    // Shares are cut at 16-byte blocks of memory: element i of the row is
    // element i + skew of the block that holds its first one.
    const V *src = static_cast<const V *>(a.logits) + (size_t)r * a.ld;
    const int skew = (int)((reinterpret_cast<uintptr_t>(src) & 15) / ELT);
    const long long lo = max((long long)me * share, (long long)skew), hi = min((long long)(me + 1) * share, (long long)skew + a.vocab);
    const int n = (int)max(0ll, hi - lo), off = n > 0 ? (int)(lo - (long long)me * share) : 0, i0 = (int)(lo - skew);   // vals[off + e] is element i0 + e
    const int blocks = (off + n + PER - 1) / PER;
    {
        // blocks wholly inside the row by one bulk copy, the rest element by element
        const int b0 = (off + PER - 1) / PER * PER, b1 = (off + n) / PER * PER;
        const bool bulk = b1 > b0;
        uint64_t *bar = reinterpret_cast<uint64_t *>(&s.bar);
        if (tid == 0) {
            ec_mbar_init(bar, 1);
            ec_fence_mbar_init();
            if (bulk) {
                ec_mbar_expect_tx(bar, (uint32_t)((b1 - b0) * ELT));
                ec_bulk_g2s(vals + b0, src + i0 + (b0 - off), (uint32_t)((b1 - b0) * ELT), bar);
            }
        }
        for (int e = tid; e < blocks * PER; e += SA_THREADS) {
            if (bulk && e >= b0 && e < b1) {
                if (e + SA_THREADS < b1) e += (b1 - 1 - e) / SA_THREADS * SA_THREADS - SA_THREADS;
                continue;
            }
            vals[e] = e >= off && e < off + n ? src[i0 + e - off] : (V)(T == EC_T_F32 ? -INFINITY : T == EC_T_F16 ? 0xfc00 : 0xff80);
        }
        for (int j = tid; j < SA_TAB; j += SA_THREADS) s.tab[j] = exp2((double)j / SA_TAB);
        __syncthreads();
        if (bulk) ec_mbar_wait(bar, 0, err);   // a wait that gave up is reported; the row's result is then void
    }
    Row row = {s, reinterpret_cast<const uint4 *>(vals), blocks, i0 - off};

    // largest logit and, where the range of a histogram needs it, the smallest
    const bool cuts = top_k > 0 || top_p < 1.0f;
    float mx = -INFINITY, mn = INFINITY;
    if (cuts)
        row.each(0, blocks, tid, SA_THREADS, [&](float v, int) {
            mx = fmaxf(mx, v);
            if (fabsf(v) < INFINITY) mn = fminf(mn, v);
        });
    else
        row.each(0, blocks, tid, SA_THREADS, [&](float v, int) { mx = fmaxf(mx, v); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    }
    if (lane == 0) { s.red[warp] = mx; s.red[SA_WARPS + warp] = mn; }
    __syncthreads();
    for (int w = 0; w < SA_WARPS; ++w) { mx = fmaxf(mx, s.red[w]); mn = fminf(mn, s.red[SA_WARPS + w]); }
    cl.sync();   // every CTA of the cluster has started: its shared memory may be written
    if (tid < ctas) {
        SaShared *o = cl.map_shared_rank(&s, tid);
        o->high[me] = mx;
        o->low[me] = mn;
    }
    cl.sync();
    for (int c = 0; c < ctas; ++c) { mx = fmaxf(mx, s.high[c]); mn = fminf(mn, s.low[c]); }

    if (mx == -INFINITY) {
        if (me == 0 && tid == 0) {
            a.ids[r] = -1;
            if (a.prob) a.prob[r] = 0.0f;
        }
        return;
    }
    if (!(temperature > 0.0f) || min_p > 1.0f || top_k == 1 || top_p <= 0.0f) {   // one candidate is left: the first of the largest
        int first = 0x7fffffff;
        row.each(0, blocks, tid, SA_THREADS, [&](float v, int p) {
            if (v == mx) first = min(first, p + row.ibase);
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
        __syncthreads();
        if (lane == 0) s.red[warp] = __int_as_float(first);
        __syncthreads();
        for (int w = 0; w < SA_WARPS; ++w) first = min(first, __float_as_int(s.red[w]));
        if (tid == 0) cl.map_shared_rank(&s, 0)->first[me] = first;
        cl.sync();
        if (me == 0 && tid == 0) {
            for (int c = 0; c < ctas; ++c) first = min(first, s.first[c]);
            a.ids[r] = first;
            if (a.prob) a.prob[r] = 1.0f;
        }
        return;
    }
    if (mx == INFINITY) {   // logits of +inf weigh the same, all others nothing
        for (int e = tid; e < blocks * PER; e += SA_THREADS)
            vals[e] = sa_value<T>(vals[e]) == INFINITY ? (V)0 : (V)(T == EC_T_F32 ? -INFINITY : T == EC_T_F16 ? 0xfc00 : 0xff80);
        __syncthreads();
        mx = mn = 0.0f;
    }
    // Below `vanish` from the largest a weight is 0: only what lies above is
    // ever a candidate.  (floor is the smallest float from there on.)
    const double vanish = (double)temperature * 0.6931471805599453 * (shift + 3);
    const float floor = fmaxf(__double2float_ru((double)mx - vanish), -FLT_MAX);
    row.weight = {(double)mx, 512.0 * 1.4426950408889634 / (double)temperature, floor, shift, s.tab};
    row.mx = mx;
    row.per_bin = (float)SA_BINS / fmaxf(fminf(mx - floor, mx - mn), 1e-30f);
    row.cut_v = -INFINITY;
    row.cut_i = 0x7fffffff;
    row.cut = false;
    const double least = min_p > 0.0f ? (double)min_p * (double)(1ull << shift) : 0.0;

    if (top_k > 0 && top_k < a.vocab && sa_select<false>(cl, row, (u64)top_k, top_p, top_k <= SA_LIST / 2)) {
        if (me != 0) return;
        int size = 0;
        for (int c = 0; c < ctas; ++c) size += s.first[c];
        sa_draw_list(a, row, r, size, top_k, top_p, least);
        return;
    }
    if (top_p < 1.0f) sa_select<true>(cl, row, 0ull, top_p, false);

    // Weights of the kept candidates in vocabulary order: of each warp's
    // contiguous piece, of the CTAs, then of the piece that holds the point.
    const int piece = (blocks + SA_WARPS - 1) / SA_WARPS;
    const u64 part = sa_warp_sum(row.sum(warp * piece, min(blocks, (warp + 1) * piece), lane, 32, least));
    __syncthreads();
    if (lane == 0) s.part[warp] = part;
    __syncthreads();
    u64 total = 0;
    for (int w = 0; w < SA_WARPS; ++w) total += s.part[w];
    if (tid < ctas) cl.map_shared_rank(&s, tid)->sums[me] = total;
    cl.sync();
    u64 before = 0;
    total = 0;
    for (int c = 0; c < ctas; ++c) {
        if (c == me) before = total;
        total += s.sums[c];
    }
    const u64 target = sa_point(a.u[r], total);
    if (target < before || target >= before + s.sums[me]) return;
    int w = 0;
    while (before + s.part[w] <= target) before += s.part[w++];
    const int end = min(blocks, (w + 1) * piece) * PER;
    for (int p0 = w * piece * PER; p0 < end; p0 += SA_THREADS) {
        const int p = p0 + tid;
        const float v = p < end ? row.at(p) : -INFINITY;
        const double x = !row.cut || row.kept(v, p) ? row.weight(v) : 0.0;
        const u64 mine = x >= least ? SaWeight::whole(x) : 0ull;
        u64 all;
        const u64 start = before + sa_scan(mine, s, all);
        if (start <= target && target < start + mine) {
            a.ids[r] = p + row.ibase;
            if (a.prob) a.prob[r] = (float)(x / (double)total);
        }
        before += all;
    }
}

int g_sample_attr[3][64];

template <int T>
int sa_launch(const ec_sample_args &a, int num_sms, int *err, cudaStream_t stream) {
    constexpr int ELT = T == EC_T_F32 ? 4 : 2, PER16 = 16 / ELT;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (!g_sample_attr[T][dev]) {
        e = cudaFuncSetAttribute(k_sample<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(k_sample<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return (int)e;
        g_sample_attr[T][dev] = 1;
    }
    int bits = 0;
    while ((1ll << bits) < a.vocab) ++bits;
    const int shift = 62 - bits < 50 ? 62 - bits : 50;
    const size_t fixed = (sizeof(SaShared) + 127) / 128 * 128;
    int ctas = 1;
    auto share_of = [&](int c) { return (int)(((long long)a.vocab + 2 * PER16 + c - 1) / c + PER16 - 1) / PER16 * PER16; };
    auto fits = [&](int c, size_t room) { return fixed + (size_t)share_of(c) * ELT <= room; };
    while (ctas < SA_MAX_CTAS && (!fits(ctas, 112 * 1024) || ((long long)a.rows * ctas < 2 * num_sms && a.vocab / ctas > 4096))) ctas *= 2;
    if (!fits(ctas, 232448)) return (int)cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * ctas));
    cfg.blockDim = dim3(SA_THREADS);
    cfg.dynamicSmemBytes = fixed + (size_t)share_of(ctas) * ELT;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)ctas;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, k_sample<T>, a, shift, share_of(ctas), err);
}

}  // namespace

extern "C" int ec_launch_sample(const ec_sample_args *a, int num_sms, int *err, cudaStream_t stream) {
    if (a->type == EC_T_F32) return sa_launch<EC_T_F32>(*a, num_sms, err, stream);
    if (a->type == EC_T_F16) return sa_launch<EC_T_F16>(*a, num_sms, err, stream);
    return sa_launch<EC_T_BF16>(*a, num_sms, err, stream);
}
