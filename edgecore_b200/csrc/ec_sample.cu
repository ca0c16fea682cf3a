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
constexpr int SA_TAB = 128;                       // entries of the 2^(j/128) table
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
    double tab[SA_TAB];        // 2^(j / 128)
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

// w(v) * 2^shift in double, not yet rounded to an integer.  With t = (v - max)
// log2(e) / T = j/128 + f, |f| <= 1/256: 2^t = 2^(j div 128) tab[j mod 128]
// e^(f ln 2), the last as its Taylor sum to the fourth power (0.0028^5 / 120,
// 2^-49 of it).  Below 2^-(shift + 2) it is 0, and so it is for NaN.
struct SaWeight {
    double mx, c;
    int shift;
    const double *tab;
    EC_DEV double operator()(float v) const {
        const double t = ((double)v - mx) * c;
        if (!(t >= -(double)(shift + 2))) return 0.0;
        const double magic = 6755399441055744.0;      // 1.5 * 2^52
        const double kd = __fma_rn(t, 128.0, magic);
        const int j = __double2loint(kd);
        const double f = __fma_rn(kd - magic, -1.0 / 128.0, t);
        double p = __fma_rn(f, 9.618129107628477e-3, 5.550410866482158e-2);   // ln2^n / n!
        p = __fma_rn(f, p, 2.402265069591007e-1);
        p = __fma_rn(f, p, 6.931471805599453e-1);
        p = __fma_rn(f, p, 1.0);
        const double s = p * tab[j & (SA_TAB - 1)];
        return __hiloint2double(__double2hiint(s) + (((j >> 7) + shift) << 20), __double2loint(s));
    }
    static EC_DEV u64 whole(double w) {                // w < 2^52, rounded to nearest
        return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;
    }
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

// One cluster of CTAs per row: each keeps its share of the row in shared
// memory, so that the logits are read from HBM once.
template <int T>
__global__ void __launch_bounds__(SA_THREADS) k_sample(const ec_sample_args a, int shift, int share, int *err) {
    EC_PDL_ENTER();
    typedef typename SaElt<T>::V V;
    constexpr int ELT = sizeof(V), PER16 = 16 / ELT;
    extern __shared__ __align__(128) unsigned char smem[];
    SaShared &s = *reinterpret_cast<SaShared *>(smem);
    V *vals = reinterpret_cast<V *>(smem + (sizeof(SaShared) + 127) / 128 * 128);
    cg::cluster_group cl = cg::this_cluster();
    const int ctas = (int)cl.num_blocks(), me = (int)cl.block_rank();
    const int r = (int)blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    // Shares are cut at 16-byte blocks of memory: element i of the row is
    // element i + skew of the block that holds its first one.
    const V *row = static_cast<const V *>(a.logits) + (size_t)r * a.ld;
    const int skew = (int)((reinterpret_cast<uintptr_t>(row) & 15) / ELT);
    const long long lo = max((long long)me * share, (long long)skew), hi = min((long long)(me + 1) * share, (long long)skew + a.vocab);
    const int n = (int)max(0ll, hi - lo), off = (int)(lo - (long long)me * share), i0 = (int)(lo - skew);   // vals[off + e] is element i0 + e
    {
        // 16-byte blocks wholly inside the row by one bulk copy, the rest element by element
        const int b0 = (off + PER16 - 1) / PER16 * PER16, b1 = (off + n) / PER16 * PER16;
        const bool bulk = b1 > b0;
        uint64_t *bar = reinterpret_cast<uint64_t *>(&s.bar);
        if (tid == 0) {
            ec_mbar_init(bar, 1);
            ec_fence_mbar_init();
            if (bulk) {
                ec_mbar_expect_tx(bar, (uint32_t)((b1 - b0) * ELT));
                ec_bulk_g2s(vals + b0, row + i0 + (b0 - off), (uint32_t)((b1 - b0) * ELT), bar);
            }
        }
        const int head = bulk ? b0 - off : n, tail = bulk ? b1 - off : n;
        for (int e = tid; e < head; e += SA_THREADS) vals[off + e] = row[i0 + e];
        for (int e = tail + tid; e < n; e += SA_THREADS) vals[off + e] = row[i0 + e];
        if (tid < SA_TAB) s.tab[tid] = exp2((double)tid / SA_TAB);
        if (tid == 0) s.found = 0;
        __syncthreads();
        if (bulk) ec_mbar_wait(bar, 0, err);   // a wait that gave up is reported; the row's result is then void
    }
    const V *mine = vals + off;

    // largest and smallest finite logit
    float mx = -INFINITY, mn = INFINITY;
    for (int e = tid; e < n; e += SA_THREADS) {
        const float v = sa_value<T>(mine[e]);
        mx = fmaxf(mx, v);
        if (fabsf(v) < INFINITY) mn = fminf(mn, v);
    }
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

    const float temperature = a.temperature ? a.temperature[r] : 1.0f, min_p = a.min_p ? a.min_p[r] : 0.0f, top_p = a.top_p ? a.top_p[r] : 1.0f;
    const int top_k = a.top_k ? a.top_k[r] : 0;
    if (mx == -INFINITY) {
        if (me == 0 && tid == 0) {
            a.ids[r] = -1;
            if (a.prob) a.prob[r] = 0.0f;
        }
        return;
    }
    if (!(temperature > 0.0f) || min_p > 1.0f || top_k == 1 || top_p <= 0.0f) {   // one candidate is left: the first of the largest
        int first = 0x7fffffff;
        for (int e = tid; e < n && first == 0x7fffffff; e += SA_THREADS)
            if (sa_value<T>(mine[e]) == mx) first = i0 + e;
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
    const bool infinite = mx == INFINITY;   // logits of +inf weigh the same, all others nothing
    auto value = [&](int e) {
        const float v = sa_value<T>(mine[e]);
        return !infinite ? v : v == INFINITY ? 0.0f : -INFINITY;
    };
    if (infinite) mx = mn = 0.0f;
    const SaWeight weight = {(double)mx, 1.4426950408889634 / (double)temperature, shift, s.tab};
    // Bins over max - logit: up to where weights vanish, or the smallest logit.
    const double vanish = (double)temperature * 0.6931471805599453 * (shift + 3);
    const float reach = vanish < (double)FLT_MAX ? (float)vanish : FLT_MAX;
    const float range = fmaxf(fminf(reach, mx - mn), 1e-30f), per_bin = (float)SA_BINS / range;
    auto bin_of = [&](float v) {   // -1: no weight
        const float x = fminf(mx - v, FLT_MAX);
        return v > -INFINITY && x <= reach ? min((int)(x * per_bin), SA_BINS - 1) : -1;
    };

    u64 cut = 0;                            // rank of the last candidate kept
    float cut_v = -INFINITY;
    int cut_i = 0x7fffffff;
    auto kept = [&](float v, int i) { return v > cut_v || (v == cut_v && i <= cut_i); };

    // Finds the candidate at which the running count (or weight, among those
    // kept so far) over the order reaches what is wanted, and cuts there.
    // With `whole`, everything up to it may be left sorted in the first CTA's
    // list instead; returns true then (all CTAs alike).
    auto select = [&](const bool mass, u64 want, const bool whole) -> bool {
        u64 above = 0, prefix = 0;
        int bits = 64, bin = -1;            // candidates of `bin` whose rank's top 64 - bits bits are `prefix`
        for (;;) {
            __syncthreads();
            for (int b = tid; b < SA_BINS; b += SA_THREADS) s.h.count[b] = s.h.limb[0][b] = s.h.limb[1][b] = s.h.limb[2][b] = 0;
            if (tid == 0) s.count = 0;
            __syncthreads();
            const int step = bits - 10 > 0 ? bits - 10 : 0;
            for (int e = tid; e < n; e += SA_THREADS) {
                const float v = value(e);
                int b = bin_of(v);
                if (b < 0 || (mass && !kept(v, i0 + e))) continue;
                if (bin >= 0) {
                    const u64 k = sa_rank(v, i0 + e);
                    if (b != bin || (bits < 64 && (k >> bits) != prefix)) continue;
                    b = SA_BINS - 1 - (int)((k >> step) & (SA_BINS - 1));
                }
                atomicAdd(&s.h.count[b], 1u);
                if (mass) {
                    const u64 w = SaWeight::whole(weight(v));
                    if (w & 0xffff) atomicAdd(&s.h.limb[0][b], (uint32_t)(w & 0xffff));
                    if (w >> 16 & 0xffff) atomicAdd(&s.h.limb[1][b], (uint32_t)(w >> 16 & 0xffff));
                    if (w >> 32) atomicAdd(&s.h.limb[2][b], (uint32_t)(w >> 32));
                }
            }
            cl.sync();
            if (me == 0) {   // join the histograms, find the crossing
                u64 cnt[2] = {0, 0}, sum[2] = {0, 0};
                for (int c = 0; c < ctas; ++c) {
                    const SaShared *o = cl.map_shared_rank(&s, c);
                    const uint2 q = reinterpret_cast<const uint2 *>(o->h.count)[tid];
                    cnt[0] += q.x;
                    cnt[1] += q.y;
                    if (mass)
#pragma unroll
                        for (int l = 0; l < 3; ++l) {
                            const uint2 m = reinterpret_cast<const uint2 *>(o->h.limb[l])[tid];
                            sum[0] += (u64)m.x << (16 * l);
                            sum[1] += (u64)m.y << (16 * l);
                        }
                }
                if (!mass) { sum[0] = cnt[0]; sum[1] = cnt[1]; }
                u64 total;
                u64 before = above + sa_scan(sum[0] + sum[1], s, total);
                if (mass && bin < 0) {
                    want = (u64)ceil((double)top_p * (double)total);
                    want = want < 1 ? 1 : want > total ? total : want;
                }
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
            const SaCtl ctl = s.ctl;
            want = ctl.want;
            if (ctl.bin < 0) return false;   // fewer than wanted have any weight: nothing to cut
            above = ctl.above;
            if (ctl.at[0] < 0) {             // everything up to the crossing goes to the list
                // how many of this CTA's do, for its place in it
                int c = 0;
                for (int b = tid; b <= ctl.bin; b += SA_THREADS) c += (int)s.h.count[b];
                u64 total;
                sa_scan((u64)c, s, total);
                if (tid == 0) cl.map_shared_rank(&s, 0)->first[me] = (int)total;
                cl.sync();
                const SaShared *o = cl.map_shared_rank(&s, 0);
                int at = 0;
                for (int q = 0; q < me; ++q) at += o->first[q];
                u64 *list = cl.map_shared_rank(&s, 0)->l.rank;
                cl.sync();                   // the first CTA's counts are read: its list may be written over them
                for (int e = tid; e < n; e += SA_THREADS) {
                    const float v = value(e);
                    const int b = bin_of(v);
                    if (b >= 0 && b <= ctl.bin) list[at + atomicAdd(&s.count, 1)] = sa_rank(v, i0 + e);
                }
                cl.sync();
                return true;
            }
            if (bin < 0) {
                bin = ctl.bin;
            } else {
                prefix = prefix << (bits - step) | ((u64)(SA_BINS - 1 - ctl.bin) & ((1ull << (bits - step)) - 1));
                bits = step;
            }
            if (ctl.crowd > SA_LIST) continue;
            u64 *list = cl.map_shared_rank(&s, 0)->l.rank;
            for (int e = tid; e < n; e += SA_THREADS) {
                const float v = value(e);
                if (bin_of(v) != bin || (mass && !kept(v, i0 + e))) continue;
                const u64 k = sa_rank(v, i0 + e);
                if (bits < 64 && (k >> bits) != prefix) continue;
                list[ctl.at[me] + atomicAdd(&s.count, 1)] = k;
            }
            cl.sync();
            if (me == 0) {
                const int size = sa_pow2(ctl.crowd);
                for (int i = tid; i < size; i += SA_THREADS)
                    if (i >= ctl.crowd) s.l.rank[i] = 0;
                sa_sort(s.l.rank, size);
                u64 w[SA_PER], sum = 0, total;
#pragma unroll
                for (int j = 0; j < SA_PER; ++j) {
                    const int i = tid * SA_PER + j;
                    w[j] = i >= ctl.crowd ? 0ull : mass ? SaWeight::whole(weight(sa_rank_value(s.l.rank[i]))) : 1ull;
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
            cut = s.ctl.cut;
            cut_v = sa_rank_value(cut);
            cut_i = sa_rank_index(cut);
            return false;
        }
    };

    const float u = a.u[r];
    auto point = [&](u64 total) -> u64 {   // the sum has to exceed it
        const double x = u > 0.0f ? (double)u * (double)total : 0.0;
        return x >= (double)total ? total - 1 : min((u64)x, total - 1);
    };
    const double least = min_p > 0.0f ? (double)min_p * (double)(1ull << shift) : 0.0;

    if (top_k > 0 && top_k < a.vocab && select(false, (u64)top_k, top_k <= SA_LIST / 2)) {
        if (me != 0) return;
        // the list holds at least top_k candidates, in no order yet
        int size = 0;
        for (int c = 0; c < ctas; ++c) size += s.first[c];
        const int full = sa_pow2(size);
        for (int i = tid; i < full; i += SA_THREADS)
            if (i >= size) s.l.rank[i] = 0;
        sa_sort(s.l.rank, full);
        u64 w[SA_PER], sum = 0, total;
        double wd[SA_PER];
#pragma unroll
        for (int j = 0; j < SA_PER; ++j) {
            const int i = tid * SA_PER + j;
            wd[j] = i < top_k && i < size ? weight(sa_rank_value(s.l.rank[i])) : 0.0;
            w[j] = SaWeight::whole(wd[j]);
            sum += w[j];
        }
        u64 before = sa_scan(sum, s, total);
        const u64 want = top_p < 1.0f ? max(1ull, min(total, (u64)ceil((double)top_p * (double)total))) : total;
        u64 kept_sum = 0;
#pragma unroll
        for (int j = 0; j < SA_PER; ++j) {   // kept: what comes before `want` is reached, and weighs enough
            const int i = tid * SA_PER + j;
            const bool keep = w[j] > 0 && before < want && (wd[j] >= least || i == 0);
            before += w[j];
            if (!keep) w[j] = 0;
            kept_sum += w[j];
            s.l.w[i] = (u64)__double_as_longlong(wd[j]);
            s.l.rank[i] = keep ? (u64)(uint32_t)~sa_rank_index(s.l.rank[i]) << 32 | (uint32_t)i : 0ull;   // lowest index largest
        }
        sa_scan(kept_sum, s, total);
        const int kept_n = sa_pow2(min(size, top_k));
        sa_sort(s.l.rank, kept_n);
        const u64 target = point(total);
        sum = 0;
#pragma unroll
        for (int j = 0; j < SA_PER; ++j) {
            const int i = tid * SA_PER + j;
            const u64 k = i < kept_n ? s.l.rank[i] : 0ull;
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
        return;
    }
    if (top_p < 1.0f) select(true, 0, false);

    // Weights of the kept candidates in vocabulary order: of each warp's
    // contiguous piece, of the CTAs, then of the piece that holds the point.
    const int piece = ((n + SA_WARPS - 1) / SA_WARPS + 31) / 32 * 32;
    auto drawn = [&](int e) -> u64 {
        const float v = value(e);
        if (!kept(v, i0 + e)) return 0ull;
        const double w = weight(v);
        return w >= least ? SaWeight::whole(w) : 0ull;
    };
    u64 sum = 0;
    for (int e = warp * piece + lane; e < min(n, (warp + 1) * piece); e += 32) sum += drawn(e);
    sum = sa_warp_sum(sum);
    __syncthreads();
    if (lane == 0) s.part[warp] = sum;
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
    const u64 target = point(total);
    if (target < before || target >= before + s.sums[me]) return;
    int w = 0;
    while (before + s.part[w] <= target) before += s.part[w++];
    const int e1 = min(n, (w + 1) * piece);
    for (int b = w * piece; b < e1; b += SA_THREADS) {
        const u64 x = b + tid < e1 ? drawn(b + tid) : 0ull;
        u64 all;
        const u64 start = before + sa_scan(x, s, all);
        if (start <= target && target < start + x) {
            a.ids[r] = i0 + b + tid;
            if (a.prob) a.prob[r] = (float)(weight(value(b + tid)) / (double)total);
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
