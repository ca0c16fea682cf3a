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
// the candidates of that bin are put in order; a bin of more than SA_LIST of
// them (equal logits) is first cut down by the bits of their order.  A top-k of
// up to SA_FAST needs no histogram: at least top_k candidates lie at or above
// the top_k-th largest of the maxima of SA_TOPS groups of the row, and those
// few are gathered and handled by one CTA.
// Measured, fp32 logits: one row of 151936 with top-k 50 and top-p 0.95 9.5 us,
// 16 CTAs whose chain of load, maximum, gather and draw it is; 128 such rows
// with settings of their own 106 us or 0.74 TB/s, where a row with top-p alone
// takes longest (histogram, join and gather, each a meeting of the cluster);
// 1000 rows of 50257 with a temperature alone 111 us (k_sample_rows).
#include "ec_common.cuh"
#include "ec_serve.h"

#include <cooperative_groups.h>
#include <float.h>
#include <stddef.h>

namespace cg = cooperative_groups;

namespace {

typedef unsigned long long u64;
constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / 32;
constexpr int SA_WORDS = 4096;                    // words of a histogram: bins of counts, or two halves of weights
constexpr int SA_LIST = 1024, SA_PER = SA_LIST / SA_THREADS;
constexpr int SA_TOPS = 256, SA_FAST = 192;       // 192 of 256: about 1.4 * 256 candidates
constexpr int SA_FEW = 256;                       // candidates that are ordered by counting
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
EC_DEV uint32_t sa_bits(float v) {
    const uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);
    return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
EC_DEV float sa_bits_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
EC_DEV u64 sa_rank(float v, int i) { return (u64)sa_bits(v) << 32 | (uint32_t)~i; }
EC_DEV float sa_rank_value(u64 r) { return sa_bits_value((uint32_t)(r >> 32)); }
EC_DEV int sa_rank_index(u64 r) { return (int)~(uint32_t)r; }

struct SaShared {
    double tab[SA_TAB];        // 2^(j / 512 + shift)
    double part2[48];          // its factors 2^(i / 16 + shift), 2^(i / 512)
    u64 part[SA_WARPS + 1];
    u64 sums[SA_MAX_CTAS];     // each CTA's weight
    u64 slices[SA_MAX_CTAS][SA_MAX_CTAS];   // [CTA][slice of the bins]: count or weight
    alignas(16) float high[SA_MAX_CTAS];
    alignas(16) float low[SA_MAX_CTAS];
    int first[SA_MAX_CTAS];
    alignas(16) uint32_t tops[SA_TOPS];   // maxima of the row's groups, in order-preserving bits
    float red[2 * SA_WARPS];
    uint32_t top;              // the top_k-th of them
    int count, place, taken;   // taken (first CTA): places of the list given away
    int bin;                   // crossing
    u64 above, cut;
    u64 bar;
    u64 rank[SA_LIST];         // candidates; in the first CTA those of the cluster
    union alignas(16) {
        uint32_t hist[SA_WORDS];
        u64 w[SA_LIST];
    };
};

// w(v) * 2^shift in double, not yet rounded to an integer.  With t = 512 (v -
// max) log2(e) / T = j + f, |f| <= 1/2: 2^(t/512) = 2^(j div 512) tab[j mod
// 512] e^(f ln 2 / 512), the last as its Taylor sum to the third power
// (0.00068^4 / 24 = 2^-46.7 of it is left out).  Nothing (2^-1000) for v below
// `floor`, where it is less than 2^-(shift + 2), for NaN and where `is` is
// false.  Nine double operations and no branch.
struct SaWeight {
    double mx, c;              // c: 512 log2(e) / T
    float floor;
    const double *tab;         // 2^(j / 512 + shift)
    EC_DEV double operator()(float v, bool is = true) const {
        const double magic = 6755399441055744.0;      // 1.5 * 2^52
        const double d = (double)fmaxf(v, floor) - mx;
        const double kd = __fma_rn(d, c, magic);
        const int j = __double2loint(kd);
        const double f = __fma_rn(d, c, magic - kd);
        double p = __fma_rn(f, 4.1353783506767136e-10, 9.163913992275265e-07);   // (ln2 / 512)^n / n!
        p = __fma_rn(f, p, 1.3538030870311431e-3);
        p = __fma_rn(f, p, 1.0);
        const double s = p * tab[j & (SA_TAB - 1)];
        const int e = is && v >= floor ? (j & ~(SA_TAB - 1)) << 11 : -(1000 << 20);
        return __hiloint2double(__double2hiint(s) + e, __double2loint(s));
    }
    // A weight (below 2^52) rounded to nearest, plus RAW: sums of these wrap
    // and are put right by the number of terms.
    static constexpr u64 RAW = 0x4330000000000000ull;
    static EC_DEV u64 raw(double w) { return (u64)__double_as_longlong(w + 4503599627370496.0); }
    static EC_DEV u64 whole(double w) { return raw(w) - RAW; }
};

static_assert(offsetof(SaShared, tops) % 16 == 0 && offsetof(SaShared, high) % 16 == 0 && offsetof(SaShared, low) % 16 == 0 && offsetof(SaShared, hist) % 16 == 0 && offsetof(SaShared, bar) % 8 == 0 &&
              alignof(SaShared) <= 128, "vector accesses");

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

// Sort list[0, n), largest first; n a power of two of at most PER * SA_THREADS.
// A thread holds PER neighbours: pairs up to 32 * PER apart are exchanged in
// registers, only the others (10 of 66 steps for 2048) through shared memory.
template <int PER> EC_DEV void sa_sort_per(u64 *list, int n) {
    const int tid = threadIdx.x;
    const bool in = tid * PER < n;
    u64 v[PER];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < PER; ++q) v[q] = in && tid * PER + q < n ? list[tid * PER + q] : 0ull;
    for (int k = 2; k <= n; k <<= 1) {
        for (int j = k >> 1; j > 0; j >>= 1) {
            if (j >= 32 * PER) {
                __syncthreads();
                if (in)
#pragma unroll
                    for (int q = 0; q < PER; ++q) list[tid * PER + q] = v[q];
                __syncthreads();
                if (in)
#pragma unroll
                    for (int q = 0; q < PER; ++q) {
                        const int i = tid * PER + q;
                        const u64 o = list[i ^ j];
                        const bool larger = ((i & j) == 0) == ((i & k) == 0);
                        v[q] = (v[q] < o) == larger ? o : v[q];
                    }
            } else if (j >= PER) {
#pragma unroll
                for (int q = 0; q < PER; ++q) {
                    const int i = tid * PER + q;
                    const u64 o = __shfl_xor_sync(0xffffffffu, v[q], j / PER);
                    const bool larger = ((i & j) == 0) == ((i & k) == 0);
                    v[q] = (v[q] < o) == larger ? o : v[q];
                }
            } else {
#pragma unroll
                for (int d = PER / 2; d > 0; d >>= 1)
                    if (j == d)
#pragma unroll
                        for (int q = 0; q < PER; ++q)
                            if ((q & d) == 0) {
                                const bool down = ((tid * PER + q) & k) == 0;
                                const u64 x = v[q], y = v[q + d];
                                const bool swap = (x < y) == down;
                                v[q] = swap ? y : x;
                                v[q + d] = swap ? x : y;
                            }
            }
        }
    }
    __syncthreads();
    if (in)
#pragma unroll
        for (int q = 0; q < PER; ++q)
            if (tid * PER + q < n) list[tid * PER + q] = v[q];
    __syncthreads();
}

__noinline__ __device__ void sa_sort(u64 *list, int n) {   // one copy: cold code costs more than the call
    if (n <= SA_THREADS) sa_sort_per<1>(list, n);
    else sa_sort_per<2>(list, n);
}
static_assert(SA_LIST <= 2 * SA_THREADS, "sa_sort");

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
    float mx, reach, per_bin;  // 1 / range of a histogram, bins per unit
    float cut_v;               // kept: larger, or equal and up to index cut_i
    int cut_i;
    bool cut;

    EC_DEV float at(int place) const { return sa_value<T>(reinterpret_cast<const V *>(blocks)[place]); }
    EC_DEV bool kept(float v, int place) const { return v > cut_v || (v == cut_v && place + ibase <= cut_i); }
    // Bin of v >= weight.floor: (max - v) in bins rounded to nearest, by the low
    // bits of a sum with 2^23.
    EC_DEV int bin(float v, int bins) const {
        return (int)min(__float_as_uint(fmaf(mx - v, per_bin, 8388608.0f)) - 0x4b000000u, (uint32_t)(bins - 1));
    }

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
    // Sum of the weights of what is kept and weighs at least `least`.
    template <bool CUT, bool LEAST> EC_DEV u64 sum(int b0, int b1, int t, int threads, double least) const {
        u64 raw = 0;
        each(b0, b1, t, threads, [&](float v, int p) {
            const double w = weight(v, !CUT || kept(v, p));
            const u64 x = SaWeight::raw(w);
            raw += LEAST && !(w >= least) ? SaWeight::RAW : x;
        });
        const int terms = b1 - b0 > t ? ((b1 - b0 - t - 1) / threads + 1) * PER : 0;
        return raw - (u64)terms * SaWeight::RAW;
    }
    EC_DEV u64 sum(int b0, int b1, int t, int threads, double least) const {
        return least > 0.0 ? (cut ? sum<true, true>(b0, b1, t, threads, least) : sum<false, true>(b0, b1, t, threads, least))
                           : (cut ? sum<true, false>(b0, b1, t, threads, least) : sum<false, false>(b0, b1, t, threads, least));
    }
};

// The candidates that `in` lets through, gathered in the first CTA's list (in
// any order); true when they fit.  The first CTA's `taken` was 0 when the
// cluster last met.  All CTAs of the cluster call it alike; it ends with the
// cluster meeting.
template <int T, typename F> EC_DEV bool sa_gather(cg::cluster_group &cl, const SaRow<T> &row, F in) {
    SaShared &s = row.s;
    const int me = (int)cl.block_rank(), tid = threadIdx.x;
    // the first CTA writes into the list at once, the others by way of their own
    int *counter = me == 0 ? &s.taken : &s.count;
    __syncthreads();
    if (tid == 0) s.count = 0;
    __syncthreads();
    row.each(0, row.n, tid, SA_THREADS, [&](float v, int p) {
        if (in(v, p)) {
            const int at = atomicAdd(counter, 1);
            if (at < SA_LIST) s.rank[at] = sa_rank(v, p + row.ibase);
        }
    });
    if (me != 0) {
        __syncthreads();
        if (tid == 0) s.place = s.count ? atomicAdd(&cl.map_shared_rank(&s, 0)->taken, s.count) : 0;
        __syncthreads();
        u64 *list = cl.map_shared_rank(s.rank, 0);
        for (int i = tid; i < min(s.count, SA_LIST); i += SA_THREADS)
            if (s.place + i < SA_LIST) list[s.place + i] = s.rank[i];
    }
    cl.sync();
    return cl.map_shared_rank(&s, 0)->taken <= SA_LIST;
}

// Finds the candidate at which the running count (MASS: weight, among those
// kept so far) over the order reaches what is wanted, and cuts there.  All
// CTAs of the cluster call it alike.
template <bool MASS, int T>
EC_DEV void sa_select(cg::cluster_group &cl, SaRow<T> &row, u64 want, float top_p) {
    SaShared &s = row.s;
    constexpr int BINS = MASS ? SA_WORDS / 2 : SA_WORDS, EACH = BINS / SA_THREADS;   // weights: low words, then high words
    const int ctas = (int)cl.num_blocks(), me = (int)cl.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int slice = BINS / ctas;
    u64 above = 0, prefix = 0;
    int bits = 64, bin = -1;   // from the second round: candidates of `bin` whose rank's top 64 - bits bits are `prefix`
    constexpr int STEP = MASS ? 11 : 12;
    const float floor = row.weight.floor;
    row.per_bin = row.reach * BINS;
    auto in_class = [&](float v, int p) {
        if (!(v >= floor) || row.bin(v, BINS) != bin || (MASS && row.cut && !row.kept(v, p))) return false;
        return bits == 64 || (sa_rank(v, p + row.ibase) >> bits) == prefix;
    };
    auto sum_of = [&](const uint32_t *h, int b) { return MASS ? (u64)h[b] + ((u64)h[BINS + b] << 32) : (u64)h[b]; };
    for (;;) {
        __syncthreads();
        for (int b = tid; b < SA_WORDS / 4; b += SA_THREADS) reinterpret_cast<uint4 *>(s.hist)[b] = make_uint4(0u, 0u, 0u, 0u);
        if (tid == 0) s.taken = 0;
        __syncthreads();
        const int step = bits - STEP > 0 ? bits - STEP : 0;
        auto add = [&](float v, int b) {
            if (!MASS) {
                atomicAdd(&s.hist[b], 1u);
            } else {
                const u64 w = SaWeight::whole(row.weight(v));
                const uint32_t lo = (uint32_t)w, old = atomicAdd(&s.hist[b], lo);
                const uint32_t hi = (uint32_t)(w >> 32) + (old + lo < lo);   // with the carry of the low word
                if (hi) atomicAdd(&s.hist[BINS + b], hi);
            }
        };
        if (bin < 0)
            row.each(0, row.n, tid, SA_THREADS, [&](float v, int p) {
                if (v >= floor && (!MASS || !row.cut || row.kept(v, p))) add(v, row.bin(v, BINS));
            });
        else
            row.each(0, row.n, tid, SA_THREADS, [&](float v, int p) {
                if (in_class(v, p)) add(v, BINS - 1 - (int)((sa_rank(v, p + row.ibase) >> step) & (BINS - 1)));
            });
        __syncthreads();
        // Every CTA tells the others its sum of each slice of the bins, so that
        // all know the slice of the crossing and join its bins themselves.
        for (int sl = warp; sl < ctas; sl += SA_WARPS) {
            u64 t = 0;
            for (int b = lane; b < slice; b += 32) t += sum_of(s.hist, sl * slice + b);
            t = sa_warp_sum(t);
            if (lane < ctas) cl.map_shared_rank(&s, lane)->slices[me][sl] = t;
        }
        cl.sync();
        u64 mine = 0, total = above;
        for (int c = 0; c < ctas; ++c) mine += lane < ctas ? s.slices[c][lane] : 0ull;
        int at = ctas;
        u64 before = above;
        if (MASS && bin < 0) {
            const u64 all = sa_warp_sum(mine);
            want = max(1ull, min(all, (u64)ceil((double)top_p * (double)all)));
        }
        for (int c = 0; c < ctas; ++c) {
            const u64 t = __shfl_sync(0xffffffffu, mine, c);
            if (at == ctas && total + t >= want) { at = c; before = total; }
            total += t;
        }
        if (at == ctas) {   // fewer than wanted have any weight: nothing to cut
            cl.sync();      // `slices` is read
            return;
        }
        // a thread's bins of that slice, from all CTAs at once
        u64 sum[EACH] = {};
        mine = 0;
        const int each = (slice + SA_THREADS - 1) / SA_THREADS;
#pragma unroll
        for (int q = 0; q < EACH; ++q)
            if (q < each && tid * each + q < slice) {
                const int b = at * slice + tid * each + q;
                if (ctas > 4) {
                    uint32_t lo[SA_MAX_CTAS], hi[SA_MAX_CTAS];
#pragma unroll
                    for (int c = 0; c < SA_MAX_CTAS; ++c) {
                        lo[c] = c < ctas ? *cl.map_shared_rank(s.hist + b, c) : 0u;
                        hi[c] = MASS && c < ctas ? *cl.map_shared_rank(s.hist + BINS + b, c) : 0u;
                    }
#pragma unroll
                    for (int c = 0; c < SA_MAX_CTAS; ++c) sum[q] += (u64)lo[c] + ((u64)hi[c] << 32);
                } else {
                    for (int c = 0; c < ctas; ++c) sum[q] += sum_of(cl.map_shared_rank(s.hist, c), b);
                }
                mine += sum[q];
            }
        before += sa_scan(mine, s, total);
#pragma unroll
        for (int q = 0; q < EACH; ++q) {
            if (sum[q] && before < want && before + sum[q] >= want) {
                s.bin = at * slice + tid * each + q;
                s.above = before;
            }
            before += sum[q];
        }
        __syncthreads();
        above = s.above;
        if (bin < 0) {
            bin = s.bin;
        } else {
            prefix = prefix << (bits - step) | ((u64)(BINS - 1 - s.bin) & ((1ull << (bits - step)) - 1));
            bits = step;
        }
        if (sa_gather(cl, row, in_class)) break;
        cl.sync();          // `taken` is read
    }
    if (me == 0) {
        const int n = s.taken;
        if (n <= SA_FEW) {   // the weight before a candidate: a loop over the others, shared out over 512 / n threads
            const int group = n <= 32 ? 16 : n <= 64 ? 8 : n <= 128 ? 4 : 2, i = tid / group;
            for (int j = tid; j < n; j += SA_THREADS) s.w[j] = MASS ? SaWeight::whole(row.weight(sa_rank_value(s.rank[j]))) : 1ull;
            __syncthreads();
            const u64 r = i < n ? s.rank[i] : 0ull;
            u64 before = 0;
            for (int j = tid % group; j < n; j += group) before += s.rank[j] > r ? s.w[j] : 0ull;
            for (int o = 1; o < group; o <<= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
            before += above;
            if (i < n && before < want && before + s.w[i] >= want) s.cut = r;
        } else {
            const int size = sa_pow2(n);
            for (int i = n + tid; i < size; i += SA_THREADS) s.rank[i] = 0;
            sa_sort(s.rank, size);
            u64 w[SA_PER], sum = 0, total;
#pragma unroll
            for (int j = 0; j < SA_PER; ++j) {
                const int i = tid * SA_PER + j;
                w[j] = i >= n ? 0ull : MASS ? SaWeight::whole(row.weight(sa_rank_value(s.rank[i]))) : 1ull;
                sum += w[j];
            }
            u64 before = above + sa_scan(sum, s, total);
#pragma unroll
            for (int j = 0; j < SA_PER; ++j) {
                if (before < want && before + w[j] >= want) s.cut = s.rank[tid * SA_PER + j];
                before += w[j];
            }
        }
        __syncthreads();
        if (tid < ctas) cl.map_shared_rank(&s, tid)->cut = s.cut;
    }
    cl.sync();
    row.cut = true;
    row.cut_v = sa_rank_value(s.cut);
    row.cut_i = sa_rank_index(s.cut);
}

// The other half of the arrival at the kernel's start: no CTA of the cluster
// is still to come.
EC_DEV void sa_cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

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
    const int tid = threadIdx.x;
    if (size <= SA_FEW) {   // by counting, as in sa_select
        const int group = size <= 32 ? 16 : size <= 64 ? 8 : size <= 128 ? 4 : 2, i = tid / group;
        if (tid == 0) s.above = 0;
        __syncthreads();
        for (int j = tid; j < size; j += SA_THREADS) s.w[j] = SaWeight::whole(row.weight(sa_rank_value(s.rank[j])));
        __syncthreads();
        const u64 mine = i < size ? s.rank[i] : 0ull;
        int place = 0;
        u64 before = 0;
        for (int j = tid % group; j < size; j += group)
            if (s.rank[j] > mine) {
                ++place;
                before += s.w[j];
            }
        for (int o = 1; o < group; o <<= 1) {
            place += __shfl_xor_sync(0xffffffffu, place, o);
            before += __shfl_xor_sync(0xffffffffu, before, o);
        }
        if (i < size && place == min(top_k, size) - 1) s.above = before + s.w[i];   // the sum over the first top_k
        __syncthreads();
        const u64 total = s.above, want = top_p < 1.0f ? max(1ull, min(total, (u64)ceil((double)top_p * (double)total))) : total;
        const double w = i < size ? row.weight(sa_rank_value(mine)) : 0.0;
        const bool keep = i < size && place < top_k && before < want && (w >= least || place == 0);
        __syncthreads();
        if (!keep && i < size && tid % group == 0) s.w[i] = 0;
        __syncthreads();
        u64 kept = 0;
        before = 0;
        for (int j = tid % group; j < size; j += group) {
            const u64 x = s.w[j];
            kept += x;
            before += (uint32_t)s.rank[j] > (uint32_t)mine ? x : 0ull;   // a lower index
        }
        for (int o = 1; o < group; o <<= 1) {
            kept += __shfl_xor_sync(0xffffffffu, kept, o);
            before += __shfl_xor_sync(0xffffffffu, before, o);
        }
        const u64 target = sa_point(a.u[r], kept);
        if (keep && tid % group == 0 && before <= target && target < before + s.w[i]) {
            a.ids[r] = sa_rank_index(mine);
            if (a.prob) a.prob[r] = (float)(w / (double)kept);
        }
        return;
    }
    const int full = sa_pow2(size);
    for (int i = tid; i < full; i += SA_THREADS)
        if (i >= size) s.rank[i] = 0;
    sa_sort(s.rank, full);
    u64 w[SA_PER], sum = 0, total;
    double wd[SA_PER];
#pragma unroll
    for (int j = 0; j < SA_PER; ++j) {
        const int i = tid * SA_PER + j;
        wd[j] = i < top_k && i < size ? row.weight(sa_rank_value(s.rank[i])) : 0.0;
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
        s.w[i] = (u64)__double_as_longlong(wd[j]);
        s.rank[i] = keep ? (u64)(uint32_t)~sa_rank_index(s.rank[i]) << 32 | (uint32_t)i : 0ull;   // lowest index largest
    }
    sa_scan(kept, s, total);
    const int most = sa_pow2(min(size, top_k));
    sa_sort(s.rank, most);
    const u64 target = sa_point(a.u[r], total);
    sum = 0;
#pragma unroll
    for (int j = 0; j < SA_PER; ++j) {
        const int i = tid * SA_PER + j;
        const u64 k = i < most ? s.rank[i] : 0ull;
        wd[j] = k ? __longlong_as_double((long long)s.w[(uint32_t)k]) : 0.0;
        w[j] = SaWeight::whole(wd[j]);
        sum += w[j];
    }
    u64 all;
    before = sa_scan(sum, s, all);
#pragma unroll
    for (int j = 0; j < SA_PER; ++j) {
        if (before <= target && target < before + w[j]) {
            a.ids[r] = (int)~(uint32_t)(s.rank[tid * SA_PER + j] >> 32);
            if (a.prob) a.prob[r] = (float)(wd[j] / (double)total);
        }
        before += w[j];
    }
}

// One cluster of CTAs per row: each keeps its share of the row in shared
// memory, so that the logits are read from HBM once.
template <int T>
__global__ void __launch_bounds__(SA_THREADS, 2) k_sample(const ec_sample_args a, int shift, int share, int *err) {
    typedef SaRow<T> Row;
    typedef typename Row::V V;
    constexpr int ELT = Row::ELT, PER = Row::PER;
    extern __shared__ __align__(128) unsigned char smem[];
    SaShared &s = *reinterpret_cast<SaShared *>(smem);
    if (threadIdx.x < SA_MAX_CTAS) {
        s.high[threadIdx.x] = -INFINITY;
        s.low[threadIdx.x] = INFINITY;
    }
    // this CTA has started, and what others write first is set (sa_cluster_wait)
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    EC_PDL_ENTER();
    V *vals = reinterpret_cast<V *>(smem + (sizeof(SaShared) + 127) / 128 * 128);
    cg::cluster_group cl = cg::this_cluster();
    const int ctas = (int)cl.num_blocks(), me = (int)cl.block_rank();
    const int r = (int)blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float temperature = a.temperature ? a.temperature[r] : 1.0f, min_p = a.min_p ? a.min_p[r] : 0.0f, top_p = a.top_p ? a.top_p[r] : 1.0f;
    const int top_k = a.top_k ? a.top_k[r] : 0;

    // Below `vanish` from the largest a weight is 0: only what lies above is
    // ever a candidate.
    const double vanish = (double)temperature * 0.6931471805599453 * (shift + 3), per_nat = 512.0 * 1.4426950408889634 / (double)temperature;

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
        if (tid == 0) { s.taken = 0; s.top = 0xffffffffu; }
        if (tid < 48) s.part2[tid] = exp2(tid < 16 ? (double)tid / 16 + shift : (double)(tid - 16) / SA_TAB);
        __syncthreads();
        for (int j = tid; j < SA_TAB; j += SA_THREADS) s.tab[j] = s.part2[j / 32] * s.part2[16 + j % 32];
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
    // the few candidates of a small top-k are found by the maxima of SA_TOPS
    // groups of threads, `group` lanes each
    const bool fast = top_k > 1 && top_k <= SA_FAST && top_k < a.vocab;
    const int group = SA_THREADS * ctas / SA_TOPS;
    float group_mx = -INFINITY;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        if (o == group) group_mx = mx;
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    }
    if (group == 32) group_mx = mx;
    if (lane == 0) { s.red[warp] = mx; s.red[SA_WARPS + warp] = mn; }
    __syncthreads();
    if (warp == 0) {
        mx = s.red[lane % SA_WARPS];
        mn = s.red[SA_WARPS + lane % SA_WARPS];
#pragma unroll
        for (int o = SA_WARPS / 2; o > 0; o >>= 1) {
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        }
    }
    sa_cluster_wait();   // every CTA of the cluster has started: its shared memory may be written
    if (tid < ctas) {
        SaShared *o = cl.map_shared_rank(&s, tid);
        o->high[me] = mx;
        o->low[me] = mn;
    }
    if (fast)
        for (int c = lane % group; c < ctas; c += group) cl.map_shared_rank(&s, c)->tops[(me * SA_THREADS + tid) / group] = sa_bits(group_mx);
    cl.sync();
    mx = -INFINITY;
    mn = INFINITY;
#pragma unroll
    for (int c = 0; c < SA_MAX_CTAS / 4; ++c) {
        const float4 h = reinterpret_cast<const float4 *>(s.high)[c], l = reinterpret_cast<const float4 *>(s.low)[c];
        mx = fmaxf(fmaxf(fmaxf(mx, h.x), fmaxf(h.y, h.z)), h.w);
        mn = fminf(fminf(fminf(mn, l.x), fminf(l.y, l.z)), l.w);
    }

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
    const bool infinite = mx == INFINITY;
    if (infinite) {   // logits of +inf weigh the same, all others nothing
        for (int e = tid; e < blocks * PER; e += SA_THREADS)
            vals[e] = sa_value<T>(vals[e]) == INFINITY ? (V)0 : (V)(T == EC_T_F32 ? -INFINITY : T == EC_T_F16 ? 0xfc00 : 0xff80);
        __syncthreads();
        mx = mn = 0.0f;
    }
    // floor: the smallest float that is not below
    const float floor = fmaxf(__double2float_ru((double)mx - vanish), -FLT_MAX);
    row.weight = {(double)mx, per_nat, floor, s.tab};
    row.mx = mx;
    row.reach = 1.0f / fmaxf(fminf(mx - floor, mx - mn), 1e-30f);
    row.cut_v = -INFINITY;
    row.cut_i = 0x7fffffff;
    row.cut = false;
    const double least = min_p > 0.0f ? (double)min_p * (double)(1ull << shift) : 0.0;

    if (top_k > 0 && top_k < a.vocab) {
        bool listed = false;
        if (fast && !infinite) {
            // the top_k-th largest of the maxima is the smallest that fewer
            // than top_k exceed: two threads count for a value
            const uint32_t v = s.tops[tid / 2];
            int larger = 0;
#pragma unroll 4
            for (int j = tid % 2; j < SA_TOPS / 4; j += 2) {
                const uint4 q = reinterpret_cast<const uint4 *>(s.tops)[j];
                larger += (q.x > v) + (q.y > v) + (q.z > v) + (q.w > v);
            }
            larger += __shfl_xor_sync(0xffffffffu, larger, 1);
            const uint32_t least_top = __reduce_min_sync(0xffffffffu, larger < top_k ? v : 0xffffffffu);
            if (lane == 0) atomicMin(&s.top, least_top);
            __syncthreads();
            const float top = sa_bits_value(s.top);
            if (top > -INFINITY) listed = sa_gather(cl, row, [&](float x, int) { return x >= top; });
        }
        if (listed) {
            if (me != 0) return;
            sa_draw_list(a, row, r, s.taken, top_k, top_p, least);
            cl.sync();   // the others have read `taken` (and left)
            return;
        }
        if (fast && !infinite) cl.sync();   // `taken` is read
        sa_select<false>(cl, row, (u64)top_k, top_p);
    }
    if (top_p < 1.0f) sa_select<true>(cl, row, 0ull, top_p);

    // Weights of the kept candidates in vocabulary order: of each warp's
    // contiguous piece, of the CTAs, then of the piece that holds the point.
    const int piece = (blocks + SA_WARPS - 1) / SA_WARPS;
    const u64 part = sa_warp_sum(row.sum(warp * piece, min(blocks, (warp + 1) * piece), lane, 32, least));
    __syncthreads();
    if (lane == 0) s.part[warp] = part;
    __syncthreads();
    if (warp == 0) {
        u64 t = lane < SA_WARPS ? s.part[lane] : 0ull;
        t = sa_warp_sum(t);
        if (lane < ctas) cl.map_shared_rank(&s, lane)->sums[me] = t;
    }
    cl.sync();
    u64 before = 0, total = 0;
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
        const double x = row.weight(v, !row.cut || row.kept(v, p));
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

constexpr int DR_THREADS = 512, DR_WARPS = DR_THREADS / 32, DR_VOCAB = 16384;
constexpr int DR_BATCH = 4;                       // 16-byte loads of a thread in flight

// A row in global memory, in aligned 16-byte blocks; its first and last may
// reach beyond it and are then read element by element.
template <int T> struct DrRow {
    typedef typename SaElt<T>::V V;
    static constexpr int ELT = sizeof(V), PER = 16 / ELT;
    const V *src;
    int skew, vocab, blocks;   // place p is element p - skew
    bool infinite;             // +inf weighs one, all else nothing
    SaWeight weight;

    EC_DEV float value(float v) const { return !infinite ? v : v == INFINITY ? 0.0f : -INFINITY; }
    EC_DEV float at(int p) const { return p >= skew && p - skew < vocab ? value(sa_value<T>(src[p - skew])) : -INFINITY; }
    EC_DEV uint4 block(int b) const {
        const int e = b * PER - skew;
        if (e >= 0 && e + PER <= vocab) return *reinterpret_cast<const uint4 *>(src + e);
        uint32_t w[4];
        for (int i = 0; i < 4; ++i) {
            w[i] = T == EC_T_F32 ? 0xff800000u : T == EC_T_F16 ? 0xfc00fc00u : 0xff80ff80u;
            for (int j = 0; j < PER / 4; ++j) {
                const int n = e + i * (PER / 4) + j;
                if (n < 0 || n >= vocab) continue;
                if constexpr (T == EC_T_F32) w[i] = __float_as_uint(src[n]);
                else w[i] = (w[i] & (j ? 0xffffu : 0xffff0000u)) | (uint32_t)src[n] << (16 * j);
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    // f(value, place) for blocks [b0, b1), taken by threads t of `threads`
    template <typename F> EC_DEV void each(int b0, int b1, int t, int threads, F f) const {
#pragma unroll 1
        for (int b = b0 + t; b < b1; b += DR_BATCH * threads) {
            uint4 u[DR_BATCH];
#pragma unroll
            for (int i = 0; i < DR_BATCH; ++i)
                if (b + i * threads < b1) u[i] = block(b + i * threads);
#pragma unroll
            for (int i = 0; i < DR_BATCH; ++i) {
                if (b + i * threads >= b1) break;
                const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    V x;
                    if constexpr (T == EC_T_F32) x = __uint_as_float(w[j]);
                    else x = (uint16_t)(w[j / 2] >> (16 * (j % 2)));
                    f(sa_value<T>(x), (b + i * threads) * PER + j);
                }
            }
        }
    }
    // A warp's sum of the weights of blocks [b0, b1)
    template <bool RARE> EC_DEV u64 sum(int b0, int b1, int lane, double least) const {
        u64 raw = 0;
        each(b0, b1, lane, 32, [&](float v, int) {
            const double w = weight(RARE ? value(v) : v);
            raw += RARE && !(w >= least) ? SaWeight::RAW : SaWeight::raw(w);
        });
        const int terms = b1 - b0 > lane ? ((b1 - b0 - lane - 1) / 32 + 1) * PER : 0;
        return sa_warp_sum(raw - (u64)terms * SaWeight::RAW);
    }
    EC_DEV u64 sum(int b0, int b1, int lane, double least) const {
        return infinite || least > 0.0 ? sum<true>(b0, b1, lane, least) : sum<false>(b0, b1, lane, least);
    }
};

// The warp of whose sum, in `part`, the point is part; `before` gains the
// sums ahead of it.
EC_DEV int dr_find(const u64 *part, u64 target, u64 &before) {
    int w = 0;
    while (w < DR_WARPS - 1 && before + part[w] <= target) before += part[w++];
    return w;
}

// Many rows without top-k and top-p: a CTA per row, which reads it twice, for
// the largest logit and for the sum, and then a 16th and a 256th of it to find
// the point.  The later readings come from L2: 1000 rows of 50257 fp32 logits
// (201 MB) read 201 MB of DRAM.  They take 111 us, 1.8 TB/s, bound by the
// instructions of the weights (about 30 for an element) and their dependence:
// the schedulers issue in 57 % of the cycles, the double pipe is busy in 26 %,
// DRAM in 22 %.  k_sample, whose SMs hold one row at a time and work on it or
// wait for it, takes 158; 16-bit logits take 100 us.  Smaller CTAs (4 of 256
// threads: 130 us) leave a longer tail and more rows in flight than L2 holds.
// Two CTAs of 512 threads leave 64 registers a thread, and 224 bytes spill (288
// with 16-bit logits); three would leave 40.
// The sums are the integers of k_sample, so the draws are the same.
template <int T> __global__ void __launch_bounds__(DR_THREADS, 2) k_sample_rows(const ec_sample_args a, int shift) {
    EC_PDL_ENTER();
    typedef DrRow<T> Row;
    constexpr int PER = Row::PER;
    __shared__ double tab[SA_TAB], part2[48];
    __shared__ float high[DR_WARPS];
    __shared__ int firsts[DR_WARPS];
    __shared__ u64 part[2][DR_WARPS];
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float temperature = a.temperature ? a.temperature[r] : 1.0f, min_p = a.min_p ? a.min_p[r] : 0.0f;
    Row row;
    row.src = static_cast<const typename Row::V *>(a.logits) + (size_t)r * a.ld;
    row.skew = (int)((reinterpret_cast<uintptr_t>(row.src) & 15) / Row::ELT);
    row.vocab = a.vocab;
    row.blocks = (row.skew + a.vocab + PER - 1) / PER;
    row.infinite = false;
    if (tid < 48) part2[tid] = exp2(tid < 16 ? (double)tid / 16 + shift : (double)(tid - 16) / SA_TAB);
    float mx = -INFINITY;
    row.each(0, row.blocks, tid, DR_THREADS, [&](float v, int) { mx = fmaxf(mx, v); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) high[warp] = mx;
    __syncthreads();
    for (int j = tid; j < SA_TAB; j += DR_THREADS) tab[j] = part2[j / 32] * part2[16 + j % 32];
    for (int w = 0; w < DR_WARPS; ++w) mx = fmaxf(mx, high[w]);
    __syncthreads();
    if (mx == -INFINITY) {
        if (tid == 0) {
            a.ids[r] = -1;
            if (a.prob) a.prob[r] = 0.0f;
        }
        return;
    }
    if (!(temperature > 0.0f) || min_p > 1.0f) {   // the first of the largest
        int first = 0x7fffffff;
        row.each(0, row.blocks, tid, DR_THREADS, [&](float v, int p) {
            if (v == mx) first = min(first, p - row.skew);
        });
        first = __reduce_min_sync(0xffffffffu, first);
        if (lane == 0) firsts[warp] = first;
        __syncthreads();
        if (tid == 0) {
            for (int w = 0; w < DR_WARPS; ++w) first = min(first, firsts[w]);
            a.ids[r] = first;
            if (a.prob) a.prob[r] = 1.0f;
        }
        return;
    }
    row.infinite = mx == INFINITY;
    if (row.infinite) mx = 0.0f;
    // as in k_sample
    const double vanish = (double)temperature * 0.6931471805599453 * (shift + 3), per_nat = 512.0 * 1.4426950408889634 / (double)temperature;
    row.weight = {(double)mx, per_nat, fmaxf(__double2float_ru((double)mx - vanish), -FLT_MAX), tab};
    const double least = min_p > 0.0f ? (double)min_p * (double)(1ull << shift) : 0.0;
    // each warp's piece of the row, then the pieces of the one with the point
    int b0 = 0, b1 = row.blocks;
    u64 before = 0, target = 0, total = 0;
    for (int level = 0; level < 2; ++level) {
        const int piece = (b1 - b0 + DR_WARPS - 1) / DR_WARPS;
        const u64 mine = row.sum(min(b1, b0 + warp * piece), min(b1, b0 + (warp + 1) * piece), lane, least);
        if (lane == 0) part[level][warp] = mine;
        __syncthreads();
        if (level == 0) {
            for (int w = 0; w < DR_WARPS; ++w) total += part[0][w];
            target = sa_point(a.u[r], total);
        }
        const int w = dr_find(part[level], target, before);
        const int from = min(b1, b0 + w * piece);
        b1 = min(b1, b0 + (w + 1) * piece);
        b0 = from;
    }
    // the piece's elements in order, a warp at a time
    if (warp != 0) return;
    for (int p0 = b0 * PER; p0 < b1 * PER; p0 += 32) {
        const float v = row.at(p0 + lane);
        const double x = row.weight(v);
        const u64 mine = p0 + lane < b1 * PER && x >= least ? SaWeight::whole(x) : 0ull;
        u64 upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        upto += before;
        if (upto > target && upto - mine <= target) {
            a.ids[r] = p0 + lane - row.skew;
            if (a.prob) a.prob[r] = (float)(x / (double)total);
        }
        before = __shfl_sync(0xffffffffu, upto, 31);
        if (before > target) return;
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
    // 148 rows of 50257: 22 us, 28 as clusters; 400 rows of 1000: 15 and 13 us,
    // 4000 of 10000: 144 and 145 us
    if (!a.top_k && !a.top_p && a.rows >= num_sms && a.vocab >= DR_VOCAB) {
        k_sample_rows<T><<<a.rows, DR_THREADS, 0, stream>>>(a, shift);
        return (int)cudaGetLastError();
    }
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
