// ec_sample.cu -- drawing one token per row of logits (ec_sample).
//
// Weights w = exp((logit - max) / T) are held as integers, w rounded to a
// multiple of 2^-shift with shift = 62 - ceil(log2 vocab): every sum of a
// row's weights fits 64 bits and is exact, so it does not depend on the order
// of its terms, atomics included.
#include "ec_common.cuh"
#include "ec_serve.h"

namespace {

constexpr int SA_THREADS = 1024, SA_WARPS = SA_THREADS / 32, SA_BINS = 256;
typedef unsigned long long u64;

// Order-preserving bits of a logit: NaN as -inf, -0 as +0.
EC_DEV uint32_t sa_key(float v) {
    if (!(v == v)) v = -INFINITY;
    if (v == 0.0f) v = 0.0f;
    const uint32_t b = __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

EC_DEV float sa_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

template <int T> EC_DEV float sa_load(const void *p, size_t i) {
    if (T == EC_T_F32) return static_cast<const float *>(p)[i];
    return ec_h2f(static_cast<const uint16_t *>(p)[i], T == EC_T_BF16);
}

// Weight of key k below the maximum mx in double.
EC_DEV double sa_exp(uint32_t k, float mx, double t) {
    const float v = sa_value(k);
    if (v == -INFINITY) return 0.0;
    if (mx == INFINITY) return v == INFINITY ? 1.0 : 0.0;
    return exp(((double)v - (double)mx) / t);
}

template <typename V, typename F> EC_DEV V sa_reduce(V v, V *part, F f) {   // over the CTA, to every thread
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < SA_WARPS; ++i) v = f(v, part[i]);
    return v;
}

// The key at which the running sum over descending keys (counts, or weights
// with `mass`) of the elements that `kept` lets through reaches `want`, and
// the sum above it.
struct SaCut { uint32_t key; u64 above; };

template <int T, bool MASS, typename K>
EC_DEV SaCut sa_select(const void *row, int n, float mx, double t, double one, u64 want, u64 *hist, K kept) {
    SaCut c = {0u, 0ull};
    for (int s = 24; s >= 0; s -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < SA_BINS; i += SA_THREADS) hist[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += SA_THREADS) {
            const uint32_t k = sa_key(sa_load<T>(row, i));
            if (s < 24 && (k >> (s + 8)) != (c.key >> (s + 8))) continue;
            if (!kept(k, i)) continue;
            const u64 w = MASS ? (u64)__double2ll_rn(sa_exp(k, mx, t) * one) : 1ull;
            if (w) atomicAdd(hist + ((k >> s) & 255u), w);
        }
        __syncthreads();
        int bin = SA_BINS - 1;
        while (bin > 0 && c.above + hist[bin] < want) c.above += hist[bin--];
        c.key |= (uint32_t)bin << s;
    }
    return c;
}

template <int T>
__global__ void __launch_bounds__(SA_THREADS) k_sample(const ec_sample_args a, int shift) {
    EC_PDL_ENTER();
    __shared__ u64 hist[SA_BINS], part[SA_THREADS];
    const int r = blockIdx.x, n = a.vocab;
    const char *row = static_cast<const char *>(a.logits) + (size_t)r * a.ld * (T == EC_T_F32 ? 4 : 2);
    const double t = a.temperature ? (double)a.temperature[r] : 1.0;
    const double one = (double)(1ull << shift);
    // the first of the largest: key, then lowest index
    u64 best = 0;
    for (int i = threadIdx.x; i < n; i += SA_THREADS) {
        const u64 k = (u64)sa_key(sa_load<T>(row, i)) << 32 | (uint32_t)(0x7fffffff - i);
        best = k > best ? k : best;
    }
    best = sa_reduce(best, part, [](u64 x, u64 y) { return x > y ? x : y; });
    const float mx = sa_value((uint32_t)(best >> 32));
    const int first = 0x7fffffff - (int)(uint32_t)best;
    const float min_p = a.min_p ? a.min_p[r] : 0.0f;
    const int top_k = a.top_k ? a.top_k[r] : 0;
    const float top_p = a.top_p ? a.top_p[r] : 1.0f;
    if (mx == -INFINITY || !(t > 0.0) || min_p > 1.0f || top_k == 1 || top_p <= 0.0f) {
        if (threadIdx.x == 0) {
            a.ids[r] = mx == -INFINITY ? -1 : first;
            if (a.prob) a.prob[r] = mx == -INFINITY ? 0.0f : 1.0f;
        }
        return;
    }
    // kept: keys above `cut`, and the first `ties` of the elements equal to it
    uint32_t cut = 0;
    u64 ties = ~0ull;
    // rank of element i among those equal to it would need a scan; `limit` is the
    // index behind the last tie that is kept instead
    int limit = n;
    auto set_limit = [&]() {   // index behind the `ties`-th element equal to cut
        // contiguous chunks, so that the count before an element is a prefix
        const int per = (n + SA_THREADS - 1) / SA_THREADS, b = min(n, (int)threadIdx.x * per), e = min(n, b + per);
        u64 c = 0;
        for (int i = b; i < e; ++i) c += sa_key(sa_load<T>(row, i)) == cut;
        __syncthreads();
        part[threadIdx.x] = c;
        __syncthreads();
        u64 before = 0;
        for (int i = 0; i < (int)threadIdx.x; ++i) before += part[i];
        __shared__ int at;
        if (threadIdx.x == 0) at = n;
        __syncthreads();
        if (before < ties && before + c >= ties)
            for (int i = b; i < e; ++i)
                if (sa_key(sa_load<T>(row, i)) == cut && ++before == ties) at = i + 1;
        __syncthreads();
        limit = at;
    };
    auto kept = [&](uint32_t k, int i) { return k > cut || (k == cut && i < limit); };
    if (top_k > 0 && top_k < n) {
        const SaCut c = sa_select<T, false>(row, n, mx, t, one, (u64)top_k, hist, [](uint32_t, int) { return true; });
        cut = c.key;
        ties = (u64)top_k - c.above;
        set_limit();
    }
    if (top_p < 1.0f) {
        u64 total = 0;
        for (int i = threadIdx.x; i < n; i += SA_THREADS) {
            const uint32_t k = sa_key(sa_load<T>(row, i));
            if (kept(k, i)) total += (u64)__double2ll_rn(sa_exp(k, mx, t) * one);
        }
        total = sa_reduce(total, part, [](u64 x, u64 y) { return x + y; });
        const u64 want = max(1ull, (u64)ceil((double)top_p * (double)total));
        const SaCut c = sa_select<T, true>(row, n, mx, t, one, want, hist, kept);
        const u64 w = (u64)__double2ll_rn(sa_exp(c.key, mx, t) * one);
        const u64 need = w ? (want - c.above + w - 1) / w : ~0ull;
        if (c.key > cut || need < ties) {
            cut = c.key;
            ties = need;
            set_limit();
        }
    }
    // weights of contiguous chunks, then of the chunk that holds the target
    auto weight = [&](int i) -> u64 {
        const uint32_t k = sa_key(sa_load<T>(row, i));
        if (!kept(k, i)) return 0ull;
        const double w = sa_exp(k, mx, t);
        return w >= (double)min_p ? (u64)__double2ll_rn(w * one) : 0ull;
    };
    const int per = (n + SA_THREADS - 1) / SA_THREADS, b = min(n, (int)threadIdx.x * per), e = min(n, b + per);
    u64 mine = 0;
    for (int i = b; i < e; ++i) mine += weight(i);
    __syncthreads();
    part[threadIdx.x] = mine;
    __syncthreads();
    u64 before = 0, total = 0;
    for (int i = 0; i < SA_THREADS; ++i) {
        if (i == (int)threadIdx.x) before = total;
        total += part[i];
    }
    const float u = a.u[r];
    const double x = u > 0.0f ? (double)u * (double)total : 0.0;
    u64 target = x >= (double)total ? total - 1 : (u64)x;   // the sum has to exceed it
    if (target >= total) target = total - 1;
    if (before <= target && target < before + mine) {
        for (int i = b; i < e; ++i) {
            const u64 w = weight(i);
            if (before + w > target) {
                a.ids[r] = i;
                if (a.prob) a.prob[r] = (float)(sa_exp(sa_key(sa_load<T>(row, i)), mx, t) * one / (double)total);
                break;
            }
            before += w;
        }
    }
}

}  // namespace

extern "C" int ec_launch_sample(const ec_sample_args *a, int, cudaStream_t stream) {
    int bits = 0;
    while ((1ll << bits) < a->vocab) ++bits;
    if (a->type == EC_T_F32) k_sample<EC_T_F32><<<a->rows, SA_THREADS, 0, stream>>>(*a, 62 - bits);
    else if (a->type == EC_T_F16) k_sample<EC_T_F16><<<a->rows, SA_THREADS, 0, stream>>>(*a, 62 - bits);
    else k_sample<EC_T_BF16><<<a->rows, SA_THREADS, 0, stream>>>(*a, 62 - bits);
    return (int)cudaGetLastError();
}
