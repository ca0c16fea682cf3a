// ec_tree.cu -- attention of drafted-token trees over a paged KV arena
// (ec_tree_attention).
#include "ec_common.cuh"
#include "ec_serve.h"

namespace {

constexpr int TA_THREADS = 128, TA_WARPS = TA_THREADS / 32, TA_DIMS = 8;   // dimensions per lane at most (head_dim 256)

template <int T> EC_DEV float ta_load(const void *p, size_t i) {
    if (T == EC_T_F32) return static_cast<const float *>(p)[i];
    return ec_h2f(static_cast<const uint16_t *>(p)[i], T == EC_T_BF16);
}

template <int T> EC_DEV void ta_store(void *p, size_t i, float v) {
    if (T == EC_T_F32) static_cast<float *>(p)[i] = v;
    else if (T == EC_T_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// One CTA per (row, query head): each warp takes every TA_WARPS-th position
// with a running maximum and sum, then the warps' parts are joined.
template <int QT, int KT>
__global__ void __launch_bounds__(TA_THREADS) k_tree_simple(const ec_kv_pages kv, const ec_tree_attn a, int *err) {
    EC_PDL_ENTER();
    __shared__ float sm[TA_WARPS], sl[TA_WARPS], so[TA_WARPS][256];
    const int row = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int lo = 0, hi = a.n_seq;   // the sequence whose rows hold `row`: the last one that starts at or before it
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.row_start[mid] <= row) lo = mid; else hi = mid;
    }
    const int b = lo, r0 = a.row_start[b], r1 = a.row_start[b + 1];
    if (row < r0 || row >= r1) return;
    const int n = r1 - r0, base = a.base[b], slot = a.slots ? a.slots[b] : b;
    if (r0 < 0 || r1 > a.rows || base < 0 || slot < 0 || slot >= kv.n_slots || (long long)base + n > (long long)kv.pages_per_slot * EC_KV_PAGE) {
        if (threadIdx.x == 0) atomicCAS(err, 0, EC_KERR_BAD_INDEX);
        return;
    }
    const unsigned long long *mask = a.mask + (size_t)row * a.mask_words;
    int depth = -1;
    for (int w = 0; w < a.mask_words; ++w) depth += __popcll(mask[w]);
    const int from = a.window > 0 ? base + depth - a.window + 1 : 0;   // lowest position that is seen
    const int hd = a.head_dim, kh = h / (a.n_head / a.n_kv_head);
    const float scale = a.scale > 0.0f ? a.scale : rsqrtf((float)hd);
    float q[TA_DIMS], o[TA_DIMS], m = -INFINITY, l = 0.0f;
    for (int i = 0; i < TA_DIMS; ++i) {
        const int d = lane + 32 * i;
        q[i] = d < hd ? ta_load<QT>(a.q, (size_t)row * a.ldq + (size_t)h * hd + d) * scale : 0.0f;
        o[i] = 0.0f;
    }
    for (int p = (from > 0 ? from : 0) / TA_WARPS * TA_WARPS + warp; p < base + n; p += TA_WARPS) {
        const int j = p - base;
        if (j < 0) {
            if (p < from) continue;
        } else {
            if (j / 64 >= a.mask_words || !(mask[j / 64] >> (j % 64) & 1)) continue;
            if (a.window > 0) {
                int dj = -1;
                for (int w = 0; w < a.mask_words; ++w) dj += __popcll(a.mask[(size_t)(r0 + j) * a.mask_words + w]);
                if (base + dj < from) continue;
            }
        }
        int page = kv.page_table[(size_t)slot * kv.pages_per_slot + p / EC_KV_PAGE];
        if (page < 0 || page >= kv.n_pages) {
            if (lane == 0) atomicCAS(err, 0, EC_KERR_BAD_INDEX);
            page = 0;
        }
        const size_t at = (size_t)page * kv.ld_page + (size_t)(p % EC_KV_PAGE) * kv.ld_pos + (size_t)kh * hd;
        float s = 0.0f;
        for (int i = 0; i < TA_DIMS; ++i)
            if (lane + 32 * i < hd) s = fmaf(q[i], ta_load<KT>(kv.k, at + lane + 32 * i), s);
        s = ec_warp_sum(s);
        const float mn = fmaxf(m, s), safe = mn == -INFINITY ? 0.0f : mn;   // NaN scores pass into the sums
        const float c = expf(m - safe), w = expf(s - safe);
        l = l * c + w;
        for (int i = 0; i < TA_DIMS; ++i)
            if (lane + 32 * i < hd) o[i] = fmaf(w, ta_load<KT>(kv.v, at + lane + 32 * i), o[i] * c);
        m = mn;
    }
    if (lane == 0) { sm[warp] = m; sl[warp] = l; }
    for (int i = 0; i < TA_DIMS; ++i) so[warp][lane + 32 * i] = o[i];
    __syncthreads();
    float mx = -INFINITY, total = 0.0f;
    for (int w = 0; w < TA_WARPS; ++w) mx = fmaxf(mx, sm[w]);
    if (mx == -INFINITY) mx = 0.0f;
    for (int w = 0; w < TA_WARPS; ++w) total += sl[w] * expf(sm[w] - mx);
    for (int d = threadIdx.x; d < hd; d += TA_THREADS) {
        float v = 0.0f;
        for (int w = 0; w < TA_WARPS; ++w) v += so[w][d] * expf(sm[w] - mx);
        ta_store<QT>(a.out, (size_t)row * a.ldo + (size_t)h * hd + d, total == 0.0f ? 0.0f : v / total);
    }
}

}  // namespace

extern "C" size_t ec_tree_attention_bytes(int, int, int, int, int, int, int) { return 0; }

extern "C" int ec_launch_tree_attention(const ec_kv_pages *kv, const ec_tree_attn *a, int, int *err, cudaStream_t stream) {
    const dim3 grid(a->rows, a->n_head);
    const bool bf = kv->type == EC_T_BF16;
    if (a->type == EC_T_F32 && !bf) k_tree_simple<EC_T_F32, EC_T_F16><<<grid, TA_THREADS, 0, stream>>>(*kv, *a, err);
    else if (a->type == EC_T_F32) k_tree_simple<EC_T_F32, EC_T_BF16><<<grid, TA_THREADS, 0, stream>>>(*kv, *a, err);
    else if (!bf) k_tree_simple<EC_T_F16, EC_T_F16><<<grid, TA_THREADS, 0, stream>>>(*kv, *a, err);
    else k_tree_simple<EC_T_BF16, EC_T_BF16><<<grid, TA_THREADS, 0, stream>>>(*kv, *a, err);
    return (int)cudaGetLastError();
}
