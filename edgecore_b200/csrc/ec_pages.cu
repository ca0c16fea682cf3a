// ec_pages.cu -- moving rows of a paged KV arena: the accepted path of a
// drafted tree to the front of its rows (ec_tree_commit), and a slot's rows
// to other slots (ec_kv_copy).
#include "ec_common.cuh"
#include "ec_serve.h"

namespace {

constexpr int PG_THREADS = 256;

// Element offset of position p of `slot` in a layer; -1 (and the error word)
// when the page table names no page of the arena.
EC_DEV long long pg_row(const ec_kv_pages &kv, int slot, int p, int *err) {
    const int page = __ldg(kv.page_table + (size_t)slot * kv.pages_per_slot + p / EC_KV_PAGE);
    if (page < 0 || page >= kv.n_pages) {
        atomicCAS(err, 0, EC_KERR_BAD_INDEX);
        return -1;
    }
    return (long long)page * kv.ld_page + (long long)(p % EC_KV_PAGE) * kv.ld_pos;
}

EC_DEV int pg_parent(const unsigned long long *mask, int node) {   // highest bit below `node`, -1: none
    for (int w = node / 64; w >= 0; --w) {
        unsigned long long v = mask[w];
        if (w == node / 64) v &= (1ull << (node % 64)) - 1ull;
        if (v) return w * 64 + 63 - __clzll((long long)v);
    }
    return -1;
}

// One CTA per sequence: walk the tree, then move the rows of the path.  A
// thread owns 16-byte columns and takes the path in order: the n-th node's
// index is at least n, so no row is overwritten before it is read.
__global__ void __launch_bounds__(PG_THREADS) k_tree_commit(const ec_kv_pages kv, const ec_tree_path a, int *err) {
    EC_PDL_ENTER();
    __shared__ int next;
    const int b = blockIdx.x;
    const int r0 = a.row_start[b], r1 = a.row_start[b + 1], base = a.base[b], slot = a.slots ? a.slots[b] : b;
    const bool good = r0 >= 0 && r1 >= r0 && r1 <= a.rows && base >= 0 && slot >= 0 && slot < kv.n_slots &&
                      (long long)base + (r1 - r0) <= (long long)kv.pages_per_slot * EC_KV_PAGE;
    if (!good && threadIdx.x == 0) atomicCAS(err, 0, EC_KERR_BAD_INDEX);
    const int n = good ? r1 - r0 : 0;
    int len = 0, node = 0;
    const int words = min(a.mask_words, (n + 63) / 64);
    const int cols = kv.dim / 8;
    while (node < n && len < a.max_path) {
        const int pick = a.picked[r0 + node];
        if (threadIdx.x == 0) a.accepted[(size_t)b * a.max_path + len] = pick;
        if (node != len) {
            const long long from = pg_row(kv, slot, base + node, err), to = pg_row(kv, slot, base + len, err);
            if (from >= 0 && to >= 0)
                for (int i = threadIdx.x; i < kv.n_layers * 2 * cols; i += PG_THREADS) {
                    const int layer = i / (2 * cols), c = i % (2 * cols);
                    uint16_t *p = static_cast<uint16_t *>(c < cols ? kv.k : kv.v) + (size_t)layer * kv.ld_layer + (size_t)(c % cols) * 8;
                    *reinterpret_cast<uint4 *>(p + to) = *reinterpret_cast<const uint4 *>(p + from);
                }
        }
        ++len;
        if (threadIdx.x == 0) next = n;
        __syncthreads();
        for (int c = node + 1 + threadIdx.x; c < n; c += PG_THREADS)
            if (c / 64 < words && a.tokens[r0 + c] == pick && pg_parent(a.mask + (size_t)(r0 + c) * a.mask_words, c) == node)
                atomicMin(&next, c);
        __syncthreads();
        node = next;
        __syncthreads();
    }
    for (int i = len + threadIdx.x; i < a.max_path; i += PG_THREADS) a.accepted[(size_t)b * a.max_path + i] = -1;
    if (threadIdx.x == 0) {
        a.n_accepted[b] = len;
        a.new_base[b] = base + len;
    }
}

EC_DEV bool pg_overlap(int a0, int a1, int b0, int b1) { return max(a0, b0) < min(a1, b1); }

// One CTA per (job, 64-position stretch).
__global__ void __launch_bounds__(PG_THREADS) k_kv_copy(const ec_kv_pages kv, int n, const int *src, const int *dst,
                                                        const int *start, const int *end, int *err) {
    EC_PDL_ENTER();
    const int j = blockIdx.y, s = src[j], d = dst[j], p0 = start[j], p1 = end[j];
    bool bad = s < 0 || s >= kv.n_slots || d < 0 || d >= kv.n_slots || p0 < 0 ||
               (long long)p1 > (long long)kv.pages_per_slot * EC_KV_PAGE || (s == d && p0 < p1);
    for (int i = threadIdx.x; i < n; i += PG_THREADS)
        if (i != j && pg_overlap(p0, p1, start[i], end[i]) && (dst[i] == d || src[i] == d || dst[i] == s)) bad = true;
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0 && blockIdx.x == 0) atomicCAS(err, 0, EC_KERR_BAD_INDEX);
        return;
    }
    const int cols = kv.dim / 8;
    for (int p = p0 + (int)blockIdx.x; p < p1; p += gridDim.x) {
        const long long from = pg_row(kv, s, p, err), to = pg_row(kv, d, p, err);
        if (from < 0 || to < 0) continue;
        for (int i = threadIdx.x; i < kv.n_layers * 2 * cols; i += PG_THREADS) {
            const int layer = i / (2 * cols), c = i % (2 * cols);
            uint16_t *q = static_cast<uint16_t *>(c < cols ? kv.k : kv.v) + (size_t)layer * kv.ld_layer + (size_t)(c % cols) * 8;
            *reinterpret_cast<uint4 *>(q + to) = *reinterpret_cast<const uint4 *>(q + from);
        }
    }
}

}  // namespace

extern "C" int ec_launch_tree_commit(const ec_kv_pages *kv, const ec_tree_path *a, int *err, cudaStream_t stream) {
    k_tree_commit<<<a->n_seq, PG_THREADS, 0, stream>>>(*kv, *a, err);
    return (int)cudaGetLastError();
}

extern "C" int ec_launch_kv_copy(const ec_kv_pages *kv, int n, const int *src, const int *dst, const int *start,
                                 const int *end, int num_sms, int *err, cudaStream_t stream) {
    k_kv_copy<<<dim3((8 * num_sms + n - 1) / n, n), PG_THREADS, 0, stream>>>(*kv, n, src, dst, start, end, err);
    return (int)cudaGetLastError();
}
