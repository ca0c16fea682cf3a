// ec_pages.cu -- moving rows of a paged KV arena: the accepted path of a
// drafted tree to the front of its rows (ec_tree_commit), and a slot's rows
// to other slots (ec_kv_copy).
#include "ec_common.cuh"
#include "ec_serve.h"

namespace {

constexpr int PG_THREADS = 256;
constexpr int PG_NODES = 512;               // nodes of a tree that a block walks at a time
constexpr int PG_BATCH = 8;                 // rows of a column in flight
constexpr int PG_SHARES = 4;                // CTAs of a sequence, at most
constexpr int PC_VECTORS = 8;               // 16-byte vectors of a thread in flight
constexpr int PC_JOBS = EC_KV_COPY_MAX;

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

// As pg_row, -1 without a report where there is no page.
EC_DEV long long pg_row_quiet(const ec_kv_pages &kv, int slot, int p) {
    const int page = __ldg(kv.page_table + (size_t)slot * kv.pages_per_slot + p / EC_KV_PAGE);
    return page < 0 || page >= kv.n_pages ? -1 : (long long)page * kv.ld_page + (long long)(p % EC_KV_PAGE) * kv.ld_pos;
}

EC_DEV uint16_t *pg_column(const ec_kv_pages &kv, int i, int cols) {   // the i-th 16 bytes of a position, over layers, K then V
    const int layer = i / (2 * cols), c = i % (2 * cols);
    return static_cast<uint16_t *>(c < cols ? kv.k : kv.v) + (size_t)layer * kv.ld_layer + (size_t)(c % cols) * 8;
}

// The accepted path.  A node continues the path if its token is the choice
// after its parent, so one pass over the nodes, all at once, leaves at each
// node its first such child, and the walk itself reads shared memory only:
// three dependent reads of global memory (the sequence, its nodes with their
// pages, the rows to move), where a search per step would pay two for every
// accepted token.  Nodes come in blocks of PG_NODES; the path goes on from
// its last node in the next block, and rows move block by block.
// A cluster of CTAs has a sequence: each walks, and moves its share of the
// 16-byte columns.  A thread has PG_BATCH rows of a column in flight before
// it stores the first; the n-th node's index is at least n, so neither a
// batch nor a later block reads a row that was overwritten before.  Only the
// cluster's first CTA writes the results, after all have read base, which
// new_base may be.
// One stream (17 nodes, 24 layers of 128): 4.0 us, the latency of launch and
// three reads.  128 sequences of 41 nodes that accept 0 to 8, 28 layers of
// 256 (29 MB): 8.9 us, 3.3 TB/s, with 4 CTAs a sequence, which all fit at
// once; 18 us with 8, which do not, 10 us with 2; 9.4 us with 4 rows in flight.
__global__ void __launch_bounds__(PG_THREADS, 4) k_tree_commit(const ec_kv_pages kv, const ec_tree_path a, int shares, int *err) {
    EC_PDL_ENTER();
    __shared__ int s_child[PG_NODES], s_token[PG_NODES], s_picked[PG_NODES], s_path[PG_NODES];
    __shared__ long long s_row[PG_NODES], s_from[PG_NODES], s_to[PG_NODES];
    __shared__ int s_found, s_tip_child;
    const int tid = threadIdx.x, b = (int)(blockIdx.x / shares), share = (int)(blockIdx.x % shares);
    const int r0 = a.row_start[b], r1 = a.row_start[b + 1], base = a.base[b], slot = a.slots ? a.slots[b] : b;
    const bool good = r0 >= 0 && r1 >= r0 && r1 <= a.rows && base >= 0 && slot >= 0 && slot < kv.n_slots &&
                      (long long)base + (r1 - r0) <= (long long)kv.pages_per_slot * EC_KV_PAGE;
    if (!good && tid == 0) atomicCAS(err, 0, EC_KERR_BAD_INDEX);
    const int n = good ? r1 - r0 : 0, words = min(a.mask_words, (n + 63) / 64);
    const int cols = kv.dim / 8, all = kv.n_layers * 2 * cols;
    int len = 0, tip = -1, tip_picked = 0;   // the path so far, its last node and the choice after it
    for (int c0 = 0; c0 < n && len < a.max_path; c0 += PG_NODES) {
        const int block = min(PG_NODES, n - c0);
        for (int i = tid; i < block; i += PG_THREADS) {
            s_token[i] = a.tokens[r0 + c0 + i];
            s_picked[i] = a.picked[r0 + c0 + i];
            s_row[i] = pg_row_quiet(kv, slot, base + c0 + i);
            s_child[i] = n;
        }
        if (tid == 0) s_tip_child = c0 == 0 ? 0 : n;   // the path starts at node 0
        __syncthreads();
        for (int i = tid; i < block; i += PG_THREADS) {
            const int c = c0 + i;
            if (c == 0 || c / 64 >= words) continue;
            const int up = pg_parent(a.mask + (size_t)(r0 + c) * a.mask_words, c);
            if (up >= c0) {
                if (s_token[i] == s_picked[up - c0]) atomicMin(&s_child[up - c0], c);
            } else if (up >= 0 && up == tip && s_token[i] == tip_picked) {
                atomicMin(&s_tip_child, c);
            }
        }
        __syncthreads();
        if (tid == 0) {
            int found = 0;
            for (int node = s_tip_child; node < n && len + found < a.max_path; node = s_child[node - c0]) s_path[found++] = node - c0;
            s_found = found;
        }
        __syncthreads();
        const int found = s_found;
        for (int i = tid; i < found; i += PG_THREADS) {
            const int from = s_path[i], to = len + i;
            long long src = s_row[from], dst = -1;
            if (c0 + from != to) {
                dst = to >= c0 ? s_row[to - c0] : pg_row_quiet(kv, slot, base + to);
                if (src < 0 || dst < 0) atomicCAS(err, 0, EC_KERR_BAD_INDEX);
            }
            s_from[i] = src;
            s_to[i] = src < 0 ? -1 : dst;
            if (share == 0) a.accepted[(size_t)b * a.max_path + to] = s_picked[from];
        }
        if (found) {
            tip = c0 + s_path[found - 1];
            tip_picked = s_picked[tip - c0];
        }
        __syncthreads();
        int first = 0;   // nodes that stay where they are
        while (first < found && s_path[first] + c0 == len + first) ++first;
        for (int i = share * PG_THREADS + tid; i < all; i += shares * PG_THREADS) {
            uint16_t *p = pg_column(kv, i, cols);
            for (int m = first; m < found; m += PG_BATCH) {
                uint4 x[PG_BATCH];
#pragma unroll
                for (int t = 0; t < PG_BATCH; ++t)
                    if (m + t < found && s_to[m + t] >= 0) x[t] = *reinterpret_cast<const uint4 *>(p + s_from[m + t]);
#pragma unroll
                for (int t = 0; t < PG_BATCH; ++t)
                    if (m + t < found && s_to[m + t] >= 0) *reinterpret_cast<uint4 *>(p + s_to[m + t]) = x[t];
            }
        }
        len += found;
        __syncthreads();
    }
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    if (share == 0)
        for (int i = len + tid; i < a.max_path; i += PG_THREADS) a.accepted[(size_t)b * a.max_path + i] = -1;
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (share == 0 && tid == 0) {
        a.n_accepted[b] = len;
        a.new_base[b] = base + len;
    }
}

// Jobs with one source and range are a group, and a group's rows are read
// once and written to every member: n forks of a prompt cost one read and n
// writes.  Every CTA judges all jobs (flags in shared memory), counts the
// groups' units -- PC_VECTORS x PG_THREADS vectors of 16 bytes, of one layer's
// K or V and within one page -- and takes every gridDim-th.  16 forks of 1733
// positions, 28 layers of 256 (845 MB): 153 us, 5.5 TB/s, bound by the writes
// (264 us when every job read for itself; 155 us with 4 vectors and twice the
// CTAs).  One fork of 45 positions, 12 layers of 768: 5.7 us, half of it the
// judging; 8 CTAs an SM take 6.4 us, 2 take 5.0 us but 158 us for the 16.
__global__ void __launch_bounds__(PG_THREADS) k_kv_copy(const ec_kv_pages kv, int n, const int *src, const int *dst,
                                                        const int *start, const int *end, int *err) {
    EC_PDL_ENTER();
    __shared__ int4 s_job[PG_THREADS];
    __shared__ unsigned char s_flag[PC_JOBS];         // 1: skipped, 2: not its group's first
    __shared__ unsigned short s_member[PC_JOBS];      // the group's jobs that are not skipped
    __shared__ long long s_warp[PG_THREADS / 32], s_sum[PG_THREADS], s_to[PG_THREADS];
    __shared__ int s_members;
    const int tid = threadIdx.x;
    // a job refused for itself: it writes and reads nothing, so it meets no other
    const auto refused = [&](int4 j) {
        return j.x < 0 || j.x >= kv.n_slots || j.y < 0 || j.y >= kv.n_slots || j.z < 0 ||
               (long long)j.w > (long long)kv.pages_per_slot * EC_KV_PAGE || (j.x == j.y && j.z < j.w);
    };
    const auto load = [&](int j) {   // a refused job as an empty range that is nobody's
        const int4 v = make_int4(src[j], dst[j], start[j], end[j]);
        return refused(v) ? make_int4(-1, -1, 0, 0) : v;
    };
    // up to PG_THREADS jobs s_job keeps all of them
    const auto job = [&](int j) { return n <= PG_THREADS ? s_job[j] : load(j); };
    for (int j0 = 0; j0 < n; j0 += PG_THREADS) {
        const int j = j0 + tid;
        const int4 me = j < n ? load(j) : make_int4(0, 0, 0, 0);
        bool bad = me.x < 0, later = bad;
        for (int i0 = 0; i0 < n; i0 += PG_THREADS) {
            __syncthreads();
            if (i0 + tid < n) s_job[tid] = i0 == j0 ? me : load(i0 + tid);
            __syncthreads();
            const int m = min(PG_THREADS, n - i0);
            for (int i = 0; i < m; ++i) {
                const int4 o = s_job[i];
                if (i0 + i == j) continue;
                if (max(me.z, o.z) < min(me.w, o.w) && (o.y == me.y || o.x == me.y || o.y == me.x)) bad = true;
                if (i0 + i < j && o.x == me.x && o.z == me.z && o.w == me.w) later = true;
            }
        }
        if (j < n) {
            s_flag[j] = (bad ? 1 : 0) | (later ? 2 : 0);
            if (bad && blockIdx.x == 0) atomicCAS(err, 0, EC_KERR_BAD_INDEX);
        }
    }
    const int cols = kv.dim / 8;
    int rows = EC_KV_PAGE;   // of a unit; it divides a page
    while (rows > 1 && rows * cols > PC_VECTORS * PG_THREADS) rows /= 2;
    long long done = 0;
    for (int j0 = 0; j0 < n; j0 += PG_THREADS) {
        const int j = j0 + tid;
        long long units = 0;
        __syncthreads();
        if (j < n && !(s_flag[j] & 2)) {
            const int4 me = job(j);
            const int p0 = me.z, p1 = me.w;
            if (p0 < p1)
                units = (long long)((p1 - 1) / rows - p0 / rows + 1) * 2 * kv.n_layers;
        }
        for (int step = 1; step < 32; step *= 2) {
            const long long before = __shfl_up_sync(~0u, units, step);
            if (tid % 32 >= step) units += before;
        }
        if (tid % 32 == 31) s_warp[tid / 32] = units;
        __syncthreads();
        for (int w = 0; w < tid / 32; ++w) units += s_warp[w];
        s_sum[tid] = units;
        __syncthreads();
        const long long total = s_sum[PG_THREADS - 1];
        int at = -1;
        // done counts the units of earlier blocks of jobs
        for (long long u = (blockIdx.x + gridDim.x - done % gridDim.x) % gridDim.x; u < total; u += gridDim.x) {
            int low = 0, high = PG_THREADS - 1;
            while (low < high) {
                const int mid = (low + high) / 2;
                if (s_sum[mid] > u) high = mid;
                else low = mid + 1;
            }
            const int4 lead = job(j0 + low);
            if (low != at) {
                at = low;
                __syncthreads();
                if (tid == 0) s_members = 0;
                __syncthreads();
                for (int i = tid; i < n; i += PG_THREADS) {
                    const int4 me = job(i);
                    if (!(s_flag[i] & 1) && me.x == lead.x && me.z == lead.z && me.w == lead.w)
                        s_member[atomicAdd(&s_members, 1)] = (unsigned short)i;   // any order: targets are apart
                }
                __syncthreads();
            }
            const int members = s_members;
            if (members == 0) continue;
            const int blocks = (lead.w - 1) / rows - lead.z / rows + 1;
            const long long v = u - (low ? s_sum[low - 1] : 0);
            const int layer = (int)(v / blocks), block = (int)(v % blocks) + lead.z / rows;   // layer: K then V of each
            const int p0 = max(lead.z, block * rows), count = (min(lead.w, (block + 1) * rows) - p0) * cols;
            uint16_t *plane = static_cast<uint16_t *>(layer & 1 ? kv.v : kv.k) + (size_t)(layer / 2) * kv.ld_layer;
            const long long from = pg_row(kv, lead.x, p0, err);
            for (int m0 = 0; m0 < members; m0 += PG_THREADS) {
                const int m1 = min(PG_THREADS, members - m0);
                __syncthreads();
                if (tid < m1) s_to[tid] = pg_row(kv, job(s_member[m0 + tid]).y, p0, err);
                __syncthreads();
                if (from < 0) continue;
                for (int i0 = tid; i0 < count; i0 += PC_VECTORS * PG_THREADS) {
                    uint4 x[PC_VECTORS];
                    long long o[PC_VECTORS];
#pragma unroll
                    for (int t = 0; t < PC_VECTORS; ++t) {
                        const int i = i0 + t * PG_THREADS;
                        o[t] = (long long)(i / cols) * kv.ld_pos + (i % cols) * 8;
                        if (i < count) x[t] = *reinterpret_cast<const uint4 *>(plane + from + o[t]);
                    }
                    for (int m = 0; m < m1; ++m) {
                        const long long to = s_to[m];
                        if (to < 0) continue;
#pragma unroll
                        for (int t = 0; t < PC_VECTORS; ++t)
                            if (i0 + t * PG_THREADS < count) *reinterpret_cast<uint4 *>(plane + to + o[t]) = x[t];
                    }
                }
            }
        }
        done += total;
    }
}

}  // namespace

extern "C" int ec_launch_tree_commit(const ec_kv_pages *kv, const ec_tree_path *a, int *err, cudaStream_t stream) {
    const int columns = kv->n_layers * 2 * (kv->dim / 8);
    int shares = 1;
    while (shares < PG_SHARES && shares * PG_THREADS < columns) shares *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(PG_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)shares;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3((unsigned)shares * (unsigned)a->n_seq);
    return (int)cudaLaunchKernelEx(&cfg, k_tree_commit, *kv, *a, shares, err);
}

extern "C" int ec_launch_kv_copy(const ec_kv_pages *kv, int n, const int *src, const int *dst, const int *start,
                                 const int *end, int num_sms, int *err, cudaStream_t stream) {
    k_kv_copy<<<4 * num_sms, PG_THREADS, 0, stream>>>(*kv, n, src, dst, start, end, err);
    return (int)cudaGetLastError();
}
