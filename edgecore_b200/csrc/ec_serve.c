/*
 * ec_serve.c -- argument checks of the serving operators on device operands
 * (ec_tree_attention, ec_tree_commit, ec_kv_copy, ec_sample).  Everything the
 * host can know is refused here with a message, before any launch; indices in
 * device memory are checked by the kernels.
 */
#include "edgecore.h"
#include "edgecore_b200.h"
#include "ec_launch.h"
#include "ec_serve.h"

#include <cuda_runtime_api.h>
#include <stdarg.h>

#define EC_EXPORT __attribute__((visibility("default")))

static int refuse(const char *fmt, ...)
{
    char msg[400];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof msg, fmt, ap);
    va_end(ap);
    ec_set_error_text(msg);
    return -1;
}

/* The current device and its SM count; -1 with a message if there is none. */
static int current_device(const char *fn, int *dev, int *sms)
{
    static int known[64];
    if (cudaGetDevice(dev) != cudaSuccess || *dev < 0 || *dev >= 64) {
        cudaGetLastError();
        return refuse("%s: no usable CUDA device", fn);
    }
    if (!known[*dev]) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *dev) != cudaSuccess) {
            cudaGetLastError();
            return refuse("%s: no usable CUDA device", fn);
        }
        known[*dev] = n;
    }
    *sms = known[*dev];
    return 0;
}

typedef struct { const void *p; const char *name; int optional, align; } operand;

/* Every operand must be there and aligned to its elements: a kernel could only
 * answer a misaligned one with a fault. */
static int aligned(const char *fn, const operand *o, int n)
{
    for (int i = 0; i < n; i++) {
        if (!o[i].p && !o[i].optional) return refuse("%s: %s must not be NULL", fn, o[i].name);
        if ((uintptr_t)o[i].p & (uintptr_t)(o[i].align - 1))
            return refuse("%s: %s must be aligned to %d bytes", fn, o[i].name, o[i].align);
    }
    return 0;
}

/* Every operand must be memory of device `dev`. */
static int on_device(const char *fn, int dev, const operand *o, int n)
{
    for (int i = 0; i < n; i++) {
        struct cudaPointerAttributes at;
        if (!o[i].p) continue;
        if (cudaPointerGetAttributes(&at, o[i].p) != cudaSuccess) {
            cudaGetLastError();
            at.type = cudaMemoryTypeUnregistered;
        }
        if (at.type == cudaMemoryTypeManaged) continue;
        if (at.type != cudaMemoryTypeDevice) return refuse("%s: %s must be device memory", fn, o[i].name);
        if (at.device != dev)
            return refuse("%s: %s is memory of device %d, the current device is %d", fn, o[i].name, at.device, dev);
    }
    return 0;
}

static int launched(const char *fn, int e)
{
    if (!e) return 0;
    return refuse("%s: launch failed: CUDA error %d (%s)", fn, e, cudaGetErrorString((cudaError_t)e));
}

static int check_pages(const char *fn, const ec_kv_pages *kv)
{
    if (!kv) return refuse("%s: no arena", fn);
    if (kv->type != EC_T_F16 && kv->type != EC_T_BF16)
        return refuse("%s: the cache must be fp16 or bf16 (type %d)", fn, kv->type);
    if (kv->n_layers < 1 || kv->n_pages < 1 || kv->n_slots < 1 || kv->pages_per_slot < 1 || kv->dim < 1)
        return refuse("%s: empty arena (%d layers, %d pages, %d slots of %d, dim %d)", fn, kv->n_layers, kv->n_pages,
                      kv->n_slots, kv->pages_per_slot, kv->dim);
    if (kv->pages_per_slot > 0x7fffffff / EC_KV_PAGE)
        return refuse("%s: %d pages per slot: positions must fit 31 bits", fn, kv->pages_per_slot);
    if (kv->dim % 8 || kv->ld_pos % 8 || kv->ld_page % 8 || kv->ld_layer % 8 || ((uintptr_t)kv->k & 15) || ((uintptr_t)kv->v & 15))
        return refuse("%s: the arena's rows must be 16-byte aligned (dim %d, strides %lld / %lld / %lld)", fn, kv->dim,
                      kv->ld_layer, kv->ld_page, kv->ld_pos);
    if (kv->ld_pos < kv->dim || kv->ld_page < kv->dim || (kv->n_layers > 1 && kv->ld_layer < kv->dim))
        return refuse("%s: the arena's strides (%lld / %lld / %lld) overlap its rows of %d", fn, kv->ld_layer,
                      kv->ld_page, kv->ld_pos, kv->dim);
    return 0;
}

EC_EXPORT int ec_tree_attention(const ec_kv_pages *kv, const ec_tree_attn *a, void *stream)
{
    static const char fn[] = "ec_tree_attention";
    if (check_pages(fn, kv)) return -1;
    if (!a) return refuse("%s: no arguments", fn);
    if (a->type != EC_T_F32 && a->type != kv->type)
        return refuse("%s: q must be fp32 or of the cache's type (type %d, cache %d)", fn, a->type, kv->type);
    if (a->n_seq < 0 || a->rows < 0) return refuse("%s: n_seq %d, rows %d", fn, a->n_seq, a->rows);
    if (a->head_dim < 8 || a->head_dim > 256 || a->head_dim % 8)
        return refuse("%s: head_dim %d (a multiple of 8 up to 256)", fn, a->head_dim);
    if (a->n_kv_head < 1 || a->n_head < a->n_kv_head || a->n_head % a->n_kv_head)
        return refuse("%s: %d query heads over %d KV heads", fn, a->n_head, a->n_kv_head);
    if ((long long)a->n_kv_head * a->head_dim != kv->dim)
        return refuse("%s: %d KV heads of %d in an arena of dim %d", fn, a->n_kv_head, a->head_dim, kv->dim);
    const long long wide = (long long)a->n_head * a->head_dim;
    if (wide > (1 << 24) || a->n_kv_head > 65535) return refuse("%s: %d heads of %d", fn, a->n_head, a->head_dim);
    if (a->rows > 1 && (a->ldq < wide || a->ldo < wide))
        return refuse("%s: row strides %lld / %lld below %lld", fn, a->ldq, a->ldo, wide);
    if (a->mask_words < 1) return refuse("%s: mask_words %d", fn, a->mask_words);
    if (a->window < 0 || a->max_len < 0) return refuse("%s: window %d, max_len %d", fn, a->window, a->max_len);
    if (!(a->scale >= 0.0f) || a->scale > 3.0e38f) return refuse("%s: scale %g", fn, (double)a->scale);
    if ((long long)a->rows * (a->n_head / a->n_kv_head) > 0x3fffffffLL || a->n_seq > 0x3fffffff) return refuse("%s: %d rows", fn, a->rows);
    if (a->n_seq == 0 || a->rows == 0) return 0;
    const int elt = a->type == EC_T_F32 ? 4 : 2;
    const operand o[] = {{a->q, "q", 0, elt}, {a->out, "out", 0, elt}, {kv->k, "k", 0, 16}, {kv->v, "v", 0, 16},
                         {kv->page_table, "page_table", 0, 4}, {a->slots, "slots", 1, 4}, {a->row_start, "row_start", 0, 4},
                         {a->base, "base", 0, 4}, {a->mask, "mask", 0, 8}, {a->work, "work", 1, 256}};
    int dev, sms;
    if (aligned(fn, o, (int)(sizeof o / sizeof o[0]))) return -1;
    if (current_device(fn, &dev, &sms) || on_device(fn, dev, o, (int)(sizeof o / sizeof o[0]))) return -1;
    int *err = ec_error_word();
    if (!err) return refuse("%s: no device error word", fn);
    return launched(fn, ec_launch_tree_attention(kv, a, sms, err, (cudaStream_t)stream));
}

EC_EXPORT size_t ec_tree_attention_work(int n_seq, int rows, int n_head, int n_kv_head, int head_dim, int max_len)
{
    int dev, sms;
    if (n_seq < 1 || rows < 1 || n_kv_head < 1 || n_head < n_kv_head || head_dim < 1 || max_len < 0) return 0;
    if (current_device("ec_tree_attention_work", &dev, &sms)) return 0;
    return ec_tree_attention_bytes(n_seq, rows, n_head, n_kv_head, head_dim, max_len, sms);
}

EC_EXPORT int ec_tree_commit(const ec_kv_pages *kv, const ec_tree_path *a, void *stream)
{
    static const char fn[] = "ec_tree_commit";
    if (check_pages(fn, kv)) return -1;
    if (!a) return refuse("%s: no arguments", fn);
    if (a->n_seq < 0 || a->n_seq > 0x0fffffff || a->rows < 0) return refuse("%s: n_seq %d, rows %d", fn, a->n_seq, a->rows);
    if (a->mask_words < 1 || a->max_path < 1) return refuse("%s: mask_words %d, max_path %d", fn, a->mask_words, a->max_path);
    if (a->n_seq == 0) return 0;
    const int none = a->rows == 0;
    const operand o[] = {{kv->k, "k", 0, 16}, {kv->v, "v", 0, 16}, {kv->page_table, "page_table", 0, 4},
                         {a->slots, "slots", 1, 4}, {a->row_start, "row_start", 0, 4}, {a->base, "base", 0, 4},
                         {a->mask, "mask", none, 8}, {a->tokens, "tokens", none, 4}, {a->picked, "picked", none, 4},
                         {a->accepted, "accepted", 0, 4}, {a->n_accepted, "n_accepted", 0, 4}, {a->new_base, "new_base", 0, 4}};
    int dev, sms;
    if (aligned(fn, o, (int)(sizeof o / sizeof o[0]))) return -1;
    if (current_device(fn, &dev, &sms) || on_device(fn, dev, o, (int)(sizeof o / sizeof o[0]))) return -1;
    int *err = ec_error_word();
    if (!err) return refuse("%s: no device error word", fn);
    return launched(fn, ec_launch_tree_commit(kv, a, err, (cudaStream_t)stream));
}

EC_EXPORT int ec_kv_copy(const ec_kv_pages *kv, int n_copies, const int *src, const int *dst, const int *start,
                         const int *end, void *stream)
{
    static const char fn[] = "ec_kv_copy";
    if (check_pages(fn, kv)) return -1;
    if (n_copies < 0 || n_copies > EC_KV_COPY_MAX) return refuse("%s: %d copies (at most %d)", fn, n_copies, EC_KV_COPY_MAX);
    if (n_copies == 0) return 0;
    const operand o[] = {{kv->k, "k", 0, 16}, {kv->v, "v", 0, 16}, {kv->page_table, "page_table", 0, 4},
                         {src, "src", 0, 4}, {dst, "dst", 0, 4}, {start, "start", 0, 4}, {end, "end", 0, 4}};
    int dev, sms;
    if (aligned(fn, o, (int)(sizeof o / sizeof o[0]))) return -1;
    if (current_device(fn, &dev, &sms) || on_device(fn, dev, o, (int)(sizeof o / sizeof o[0]))) return -1;
    int *err = ec_error_word();
    if (!err) return refuse("%s: no device error word", fn);
    return launched(fn, ec_launch_kv_copy(kv, n_copies, src, dst, start, end, sms, err, (cudaStream_t)stream));
}

EC_EXPORT int ec_sample(int *ids, float *prob, const void *logits, int type, long long ld, int rows, int vocab,
                        const float *temperature, const int *top_k, const float *top_p, const float *min_p,
                        const float *u, void *stream)
{
    static const char fn[] = "ec_sample";
    if (type != EC_T_F32 && type != EC_T_F16 && type != EC_T_BF16) return refuse("%s: type %d", fn, type);
    if (rows < 0 || vocab < 1) return refuse("%s: rows %d, vocab %d", fn, rows, vocab);
    if (vocab > EC_SAMPLE_MAX_VOCAB) return refuse("%s: vocab %d (at most %d)", fn, vocab, EC_SAMPLE_MAX_VOCAB);
    if (rows > 0x07ffffff) return refuse("%s: rows %d", fn, rows);
    if (rows > 1 && ld < vocab) return refuse("%s: row stride %lld below vocab %d", fn, ld, vocab);
    if (rows == 0) return 0;
    const operand o[] = {{ids, "ids", 0, 4}, {prob, "prob", 1, 4}, {logits, "logits", 0, type == EC_T_F32 ? 4 : 2},
                         {temperature, "temperature", 1, 4}, {top_k, "top_k", 1, 4}, {top_p, "top_p", 1, 4},
                         {min_p, "min_p", 1, 4}, {u, "u", 0, 4}};
    int dev, sms;
    if (aligned(fn, o, (int)(sizeof o / sizeof o[0]))) return -1;
    if (current_device(fn, &dev, &sms) || on_device(fn, dev, o, (int)(sizeof o / sizeof o[0]))) return -1;
    const ec_sample_args a = {ids, prob, logits, ld, type, rows, vocab, temperature, top_k, top_p, min_p, u};
    int *err = ec_error_word();
    if (!err) return refuse("%s: no device error word", fn);
    return launched(fn, ec_launch_sample(&a, sms, err, (cudaStream_t)stream));
}
