/*
 * ec_serve.h -- internal interface between the checks of the serving
 * operators (ec_serve.c) and their kernels (ec_tree.cu, ec_pages.cu,
 * ec_sample.cu).  Every launcher enqueues on `stream` and returns a
 * cudaError_t-compatible int; its arguments have passed the checks.  `err`
 * is the device error word (ec_error_word).
 */
#ifndef EC_SERVE_H
#define EC_SERVE_H

#include "edgecore_b200.h"
#include <cuda_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

int ec_launch_tree_attention(const ec_kv_pages *kv, const ec_tree_attn *a, int num_sms, int *err, cudaStream_t stream);
size_t ec_tree_attention_bytes(int n_seq, int rows, int n_head, int n_kv_head, int head_dim, int max_len, int num_sms);
int ec_launch_tree_commit(const ec_kv_pages *kv, const ec_tree_path *a, int *err, cudaStream_t stream);
int ec_launch_kv_copy(const ec_kv_pages *kv, int n, const int *src, const int *dst, const int *start, const int *end,
                      int num_sms, int *err, cudaStream_t stream);

#define EC_KV_COPY_MAX 4096          /* jobs of a call: every CTA keeps a flag of each */

typedef struct {
    int *ids;
    float *prob;
    const void *logits;
    long long ld;
    int type, rows, vocab;
    const float *temperature;
    const int *top_k;
    const float *top_p, *min_p, *u;
} ec_sample_args;
int ec_launch_sample(const ec_sample_args *a, int num_sms, int *err, cudaStream_t stream);
#define EC_SAMPLE_MAX_VOCAB 750000   /* a cluster of 16 CTAs holds a row in shared memory */

#ifdef __cplusplus
}
#endif

#endif /* EC_SERVE_H */
