/*
 * The Qwen3 text model's structures, shared by its encoder (qwen3.c) and its
 * use as a language model (qwen3_lm.c).
 */
#ifndef IRIS_QWEN3_INTERNAL_H
#define IRIS_QWEN3_INTERNAL_H

#include "iris_internal.h"

#define Q3_EPS 1e-6f        /* QWEN3_RMS_NORM_EPS */
#define Q3_MAX_SEQ 512      /* QWEN3_MAX_SEQ_LEN: the reference pads every prompt to it */

typedef struct {
    uint16_t *w_qkv;   /* [(nh + 2 nkv) * 128, H] */
    uint16_t *w_o;     /* [H, nh * 128] */
    uint16_t *w_gu;    /* [2F, H], gate/up rows interleaved in blocks of 128 */
    uint16_t *w_down;  /* [H, F] */
    float *ln1, *ln2, *qn, *kn;
    CUtensorMap tm_qkv, tm_o, tm_gu, tm_down;
} q3_layer_t;

typedef struct {
    int valid, S;
    int *ids;
    uint8_t *mask;
    float *x, *qkv, *out, *cosb, *sinb;
    float *ws;          /* split-K workspace of the H-wide projections (few output tiles at 512 rows) */
    size_t ws_bytes;
    uint16_t *xn, *q, *k, *v, *attn, *mlp;
    CUtensorMap tm_xn, tm_attn, tm_mlp;
    cudaGraph_t graph;
    cudaGraphExec_t gexec;
    int graph_ok, graph_mode;
    uint64_t graph_kernels;
} q3_plan_t;

struct iris_cuda_qwen3 {
    iris_cuda_qwen3_config_t cfg;
    int mode;              /* 0 Flux, 1 Z-Image extraction */
    int nlayers;           /* layers held on the device */
    uint16_t *embed;       /* [vocab, H] */
    q3_layer_t *layers;
    float *ones;           /* [H] gate of the residual GEMM epilogues */
    /* the language model's end (load_lm / random_lm; NULL in an encoder) */
    float *norm;           /* [H] */
    uint16_t *head;        /* [head_rows, H]: the embeddings, or weights of its own; rows >= vocab are 0 */
    int head_rows;         /* vocab rounded up to 128 (the GEMM's tile) */
    int head_own;          /* head is not embed */
    CUtensorMap tm_head;
    q3_plan_t plan;
    size_t weight_bytes;
    int sessions;          /* that use it; iris_cuda_qwen3_free waits for the last */
    int freed;
};

typedef struct {
    int rc;
    uint64_t kernels;
    /* profiling (iris_cuda_qwen3_profile): an event after every launch */
    iris_cuda_kernel_time_t *prof;
    cudaEvent_t *ev;
    int nprof, maxprof;
    double flops;  /* algorithmic FLOPs of the next accounted launch */
} q3_enq_t;

/* account a launch; an error stops the rest of the queue */
void iris_q3_done(q3_enq_t *E, cudaError_t e, const char *what, int n);
/* out[M, N] = a[M, K] b[N, K]^T through the given epilogue */
void iris_q3_gemm(q3_enq_t *E, const char *name, const CUtensorMap *ta, const CUtensorMap *tb, int M, int N, int K,
                  int mode, void *out, int ldo, const float *gate, void *mlp_out, int ld_mlp, float *ws,
                  size_t ws_bytes);

#endif
