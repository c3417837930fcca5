/*
 * The Qwen3 text model as a language model: sessions with a paged key-value
 * cache, fed any mix of prompts and single tokens.  The decoder layers are the
 * encoder's (qwen3.c) with its rotation and attention replaced by the
 * operators of lm_kernels.cu: the QKV projection's rows go through
 * iris_launch_rope_append into the layer's pages, and every row attends over
 * its sequence's pages.  Then the final norm, the head's GEMM, and the log
 * probabilities.  A step whose token count and top_k come again is a CUDA graph
 * (lm_run).
 */
#include "qwen3_internal.h"

#include <math.h>
#include <stdlib.h>
#include <string.h>

#define LM_PAGE 16          /* tokens of a page */
#define LM_MAX_TOKENS 8192  /* of a step: the logits are f32 [tokens, vocab] */
#define LM_SIZES 16         /* of steps, remembered */
#define LM_DRAW (-1)

/* a size of step: its graph, once captured */
typedef struct {
    int tokens, top_k;      /* tokens 0: none; top_k LM_DRAW: a token is drawn behind each */
    uint64_t used;          /* the step that last had it */
    cudaGraph_t graph;
    cudaGraphExec_t gexec;  /* NULL before its second step */
    uint64_t kernels;
} lm_size_t;

struct iris_cuda_qwen3_lm {
    iris_cuda_qwen3_t *m;
    int num_seqs, max_len, max_tokens, blocks;
    /* host: tokens each sequence holds, the same in the step being checked, and which step last named it */
    int *len, *next;
    uint64_t *named, step;
    /* device */
    int32_t *table;         /* [num_seqs, blocks], shared by all layers */
    uint16_t *pools;        /* [layers][k, v][pages, LM_PAGE, kv_heads, 128] */
    size_t pool_elems;      /* of one pool */
    int32_t *in, *h_in;     /* a step's ids, seq, pos, targets: [4][tokens]; the same on the host */
    float *x, *qkv, *logits, *ws;
    size_t ws_bytes;
    uint16_t *xn, *q, *attn, *mlp;
    void *attn_ws, *lp_ws;
    float *out;             /* logprob, entropy, top_logprobs: [2 + 32][max_tokens] */
    int32_t *out_ids;       /* [max_tokens, 32] */
    double *draw, *h_draw;  /* a step's settings of draws: uniform [tokens], then f32 temperature, top_p, min_p and int32 top_k
                               [4][tokens]; the same on the host */
    CUtensorMap tm_xn, tm_attn, tm_mlp;
    iris_gpu_rope_t rope;
    lm_size_t sizes[LM_SIZES];
};

static void lm_size_free(lm_size_t *z) {
    if (z->gexec) {
        cudaGraphExecDestroy(z->gexec);
        cudaGraphDestroy(z->graph);
    }
    memset(z, 0, sizeof(*z));
}

void iris_cuda_qwen3_lm_free(iris_cuda_qwen3_lm_t *lm) {
    if (!lm) return;
    if (g_rt.initialized) cudaStreamSynchronize(g_rt.stream);
    for (int i = 0; i < LM_SIZES; i++) lm_size_free(&lm->sizes[i]);
    void *b[] = {lm->table, lm->pools, lm->in, lm->x, lm->qkv, lm->logits, lm->ws, lm->xn, lm->q, lm->attn, lm->mlp,
                 lm->attn_ws, lm->lp_ws, lm->out, lm->out_ids, lm->draw};
    for (size_t i = 0; i < sizeof(b) / sizeof(b[0]); i++) iris_dfree(b[i]);
    free(lm->h_in);
    free(lm->h_draw);
    free(lm->len);
    free(lm->next);
    free(lm->named);
    iris_cuda_qwen3_t *m = lm->m;
    free(lm);
    if (--m->sessions == 0 && m->freed) iris_cuda_qwen3_free(m);
}

static void lm_cache(const iris_cuda_qwen3_lm_t *lm, int layer, iris_gpu_kv_cache_t *c) {
    const int nkv = lm->m->cfg.kv_heads;
    memset(c, 0, sizeof(*c));
    c->k = lm->pools + (size_t)(2 * layer) * lm->pool_elems;
    c->v = lm->pools + (size_t)(2 * layer + 1) * lm->pool_elems;
    c->table = lm->table;
    c->num_pages = lm->num_seqs * lm->blocks;
    c->page_size = LM_PAGE;
    c->kv_heads = nkv;
    c->head_dim = 128;
    c->num_seqs = lm->num_seqs;
    c->max_blocks = lm->blocks;
    c->table_stride = lm->blocks;
    c->head_stride = 128;
    c->token_stride = (int64_t)nkv * 128;
    c->page_stride = (int64_t)LM_PAGE * nkv * 128;
}

iris_cuda_qwen3_lm_t *iris_cuda_qwen3_lm_create(iris_cuda_qwen3_t *m, int num_seqs, int max_len, int max_tokens) {
    if (!m || !m->head) { iris_fail(IRIS_CUDA_ERR_ARG, "language model session: needs a model of load_lm / random_lm"); return NULL; }
    if (num_seqs < 1 || max_len < 1 || max_tokens < 1 || max_tokens > LM_MAX_TOKENS ||
        (int64_t)num_seqs * (((int64_t)max_len + LM_PAGE - 1) / LM_PAGE) > (1 << 30)) {
        iris_fail(IRIS_CUDA_ERR_ARG, "language model session: %d sequences of %d tokens, steps of %d (1..%d)", num_seqs,
                  max_len, max_tokens, LM_MAX_TOKENS);
        return NULL;
    }
    iris_cuda_qwen3_lm_t *lm = (iris_cuda_qwen3_lm_t *)calloc(1, sizeof(*lm));
    if (!lm) { iris_fail(IRIS_CUDA_ERR_OOM, "language model session"); return NULL; }
    const iris_cuda_qwen3_config_t *c = &m->cfg;
    lm->m = m;
    m->sessions++;
    lm->num_seqs = num_seqs;
    lm->max_len = max_len;
    lm->max_tokens = max_tokens;
    lm->blocks = (int)(((int64_t)max_len + LM_PAGE - 1) / LM_PAGE);
    const size_t T = (size_t)max_tokens, H = (size_t)c->hidden, F = (size_t)c->intermediate;
    const size_t qd = (size_t)c->heads * 128, nq = (size_t)(c->heads + 2 * c->kv_heads) * 128;
    const size_t pages = (size_t)num_seqs * lm->blocks;
    lm->pool_elems = pages * LM_PAGE * c->kv_heads * 128;
    int rc = 0;
    iris_gpu_kv_cache_t cache;
    lm_cache(lm, 0, &cache);
    lm->len = (int *)calloc((size_t)num_seqs, sizeof(int));
    lm->next = (int *)calloc((size_t)num_seqs, sizeof(int));
    lm->named = (uint64_t *)calloc((size_t)num_seqs, sizeof(uint64_t));
    lm->h_in = (int32_t *)malloc(4 * T * 4);
    lm->h_draw = (double *)malloc(24 * T);
    if (!lm->len || !lm->next || !lm->named || !lm->h_in || !lm->h_draw) rc = iris_fail(IRIS_CUDA_ERR_OOM, "language model session");
#define ALLOC(dst, bytes) \
    do { if (!rc && !((dst) = iris_dmalloc(bytes))) rc = iris_fail(IRIS_CUDA_ERR_OOM, "language model session"); } while (0)
    ALLOC(lm->table, pages * 4);
    ALLOC(lm->pools, (size_t)2 * c->layers * lm->pool_elems * 2);
    ALLOC(lm->in, 4 * T * 4);
    ALLOC(lm->x, T * H * 4);
    ALLOC(lm->qkv, T * nq * 4);
    ALLOC(lm->logits, T * m->head_rows * 4);
    lm->ws_bytes = 4 * T * H * 4;  /* split-K partial sums of the H-wide projections */
    ALLOC(lm->ws, lm->ws_bytes);
    ALLOC(lm->xn, T * H * 2);
    ALLOC(lm->q, T * qd * 2);
    ALLOC(lm->attn, T * qd * 2);
    ALLOC(lm->mlp, T * F * 2);
    ALLOC(lm->attn_ws, iris_paged_attention_ws_bytes(&cache, c->heads, g_rt.num_sms));
    ALLOC(lm->lp_ws, iris_logprobs_ws_bytes(max_tokens, c->vocab));
    ALLOC(lm->out, (2 + 32) * T * 4);
    ALLOC(lm->out_ids, 32 * T * 4);
    ALLOC(lm->draw, 24 * T);
#undef ALLOC
    if (!rc) {
        /* sequence s has the pages [s * blocks, (s + 1) * blocks) */
        int32_t *t = (int32_t *)malloc(pages * 4);
        if (!t) rc = iris_fail(IRIS_CUDA_ERR_OOM, "page table");
        for (size_t i = 0; !rc && i < pages; i++) t[i] = (int32_t)i;
        if (!rc) rc = iris_h2d(lm->table, t, pages * 4);
        free(t);
    }
    if (!rc) rc = iris_gpu_rope_init(&lm->rope, IRIS_ROPE_HALF, 128, (double)c->rope_theta, NULL);
    /* rows past a step's tokens hold an earlier step's values: a GEMM reads them into rows it does not store */
    if (!rc) rc = iris_cuda_check(cudaMemsetAsync(lm->xn, 0, T * H * 2, g_rt.stream), "clear");
    if (!rc) rc = iris_cuda_check(cudaMemsetAsync(lm->attn, 0, T * qd * 2, g_rt.stream), "clear");
    if (!rc) rc = iris_cuda_check(cudaMemsetAsync(lm->mlp, 0, T * F * 2, g_rt.stream), "clear");
    if (!rc && (iris_make_tmap_bf16(&lm->tm_xn, lm->xn, T, H, H, 128) ||
                iris_make_tmap_bf16(&lm->tm_attn, lm->attn, T, qd, qd, 128) ||
                iris_make_tmap_bf16(&lm->tm_mlp, lm->mlp, T, F, F, 128)))
        rc = iris_fail(IRIS_CUDA_ERR_CUDA, "language model activation tensor map");
    if (rc) { iris_cuda_qwen3_lm_free(lm); return NULL; }
    return lm;
}

size_t iris_cuda_qwen3_lm_cache_bytes(const iris_cuda_qwen3_lm_t *lm) {
    return lm ? (size_t)2 * lm->m->cfg.layers * lm->pool_elems * 2 : 0;
}

int iris_cuda_qwen3_lm_length(const iris_cuda_qwen3_lm_t *lm, int seq) {
    if (!lm || seq < 0 || seq >= lm->num_seqs) return iris_fail(IRIS_CUDA_ERR_ARG, "sequence %d", seq);
    return lm->len[seq];
}

static int lm_enqueue(iris_cuda_qwen3_lm_t *lm, int T, int top_k, q3_enq_t *E) {
    const iris_cuda_qwen3_t *m = lm->m;
    const iris_cuda_qwen3_config_t *c = &m->cfg;
    const int H = c->hidden, F = c->intermediate, nh = c->heads, nkv = c->kv_heads, qd = nh * 128;
    const int nq = (nh + 2 * nkv) * 128;
    const int32_t *ids = lm->in, *seq = ids + T, *pos = seq + T, *targets = pos + T;
    cudaStream_t st = g_rt.stream;
    int n = 1;
    iris_q3_done(E, iris_launch_embed_rows(ids, T, m->embed, c->vocab, H, lm->x, st), "embed", 1);
    for (int i = 0; i < c->layers && !E->rc; i++) {
        const q3_layer_t *L = &m->layers[i];
        iris_q3_done(E, iris_launch_rmsnorm(lm->x, H, L->ln1, NULL, lm->xn, H, T, H, Q3_EPS, NULL, st), "rmsnorm", 1);
        iris_q3_gemm(E, "qkv", &lm->tm_xn, &L->tm_qkv, T, nq, H, IRIS_EPI_F32, lm->qkv, nq, NULL, NULL, 0, NULL, 0);
        IrisRopeAppend r;
        memset(&r, 0, sizeof(r));
        lm_cache(lm, i, &r.cache);
        r.rope = lm->rope;
        r.q_out = lm->q;
        r.q = lm->qkv;
        r.k = lm->qkv + qd;
        r.v = lm->qkv + qd + nkv * 128;
        r.ldq_out = qd;
        r.ldq = r.ldk = r.ldv = nq;
        r.q_norm = L->qn;
        r.k_norm = L->kn;
        r.eps = Q3_EPS;
        r.seq = seq;
        r.pos = pos;
        r.tokens = T;
        r.heads = nh;
        if (!E->rc) iris_q3_done(E, iris_launch_rope_append(&r, 1, g_rt.num_sms, st), "rope append", 1);
        IrisPagedAttention a = {r.cache, lm->attn, lm->q, qd, qd, seq, pos, T, nh, 1.0f / sqrtf(128.0f), (float *)lm->attn_ws,
                                {0, 0}, {NULL, NULL, 0, 0, 0, 0, {0, 0}}};
        if (!E->rc) {
            const cudaError_t e = iris_launch_paged_attention(&a, g_rt.num_sms, st, &n);
            iris_q3_done(E, e, "attention", n);
        }
        iris_q3_gemm(E, "o_proj", &lm->tm_attn, &L->tm_o, T, H, qd, IRIS_EPI_RESID_GATE, lm->x, H, m->ones, NULL, 0, lm->ws,
                     lm->ws_bytes);
        iris_q3_done(E, iris_launch_rmsnorm(lm->x, H, L->ln2, NULL, lm->xn, H, T, H, Q3_EPS, NULL, st), "rmsnorm", 1);
        iris_q3_gemm(E, "gate_up", &lm->tm_xn, &L->tm_gu, T, 2 * F, H, IRIS_EPI_SWIGLU, NULL, 0, NULL, lm->mlp, F, NULL, 0);
        iris_q3_gemm(E, "down", &lm->tm_mlp, &L->tm_down, T, H, F, IRIS_EPI_RESID_GATE, lm->x, H, m->ones, NULL, 0, lm->ws,
                     lm->ws_bytes);
    }
    iris_q3_done(E, iris_launch_rmsnorm(lm->x, H, m->norm, NULL, lm->xn, H, T, H, Q3_EPS, NULL, st), "rmsnorm", 1);
    iris_q3_gemm(E, "head", &lm->tm_xn, &m->tm_head, T, m->head_rows, H, IRIS_EPI_F32, lm->logits, m->head_rows, NULL, NULL, 0,
                 NULL, 0);
    if (top_k == LM_DRAW) {
        const float *set = (const float *)(lm->draw + T);
        IrisSample d = {lm->logits, m->head_rows, T, c->vocab, set, set + T, set + 2 * T, (const int32_t *)(set + 3 * T), lm->draw,
                        lm->out_ids, NULL, lm->out, 0, 0};
        if (!E->rc) iris_q3_done(E, iris_launch_sample(&d, 1, g_rt.num_sms, st), "draw", 1);
        return E->rc;
    }
    IrisLogprobs p = {lm->logits, m->head_rows, T, c->vocab, top_k, targets, lm->out, lm->out + lm->max_tokens,
                      lm->out + 2 * lm->max_tokens, lm->out_ids, lm->lp_ws};
    if (!E->rc) {
        const cudaError_t e = iris_launch_logprobs(&p, 1, g_rt.num_sms, st, &n);
        iris_q3_done(E, e, "log probabilities", n);
    }
    return E->rc;
}

/* A size's first step is queued kernel by kernel and its second captured: a graph spares 0.25 ms of 3.9 (Qwen3-4B, 8
 * tokens), making one costs 1.2.  The LM_SIZES sizes used last are kept, so that prompts and single tokens may alternate. */
static int lm_run(iris_cuda_qwen3_lm_t *lm, int T, int top_k) {
    if (iris_fault("launch")) return iris_fail(IRIS_CUDA_ERR_INJECTED, "injected launch failure");
    q3_enq_t E;
    memset(&E, 0, sizeof(E));
    lm_size_t *z = lm->sizes;  /* this size, or the one not used for longest */
    for (int i = 0; i < LM_SIZES; i++) {
        if (lm->sizes[i].tokens == T && lm->sizes[i].top_k == top_k) { z = &lm->sizes[i]; break; }
        if (lm->sizes[i].used < z->used) z = &lm->sizes[i];
    }
    const int known = z->tokens == T && z->top_k == top_k;
    if (!known || getenv("IRIS_CUDA_NO_GRAPH")) {
        if (!known) {
            lm_size_free(z);
            z->tokens = T;
            z->top_k = top_k;
        }
        z->used = lm->step;
        const int rc = lm_enqueue(lm, T, top_k, &E);
        iris_count_launch(E.kernels);
        return rc;
    }
    z->used = lm->step;
    if (!z->gexec) {
        cudaError_t e = cudaStreamBeginCapture(g_rt.stream, cudaStreamCaptureModeThreadLocal);
        if (e != cudaSuccess) return iris_cuda_check(e, "begin capture");
        const int rc = lm_enqueue(lm, T, top_k, &E);
        cudaGraph_t g = NULL;
        e = cudaStreamEndCapture(g_rt.stream, &g);
        if (rc) { if (g) cudaGraphDestroy(g); return rc; }
        if (e != cudaSuccess) return iris_cuda_check(e, "end capture");
        e = cudaGraphInstantiate(&z->gexec, g, 0);
        if (e != cudaSuccess) { z->gexec = NULL; cudaGraphDestroy(g); return iris_cuda_check(e, "graph instantiate"); }
        z->graph = g;
        z->kernels = E.kernels;
    }
    iris_count_launch(z->kernels);
    return iris_cuda_check(cudaGraphLaunch(z->gexec, g_rt.stream), "graph launch");
}

/* the step's sequences and positions against what the sequences hold; lm->next gets the lengths after it */
static int lm_check(iris_cuda_qwen3_lm_t *lm, const int *seq, const int *pos, int T) {
    lm->step++;
    for (int t = 0; t < T; t++) {
        const int s = seq[t], p = pos[t];
        if (s < 0 || s >= lm->num_seqs || p < 0 || p >= lm->max_len)
            return iris_fail(IRIS_CUDA_ERR_ARG, "token %d: position %d of sequence %d (%d sequences of %d)", t, p, s,
                             lm->num_seqs, lm->max_len);
        const int first = lm->named[s] != lm->step;
        if (first ? p > lm->len[s] : p != lm->next[s])
            return iris_fail(IRIS_CUDA_ERR_ARG, "token %d: position %d of sequence %d, which holds %d", t, p, s,
                             first ? lm->len[s] : lm->next[s]);
        lm->named[s] = lm->step;
        lm->next[s] = p + 1;
    }
    return 0;
}

/* what every step's arguments have to be */
static int lm_args(iris_cuda_qwen3_lm_t *lm, const int *ids, const int *seq, const int *pos, int tokens) {
    if (!lm || !ids || !seq || !pos) return iris_fail(IRIS_CUDA_ERR_ARG, "null argument");
    if (tokens < 1 || tokens > lm->max_tokens)
        return iris_fail(IRIS_CUDA_ERR_ARG, "step of %d tokens (1..%d)", tokens, lm->max_tokens);
    return lm_check(lm, seq, pos, tokens);
}

typedef struct { void *to; const void *from; size_t bytes; } lm_out_t;

/* the step itself; its outputs back to the host */
static int lm_feed(iris_cuda_qwen3_lm_t *lm, const int *ids, const int *seq, const int *pos, const int *targets, int tokens,
                   int top_k, const lm_out_t *outs, int n_outs) {
    const size_t n = (size_t)tokens;
    memcpy(lm->h_in, ids, n * 4);
    memcpy(lm->h_in + n, seq, n * 4);
    memcpy(lm->h_in + 2 * n, pos, n * 4);
    if (targets) memcpy(lm->h_in + 3 * n, targets, n * 4);
    else memset(lm->h_in + 3 * n, 0xFF, n * 4);  /* -1 */
    int rc = iris_h2d(lm->in, lm->h_in, 4 * n * 4);
    if (!rc) rc = lm_run(lm, tokens, top_k);
    for (int i = 0; !rc && i < n_outs; i++)
        if (outs[i].to && outs[i].bytes)
            rc = iris_cuda_check(cudaMemcpyAsync(outs[i].to, outs[i].from, outs[i].bytes, cudaMemcpyDeviceToHost, g_rt.stream),
                                 "outputs");
    const int done = iris_cuda_synchronize();
    if (!rc) rc = done;
    if (!rc)
        for (int t = 0; t < tokens; t++) lm->len[seq[t]] = lm->next[seq[t]];
    return rc;
}

int iris_cuda_qwen3_lm_step(iris_cuda_qwen3_lm_t *lm, const int *ids, const int *seq, const int *pos,
                            const int *targets, int tokens, int top_k, float *logprob, float *entropy, int *top_ids,
                            float *top_logprobs) {
    if (lm && (top_k < 0 || top_k > 32 || top_k > lm->m->cfg.vocab))
        return iris_fail(IRIS_CUDA_ERR_ARG, "top_k %d (0..min(32, vocabulary))", top_k);
    const int rc = lm_args(lm, ids, seq, pos, tokens);
    if (rc) return rc;
    const size_t n = (size_t)tokens, T = (size_t)lm->max_tokens, k = (size_t)top_k;
    const lm_out_t outs[] = {{logprob, lm->out, n * 4}, {entropy, lm->out + T, n * 4}, {top_logprobs, lm->out + 2 * T, n * k * 4},
                             {top_ids, lm->out_ids, n * k * 4}};
    return lm_feed(lm, ids, seq, pos, targets, tokens, top_k, outs, 4);
}

int iris_cuda_qwen3_lm_sample(iris_cuda_qwen3_lm_t *lm, const int *ids, const int *seq, const int *pos, int tokens,
                              const float *temperature, const int *top_k, const float *top_p, const float *min_p,
                              const double *uniform, int *next, float *logprobs) {
    if (!uniform || !next) return iris_fail(IRIS_CUDA_ERR_ARG, "null argument");
    int rc = lm_args(lm, ids, seq, pos, tokens);
    if (rc) return rc;
    const size_t n = (size_t)tokens;
    float *set = (float *)(lm->h_draw + n);
    int32_t *k = (int32_t *)(set + 3 * n);
    memcpy(lm->h_draw, uniform, n * 8);
    for (size_t t = 0; t < n; t++) {
        set[t] = temperature ? temperature[t] : 1.0f;
        set[n + t] = top_p ? top_p[t] : 1.0f;
        set[2 * n + t] = min_p ? min_p[t] : 0.0f;
        k[t] = top_k ? top_k[t] : 0;
    }
    rc = iris_h2d(lm->draw, lm->h_draw, 24 * n);
    if (rc) return rc;
    const lm_out_t outs[] = {{next, lm->out_ids, n * 4}, {logprobs, lm->out, n * 4}};
    return lm_feed(lm, ids, seq, pos, NULL, tokens, LM_DRAW, outs, 2);
}
