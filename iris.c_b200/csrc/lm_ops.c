/*
 * Language-model operators (layer 4 of iris_cuda.h): argument checks, the
 * rotation's frequencies, and the launches of lm_kernels.cu.
 *
 * Every check of host-visible arguments runs before the device is touched, so
 * a refused call queues nothing and needs no GPU.
 */
#include "gpu_ops_internal.h"

#include <limits.h>
#include <math.h>
#include <string.h>

#define LM_FAIL(...) op_fail(IRIS_CUDA_ERR_ARG, __VA_ARGS__)

static int misaligned(const void *p, size_t a) { return ((uintptr_t)p & (a - 1)) != 0; }

/* ------------------------------------------------------------------ device side of a call
 * The calls run on the library's device whatever the calling thread's current
 * one is.  Every pointer has to be that device's memory (or managed): a host
 * pointer, or one of a device that this one can not reach, would fault. */
typedef struct { int prev; } lm_dev_t;

static int lm_enter(lm_dev_t *d, const char *what, const void *const *ptrs, int n) {
    d->prev = -1;
    int rc = iris_rt_ensure();
    if (rc) return op_fail(rc, "%s: %s", what, "no usable device");
    for (int i = 0; i < n; i++) {
        if (!ptrs[i]) continue;
        struct cudaPointerAttributes at;
        cudaError_t e = cudaPointerGetAttributes(&at, ptrs[i]);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return LM_FAIL("%s: pointer %d: %s", what, i, cudaGetErrorString(e));
        }
        if (at.type != cudaMemoryTypeManaged && (at.type != cudaMemoryTypeDevice || at.device != g_rt.device))
            return LM_FAIL("%s: pointer %d is not memory of device %d", what, i, g_rt.device);
    }
    int cur = -1;
    if (op_check(cudaGetDevice(&cur), what)) return IRIS_CUDA_ERR_CUDA;
    if (cur != g_rt.device) {
        if (op_check(cudaSetDevice(g_rt.device), what)) return IRIS_CUDA_ERR_CUDA;
        d->prev = cur;
    }
    return 0;
}

static int lm_leave(lm_dev_t *d, cudaError_t e, const char *what, int launches) {
    if (d->prev >= 0) cudaSetDevice(d->prev);
    if (e == cudaSuccess) iris_count_launch((uint64_t)launches);
    return op_check(e, what);
}

/* ------------------------------------------------------------------ paged cache */
static int cache_check(const iris_gpu_kv_cache_t *c, const char *what) {
    if (!c || !c->k || !c->v || !c->table) return LM_FAIL("%s: null cache, pool or page table", what);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return LM_FAIL("%s: head_dim %d (64, 128 or 256)", what, c->head_dim);
    if (c->num_pages < 1 || c->page_size < 1 || c->kv_heads < 1 || c->num_seqs < 1 || c->max_blocks < 1)
        return LM_FAIL("%s: cache of %d pages of %d tokens, %d heads, table %d x %d", what, c->num_pages, c->page_size,
                       c->kv_heads, c->num_seqs, c->max_blocks);
    if (c->kv_heads > 65535) return LM_FAIL("%s: %d key-value heads (at most 65535)", what, c->kv_heads);
    if (misaligned(c->k, 16) || misaligned(c->v, 16) || misaligned(c->table, 4))
        return LM_FAIL("%s: misaligned pointer (pools need 16-byte, the table 4-byte alignment)", what);
    if (c->page_stride < 0 || c->token_stride < 0 || c->head_stride < 0 || c->page_stride % 8 || c->token_stride % 8 ||
        c->head_stride % 8 || (c->num_pages > 1 && !c->page_stride) || (c->page_size > 1 && !c->token_stride) ||
        (c->kv_heads > 1 && !c->head_stride))
        return LM_FAIL("%s: strides %lld / %lld / %lld of pages, slots and heads (positive multiples of 8)", what,
                       (long long)c->page_stride, (long long)c->token_stride, (long long)c->head_stride);
    if (c->table_stride < 0 || (c->num_seqs > 1 && c->table_stride < c->max_blocks))
        return LM_FAIL("%s: table stride %lld under its %d entries", what, (long long)c->table_stride, c->max_blocks);
    return 0;
}

/* ------------------------------------------------------------------ rotary positions */
static int rope_layout_check(const iris_gpu_rope_t *r, int layout, int rot_dim, const char *what) {
    if (!r) return LM_FAIL("%s: null rotation", what);
    if (layout != IRIS_ROPE_HALF && layout != IRIS_ROPE_INTERLEAVED) return LM_FAIL("%s: layout %d", what, layout);
    if (rot_dim < 16 || rot_dim > 256 || rot_dim % 16)
        return LM_FAIL("%s: rot_dim %d (a multiple of 16, 16 to 256)", what, rot_dim);
    return 0;
}

int iris_gpu_rope_init_freqs(iris_gpu_rope_t *rope, int layout, int rot_dim, const double *freqs, double amplitude) {
    if (rope_layout_check(rope, layout, rot_dim, "rope_init")) return IRIS_CUDA_ERR_ARG;
    if (!freqs) return LM_FAIL("rope_init: null frequencies");
    if (!isfinite((float)amplitude) || !((float)amplitude > 0.0f)) return LM_FAIL("rope_init: amplitude %g", amplitude);
    for (int i = 0; i < rot_dim / 2; i++)
        if (!isfinite(freqs[i]) || freqs[i] < 0.0) return LM_FAIL("rope_init: frequency %d is %g", i, freqs[i]);
    memset(rope, 0, sizeof(*rope));
    rope->layout = layout;
    rope->rot_dim = rot_dim;
    rope->amplitude = (float)amplitude;
    for (int i = 0; i < rot_dim / 2; i++) {
        /* turns per position, its whole part dropped: positions are whole, so it never shows */
        const double t = freqs[i] / 6.283185307179586476925286766559;
        rope->turns[i] = (uint64_t)ldexp(t - floor(t), 64);
    }
    return 0;
}

int iris_gpu_rope_init(iris_gpu_rope_t *rope, int layout, int rot_dim, double theta,
                       const iris_gpu_rope_scaling_t *scaling) {
    if (rope_layout_check(rope, layout, rot_dim, "rope_init")) return IRIS_CUDA_ERR_ARG;
    if (!isfinite(theta) || theta <= 0.0) return LM_FAIL("rope_init: theta %g", theta);
    if (scaling && (!isfinite(scaling->factor) || scaling->factor <= 0.0 || !isfinite(scaling->original_len) ||
                    scaling->original_len < 0.0))
        return LM_FAIL("rope_init: scaling factor %g over %g positions", scaling->factor, scaling->original_len);
    if (scaling && scaling->original_len > 0.0 &&
        !(isfinite(scaling->low) && isfinite(scaling->high) && scaling->low < scaling->high))
        return LM_FAIL("rope_init: scaling by parts between %g and %g turns", scaling->low, scaling->high);
    double f[128];
    for (int i = 0; i < rot_dim / 2; i++) {
        f[i] = pow(theta, -2.0 * i / rot_dim);
        if (!scaling) continue;
        double keep = 0.0;
        if (scaling->original_len > 0.0) {
            const double r = scaling->original_len * f[i] / 6.283185307179586476925286766559;
            keep = (r - scaling->low) / (scaling->high - scaling->low);
            keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
        }
        f[i] *= keep + (1.0 - keep) / scaling->factor;
    }
    return iris_gpu_rope_init_freqs(rope, layout, rot_dim, f, scaling ? scaling->amplitude : 1.0);
}

int iris_gpu_rope_append(const iris_gpu_kv_cache_t *cache, const iris_gpu_rope_t *rope, void *q_out, int64_t ldq_out,
                         const void *q, const void *k, const void *v, int64_t ldq, int64_t ldk, int64_t ldv, int f32,
                         const float *q_norm, const float *k_norm, float eps, const int32_t *seq, const int32_t *pos,
                         int tokens, int heads, void *stream) {
    const char *what = "rope_append";
    if (cache_check(cache, what)) return IRIS_CUDA_ERR_ARG;
    if (tokens < 0 || heads < 0 || heads > 65535) return LM_FAIL("%s: %d tokens, %d heads", what, tokens, heads);
    /* a batch of no rows may have no tensors */
    if (tokens && (!k || !v || !seq || !pos || (heads && (!q || !q_out)))) return LM_FAIL("%s: null pointer", what);
    if (rope) {
        if (rope_layout_check(rope, rope->layout, rope->rot_dim, what)) return IRIS_CUDA_ERR_ARG;
        if (rope->rot_dim > cache->head_dim)
            return LM_FAIL("%s: rot_dim %d over head_dim %d", what, rope->rot_dim, cache->head_dim);
    }
    if (!(eps >= 0.0f)) return LM_FAIL("%s: eps %g", what, (double)eps);
    const int64_t hd = cache->head_dim, step = f32 ? 4 : 8;
    if (ldk % step || ldv % step || ldk < cache->kv_heads * hd || ldv < cache->kv_heads * hd ||
        (heads && (ldq % step || ldq_out % 8 || ldq < heads * hd || ldq_out < heads * hd)))
        return LM_FAIL("%s: row strides %lld, %lld, %lld to %lld (at least the row, multiples of 8, f32 of 4)", what,
                       (long long)ldq, (long long)ldk, (long long)ldv, (long long)ldq_out);
    if (misaligned(k, 16) || misaligned(v, 16) || (heads && (misaligned(q, 16) || misaligned(q_out, 16))) ||
        misaligned(q_norm, 16) || misaligned(k_norm, 16) || misaligned(seq, 4) || misaligned(pos, 4))
        return LM_FAIL("%s: misaligned pointer (16 bytes; seq and pos 4)", what);
    if (tokens && heads && q_out == q && (f32 || ldq != ldq_out))
        return LM_FAIL("%s: q_out on q needs bf16 and one row stride", what);
    if (!tokens) return 0;
    const void *ptrs[] = {cache->k, cache->v, cache->table, q_out, q, k, v, q_norm, k_norm, seq, pos};
    lm_dev_t d;
    int rc = lm_enter(&d, what, ptrs, (int)(sizeof(ptrs) / sizeof(ptrs[0])));
    if (rc) return rc;
    IrisRopeAppend a;
    memset(&a, 0, sizeof(a));
    a.cache = *cache;
    if (rope) a.rope = *rope;
    a.q_out = q_out;
    a.q = q;
    a.k = k;
    a.v = v;
    a.ldq_out = ldq_out;
    a.ldq = ldq;
    a.ldk = ldk;
    a.ldv = ldv;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.eps = eps;
    a.seq = seq;
    a.pos = pos;
    a.tokens = tokens;
    a.heads = heads;
    return lm_leave(&d, iris_launch_rope_append(&a, f32 != 0, g_rt.num_sms, (cudaStream_t)stream), what, 1);
}

/* ------------------------------------------------------------------ attention over the cache */
static int heads_check(const iris_gpu_kv_cache_t *c, int heads, const char *what) {
    if (heads < 1 || heads > 65535 || heads % c->kv_heads)
        return LM_FAIL("%s: %d query heads on %d key-value heads", what, heads, c->kv_heads);
    return 0;
}

size_t iris_gpu_attention_paged_workspace(const iris_gpu_kv_cache_t *cache, int heads) {
    const char *what = "attention_paged_workspace";
    if (cache_check(cache, what) || heads_check(cache, heads, what)) return 0;
    if (iris_rt_ensure()) { op_fail(IRIS_CUDA_ERR_NODEV, "%s: no usable device", what); return 0; }
    return iris_paged_attention_ws_bytes(cache, heads, g_rt.num_sms);
}

int iris_gpu_attention_paged(const iris_gpu_kv_cache_t *cache, void *out, const void *q, int64_t ldo, int64_t ldq,
                             const int32_t *seq, const int32_t *pos, int rows, int heads, float scale,
                             void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "attention_paged";
    if (cache_check(cache, what) || heads_check(cache, heads, what)) return IRIS_CUDA_ERR_ARG;
    if (rows < 0 || (!seq && rows > cache->num_seqs))
        return LM_FAIL("%s: %d rows for %d sequences", what, rows, cache->num_seqs);
    if (rows && (!out || !q || !pos || !workspace)) return LM_FAIL("%s: null pointer", what);
    const int64_t width = (int64_t)heads * cache->head_dim;
    if (ldo % 8 || ldq % 8 || ldo < width || ldq < width)
        return LM_FAIL("%s: row strides %lld to %lld (at least %lld, multiples of 8)", what, (long long)ldq,
                       (long long)ldo, (long long)width);
    if (!isfinite(scale)) return LM_FAIL("%s: scale %g", what, (double)scale);
    if (misaligned(out, 16) || misaligned(q, 16) || misaligned(workspace, 16) || misaligned(seq, 4) || misaligned(pos, 4))
        return LM_FAIL("%s: misaligned pointer (16 bytes; seq and pos 4)", what);
    if (!rows) return 0;
    const void *ptrs[] = {cache->k, cache->v, cache->table, out, q, seq, pos, workspace};
    lm_dev_t d;
    int rc = lm_enter(&d, what, ptrs, (int)(sizeof(ptrs) / sizeof(ptrs[0])));
    if (rc) return rc;
    const size_t need = iris_paged_attention_ws_bytes(cache, heads, g_rt.num_sms);
    if (workspace_bytes < need) {
        lm_leave(&d, cudaSuccess, what, 0);
        return LM_FAIL("%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
    }
    IrisPagedAttention a = {*cache, out, q, ldo, ldq, seq, pos, rows, heads, scale, (float *)workspace, {0, 0}};
    int launches = 0;
    cudaError_t e = iris_launch_paged_attention(&a, g_rt.num_sms, (cudaStream_t)stream, &launches);
    return lm_leave(&d, e, what, launches);
}

/* ------------------------------------------------------------------ log probabilities */
static int logprobs_shape(int rows, int vocab, const char *what) {
    /* ids are int32; 2^40 logits, more than any device holds, are under 2^32 parts (of 1024 values or a row's rest) */
    if (rows < 0 || vocab < 1 || vocab > (1 << 30) || (int64_t)rows * vocab > (int64_t)1 << 40)
        return LM_FAIL("%s: %d rows of %d logits", what, rows, vocab);
    return 0;
}

size_t iris_gpu_token_logprobs_workspace(int rows, int vocab) {
    if (logprobs_shape(rows, vocab, "token_logprobs_workspace")) return 0;
    return iris_logprobs_ws_bytes(rows, vocab);
}

int iris_gpu_token_logprobs(const void *logits, int f32, int64_t ld, int rows, int vocab, const int32_t *targets,
                            float *logprob, float *entropy, int top_k, int32_t *top_ids, float *top_logprobs,
                            void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "token_logprobs";
    if (logprobs_shape(rows, vocab, what)) return IRIS_CUDA_ERR_ARG;
    if (ld < vocab) return LM_FAIL("%s: row stride %lld under %d logits", what, (long long)ld, vocab);
    if (top_k < 0 || top_k > 32 || top_k > vocab) return LM_FAIL("%s: top_k %d (0 to min(32, vocab))", what, top_k);
    if (rows && (!logits || !workspace || (logprob && !targets))) return LM_FAIL("%s: null pointer", what);
    if (rows && top_k && !top_ids && !top_logprobs) return LM_FAIL("%s: top_k %d without an output", what, top_k);
    if (misaligned(logits, f32 ? 4 : 2) || misaligned(targets, 4) || misaligned(logprob, 4) || misaligned(entropy, 4) ||
        misaligned(top_ids, 4) || misaligned(top_logprobs, 4) || misaligned(workspace, 16))
        return LM_FAIL("%s: misaligned pointer", what);
    const size_t need = iris_logprobs_ws_bytes(rows, vocab);
    if (rows && workspace_bytes < need) return LM_FAIL("%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, need);
    if (!rows || (!logprob && !entropy && !top_k)) return 0;
    const void *ptrs[] = {logits, targets, logprob, entropy, top_ids, top_logprobs, workspace};
    lm_dev_t d;
    int rc = lm_enter(&d, what, ptrs, (int)(sizeof(ptrs) / sizeof(ptrs[0])));
    if (rc) return rc;
    IrisLogprobs a = {logits, ld, rows, vocab, top_k, targets, logprob, entropy, top_logprobs, top_ids, workspace};
    int launches = 0;
    cudaError_t e = iris_launch_logprobs(&a, f32 != 0, g_rt.num_sms, (cudaStream_t)stream, &launches);
    return lm_leave(&d, e, what, launches);
}
