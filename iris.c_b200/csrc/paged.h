/*
 * Index arithmetic of the paged-cache attention, shared by the kernels
 * (lm_kernels.cu) and by its host test: which keys a row sees, where a key
 * lies, and how the key tiles of all rows are shared out.
 *
 * Work is counted in tiles of IRIS_PAGED_TILE keys.  A unit is one row, one
 * key-value head and up to 8 or 16 of the query heads on it; a row has
 * `units` of them, each of as many tiles as the row's keys fill.  All tiles of
 * all rows stand in one line (row by row, unit by unit, tile by tile) that is
 * cut into equal shares, one per CTA, whatever the rows' lengths.  To begin and
 * finish a unit takes a CTA about as long as a tile, so that every unit has one
 * empty place in the line behind its tiles (IRIS_PAGED_EXTRA).  Where a call
 * has several rows of a sequence, a unit can be a run of them instead of one
 * (iris_paged_run); the first stands in the line for all.  A unit cut
 * by a share's border is summed in pieces: a CTA leaves at most two, slot 2 c
 * for a piece whose unit began in an earlier share, slot 2 c + 1 for one that
 * begins here and goes on.
 */
#ifndef IRIS_PAGED_H
#define IRIS_PAGED_H

#include <stdint.h>

#include "iris_cuda.h"

#ifdef __CUDACC__
#define IRIS_HD __host__ __device__ __forceinline__
#else
#define IRIS_HD static inline
#endif

#define IRIS_PAGED_TILE 64
#define IRIS_PAGED_EXTRA 1

/* query heads of a unit, where `group` of them share a key-value head: the 16 rows of a matrix instruction hold up to
 * 8 heads twice (see the kernel) or up to 16 once, so that groups of up to 16 read the cache once */
IRIS_HD int iris_paged_heads(int group) { return group > 8 ? 16 : 8; }

/* units of a row */
IRIS_HD int iris_paged_units(const iris_gpu_kv_cache_t *c, int heads) {
    const int group = heads / c->kv_heads, n = iris_paged_heads(group);
    return c->kv_heads * ((group + n - 1) / n);
}

/* sequence of row t, or -1 */
IRIS_HD int iris_paged_seq(const iris_gpu_kv_cache_t *c, const int32_t *seq, int t) {
    const int s = seq ? seq[t] : t;
    return s >= 0 && s < c->num_seqs ? s : -1;
}

/* keys that a row at position `pos` sees (no more than the table has room for) */
IRIS_HD int iris_paged_len(const iris_gpu_kv_cache_t *c, int pos) {
    const int64_t room = (int64_t)c->max_blocks * c->page_size;
    const int64_t len = pos < 0 ? 0 : (int64_t)pos + 1;
    const int64_t n = len < room ? len : room;
    return n < 0x7FFFFFFF ? (int)n : 0x7FFFFFFF;
}

IRIS_HD int iris_paged_tiles(int len) { return len / IRIS_PAGED_TILE + (len % IRIS_PAGED_TILE != 0); }

/* places in the line of one unit of row t */
IRIS_HD int iris_paged_row_places(const iris_gpu_kv_cache_t *c, const int32_t *seq, const int32_t *pos, int t) {
    const int n = iris_paged_seq(c, seq, t) < 0 ? 0 : iris_paged_tiles(iris_paged_len(c, pos[t]));
    return n ? n + IRIS_PAGED_EXTRA : 0;
}

/* A run: consecutive rows of one sequence, none past a multiple of `span` rows.
 * The number of rows in the run that begins at row t and the most keys that one
 * of them sees; 0 where row t is not the first of its run, or padding. */
IRIS_HD int iris_paged_run(const iris_gpu_kv_cache_t *c, const int32_t *seq, const int32_t *pos, int rows, int span, int t,
                           int *len) {
    const int in = t % span, s = seq[t], end = rows - t < span - in ? rows : t - in + span;
    int n = 0, most = -1, more = 1;
    *len = 0;
    if (s < 0 || s >= c->num_seqs || (in && seq[t - 1] == s)) return 0;
    for (int r = t; r < end; r++) {  /* no way out, so that the loads need not wait for one another */
        const int p = pos[r];
        more &= seq[r] == s;
        n += more;
        most = more && p > most ? p : most;
    }
    *len = iris_paged_len(c, most);
    return n;
}
IRIS_HD int iris_paged_run_places(const iris_gpu_kv_cache_t *c, const int32_t *seq, const int32_t *pos, int rows, int span,
                                  int t) {
    int len;
    iris_paged_run(c, seq, pos, rows, span, t, &len);
    return len ? iris_paged_tiles(len) + IRIS_PAGED_EXTRA : 0;
}

/* p / page_size for 0 <= p < 2^31 as p * mul >> shift: shift = 31 + ceil(log2 page_size), mul = ceil(2^shift /
 * page_size) <= 2^32 - 1, and p (mul page_size - 2^shift) < 2^31 page_size <= 2^shift keeps the floor */
typedef struct { uint32_t mul; int shift; } iris_paged_div_t;
IRIS_HD iris_paged_div_t iris_paged_div(int page_size) {
    iris_paged_div_t d;
    d.shift = 31;
    while (((uint64_t)1 << (d.shift - 31)) < (uint64_t)page_size) d.shift++;
    d.mul = (uint32_t)((((uint64_t)1 << d.shift) + page_size - 1) / page_size);
    return d;
}
IRIS_HD int iris_paged_block(iris_paged_div_t d, int p) { return (int)(((uint64_t)(uint32_t)p * d.mul) >> d.shift); }

/* page of block b of sequence s, or -1 where the table or the pool has none */
IRIS_HD int iris_paged_page(const iris_gpu_kv_cache_t *c, int s, int b) {
    if (b >= c->max_blocks) return -1;
    const int page = c->table[(int64_t)s * c->table_stride + b];
    return page >= 0 && page < c->num_pages ? page : -1;
}

/* element offset in the pools of `slot` (head 0) of `page` */
IRIS_HD int64_t iris_paged_offset(const iris_gpu_kv_cache_t *c, int page, int slot) {
    return (int64_t)page * c->page_stride + (int64_t)slot * c->token_stride;
}

/* places in a share */
IRIS_HD int64_t iris_paged_share(int64_t total, int ctas) { return total <= ctas ? 1 : (total + ctas - 1) / ctas; }
IRIS_HD uint32_t iris_paged_share32(uint32_t total, uint32_t ctas) { return total <= ctas ? 1 : (total - 1) / ctas + 1; }

/* A place in the line. */
typedef struct {
    int64_t left; /* places of the share from this one on */
    int t;        /* row                          */
    int s, len;   /* its sequence and visible keys */
    int n;        /* tiles of each of its units   */
    int u;        /* unit                         */
    int i;        /* tile of the unit             */
    int rows;     /* rows of the call, span: of which a unit may hold so many (0: one row a unit, `rows` and `count` unused) */
    int span, count; /* count: rows of this run   */
} iris_paged_at_t;

IRIS_HD void iris_paged_row(iris_paged_at_t *a, const iris_gpu_kv_cache_t *c, const int32_t *seq, const int32_t *pos) {
    a->s = iris_paged_seq(c, seq, a->t);
    if (a->span) a->count = iris_paged_run(c, seq, pos, a->rows, a->span, a->t, &a->len);
    else a->len = a->s < 0 ? 0 : iris_paged_len(c, pos[a->t]);
    a->n = iris_paged_tiles(a->len);
}

/* whether another tile of the share comes after this one, and which */
IRIS_HD int iris_paged_more(const iris_paged_at_t *a) {
    return a->i + 1 < a->n ? a->left > 1 : a->left > 1 + IRIS_PAGED_EXTRA;
}
IRIS_HD void iris_paged_unit(iris_paged_at_t *a, int units, const iris_gpu_kv_cache_t *c, const int32_t *seq,
                             const int32_t *pos) {
    a->i = 0;
    if (++a->u < units) return;
    a->u = 0;
    do {
        a->t += a->span && a->count > 1 ? a->count : 1;
        iris_paged_row(a, c, seq, pos);
    } while (a->n == 0);
}
IRIS_HD void iris_paged_next(iris_paged_at_t *a, int units, const iris_gpu_kv_cache_t *c, const int32_t *seq,
                             const int32_t *pos) {
    a->left--;
    if (++a->i < a->n) return;
    a->left -= IRIS_PAGED_EXTRA;
    iris_paged_unit(a, units, c, seq, pos);
}

/* The first tile at or after place `rest` of row a->t's units, of a share of
 * `left` places from there; 0 if the share has none. */
IRIS_HD int iris_paged_start(iris_paged_at_t *a, int64_t rest, int64_t left, int units, const iris_gpu_kv_cache_t *c,
                             const int32_t *seq, const int32_t *pos) {
    iris_paged_row(a, c, seq, pos);
    const int places = a->n + IRIS_PAGED_EXTRA;
    a->u = rest <= 0x7FFFFFFF ? (int)((uint32_t)rest / (uint32_t)places) : (int)(rest / places);
    a->i = (int)(rest - (int64_t)a->u * places);
    a->left = left;
    if (a->i < a->n) return 1;
    const int skip = places - a->i;  /* empty places */
    if (left <= skip) return 0;
    a->left -= skip;
    iris_paged_unit(a, units, c, seq, pos);
    return 1;
}

/* Share c begins at tile `at.i` of a unit.  The number of later shares that
 * hold pieces of that unit when c is the first after the one it began in,
 * else 0.  The pieces then are slot 2 (c - 1) + 1 and slots 2 c, 2 (c + 1), ... */
IRIS_HD int iris_paged_join(const iris_paged_at_t *at, int64_t share) {
    if (at->i == 0 || at->i > share) return 0;
    return (int)((at->n - at->i + share - 1) / share);
}

/* The same from the unit: its first tile is place `begin` of the line, n tiles.
 * Returns the number of later shares that hold pieces of it, *border the first. */
IRIS_HD int iris_paged_cut(int64_t begin, int n, int64_t share, int *border) {
    const int64_t c = begin / share + 1, over = begin + n - c * share;
    *border = (int)c;
    return over > 0 ? (int)((over + share - 1) / share) : 0;
}

#endif
