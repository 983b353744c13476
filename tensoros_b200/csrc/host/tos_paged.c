/*
 * tos_paged.c - entry points of the paged-cache operators, over caches in floats
 * and in 8 bits, and of sampling a batch: argument checks, the rotation's
 * frequency table, and the hand-over to the tosk_* launchers (paged_rotary.cu,
 * paged_attention.cu, paged8_store.cu, paged8_decode.cu, sample_rows.cu).
 */
#include <math.h>
#include <stdlib.h>
#include <string.h>

#include "tos_internal.h"

#define MAX_HEAD_DIM 256
#define MAX_ROWS (1 << 30)   /* packed rows of a sequence: 32-bit arithmetic with room */
/* Keys of a sequence: unsplit, a piece of work over them takes 1 s at 4 us a
 * key tile.  No bounded wait of the kernels spans more than one piece, and they
 * end after 2 s; what rows with infinities and NaN take comes after the last. */
#define MAX_KEYS (1 << 25)
#define MAX_SEQS 65535
/* Keys that a call over an 8-bit cache lays out as fp16: pages of 128 in 32-bit arithmetic with room. */
#define MAX_TOTAL_KEYS ((int64_t)1 << 32)

struct tos_rotary {
    tosk_rotary_t r;
    int rot_dim;
};

/* Makes the library's device current for one call. */
static int device_enter(int *before)
{
    int rc = tos_ensure_init();
    if (rc) return rc;
    if (cudaGetDevice(before) != cudaSuccess) return TOS_ECUDA;
    if (*before != tos_g.device && cudaSetDevice(tos_g.device) != cudaSuccess) return TOS_ECUDA;
    return TOS_OK;
}

static int device_leave(int before, int cuda_rc)
{
    if (before != tos_g.device) cudaSetDevice(before);
    return tos_set_status(tos_from_cuda(cuda_rc));
}

static int is_float(int t) { return t == TOS_TYPE_F32 || t == TOS_TYPE_F16; }

static int aligned_to(const void *p, int type) { return ((uintptr_t)p & (type == TOS_TYPE_F16 ? 1 : 3)) == 0; }

static int rows_check(const tos_rows_t *r, int heads, int hd)
{
    if (!r || !r->ptr || r->stride < (int64_t)heads * hd || r->stride > ((int64_t)1 << 40)) return TOS_EINVAL;
    if (!is_float(r->type)) return TOS_ENOTSUP;
    return aligned_to(r->ptr, r->type) ? TOS_OK : TOS_EINVAL;
}

static int paged_check(const tos_paged_kv_t *c)
{
    if (!c || !c->k || !c->v || !c->table) return TOS_EINVAL;
    if (c->n_pages <= 0 || c->page_size <= 0 || c->n_kv <= 0 || c->head_dim <= 0 || c->n_seqs < 0 ||
        c->table_stride <= 0)
        return TOS_EINVAL;
    if (!is_float(c->type) || c->head_dim > MAX_HEAD_DIM || c->n_kv > (1 << 20)) return TOS_ENOTSUP;
    if (!aligned_to(c->k, c->type) || !aligned_to(c->v, c->type) || ((uintptr_t)c->table & 3)) return TOS_EINVAL;
    return TOS_OK;
}

static tosk_paged_t paged_of(const tos_paged_kv_t *c)
{
    tosk_paged_t p = {c->k, c->v, c->type, c->n_pages, c->page_size, c->n_kv, c->head_dim,
                      c->table, c->n_seqs, c->table_stride};
    return p;
}

static tosk_rows_t rows_of(const tos_rows_t *src, const tos_rows_t *dst)
{
    tosk_rows_t r = {src ? src->ptr : NULL, dst ? dst->ptr : NULL, src ? src->stride : 0, dst ? dst->stride : 0,
                     src ? src->type : 0, dst ? dst->type : 0};
    return r;
}

/* source and destination rows of one kind of head (none when heads is 0) */
static int pair_check(const tos_rows_t *src, const tos_rows_t *dst, int heads, int hd)
{
    if (heads == 0) return src || dst ? TOS_EINVAL : TOS_OK;
    int rc = rows_check(src, heads, hd);
    if (!rc) rc = rows_check(dst, heads, hd);
    if (!rc && src->ptr == dst->ptr && (src->type != dst->type || src->stride != dst->stride)) rc = TOS_EINVAL;
    return rc;
}

/* ------------------------------------------------------------- rotation */

static int is_yarn(int scaling) { return scaling == TOS_ROTARY_SCALE_YARN || scaling == TOS_ROTARY_SCALE_YARN_UNROUNDED; }

/* The pair index at which a rotation makes `turns` turns in ctx positions. */
static long double yarn_edge(int rot, double base, double turns, int ctx)
{
    return rot * logl((long double)ctx / (turns * 2.0L * (long double)M_PI)) / (2.0L * logl((long double)base));
}

/* Where the blend of a YARN rotation begins and ends. */
static void yarn_edges(const tos_rotary_desc_t *d, long double *lo, long double *hi)
{
    *lo = yarn_edge(d->rot_dim, d->base, d->beta_fast, d->orig_ctx);
    *hi = yarn_edge(d->rot_dim, d->base, d->beta_slow, d->orig_ctx);
    if (d->scaling == TOS_ROTARY_SCALE_YARN_UNROUNDED) return;
    *lo = fminl(fmaxl(floorl(*lo), 0), d->rot_dim - 1);
    *hi = fminl(fmaxl(ceill(*hi), 0), d->rot_dim - 1);
    if (*lo == *hi) *hi += 0.001L;
}

static int rotary_desc_ok(const tos_rotary_desc_t *d)
{
    if (d->rot_dim < 2 || (d->rot_dim & 1) || d->rot_dim > MAX_HEAD_DIM) return 0;
    if (d->layout != TOS_ROTARY_INTERLEAVED && d->layout != TOS_ROTARY_HALF) return 0;
    if (!(d->base > 0.0f) || !isfinite(d->base)) return 0;
    if (d->scaling < TOS_ROTARY_SCALE_NONE || d->scaling > TOS_ROTARY_SCALE_YARN) return 0;
    if (d->scaling != TOS_ROTARY_SCALE_NONE && (!(d->factor >= 1.0f) || !isfinite(d->factor))) return 0;
    if (is_yarn(d->scaling) &&
        (d->orig_ctx <= 0 || !(d->base > 1.0f) || !(d->beta_slow > 0.0f) || !(d->beta_fast > d->beta_slow) ||
         !isfinite(d->beta_fast) || !isfinite(d->attn_factor)))
        return 0;
    if (d->freq_factors)
        for (int i = 0; i < d->rot_dim / 2; i++)
            if (!(d->freq_factors[i] > 0.0f) || !isfinite(d->freq_factors[i])) return 0;
    return 1;
}

int tos_rotary_create(tos_rotary_t **out, const tos_rotary_desc_t *d)
{
    if (!out || !d || !rotary_desc_ok(d)) return tos_set_status(TOS_EINVAL);
    int before;
    int rc = device_enter(&before);
    if (rc) return tos_set_status(rc);
    const int n = d->rot_dim / 2;
    unsigned long long turn[MAX_HEAD_DIM / 2];
    for (int i = 0; i < n; i++) {
        long double theta = powl((long double)d->base, -2.0L * i / d->rot_dim);
        if (d->freq_factors) theta /= d->freq_factors[i];
        if (d->scaling == TOS_ROTARY_SCALE_LINEAR) theta /= d->factor;
        if (is_yarn(d->scaling)) {
            long double lo, hi;
            yarn_edges(d, &lo, &hi);
            long double g = (i - lo) / (hi - lo);
            g = g < 0 ? 0 : g > 1 ? 1 : g;
            theta *= (1 - g) + g / d->factor;
        }
        /* a fraction of a turn per position; whole turns drop out */
        long double f = theta / (2.0L * acosl(-1.0L));
        f -= floorl(f);
        turn[i] = (unsigned long long)ldexpl(f, 64);
    }
    tos_rotary_t *r = (tos_rotary_t *)calloc(1, sizeof(*r));
    if (!r) { device_leave(before, 0); return tos_set_status(TOS_ENOMEM); }
    r->rot_dim = d->rot_dim;
    r->r.rot = d->rot_dim;
    r->r.half = d->layout == TOS_ROTARY_HALF;
    r->r.mag = is_yarn(d->scaling) ? d->attn_factor * (1.0f + 0.1f * logf(d->factor)) : 1.0f;
    int e = cudaMalloc((void **)&r->r.turn, (size_t)n * sizeof(turn[0]));
    if (!e) e = cudaMemcpyAsync(r->r.turn, turn, (size_t)n * sizeof(turn[0]), cudaMemcpyHostToDevice, tos_g.stream);
    if (!e) e = cudaStreamSynchronize(tos_g.stream);
    if (e) {
        if (r->r.turn) cudaFree(r->r.turn);
        free(r);
    } else {
        *out = r;
    }
    return device_leave(before, e);
}

void tos_rotary_destroy(tos_rotary_t *r)
{
    if (!r) return;
    cudaFree(r->r.turn);
    free(r);
}

static int rotary_args_check(const tos_rotary_t *rot, const int *pos, int hd, const float *qn, const float *kn, float eps)
{
    if (rot && (rot->rot_dim > hd || !pos)) return TOS_EINVAL;
    if (((uintptr_t)qn & 3) || ((uintptr_t)kn & 3) || ((uintptr_t)pos & 3)) return TOS_EINVAL;
    if ((qn || kn) && !(eps >= 0.0f && isfinite(eps))) return TOS_EINVAL;
    return TOS_OK;
}

int tos_qk_norm_rotary_dev(const tos_rows_t *q, const tos_rows_t *q_out, const tos_rows_t *k,
                           const tos_rows_t *k_out, int n_tokens, int n_heads, int n_kv, int head_dim,
                           const float *q_norm, const float *k_norm, float eps, const tos_rotary_t *rot,
                           const int *pos, void *stream)
{
    if (n_tokens < 0 || n_heads < 0 || n_kv < 0 || head_dim <= 0 || (head_dim & 1)) return tos_set_status(TOS_EINVAL);
    if (head_dim > MAX_HEAD_DIM || n_heads > (1 << 20) || n_kv > (1 << 20)) return tos_set_status(TOS_ENOTSUP);
    int rc = pair_check(q, q_out, n_heads, head_dim);
    if (!rc) rc = pair_check(k, k_out, n_kv, head_dim);
    if (!rc) rc = rotary_args_check(rot, pos, head_dim, q_norm, k_norm, eps);
    if (!rc && n_heads && n_kv && q->type != k->type) rc = TOS_ENOTSUP;
    if (rc) return tos_set_status(rc);
    int before;
    if ((rc = device_enter(&before))) return tos_set_status(rc);
    if (n_tokens == 0 || n_heads + n_kv == 0) return device_leave(before, 0);
    tosk_rotary_args_t a;
    memset(&a, 0, sizeof(a));
    a.q = rows_of(q, q_out);
    a.k = rows_of(k, k_out);
    a.n_tokens = n_tokens; a.n_heads = n_heads; a.n_kv = n_kv; a.hd = head_dim;
    a.q_norm = q_norm; a.k_norm = k_norm; a.eps = eps;
    if (rot) a.rot = rot->r;
    a.pos = pos;
    return device_leave(before, tosk_rotary_rows(&a, tos_pick_stream(stream)));
}

int tos_kv_append_paged_dev(const tos_paged_kv_t *kv, const tos_rows_t *k, const tos_rows_t *v,
                            const tos_rows_t *q, const tos_rows_t *q_out, int n_tokens, int n_heads,
                            const int *seq, const int *slot, const int *pos, const float *q_norm,
                            const float *k_norm, float eps, const tos_rotary_t *rot, void *stream)
{
    int rc = paged_check(kv);
    if (rc) return tos_set_status(rc);
    if (n_tokens < 0 || n_heads < 0 || (kv->head_dim & 1)) return tos_set_status(TOS_EINVAL);
    if (n_heads > (1 << 20)) return tos_set_status(TOS_ENOTSUP);
    rc = rows_check(k, kv->n_kv, kv->head_dim);
    if (!rc) rc = rows_check(v, kv->n_kv, kv->head_dim);
    if (!rc) rc = pair_check(q, q_out, n_heads, kv->head_dim);
    if (!rc) rc = rotary_args_check(rot, pos, kv->head_dim, q_norm, k_norm, eps);
    if (!rc && n_tokens && (!seq || !slot || ((uintptr_t)seq & 3) || ((uintptr_t)slot & 3))) rc = TOS_EINVAL;
    if (!rc && (k->type != v->type || (n_heads && q->type != k->type))) rc = TOS_ENOTSUP;
    if (rc) return tos_set_status(rc);
    int before;
    if ((rc = device_enter(&before))) return tos_set_status(rc);
    if (n_tokens == 0) return device_leave(before, 0);
    tosk_rotary_args_t a;
    memset(&a, 0, sizeof(a));
    a.q = rows_of(q, q_out);
    a.k = rows_of(k, NULL);
    a.v = rows_of(v, NULL);
    a.n_tokens = n_tokens; a.n_heads = n_heads; a.n_kv = kv->n_kv; a.hd = kv->head_dim;
    a.q_norm = q_norm; a.k_norm = k_norm; a.eps = eps;
    if (rot) a.rot = rot->r;
    a.pos = pos;
    a.append = 1;
    a.kv = paged_of(kv);
    a.seq = seq; a.slot = slot;
    return device_leave(before, tosk_rotary_rows(&a, tos_pick_stream(stream)));
}

/* ------------------------------------------------------------ attention */

static int attn_rows_check(const tos_rows_t *out, const tos_rows_t *q, int n_heads, int n_kv, int head_dim, float scale)
{
    if (n_heads <= 0 || n_heads % n_kv || !isfinite(scale * 1.5f)) return TOS_EINVAL;
    if (n_heads > (1 << 20)) return TOS_ENOTSUP;
    int rc = rows_check(out, n_heads, head_dim);
    if (!rc) rc = rows_check(q, n_heads, head_dim);
    if (!rc && out->ptr == q->ptr) rc = TOS_EINVAL;
    if (!rc && out->type != q->type) rc = TOS_ENOTSUP;
    return rc;
}

static int attn_check(const tos_rows_t *out, const tos_rows_t *q, const tos_paged_kv_t *kv, int n_heads, float scale)
{
    int rc = paged_check(kv);
    return rc ? rc : attn_rows_check(out, q, n_heads, kv->n_kv, kv->head_dim, scale);
}

static int ws_check(void *ws, size_t bytes, size_t need)
{
    if (need == 0) return TOS_OK;
    return ws && bytes >= need && ((uintptr_t)ws & 15) == 0 ? TOS_OK : TOS_EINVAL;
}

/* The 8-bit cache's workspaces begin with pools that are copied from in 16-byte pieces and by TMA. */
static int ws256_check(void *ws, size_t bytes, size_t need)
{
    return ws_check(ws, bytes, need) || (need && ((uintptr_t)ws & 255)) ? TOS_EINVAL : TOS_OK;
}

size_t tos_attention_prompt_paged_workspace_bytes(int n_seqs, int total_q, int max_q, int max_kv, int n_heads,
                                                  int n_kv, int head_dim)
{
    if (n_seqs <= 0 || total_q <= 0 || max_q <= 0 || max_kv < 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv ||
        head_dim <= 0 || head_dim > MAX_HEAD_DIM)
        return 0;
    return tosk_paged_prompt_ws_bytes(n_seqs, total_q, max_kv, n_heads, n_kv, head_dim);
}

static tosk_paged_attn_t attn_of(const tos_rows_t *out, const tos_rows_t *q, const tos_paged_kv_t *kv,
                                 const int *kv_len, int n_heads, float scale, void *ws, size_t ws_bytes)
{
    tosk_paged_attn_t a;
    memset(&a, 0, sizeof(a));
    a.out = out->ptr; a.out_stride = out->stride;
    a.q = q->ptr; a.q_stride = q->stride;
    a.type = q->type;
    a.kv = paged_of(kv);
    a.kv_len = kv_len;
    a.n_heads = n_heads;
    a.scale = scale;
    a.ws = ws; a.ws_bytes = ws_bytes;
    a.err = tos_g.err_dev;
    return a;
}

int tos_attention_prompt_paged_dev(const tos_rows_t *out, const tos_rows_t *q, const tos_paged_kv_t *kv,
                                   const int *cu_q, const int *kv_len, int n_seqs, int total_q, int max_q,
                                   int max_kv, int n_heads, float scale, void *ws, size_t ws_bytes, void *stream)
{
    int rc = attn_check(out, q, kv, n_heads, scale);
    if (!rc && (n_seqs < 0 || n_seqs > kv->n_seqs || total_q < 0 || max_q < 0 || max_kv < 0)) rc = TOS_EINVAL;
    if (!rc && n_seqs && (!cu_q || !kv_len || ((uintptr_t)cu_q & 3) || ((uintptr_t)kv_len & 3))) rc = TOS_EINVAL;
    if (!rc && (max_kv > MAX_KEYS || n_seqs > MAX_SEQS || (int64_t)max_q * (n_heads / kv->n_kv) > MAX_ROWS))
        rc = TOS_ENOTSUP;
    if (!rc)
        rc = ws_check(ws, ws_bytes, tos_attention_prompt_paged_workspace_bytes(n_seqs, total_q, max_q, max_kv,
                                                                               n_heads, kv->n_kv, kv->head_dim));
    if (rc) return tos_set_status(rc);
    int before;
    if ((rc = device_enter(&before))) return tos_set_status(rc);
    if (n_seqs == 0 || total_q == 0 || max_q == 0) return device_leave(before, 0);
    tosk_paged_attn_t a = attn_of(out, q, kv, kv_len, n_heads, scale, ws, ws_bytes);
    a.cu_q = cu_q;
    a.n_seqs = n_seqs; a.total_q = total_q; a.max_q = max_q; a.max_kv = max_kv;
    return device_leave(before, tosk_paged_prompt(&a, tos_pick_stream(stream)));
}

size_t tos_attention_decode_paged_workspace_bytes(int n_seqs, int max_kv, int prefix_len, int n_heads, int n_kv,
                                                  int head_dim)
{
    if (n_seqs <= 0 || max_kv < 0 || prefix_len < 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || head_dim <= 0 ||
        head_dim > MAX_HEAD_DIM)
        return 0;
    return tosk_paged_decode_ws_bytes(n_seqs, max_kv, prefix_len, n_heads, n_kv, head_dim);
}

int tos_attention_decode_paged_dev(const tos_rows_t *out, const tos_rows_t *q, const tos_paged_kv_t *kv,
                                   const int *kv_len, int n_seqs, int max_kv, const int *prefix_table,
                                   int prefix_len, int n_heads, float scale, void *ws, size_t ws_bytes, void *stream)
{
    int rc = attn_check(out, q, kv, n_heads, scale);
    if (!rc && (n_seqs < 0 || n_seqs > kv->n_seqs || max_kv < 0 || prefix_len < 0)) rc = TOS_EINVAL;
    if (!rc && n_seqs && (!kv_len || ((uintptr_t)kv_len & 3))) rc = TOS_EINVAL;
    if (!rc && prefix_len && (!prefix_table || ((uintptr_t)prefix_table & 3))) rc = TOS_EINVAL;
    if (!rc && (max_kv > MAX_KEYS || prefix_len > MAX_KEYS || n_seqs > MAX_SEQS ||
                (int64_t)n_seqs * (n_heads / kv->n_kv) > MAX_ROWS))
        rc = TOS_ENOTSUP;
    if (!rc)
        rc = ws_check(ws, ws_bytes, tos_attention_decode_paged_workspace_bytes(n_seqs, max_kv, prefix_len, n_heads,
                                                                               kv->n_kv, kv->head_dim));
    if (rc) return tos_set_status(rc);
    int before;
    if ((rc = device_enter(&before))) return tos_set_status(rc);
    if (n_seqs == 0) return device_leave(before, 0);
    tosk_paged_attn_t a = attn_of(out, q, kv, kv_len, n_heads, scale, ws, ws_bytes);
    a.n_seqs = a.total_q = n_seqs;
    a.max_q = 1;
    a.max_kv = max_kv;
    a.prefix_table = prefix_table;
    a.prefix_len = prefix_len;
    return device_leave(before, tosk_paged_decode(&a, tos_pick_stream(stream)));
}

/* --------------------------------------------------------- cache in 8 bits */

static int paged8_check(const tos_paged8_kv_t *c)
{
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->table) return TOS_EINVAL;
    if (c->n_pages <= 0 || c->page_size <= 0 || c->n_kv <= 0 || c->head_dim <= 0 || c->n_seqs < 0 ||
        c->table_stride <= 0 || c->block <= 0 || (c->block & (c->block - 1)) || c->page_size % c->block)
        return TOS_EINVAL;
    if ((c->type != TOS_TYPE_I8 && c->type != TOS_TYPE_F8_E4M3) || c->head_dim > MAX_HEAD_DIM || c->n_kv > (1 << 20) ||
        c->block > 1024)
        return TOS_ENOTSUP;
    if (((uintptr_t)c->k & 15) || ((uintptr_t)c->v & 15) || ((uintptr_t)c->k_scale & 3) || ((uintptr_t)c->v_scale & 3) ||
        ((uintptr_t)c->table & 3))
        return TOS_EINVAL;
    return TOS_OK;
}

static tosk_paged8_t paged8_of(const tos_paged8_kv_t *c)
{
    tosk_paged8_t p = {c->k, c->v, c->k_scale, c->v_scale, c->type, c->block, c->n_pages, c->page_size, c->n_kv,
                       c->head_dim, c->table, c->n_seqs, c->table_stride};
    return p;
}

static int packed_check(const tos_paged8_kv_t *kv, const int *cu, const int *kv_len, int n_seqs, int n_tokens)
{
    if (n_seqs < 0 || n_seqs > kv->n_seqs || n_tokens < 0) return TOS_EINVAL;
    if (n_seqs && (!cu || !kv_len || ((uintptr_t)cu & 3) || ((uintptr_t)kv_len & 3))) return TOS_EINVAL;
    return n_seqs > MAX_SEQS || n_tokens > MAX_ROWS ? TOS_ENOTSUP : TOS_OK;
}

int tos_kv_append_paged8_dev(const tos_paged8_kv_t *kv, const tos_rows_t *k, const tos_rows_t *v, const int *cu,
                             const int *kv_len, int n_seqs, int n_tokens, void *stream)
{
    int rc = paged8_check(kv);
    if (!rc) rc = rows_check(k, kv->n_kv, kv->head_dim);
    if (!rc) rc = rows_check(v, kv->n_kv, kv->head_dim);
    if (!rc) rc = packed_check(kv, cu, kv_len, n_seqs, n_tokens);
    if (!rc && k->type != v->type) rc = TOS_ENOTSUP;
    if (rc) return tos_set_status(rc);
    int before;
    if ((rc = device_enter(&before))) return tos_set_status(rc);
    if (n_seqs == 0 || n_tokens == 0) return device_leave(before, 0);
    tosk_paged8_io_t io = {paged8_of(kv), rows_of(k, NULL), rows_of(v, NULL), cu, kv_len, n_seqs, n_tokens};
    return device_leave(before, tosk_paged8_put(&io, tos_pick_stream(stream)));
}

int tos_kv_read_paged8_dev(const tos_paged8_kv_t *kv, const tos_rows_t *k_out, const tos_rows_t *v_out, const int *cu,
                           const int *kv_len, int n_seqs, int n_tokens, void *stream)
{
    int rc = paged8_check(kv);
    if (!rc && !k_out && !v_out) rc = TOS_EINVAL;
    if (!rc && k_out) rc = rows_check(k_out, kv->n_kv, kv->head_dim);
    if (!rc && v_out) rc = rows_check(v_out, kv->n_kv, kv->head_dim);
    if (!rc) rc = packed_check(kv, cu, kv_len, n_seqs, n_tokens);
    if (!rc && k_out && v_out && k_out->type != v_out->type) rc = TOS_ENOTSUP;
    if (rc) return tos_set_status(rc);
    int before;
    if ((rc = device_enter(&before))) return tos_set_status(rc);
    if (n_seqs == 0 || n_tokens == 0) return device_leave(before, 0);
    tosk_paged8_io_t io = {paged8_of(kv), rows_of(NULL, k_out), rows_of(NULL, v_out), cu, kv_len, n_seqs, n_tokens};
    return device_leave(before, tosk_paged8_get(&io, tos_pick_stream(stream)));
}

static tosk_paged_attn_t attn8_of(const tos_rows_t *out, const tos_rows_t *q, const int *kv_len, int n_heads, float scale,
                                  void *ws, size_t ws_bytes)
{
    tosk_paged_attn_t a;
    memset(&a, 0, sizeof(a));
    a.out = out->ptr; a.out_stride = out->stride;
    a.q = q->ptr; a.q_stride = q->stride;
    a.type = q->type;
    a.kv_len = kv_len;
    a.n_heads = n_heads;
    a.scale = scale;
    a.ws = ws; a.ws_bytes = ws_bytes;
    a.err = tos_g.err_dev;
    return a;
}

size_t tos_attention_prompt_paged8_workspace_bytes(int n_seqs, int total_q, int max_q, int64_t total_kv, int max_kv,
                                                   int n_heads, int n_kv, int head_dim)
{
    if (n_seqs <= 0 || total_q <= 0 || max_q <= 0 || total_kv < 0 || max_kv < 0 || n_heads <= 0 || n_kv <= 0 ||
        n_heads % n_kv || head_dim <= 0 || head_dim > MAX_HEAD_DIM)
        return 0;
    return tosk_paged8_prompt_ws_bytes(n_seqs, total_q, total_kv, max_kv, n_heads, n_kv, head_dim);
}

int tos_attention_prompt_paged8_dev(const tos_rows_t *out, const tos_rows_t *q, const tos_paged8_kv_t *kv,
                                    const int *cu_q, const int *kv_len, int n_seqs, int total_q, int max_q,
                                    int64_t total_kv, int max_kv, int n_heads, float scale, void *ws, size_t ws_bytes,
                                    void *stream)
{
    int rc = paged8_check(kv);
    if (!rc) rc = attn_rows_check(out, q, n_heads, kv->n_kv, kv->head_dim, scale);
    if (!rc) rc = packed_check(kv, cu_q, kv_len, n_seqs, total_q);
    if (!rc && (max_q < 0 || max_kv < 0 || total_kv < 0)) rc = TOS_EINVAL;
    if (!rc && (max_kv > MAX_KEYS || (int64_t)max_q * (n_heads / kv->n_kv) > MAX_ROWS || total_kv > MAX_TOTAL_KEYS))
        rc = TOS_ENOTSUP;
    const int none = n_seqs == 0 || total_q == 0 || max_q == 0;
    if (!rc && !none)
        rc = ws256_check(ws, ws_bytes, tos_attention_prompt_paged8_workspace_bytes(n_seqs, total_q, max_q, total_kv, max_kv,
                                                                                   n_heads, kv->n_kv, kv->head_dim));
    if (rc) return tos_set_status(rc);
    int before;
    if ((rc = device_enter(&before))) return tos_set_status(rc);
    if (none) return device_leave(before, 0);
    tosk_paged_attn_t a = attn8_of(out, q, kv_len, n_heads, scale, ws, ws_bytes);
    a.cu_q = cu_q;
    a.n_seqs = n_seqs; a.total_q = total_q; a.max_q = max_q; a.max_kv = max_kv;
    tosk_paged8_t c = paged8_of(kv);
    return device_leave(before, tosk_paged8_prompt(&a, &c, total_kv, tos_pick_stream(stream)));
}

size_t tos_attention_decode_paged8_workspace_bytes(int n_seqs, int max_kv, int n_heads, int n_kv, int head_dim)
{
    if (n_seqs <= 0 || max_kv < 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || head_dim <= 0 ||
        head_dim > MAX_HEAD_DIM)
        return 0;
    return tosk_paged8_decode_ws_bytes(n_seqs, max_kv, n_heads, n_kv, head_dim);
}

int tos_attention_decode_paged8_dev(const tos_rows_t *out, const tos_rows_t *q, const tos_paged8_kv_t *kv,
                                    const int *kv_len, int n_seqs, int max_kv, int n_heads, float scale, void *ws,
                                    size_t ws_bytes, void *stream)
{
    int rc = paged8_check(kv);
    if (!rc) rc = attn_rows_check(out, q, n_heads, kv->n_kv, kv->head_dim, scale);
    if (!rc && (n_seqs < 0 || n_seqs > kv->n_seqs || max_kv < 0)) rc = TOS_EINVAL;
    if (!rc && n_seqs && (!kv_len || ((uintptr_t)kv_len & 3))) rc = TOS_EINVAL;
    if (!rc && (max_kv > MAX_KEYS || n_seqs > MAX_SEQS || (int64_t)n_seqs * (n_heads / kv->n_kv) > MAX_ROWS ||
                (kv->head_dim % 16 && (int64_t)n_seqs * max_kv > MAX_TOTAL_KEYS)))
        rc = TOS_ENOTSUP;
    if (!rc)
        rc = ws256_check(ws, ws_bytes, tos_attention_decode_paged8_workspace_bytes(n_seqs, max_kv, n_heads, kv->n_kv,
                                                                                   kv->head_dim));
    if (rc) return tos_set_status(rc);
    int before;
    if ((rc = device_enter(&before))) return tos_set_status(rc);
    if (n_seqs == 0) return device_leave(before, 0);
    tosk_paged_attn_t a = attn8_of(out, q, kv_len, n_heads, scale, ws, ws_bytes);
    a.n_seqs = a.total_q = n_seqs;
    a.max_q = 1;
    a.max_kv = max_kv;
    tosk_paged8_t c = paged8_of(kv);
    return device_leave(before, tosk_paged8_decode(&a, &c, tos_pick_stream(stream)));
}

/* --------------------------------------------------------- sampling a batch */

#define MAX_VOCAB (1 << 20)   /* the sums of weights: 62 bits for as many */
#define MAX_SAMPLE_ROWS (1 << 24)

int tos_sample_rows_dev(const tos_rows_t *logits, int n_rows, int n_vocab, const tos_sample_params_t *params,
                        const float *u, int *token, float *prob, int *kept, void *stream)
{
    if (n_rows < 0 || n_vocab <= 0) return tos_set_status(TOS_EINVAL);
    if (n_vocab > MAX_VOCAB || n_rows > MAX_SAMPLE_ROWS) return tos_set_status(TOS_ENOTSUP);
    int rc = rows_check(logits, 1, n_vocab);
    if (!rc && n_rows && (!u || !token)) rc = TOS_EINVAL;
    const tos_sample_params_t none = {NULL, NULL, NULL, NULL};
    if (!params) params = &none;
    if (!rc && (((uintptr_t)u | (uintptr_t)token | (uintptr_t)prob | (uintptr_t)kept | (uintptr_t)params->temperature |
                 (uintptr_t)params->top_k | (uintptr_t)params->top_p | (uintptr_t)params->min_p) & 3))
        rc = TOS_EINVAL;
    if (rc) return tos_set_status(rc);
    int before;
    if ((rc = device_enter(&before))) return tos_set_status(rc);
    if (n_rows == 0) return device_leave(before, 0);
    tosk_sample_t a = {logits->ptr, logits->stride, logits->type, n_rows, n_vocab, params->temperature, params->top_k,
                       params->top_p, params->min_p, u, token, prob, kept};
    return device_leave(before, tosk_sample_rows(&a, tos_pick_stream(stream)));
}
