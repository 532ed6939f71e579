/* SPDX-License-Identifier: MIT
 *
 * The paged key-value cache's entry points (ornith_hip.h): arguments are
 * checked here, the work is in csrc/kernels/kv*.hip.  C99.
 *
 * What only the device knows (page numbers, slots, lengths) is checked by the
 * kernels: a word of pinned host memory per kind of mistake, which stays
 * untouched by correct calls and is looked at after the stream has ended.
 */
#include "call.h"

#include <math.h>
#include <stdio.h>
#include <string.h>

void *orn_kv_ws_get(gpu_context *ctx, size_t bytes)
{
    orn_workspace *w = &ctx->kv_ws;
    if (bytes <= w->bytes) return w->base;
    hipStreamSynchronize(ctx->stream);
    if (w->base) hipFree(w->base);
    w->base = NULL;
    w->bytes = 0;
    const size_t want = bytes + (bytes >> 3);
    if (hipMalloc(&w->base, want) != hipSuccess) {
        (void)hipGetLastError(); /* reported here, not by the next launch */
        w->base = NULL;
        orn_set_err(ctx, ORN_ENOMEM, "workspace allocation of %zu bytes failed", want);
        return NULL;
    }
    w->bytes = want;
    return w->base;
}

int gpu_kv_check(gpu_context *ctx)
{
    return ctx ? idle(ctx, 0, "gpu_kv_check") : ORN_EINVAL;
}

static int elem_bytes(int type)
{
    return type == ORN_KV_F32 ? 4 : type == ORN_KV_E4M3 ? 1 : 2;
}

/* The pages' description checked, and as the kernels take it. */
static int pages_ok(gpu_context *ctx, const ornith_kv_pages *kv, ornk_kv_pages *p, const char *who)
{
    if (!kv || !kv->K || !kv->V)
        return orn_set_err(ctx, ORN_EINVAL, "%s: no pages", who);
    if (kv->type < ORN_KV_F32 || kv->type > ORN_KV_E4M3)
        return orn_set_err(ctx, ORN_EUNSUPPORTED, "%s: cache type %d", who, kv->type);
    if (kv->head_dim < 1 || kv->head_dim > 256)
        return orn_set_err(ctx, ORN_EUNSUPPORTED, "%s: head_dim %d is not 1 to 256", who,
                           kv->head_dim);
    if (kv->page_size < 8 || kv->page_size > 1024 || (kv->page_size & (kv->page_size - 1)))
        return orn_set_err(ctx, ORN_EUNSUPPORTED,
                           "%s: page_size %d is not a power of two from 8 to 1024", who,
                           kv->page_size);
    if (kv->n_pages < 1 || kv->n_kv_heads < 1 || kv->n_kv_heads > 32767 ||
        (long long)kv->n_pages * kv->page_size > 0x7fffffffll)
        return orn_set_err(ctx, ORN_EINVAL, "%s: %d pages of %d slots, %d kv heads", who,
                           kv->n_pages, kv->page_size, kv->n_kv_heads);
    if (span(kv->n_kv_heads, kv->page_size, kv->head_dim, 1, elem_bytes(kv->type)) > UINT32_MAX)
        return orn_set_err(ctx, ORN_EUNSUPPORTED, "%s: a page of 4 GB or more", who);
    const size_t n = span(kv->n_pages, kv->n_kv_heads, kv->page_size, kv->head_dim,
                          elem_bytes(kv->type));
    if (!holds(kv->K, n) || !holds(kv->V, n))
        return orn_set_err(ctx, ORN_EINVAL, "%s: K or V is smaller than its pages", who);
    if (kv->K == kv->V) return orn_set_err(ctx, ORN_EINVAL, "%s: K is V", who);
    const float ks = kv->k_scale == 0.0f ? 1.0f : kv->k_scale;
    const float vs = kv->v_scale == 0.0f ? 1.0f : kv->v_scale;
    /* below, a scale is subnormal and has fewer digits; above, hardly a stored value is finite */
    if (kv->type == ORN_KV_E4M3 &&
        !(ks >= 0x1p-126f && ks <= 0x1p126f && vs >= 0x1p-126f && vs <= 0x1p126f))
        return orn_set_err(ctx, ORN_EINVAL, "%s: k_scale and v_scale are from 2^-126 to 2^126", who);
    memset(p, 0, sizeof *p);
    p->k = kv->K->dev;
    p->v = kv->V->dev;
    p->type = kv->type;
    p->n_pages = kv->n_pages;
    p->page = kv->page_size;
    while ((1 << p->page_log2) < kv->page_size) ++p->page_log2;
    p->kv = kv->n_kv_heads;
    p->hd = kv->head_dim;
    p->k_scale = kv->type == ORN_KV_E4M3 ? ks : 1.0f;
    p->v_scale = kv->type == ORN_KV_E4M3 ? vs : 1.0f;
    return ORN_OK;
}

/* The rotation checked; every pair's axis, and its revolutions per position:
 * base^(-p/R) / 2 pi, in 64 bits.  Each frequency is the one before it times
 * base^(-1/R), so pair p's is off by p roundings of 2^-53 and p times the rounding of
 * base^(-1/R) itself, about 2 p in all. */
static int rope_ok(gpu_context *ctx, const ornith_rope_axes *r, int hd, ornk_rope_args *a,
                   const char *who)
{
    if (r->n_axes < 1 || r->n_axes > ORN_ROPE_MAX_AXES)
        return orn_set_err(ctx, ORN_EINVAL, "%s: %d axes", who, r->n_axes);
    int R = 0, left[ORN_ROPE_MAX_AXES] = {0};
    for (int i = 0; i < r->n_axes; ++i) {
        if (r->pairs[i] < 0 || r->pairs[i] > ORN_ROPE_MAX_PAIRS)
            return orn_set_err(ctx, ORN_EINVAL, "%s: axis %d has %d pairs", who, i, r->pairs[i]);
        R += left[i] = r->pairs[i];
    }
    if (R > ORN_ROPE_MAX_PAIRS || 2 * R > hd)
        return orn_set_err(ctx, ORN_EINVAL, "%s: %d pairs in a head of %d", who, R, hd);
    if (!(r->base > 0.0 && r->base < INFINITY))
        return orn_set_err(ctx, ORN_EINVAL, "%s: base %g", who, r->base);
    for (int p = 0, ax = 0; p < R; ++p) {
        while (!left[ax]) ax = (ax + 1) % r->n_axes;
        a->axis[p] = (uint8_t)ax;
        --left[ax];
        if (r->interleaved) ax = (ax + 1) % r->n_axes;
    }
    const double step = R ? pow(r->base, -1.0 / R) : 1.0;
    double f = 0.15915494309189533577; /* 1 / 2 pi */
    for (int p = 0; p < R; ++p, f *= step) {
        if (!(f * 2147483648.0 < INFINITY)) /* no angle at the farthest position */
            return orn_set_err(ctx, ORN_EINVAL, "%s: base %g", who, r->base);
        a->turns[p] = f;
    }
    a->R = R;
    a->halves = r->halves != 0;
    return ORN_OK;
}

/* The heads' norms checked. */
static int norm_ok(gpu_context *ctx, const ornith_head_norm *n, int heads, int kv, int hd,
                   ornk_rope_args *a, const char *who)
{
    if (n->kind != ORN_NORM_RMS && n->kind != ORN_NORM_L2)
        return orn_set_err(ctx, ORN_EUNSUPPORTED, "%s: norm %d", who, n->kind);
    if (!(n->eps >= 0.0f && n->eps < INFINITY))
        return orn_set_err(ctx, ORN_EINVAL, "%s: eps %g", who, (double)n->eps);
    const int each = n->per_head != 0;
    if ((n->q_weight && heads && !holds(n->q_weight, span(each ? heads : 1, hd, 1, 1, 4))) ||
        (n->k_weight && kv && !holds(n->k_weight, span(each ? kv : 1, hd, 1, 1, 4))))
        return orn_set_err(ctx, ORN_EINVAL, "%s: weights too small", who);
    a->norm = 1 + n->kind;
    a->per_head = each;
    a->eps = n->eps;
    a->qw = n->q_weight && heads ? (const float *)n->q_weight->dev : NULL;
    a->kw = n->k_weight && kv ? (const float *)n->k_weight->dev : NULL;
    return ORN_OK;
}

/* gpu_rope_axes, and with a norm gpu_norm_rope_axes, where rope may be NULL. */
static int rope_axes(gpu_context *ctx, gpu_buffer *q_out, gpu_buffer *k_out, const gpu_buffer *Q,
                     const gpu_buffer *K, int n_tokens, int n_heads, int n_kv_heads, int head_dim,
                     const ornith_head_norm *norm, const gpu_buffer *positions,
                     const ornith_rope_axes *rope, unsigned flags, const char *who)
{
    if (!ctx) return ORN_EINVAL;
    if (!positions != !rope || (!rope && !norm) || n_tokens < 0 || n_heads < 0 || n_kv_heads < 0 || n_heads > 65535 ||
        n_kv_heads > 65535 || head_dim < 1 || !Q != !n_heads || !q_out != !n_heads ||
        !K != !n_kv_heads || !k_out != !n_kv_heads)
        return orn_set_err(ctx, ORN_EINVAL, "%s: bad arguments", who);
    if (head_dim > 4096)
        return orn_set_err(ctx, ORN_EUNSUPPORTED, "%s: head_dim %d > 4096", who, head_dim);
    ornk_rope_args a;
    memset(&a, 0, sizeof a);
    int rc = ORN_OK;
    if ((rope && (rc = rope_ok(ctx, rope, head_dim, &a, who))) ||
        (norm && (rc = norm_ok(ctx, norm, n_heads, n_kv_heads, head_dim, &a, who))))
        return rc;
    const size_t nq = span(n_tokens, n_heads, head_dim, 1, 4);
    const size_t nk = span(n_tokens, n_kv_heads, head_dim, 1, 4);
    if ((rope && !holds(positions, span(rope->n_axes, n_tokens, 1, 1, 4))) ||
        (Q && (!holds(Q, nq) || !holds(q_out, nq))) || (K && (!holds(K, nk) || !holds(k_out, nk))))
        return orn_set_err(ctx, ORN_EINVAL, "%s: buffer too small", who);
    const gpu_buffer *in[] = {positions, norm ? norm->q_weight : NULL, norm ? norm->k_weight : NULL};
    for (int i = 0; i < 3; ++i)
        if (in[i] && (in[i] == q_out || in[i] == k_out))
            return orn_set_err(ctx, ORN_EINVAL, "%s: an output aliases another argument", who);
    if ((Q && (q_out == K || q_out == k_out)) || (K && k_out == Q))
        return orn_set_err(ctx, ORN_EINVAL, "%s: an output aliases another argument", who);
    if (!n_tokens || !(n_heads + n_kv_heads)) return idle(ctx, flags, who);
    a.q = Q ? (const float *)Q->dev : NULL;
    a.q_out = Q ? (float *)q_out->dev : NULL;
    a.k = K ? (const float *)K->dev : NULL;
    a.k_out = K ? (float *)k_out->dev : NULL;
    a.pos = rope ? (const int *)positions->dev : NULL;
    a.T = n_tokens;
    a.heads = n_heads;
    a.kv = n_kv_heads;
    a.hd = head_dim;
    int prev;
    if ((rc = enter(ctx, &prev))) return rc;
    rc = orn_hip_check(ctx, (hipError_t)ornk_rope_append(NULL, &a, ctx->stream), who);
    return leave(ctx, rc, flags, prev, who);
}

int gpu_rope_axes(gpu_context *ctx, gpu_buffer *q_out, gpu_buffer *k_out, const gpu_buffer *Q,
                  const gpu_buffer *K, int n_tokens, int n_heads, int n_kv_heads, int head_dim,
                  const gpu_buffer *positions, const ornith_rope_axes *rope, unsigned flags)
{
    return rope_axes(ctx, q_out, k_out, Q, K, n_tokens, n_heads, n_kv_heads, head_dim, NULL,
                     positions, rope, flags, "gpu_rope_axes");
}

int gpu_norm_rope_axes(gpu_context *ctx, gpu_buffer *q_out, gpu_buffer *k_out, const gpu_buffer *Q,
                       const gpu_buffer *K, int n_tokens, int n_heads, int n_kv_heads, int head_dim,
                       const ornith_head_norm *norm, const gpu_buffer *positions,
                       const ornith_rope_axes *rope, unsigned flags)
{
    static const char who[] = "gpu_norm_rope_axes";
    if (ctx && !norm) return orn_set_err(ctx, ORN_EINVAL, "%s: no norm", who);
    return rope_axes(ctx, q_out, k_out, Q, K, n_tokens, n_heads, n_kv_heads, head_dim, norm,
                     positions, rope, flags, who);
}

/* gpu_kv_append, and with a norm gpu_norm_kv_append, whose queries need no rotation. */
static int kv_append(gpu_context *ctx, const ornith_kv_pages *kv, const gpu_buffer *K,
                     const gpu_buffer *V, int n_tokens, const gpu_buffer *slots, gpu_buffer *q_out,
                     const gpu_buffer *Q, int n_heads, const ornith_head_norm *norm,
                     const gpu_buffer *positions, const ornith_rope_axes *rope, unsigned flags,
                     const char *who)
{
    if (!ctx) return ORN_EINVAL;
    ornk_kv_pages p;
    int rc = pages_ok(ctx, kv, &p, who);
    if (rc) return rc;
    if (!K || !V || !slots || n_tokens < 0 || n_heads < 0 || n_heads > 65535 || !Q != !n_heads ||
        !q_out != !n_heads || !rope != !positions || (Q && !rope && !norm))
        return orn_set_err(ctx, ORN_EINVAL, "%s: bad arguments", who);
    ornk_rope_args a;
    memset(&a, 0, sizeof a);
    if ((rope && (rc = rope_ok(ctx, rope, p.hd, &a, who))) ||
        (norm && (rc = norm_ok(ctx, norm, n_heads, p.kv, p.hd, &a, who))))
        return rc;
    const size_t nq = span(n_tokens, n_heads, p.hd, 1, 4), nk = span(n_tokens, p.kv, p.hd, 1, 4);
    if (!holds(K, nk) || !holds(V, nk) || !holds(slots, span(n_tokens, 1, 1, 1, 4)) ||
        (Q && (!holds(Q, nq) || !holds(q_out, nq))) ||
        (rope && !holds(positions, span(rope->n_axes, n_tokens, 1, 1, 4))))
        return orn_set_err(ctx, ORN_EINVAL, "%s: buffer too small", who);
    const gpu_buffer *in[] = {K, V, Q, slots, positions, norm ? norm->q_weight : NULL,
                              norm ? norm->k_weight : NULL};
    for (int i = 0; i < 7; ++i)
        if (in[i] && (in[i] == kv->K || in[i] == kv->V || (in[i] == q_out && i != 2)))
            return orn_set_err(ctx, ORN_EINVAL, "%s: an output aliases another argument", who);
    if (q_out && (q_out == kv->K || q_out == kv->V))
        return orn_set_err(ctx, ORN_EINVAL, "%s: q_out is the cache", who);
    if (!n_tokens) return idle(ctx, flags, who);
    a.q = Q ? (const float *)Q->dev : NULL;
    a.q_out = Q ? (float *)q_out->dev : NULL;
    a.k = (const float *)K->dev;
    a.v = (const float *)V->dev;
    a.pos = rope ? (const int *)positions->dev : NULL;
    a.slots = (const int *)slots->dev;
    a.T = n_tokens;
    a.heads = n_heads;
    a.kv = p.kv;
    a.hd = p.hd;
    int prev;
    if ((rc = enter(ctx, &prev))) return rc;
    if (!(rc = err_words(ctx, &p.err)))
        rc = orn_hip_check(ctx, (hipError_t)ornk_rope_append(&p, &a, ctx->stream), who);
    return leave(ctx, rc, flags, prev, who);
}

int gpu_kv_append(gpu_context *ctx, const ornith_kv_pages *kv, const gpu_buffer *K,
                  const gpu_buffer *V, int n_tokens, const gpu_buffer *slots, gpu_buffer *q_out,
                  const gpu_buffer *Q, int n_heads, const gpu_buffer *positions,
                  const ornith_rope_axes *rope, unsigned flags)
{
    return kv_append(ctx, kv, K, V, n_tokens, slots, q_out, Q, n_heads, NULL, positions, rope, flags,
                     "gpu_kv_append");
}

int gpu_norm_kv_append(gpu_context *ctx, const ornith_kv_pages *kv, const gpu_buffer *K,
                       const gpu_buffer *V, int n_tokens, const gpu_buffer *slots,
                       gpu_buffer *q_out, const gpu_buffer *Q, int n_heads,
                       const ornith_head_norm *norm, const gpu_buffer *positions,
                       const ornith_rope_axes *rope, unsigned flags)
{
    static const char who[] = "gpu_norm_kv_append";
    if (ctx && !norm) return orn_set_err(ctx, ORN_EINVAL, "%s: no norm", who);
    return kv_append(ctx, kv, K, V, n_tokens, slots, q_out, Q, n_heads, norm, positions, rope, flags,
                     who);
}

/* The sequences' table and lengths; *bound: the largest length there may be. */
static int seqs_ok(gpu_context *ctx, const ornk_kv_pages *p, int n_seqs, const gpu_buffer *table,
                   int max_pages, const gpu_buffer *lens, int max_len, int *bound, const char *who)
{
    if (!table || !lens || n_seqs < 0 || max_pages < 0 || max_len < 0)
        return orn_set_err(ctx, ORN_EINVAL, "%s: bad arguments", who);
    if (n_seqs > 65535)
        return orn_set_err(ctx, ORN_EUNSUPPORTED, "%s: %d sequences (at most 65535)", who, n_seqs);
    const long long width = (long long)max_pages * p->page;
    if (width > 0x7fff0000ll || max_len > width)  /* indexes a stretch past a length fit an int */
        return orn_set_err(ctx, ORN_EINVAL, "%s: max_len %d, and %d pages of %d in the table", who,
                           max_len, max_pages, p->page);
    if (!holds(table, span(n_seqs, max_pages, 1, 1, 4)) || !holds(lens, span(n_seqs, 1, 1, 1, 4)))
        return orn_set_err(ctx, ORN_EINVAL, "%s: table or lens too small", who);
    *bound = max_len ? max_len : (int)width;
    return ORN_OK;
}

int gpu_kv_attend(gpu_context *ctx, const ornith_kv_pages *kv, gpu_buffer *out,
                  const gpu_buffer *Q, int n_seqs, int n_heads, const gpu_buffer *table,
                  int max_pages, const gpu_buffer *lens, const ornith_attend_opts *opts)
{
    static const char who[] = "gpu_kv_attend";
    static const ornith_attend_opts none;
    if (!ctx) return ORN_EINVAL;
    const ornith_attend_opts *o = opts ? opts : &none;
    ornk_kv_pages p;
    int bound, rc = pages_ok(ctx, kv, &p, who);
    if (rc || (rc = seqs_ok(ctx, &p, n_seqs, table, max_pages, lens, o->max_len, &bound, who)))
        return rc;
    if (!out || !Q || n_heads < 1 || n_heads > 65535 || n_heads % p.kv)
        return orn_set_err(ctx, ORN_EINVAL, "%s: bad arguments, or %d heads over %d kv heads", who,
                           n_heads, p.kv);
    if ((size_t)n_seqs * p.kv * ((n_heads / p.kv + 15) / 16) > 1 << 21)
        return orn_set_err(ctx, ORN_EUNSUPPORTED, "%s: %d sequences of %d kv heads", who, n_seqs, p.kv);
    if (!isfinite(o->scale)) return orn_set_err(ctx, ORN_EINVAL, "%s: scale", who);
    const size_t nq = span(n_seqs, n_heads, p.hd, 1, 4);
    if (!holds(Q, nq) || !holds(out, nq))
        return orn_set_err(ctx, ORN_EINVAL, "%s: Q or out too small", who);
    if (o->score_in && !o->score_out)
        return orn_set_err(ctx, ORN_EINVAL, "%s: score_in without score_out", who);
    if (o->score_new < 0) return orn_set_err(ctx, ORN_EINVAL, "%s: score_new", who);
    if (o->score_out) {
        const size_t ns = o->score_stride < 0 ? SIZE_MAX
                                              : span(n_seqs, p.kv, o->score_stride, 1, 4);
        if (o->score_stride < bound || !holds(o->score_out, ns) ||
            (o->score_in && !holds(o->score_in, ns)))
            return orn_set_err(ctx, ORN_EINVAL, "%s: scores too small for lengths of %d", who,
                               bound);
    }
    const gpu_buffer *in[] = {Q, table, lens, kv->K, kv->V, o->score_in};
    for (int i = 0; i < 6; ++i)
        if (in[i] && (in[i] == out || (in[i] == o->score_out && i < 5)))
            return orn_set_err(ctx, ORN_EINVAL, "%s: an output aliases another argument", who);
    if (out == o->score_out) return orn_set_err(ctx, ORN_EINVAL, "%s: out is score_out", who);
    if (!n_seqs) return idle(ctx, o->flags, who);
    ornk_attend_args a;
    memset(&a, 0, sizeof a);
    a.q = (const float *)Q->dev;
    a.out = (float *)out->dev;
    a.table = (const int *)table->dev;
    a.lens = (const int *)lens->dev;
    a.n_seqs = n_seqs;
    a.heads = n_heads;
    a.max_pages = max_pages;
    a.max_len = bound;
    a.scale = o->scale != 0.0f ? o->scale : 1.0f / sqrtf((float)p.hd);
    a.score_in = o->score_in ? (const float *)o->score_in->dev : NULL;
    a.score_out = o->score_out ? (float *)o->score_out->dev : NULL;
    a.score_stride = (size_t)o->score_stride;
    a.decay = o->decay;
    a.score_new = o->score_new;
    int prev;
    if ((rc = enter(ctx, &prev))) return rc;
    if (!(rc = err_words(ctx, &p.err))) {
        const size_t ws = ornk_kv_attend_ws(&p, &a);
        if (ws && !(a.ws = orn_kv_ws_get(ctx, ws))) rc = ORN_ENOMEM;
    }
    if (!rc) rc = orn_hip_check(ctx, (hipError_t)ornk_kv_attend(&p, &a, ctx->stream), who);
    return leave(ctx, rc, o->flags, prev, who);
}

int gpu_kv_evict(gpu_context *ctx, const ornith_kv_pages *kv, int n_seqs, const gpu_buffer *table,
                 int max_pages, const gpu_buffer *lens, const gpu_buffer *score, int score_stride,
                 const gpu_buffer *dst_table, int dst_pages, gpu_buffer *dst_lens,
                 gpu_buffer *dst_score, int dst_stride, gpu_buffer *kept,
                 const ornith_evict_opts *opts)
{
    static const char who[] = "gpu_kv_evict";
    if (!ctx) return ORN_EINVAL;
    ornk_kv_pages p;
    int bound, rc = pages_ok(ctx, kv, &p, who);
    if (rc) return rc;
    if (!opts || opts->keep < 1 || opts->sink < 0 || opts->recent < 0 ||
        (long long)opts->sink + opts->recent > opts->keep)
        return orn_set_err(ctx, ORN_EINVAL, "%s: keep >= sink + recent, at least 1", who);
    if ((rc = seqs_ok(ctx, &p, n_seqs, table, max_pages, lens, opts->max_len, &bound, who)))
        return rc;
    if (!score || !dst_table || !dst_lens || !kept || dst_pages < 0)
        return orn_set_err(ctx, ORN_EINVAL, "%s: bad arguments", who);
    const int most = opts->keep < bound ? opts->keep : bound; /* the longest result */
    if (most > 1 << 27) /* 2^25 stretches of 4 rows: 32 launches of the mover */
        return orn_set_err(ctx, ORN_EUNSUPPORTED, "%s: %d tokens kept (at most 2^27)", who, most);
    if ((long long)dst_pages * p.page < most || !holds(dst_table, span(n_seqs, dst_pages, 1, 1, 4)))
        return orn_set_err(ctx, ORN_EINVAL, "%s: dst_table has no room for %d tokens", who, most);
    if (score_stride < bound || !holds(score, span(n_seqs, p.kv, score_stride, 1, 4)) ||
        (dst_score &&
         (dst_stride < most || !holds(dst_score, span(n_seqs, p.kv, dst_stride, 1, 4)))))
        return orn_set_err(ctx, ORN_EINVAL, "%s: scores too small", who);
    if (!holds(dst_lens, span(n_seqs, 1, 1, 1, 4)) ||
        !holds(kept, span(n_seqs, p.kv, opts->keep, 1, 4)))
        return orn_set_err(ctx, ORN_EINVAL, "%s: dst_lens or kept too small", who);
    if (dst_table == table && dst_pages != max_pages)
        return orn_set_err(ctx, ORN_EINVAL, "%s: one table of two widths", who);
    if (dst_score == score && dst_stride != score_stride)
        return orn_set_err(ctx, ORN_EINVAL, "%s: one score buffer of two strides", who);
    const gpu_buffer *all[] = {kv->K, kv->V, table, lens, score, dst_table, dst_lens, dst_score, kept};
    for (int i = 0; i < 9; ++i)
        for (int j = i + 1; j < 9; ++j)
            if (all[i] && all[i] == all[j] && !(i == 2 && j == 5) && !(i == 3 && j == 6) &&
                !(i == 4 && j == 7))
                return orn_set_err(ctx, ORN_EINVAL, "%s: two arguments are one buffer", who);
    if (!n_seqs) return idle(ctx, opts->flags, who);
    ornk_evict_args a;
    memset(&a, 0, sizeof a);
    a.table = (const int *)table->dev;
    a.lens = (const int *)lens->dev;
    a.dst_table = (const int *)dst_table->dev;
    a.score = (const float *)score->dev;
    a.dst_score = dst_score ? (float *)dst_score->dev : NULL;
    a.score_stride = (size_t)score_stride;
    a.dst_stride = (size_t)dst_stride;
    a.dst_lens = (int *)dst_lens->dev;
    a.kept = (int *)kept->dev;
    a.n_seqs = n_seqs;
    a.max_pages = max_pages;
    a.dst_pages = dst_pages;
    a.max_len = bound;
    a.keep = opts->keep;
    a.sink = opts->sink;
    a.recent = opts->recent;
    a.in_place = dst_table == table;
    int prev;
    if ((rc = enter(ctx, &prev))) return rc;
    if (!(rc = err_words(ctx, &p.err)) &&
        !(a.counts = (int *)orn_kv_ws_get(ctx, (size_t)n_seqs * sizeof(int))))
        rc = ORN_ENOMEM;
    if (!rc) rc = orn_hip_check(ctx, (hipError_t)ornk_kv_evict(&p, &a, ctx->stream), who);
    return leave(ctx, rc, opts->flags, prev, who);
}
