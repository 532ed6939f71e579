/* SPDX-License-Identifier: MIT
 *
 * gpu_linear_attend (ornith_hip.h): arguments are checked here, the work is in
 * csrc/kernels/linear.hip, which checks the numbers in device buffers.  C99.
 */
#include "call.h"

#include <math.h>
#include <string.h>

int gpu_linear_attend(gpu_context *ctx, const ornith_linear_states *st, gpu_buffer *out,
                      const gpu_buffer *Q, const gpu_buffer *K, const gpu_buffer *V, int q_heads,
                      int k_heads, int v_heads, int n_tokens, const gpu_buffer *decay, int n_seqs,
                      const gpu_buffer *starts, const gpu_buffer *slots_in,
                      const gpu_buffer *slots_out, const ornith_linear_opts *opts)
{
    static const char who[] = "gpu_linear_attend";
    static const ornith_linear_opts none;
    if (!ctx) return ORN_EINVAL;
    const ornith_linear_opts *o = opts ? opts : &none;
    if (!st || !out || !Q || !K || !V || !decay || n_tokens < 0 || n_seqs < 0 || o->max_len < 0 ||
        (!starts && n_seqs != n_tokens))
        return orn_set_err(ctx, ORN_EINVAL, "%s: bad arguments", who);
    const int H = st->n_heads, dk = st->key_dim, dv = st->value_dim;
    if (H < 1 || H > 65535 || dk < 1 || dk > 256 || dv < 1 || dv > 256 || n_seqs > 65535)
        return orn_set_err(ctx, ORN_EUNSUPPORTED, "%s: %d sequences, %d heads of %d x %d", who, n_seqs,
                           H, dk, dv);
    if (q_heads < 1 || k_heads < 1 || v_heads < 1 || H % q_heads || H % k_heads || H % v_heads)
        return orn_set_err(ctx, ORN_EINVAL, "%s: %d, %d and %d heads for %d", who, q_heads, k_heads,
                           v_heads, H);
    if (n_tokens > 0x7fff0000) /* indexes a chunk past the end fit an int */
        return orn_set_err(ctx, ORN_EUNSUPPORTED, "%s: %d tokens (at most 2^31 - 2^16)", who, n_tokens);
    if (!isfinite(o->scale)) return orn_set_err(ctx, ORN_EINVAL, "%s: scale", who);
    if (!holds(Q, span(n_tokens, q_heads, dk, 1, 4)) || !holds(K, span(n_tokens, k_heads, dk, 1, 4)) ||
        !holds(V, span(n_tokens, v_heads, dv, 1, 4)) || !holds(out, span(n_tokens, H, dv, 1, 4)) ||
        !holds(decay, span(o->per_token ? n_tokens : 1, H, 1, 1, 4)) ||
        (starts && !holds(starts, span((size_t)n_seqs + 1, 1, 1, 1, 4))) ||
        (slots_in && !holds(slots_in, span(n_seqs, 1, 1, 1, 4))) ||
        (slots_out && !holds(slots_out, span(n_seqs, 1, 1, 1, 4))))
        return orn_set_err(ctx, ORN_EINVAL, "%s: buffer too small", who);
    if (slots_in || slots_out) {
        if (st->n_slots < 0 || !holds(st->S, span(st->n_slots, H, dk, dv, 4)))
            return orn_set_err(ctx, ORN_EINVAL, "%s: no room for %d states", who, st->n_slots);
    }
    const gpu_buffer *in[] = {Q, K, V, decay, starts, slots_in, slots_out};
    for (int i = 0; i < 7; ++i)
        if (in[i] && (in[i] == out || in[i] == st->S))
            return orn_set_err(ctx, ORN_EINVAL, "%s: an output aliases another argument", who);
    if (out == st->S) return orn_set_err(ctx, ORN_EINVAL, "%s: out is the states", who);
    if (!n_seqs) return idle(ctx, o->flags, who);
    ornk_linear_args a;
    memset(&a, 0, sizeof a);
    a.q = (const float *)Q->dev;
    a.k = (const float *)K->dev;
    a.v = (const float *)V->dev;
    a.decay = (const float *)decay->dev;
    a.out = (float *)out->dev;
    a.S = slots_in || slots_out ? (float *)st->S->dev : NULL;
    a.starts = starts ? (const int *)starts->dev : NULL;
    a.in = slots_in ? (const int *)slots_in->dev : NULL;
    a.out_slots = slots_out ? (const int *)slots_out->dev : NULL;
    a.n_seqs = n_seqs;
    a.n_tokens = n_tokens;
    a.n_slots = st->n_slots;
    a.heads = H;
    a.qh = q_heads;
    a.kh = k_heads;
    a.vh = v_heads;
    a.dk = dk;
    a.dv = dv;
    a.max_len = !starts ? 1 : o->max_len && o->max_len < n_tokens ? o->max_len : n_tokens;
    a.per_token = o->per_token != 0;
    a.complement = o->complement != 0;
    a.scale = o->scale != 0.0f ? o->scale : 1.0f / sqrtf((float)dk);
    int prev, rc;
    if ((rc = enter(ctx, &prev))) return rc;
    if (!(rc = err_words(ctx, &a.err))) {
        const size_t ws = ornk_linear_ws(&a);
        if (ws && !(a.ws = orn_kv_ws_get(ctx, ws))) rc = ORN_ENOMEM;
    }
    if (!rc) rc = orn_hip_check(ctx, (hipError_t)ornk_linear(&a, ctx->stream), who);
    return leave(ctx, rc, o->flags, prev, who);
}
