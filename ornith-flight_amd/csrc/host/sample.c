/* SPDX-License-Identifier: MIT
 *
 * gpu_sample (ornith_hip.h): arguments are checked here, the requests and random
 * numbers, which only the device knows, by csrc/kernels/sample.hip.  C99.
 */
#include "call.h"

#include <string.h>

int gpu_sample(gpu_context *ctx, gpu_buffer *tokens, gpu_buffer *prob, const gpu_buffer *logits,
               int n_rows, int n_vocab, int row_stride, const gpu_buffer *requests,
               const gpu_buffer *u, unsigned flags)
{
    static const char who[] = "gpu_sample";
    if (!ctx) return ORN_EINVAL;
    if (!tokens || !logits || !requests || !u || n_rows < 0 || n_vocab < 1 ||
        (row_stride && row_stride < n_vocab))
        return orn_set_err(ctx, ORN_EINVAL, "%s: bad arguments", who);
    if (n_rows > 65535 || n_vocab > ORN_SAMPLE_MAX_VOCAB)
        return orn_set_err(ctx, ORN_EUNSUPPORTED, "%s: %d rows of %d tokens", who, n_rows, n_vocab);
    const size_t stride = row_stride ? (size_t)row_stride : (size_t)n_vocab;
    const size_t n = n_rows ? ((size_t)n_rows - 1) * stride + (size_t)n_vocab : 0; /* < 2^48 */
    if (!holds(logits, 4 * n) || !holds(tokens, 4 * (size_t)n_rows) || !holds(u, 4 * (size_t)n_rows) ||
        (prob && !holds(prob, 4 * (size_t)n_rows)) ||
        !holds(requests, sizeof(ornith_sample_request) * (size_t)n_rows))
        return orn_set_err(ctx, ORN_EINVAL, "%s: buffer too small", who);
    const gpu_buffer *in[] = {logits, requests, u};
    for (int i = 0; i < 3; ++i)
        if (in[i] == tokens || in[i] == prob)
            return orn_set_err(ctx, ORN_EINVAL, "%s: an output aliases another argument", who);
    if (tokens == prob) return orn_set_err(ctx, ORN_EINVAL, "%s: tokens is prob", who);
    if (!n_rows) return idle(ctx, flags, who);
    ornk_sample_args a;
    memset(&a, 0, sizeof a);
    a.logits = (const float *)logits->dev;
    a.u = (const float *)u->dev;
    a.requests = requests->dev;
    a.tokens = (int *)tokens->dev;
    a.prob = prob ? (float *)prob->dev : NULL;
    a.rows = n_rows;
    a.n = n_vocab;
    a.stride = stride;
    /* a token's weight relative to the largest in as many bits as leave 62 for the sum,
     * and no more than a double's sum with 2^52 has */
    int bits = 51;
    while ((size_t)n_vocab > (size_t)1 << (62 - bits)) --bits; /* 42 at the largest */
    a.unit = (double)((uint64_t)1 << bits);
    int prev, rc;
    if ((rc = enter(ctx, &prev))) return rc;
    if (!(rc = err_words(ctx, &a.err))) {
        const size_t ws = ornk_sample_ws(&a);
        if (ws && !(a.ws = orn_kv_ws_get(ctx, ws))) rc = ORN_ENOMEM;
    }
    if (!rc) rc = orn_hip_check(ctx, (hipError_t)ornk_sample(&a, ctx->stream), who);
    return leave(ctx, rc, flags, prev, who);
}
