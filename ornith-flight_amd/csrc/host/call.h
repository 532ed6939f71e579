/* SPDX-License-Identifier: MIT
 *
 * What the entry points of a decode step (kv.c, linear.c, sample.c) begin and end
 * with: sizes of buffers, the context's device, the stream's end and what the
 * kernels reported.
 */
#ifndef ORNITH_HOST_CALL_H
#define ORNITH_HOST_CALL_H

#include <stdio.h>

#include "internal.h"

/* a * b * c * d * elem bytes, SIZE_MAX where that passes 64 bits */
static inline size_t span(size_t a, size_t b, size_t c, size_t d, size_t elem)
{
    size_t n = a;
    if (__builtin_mul_overflow(n, b, &n) || __builtin_mul_overflow(n, c, &n) ||
        __builtin_mul_overflow(n, d, &n) || __builtin_mul_overflow(n, elem, &n))
        return SIZE_MAX;
    return n;
}

static inline int holds(const gpu_buffer *b, size_t bytes) { return b && b->dev && bytes <= b->size; }

/* Calls run on the context's device, whichever is current. */
static inline int enter(gpu_context *ctx, int *prev)
{
    *prev = ctx->device;
    int rc = orn_hip_check(ctx, hipGetDevice(prev), "hipGetDevice");
    if (!rc && *prev != ctx->device)
        rc = orn_hip_check(ctx, hipSetDevice(ctx->device), "hipSetDevice");
    return rc;
}

static inline int report(gpu_context *ctx, const char *who)
{
    static const char *const what[ORNK_KV_ERR_WORDS] = {
        "a page number of row %d is outside the pages", "slot of token %d is outside the pages",
        "the length of sequence %d is outside its bounds",
        "a slot of sequence %d is outside the states",
        "the tokens of sequence %d are outside their bounds",
        "the request or the random number of row %d is outside its bounds"};
    int rc = ORN_OK;
    for (int i = 0; i < ORNK_KV_ERR_WORDS; ++i) {
        volatile int *w = ctx->ctl_host + ORN_CTL_KV + i;
        const int at = *w;
        if (!at) continue;
        *w = 0;
        if (rc) continue;
        char msg[96];
        snprintf(msg, sizeof msg, what[i], at - 1);
        rc = orn_set_err(ctx, ORN_EINVAL, "%s: %s (this call or an earlier asynchronous one)", who,
                         msg);
    }
    return rc;
}

static inline int leave(gpu_context *ctx, int rc, unsigned flags, int prev, const char *who)
{
    if (!rc && !(flags & ORN_KV_ASYNC)) {
        rc = orn_hip_check(ctx, hipStreamSynchronize(ctx->stream), who);
        if (!rc) rc = report(ctx, who);
    }
    if (prev != ctx->device) (void)hipSetDevice(prev);
    return rc;
}

/* A call with nothing of its own to do. */
static inline int idle(gpu_context *ctx, unsigned flags, const char *who)
{
    int prev;
    const int rc = enter(ctx, &prev);
    return rc ? rc : leave(ctx, ORN_OK, flags, prev, who);
}

static inline int err_words(gpu_context *ctx, int **err)
{
    void *d = NULL;
    const int rc = orn_hip_check(ctx, hipHostGetDevicePointer(&d, ctx->ctl_host, 0),
                                 "hipHostGetDevicePointer");
    *err = (int *)d + ORN_CTL_KV;
    return rc;
}

#endif /* ORNITH_HOST_CALL_H */
