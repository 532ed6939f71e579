/* The paged cache's entry points (csrc/host/kv.c) without a GPU: HIP calls and
 * kernel launches that only count, for the tests of what the host refuses. */
#include "../ornith-flight_amd/csrc/host/kv.c"

#include <stdlib.h>

int kv_launches, kv_syncs, kv_device, kv_no_room;
ornk_rope_args kv_rope;
ornk_attend_args kv_attend;
ornk_evict_args kv_evict;

int orn_set_err(gpu_context *ctx, int code, const char *fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(ctx->err, sizeof ctx->err, fmt, ap);
    va_end(ap);
    return code;
}

int orn_hip_check(gpu_context *ctx, hipError_t e, const char *what)
{
    return e == hipSuccess ? ORN_OK : orn_set_err(ctx, ORN_EHIP, "%s: %d", what, (int)e);
}

hipError_t hipGetDevice(int *d) { return *d = kv_device, hipSuccess; }
hipError_t hipSetDevice(int d) { return kv_device = d, hipSuccess; }
hipError_t hipHostGetDevicePointer(void **d, void *h, unsigned f) { return *d = h, hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t s) { return ++kv_syncs, hipSuccess; }
hipError_t hipGetLastError(void) { return hipSuccess; }
hipError_t hipFree(void *p) { return free(p), hipSuccess; }
hipError_t hipMalloc(void **p, size_t n)
{
    *p = kv_no_room ? NULL : malloc(n < 4096 ? n : 4096);
    return *p ? hipSuccess : hipErrorOutOfMemory;
}

int ornk_rope_append(const ornk_kv_pages *p, const ornk_rope_args *a, hipStream_t s)
{
    return kv_rope = *a, ++kv_launches, hipSuccess;
}
size_t ornk_kv_attend_ws(const ornk_kv_pages *p, const ornk_attend_args *a) { return 64; }
int ornk_kv_attend(const ornk_kv_pages *p, const ornk_attend_args *a, hipStream_t s)
{
    return kv_attend = *a, ++kv_launches, hipSuccess;
}
int ornk_kv_evict(const ornk_kv_pages *p, const ornk_evict_args *a, hipStream_t s)
{
    return kv_evict = *a, ++kv_launches, hipSuccess;
}

gpu_context *kv_test_context(int device)
{
    gpu_context *c = calloc(1, sizeof *c);
    c->ctl_host = calloc(64, sizeof(int));
    c->device = device;
    return c;
}
gpu_buffer *kv_test_buffer(size_t size)
{
    gpu_buffer *b = calloc(1, sizeof *b);
    b->dev = b;
    b->size = size;
    return b;
}
const char *kv_test_error(gpu_context *c) { return c->err; }
/* an error word, as a kernel sets it */
void kv_test_mark(gpu_context *c, int what, int at) { c->ctl_host[ORN_CTL_KV + what] = 1 + at; }
double kv_test_turns(int p) { return kv_rope.turns[p]; }
int kv_test_axis(int p) { return kv_rope.axis[p]; }
int kv_test_workspace(gpu_context *c) { return c->kv_ws.base != NULL; }
