/* The entry points of linear attention and sampling (csrc/host/linear.c, sample.c)
 * without a GPU: HIP calls and kernel launches that only count, for the tests of what
 * the host refuses. */
#include "../ornith-flight_amd/csrc/host/linear.c"
#include "../ornith-flight_amd/csrc/host/sample.c"

#include <stdlib.h>

int decode_launches, decode_device, decode_no_room;
ornk_linear_args decode_linear;
ornk_sample_args decode_sample;

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

void *orn_kv_ws_get(gpu_context *ctx, size_t bytes) { return decode_no_room ? NULL : ctx; }
hipError_t hipGetDevice(int *d) { return *d = decode_device, hipSuccess; }
hipError_t hipSetDevice(int d) { return decode_device = d, hipSuccess; }
hipError_t hipHostGetDevicePointer(void **d, void *h, unsigned f) { return *d = h, hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t s) { return hipSuccess; }

size_t ornk_linear_ws(const ornk_linear_args *a) { return 64; }
int ornk_linear(const ornk_linear_args *a, hipStream_t s)
{
    return decode_linear = *a, ++decode_launches, hipSuccess;
}
size_t ornk_sample_ws(const ornk_sample_args *a) { return 64; }
int ornk_sample(const ornk_sample_args *a, hipStream_t s)
{
    return decode_sample = *a, ++decode_launches, hipSuccess;
}

gpu_context *decode_context(int device)
{
    gpu_context *c = calloc(1, sizeof *c);
    c->ctl_host = calloc(64, sizeof(int));
    c->device = device;
    return c;
}
gpu_buffer *decode_buffer(size_t size)
{
    gpu_buffer *b = calloc(1, sizeof *b);
    b->dev = b;
    b->size = size;
    return b;
}
const char *decode_error(gpu_context *c) { return c->err; }
/* an error word, as a kernel sets it */
void decode_mark(gpu_context *c, int what, int at) { c->ctl_host[ORN_CTL_KV + what] = 1 + at; }
double decode_unit(void) { return decode_sample.unit; }
int decode_max_len(void) { return decode_linear.max_len; }
