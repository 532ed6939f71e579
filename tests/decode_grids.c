/* The launches of linear attention and sampling (csrc/kernels/linear.hip, sample.hip, their
 * host side) without a GPU.  For a line on standard input of
 *   l n_seqs heads dk dv max_len      linear attention
 *   s rows n 0 0 0                    sampling
 * a line of "kernel x y z bytes" for each launch, side by side: the kernel's name as the
 * compiler forms it, its grid, and the bytes of the call's workspace. */
#include "../ornith-flight_amd/csrc/kernels/launch.h"
#include <hip/hip_runtime_api.h>

#include <stdio.h>
#include <string.h>

static dim3 grid, block;
static size_t room;
static struct {
    const void *f;
    const char *name;
} kernels[256];
static int n_kernels;

hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t lds, hipStream_t s)
{
    return grid = g, block = b, hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *lds, hipStream_t *s)
{
    return *g = grid, *b = block, *lds = 0, *s = NULL, hipSuccess;
}
hipError_t hipLaunchKernel(const void *f, dim3 g, dim3 b, void **args, size_t lds, hipStream_t s)
{
    for (int i = 0; i < n_kernels; ++i)
        if (kernels[i].f == f) printf("%s %u %u %u %zu ", kernels[i].name, g.x, g.y, g.z, room);
    return hipSuccess;
}
hipError_t hipGetLastError(void) { return hipSuccess; }
void **__hipRegisterFatBinary(const void *data) { return NULL; }
void __hipUnregisterFatBinary(void **m) {}
void __hipRegisterFunction(void **m, const void *f, char *name, const char *dev, unsigned limit, void *t,
                           void *b, dim3 *bd, dim3 *gd, int *w)
{
    if (n_kernels < 256) kernels[n_kernels].f = f, kernels[n_kernels++].name = dev;
}

int main(void)
{
    char what;
    int a, b, c, d, e;
    while (scanf(" %c%d%d%d%d%d", &what, &a, &b, &c, &d, &e) == 6) {
        if (what == 'l') {
            ornk_linear_args l;
            memset(&l, 0, sizeof l);
            l.n_seqs = a, l.heads = b, l.dk = c, l.dv = d, l.max_len = e;
            room = ornk_linear_ws(&l);
            ornk_linear(&l, NULL);
        } else {
            ornk_sample_args s;
            memset(&s, 0, sizeof s);
            s.rows = a, s.n = b, s.stride = b;
            room = ornk_sample_ws(&s);
            ornk_sample(&s, NULL);
        }
        printf("\n");
    }
    return 0;
}
