/* The launches of the paged cache's kernels (csrc/kernels/kv*.hip, their host side)
 * without a GPU.  For a line on standard input of
 *   e hd type kv n_seqs max_len keep in_place        an eviction
 *   a hd type kv n_seqs max_len heads score          an attention
 *   r hd R halves kv T heads slots                   a rotation or an append
 * a line of "x y z threads" for each launch, side by side. */
#include "../ornith-flight_amd/csrc/kernels/launch.h"
#include <hip/hip_runtime_api.h>

#include <stdio.h>
#include <string.h>

static dim3 grid, block;

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
    printf("%u %u %u %u ", g.x, g.y, g.z, b.x * b.y * b.z);
    return hipSuccess;
}
hipError_t hipGetLastError(void) { return hipSuccess; }
void **__hipRegisterFatBinary(const void *data) { return NULL; }
void __hipUnregisterFatBinary(void **m) {}
void __hipRegisterFunction(void **m, const void *f, char *name, const char *dev, unsigned limit, void *t,
                           void *b, dim3 *bd, dim3 *gd, int *w)
{
}

int main(void)
{
    char what;
    int a, b, c, d, e, f, g;
    while (scanf(" %c%d%d%d%d%d%d%d", &what, &a, &b, &c, &d, &e, &f, &g) == 8) {
        ornk_kv_pages p;
        memset(&p, 0, sizeof p);
        p.hd = a;
        p.page = 16;
        p.page_log2 = 4;
        if (what == 'r') {
            static ornk_rope_args r;
            p.kv = r.kv = d;
            r.hd = a, r.R = b, r.halves = c, r.T = e, r.heads = f;
            r.slots = g ? &a : NULL;
            ornk_rope_append(&p, &r, NULL);
        } else if (what == 'a') {
            ornk_attend_args t;
            memset(&t, 0, sizeof t);
            p.type = b, p.kv = c;
            t.n_seqs = d, t.max_len = e, t.heads = f;
            t.score_out = g ? (float *)&a : NULL;
            ornk_kv_attend(&p, &t, NULL);
        } else {
            ornk_evict_args t;
            memset(&t, 0, sizeof t);
            p.type = b, p.kv = c;
            t.n_seqs = d, t.max_len = e, t.keep = f, t.in_place = g;
            ornk_kv_evict(&p, &t, NULL);
        }
        printf("\n");
    }
    return 0;
}
