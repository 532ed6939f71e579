/* The paged cache's workspace (csrc/host/kv.c) as it grows: prints w for a wait for
 * the stream, f for a free and m for an allocation, in order, a line for each of the
 * sizes given. */
#include "../ornith-flight_amd/csrc/host/kv.c"

#include <stdlib.h>

hipError_t hipStreamSynchronize(hipStream_t s) { return putchar('w'), hipSuccess; }
hipError_t hipFree(void *p) { return putchar('f'), free(p), hipSuccess; }
hipError_t hipMalloc(void **p, size_t n) { return putchar('m'), *p = malloc(n), hipSuccess; }

int main(int argc, char **argv)
{
    static gpu_context ctx;
    for (int i = 1; i < argc; ++i) {
        const size_t n = strtoul(argv[i], NULL, 10);
        char *p = orn_kv_ws_get(&ctx, n);
        if (n) p[0] = p[n - 1] = 1;
        putchar('\n');
    }
    return 0;
}
