/* A HIP runtime of host memory for tests of the library's host code without a GPU: allocations come from malloc up to a
 * budget, copies happen at once, kernels do nothing, and a flag says that every stream is being captured. */
#include <stdlib.h>
#include <string.h>

long long hh_live, hh_budget = 1LL << 62, hh_mallocs, hh_syncs, hh_launches;
int hh_capturing;
static int last; /* a failed call's error stays until it is asked for */

struct block { void *p; size_t n; struct block *next; };
static struct block *blocks;
static long long scratch[1 << 20];

int hipMalloc(void **out, size_t n) {
    *out = NULL;
    if (hh_live + (long long)n > hh_budget) return last = 2; /* out of memory */
    struct block *b = malloc(sizeof *b);
    b->p = calloc(1, n ? n : 1);
    b->n = n;
    b->next = blocks;
    blocks = b;
    hh_live += n;
    ++hh_mallocs;
    *out = b->p;
    return 0;
}
int hipFree(void *p) {
    for (struct block **at = &blocks; *at; at = &(*at)->next)
        if ((*at)->p == p) {
            struct block *b = *at;
            *at = b->next;
            hh_live -= b->n;
            free(b->p);
            free(b);
            return 0;
        }
    return p ? 1 : 0;
}
int hipMemset(void *p, int v, size_t n) { memset(p, v, n); return 0; }
int hipMemcpy(void *to, const void *from, size_t n, int kind) { memcpy(to, from, n); return 0; }
int hipMemcpyAsync(void *to, const void *from, size_t n, int kind, void *stream) { memcpy(to, from, n); return 0; }
int hipDeviceSynchronize(void) { ++hh_syncs; return 0; }
int hipGetDevice(int *d) { *d = 0; return 0; }
int hipSetDevice(int d) { return d != 0; }
int hipGetLastError(void) { int e = last; last = 0; return e; }
const char *hipGetErrorString(int e) { return e == 2 ? "out of memory" : "error"; }
int hipGetSymbolAddress(void **out, const void *symbol) { *out = scratch; return 0; }
int hipStreamCreateWithFlags(void **s, unsigned flags) { *s = &hh_capturing; return 0; }
int hipStreamDestroy(void *s) { return 0; }
int hipStreamSynchronize(void *s) { return 0; }
int hipStreamIsCapturing(void *s, int *status) { *status = hh_capturing; return 0; }
int hipLaunchKernel(const void *f, ...) { ++hh_launches; return 0; }
int hipFuncSetAttribute(const void *f, int a, int v) { return 0; }
/* (the grid and block of a launch are passed and taken back in registers or on the stack by value: nothing is kept) */
int __hipPushCallConfiguration() { return 0; }
int __hipPopCallConfiguration(void *grid, void *block, size_t *shared, void **stream) { memset(grid, 0, 12); memset(block, 0, 12); *shared = 0; *stream = NULL; return 0; }
void **__hipRegisterFatBinary(const void *data) { static void *h; return &h; }
void __hipRegisterFunction() {}
void __hipRegisterVar() {}
void __hipUnregisterFatBinary(void **h) {}
