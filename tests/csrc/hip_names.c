/* Stands in for the HIP runtime where only the host side of an entry runs, and
 * notes which kernels it launches: their names, in order, and their grids. */
#include <stddef.h>

typedef struct { unsigned x, y, z; } dim3_;

enum { MOST_KERNELS = 4096, MOST_LAUNCHES = 64 };
static struct { const void *function; const char *name; } kernels[MOST_KERNELS];
static int kernel_count;
static dim3_ grid_of, block_of;
static size_t shared_of;

int names_launches;
const char *names_of[MOST_LAUNCHES];
dim3_ names_grids[MOST_LAUNCHES], names_blocks[MOST_LAUNCHES];

void **__hipRegisterFatBinary(const void *data) { (void)data; return NULL; }
void __hipUnregisterFatBinary(void **m) { (void)m; }
void __hipRegisterFunction(void **m, const void *f, char *d, const char *n, unsigned l, void *t,
                           void *b, void *bd, void *gd, int *w) {
    (void)m, (void)d, (void)l, (void)t, (void)b, (void)bd, (void)gd, (void)w;
    if (kernel_count < MOST_KERNELS) {
        kernels[kernel_count].function = f;
        kernels[kernel_count++].name = n;
    }
}
void __hipRegisterVar(void **m, void *v, char *h, char *d, int e, size_t s, int c, int g) {
    (void)m, (void)v, (void)h, (void)d, (void)e, (void)s, (void)c, (void)g;
}

int __hipPushCallConfiguration(dim3_ grid, dim3_ block, size_t shared, void *stream) {
    (void)stream;
    grid_of = grid, block_of = block, shared_of = shared;
    return 0;
}
int __hipPopCallConfiguration(dim3_ *grid, dim3_ *block, size_t *shared, void **stream) {
    *grid = grid_of, *block = block_of, *shared = shared_of, *stream = NULL;
    return 0;
}
int hipLaunchKernel(const void *f, dim3_ grid, dim3_ block, void **args, size_t shared,
                    void *stream) {
    (void)args, (void)shared, (void)stream;
    const char *name = "";
    for (int i = 0; i < kernel_count; ++i)
        if (kernels[i].function == f) name = kernels[i].name;
    if (names_launches < MOST_LAUNCHES) {
        names_of[names_launches] = name;
        names_grids[names_launches] = grid;
        names_blocks[names_launches] = block;
    }
    ++names_launches;
    return 0;
}
int hipGetLastError(void) { return 0; }
