/* Stands in for the HIP runtime where only the host side of an entry runs: a
 * launch is noted and counts as accepted. */
#include <stddef.h>

typedef struct { unsigned x, y, z; } dim3_;

static dim3_ grid_of, block_of;
static size_t shared_of;

int stub_launches;
double stub_most_threads; /* of a grid's dimension */
size_t stub_most_shared;

void **__hipRegisterFatBinary(const void *data) { (void)data; return NULL; }
void __hipUnregisterFatBinary(void **m) { (void)m; }
void __hipRegisterFunction(void **m, const void *f, char *d, const char *n, unsigned l, void *t,
                           void *b, void *bd, void *gd, int *w) {
    (void)m, (void)f, (void)d, (void)n, (void)l, (void)t, (void)b, (void)bd, (void)gd, (void)w;
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
    (void)f, (void)args, (void)stream;
    ++stub_launches;
    const double across[] = {(double)grid.x * block.x, (double)grid.y * block.y,
                             (double)grid.z * block.z};
    for (int i = 0; i < 3; ++i)
        if (across[i] > stub_most_threads) stub_most_threads = across[i];
    if (shared > stub_most_shared) stub_most_shared = shared;
    return grid.x && grid.y && grid.z && block.x ? 0 : 9;
}
int hipGetLastError(void) { return 0; }
