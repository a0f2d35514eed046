/* launch_hook.c -- stands in for the runtime's launch in a process without a card: loaded before the library, it notes each
 * launch's grid, workgroup and first argument's first words, and refuses what the runtime refuses: a dimension of 2^32 work
 * items or more, or of nothing. No kernel runs. */
#include <stddef.h>
#include <stdint.h>
#include <string.h>

typedef struct {
    uint32_t x, y, z;
} Dim;

enum { kMost = 4096, kWords = 24 };
static struct {
    Dim grid, block;
    int64_t words[kWords];
} launches[kMost];
static int count, error;

/* a <<<>>> launch's configuration, handed from the call to the kernel's stub */
static Dim the_grid, the_block;
static size_t the_lds;
static void* the_stream;
int __hipPushCallConfiguration(Dim grid, Dim block, size_t lds, void* stream) {
    the_grid = grid, the_block = block, the_lds = lds, the_stream = stream;
    return 0;
}
int __hipPopCallConfiguration(Dim* grid, Dim* block, size_t* lds, void** stream) {
    *grid = the_grid, *block = the_block, *lds = the_lds, *stream = the_stream;
    return 0;
}

int hipLaunchKernel(const void* kernel, Dim grid, Dim block, void** args, size_t lds, void* stream) {
    (void)kernel, (void)lds, (void)stream;
    if (count < kMost) {
        launches[count].grid = grid;
        launches[count].block = block;
        memcpy(launches[count].words, args[0], sizeof launches[count].words);
    }
    ++count;
    const uint64_t x = (uint64_t)grid.x * block.x, y = (uint64_t)grid.y * block.y, z = (uint64_t)grid.z * block.z;
    if (!x || !y || !z || x >> 32 || y >> 32 || z >> 32 || grid.y > 65535 || grid.z > 65535 || (uint64_t)block.x * block.y * block.z > 1024)
        return error = 9; /* hipErrorInvalidConfiguration */
    return 0;
}
int hipGetLastError(void) {
    const int e = error;
    error = 0;
    return e;
}
void hook_clear(void) { count = error = 0; }
int hook_count(void) { return count; }
/* grid x y z, workgroup x y z, then the first argument's words */
void hook_launch(int i, int64_t* out) {
    const Dim* d = &launches[i].grid;
    out[0] = d->x, out[1] = d->y, out[2] = d->z;
    d = &launches[i].block;
    out[3] = d->x, out[4] = d->y, out[5] = d->z;
    memcpy(out + 6, launches[i].words, sizeof launches[i].words);
}
