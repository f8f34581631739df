/* Stands in for the HIP runtime's calls that launch kernels: writes down what would be launched, and launches nothing.
 * Loaded (RTLD_GLOBAL) ahead of a library under test in a process of its own; needs no GPU.  Output, a line each:
 *   launch KERNEL gx gy gz bx by bz DYNAMIC_LDS
 *   raise KERNEL BYTES          (hipFuncAttributeMaxDynamicSharedMemorySize) */
#include <stddef.h>
#include <stdio.h>

typedef struct {
  unsigned x, y, z;
} dim3;

enum { kMax = 4096 };
static const void* host[kMax];
static const char* names[kMax];
static int known;

static const char* name_of(const void* f) {
  for (int i = 0; i < known; ++i)
    if (host[i] == f) return names[i];
  return "?";
}

void __hipRegisterFunction(void** modules, const void* function, char* device_function, const char* device_name, unsigned limit,
                           void* tid, void* bid, dim3* block, dim3* grid, int* wsize) {
  (void)modules, (void)device_function, (void)limit, (void)tid, (void)bid, (void)block, (void)grid, (void)wsize;
  if (known < kMax) {
    host[known] = function;
    names[known++] = device_name;
  }
}

static dim3 next_grid, next_block;
static size_t next_shared;
static void* next_stream;

int __hipPushCallConfiguration(dim3 grid, dim3 block, size_t shared, void* stream) {
  next_grid = grid, next_block = block, next_shared = shared, next_stream = stream;
  return 0;
}

int __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* shared, void** stream) {
  *grid = next_grid, *block = next_block, *shared = next_shared, *stream = next_stream;
  return 0;
}

int hipLaunchKernel(const void* function, dim3 grid, dim3 block, void** args, size_t shared, void* stream) {
  (void)args, (void)stream;
  printf("launch %s %u %u %u %u %u %u %zu\n", name_of(function), grid.x, grid.y, grid.z, block.x, block.y, block.z, shared);
  fflush(stdout);
  return 0;
}

int hipFuncSetAttribute(const void* function, int attribute, int value) {
  (void)attribute;
  printf("raise %s %d\n", name_of(function), value);
  fflush(stdout);
  return 0;
}

int hipGetDevice(int* device) {
  *device = 0;
  return 0;
}

int hipGetLastError(void) { return 0; }
