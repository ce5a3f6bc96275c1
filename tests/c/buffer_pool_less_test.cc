// A buffer of more than is needed where there is memory for it, and of what is needed where there is not (csrc/buffer_pool.cuh), against a
// fake of the CUDA calls that the pool makes.
#include "../../cwick_b200/csrc/buffer_pool.cuh"

#include <cstdio>
#include <cstdlib>

constexpr size_t MB = 1u << 20;
static size_t memory = 100 * MB;
static int mallocs, cleared;
static cudaError_t other = cudaSuccess;

extern "C" {
cudaError_t cudaMalloc(void **p, size_t n) {
    mallocs++;
    if (other != cudaSuccess) return other;
    if (n > memory) return cudaErrorMemoryAllocation;
    *p = malloc(1);
    return cudaSuccess;
}
cudaError_t cudaFree(void *p) { free(p); return cudaSuccess; }
cudaError_t cudaGetLastError(void) { cleared++; return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus *st) { *st = cudaStreamCaptureStatusNone; return cudaSuccess; }
}

#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

int main() {
    CwkBufferPool pool;
    void *p = nullptr;
    size_t n = 0;
    CHECK(pool.alloc(0, 80 * MB, 40 * MB, &p, &n) == cudaSuccess && n == 80 * MB && mallocs == 1);
    pool.free(0, p, n, false);
    CHECK(pool.alloc(0, 180 * MB, 90 * MB, &p, &n) == cudaSuccess && n == 90 * MB && mallocs == 3 && cleared == 1);
    pool.free(0, p, n, false);
    p = nullptr; n = 0; mallocs = 0;
    CHECK(pool.alloc(0, 240 * MB, 120 * MB, &p, &n) == cudaErrorMemoryAllocation && p == nullptr && n == 0 && mallocs == 2);
    CHECK(pool.alloc(0, 120 * MB, 120 * MB, &p, &n) == cudaErrorMemoryAllocation && mallocs == 3);
    other = cudaErrorUnknown;                              // no lack of memory: not tried again
    CHECK(pool.alloc(0, 80 * MB, 40 * MB, &p, &n) == cudaErrorUnknown && p == nullptr && mallocs == 4);
    printf("ok\n");
    return 0;
}
