/* In front of fake_cudart.c: what the token-by-token operators ask of a runtime besides, and where their words lie: the page-locked ones that a kernel sets when
 * it gives up (64 bytes), and the counters (serving_counters of them, set by the test before they are made). */
#define _GNU_SOURCE
#include <cuda_runtime_api.h>
#include <dlfcn.h>

size_t serving_counters;
int* gave_up_word;
unsigned* counter_words;

cudaError_t cudaHostAlloc(void** p, size_t n, unsigned f) {
    cudaError_t (*next)(void**, size_t, unsigned) = dlsym(RTLD_NEXT, "cudaHostAlloc");
    const cudaError_t e = next(p, n, f);
    if (!e && n == 64) gave_up_word = *p;
    return e;
}
cudaError_t cudaMalloc(void** p, size_t n) {
    cudaError_t (*next)(void**, size_t) = dlsym(RTLD_NEXT, "cudaMalloc");
    const cudaError_t e = next(p, n);
    if (!e && serving_counters && n == serving_counters) counter_words = *p;
    return e;
}
cudaError_t cudaStreamIsCapturing(cudaStream_t s, enum cudaStreamCaptureStatus* c) { (void)s; *c = cudaStreamCaptureStatusNone; return cudaSuccess; }
