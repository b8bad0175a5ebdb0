// A CUDA runtime that launches nothing: the host side of the leaky scan linked
// against it shows what a call makes of a launch that is refused.  fake_fail(n)
// refuses the n-th launch from then on (-1: none), as the runtime does: the
// status is returned and kept for cudaGetLastError.
#include "common.h"

static int g_launches, g_fail = -1;
static cudaError_t g_last = cudaSuccess;
static cudaError_t launched() {
    if (g_launches++ != g_fail) return cudaSuccess;
    return g_last = cudaErrorInvalidConfiguration;
}

extern "C" {
void** __cudaRegisterFatBinary(void*) {
    static void* handle;
    return &handle;
}
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, uint3*, uint3*, dim3*, dim3*, int*) {}

static dim3 g_grid, g_block;
unsigned __cudaPushCallConfiguration(dim3 grid, dim3 block, size_t, void*) {
    g_grid = grid;
    g_block = block;
    return 0;
}
cudaError_t __cudaPopCallConfiguration(dim3* grid, dim3* block, size_t* smem, void* stream) {
    *grid = g_grid;
    *block = g_block;
    *smem = 0;
    *(void**)stream = nullptr;
    return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void*, dim3, dim3, void**, size_t, cudaStream_t) { return launched(); }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t*, const void*, void**) { return launched(); }
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaGetDevice(int* d) {
    *d = 0;
    return cudaSuccess;
}
cudaError_t cudaMemsetAsync(void*, int, size_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaMemset2DAsync(void*, size_t, int, size_t, size_t, cudaStream_t) { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "refused"; }
cudaError_t cudaGetLastError() {
    const cudaError_t e = g_last;
    g_last = cudaSuccess;
    return e;
}

void fake_fail(int n) {
    g_launches = 0;
    g_fail = n;
    g_last = cudaSuccess;
}
int fake_launches() { return g_launches; }

// a scan of dense contiguous rows, and its gradient: an SNN_* code
int fake_scan(int type, int flags, int64_t b, int64_t t, int64_t d, int grad) {
    snn_scan s = {type, flags, b, t, d, nullptr};
    snn_rows r[5];
    for (int i = 0; i < 5; ++i) r[i] = {(void*)(uintptr_t)((i + 1) << 20), t * d, d};
    float *saved = (float*)(uintptr_t)(8 << 20), *h = (float*)(uintptr_t)(9 << 20);
    void* work = (void*)(uintptr_t)(10 << 20);
    try {
        if (grad)
            snnb::leaky_scan_grad(&s, &r[0], &r[1], saved, &r[2], h, &r[3], flags & SNN_SCAN_RASTER ? nullptr : &r[4], h,
                                  work, 1ll << 40, nullptr);
        else
            snnb::leaky_scan(&s, &r[0], &r[1], h, &r[2], h, saved, work, 1ll << 40, nullptr);
    } catch (const snnb::Error& e) {
        return e.code;
    }
    return SNN_OK;
}
}
