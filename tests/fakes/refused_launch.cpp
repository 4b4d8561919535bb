// A CUDA runtime that refuses one kernel launch, and the parts of libhexcuda's
// runtime that the paged-cache launchers call: linked with their objects, it shows
// on the CPU what an entry does once a launch of its own was refused.
#include <cuda.h>
#include <stdarg.h>
#include <stdio.h>

#include "hx_internal.h"

static int g_launches, g_refuse;
static cudaError_t g_error = cudaSuccess;

static cudaError_t launch() {
    if (++g_launches != g_refuse) return cudaSuccess;
    return g_error = cudaErrorLaunchOutOfResources;
}
static CUresult encode(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                       const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                       CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                       CUtensorMapFloatOOBfill) {
    return CUDA_SUCCESS;
}

extern "C" {
cudaError_t cudaLaunchKernel(const void *, dim3, dim3, void **, size_t, cudaStream_t) { return launch(); }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t *, const void *, void **) { return launch(); }
cudaError_t cudaGetLastError() {
    const cudaError_t e = g_error;
    g_error = cudaSuccess;
    return e;
}
cudaError_t cudaFuncSetAttribute(const void *, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaFuncGetAttributes(cudaFuncAttributes *a, const void *) {
    *a = cudaFuncAttributes();
    a->numRegs = 168;
    return cudaSuccess;
}
cudaError_t cudaOccupancyMaxActiveBlocksPerMultiprocessorWithFlags(int *n, const void *, int, size_t,
                                                                   unsigned) {
    *n = 8;
    return cudaSuccess;
}
cudaError_t cudaOccupancyMaxActiveBlocksPerMultiprocessor(int *n, const void *, int, size_t) {
    *n = 8;
    return cudaSuccess;
}
cudaError_t cudaGetDriverEntryPoint(const char *, void **p, unsigned long long,
                                    cudaDriverEntryPointQueryResult *r) {
    *p = reinterpret_cast<void *>(encode);
    *r = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
void **__cudaRegisterFatBinary(void *) {
    static void *handle;
    return &handle;
}
void __cudaRegisterFatBinaryEnd(void **) {}
void __cudaUnregisterFatBinary(void **) {}
void __cudaRegisterFunction(void **, const char *, char *, const char *, int, uint3 *, uint3 *, dim3 *,
                            dim3 *, int *) {}
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, cudaStream_t) { return 0; }
cudaError_t __cudaPopCallConfiguration(dim3 *, dim3 *, size_t *, void *) { return cudaSuccess; }

HX_EXPORT void refuse(int nth) {
    g_refuse = nth;
    g_launches = 0;
    g_error = cudaSuccess;
}
HX_EXPORT int launches() { return g_launches; }
}

namespace hx {
static Dev g_dev;
Dev *get_dev(int) {
    g_dev.ordinal = 0;
    g_dev.sms = 148;
    return &g_dev;
}
int fail(int code, const char *, ...) { return code; }
int check(cudaError_t e, const char *) { return e == cudaSuccess ? HEXCUDA_OK : HEXCUDA_ERR_CUDA; }
void launch_begin(Dev *) {}
int launch_end(Dev *, const char *, int) { return check(cudaGetLastError(), ""); }
void note_mech(unsigned) {}
}  // namespace hx
