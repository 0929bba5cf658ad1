// A stand-in for the CUDA runtime calls of a launch, loaded ahead of the runtime by tests/test_first_calls_host.py: attributes take their time and may fail a number of times
// (FAIL_ATTRIBUTES), and a launch that asks for more shared memory than its kernel has been allowed so far fails, as on a device.  No GPU is touched.
#include <atomic>
#include <chrono>
#include <cstdlib>
#include <map>
#include <mutex>
#include <thread>
#include <cuda.h>
#include <cuda_runtime_api.h>

static std::mutex mu;
static std::map<const void*, int> allowed;
static std::atomic<int> fails{getenv("FAIL_ATTRIBUTES") ? atoi(getenv("FAIL_ATTRIBUTES")) : 0};

static CUresult encode(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                       CUtensorMapL2promotion, CUtensorMapFloatOOBfill) { return CUDA_SUCCESS; }

extern "C" {
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) { *v = 148; return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaThreadExchangeStreamCaptureMode(cudaStreamCaptureMode*) { return cudaSuccess; }
cudaError_t cudaHostRegister(void*, size_t, unsigned) { return cudaSuccess; }
cudaError_t cudaHostGetDevicePointer(void** d, void* h, unsigned) { *d = h; return cudaSuccess; }
cudaError_t cudaGetDriverEntryPoint(const char*, void** fn, unsigned long long, cudaDriverEntryPointQueryResult* r) {
    std::this_thread::sleep_for(std::chrono::milliseconds(20));
    *fn = (void*)encode;
    if (r) *r = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
cudaError_t cudaFuncSetAttribute(const void* f, cudaFuncAttribute a, int v) {
    std::this_thread::sleep_for(std::chrono::milliseconds(20));
    if (fails.fetch_sub(1) > 0) return cudaErrorMemoryAllocation;
    std::lock_guard<std::mutex> lk(mu);
    if (a == cudaFuncAttributeMaxDynamicSharedMemorySize) allowed[f] = v;
    return cudaSuccess;
}
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* f, void**) {
    std::lock_guard<std::mutex> lk(mu);
    const auto it = allowed.find(f);
    return (int)c->dynamicSmemBytes <= (it == allowed.end() ? 48 * 1024 : it->second) ? cudaSuccess : cudaErrorInvalidValue;
}
}
