// stub_hip.h -- a HIP runtime for CPU tests of the host library: csrc/fa_host.cpp is compiled into a
// test program together with these definitions and without the real runtime.  Nothing runs on a GPU;
// launches are recorded, and a yield after each gives other threads their chance to come between.
// Modules "load" from any existing file, and hold every function but those that stub::absent names.
#ifndef STUB_HIP_H
#define STUB_HIP_H

#include <hip/hip_runtime.h>

#include <cstdlib>
#include <cstring>
#include <mutex>
#include <string>
#include <thread>
#include <vector>

namespace stub {
struct Launch {
    int call;   // the caller's number of its call (stub::call)
    std::string name;
};
inline thread_local int call = 0;
inline std::mutex mu;
inline std::vector<Launch> launches;
inline std::string absent;             // functions whose names start with this are in no module
inline int yields = 1;
inline std::vector<std::string> loaded;
inline std::vector<size_t> allocations;
inline int synchronized = 0;           // streams, by hipStreamSynchronize
}  // namespace stub

extern "C" {
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipGetDeviceCount(int* n) { return *n = 1, hipSuccess; }
hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int) {
    std::memset(p, 0, sizeof(*p));
    p->multiProcessorCount = 256;
    return hipSuccess;
}
hipError_t hipMalloc(void** p, size_t n) {
    std::lock_guard<std::mutex> lock(stub::mu);
    stub::allocations.push_back(n);
    return *p = std::malloc(64), hipSuccess;   // an address of its own; the memory itself is not used
}
hipError_t hipFree(void* p) { return std::free(p), hipSuccess; }
hipError_t hipMallocAsync(void** p, size_t n, hipStream_t) { return hipMalloc(p, n); }
hipError_t hipFreeAsync(void* p, hipStream_t) { return hipFree(p); }
hipError_t hipHostMalloc(void** p, size_t n, unsigned) { return *p = std::malloc(n), hipSuccess; }
hipError_t hipHostFree(void* p) { return std::free(p), hipSuccess; }
hipError_t hipMemGetInfo(size_t* f, size_t* t) { return *f = *t = size_t(1) << 38, hipSuccess; }
hipError_t hipMemcpyAsync(void*, const void*, size_t, hipMemcpyKind, hipStream_t) { return hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { return *e = nullptr, hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { return *s = nullptr, hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) {
    std::lock_guard<std::mutex> lock(stub::mu);
    return ++stub::synchronized, hipSuccess;
}
hipError_t hipStreamGetCaptureInfo(hipStream_t, hipStreamCaptureStatus* st, unsigned long long* id) {
    return *st = hipStreamCaptureStatusNone, *id = 0, hipSuccess;
}
hipError_t hipThreadExchangeStreamCaptureMode(hipStreamCaptureMode*) { return hipSuccess; }
hipError_t hipModuleLoad(hipModule_t* m, const char* path) {
    std::lock_guard<std::mutex> lock(stub::mu);
    stub::loaded.push_back(path);
    *m = reinterpret_cast<hipModule_t>(stub::loaded.size());
    return hipSuccess;
}
hipError_t hipModuleUnload(hipModule_t) { return hipSuccess; }
hipError_t hipModuleGetFunction(hipFunction_t* f, hipModule_t, const char* name) {
    if (!stub::absent.empty() && std::strncmp(name, stub::absent.c_str(), stub::absent.size()) == 0)
        return hipErrorNotFound;
    *f = reinterpret_cast<hipFunction_t>(strdup(name));
    return hipSuccess;
}
hipError_t hipModuleLaunchKernel(hipFunction_t f, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned,
                                 hipStream_t, void**, void**) {
    {
        std::lock_guard<std::mutex> lock(stub::mu);
        stub::launches.push_back({stub::call, reinterpret_cast<const char*>(f)});
    }
    for (int i = 0; i < stub::yields; ++i) std::this_thread::yield();
    return hipSuccess;
}
}

static char stub_scratch[64];
int fa_scratch_init(int) { return 0; }
void* fa_scratch_ptr(int) { return stub_scratch; }

#endif
