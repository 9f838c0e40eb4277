// A step of AdamW over more tensors than one launch takes, of which a late one lies in host memory, on a HIP runtime made of the functions below: it
// has no device, counts launches by the kernels' names and refuses allocations beyond `most`.  Without memory for that tensor nothing is
// launched; with it everything is.  Ends with 1 and a line that says what did not hold.
#include <hip/hip_runtime.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <map>
#include <string>
#include <vector>

#include "ptl_api.h"

static char arena[4 << 20];  // what stands for device memory that the program has
static size_t most;          // bytes of the largest allocation that is granted
static std::map<const void *, std::string> &names() {  // (kernels are registered before this file's own variables are there)
    static std::map<const void *, std::string> m;
    return m;
}
static int steps, copies, others;

extern "C" {
void **__hipRegisterFatBinary(const void *) { return nullptr; }
void __hipUnregisterFatBinary(void **) {}
void __hipRegisterFunction(void **, const void *host, char *, const char *name, unsigned, void *, void *, void *, void *, int *) { names()[host] = name; }
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *lds, hipStream_t *stream) {
    *grid = *block = dim3(1);
    *lds = 0;
    *stream = nullptr;
    return hipSuccess;
}
hipError_t hipLaunchKernel(const void *f, dim3, dim3, void **, size_t, hipStream_t) {
    const std::string &n = names()[f];
    ++(n.find("adamw") != std::string::npos ? steps : n.find("stage_copy") != std::string::npos ? copies : others);
    return hipSuccess;
}
hipError_t hipMalloc(void **p, size_t n) {
    *p = n <= most ? malloc(n) : nullptr;
    return *p ? hipSuccess : hipErrorOutOfMemory;
}
hipError_t hipFree(void *p) {
    free(p);
    return hipSuccess;
}
hipError_t hipHostMalloc(void **p, size_t n, unsigned) { return hipMalloc(p, n); }
hipError_t hipHostFree(void *p) { return hipFree(p); }
hipError_t hipMemset(void *p, int v, size_t n) {
    memset(p, v, n);
    return hipSuccess;
}
hipError_t hipMemcpyAsync(void *to, const void *from, size_t n, hipMemcpyKind, hipStream_t) {
    memcpy(to, from, n);
    return hipSuccess;
}
hipError_t hipPointerGetAttributes(hipPointerAttribute_t *a, const void *p) {
    if (p < arena || p >= arena + sizeof(arena)) return hipErrorInvalidValue;
    a->type = hipMemoryTypeDevice;
    return hipSuccess;
}
hipError_t hipMemGetAddressRange(hipDeviceptr_t *base, size_t *n, hipDeviceptr_t) {
    *base = arena;
    *n = sizeof(arena);
    return hipSuccess;
}
hipError_t hipGetDevice(int *d) { return *d = 0, hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDeviceCount(int *n) { return *n = 1, hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600 *p, int) {
    memset(p, 0, sizeof(*p));
    p->multiProcessorCount = 256;
    return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
const char *hipGetErrorString(hipError_t e) { return e == hipErrorOutOfMemory ? "out of memory" : "error"; }
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s) { return *s = hipStreamCaptureStatusNone, hipSuccess; }
hipError_t hipEventCreate(hipEvent_t *e) { return *e = nullptr, hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t *e, unsigned) { return hipEventCreate(e); }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float *ms, hipEvent_t, hipEvent_t) { return *ms = 0, hipSuccess; }
}
namespace ptl {
int dw_noalloc_setup(int) { return 0; }  // (of the layers, which are not linked)
}

static bool expect(const char *what, int got, int want) {
    if (got != want) printf("%s: %d instead of %d\n", what, got, want);
    return got == want;
}

int main() {
    const int count = 70, n = 1000, late = 69, large = 9 << 20;  // (36 MB: a buffer of its own)
    std::vector<blob> w(count);
    std::vector<adamw_state> s(count);
    std::vector<adamw_args> list(count);
    std::vector<float> host(4 * (size_t)large, 1.f), small(count * 4 * (size_t)n, 1.f);
    adamw_step step = {0.9f, 0.999f, 1e-8f, 1, nullptr, nullptr};
    auto place = [&](int i, float *at, int dim) {
        w[i] = {};
        w[i].data = at;
        w[i].diff = at + dim;
        w[i].dim = dim;
        s[i] = {};
        s[i].m = at + 2 * (size_t)dim;
        s[i].v = at + 3 * (size_t)dim;
        list[i] = {&w[i], nullptr, &s[i], nullptr, 0.1f, 0.f};
    };
    bool ok = true;
    for (int i = 0; i < count; ++i) place(i, reinterpret_cast<float *>(arena) + 4 * (size_t)n * i, n);
    place(late, host.data(), large);
    most = 8 << 20;
    ok &= expect("status without memory", ptl_adamw_fp32_multi(list.data(), count, &step), 2);
    ok &= expect("launches without memory", steps, 0);
    for (float f : host) ok &= f == 1.f;
    most = (size_t)1 << 30;
    ok &= expect("status with memory", ptl_adamw_fp32_multi(list.data(), count, &step), 0);
    ok &= expect("launches with memory", steps, 3);
    // small tensors of the host: they are fetched together, 16 to a launch, and so are the results written back (the weights and both moments)
    steps = copies = 0;
    for (int i = 0; i < count; ++i) place(i, small.data() + 4 * (size_t)n * i, n);
    ok &= expect("status of host tensors", ptl_adamw_fp32_multi(list.data(), count, &step), 0);
    ok &= expect("launches of host tensors", steps, 3);
    ok &= expect("copies of host tensors", copies, (count * 4 + 15) / 16 + (count * 3 + 15) / 16);
    ok &= expect("other launches", others, 0);
    return ok ? 0 : 1;
}
