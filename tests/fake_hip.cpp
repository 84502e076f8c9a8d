// A stand-in for the HIP runtime, for tests of the library's host side without a GPU: loaded with RTLD_GLOBAL before
// libaesir_hip.so it answers its HIP calls. Device memory is host memory; of the kernels only those that bring tables to the
// device and copy pages do anything. Launches and host allocations can be made to fail from the test.
#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <map>
#include <new>
#include <string>

static long g_fail_launch = 0, g_fail_new = 0;  // count down to the one that fails; 0: none
static long g_launches = 0, g_news = 0;
static int g_capturing = 0;
static hipError_t g_last = hipSuccess;
static int32_t *g_table = nullptr;

static std::map<const void *, std::string> &names() {
    static auto *m = new std::map<const void *, std::string>();
    return *m;
}

void *operator new(size_t n) {
    g_news++;
    if (g_fail_new > 0 && --g_fail_new == 0) throw std::bad_alloc();
    if (void *p = std::malloc(n ? n : 1)) return p;
    throw std::bad_alloc();
}
void operator delete(void *p) noexcept { std::free(p); }
void operator delete(void *p, size_t) noexcept { std::free(p); }

struct Upload {  // the arguments of kv4_upload_kernel
    const uint32_t *src;
    uint32_t *dst;
    int32_t words, fill;
    int32_t *table;
    int32_t updates;
};

struct Move {
    int32_t src, dst;
};

extern "C" {

void fake_fail_launch(long n) { g_fail_launch = n; }
void fake_fail_new(long n) { g_fail_new = n; }
long fake_launches() { return g_launches; }
long fake_news() { return g_news; }
void fake_capturing(int on) { g_capturing = on; }
int32_t *fake_table() { return g_table; }

void **__hipRegisterFatBinary(const void *) { return (void **)calloc(1, sizeof(void *)); }
void __hipUnregisterFatBinary(void **) {}
void __hipRegisterFunction(void **, const void *host, char *, const char *name, unsigned, void *, void *, void *, void *, int *) { names()[host] = name; }
void __hipRegisterVar(void **, void *, char *, char *, int, size_t, int, int) {}

static struct {
    dim3 grid, block;
    size_t shared;
    hipStream_t stream;
} g_config;

hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t shared, hipStream_t stream) {
    g_config = {grid, block, shared, stream};
    return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *shared, hipStream_t *stream) {
    *grid = g_config.grid;
    *block = g_config.block;
    *shared = g_config.shared;
    *stream = g_config.stream;
    return hipSuccess;
}

hipError_t hipLaunchKernel(const void *f, dim3, dim3, void **args, size_t, hipStream_t) {
    g_launches++;
    if (g_fail_launch > 0 && --g_fail_launch == 0) return g_last = hipErrorLaunchFailure;
    const std::string &name = names()[f];
    if (name.find("kv4_upload_kernel") != std::string::npos) {
        const Upload &u = *(const Upload *)args[0];
        if (u.words) std::memcpy(u.dst, u.src, 4 * (size_t)u.words);
        for (int32_t i = 0; i < u.fill; i++) u.dst[u.words + i] = 0x7FFFFFFF;
        for (int32_t i = 0; i < u.updates; i++) u.table[u.src[u.words + 2 * i]] = (int32_t)u.src[u.words + 2 * i + 1];
        g_table = u.table;
    } else if (name.find("kv4_copy_kernel") != std::string::npos) {
        char *pool = *(char **)args[0];
        const int64_t bytes = *(int64_t *)args[1];
        const Move *m = *(const Move **)args[2];
        for (int i = 0; i < *(int *)args[3]; i++) std::memcpy(pool + m[i].dst * bytes, pool + m[i].src * bytes, (size_t)bytes);
    }
    return hipSuccess;
}

hipError_t hipGetLastError() {
    const hipError_t e = g_last;
    g_last = hipSuccess;
    return e;
}
const char *hipGetErrorString(hipError_t) { return "made to fail"; }
hipError_t hipGetDeviceCount(int *n) { return *n = 1, hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600 *p, int) {
    std::memset(p, 0, sizeof *p);
    p->multiProcessorCount = 256;
    std::strcpy(p->gcnArchName, "none");
    return hipSuccess;
}
#undef hipMalloc
#undef hipHostMalloc
hipError_t hipMalloc(void **p, size_t n) { return (*p = std::aligned_alloc(4096, (n + 4095) / 4096 * 4096)) ? hipSuccess : hipErrorOutOfMemory; }
hipError_t hipFree(void *p) { return std::free(p), hipSuccess; }
hipError_t hipHostMalloc(void **p, size_t n, unsigned) { return hipMalloc(p, n); }
hipError_t hipHostFree(void *p) { return hipFree(p); }
hipError_t hipMemsetAsync(void *p, int x, size_t n, hipStream_t) { return std::memset(p, x, n), hipSuccess; }
hipError_t hipMemcpyAsync(void *d, const void *s, size_t n, hipMemcpyKind, hipStream_t) { return std::memcpy(d, s, n), hipSuccess; }
hipError_t hipStreamCreateWithFlags(hipStream_t *s, unsigned) { return *s = (hipStream_t)std::malloc(1), hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t s) { return std::free(s), hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s) {
    *s = g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
    return hipSuccess;
}
hipError_t hipEventCreate(hipEvent_t *e) { return *e = (hipEvent_t)std::malloc(1), hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t e) { return std::free(e), hipSuccess; }

}  // extern "C"
