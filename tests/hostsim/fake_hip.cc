// TEST INFRASTRUCTURE: the few calls of the HIP runtime that the host side of psgpu_proj.hip makes, on a machine with two devices and
// no kernels: memory is the host's, launches do nothing, and every call is written down with the thread that made it.
// tests/test_net_host.py holds the order of the calls against what the header promises.  Not a product path.
#include <hip/hip_runtime_api.h>
#include <cstdarg>
#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>
#include <string>
#include <unistd.h>

static std::mutex g_mutex;
static std::string g_log;
static std::map<uintptr_t, std::pair<size_t, int>> g_memory;            // address -> bytes, device
static thread_local int t_device = 0, t_name = 0;

static void note(const char *what, int arg)
{
    {
        std::lock_guard<std::mutex> lock(g_mutex);
        g_log += std::to_string(t_name) + " " + what + " " + std::to_string(arg) + "\n";
    }
    usleep(300);                                                        // (another thread's turn)
}
static int device_of(const void *p)
{
    std::lock_guard<std::mutex> lock(g_mutex);
    auto it = g_memory.upper_bound((uintptr_t)p);
    if (it == g_memory.begin()) return -1;
    --it;
    return (uintptr_t)p < it->first + it->second.first ? it->second.second : -1;
}

extern "C" {
void fake_name(int name) { t_name = name; }
void fake_place(void *p, size_t n, int device) { std::lock_guard<std::mutex> lock(g_mutex); g_memory[(uintptr_t)p] = {n, device}; }
size_t fake_log(char *to, size_t room)
{
    std::lock_guard<std::mutex> lock(g_mutex);
    const size_t n = g_log.size() < room ? g_log.size() : room;
    memcpy(to, g_log.data(), n);
    g_log.clear();
    return n;
}

hipError_t hipGetDevice(int *d) { *d = t_device; return hipSuccess; }
hipError_t hipSetDevice(int d) { t_device = d; return hipSuccess; }
hipError_t hipDeviceSynchronize() { note("sync", t_device); return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
const char *hipGetErrorString(hipError_t) { return "error"; }
hipError_t hipMalloc(void **p, size_t n) { *p = calloc(n ? n : 1, 1); fake_place(*p, n ? n : 1, t_device); return hipSuccess; }
hipError_t hipFree(void *p)
{
    if (p) { std::lock_guard<std::mutex> lock(g_mutex); g_memory.erase((uintptr_t)p); }
    free(p);
    return hipSuccess;
}
hipError_t hipMemcpy(void *to, const void *from, size_t n, hipMemcpyKind) { note("copy", device_of(from)); memcpy(to, from, n); return hipSuccess; }
hipError_t hipMemset(void *p, int v, size_t n) { memset(p, v, n); return hipSuccess; }
hipError_t hipPointerGetAttributes(hipPointerAttribute_t *at, const void *p)
{
    const int d = device_of(p);
    if (d < 0) return hipErrorInvalidValue;
    memset(at, 0, sizeof *at);
    at->type = hipMemoryTypeDevice;
    at->device = d;
    return hipSuccess;
}
hipError_t hipLaunchKernel(const void *, dim3, dim3, void **, size_t, hipStream_t) { note("launch", t_device); return hipSuccess; }
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3 *, dim3 *, size_t *, hipStream_t *) { return hipSuccess; }
void **__hipRegisterFatBinary(const void *) { static void *none; return &none; }
void __hipRegisterFunction(void **, const void *, char *, const char *, int, void *, void *, void *, void *, int *) {}
void __hipUnregisterFatBinary(void **) {}
char __hip_fatbin[16];
int32_t psgpu_get_device() { return t_device; }
}

void psgpu_set_error(const char *, ...) {}
void psgpu_clear_error() {}
int net_check_device(int *d) { if (d) *d = t_device; return 0; }
