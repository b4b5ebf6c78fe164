// What the operators around the index share on the host: the device check and the word that lost waits raise.
#include "operators_common.cuh"

namespace cpb {
namespace op {
namespace {

__device__ uint32_t g_operator_status;
std::mutex g_mutex;
uint32_t* g_status_ptr[kMaxDevices] = {};
std::atomic<bool> g_device_ok[kMaxDevices];

}  // namespace

int check_device() {
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        set_error("no CUDA device available: this library has no CPU path");
        return CPHNSW_B200_E_CUDA;
    }
    if (dev < 0 || dev >= kMaxDevices) {
        set_error("device ordinal %d not supported", dev);
        return CPHNSW_B200_E_UNSUPPORTED;
    }
    if (g_device_ok[dev].load(std::memory_order_acquire)) return 0;
    int major = 0;
    CPB_CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
    if (major != 10) {
        set_error("device %d is sm_%dx; this library is built for sm_100a only", dev, major);
        return CPHNSW_B200_E_CUDA;
    }
    g_device_ok[dev].store(true, std::memory_order_release);
    return 0;
}

int sm_count(int* out) {
    static std::atomic<int> known[kMaxDevices];
    int dev = 0;
    CPB_CUDA(cudaGetDevice(&dev));
    int v = known[dev % kMaxDevices].load(std::memory_order_relaxed);
    if (!v) {
        CPB_CUDA(cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev));
        known[dev % kMaxDevices].store(v, std::memory_order_relaxed);
    }
    *out = v;
    return 0;
}

// (the symbol in host code is only a stand-in: the address is asked for once per device, with that device current)
int status_word(uint32_t** out) {
    int dev = -1;
    CPB_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= kMaxDevices) {
        set_error("device ordinal %d not supported", dev);
        return CPHNSW_B200_E_UNSUPPORTED;
    }
    std::lock_guard<std::mutex> lock(g_mutex);
    if (!g_status_ptr[dev]) {
        void* p = nullptr;
        CPB_CUDA(cudaGetSymbolAddress(&p, g_operator_status));
        g_status_ptr[dev] = static_cast<uint32_t*>(p);
    }
    *out = g_status_ptr[dev];
    return 0;
}

}  // namespace op
}  // namespace cpb

extern "C" int cphnsw_b200_operator_status(void) {
    using namespace cpb;
    CPB_TRY(op::check_device());
    uint32_t* d = nullptr;
    CPB_TRY(op::status_word(&d));
    uint32_t v = 0;
    CPB_CUDA(cudaDeviceSynchronize());
    CPB_CUDA(cudaMemcpy(&v, d, sizeof v, cudaMemcpyDeviceToHost));
    if (v == kStatusOk) return 0;
    CPB_CUDA(cudaMemset(d, 0, sizeof v));
    set_error("an operator's kernel gave up a wait: results since the last check are not valid");
    return CPHNSW_B200_E_DEVICE_WAIT;
}
