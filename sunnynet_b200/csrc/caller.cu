// Checks and device selection of the enqueue-only entry points (caller.cuh).
#include "caller.cuh"

#include <cuda.h>

#include <atomic>

namespace sn {
namespace {

// cuMemGetAddressRange, through the runtime (no link against the driver).
typedef CUresult (*RangeFn)(CUdeviceptr*, size_t*, CUdeviceptr);
RangeFn range_fn() {
    static const RangeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuMemGetAddressRange", &p, cudaEnableDefault, &q) !=
                cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<RangeFn>(p);
    }();
    return fn;
}

constexpr int kMaxDevices = 64;
std::atomic<int> g_sms[kMaxDevices];  // 0: not asked yet

}  // namespace

int CallerDevice::add(const char* what, const ArgPtr& a) {
    if (!a.p) return SN_OK;
    if ((uintptr_t)a.p % a.align)
        return fail(SN_E_INVAL, "%s: an array is not aligned to its elements", what);
    if (known((uintptr_t)a.p)) return SN_OK;
    cudaPointerAttributes at;
    if (cudaPointerGetAttributes(&at, a.p) != cudaSuccess) {
        cudaGetLastError();
        return fail(SN_E_DEVICE, "%s: no CUDA device", what);
    }
    if (at.type == cudaMemoryTypeManaged) return SN_OK;
    if (at.type != cudaMemoryTypeDevice)
        return fail(SN_E_INVAL, "%s: every array must be device memory", what);
    if (device_ < 0) device_ = at.device;
    if (at.device != device_)
        return fail(SN_E_INVAL, "%s: arrays of devices %d and %d", what, device_, at.device);
    if (asked_++ < 8) return SN_OK;  // a few arrays: a range costs more than it saves
    CUdeviceptr base = 0;
    size_t size = 0;
    if (const RangeFn range = range_fn())
        if (range(&base, &size, (CUdeviceptr)a.p) == CUDA_SUCCESS)
            spans_[next_++ % 16] = {(uintptr_t)base, (uintptr_t)size};
    return SN_OK;
}

int CallerDevice::select(const char* what) {
    int now = 0;
    SN_TRY(cuda_check(cudaGetDevice(&now), what));
    if (device_ < 0) device_ = now;
    if (device_ >= kMaxDevices)
        return fail(SN_E_UNSUPPORTED, "%s: device ordinal %d", what, device_);
    if (device_ != now) {
        SN_TRY(cuda_check(cudaSetDevice(device_), what));
        restore_ = now;
    }
    sms_ = g_sms[device_].load(std::memory_order_relaxed);
    if (!sms_) {
        int major = 0, sms = 0;
        SN_TRY(cuda_check(
            cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device_), what));
        SN_TRY(cuda_check(
            cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device_), what));
        if (major < 10)
            return fail(SN_E_UNSUPPORTED, "%s: device %d is sm_%d0; this build targets sm_100a",
                        what, device_, major);
        g_sms[device_].store(sms, std::memory_order_relaxed);
        sms_ = sms;
    }
    return SN_OK;
}

}  // namespace sn
