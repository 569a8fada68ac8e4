// Entry points that only enqueue: the arrays are device memory, the stream is
// an argument, workspaces are the caller's. Such a call reads and writes no
// state of the library runtime (no staging, no shared scratch, no
// synchronisation), so it can be captured into a graph and calls on several
// streams or devices do not meet.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "runtime.cuh"

namespace sn {

// One array argument: its address and the alignment its element type needs.
// A null pointer is an absent optional argument.
struct ArgPtr {
    const void* p;
    unsigned align;
};

// Makes the device that owns the arrays current for the scope of a call (its
// kernels launch there whatever device the calling thread had selected).
class CallerDevice {
  public:
    // SN_OK when every array present is memory of one sm_100 device (managed
    // memory goes with any), aligned to its elements.
    int enter(const char* what, std::initializer_list<ArgPtr> args) {
        for (const ArgPtr& a : args) SN_TRY(add(what, a));
        return select(what);
    }
    int add(const char* what, const ArgPtr& a);
    int select(const char* what);
    int num_sms() const { return sms_; }
    CallerDevice();
    CallerDevice(const CallerDevice&) = delete;
    CallerDevice& operator=(const CallerDevice&) = delete;
    ~CallerDevice() {
        if (restore_ >= 0) cudaSetDevice(restore_);
    }

  private:
    bool known(uintptr_t p) const {
        for (const Span& r : spans_)
            if (p - r.base < r.size) return true;
        return false;
    }

    // Allocations that arrays of this call were found in, the last few: lists of
    // hundreds of tensors lie in a handful of an allocator's blocks.
    struct Span {
        uintptr_t base = 0, size = 0;
    };
    Span spans_[16];
    unsigned next_ = 0, asked_ = 0;
    int device_, restore_ = -1, sms_ = 0;
    bool told_;  // the caller vouches for its arrays (sn_abi_arrays_on)
    // (that counts for one call: entry points construct this before they return for any reason)
};

// Bytes of one element of an SN_F32 / SN_BF16 / SN_F16 array, 0 for others.
inline unsigned dtype_size(int dtype) {
    return dtype == SN_F32 ? 4u : dtype == SN_BF16 || dtype == SN_F16 ? 2u : 0u;
}

}  // namespace sn
