// Shared by the operators that stand beside the net (scs_optim.hip, scs_lowrank.hip): element types, the device a call runs on, errors.
#pragma once
#include <exception>
#include <utility>

#include "scs_common.h"

namespace scs {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(__bf16 x) { return (float)x; }
template <class T> __device__ __forceinline__ T from_f32(float x);                            // to the nearest, ties to even
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ _Float16 from_f32<_Float16>(float x) { return (_Float16)x; }
template <> __device__ __forceinline__ __bf16 from_f32<__bf16>(float x) { return (__bf16)x; }

int handle_device(scs_handle h);          // (scs_api.hip)

// The handle's device is current inside a call and the caller's again behind it.
struct DeviceGuard {
    int before = -1, rc = SCS_OK;
    explicit DeviceGuard(int device) {
        hipError_t e = hipGetDevice(&before);
        if (e == hipSuccess && before != device) e = hipSetDevice(device);
        else if (e == hipSuccess) before = -1;
        if (e != hipSuccess) { set_error("selecting device %d failed: %s", device, hipGetErrorString(e)); rc = SCS_ERR_HIP; before = -1; }
    }
    ~DeviceGuard() { if (before >= 0) (void)hipSetDevice(before); }
    DeviceGuard(const DeviceGuard&) = delete;
};

// No C++ exception crosses the C boundary.
template <class F> int guarded(F&& f) {
    try { return f(); }
    catch (const std::exception& e) { set_error("%s", e.what()); return SCS_ERR_ARG; }
    catch (...) { set_error("unknown exception"); return SCS_ERR_ARG; }
}

}  // namespace scs
