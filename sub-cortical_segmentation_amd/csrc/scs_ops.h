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

// ---- four consecutive elements of a type, held as loaded
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
template <class T> struct Vec4;
template <> struct Vec4<float> { typedef f32x4 raw; };
template <> struct Vec4<__bf16> { typedef u32x2 raw; };
template <> struct Vec4<_Float16> { typedef u32x2 raw; };
// four consecutive elements at any element alignment (the global loads of gfx950 need none)
template <class R> struct __attribute__((packed, aligned(2))) Loose { R v; };

template <class T> __device__ __forceinline__ void raw_load(typename Vec4<T>::raw& r, const T* p, int left) {
    if (left >= 4) r = reinterpret_cast<const Loose<typename Vec4<T>::raw>*>(p)->v;
    else {
        T e[4] = {};
        for (int i = 0; i < 3; ++i) if (i < left) e[i] = p[i];
        __builtin_memcpy(&r, e, sizeof(r));
    }
}
template <class T> __device__ __forceinline__ void raw_store(const typename Vec4<T>::raw& r, T* p, int left) {
    if (left >= 4) reinterpret_cast<Loose<typename Vec4<T>::raw>*>(p)->v = r;
    else {
        T e[4];
        __builtin_memcpy(e, &r, sizeof(r));
        for (int i = 0; i < 3; ++i) if (i < left) p[i] = e[i];
    }
}
template <class T> __device__ __forceinline__ void unpack(const typename Vec4<T>::raw& r, float (&f)[4]) {
    T e[4];
    __builtin_memcpy(e, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = to_f32(e[i]);
}
template <class T> __device__ __forceinline__ typename Vec4<T>::raw pack(const float (&f)[4]) {
    T e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = from_f32<T>(f[i]);           // to the nearest, ties to even
    typename Vec4<T>::raw r;
    __builtin_memcpy(&r, e, sizeof(r));
    return r;
}

// ---- vectors of elements at any element alignment
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
template <class T> __device__ __forceinline__ typename Vec4<T>::raw at4(const T* p) { return reinterpret_cast<const Loose<typename Vec4<T>::raw>*>(p)->v; }
template <class T> __device__ __forceinline__ u32x4 at16(const T* p) { return reinterpret_cast<const Loose<u32x4>*>(p)->v; }
// 16 bytes of elements at any element alignment, zeros behind `left`
template <class T> __device__ __forceinline__ u32x4 load16(const T* p, int64_t left) {
    constexpr int N = 16 / sizeof(T);
    if (left >= N) return at16(p);
    T e[N] = {};
    for (int i = 0; i < N - 1; ++i) if (i < left) e[i] = p[i];
    u32x4 r;
    __builtin_memcpy(&r, e, 16);
    return r;
}

// ---- operands of the 16-bit matrix cores
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <class T> struct Frag;
template <> struct Frag<__bf16> { typedef __bf16 v8 __attribute__((ext_vector_type(8))); };
template <> struct Frag<_Float16> { typedef _Float16 v8 __attribute__((ext_vector_type(8))); };
__device__ __forceinline__ f32x4 mfma16(Frag<__bf16>::v8 a, Frag<__bf16>::v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma16(Frag<_Float16>::v8 a, Frag<_Float16>::v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

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
