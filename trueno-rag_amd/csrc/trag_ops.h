// What the operators on a caller's device arrays share (trag_q8.hip, trag_matmul_q8.hip,
// trag_distill.hip): element types, 16 bytes of them at a time, and the checks of an entry point that
// has no handle to ask for its device.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>
#include <new>
#include <string>
#include "trag.h"
#include "trag_error.h"

namespace trag {

inline uint32_t dtype_bytes(uint32_t dtype) { return dtype == TRAG_F32 ? 4u : 2u; }
inline bool aligned_to(const void* p, uint32_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1u)) == 0; }

// ---- element types, W consecutive elements (16 bytes) at a time. A caller's rows may start at any element (odd
// widths, odd strides), so the wide accesses ask for element alignment only; the hardware serves unaligned 16-byte
// accesses, and an aligned row pays nothing for it. `round`: a result is rounded to f32 and then to the type.
struct F32 {
    typedef float elem;
    static constexpr int W = 4;
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
    static __device__ __forceinline__ float round(float v) { return v; }
};
struct F16 {
    typedef _Float16 elem;
    static constexpr int W = 8;
    typedef _Float16 vec __attribute__((ext_vector_type(8), aligned(2)));
    // (the value is hidden from the compiler, which would fold a product and its conversion into a mixed-precision
    // multiply with a single rounding)
    static __device__ __forceinline__ _Float16 round(float v) {
        asm("" : "+v"(v));
        return (_Float16)v;
    }
};
struct BF16 {
    typedef __bf16 elem;
    static constexpr int W = 8;
    typedef __bf16 vec __attribute__((ext_vector_type(8), aligned(2)));
    static __device__ __forceinline__ __bf16 round(float v) { return (__bf16)v; }
};
template <typename T>
__device__ __forceinline__ typename T::vec load_vec(const typename T::elem* p) { return *reinterpret_cast<const typename T::vec*>(p); }
template <typename T>
__device__ __forceinline__ void store_vec(typename T::elem* p, typename T::vec v) { *reinterpret_cast<typename T::vec*>(p) = v; }
template <typename T>
__device__ __forceinline__ typename T::vec fill_vec(float v) {
    typename T::vec r;
#pragma unroll
    for (int i = 0; i < T::W; ++i) r[i] = T::round(v);
    return r;
}

// ---- entry points without a handle. The device is the stream's; for the default stream it is the one the
// arrays live on. Arrays that are not device memory of that device are refused on the host: a kernel would fault.
struct OpDevice {
    int prev = -1;
    bool switched = false;
    trag_status status = TRAG_OK;
    int dev = -1;

    OpDevice(const char* who, void* hip_stream, std::initializer_list<const void*> arrays) {
        int count = 0;
        if (hipGetDeviceCount(&count) != hipSuccess || count == 0) {
            (void)hipGetLastError();
            status = set_error(TRAG_DEVICE_ERROR, std::string(who) + ": no HIP device available (this library has no CPU path)");
            return;
        }
        if (hip_stream) {
            hipDevice_t d = -1;
            if (hipStreamGetDevice((hipStream_t)hip_stream, &d) == hipSuccess) dev = (int)d;
            else (void)hipGetLastError();
        }
        for (const void* p : arrays) {
            if (!p) continue;
            hipPointerAttribute_t at{};
            const hipError_t e = hipPointerGetAttributes(&at, p);
            if (e != hipSuccess) (void)hipGetLastError();
            if (e != hipSuccess || (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged && at.type != hipMemoryTypeHost)) {
                status = set_error(TRAG_INVALID_ARG, std::string(who) + ": an array is not device memory");
                return;
            }
            if (at.type != hipMemoryTypeDevice) continue;
            if (dev < 0) dev = at.device;
            if (at.device != dev) {
                status = set_error(TRAG_INVALID_ARG, std::string(who) + ": an array lives on device " + std::to_string(at.device) +
                                                     ", the call runs on device " + std::to_string(dev));
                return;
            }
        }
        if (dev >= 0 && hipGetDevice(&prev) == hipSuccess && prev != dev) switched = hipSetDevice(dev) == hipSuccess;
        // (an error that a call of the program's before this one has left behind: op_launched would take it for the launch's; the
        // runtime's record of it cannot be put back, so the message says what it was)
        const hipError_t left = hipGetLastError();
        if (left != hipSuccess)
            (void)set_error(TRAG_OK, std::string(who) + ": an earlier HIP call of the program had failed (" + hipGetErrorString(left) + "); its error is cleared");
    }
    ~OpDevice() {
        if (switched) (void)hipSetDevice(prev);
    }
    OpDevice(const OpDevice&) = delete;
    OpDevice& operator=(const OpDevice&) = delete;
};

inline trag_status op_launched(const char* who) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(TRAG_DEVICE_ERROR, std::string(who) + ": " + hipGetErrorString(e));
    return TRAG_OK;
}

// No C++ exception leaves a C entry point (a message that cannot be allocated is the one source).
template <typename F>
inline trag_status op_entry(F&& body) noexcept {
    try {
        return body();
    } catch (const std::bad_alloc&) {
        return TRAG_OOM;
    } catch (...) {
        return TRAG_DEVICE_ERROR;
    }
}

}  // namespace trag
