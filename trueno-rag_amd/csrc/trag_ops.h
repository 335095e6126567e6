// What the operators on a caller's device arrays share (trag_q8.hip, trag_matmul_q8.hip,
// trag_distill.hip): element types, eight elements at a time, workgroup reductions, and the checks
// of an entry point that has no handle to ask for its device.
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

// ---- element types: 8 consecutive elements as floats. A caller's rows may start at any element (odd widths,
// odd strides), so the wide accesses ask for element alignment only; the hardware serves unaligned 16-byte
// accesses, and an aligned row pays nothing for it.
struct F32 {
    typedef float elem;
    typedef float vec4 __attribute__((ext_vector_type(4), aligned(4)));
    static __device__ __forceinline__ float load(const elem* p) { return *p; }
    static __device__ __forceinline__ void store(elem* p, float v) { *p = v; }
    static __device__ __forceinline__ void load8(const elem* p, float (&v)[8]) {
        const vec4 a = *reinterpret_cast<const vec4*>(p), b = *reinterpret_cast<const vec4*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    }
    static __device__ __forceinline__ void store8(elem* p, const float (&v)[8]) {
        vec4 a, b;
#pragma unroll
        for (int i = 0; i < 4; ++i) { a[i] = v[i]; b[i] = v[4 + i]; }
        *reinterpret_cast<vec4*>(p) = a;
        *reinterpret_cast<vec4*>(p + 4) = b;
    }
};

struct F16 {
    // A result is rounded to f32 and then to f16, as in the other types: the product in front of the conversion is hidden
    // from the compiler, which would fold the two into a mixed-precision multiply with a single rounding.
    static __device__ __forceinline__ _Float16 round(float v) {
        asm("" : "+v"(v));
        return (_Float16)v;
    }
    typedef _Float16 elem;
    typedef _Float16 vec8 __attribute__((ext_vector_type(8), aligned(2)));
    static __device__ __forceinline__ float load(const elem* p) { return (float)*p; }
    static __device__ __forceinline__ void store(elem* p, float v) { *p = round(v); }
    static __device__ __forceinline__ void load8(const elem* p, float (&v)[8]) {
        const vec8 a = *reinterpret_cast<const vec8*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
    }
    static __device__ __forceinline__ void store8(elem* p, const float (&v)[8]) {
        vec8 a;
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = round(v[i]);
        *reinterpret_cast<vec8*>(p) = a;
    }
};

struct BF16 {
    typedef __bf16 elem;
    typedef __bf16 vec8 __attribute__((ext_vector_type(8), aligned(2)));
    static __device__ __forceinline__ float load(const elem* p) { return (float)*p; }
    static __device__ __forceinline__ void store(elem* p, float v) { *p = (__bf16)v; }
    static __device__ __forceinline__ void load8(const elem* p, float (&v)[8]) {
        const vec8 a = *reinterpret_cast<const vec8*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
    }
    static __device__ __forceinline__ void store8(elem* p, const float (&v)[8]) {
        vec8 a;
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = (__bf16)v[i];
        *reinterpret_cast<vec8*>(p) = a;
    }
};

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
