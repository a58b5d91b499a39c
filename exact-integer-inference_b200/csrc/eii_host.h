// Host-side helpers shared by the translation units of libeii.so: the thread-local error message
// behind eii_last_error(), the CUDA error check, and a guard for the caller's current device.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "eii.h"

namespace eii {

// Records the message of a failed call on this thread and returns `code`.
int fail(int code, const char* fmt, ...);

#define CK(call)                                                                                      \
    do {                                                                                              \
        cudaError_t e_ = (call);                                                                      \
        if (e_ != cudaSuccess) {                                                                      \
            cudaGetLastError(); /* reported here, so no later launch is to find it */                 \
            return fail(EII_ERR_CUDA, "%s: %s (%s:%d)", #call, cudaGetErrorString(e_), __FILE__, __LINE__); \
        }                                                                                             \
    } while (0)
#define TRY(...)                         \
    do {                                 \
        int rc_ = (__VA_ARGS__);         \
        if (rc_ != EII_OK) return rc_;   \
    } while (0)

// Makes `device` current for a scope and restores the caller's device afterwards.
struct DeviceGuard {
    int before = -1;
    cudaError_t st = cudaSuccess;
    explicit DeviceGuard(int device) {
        st = cudaGetDevice(&before);
        if (st == cudaSuccess && before != device) st = cudaSetDevice(device);
        else before = -1;
    }
    ~DeviceGuard() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// A device array that a kernel reads or writes element by element.
inline int check_aligned(const char* name, const void* p, int bytes) {
    if (reinterpret_cast<uintptr_t>(p) % bytes) return fail(EII_ERR_ARG, "%s must be %d-byte aligned", name, bytes);
    return EII_OK;
}

// `device` exists and is sm_100 (EII_ERR_CUDA / EII_ERR_ARG otherwise); leaves the current device alone.
int check_device(int device);

}  // namespace eii
