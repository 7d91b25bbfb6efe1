// What the files behind the C ABI share: errors as status codes, and a
// context's devices and caches.
#pragma once

#include <cuda_runtime.h>

#include <new>
#include <string>

#include "error.h"

#define SHIELD_CUDA(x)                                                                                 \
    do {                                                                                               \
        cudaError_t e_ = (x);                                                                          \
        if (e_ != cudaSuccess) {                                                                       \
            cudaGetLastError(); /* reported here: no later launch may take it for its own */           \
            throw ::shield::Error(e_ == cudaErrorMemoryAllocation ? SHIELD_ERR_NOMEM : SHIELD_ERR_CUDA, \
                                  std::string(#x) + " failed: " + cudaGetErrorString(e_));             \
        }                                                                                              \
    } while (0)

namespace shield {

namespace kv {
struct State;
}

// Sets the calling thread's shield_last_error message.
void set_last_error(const char *message);

// Runs f and turns what it throws into a status code and a message.
template <class F>
shield_status guarded(F &&f) {
    try {
        f();
        set_last_error("");
        return SHIELD_OK;
    } catch (const Error &e) {
        set_last_error(e.what());
        return e.code;
    } catch (const std::bad_alloc &) {
        set_last_error("host memory exhausted");
        return SHIELD_ERR_NOMEM;
    } catch (const std::exception &e) {
        set_last_error(e.what());
        return SHIELD_ERR_CUDA;
    }
}

// One GPU of a context.
struct DeviceView {
    int ordinal = 0;
    int sms = 0;
    cudaStream_t stream = nullptr;
};
DeviceView device_view(shield_ctx *ctx, int32_t device);  // SHIELD_ERR_RANGE outside the context
kv::State &kv_state(shield_ctx *ctx);

// Makes a device current for a scope and the caller's current again after it.
struct DeviceScope {
    int before = -1;
    explicit DeviceScope(int ordinal) {
        if (cudaGetDevice(&before) != cudaSuccess) before = -1;
        if (before == ordinal) before = -1;
        else SHIELD_CUDA(cudaSetDevice(ordinal));
    }
    ~DeviceScope() {
        if (before >= 0) cudaSetDevice(before);
    }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope &operator=(const DeviceScope &) = delete;
};

}  // namespace shield
