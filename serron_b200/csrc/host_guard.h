// Host side of the C ABI's entry points: argument checks with messages, CUDA errors as exceptions that never leave
// the library, and the caller's device restored after each call.
#pragma once

#include "serron_b200.h"

#include <cuda_runtime.h>

#include <sstream>
#include <stdexcept>
#include <string>

#include "common.cuh"

namespace serron {

void set_last_error(const std::string& message);  // api.cu: the message serron_last_error returns

struct Failure {
    int code;
    std::string message;
};

template <typename... Args>
std::string concat(const Args&... args) {
    std::ostringstream oss;
    ((oss << args), ...);
    return oss.str();
}

#define SB_CHECK(cond, ...)                                                                      \
    do {                                                                                         \
        if (!(cond)) throw ::serron::Failure{SERRON_ERR_INVALID, ::serron::concat(__VA_ARGS__)}; \
    } while (0)

#define SB_CUDA(expr)                                                                                          \
    do {                                                                                                       \
        const cudaError_t err_ = (expr);                                                                       \
        if (err_ != cudaSuccess)                                                                               \
            throw ::serron::Failure{SERRON_ERR_CUDA,                                                           \
                                    ::serron::concat("serron: CUDA error ", cudaGetErrorName(err_), ": ",      \
                                                     cudaGetErrorString(err_), " (", #expr, ")")};             \
    } while (0)

template <typename F>
int guarded(F&& f) {
    try {
        f();
        return SERRON_OK;
    } catch (const Failure& e) {
        set_last_error(e.message);
        return e.code;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return SERRON_ERR_INVALID;
    }
}

// Makes `device` current for the scope of a call and restores the previous device.
struct DeviceScope {
    int previous = -1;
    explicit DeviceScope(int device) {
        if (cudaGetDevice(&previous) != cudaSuccess) previous = -1;
        cudaGetLastError();
        if (previous != device) SB_CUDA(cudaSetDevice(device));
    }
    ~DeviceScope() {
        int now = -1;
        if (previous >= 0 && cudaGetDevice(&now) == cudaSuccess && now != previous) cudaSetDevice(previous);
    }
};

inline size_t elem_size(int dtype) { return dtype == kF64 ? 8 : dtype == kF32 ? 4 : 2; }

}  // namespace serron
