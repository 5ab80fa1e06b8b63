// Host-side errors of the C ABI: a C++ exception per status code inside the library, turned
// into the code and a thread-local message at every C entry point.
#pragma once
#include <cuda_runtime.h>

#include <new>
#include <stdexcept>
#include <string>

#include "../../include/cora_b200.h"

namespace cora {

extern thread_local std::string g_last_error;  // defined in engine.cu

struct Error : std::runtime_error {
    int code;
    Error(int c, const std::string &m) : std::runtime_error(m), code(c) {}
};
[[noreturn]] inline void fail(int code, const std::string &msg) { throw Error(code, msg); }

#define CUDA_TRY(call)                                                                  \
    do {                                                                                \
        cudaError_t e_ = (call);                                                        \
        if (e_ != cudaSuccess)                                                          \
            ::cora::fail(CORA_ECUDA, std::string(#call) + ": " + cudaGetErrorString(e_)); \
    } while (0)

template <typename F>
int guarded(F &&f) {
    try {
        f();
        return CORA_OK;
    } catch (const Error &e) {
        g_last_error = e.what();
        return e.code;
    } catch (const std::bad_alloc &e) {
        g_last_error = e.what();
        return CORA_ENOMEM;
    } catch (const std::exception &e) {
        g_last_error = e.what();
        return CORA_ERUNTIME;
    }
}

}  // namespace cora
