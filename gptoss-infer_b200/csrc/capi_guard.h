// The C ABI's error convention, shared by the files that implement it: an exception becomes -1 plus the calling
// thread's message (gptoss_last_error).
#pragma once
#include <cuda_runtime.h>

#include <exception>
#include <string>

namespace gpt {

std::string& last_error_slot();           // the calling thread's message (capi.cu)

// Ends a failed call: takes the CUDA runtime's last error, which the next launch check would report as its own (a failed
// allocation stays there), and keeps the message. Never throws.
inline void keep_error(const char* what) noexcept {
    cudaGetLastError();
    try {
        last_error_slot() = what;
    } catch (...) {                           // no memory for the message
        last_error_slot().clear();
    }
}

template <class F>
int abi_guard(F&& f) {
    try {
        f();
        return 0;
    } catch (const std::exception& e) {
        keep_error(e.what());
    } catch (...) {
        keep_error("unknown error");
    }
    return -1;
}

}  // namespace gpt
