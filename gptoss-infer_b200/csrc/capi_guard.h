// The C ABI's error convention, shared by the files that implement it: an exception becomes -1 plus the calling
// thread's message (gptoss_last_error).
#pragma once
#include <exception>
#include <string>

namespace gpt {

std::string& last_error_slot();           // the calling thread's message (capi.cu)

template <class F>
int abi_guard(F&& f) {
    try {
        f();
        return 0;
    } catch (const std::exception& e) {
        last_error_slot() = e.what();
    } catch (...) {
        last_error_slot() = "unknown error";
    }
    return -1;
}

}  // namespace gpt
