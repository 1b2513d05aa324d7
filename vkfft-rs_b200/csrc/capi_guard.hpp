// What the extern "C" sources share: the context handle and the wrapper that turns
// exceptions into statuses.
#pragma once

#include <string>
#include <utility>

#include "runtime.hpp"

struct b200fft_context {
    b200fft::Context *ctx;
};

namespace b200fft {

void set_last_error(std::string message);  // the thread's b200fft_last_error_string()

template <typename F>
b200fft_status guarded(F &&f) {
    try {
        f();
        return B200FFT_OK;
    } catch (const FftError &e) {
        set_last_error(e.message);
        return e.code;
    } catch (const std::bad_alloc &) {
        set_last_error("CUDA runtime error: host allocation failed");
        return B200FFT_NATIVE_RUNTIME;
    } catch (const std::exception &e) {
        set_last_error(std::string("CUDA runtime error: ") + e.what());
        return B200FFT_NATIVE_RUNTIME;
    }
}

inline void need(const void *p, const char *what) {
    if (!p) throw FftError(B200FFT_VALUE_OUT_OF_RANGE, std::string(what) + " must not be null");
}

}  // namespace b200fft
