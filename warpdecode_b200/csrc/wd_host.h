// What the translation units of the library share on the host: the calling thread's error text, and the device of a call.
#pragma once

#include <cuda_runtime.h>

#include <exception>
#include <new>
#include <string>

#include "../../include/warpdecode_b200.h"

namespace wd_host {

int set_error(int code, const std::string &msg);        // (wd_engine.cu) the text behind wd_last_error(); returns code

#define WD_TRY_CUDA(call)                                                                                       \
    do {                                                                                                        \
        cudaError_t e__ = (call);                                                                               \
        if (e__ != cudaSuccess) return wd_host::set_error(WD_E_CUDA, std::string(#call) + ": " + cudaGetErrorString(e__)); \
    } while (0)

// The device of a call, and the thread's own one again behind it.
class OnDevice {
public:
    explicit OnDevice(int device) {
        if (cudaGetDevice(&before_) != cudaSuccess) before_ = device;
        if (before_ != device) ok_ = cudaSetDevice(device) == cudaSuccess, changed_ = ok_;
        if (!ok_) cudaGetLastError();       // (the caller says so; a later launch is not to be blamed for it)
    }
    ~OnDevice() {
        if (changed_) cudaSetDevice(before_);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
    bool ok() const { return ok_; }

private:
    int before_ = 0;
    bool ok_ = true, changed_ = false;
};

// No exception leaves a C entry.
template <class F>
int guarded(F &&f) {
    try {
        return f();
    } catch (const std::bad_alloc &) {
        return set_error(WD_E_NOMEM, "out of host memory");
    } catch (const std::exception &e) {
        return set_error(WD_E_STATE, e.what());
    } catch (...) {
        return set_error(WD_E_STATE, "unexpected failure");
    }
}

}  // namespace wd_host
