// What translation units other than backend.cu see of a device context.
#pragma once
#include <cuda_runtime.h>

namespace pgb {

struct CtxRef {
    int device, sms;
    cudaStream_t stream;
    int *err;  // the device error word
};

int ctx_of(int device, CtxRef *ref);  // 0 when the device was not initialised
void count_launches(int n);
void forget_opt_ins();  // attn.cu: kernel attributes are set anew (at shutdown)

// Makes a context's device current for one call and puts the caller's back.
class DeviceGuard {
  public:
    explicit DeviceGuard(int device) {
        ok_ = cudaGetDevice(&was_) == cudaSuccess;
        if (ok_ && was_ != device) {
            ok_ = cudaSetDevice(device) == cudaSuccess;
            back_ = ok_;
        }
    }
    ~DeviceGuard() {
        if (back_) cudaSetDevice(was_);
    }
    bool ok() const { return ok_; }

  private:
    int was_ = 0;
    bool ok_ = false, back_ = false;
};

}  // namespace pgb
