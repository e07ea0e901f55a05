// The current device of an entry point's call.
#pragma once

#include <hip/hip_runtime.h>

namespace airkv {

// The pool's device is the current one while this lives.
class OnDevice {
public:
    explicit OnDevice(int device) {
        status_ = hipGetDevice(&before_);
        if (status_ == hipSuccess && before_ != device) {
            status_ = hipSetDevice(device);
            changed_ = status_ == hipSuccess;
        }
    }
    ~OnDevice() {
        if (changed_) (void)hipSetDevice(before_);
    }
    hipError_t status() const { return status_; }

private:
    int before_ = 0;
    bool changed_ = false;
    hipError_t status_;
};

}  // namespace airkv
