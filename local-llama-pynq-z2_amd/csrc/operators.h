// Operators on device memory (include/llm_hip.h): argument checks shared by the entry points (internal header).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/llm_hip.h"
#include "host_common.h"

// Bytes of a value of an LLM_* type (0: no such type).
static inline int op_type_bytes(int type) {
    return type == LLM_F32 ? 4 : type == LLM_BF16 ? 2 : type == LLM_I8 || type == LLM_E4M3 ? 1 : 0;
}
static inline bool op_scaled(int type) { return type == LLM_I8 || type == LLM_E4M3; }

// The device that holds all these addresses, made current for the call; the caller's device comes back at the end.
// An address that is not device memory (host memory would fault the kernel) or lies on another device is refused.
class OpDevice {
  public:
    explicit OpDevice(const char *who) : who_(who) {}
    ~OpDevice() {
        if (back_ >= 0) (void)hipSetDevice(back_);
    }
    bool holds(const void *p, const char *what) {
        hipPointerAttribute_t at;
        if (!p || hipPointerGetAttributes(&at, p) != hipSuccess ||
            (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged)) {
            (void)hipGetLastError();
            fprintf(stderr, "%s: %s is not device memory\n", who_, what);
            return false;
        }
        if (dev_ >= 0 && at.device != dev_) {
            fprintf(stderr, "%s: %s lies on device %d, other arguments on device %d\n", who_, what, at.device, dev_);
            return false;
        }
        dev_ = at.device;
        return true;
    }
    bool select() {
        int cur = -1;
        if (hipGetDevice(&cur) != hipSuccess) return false;
        if (cur == dev_) return true;
        if (hipSetDevice(dev_) != hipSuccess) {
            fprintf(stderr, "%s: cannot select device %d\n", who_, dev_);
            return false;
        }
        back_ = cur;
        return true;
    }
    int device() const { return dev_; }

  private:
    const char *who_;
    int dev_ = -1, back_ = -1;
};

// A cache that the kernels can walk: whole rows of 16 to 256 values in steps of 16, 4-byte aligned, strides that fit the
// kernels' 32-bit offsets within 64 positions.  Prints what is wrong.  dev NULL: the addresses are not looked up.
bool op_check_cache(const llm_kv *c, OpDevice *dev, const char *who);
// Rows of activations beside it: fp32 or bf16, vectors of 4 values aligned.
bool op_check_rows(const llm_rows *r, const char *what, OpDevice *dev, const char *who);
