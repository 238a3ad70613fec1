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

  private:
    const char *who_;
    int dev_ = -1, back_ = -1;
};

// A cache that the kernels can walk: whole rows of 16 to 256 values in steps of 16, 4-byte aligned, strides that fit the
// kernels' 32-bit offsets within 64 positions.  Prints what is wrong.  dev NULL: the addresses are not looked up.
bool op_check_cache(const llm_kv *c, OpDevice *dev, const char *who);
// Rows of activations beside it: fp32 or bf16, vectors of 4 values aligned.
bool op_check_rows(const llm_rows *r, const char *what, OpDevice *dev, const char *who);

// Memory that a call writes: sequences, heads and tokens whose stride is zero lie on one another, and what is left there would
// depend on timing.  Prints what is wrong.  dims, strides: of as many as there are.
static inline bool op_check_apart(const char *who, const char *what, int dims, const int *count, const int64_t *stride) {
    for (int i = 0; i < dims; i++)
        if (count[i] > 1 && stride[i] == 0) {
            fprintf(stderr, "%s: a stride of zero in %s, which is written\n", who, what);
            return false;
        }
    return true;
}

// The launches behind the entry points, for callers that know their arguments to be right (the model).

struct KvCall {
    const int *pos; // NULL: pos0 for every sequence
    int pos0;
    int by_pos;     // writes: the row of position p is row p of the rows, not the t-th
    const int *n;
    int max_n, zero_rest;
};
hipError_t launch_kv(bool write, const llm_kv &c, const llm_rows &k, const llm_rows &v, const KvCall &q, hipStream_t st);
// Of every sequence (the model: layer), rows pos0 + path[j] to pos0 + j; path rises, path[j] < 64.
hipError_t launch_kv_keep(const llm_kv &c, int pos0, const uint8_t *path, int n, hipStream_t st);

struct TreeCall {
    int n_heads;
    const int *lens, *n;
    const uint64_t *mask;
    int max_n, max_len;
    float scale;
    int zero_rest;
    void *work; // llm_tree_attention_work()
};
hipError_t launch_tree_attention(const llm_kv &c, const llm_rows &q, const llm_rows &out, const TreeCall &t, hipStream_t st);

struct LogprobsCall {
    const void *logits;
    int type, rows, vocab;
    int64_t stride;
    float temperature;
    const int *tokens;
    int n_tokens;
    float *logp, *entropy, *lse;
    int top, *top_ids;
    float *top_logp;
    void *work; // llm_logprobs_work()
};
hipError_t launch_logprobs(const LogprobsCall &q, hipStream_t st);
