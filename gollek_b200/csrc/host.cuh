// host.cuh -- host helpers that the translation units of libgollek_kernels.so share: the
// last-error message, CUDA error checks, the caller's device, the tensor-map encoder and
// the library's per-(device, stream) scratch.  Defined in gollek_kernels.cu.
#pragma once

#include <cudaTypedefs.h>

#include <string>

#include "common.cuh"

namespace gk {

extern thread_local std::string t_last_error;

// Records the message of a failed call on this thread and returns `code`.
int fail(int code, const char *fmt, ...);
int cuda_fail(cudaError_t e, const char *what);

#define GK_CUDA(call, what)                        \
    do {                                           \
        cudaError_t e_ = (call);                   \
        if (e_ != cudaSuccess) return cuda_fail(e_, what); \
    } while (0)

// Restores the caller's current device on scope exit.
struct DeviceGuard {
    int prev = -1;
    explicit DeviceGuard(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (dev >= 0 && dev != prev) cudaSetDevice(dev);
    }
    ~DeviceGuard() {
        int cur = -1;
        if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
    }
};

PFN_cuTensorMapEncodeTiled_v12000 encode_fn();
int sm_count(int dev);
// The library's scratch: kSplitK begins with arrival counters that are zero between calls; kPlan
// holds whatever the last ragged or shared-prefix call left there.  Never one for the other.
enum class Scratch { kSplitK, kPlan };
int library_workspace(int dev, void *stream, Scratch kind, size_t bytes, void **out, size_t *cap_out = nullptr);
int dtype_bytes(int dt);

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Reads (and with clear, resets) the status word of gollek_varlen.cu's kernels on the
// current device: a __device__ variable belongs to its translation unit.
cudaError_t varlen_status(bool clear, unsigned *out);

}  // namespace gk
