// Launchers of the training-side kernels, for the C ABI.  Element types are the header's
// SCMIAC_F32 / SCMIAC_F16 / SCMIAC_BF16.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>

namespace scmiac {

// linear_kernels.hip
struct LinearArgs {
    const void *x, *w, *bias, *residual;
    long long ldx, ldw, ldr;      // row strides in elements
    long long m, n, k;
    int dtype, act;
};
size_t linear_workspace_bytes(long long m, long long n, long long k, int dtype, int act, int backward);
hipError_t launch_linear_forward(const LinearArgs& a, void* y, void* z, void* ws, hipStream_t stream);
hipError_t launch_linear_backward(const LinearArgs& a, const void* z, const void* dy, void* dx, void* dw, void* dbias,
                                  void* ws, hipStream_t stream);

// distill_kernels.hip
size_t top_logits_workspace_bytes(long long n, long long v, int k, int dtype);
hipError_t launch_top_logits(const void* x, long long ld, long long n, long long v, int dtype, int k, float temperature,
                             void* values, int* idx, float* lse, void* ws, hipStream_t stream);
struct DistillArgs {
    const void* x;
    long long ld, n, v;
    int dtype;
    const int* idx;
    const float* top;
    int k;
    const float* teacher_lse;     // NULL: softmax over the listed classes
    float temperature, teacher_temperature;
};
size_t distill_workspace_bytes(long long n, long long v, int dtype);
hipError_t launch_distill_forward(const DistillArgs& a, int reduction, float* loss, float* row_stats, float* scale,
                                  void* ws, hipStream_t stream);
hipError_t launch_distill_backward(const DistillArgs& a, const float* row_stats, const float* grad, long long grad_stride,
                                   const float* scale, void* dx, long long ldd, hipStream_t stream);

}  // namespace scmiac
