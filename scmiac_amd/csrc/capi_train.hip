// extern "C" boundary of the training-side kernels (declared in include/scmiac_hip.h).
#include <float.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include "../../include/scmiac_hip.h"
#include "api_error.h"
#include "train_kernels.h"

using namespace scmiac;

namespace {

constexpr int64_t kMaxRows = ((int64_t)1 << 24) - 1;    // blocks of 256 threads in one launch
constexpr int64_t kMaxWidth = ((int64_t)1 << 31) - 1;
constexpr int64_t kMaxTiles = ((int64_t)1 << 23) - 1024;  // two products and their splits in one launch

__attribute__((format(printf, 2, 3))) int fail(int code, const char* fmt, ...) {
    char text[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof(text), fmt, ap);
    va_end(ap);
    return api_fail(code, text);
}
int done(hipError_t e, const char* what) {
    return e == hipSuccess ? SCMIAC_OK : fail(SCMIAC_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}
// (of a denormal one neither 1 / v nor log2(e) / v need be finite)
bool is_temperature(float v) { return v >= FLT_MIN && v < INFINITY; }

int check_dtype(int dtype) {
    if (dtype < SCMIAC_F32 || dtype > SCMIAC_BF16) return fail(SCMIAC_ERR_ARG, "dtype=%d is none of SCMIAC_F32/F16/BF16", dtype);
    return SCMIAC_OK;
}
int check_workspace(const void* ws, size_t have, size_t need) {
    if ((reinterpret_cast<uintptr_t>(ws) & 15) != 0) return fail(SCMIAC_ERR_WORKSPACE, "workspace is not aligned to 16 bytes");
    if (need > have || (need && !ws)) return fail(SCMIAC_ERR_WORKSPACE, "workspace holds %zu bytes, %zu needed", have, need);
    return SCMIAC_OK;
}

int check_linear(int64_t m, int64_t n, int64_t k, int dtype, int act) {
    if (int rc = check_dtype(dtype)) return rc;
    if (act < SCMIAC_ACT_NONE || act > SCMIAC_ACT_SILU) return fail(SCMIAC_ERR_ARG, "act=%d is no SCMIAC_ACT_*", act);
    if (m < 0 || n < 1 || k < 1 || m > kMaxWidth || n > kMaxWidth || k > kMaxWidth)
        return fail(SCMIAC_ERR_ARG, "m=%lld, n=%lld, k=%lld: needs 0 <= m, 1 <= n, k, below 2^31", (long long)m, (long long)n,
                    (long long)k);
    const int64_t tm = (m + 63) / 64, tn = (n + 63) / 64, tk = (k + 63) / 64;
    if (tm * tn > kMaxTiles || tm * tk > kMaxTiles || tn * tk > kMaxTiles)
        return fail(SCMIAC_ERR_ARG, "m=%lld, n=%lld, k=%lld: a product of more than 2^23 - 1024 tiles of 64 x 64", (long long)m, (long long)n,
                    (long long)k);
    return SCMIAC_OK;
}

int check_rows(int64_t ld, int64_t n, int64_t v, int dtype) {
    if (int rc = check_dtype(dtype)) return rc;
    if (n < 0 || n > kMaxRows) return fail(SCMIAC_ERR_ARG, "n=%lld rows outside 0..2^24-1", (long long)n);
    if (v < 1 || v > kMaxWidth) return fail(SCMIAC_ERR_ARG, "v=%lld classes outside 1..2^31-1", (long long)v);
    if (ld < 0) return fail(SCMIAC_ERR_ARG, "negative row stride");
    return SCMIAC_OK;
}
int check_top(int64_t n, int64_t v, int k, int dtype) {
    if (int rc = check_rows(0, n, v, dtype)) return rc;
    if (k < 1 || k > SCMIAC_TOP_MAX_K) return fail(SCMIAC_ERR_ARG, "k=%d outside 1..%d", k, SCMIAC_TOP_MAX_K);
    return SCMIAC_OK;
}
int check_distill(int64_t ld, int64_t n, int64_t v, int dtype, int k, float temperature, float teacher_temperature) {
    if (int rc = check_rows(ld, n, v, dtype)) return rc;
    if (k < 1 || k > SCMIAC_DISTILL_MAX_K) return fail(SCMIAC_ERR_ARG, "k=%d outside 1..%d", k, SCMIAC_DISTILL_MAX_K);
    if (!is_temperature(temperature) || !is_temperature(teacher_temperature))
        return fail(SCMIAC_ERR_ARG, "temperatures must be positive, finite and at least 2^-126");
    return SCMIAC_OK;
}

}  // namespace

extern "C" {

int scmiac_linear_workspace_size(int64_t m, int64_t n, int64_t k, int dtype, int act, int backward, size_t* bytes) {
    if (!bytes) return fail(SCMIAC_ERR_ARG, "bytes is NULL");
    if (int rc = check_linear(m, n, k, dtype, act)) return rc;
    *bytes = linear_workspace_bytes(m, n, k, dtype, act, backward);
    return SCMIAC_OK;
}

int scmiac_linear_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* residual,
                          int64_t ldr, int64_t m, int64_t n, int64_t k, int dtype, int act, void* y, void* z,
                          void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_linear(m, n, k, dtype, act)) return rc;
    if (m == 0) return SCMIAC_OK;
    if (!x || !w || !y) return fail(SCMIAC_ERR_ARG, "NULL device pointer");
    if (ldx < 0 || ldw < 0 || ldr < 0) return fail(SCMIAC_ERR_ARG, "negative row stride");
    if (int rc = check_workspace(workspace, workspace_bytes, linear_workspace_bytes(m, n, k, dtype, act, 0))) return rc;
    const LinearArgs a = {x, w, bias, residual, ldx, ldw, ldr, m, n, k, dtype, act};
    return done(launch_linear_forward(a, y, z, workspace, static_cast<hipStream_t>(stream)), "linear_forward");
}

int scmiac_linear_backward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* z, const void* dy, int64_t m,
                           int64_t n, int64_t k, int dtype, int act, void* dx, void* dw, void* dbias, void* workspace,
                           size_t workspace_bytes, void* stream) {
    if (int rc = check_linear(m, n, k, dtype, act)) return rc;
    if (m == 0 && !dw && !dbias) return SCMIAC_OK;
    if (m > 0 && (!dy || (dx && !w) || (dw && !x) || (act != SCMIAC_ACT_NONE && !z)))
        return fail(SCMIAC_ERR_ARG, "NULL device pointer");
    if (ldx < 0 || ldw < 0) return fail(SCMIAC_ERR_ARG, "negative row stride");
    if (int rc = check_workspace(workspace, workspace_bytes, linear_workspace_bytes(m, n, k, dtype, act, 1))) return rc;
    const LinearArgs a = {x, w, nullptr, nullptr, ldx, ldw, 0, m, n, k, dtype, act};
    return done(launch_linear_backward(a, z, dy, m > 0 ? dx : nullptr, dw, dbias, workspace, static_cast<hipStream_t>(stream)),
                "linear_backward");
}

int scmiac_top_logits_workspace_size(int64_t n, int64_t v, int k, int dtype, size_t* bytes) {
    if (!bytes) return fail(SCMIAC_ERR_ARG, "bytes is NULL");
    if (int rc = check_top(n, v, k, dtype)) return rc;
    *bytes = n > 0 ? top_logits_workspace_bytes(n, v, k, dtype) : 0;
    return SCMIAC_OK;
}

int scmiac_top_logits(const void* x, int64_t ld, int64_t n, int64_t v, int dtype, int k, float temperature, void* values,
                      int32_t* idx, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_top(n, v, k, dtype)) return rc;
    if (ld < 0) return fail(SCMIAC_ERR_ARG, "negative row stride");
    if (!is_temperature(temperature)) return fail(SCMIAC_ERR_ARG, "temperature must be positive, finite and at least 2^-126");
    if (n == 0) return SCMIAC_OK;
    if (!x || !values || !idx || !lse) return fail(SCMIAC_ERR_ARG, "NULL device pointer");
    if (int rc = check_workspace(workspace, workspace_bytes, top_logits_workspace_bytes(n, v, k, dtype))) return rc;
    return done(launch_top_logits(x, ld, n, v, dtype, k, temperature, values, idx, lse, workspace,
                                  static_cast<hipStream_t>(stream)),
                "top_logits");
}

int scmiac_distill_workspace_size(int64_t n, int64_t v, int dtype, size_t* bytes) {
    if (!bytes) return fail(SCMIAC_ERR_ARG, "bytes is NULL");
    if (int rc = check_rows(0, n, v, dtype)) return rc;
    *bytes = distill_workspace_bytes(n, v, dtype);
    return SCMIAC_OK;
}

int scmiac_distill_forward(const void* x, int64_t ld, int64_t n, int64_t v, int dtype, const int32_t* idx, const float* top,
                           int k, const float* teacher_lse, float temperature, float teacher_temperature, int reduction,
                           float* loss, float* row_stats, float* scale, void* workspace, size_t workspace_bytes,
                           void* stream) {
    if (int rc = check_distill(ld, n, v, dtype, k, temperature, teacher_temperature)) return rc;
    if (reduction < SCMIAC_REDUCE_NONE || reduction > SCMIAC_REDUCE_SUM)
        return fail(SCMIAC_ERR_ARG, "reduction=%d is no SCMIAC_REDUCE_*", reduction);
    if (n == 0 && reduction == SCMIAC_REDUCE_NONE) return SCMIAC_OK;
    if (!loss || (reduction != SCMIAC_REDUCE_NONE && !scale) || (n > 0 && (!x || !idx || !top || !row_stats)))
        return fail(SCMIAC_ERR_ARG, "NULL device pointer");
    if (int rc = check_workspace(workspace, workspace_bytes, distill_workspace_bytes(n, v, dtype))) return rc;
    const DistillArgs a = {x, ld, n, v, dtype, idx, top, k, teacher_lse, temperature, teacher_temperature};
    return done(launch_distill_forward(a, reduction, loss, row_stats, scale, workspace, static_cast<hipStream_t>(stream)),
                "distill_forward");
}

int scmiac_distill_backward(const void* x, int64_t ld, int64_t n, int64_t v, int dtype, const int32_t* idx, const float* top,
                            int k, float temperature, float teacher_temperature, const float* row_stats, const float* grad,
                            int64_t grad_stride, const float* scale, void* dx, int64_t ldd, void* stream) {
    if (int rc = check_distill(ld, n, v, dtype, k, temperature, teacher_temperature)) return rc;
    if (ldd < v && n > 1) return fail(SCMIAC_ERR_ARG, "rows of the gradient overlap: stride %lld, %lld classes", (long long)ldd, (long long)v);
    if (grad_stride < 0) return fail(SCMIAC_ERR_ARG, "negative gradient stride");
    if (n == 0) return SCMIAC_OK;
    if (!x || !idx || !top || !row_stats || !grad || !dx) return fail(SCMIAC_ERR_ARG, "NULL device pointer");
    const DistillArgs a = {x, ld, n, v, dtype, idx, top, k, nullptr, temperature, teacher_temperature};
    return done(launch_distill_backward(a, row_stats, grad, grad_stride, scale, dx, ldd, static_cast<hipStream_t>(stream)),
                "distill_backward");
}

}  // extern "C"
