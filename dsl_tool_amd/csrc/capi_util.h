// Status, message and argument checks shared by the extern "C" entry points
// (capi.hip, capi_serve.hip).
#pragma once

#include <cstdarg>
#include <cstdio>
#include <string>

#include "dsl_gemm.h"
#include "launch.h"

namespace dsl {
namespace capi {

inline thread_local std::string g_err;

inline int fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_err = buf;
  return code;
}

inline int ok() {
  g_err.clear();
  return DSL_OK;
}

inline int hip_status(hipError_t e, const char *what) {
  if (e == hipSuccess) return ok();
  return fail(DSL_ERR_HIP, "%s: HIP error %d (%s)", what, (int)e, hipGetErrorString(e));
}

inline bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Common checks of a bf16 / fp32 input matrix.
inline int check_input(const char *fn, const void *x, int64_t rows, int64_t cols, int64_t sr,
                int64_t sc, int x_dtype) {
  if (x_dtype != DSL_IN_BF16 && x_dtype != DSL_IN_F32)
    return fail(DSL_ERR_ARG, "%s: unknown x_dtype %d", fn, x_dtype);
  if (rows < 0 || cols < 0) return fail(DSL_ERR_ARG, "%s: negative shape (%lld, %lld)", fn,
                                        (long long)rows, (long long)cols);
  if (rows == 0 || cols == 0) return DSL_OK;
  if (!x) return fail(DSL_ERR_ARG, "%s: input pointer is NULL", fn);
  if (!aligned(x, x_dtype == DSL_IN_F32 ? 4 : 2))
    return fail(DSL_ERR_ARG, "%s: input must be aligned to its element size", fn);
  if (sr <= 0 || sc <= 0)
    return fail(DSL_ERR_ARG, "%s: strides must be positive (got %lld, %lld)", fn, (long long)sr,
                (long long)sc);
  if (rows >= (int64_t)1 << 31 || cols >= (int64_t)1 << 31)
    return fail(DSL_ERR_ARG, "%s: dimensions must be < 2^31", fn);
  return DSL_OK;
}

inline int check_out(const char *fn, const void *q, const char *name) {
  if (!q) return fail(DSL_ERR_ARG, "%s: %s is NULL", fn, name);
  if (!aligned(q, 16)) return fail(DSL_ERR_ARG, "%s: %s must be 16-byte aligned", fn, name);
  return DSL_OK;
}

inline int check_gemm_dims(const char *fn, int64_t m, int64_t n, int64_t k, int64_t ldc, int kmult,
                    int out_dtype) {
  if (m < 0 || n < 0 || k <= 0)
    return fail(DSL_ERR_ARG, "%s: need m >= 0, n >= 0, k > 0 (got %lld, %lld, %lld)", fn,
                (long long)m, (long long)n, (long long)k);
  if (m >= (int64_t)1 << 31 || n >= (int64_t)1 << 31 || k >= (int64_t)1 << 31)
    return fail(DSL_ERR_ARG, "%s: dimensions must be < 2^31", fn);
  if (k % kmult != 0)
    return fail(DSL_ERR_ARG, "%s: k=%lld must be a multiple of %d", fn, (long long)k, kmult);
  if (ldc < n) return fail(DSL_ERR_ARG, "%s: ldc=%lld < n=%lld", fn, (long long)ldc, (long long)n);
  if (out_dtype != DSL_OUT_BF16 && out_dtype != DSL_OUT_F32)
    return fail(DSL_ERR_ARG, "%s: unknown out_dtype %d", fn, out_dtype);
  return DSL_OK;
}

}  // namespace capi
}  // namespace dsl
