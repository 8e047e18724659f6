// Argument checks shared by the C entry points of the block operators (internal
// linkage).
#pragma once

#include <cstdarg>
#include <cstdio>
#include <initializer_list>

#include "mx_common.cuh"
#include "sc_common.cuh"

namespace scmp {
namespace {

int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  set_last_error(buf);
  return code;
}
int cuda_fail(cudaError_t e, const char *what) {
  return fail(SCMP_ECUDA, "%s: %s", what, cudaGetErrorString(e));
}

constexpr int64_t kMaxRows = INT32_MAX - 1023;  // a tile's coordinates stay 32-bit

bool known_dtype(int d) { return d >= SCMP_F32 && d <= SCMP_F16; }
int64_t dtype_bytes(int d) { return d == SCMP_F32 ? 4 : 2; }
bool aligned(std::initializer_list<const void *> ptrs, int64_t to) {
  uintptr_t a = 0;
  for (const void *p : ptrs) a |= reinterpret_cast<uintptr_t>(p);
  return (a & (uintptr_t)(to - 1)) == 0;
}
int check_elements(std::initializer_list<const void *> ptrs, int dtype) {
  if (!aligned(ptrs, dtype_bytes(dtype)))
    return fail(SCMP_EINVAL, "a pointer is not aligned to its elements of %lld bytes",
                (long long)dtype_bytes(dtype));
  return SCMP_OK;
}

}  // namespace
}  // namespace scmp
