// What the prompt-width operators' C entry points share: refusals that name the argument, and
// the carving of the caller's workspace.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "abi_errors.h"
#include "prompt_ops.h"

namespace mono {
namespace prompt {

inline int refuse(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
inline int refuse(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return mono::abi_fail(MONO_EINVAL, buf);
}

inline int launched(hipError_t e, const char* what) {
  if (e == hipSuccess) return mono::abi_ok();
  char buf[256];
  snprintf(buf, sizeof buf, "launching %s: %s", what, hipGetErrorString(e));
  return mono::abi_fail(MONO_EHIP, buf);
}

// a device pointer that the launches' vector loads and stores can use
inline int need(const void* p, const char* name, size_t align) {
  if (!p) return refuse("argument %s must be a device pointer, got NULL", name);
  if (reinterpret_cast<uintptr_t>(p) % align) return refuse("argument %s must be %zu-byte aligned, got %p", name, align, p);
  return MONO_OK;
}

inline int need_rows(int64_t rows, const char* name) {
  if (rows < 0 || rows > MAX_ROWS) return refuse("%s must be in [0, %lld], got %lld", name, (long long)MAX_ROWS, (long long)rows);
  return MONO_OK;
}

inline int need_stride(int64_t stride, int64_t least, int64_t multiple, const char* name) {
  if (stride < least || stride % multiple)
    return refuse("%s must be a multiple of %lld that is at least %lld, got %lld", name, (long long)multiple, (long long)least,
                  (long long)stride);
  return MONO_OK;
}

// Carves the caller's workspace into 256-byte aligned pieces; with no base it only adds
// up what a call needs.
struct Space {
  char* base;
  size_t off = 0;
  template <class T>
  T* take(size_t n) {
    T* p = base ? reinterpret_cast<T*>(base + off) : nullptr;
    off += (n * sizeof(T) + 255) & ~size_t(255);
    return p;
  }
  Rows rows(int64_t n, int k) {
    uint8_t* q = take<uint8_t>((size_t)n * k);
    return Rows{q, take<float>((size_t)n * (k / BLK)), (int)n};
  }
};

inline int need_space(const void* ws, int64_t bytes, size_t least) {
  if (bytes < 0 || (size_t)bytes < least) return refuse("workspace must hold %zu bytes, got %lld", least, (long long)bytes);
  return need(ws, "workspace", 256);
}

}  // namespace prompt
}  // namespace mono
