// Argument checks shared by the kernel-level C entry points.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <exception>
#include <initializer_list>
#include <string>

#include "../../include/inl_cuda.h"

namespace inl {

int record_error(int code, const std::string& msg);

struct HookPtr {
  const void* p;
  int align;  // element size
  const char* name;
};

// Every pointer given (NULL ones are the caller's to judge) on an element
// boundary: no device needed.
inline int check_aligned(const char* what, std::initializer_list<HookPtr> ptrs) {
  for (const HookPtr& h : ptrs)
    if (h.p && (reinterpret_cast<uintptr_t>(h.p) % static_cast<uintptr_t>(h.align)) != 0)
      return record_error(INL_ERR_INVALID_INPUT, std::string(what) + ": " + h.name + " is not element-aligned");
  return INL_OK;
}

// Memory of the current device, managed memory or pinned host memory. The rest
// is refused, since a kernel that touches it may fault and take the context with
// it: pageable host memory, and another device's, of which a pointer does not
// tell whether this device was given access to it.
inline int check_reachable(const char* what, std::initializer_list<HookPtr> ptrs) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return record_error(INL_ERR_CONFIG, std::string(what) + ": no CUDA device: " + cudaGetErrorString(e));
  }
  for (const HookPtr& h : ptrs) {
    if (!h.p) continue;
    cudaPointerAttributes at;
    e = cudaPointerGetAttributes(&at, h.p);
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      return record_error(INL_ERR_CONFIG, std::string(what) + ": " + cudaGetErrorString(e));
    }
    if (at.type == cudaMemoryTypeUnregistered || (at.type == cudaMemoryTypeDevice && at.device != dev))
      return record_error(INL_ERR_INVALID_INPUT,
                          std::string(what) + ": " + h.name + " is not memory of the current device");
  }
  return INL_OK;
}

// The status e that a launch returned. An error that an earlier call left on
// this thread is not taken for the launch's, and stays for its owner to read.
inline int launched(const char* what, cudaError_t e) {
  if (e == cudaSuccess) return INL_OK;
  (void)cudaGetLastError();  // the launch's own
  return record_error(INL_ERR_INFERENCE, std::string(what) + " launch failed: " + cudaGetErrorString(e));
}

// Runs the body of a C entry point; no C++ exception leaves it.
template <typename F>
int guarded(F&& body) noexcept {
  try {
    return body();
  } catch (...) {
    return INL_ERR_INFERENCE;
  }
}

}  // namespace inl
