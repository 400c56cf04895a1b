// What the entry points of the paged 4-bit key/value cache share.
#pragma once
#include <cuda_fp16.h>

#include "glc_internal.h"
#include "kv_plan.h"
#include "sm100.cuh"

namespace glc {

static_assert(KV_BAD_ARGUMENT == GLC_DEV_BAD_ARGUMENT, "one code");

// Host checks shared by the entry points; 0 or a GLC_ERR_* code.
int kv_check(Context* ctx, const char* what, const glc_kv_cache* cache, const glc_kv_batch* batch);

// Makes the context's device current for the scope (a caller may have another
// one current; launches and allocations go by it).
struct DeviceScope {
  int before = -1;
  explicit DeviceScope(const Context* c) {
    int d = -1;
    if (cudaGetDevice(&d) == cudaSuccess && d != c->device && cudaSetDevice(c->device) == cudaSuccess) before = d;
  }
  ~DeviceScope() {
    if (before >= 0) cudaSetDevice(before);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
};

}  // namespace glc
