// Shared host-side helpers of libstt_mi355x.so: error reporting.
#pragma once
#include <hip/hip_runtime.h>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <vector>

#include "../../include/stt_mi355x.h"

// Records a message for stt_last_error() and returns `code`.
int stt_fail(int code, const char* fmt, ...);

#define STT_HIP_OR_FAIL(expr, cleanup)                                                  \
  do {                                                                                  \
    hipError_t e_ = (expr);                                                             \
    if (e_ != hipSuccess) {                                                             \
      cleanup;                                                                          \
      return stt_fail(STT_ERR_HIP, "%s failed: %s (%s:%d)", #expr, hipGetErrorString(e_), \
                      __FILE__, __LINE__);                                              \
    }                                                                                   \
  } while (0)

// Workgroup barrier for LDS traffic alone: this wave's LDS operations are done, loads from global memory stay
// in flight (__syncthreads also waits for those, which exposes their latency at every step of a pipelined
// loop).
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);      // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
