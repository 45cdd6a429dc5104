// Host helpers of stk_capi.cu that the other C entry points share: the
// thread's error message and the device's SM count.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace stk {

int host_fail(int code, const char* msg);
int host_cuda_fail(cudaError_t e, const char* where);
int host_device_sms(int* sms);

inline bool aligned_to(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace stk

// No C++ exception leaves a C entry point.
#define STK_ENTRY_BEGIN try {
#define STK_ENTRY_END                                              \
  }                                                                \
  catch (...) {                                                    \
    return STK_ECUDA;                                              \
  }
