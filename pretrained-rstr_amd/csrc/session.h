// session.h -- what the translation units of the C ABI share: the session, its
// error reporting and the device allocation that every handle uses.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>

#include <string>

#include "../../include/rstr_hip.h"

struct rstr_session {
  int device = 0;
  hipStream_t stream = nullptr;
  std::string err;
  void* scratch = nullptr;  // device address of this GPU's static staging array
};

namespace rstr {

// Leaves `msg` with the session (or with the thread's open error) and returns `code`.
int fail(rstr_session* s, int code, const std::string& msg);

// hipMalloc, tried again without the blocks that the pools of this GPU keep
// for isolated attention when it does not fit.
hipError_t device_alloc(void** p, size_t bytes);

}  // namespace rstr

#define HIPCHK(S, expr)                                                                  \
  do {                                                                                   \
    hipError_t e_ = (expr);                                                              \
    if (e_ != hipSuccess)                                                                \
      return fail((S), e_ == hipErrorOutOfMemory ? RSTR_E_OOM : RSTR_E_HIP,              \
                  std::string(#expr) + ": " + hipGetErrorString(e_));                    \
  } while (0)
