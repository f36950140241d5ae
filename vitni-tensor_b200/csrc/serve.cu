// serve.cu -- the batched serving operators' error message (vtq_device_last_error).
#include "serve.h"

#include <cstdarg>
#include <cstdio>

namespace {
thread_local char g_serve_error[256] = "";
}

namespace vtq {

vtq_status serve_fail(vtq_status s, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_serve_error, sizeof g_serve_error, fmt, ap);
  va_end(ap);
  return s;
}

vtq_status serve_cuda(cudaError_t e, const char* where) {
  if (e == cudaSuccess) return VTQ_OK;
  return serve_fail(e == cudaErrorMemoryAllocation ? VTQ_ERR_OOM : VTQ_ERR_GPU, "gpu error: %s: %s",
                    where, cudaGetErrorString(e));
}

}  // namespace vtq

extern "C" const char* vtq_device_last_error(void) { return g_serve_error; }
