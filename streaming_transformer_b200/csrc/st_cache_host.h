// st_cache_host.h -- host side shared by the window-cache operators: error
// messages, argument checks and the device of a call.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/streaming_b200.h"

namespace st {

// Records `what` + `msg` for st_cache_error() and returns `code`. No exception
// leaves it (or anything else here): the callers are C entry points.
int cache_fail(int code, const char* msg, const char* what = "") noexcept;
// ST_OK, or ST_ERR_CUDA with the message of `e`.
int cache_cuda(cudaError_t e, const char* what);

inline int mode_bytes(int mode) { return mode == ST_MODE_FP32 ? 4 : 2; }

// Checks a cache descriptor; `writes`: its rows are written, so streams and
// heads may not overlap.
int check_cache(const st_cache* c, bool writes);
// Checks rows [rows][heads][head_dim] of `mode`; `writes` as above.
int check_rows(const st_rows& r, const char* name, int mode, int64_t rows, int heads, int head_dim, bool writes);
// Checks that `p` (NULL passes) is on a boundary of `bytes`, the size of the values that a kernel loads from it.
int check_aligned(const void* p, const char* name, unsigned bytes);

// Makes `device` current for the calls of a scope and restores the caller's;
// status() is an ST_ERR_CUDA when the device cannot be taken or an error of an
// earlier launch is pending on this thread (it belongs to its caller and is
// reported without being cleared).
class DeviceScope {
 public:
  explicit DeviceScope(int device);
  ~DeviceScope();
  int status() const { return status_; }

 private:
  int previous_ = -1, status_ = ST_OK;
};

// SM count of `device`, read once per process.
int sm_count(int device);

}  // namespace st
