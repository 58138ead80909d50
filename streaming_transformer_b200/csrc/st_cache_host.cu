// st_cache_host.cu -- argument checks and error messages of the window-cache
// operators (st_cache_*, st_window_attention). Everything a device could not
// refuse by itself is refused here, before any launch.
#include "st_cache_host.h"

#include <atomic>
#include <string>

namespace st {

namespace {
thread_local std::string g_cache_error;
constexpr int kMaxDevices = 64;
std::atomic<int> g_sms[kMaxDevices];

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Two nested strides over `outer` x `inner` blocks of `block` units leave the
// blocks apart: one of the two encloses the other.
bool apart(int64_t outer, int64_t outer_stride, int64_t inner, int64_t inner_stride, int64_t block) {
  if (inner == 1) inner_stride = block;
  if (outer == 1) outer_stride = block;
  if (inner_stride < block || outer_stride < block) return false;
  return outer == 1 || inner == 1 || outer_stride >= (inner - 1) * inner_stride + block ||
         inner_stride >= (outer - 1) * outer_stride + block;
}
// Strides beyond this many units could overflow a 64-bit byte offset.
constexpr int64_t kMaxStride = (int64_t)1 << 40;
}  // namespace

int cache_fail(int code, const char* msg, const char* what) noexcept {
  try {
    g_cache_error = what;
    g_cache_error += msg;
  } catch (...) {  // no memory for the message: the code still says what kind of error it was
    g_cache_error.clear();
  }
  return code;
}

int cache_cuda(cudaError_t e, const char* what) {
  return e == cudaSuccess ? ST_OK : cache_fail(ST_ERR_CUDA, cudaGetErrorString(e), what);
}

int check_cache(const st_cache* c, bool writes) {
  if (!c) return cache_fail(ST_ERR_INVALID, "null cache");
  if (c->device < 0 || c->device >= kMaxDevices) return cache_fail(ST_ERR_INVALID, "device ordinal out of range");
  if (c->type < ST_MODE_FP32 || c->type > ST_CACHE_INT4) return cache_fail(ST_ERR_INVALID, "unknown cache type");
  if (c->streams < 1 || c->streams > 65535 || c->heads < 1 || c->heads > 65535)
    return cache_fail(ST_ERR_INVALID, "cache streams and heads are 1 to 65535");
  const bool four = c->type == ST_CACHE_INT4;
  if (c->head_dim < 8 || c->head_dim > ST_CACHE_MAX_HEAD_DIM || c->head_dim % (four ? ST_CACHE_GROUP : 8))
    return cache_fail(ST_ERR_INVALID, four ? "head_dim of a 4-bit cache is a multiple of 32 up to 256"
                                           : "head_dim is a multiple of 8 up to 256");
  if (c->sinks < 0 || c->window < 1 || (int64_t)c->sinks + c->window > (1 << 30))
    return cache_fail(ST_ERR_INVALID, "a cache has sinks >= 0 and window >= 1, at most 2^30 slots");
  if (!c->keys || !c->values) return cache_fail(ST_ERR_INVALID, "null cache rows");
  if (!aligned16(c->keys) || !aligned16(c->values))
    return cache_fail(ST_ERR_INVALID, "cache rows must start on a 16-byte boundary");
  if (four != (c->key_scales != nullptr) || four != (c->value_scales != nullptr))
    return cache_fail(ST_ERR_INVALID, "a 4-bit cache has scales, any other has none");
  if (four && (!aligned16(c->key_scales) || !aligned16(c->value_scales)))
    return cache_fail(ST_ERR_INVALID, "cache scales must start on a 16-byte boundary");
  if (c->stream_stride < 0 || c->head_stride < 0 || c->stream_stride > kMaxStride || c->head_stride > kMaxStride)
    return cache_fail(ST_ERR_INVALID, "cache strides out of range");
  if (writes && !apart(c->streams, c->stream_stride, c->heads, c->head_stride, (int64_t)c->sinks + c->window))
    return cache_fail(ST_ERR_INVALID, "cache strides let streams or heads overlap");
  return ST_OK;
}

int check_rows(const st_rows& r, const char* name, int mode, int64_t rows, int heads, int head_dim, bool writes) {
  if (!r.data) return cache_fail(ST_ERR_INVALID, ": null pointer", name);
  if (!aligned16(r.data)) return cache_fail(ST_ERR_INVALID, ": must start on a 16-byte boundary", name);
  if (r.row_stride < 0 || r.head_stride < 0 || r.row_stride > kMaxStride || r.head_stride > kMaxStride)
    return cache_fail(ST_ERR_INVALID, ": strides out of range", name);
  const int per = 16 / mode_bytes(mode);
  if (r.row_stride % per || r.head_stride % per)
    return cache_fail(ST_ERR_INVALID, ": strides must be multiples of 16 bytes", name);
  if (writes && !apart(rows, r.row_stride, heads, r.head_stride, head_dim))
    return cache_fail(ST_ERR_INVALID, ": strides let rows overlap", name);
  return ST_OK;
}

int check_aligned(const void* p, const char* name, unsigned bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0
             ? ST_OK : cache_fail(ST_ERR_INVALID, " must be on a boundary of the size of its values", name);
}

DeviceScope::DeviceScope(int device) {
  const cudaError_t pending = cudaPeekAtLastError();
  int current = 0;
  status_ = cache_cuda(cudaGetDevice(&current), "cudaGetDevice: ");
  if (status_ == ST_OK && pending != cudaSuccess)
    status_ = cache_fail(ST_ERR_CUDA, cudaGetErrorString(pending), "an earlier CUDA error is pending: ");
  if (status_ == ST_OK && current != device) {
    status_ = cache_cuda(cudaSetDevice(device), "cudaSetDevice: ");
    if (status_ == ST_OK) previous_ = current;
  }
  if (status_ != ST_OK && pending == cudaSuccess) cudaGetLastError();  // reported here, so not left pending
}

DeviceScope::~DeviceScope() {
  if (previous_ >= 0) cudaSetDevice(previous_);
}

int sm_count(int device) {
  int n = g_sms[device].load(std::memory_order_relaxed);
  if (!n) {
    const bool pending = cudaPeekAtLastError() != cudaSuccess;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
      if (!pending) cudaGetLastError();  // the call that needs the device reports it
      return 1;
    }
    g_sms[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

}  // namespace st

extern "C" const char* st_cache_error(void) { return st::g_cache_error.c_str(); }
