// st_window.cu -- causal attention of packed sequences with a sliding window
// and sinks (st_window_attention).
//
// A group of lanes takes one query row of one head and walks the keys it sees:
// the sinks before the window, then the window. One pass, with a running
// maximum and sum in fp32.
#include "st_cache.cuh"
#include "st_cache_host.h"

namespace st {
namespace {

constexpr int kWindowThreads = 128;

struct WindowArgs {
  const void* q; const void* k; const void* v; void* out;
  long long q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;  // elements
  const int* starts;
  int rows, sequences, heads, kv_heads, head_dim, window, sinks;
  float scale;
};

// The sequence that owns `row`, as its first row; -1 outside every sequence.
__device__ int sequence_start(const WindowArgs& a, int row) {
  if (!a.starts) return 0;
  int lo = 0, hi = a.sequences;  // the first sequence that ends behind the row
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.starts[mid + 1] <= row) lo = mid + 1;
    else hi = mid;
  }
  if (lo == a.sequences) return -1;
  const int first = clamp_row(a.starts[lo], a.rows);
  return first <= row ? first : -1;
}

template <typename T, int LANES>
__global__ void __launch_bounds__(kWindowThreads) k_window_rows(const WindowArgs a) {
  const int lane = threadIdx.x % LANES, h = blockIdx.y, kv = h / (a.heads / a.kv_heads);
  const unsigned mask = LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u) << ((threadIdx.x & 31) / LANES * LANES);
  const long long row = (long long)blockIdx.x * (kWindowThreads / LANES) + threadIdx.x / LANES;
  if (row >= a.rows) return;
  const int start = sequence_start(a, (int)row);
  if (start < 0) return;
  const bool on = lane * 8 < a.head_dim;
  float q[8] = {}, acc[8] = {}, m = -INFINITY, l = 0.f;
  if (on) load8(static_cast<const T*>(a.q) + row * a.q_row + h * a.q_head + lane * 8, q);
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] *= a.scale;
  const T* kp = static_cast<const T*>(a.k) + kv * a.k_head + lane * 8;
  const T* vp = static_cast<const T*>(a.v) + kv * a.v_head + lane * 8;
  const int low = (int)max((long long)start, row - a.window + 1);  // first row of the window
  int j = start < low && a.sinks > 0 ? start : low;
  while (j <= row) {
    float k[8] = {}, v[8] = {}, dot = 0.f;
    if (on) {
      load8(kp + j * a.k_row, k);
      load8(vp + j * a.v_row, v);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) dot = fmaf(q[i], k[i], dot);
#pragma unroll
    for (int o = 1; o < LANES; o *= 2) dot += __shfl_xor_sync(mask, dot, o);
    const float top = fmaxf(m, dot), keep = top == -INFINITY ? 1.f : __expf(m - top);
    const float p = __expf(dot - (top == -INFINITY ? 0.f : top));  // a NaN stays one
    m = top;
    l = fmaf(l, keep, p);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(acc[i], keep, p * v[i]);
    ++j;
    if (j < low && j - start >= a.sinks) j = low;
  }
  const float inv = l > 0.f ? 1.f / l : NAN;
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] *= inv;
  if (on) store8(static_cast<T*>(a.out) + row * a.o_row + h * a.o_head + lane * 8, acc);
}

template <typename T, int LANES>
void launch_rows(const WindowArgs& a, cudaStream_t s) {
  const long long per = kWindowThreads / LANES;
  k_window_rows<T, LANES><<<dim3((unsigned)((a.rows + per - 1) / per), a.heads), kWindowThreads, 0, s>>>(a);
}

template <typename T>
void launch_window(const WindowArgs& a, cudaStream_t s) {
  switch (lanes_per_row(a.head_dim)) {
    case 1: launch_rows<T, 1>(a, s); break;
    case 2: launch_rows<T, 2>(a, s); break;
    case 4: launch_rows<T, 4>(a, s); break;
    case 8: launch_rows<T, 8>(a, s); break;
    case 16: launch_rows<T, 16>(a, s); break;
    default: launch_rows<T, 32>(a, s); break;
  }
}

}  // namespace
}  // namespace st

using namespace st;

extern "C" int st_window_attention(const st_window* p, void* stream) {
  if (!p) return cache_fail(ST_ERR_INVALID, "null arguments");
  if (p->device < 0 || p->device >= 64) return cache_fail(ST_ERR_INVALID, "device ordinal out of range");
  if (p->mode < ST_MODE_FP32 || p->mode > ST_MODE_BF16) return cache_fail(ST_ERR_INVALID, "unknown row mode");
  if (p->kv_heads < 1 || p->heads < 1 || p->heads > 65535 || p->heads % p->kv_heads)
    return cache_fail(ST_ERR_INVALID, "query heads are a multiple of the key heads, up to 65535");
  if (p->head_dim < 8 || p->head_dim > ST_CACHE_MAX_HEAD_DIM || p->head_dim % 8)
    return cache_fail(ST_ERR_INVALID, "head_dim is a multiple of 8 up to 256");
  if (p->rows < 0 || p->rows > INT32_MAX) return cache_fail(ST_ERR_INVALID, "rows are 0 to 2^31 - 1");
  if (p->window < 1 || p->sinks < 0) return cache_fail(ST_ERR_INVALID, "window is at least 1 and sinks at least 0");
  if (p->starts ? p->sequences < 0 : p->sequences != 1)
    return cache_fail(ST_ERR_INVALID, "without starts there is one sequence");
  if (!(p->scale > -3.0e38f && p->scale < 3.0e38f)) return cache_fail(ST_ERR_INVALID, "scale must be finite");
  if (p->rows == 0 || p->sequences == 0) return ST_OK;
  int rc;
  if ((rc = check_rows(p->q, "q", p->mode, p->rows, p->heads, p->head_dim, false)) != ST_OK ||
      (rc = check_rows(p->k, "k", p->mode, p->rows, p->kv_heads, p->head_dim, false)) != ST_OK ||
      (rc = check_rows(p->v, "v", p->mode, p->rows, p->kv_heads, p->head_dim, false)) != ST_OK ||
      (rc = check_rows(p->out, "out", p->mode, p->rows, p->heads, p->head_dim, true)) != ST_OK)
    return rc;
  DeviceScope scope(p->device);
  if (scope.status() != ST_OK) return scope.status();
  WindowArgs a{};
  a.q = p->q.data; a.k = p->k.data; a.v = p->v.data; a.out = p->out.data;
  a.q_row = p->q.row_stride; a.q_head = p->q.head_stride;
  a.k_row = p->k.row_stride; a.k_head = p->k.head_stride;
  a.v_row = p->v.row_stride; a.v_head = p->v.head_stride;
  a.o_row = p->out.row_stride; a.o_head = p->out.head_stride;
  a.starts = p->starts; a.rows = (int)p->rows; a.sequences = p->sequences;
  a.heads = p->heads; a.kv_heads = p->kv_heads; a.head_dim = p->head_dim;
  a.window = p->window; a.sinks = p->sinks; a.scale = p->scale;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p->mode == ST_MODE_FP32) launch_window<float>(a, s);
  else if (p->mode == ST_MODE_FP16) launch_window<__half>(a, s);
  else launch_window<__nv_bfloat16>(a, s);
  return cache_cuda(cudaGetLastError(), "window attention launch: ");
}
