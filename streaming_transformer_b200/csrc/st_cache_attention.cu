// st_cache_attention.cu -- one query row per stream over its cache
// (st_cache_attention).
//
// Softmax in one pass: a group of lanes takes a slot, its running maximum m,
// sum l and weighted values are fp32, and groups, then warps, are merged with
// exp(m - max m) at the end.
#include "st_cache.cuh"
#include "st_cache_host.h"

namespace st {
namespace {

constexpr int kAttendThreads = 128;

struct AttendArgs {
  const void* q; void* out;
  long long q_row, q_head, o_row, o_head;  // elements
  const void* keys; const void* values;
  const unsigned* key_scales; const unsigned* value_scales;
  long long stream_stride, head_stride;  // cache rows
  const long long* positions;
  int streams, heads, kv_heads, head_dim, slots;
  float scale;
};

template <typename T, int LANES, bool INT4>
__device__ __forceinline__ void load_row8(const void* rows, const unsigned* scales, long long at, int lane, int head_dim,
                                          float (&f)[8]) {
  if (INT4)
    decode8(static_cast<const unsigned*>(rows)[at * (head_dim / 8) + lane], scales[at * (head_dim / 32) + lane / 4], f);
  else
    load8(static_cast<const T*>(rows) + at * head_dim + lane * 8, f);
}

template <typename T, int LANES, bool INT4>
__global__ void __launch_bounds__(kAttendThreads) k_cache_attention(const AttendArgs a) {
  constexpr int kGroups = kAttendThreads / LANES;
  __shared__ float sh_m[kGroups], sh_l[kGroups], sh_acc[kGroups][LANES * 8];
  const int h = blockIdx.x, stream = blockIdx.y, kv = h / (a.heads / a.kv_heads);
  const int group = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const bool on = lane * 8 < a.head_dim;
  const int seen = slots_seen(a.positions[stream], a.slots);
  float q[8] = {}, acc[8] = {}, m = -INFINITY, l = 0.f;
  if (on) load8(static_cast<const T*>(a.q) + stream * a.q_row + h * a.q_head + lane * 8, q);
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] *= a.scale;
  const long long base = stream * a.stream_stride + kv * a.head_stride;
  for (int first = 0; first < seen; first += kGroups) {
    const int slot = first + group;
    float k[8] = {}, v[8] = {}, dot = 0.f;
    if (on && slot < seen) {
      load_row8<T, LANES, INT4>(a.keys, a.key_scales, base + slot, lane, a.head_dim, k);
      load_row8<T, LANES, INT4>(a.values, a.value_scales, base + slot, lane, a.head_dim, v);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) dot = fmaf(q[i], k[i], dot);
#pragma unroll
    for (int o = 1; o < LANES; o *= 2) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (slot >= seen) continue;  // only in the last pass
    const float top = fmaxf(m, dot), keep = top == -INFINITY ? 1.f : __expf(m - top);
    const float p = __expf(dot - (top == -INFINITY ? 0.f : top));  // a NaN stays one
    m = top;
    l = fmaf(l, keep, p);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(acc[i], keep, p * v[i]);
  }
  if (lane == 0) {
    sh_m[group] = m;
    sh_l[group] = l;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) sh_acc[group][lane * 8 + i] = acc[i];
  __syncthreads();
  for (int d = threadIdx.x; d < a.head_dim; d += kAttendThreads) {
    float top = -INFINITY, sum = 0.f, o = 0.f;
    for (int g = 0; g < kGroups; ++g) top = fmaxf(top, sh_m[g]);
    for (int g = 0; g < kGroups; ++g) {
      const float w = sh_m[g] == -INFINITY ? 0.f : __expf(sh_m[g] - top);
      sum = fmaf(sh_l[g], w, sum);
      o = fmaf(sh_acc[g][d], w, o);
    }
    static_cast<T*>(a.out)[stream * a.o_row + h * a.o_head + d] = static_cast<T>(sum > 0.f ? o / sum : seen ? NAN : 0.f);
  }
}

template <typename T, bool INT4>
void launch_attention(const AttendArgs& a, cudaStream_t s) {
  const dim3 grid(a.heads, a.streams);
  switch (lanes_per_row(a.head_dim)) {
    case 1: if constexpr (!INT4) k_cache_attention<T, 1, INT4><<<grid, kAttendThreads, 0, s>>>(a); break;
    case 2: if constexpr (!INT4) k_cache_attention<T, 2, INT4><<<grid, kAttendThreads, 0, s>>>(a); break;
    case 4: k_cache_attention<T, 4, INT4><<<grid, kAttendThreads, 0, s>>>(a); break;
    case 8: k_cache_attention<T, 8, INT4><<<grid, kAttendThreads, 0, s>>>(a); break;
    case 16: k_cache_attention<T, 16, INT4><<<grid, kAttendThreads, 0, s>>>(a); break;
    default: k_cache_attention<T, 32, INT4><<<grid, kAttendThreads, 0, s>>>(a); break;
  }
}

int check_heads(const st_cache* c, int heads) {
  return heads < 1 || heads > 65535 || heads % c->heads
             ? cache_fail(ST_ERR_INVALID, "query heads are a multiple of the cache's heads, up to 65535") : ST_OK;
}

}  // namespace
}  // namespace st

using namespace st;

extern "C" {

int st_cache_attention_workspace(const st_cache* c, int heads, size_t* bytes) {
  int rc = check_cache(c, false);
  if (rc != ST_OK || (rc = check_heads(c, heads)) != ST_OK) return rc;
  if (!bytes) return cache_fail(ST_ERR_INVALID, "null pointer");
  *bytes = 0;
  return ST_OK;
}

int st_cache_attention(const st_cache* c, const st_attend* p, void* stream) {
  int rc = check_cache(c, false);
  if (rc != ST_OK) return rc;
  if (!p) return cache_fail(ST_ERR_INVALID, "null arguments");
  if (p->mode < ST_MODE_FP32 || p->mode > ST_MODE_BF16) return cache_fail(ST_ERR_INVALID, "unknown row mode");
  if (c->type == ST_CACHE_INT4 ? p->mode == ST_MODE_FP32 : p->mode != c->type)
    return cache_fail(ST_ERR_INVALID, "rows are of the cache's type, or fp16 or bf16 for a 4-bit cache");
  if ((rc = check_heads(c, p->heads)) != ST_OK ||
      (rc = check_rows(p->q, "q", p->mode, c->streams, p->heads, c->head_dim, false)) != ST_OK ||
      (rc = check_rows(p->out, "out", p->mode, c->streams, p->heads, c->head_dim, true)) != ST_OK)
    return rc;
  if (!p->positions) return cache_fail(ST_ERR_INVALID, "null positions");
  if (!(p->scale > -3.0e38f && p->scale < 3.0e38f)) return cache_fail(ST_ERR_INVALID, "scale must be finite");
  DeviceScope scope(c->device);
  if (scope.status() != ST_OK) return scope.status();
  AttendArgs a{};
  a.q = p->q.data; a.out = p->out.data;
  a.q_row = p->q.row_stride; a.q_head = p->q.head_stride;
  a.o_row = p->out.row_stride; a.o_head = p->out.head_stride;
  a.keys = c->keys; a.values = c->values;
  a.key_scales = static_cast<const unsigned*>(c->key_scales);
  a.value_scales = static_cast<const unsigned*>(c->value_scales);
  a.stream_stride = c->stream_stride; a.head_stride = c->head_stride;
  a.positions = reinterpret_cast<const long long*>(p->positions);
  a.streams = c->streams; a.heads = p->heads; a.kv_heads = c->heads; a.head_dim = c->head_dim;
  a.slots = c->sinks + c->window;
  a.scale = p->scale;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool four = c->type == ST_CACHE_INT4;
  if (p->mode == ST_MODE_FP32) launch_attention<float, false>(a, s);
  else if (p->mode == ST_MODE_FP16) four ? launch_attention<__half, true>(a, s) : launch_attention<__half, false>(a, s);
  else four ? launch_attention<__nv_bfloat16, true>(a, s) : launch_attention<__nv_bfloat16, false>(a, s);
  return cache_cuda(cudaGetLastError(), "cache attention launch: ");
}

}  // extern "C"
