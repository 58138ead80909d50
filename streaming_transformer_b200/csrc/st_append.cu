// st_append.cu -- per-head norm, rotation and cache insert in one pass
// (st_cache_append), and the values 4-bit rows stand for (st_cache_unpack).
//
// One CTA takes one row (one position of one stream) with all its heads. The
// angles depend on the position alone, so each pair's cosine and sine is found
// once per row and shared by every head through shared memory: position *
// frequency / (2 pi) in 64 bits, the whole turns dropped there, and only the
// fraction goes to sincospi in fp32 (a position of 2^20 keeps an angle to
// 2^-24 turns, where an fp32 product would lose it to 2^-4).
// A head's row is a group of lanes with 8 columns each; the mean square is a
// shuffle sum inside the group. Every row is read once and written once: the
// bound is memory. The first rows of every group are on their way before the
// CTA knows whose they are.
#include "st_cache.cuh"
#include "st_cache_host.h"

namespace st {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kMaxPairs = ST_CACHE_MAX_HEAD_DIM / 2;

struct AppendArgs {
  void* q; void* k; void* v; void* q_out; void* k_out;
  long long q_row, q_head, k_row, k_head, v_row, v_head, qo_row, qo_head, ko_row, ko_head;  // elements
  void* keys; void* values;
  unsigned* key_scales; unsigned* value_scales;
  long long stream_stride, head_stride;  // cache rows
  const float* q_gain; const float* k_gain;
  const double* frequencies;
  const long long* positions;
  const int* starts;
  int rows, streams, heads, kv_heads, head_dim, rotary, sinks, window;
  float epsilon, per_column;  // per_column: 1 / head_dim
};

// 8 columns as they were loaded.
template <typename T>
struct Raw8 {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
  }
};
constexpr int kAhead = 3;  // rows a group of lanes loads ahead of their use

template <typename T, int LANES, bool INT4>
__global__ void __launch_bounds__(kAppendThreads, 5) k_cache_append(const AppendArgs a) {
  __shared__ alignas(16) float2 turn[kMaxPairs];
  __shared__ int sh_slot;
  const int row = blockIdx.x, tid = threadIdx.x;
  constexpr int kGroups = kAppendThreads / LANES;
  const int lane = tid % LANES, col = lane * 8;
  const unsigned mask = LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u) << ((tid & 31) / LANES * LANES);
  const bool on = col < a.head_dim;
  const int tasks = a.heads + 2 * a.kv_heads;
  // task: a query head, then the key heads, then the value heads
  const T* const q_row = static_cast<const T*>(a.q) + row * a.q_row + col;
  const T* const k_row = static_cast<const T*>(a.k) + row * a.k_row + col;
  const T* const v_row = static_cast<const T*>(a.v) + row * a.v_row + col;
  auto source = [&](int task) {
    const int k = task - a.heads, v = k - a.kv_heads;
    const long long stride = k < 0 ? a.q_head : v < 0 ? a.k_head : a.v_head;
    return (k < 0 ? q_row : v < 0 ? k_row : v_row) + (k < 0 ? task : v < 0 ? k : v) * stride;
  };
  Raw8<T> ahead[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    const int task = tid / LANES + u * kGroups;
    if (on && task < tasks) ahead[u].load(source(task));
  }
  // the stream that owns this row: the number of streams that end at or before it
  int stream = row, first = row, last = row + 1;
  if (a.starts) {
    // by 256 at a time: the last stream of each stretch, then the stretch that the row is in
    const int stretch = (a.streams + kAppendThreads - 1) / kAppendThreads;  // at most 256
    const int end = tid * stretch + stretch - 1;
    int ended = __syncthreads_count(end < a.streams && a.starts[end + 1] <= row);
    if (stretch > 1) {
      const int s = ended * stretch + tid;
      ended = ended * stretch + __syncthreads_count(tid < stretch && s < a.streams && a.starts[s + 1] <= row);
    }
    stream = ended;
    if (stream >= a.streams) return;  // behind the last stream
    first = clamp_row(a.starts[stream], a.rows);
    last = clamp_row(a.starts[stream + 1], a.rows);
    if (row < first || row >= last) return;  // before the first stream
  }
  const long long p0 = a.positions[stream];
  const bool idle = p0 < 0;
  const long long position = p0 + (row - first);
  for (int p = tid; p < (a.rotary + 3) / 4 * 4; p += kAppendThreads) {  // a lane's 4 pairs: those past the last turn by 0
    if (p >= a.rotary) {
      turn[p] = make_float2(1.f, 0.f);
      continue;
    }
    const double t = (double)position * a.frequencies[p] * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(2.f * (float)(t - rint(t)), &s, &c);
    turn[p] = make_float2(c, s);
  }
  if (tid == kAppendThreads - 1) {  // in a warp that has no pairs, mostly
    // inserted: sink positions, and those the stream's last `window` rows hold
    const long long newest = p0 + (last - 1 - first);
    int slot = -1;
    if (!idle && position >= 0) {  // a sum past 2^63 is not inserted
      if (position < a.sinks) slot = (int)position;
      else if (position > newest - a.window) slot = a.sinks + (int)((position - a.sinks) % a.window);
    }
    sh_slot = slot;
  }
  __syncthreads();
  const int slot = sh_slot;
  for (int first = tid / LANES; first < tasks; first += kAhead * kGroups) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int task = first + u * kGroups;
      if (task >= tasks) break;
      const bool is_q = task < a.heads, is_v = task >= a.heads + a.kv_heads;
      const int head = is_q ? task : is_v ? task - a.heads - a.kv_heads : task - a.heads;
      float f[8] = {};
      if (on && !idle) load8(reinterpret_cast<const T*>(ahead[u].u), f);
      if (on && task + kAhead * kGroups < tasks) ahead[u].load(source(task + kAhead * kGroups));
      if (!is_v && !idle) {
        const float* gain = is_q ? a.q_gain : a.k_gain;
        if (gain) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) sum = fmaf(f[i], f[i], sum);
#pragma unroll
          for (int o = 1; o < LANES; o *= 2) sum += __shfl_xor_sync(mask, sum, o);
          const float scale = rsqrtf(fmaf(sum, a.per_column, a.epsilon));
          if (on) {
            float g[8];
            load8(gain + col, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = f[i] * scale * g[i];
          }
        }
        if (col / 2 < a.rotary) {
          const float4* w = reinterpret_cast<const float4*>(&turn[col / 2]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float4 t = w[i];
            const float x0 = f[4 * i], y0 = f[4 * i + 1], x1 = f[4 * i + 2], y1 = f[4 * i + 3];
            f[4 * i] = x0 * t.x - y0 * t.y;
            f[4 * i + 1] = x0 * t.y + y0 * t.x;
            f[4 * i + 2] = x1 * t.z - y1 * t.w;
            f[4 * i + 3] = x1 * t.w + y1 * t.z;
          }
        }
      }
      if (is_q) {
        if (on) store8(static_cast<T*>(a.q_out) + row * a.qo_row + head * a.qo_head + col, f);
        continue;
      }
      if (!is_v && a.k_out && on) store8(static_cast<T*>(a.k_out) + row * a.ko_row + head * a.ko_head + col, f);
      if (slot < 0) continue;
      const long long at = stream * a.stream_stride + head * a.head_stride + slot;
      if (INT4) {
        unsigned pair;
        const unsigned codes = encode8(f, mask, &pair);
        if (on) {
          static_cast<unsigned*>(is_v ? a.values : a.keys)[at * (a.head_dim / 8) + lane] = codes;
          if (lane % 4 == 0) (is_v ? a.value_scales : a.key_scales)[at * (a.head_dim / 32) + lane / 4] = pair;
        }
      } else if (on) {
        store8(static_cast<T*>(is_v ? a.values : a.keys) + at * a.head_dim + col, f);
      }
    }
  }
}

template <typename T, bool INT4>
void launch_append(const AppendArgs& a, cudaStream_t s) {
  switch (lanes_per_row(a.head_dim)) {
    case 1: if constexpr (!INT4) k_cache_append<T, 1, INT4><<<a.rows, kAppendThreads, 0, s>>>(a); break;
    case 2: if constexpr (!INT4) k_cache_append<T, 2, INT4><<<a.rows, kAppendThreads, 0, s>>>(a); break;
    case 4: k_cache_append<T, 4, INT4><<<a.rows, kAppendThreads, 0, s>>>(a); break;
    case 8: k_cache_append<T, 8, INT4><<<a.rows, kAppendThreads, 0, s>>>(a); break;
    case 16: k_cache_append<T, 16, INT4><<<a.rows, kAppendThreads, 0, s>>>(a); break;
    default: k_cache_append<T, 32, INT4><<<a.rows, kAppendThreads, 0, s>>>(a); break;
  }
}

struct UnpackArgs {
  const unsigned* codes[2];
  const unsigned* scales[2];
  void* out[2];
  long long stream_stride, head_stride;
  int heads, slots, pieces;  // pieces: of 8 columns, per row
};

// A thread takes 8 columns of a key row and of the value row beside it.
template <typename T>
__global__ void __launch_bounds__(256) k_cache_unpack(const UnpackArgs a) {
  const long long begin = blockIdx.x * 256ll;
  const int head = blockIdx.y, stream = blockIdx.z;
  const int slot0 = (int)(begin / a.pieces), local = (int)(begin - (long long)slot0 * a.pieces) + threadIdx.x;
  const int slot = slot0 + local / a.pieces, piece = local % a.pieces;
  if (slot >= a.slots) return;
  const long long at = stream * a.stream_stride + head * a.head_stride + slot;
  const long long to = (((long long)stream * a.heads + head) * a.slots + slot) * a.pieces + piece;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    float f[8];
    decode8(a.codes[side][at * a.pieces + piece], a.scales[side][at * (a.pieces / 4) + piece / 4], f);
    store8(static_cast<T*>(a.out[side]) + to * 8, f);
  }
}

}  // namespace
}  // namespace st

using namespace st;

extern "C" {

int st_cache_append(const st_cache* c, const st_append* p, void* stream) {
  int rc = check_cache(c, true);
  if (rc != ST_OK) return rc;
  if (!p) return cache_fail(ST_ERR_INVALID, "null arguments");
  if (p->mode < ST_MODE_FP32 || p->mode > ST_MODE_BF16) return cache_fail(ST_ERR_INVALID, "unknown row mode");
  if (c->type == ST_CACHE_INT4 ? p->mode == ST_MODE_FP32 : p->mode != c->type)
    return cache_fail(ST_ERR_INVALID, "rows are of the cache's type, or fp16 or bf16 for a 4-bit cache");
  if (p->heads < 1 || p->heads > 65535) return cache_fail(ST_ERR_INVALID, "query heads are 1 to 65535");
  if (p->rows < 0 || p->rows > INT32_MAX) return cache_fail(ST_ERR_INVALID, "rows are 0 to 2^31 - 1");
  if (!p->starts && p->rows != c->streams)
    return cache_fail(ST_ERR_INVALID, "without starts there is one row for each stream");
  if (p->rows == 0) return ST_OK;
  if ((rc = check_rows(p->q, "q", p->mode, p->rows, p->heads, c->head_dim, false)) != ST_OK ||
      (rc = check_rows(p->k, "k", p->mode, p->rows, c->heads, c->head_dim, false)) != ST_OK ||
      (rc = check_rows(p->v, "v", p->mode, p->rows, c->heads, c->head_dim, false)) != ST_OK ||
      (rc = check_rows(p->q_out, "q_out", p->mode, p->rows, p->heads, c->head_dim, true)) != ST_OK ||
      (p->k_out.data && (rc = check_rows(p->k_out, "k_out", p->mode, p->rows, c->heads, c->head_dim, true)) != ST_OK))
    return rc;
  if (!p->positions) return cache_fail(ST_ERR_INVALID, "null positions");
  if (!(p->epsilon >= 0.f) || p->epsilon > 3.0e38f) return cache_fail(ST_ERR_INVALID, "epsilon must be finite and >= 0");
  if (p->rotary < 0 || p->rotary > c->head_dim / 2 || (p->rotary && !p->frequencies))
    return cache_fail(ST_ERR_INVALID, "rotary is 0 to head_dim / 2, with a frequency for each");
  for (const float* g : {p->q_gain, p->k_gain})
    if (reinterpret_cast<uintptr_t>(g) % 16) return cache_fail(ST_ERR_INVALID, "gains must start on a 16-byte boundary");
  DeviceScope scope(c->device);
  if (scope.status() != ST_OK) return scope.status();
  AppendArgs a{};
  a.q = p->q.data; a.k = p->k.data; a.v = p->v.data; a.q_out = p->q_out.data; a.k_out = p->k_out.data;
  a.q_row = p->q.row_stride; a.q_head = p->q.head_stride;
  a.k_row = p->k.row_stride; a.k_head = p->k.head_stride;
  a.v_row = p->v.row_stride; a.v_head = p->v.head_stride;
  a.qo_row = p->q_out.row_stride; a.qo_head = p->q_out.head_stride;
  a.ko_row = p->k_out.row_stride; a.ko_head = p->k_out.head_stride;
  a.keys = c->keys; a.values = c->values;
  a.key_scales = static_cast<unsigned*>(c->key_scales); a.value_scales = static_cast<unsigned*>(c->value_scales);
  a.stream_stride = c->stream_stride; a.head_stride = c->head_stride;
  a.q_gain = p->q_gain; a.k_gain = p->k_gain; a.frequencies = p->frequencies;
  a.positions = reinterpret_cast<const long long*>(p->positions); a.starts = p->starts;
  a.rows = (int)p->rows; a.streams = c->streams; a.heads = p->heads; a.kv_heads = c->heads;
  a.head_dim = c->head_dim; a.rotary = p->rotary; a.sinks = c->sinks; a.window = c->window; a.epsilon = p->epsilon;
  a.per_column = 1.0f / (float)c->head_dim;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool four = c->type == ST_CACHE_INT4;
  if (p->mode == ST_MODE_FP32) launch_append<float, false>(a, s);
  else if (p->mode == ST_MODE_FP16) four ? launch_append<__half, true>(a, s) : launch_append<__half, false>(a, s);
  else four ? launch_append<__nv_bfloat16, true>(a, s) : launch_append<__nv_bfloat16, false>(a, s);
  return cache_cuda(cudaGetLastError(), "append launch: ");
}

int st_cache_unpack(const st_cache* c, int mode, void* keys, void* values, void* stream) {
  int rc = check_cache(c, false);
  if (rc != ST_OK) return rc;
  if (c->type != ST_CACHE_INT4) return cache_fail(ST_ERR_INVALID, "only a 4-bit cache is unpacked");
  if (mode < ST_MODE_FP32 || mode > ST_MODE_BF16) return cache_fail(ST_ERR_INVALID, "unknown row mode");
  if (!keys || !values) return cache_fail(ST_ERR_INVALID, "null pointer");
  if (reinterpret_cast<uintptr_t>(keys) % 16 || reinterpret_cast<uintptr_t>(values) % 16)
    return cache_fail(ST_ERR_INVALID, "outputs must start on a 16-byte boundary");
  DeviceScope scope(c->device);
  if (scope.status() != ST_OK) return scope.status();
  UnpackArgs a{};
  a.codes[0] = static_cast<const unsigned*>(c->keys); a.codes[1] = static_cast<const unsigned*>(c->values);
  a.scales[0] = static_cast<const unsigned*>(c->key_scales); a.scales[1] = static_cast<const unsigned*>(c->value_scales);
  a.out[0] = keys; a.out[1] = values;
  a.stream_stride = c->stream_stride; a.head_stride = c->head_stride;
  a.heads = c->heads; a.slots = c->sinks + c->window; a.pieces = c->head_dim / 8;
  const dim3 grid((unsigned)(((long long)a.slots * a.pieces + 255) / 256), c->heads, c->streams);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (mode == ST_MODE_FP32) k_cache_unpack<float><<<grid, 256, 0, s>>>(a);
  else if (mode == ST_MODE_FP16) k_cache_unpack<__half><<<grid, 256, 0, s>>>(a);
  else k_cache_unpack<__nv_bfloat16><<<grid, 256, 0, s>>>(a);
  return cache_cuda(cudaGetLastError(), "unpack launch: ");
}

}  // extern "C"
