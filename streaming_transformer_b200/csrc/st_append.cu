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
// shuffle sum inside the group. Every row that a result or a slot needs is read
// once and written once. 8192 fp32 rows of 8 streams, 32 and 8 heads of 128, take
// 68 us if all are inserted (window 4096), 0.90 of the copy bandwidth, and 57 with
// a window of 512. 16-bit rows are bound by instructions, as 8 columns
// cost as many whatever their type: 16384 take 79 to 82 us if all are inserted, and
// 66 with a window of 512 (72 into 4-bit rows).
// All that a CTA needs is on its way before it knows whose its row is.
#include "st_cache.cuh"
#include "st_cache_host.h"

namespace st {
namespace {

constexpr int kMaxPairs = ST_CACHE_MAX_HEAD_DIM / 2;

struct AppendArgs {
  void* q; void* k; void* v; void* q_out; void* k_out;
  long long q_row, k_row, v_row, qo_row, ko_row;  // elements
  // pieces of 16 bytes: a head's address is then one multiply-add of 32 bits (16384 16-bit rows: 82.3 us from 64-bit
  // strides, 79.3)
  int q_head, k_head, v_head, qo_head, ko_head;
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
  uint4 u[sizeof(T) / 2] = {};
  __device__ __forceinline__ void load(const uint4* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = p[i];
  }
};

template <typename T, int LANES, bool INT4, int THREADS>
__global__ void __launch_bounds__(THREADS, 1280 / THREADS) k_cache_append(const AppendArgs a) {
  // of every 8 columns the first half in one list and the second in another, which a warp reads without bank conflicts:
  // cosine and sine of 2 pairs, gains of 4 columns
  __shared__ float4 turn[2][kMaxPairs / 4], gains[2][2][kMaxPairs / 4];
  __shared__ long long sh_position;
  __shared__ int sh_stream, sh_first, sh_last, sh_slot;
  const int row = blockIdx.x, tid = threadIdx.x;
  constexpr int kGroups = THREADS / LANES;
  // Rows a group of lanes loads ahead of their use, and copies of the loop's body. With 3 the instruction cache misses
  // (8192 fp32 rows 58.5 us, with 3 60.7) or registers run short (256 fp32 rows 3.4 and 3.9).
  constexpr int kAhead = 2;
  static_assert(kMaxPairs <= THREADS && ST_CACHE_MAX_HEAD_DIM / 2 <= THREADS, "a thread for each pair, and for each 4 gains");
  const int lane = tid % LANES, col = lane * 8;
  const unsigned mask = LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u) << ((tid & 31) / LANES * LANES);
  const bool on = col < a.head_dim;
  const int tasks = a.heads + 2 * a.kv_heads;
  // task: a query head, then the key heads, then the value heads
  auto at_row = [&](const void* rows, long long stride) {  // this thread's columns of head 0
    return reinterpret_cast<const uint4*>(static_cast<const T*>(rows) + row * stride + col);
  };
  const uint4 *const q_row = at_row(a.q, a.q_row), *const k_row = at_row(a.k, a.k_row), *const v_row = at_row(a.v, a.v_row);
  auto source = [&](int task) {
    const int k = task - a.heads, v = k - a.kv_heads;
    const int stride = k < 0 ? a.q_head : v < 0 ? a.k_head : a.v_head;
    return (k < 0 ? q_row : v < 0 ? k_row : v_row) + (long long)(k < 0 ? task : v < 0 ? k : v) * stride;
  };
  auto result = [&](void* rows, long long row_stride, int head, int stride) {
    return reinterpret_cast<T*>(const_cast<uint4*>(at_row(rows, row_stride)) + (long long)head * stride);
  };
  Raw8<T> ahead[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    const int task = tid / LANES + u * kGroups;
    if (on && task < tasks) ahead[u].load(source(task));
  }
  // What else the row needs is loaded beside them, each value by the thread that may use it, so that the CTA waits for
  // memory once.
  const double frequency = tid < a.rotary ? a.frequencies[tid] : 0.0;
  const int side = tid >= a.head_dim / 4, gain_col = (tid - side * (a.head_dim / 4)) * 4;
  const float* const gain = side ? a.k_gain : a.q_gain;
  const bool has_gain = gain && gain_col < a.head_dim;
  float4 gain4;
  if (has_gain) gain4 = *reinterpret_cast<const float4*>(gain + gain_col);
  // the stream that owns this row
  int stream = row, first = row, last = row + 1;
  long long p0;
  if (a.starts) {
    // one of the first THREADS, or of the stretch of so many that lies behind all that end at or before this row
    int base = 0, span = a.streams;
    while (span > THREADS) {
      span = (span + THREADS - 1) / THREADS;
      const int end = base + tid * span + span - 1;
      base += __syncthreads_count(end < a.streams && a.starts[end + 1] <= row) * span;
    }
    const int s = base + tid;
    bool mine = false;
    if (tid < span && s < a.streams) {
      const int from = a.starts[s], to = a.starts[s + 1];
      const long long position = a.positions[s];
      mine = from <= row && row < to;
      if (mine) {
        sh_stream = s;
        sh_first = clamp_row(from, a.rows);
        sh_last = clamp_row(to, a.rows);
        sh_position = position;
      }
    }
    if (!__syncthreads_or(mine)) return;  // a row of no stream
    stream = sh_stream;
    first = sh_first;
    last = sh_last;
    p0 = sh_position;
  } else {
    p0 = a.positions[row];
  }
  if (p0 < 0) {  // idle
    const float zeros[8] = {};
    for (int task = tid / LANES; on && task < a.heads + (a.k_out ? a.kv_heads : 0); task += kGroups)
      store8(task < a.heads ? result(a.q_out, a.qo_row, task, a.qo_head)
                            : result(a.k_out, a.ko_row, task - a.heads, a.ko_head), zeros);
    return;
  }
  const long long position = p0 + (row - first);
  auto pair_turn = [&](int p) -> float2& { return reinterpret_cast<float2*>(&turn[p / 2 % 2][p / 4])[p % 2]; };
  if (has_gain) gains[side][gain_col / 4 % 2][gain_col / 8] = gain4;
  if (tid < a.rotary) {
    const double t = (double)position * frequency * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(2.f * (float)(t - rint(t)), &s, &c);
    pair_turn(tid) = make_float2(c, s);
  }
  if (tid == THREADS - 1) {  // in a warp that has no pairs, mostly
    // inserted: sink positions, and those the stream's last `window` rows hold
    const long long newest = p0 + (last - 1 - first);
    int slot = -1;
    if (position >= 0) {  // a sum past 2^63 is not inserted
      if (position < a.sinks) slot = (int)position;
      else if (position > newest - a.window) slot = a.sinks + (int)((position - a.sinks) % a.window);
    }
    sh_slot = slot;
  }
  __syncthreads();
  const int slot = sh_slot;
  // A row that is not inserted has no use for its values, nor for keys that are not asked for (16384 rows, a quarter of
  // them inserted: 65.5 us, with the loads 79.3, of which conditions that this loop no longer has took 2).
  const int end = slot >= 0 ? tasks : a.heads + (a.k_out ? a.kv_heads : 0), turns = a.rotary - col / 2;
  for (int next = tid / LANES; next < end; next += kAhead * kGroups) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int task = next + u * kGroups;
      if (task >= end) break;
      const bool is_q = task < a.heads, is_v = task >= a.heads + a.kv_heads;
      const int head = is_q ? task : is_v ? task - a.heads - a.kv_heads : task - a.heads;
      float f[8];  // zeros past head_dim
      load8(reinterpret_cast<const T*>(ahead[u].u), f);
      if (on && task + kAhead * kGroups < end) ahead[u].load(source(task + kAhead * kGroups));
      if (!is_v) {
        if (is_q ? a.q_gain : a.k_gain) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) sum = fmaf(f[i], f[i], sum);
#pragma unroll
          for (int o = 1; o < LANES; o *= 2) sum += __shfl_xor_sync(mask, sum, o);
          const float scale = rsqrtf(fmaf(sum, a.per_column, a.epsilon));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float4 g = gains[!is_q][i][lane];
            f[4 * i] *= scale * g.x;
            f[4 * i + 1] *= scale * g.y;
            f[4 * i + 2] *= scale * g.z;
            f[4 * i + 3] *= scale * g.w;
          }
        }
        auto rotate = [&](int pair, float c, float s) {
          const float x = f[2 * pair], y = f[2 * pair + 1];
          f[2 * pair] = x * c - y * s;
          f[2 * pair + 1] = x * s + y * c;
        };
        if (turns >= 4) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float4 t = turn[i][lane];
            rotate(2 * i, t.x, t.y);
            rotate(2 * i + 1, t.z, t.w);
          }
        } else if (turns > 0) {  // the lane where the rotated columns end
#pragma unroll
          for (int i = 0; i < 3; ++i)
            if (i < turns) rotate(i, pair_turn(col / 2 + i).x, pair_turn(col / 2 + i).y);
        }
      }
      if (is_q) {
        if (on) store8(result(a.q_out, a.qo_row, head, a.qo_head), f);
        continue;
      }
      if (!is_v && a.k_out && on) store8(result(a.k_out, a.ko_row, head, a.ko_head), f);
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

// Rows that are resident all at once, 5 CTAs on each of 148 SMs, have 256 threads each: fewer heads one after another
// (16 heads of 64, 256 rows: 2.8 us, with 128 threads 3.2; 700: 4.0 and 4.1). More rows have 128, as a CTA's threads
// wait together for what it does once (1000 rows: 4.5 us, with 256 threads 5.4; 3000: 11.3 and 13.5).
constexpr int kFewRows = 5 * 148;

template <typename T, bool INT4, int THREADS>
void launch_append(const AppendArgs& a, cudaStream_t s) {
  switch (lanes_per_row(a.head_dim)) {
    case 1: if constexpr (!INT4) k_cache_append<T, 1, INT4, THREADS><<<a.rows, THREADS, 0, s>>>(a); break;
    case 2: if constexpr (!INT4) k_cache_append<T, 2, INT4, THREADS><<<a.rows, THREADS, 0, s>>>(a); break;
    case 4: k_cache_append<T, 4, INT4, THREADS><<<a.rows, THREADS, 0, s>>>(a); break;
    case 8: k_cache_append<T, 8, INT4, THREADS><<<a.rows, THREADS, 0, s>>>(a); break;
    case 16: k_cache_append<T, 16, INT4, THREADS><<<a.rows, THREADS, 0, s>>>(a); break;
    default: k_cache_append<T, 32, INT4, THREADS><<<a.rows, THREADS, 0, s>>>(a); break;
  }
}
template <typename T, bool INT4>
void launch_append(const AppendArgs& a, cudaStream_t s) {
  a.rows <= kFewRows ? launch_append<T, INT4, 256>(a, s) : launch_append<T, INT4, 128>(a, s);
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
  if ((rc = check_aligned(p->positions, "positions", 8)) != ST_OK || (rc = check_aligned(p->starts, "starts", 4)) != ST_OK ||
      (rc = check_aligned(p->rotary ? p->frequencies : nullptr, "frequencies", 8)) != ST_OK)
    return rc;
  for (const float* g : {p->q_gain, p->k_gain})
    if (reinterpret_cast<uintptr_t>(g) % 16) return cache_fail(ST_ERR_INVALID, "gains must start on a 16-byte boundary");
  AppendArgs a{};
  a.q = p->q.data; a.k = p->k.data; a.v = p->v.data; a.q_out = p->q_out.data; a.k_out = p->k_out.data;
  const int per = p->mode == ST_MODE_FP32 ? 4 : 8;
  const struct { const st_rows* rows; int heads; long long* row; int* head; const char* name; } sides[] = {
      {&p->q, p->heads, &a.q_row, &a.q_head, "q"}, {&p->k, c->heads, &a.k_row, &a.k_head, "k"},
      {&p->v, c->heads, &a.v_row, &a.v_head, "v"}, {&p->q_out, p->heads, &a.qo_row, &a.qo_head, "q_out"},
      {&p->k_out, c->heads, &a.ko_row, &a.ko_head, "k_out"}};
  for (const auto& x : sides) {
    if (!x.rows->data) continue;  // no k_out
    const long long stride = x.heads > 1 ? x.rows->head_stride / per : 0;
    if (stride > INT32_MAX) return cache_fail(ST_ERR_INVALID, ": head strides are up to 2^31 - 1 times 16 bytes", x.name);
    *x.row = x.rows->row_stride;
    *x.head = (int)stride;
  }
  DeviceScope scope(c->device);
  if (scope.status() != ST_OK) return scope.status();
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
