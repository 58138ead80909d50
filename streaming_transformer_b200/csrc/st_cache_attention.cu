// st_cache_attention.cu -- one query row per stream over its cache
// (st_cache_attention).
//
// The bound is memory: every seen key and value row has to be read, and each
// byte of a 16-bit row meets one multiply-add per query head of its group. A
// kernel for a head alone would read the rows once per head, so a CTA takes all
// query heads of a key head, up to 16 (8 past 128 columns, 4 of fp32 rows); more
// are dealt to CTAs that each read the rows. 16-bit and 4-bit rows
// go through mma.sync: a tile of 16 slots is only 16 x 8 x head_dim
// multiply-adds, a few percent of what even the warp-level instruction does, and
// its fragments load straight from global memory into the registers that feed
// it. (A tcgen05 tile has at least 64 rows where there are 1 to 16 heads, and
// wants both operands through shared memory.)
//
// Fragments. A 16-byte load gives a lane 8 columns of a row. The columns of a
// product may be summed in any order, so they are dealt to the k index of the
// instruction as they arrive: with lane = 4 g + t,
//   S^T = K Q^T:  lane (g, t) loads columns 32 j + 8 t .. + 7 of slots g and
//                 g + 8 (rows of A) and of query head g (column of B) alike;
//   O^T = V^T P^T: lane (g, t) loads columns 64 i + 8 g .. + 7 of slots 2 t,
//                 2 t + 1, 2 t + 8, 2 t + 9; word m of the 4 holds the value
//                 pairs of rows g and g + 8 of m-tile (i, m), so output rows are
//                 columns 64 i + 8 g + 2 m and + 1.
// S^T leaves slots in rows and heads in columns; movmatrix turns each 8 x 8
// piece of P into the B operand of the second product.
//
// That holds 4 (head_dim 128) to 2 (64) KB in flight a warp, in registers. 4-bit
// rows are too short for it: they go through a ring in shared memory, two stages
// of 16 or 32 slots for each warp, filled by 16-byte cp.async (zeros past the last
// slot). Rows there are an odd number of 16-byte units apart, so that
// neither product's reads meet in a bank.
//
// 4-bit rows: the codes enter the products as they are. A nibble in the low
// byte of a 16-bit word is that many of the type's smallest steps (c 2^-24 in
// fp16, c 2^-133 in bf16; 16 c for the byte's high nibble), which the
// instruction takes exactly, so a word of 8 codes costs four masks and a shift.
// Queries are scaled by a power of two per head beforehand so that sums come out
// as normal numbers (and by 1/16 where they meet a high nibble). A product stays
// within one group of 32 columns, whose scale and lowest value then enter in
// fp32: sum q k = scale * sum q c + lowest * sum q. For values the scale is
// folded into the weight before its one rounding, to bf16 (times 2^70: its range
// takes scales from 2^-56 to 2^56). For fp16 rows, which have 3 bits more, the
// weight is a sum of two bf16, each with a product of its own (fp16 itself has no
// room for the scales; 256 Large streams, 516 slots: 55 us, at bf16 48). Codes are 0..15 where the values lie about
// 0, so that rounding would count double; the fp32 sum beside the product takes
// p * (lowest + 7.5 scale) - 7.5 * (the rounded weight), which leaves the error
// with the code's distance from 7.5. Turning codes into 16-bit values first took
// 1.7 times the instructions, which bound the kernel (256 Large streams, 516
// slots: 58 us, now 48), and rounded each value once more.
//
// Softmax statistics are fp32: a running maximum per head (in units of log2),
// the sum of unrounded weights, and output sums. Weights are rounded to the 16
// bits that the instruction takes, relative to the running maximum; for fp16
// they are kept 2^10 higher, so that none that counts is a denormal.
//
// Split. Slots are dealt to splits x 4 warps so that all SMs pull memory at
// once; the parts of a CTA meet in shared memory, those of several CTAs in the
// workspace, where k_merge joins them in split order (no atomics: the same
// call gives the same bits). Parts follow the slots seen, which only the device
// knows; the number of splits follows the cache's size.
#include "st_cache.cuh"
#include "st_cache_host.h"

#include <algorithm>

namespace st {
namespace {

constexpr int kAttendWarps = 4;
constexpr int kAttendThreads = 32 * kAttendWarps;
constexpr float kLog2e = 1.4426950408889634f;

struct AttendArgs {
  const void* q; void* out;
  long long q_row, q_head, o_row, o_head;  // elements
  const void* keys; const void* values;
  const unsigned* key_scales; const unsigned* value_scales;
  long long stream_stride, head_stride;  // cache rows
  const long long* positions;
  float* parts;   // [stream][head][split]{m, l}, then from `sums_at` on [stream][head][split][head_dim]
  long long sums_at;  // floats, a multiple of 4
  int streams, heads, kv_heads, group, head_dim, slots, splits, blocks;  // blocks of query heads a key head
  float scale2;   // scale * log2(e)
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                    unsigned b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned transpose8x8(unsigned v) {
  unsigned r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Rows are read once: whole sectors, no place in L1.
__device__ __forceinline__ uint4 ld_row16(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
// 16, 8 or 4 bytes to shared memory, zeros unless `in`.
template <int N>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool in) {
  const unsigned to = (unsigned)__cvta_generic_to_shared(dst);
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(in ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(src), "n"(N), "r"(in ? N : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Part of this CTA's split in tiles of `tile` slots: [first, last).
__device__ __forceinline__ void split_slots(int seen, int tile, int split, int splits, int& first, int& last) {
  const int tiles = (seen + tile - 1) / tile, per = (tiles + splits - 1) / splits;
  first = (int)min((long long)seen, (long long)split * per * tile);
  last = (int)min((long long)seen, (long long)first + (long long)per * tile);
}

// Writes one head's result, or its part of it. `o` is unnormalised.
template <typename T>
__device__ __forceinline__ void put_result(const AttendArgs& a, int stream, int h, int split, int d, float m, float l,
                                           float o, int seen) {
  if (a.splits == 1) {
    static_cast<T*>(a.out)[stream * a.o_row + h * a.o_head + d] = static_cast<T>(seen ? o / l : 0.f);
    return;
  }
  const long long at = ((long long)stream * a.heads + h) * a.splits + split;
  if (d == 0) reinterpret_cast<float2*>(a.parts)[at] = make_float2(m, l);
  a.parts[a.sums_at + at * a.head_dim + d] = o;
}

__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---------------------------------------------------------------- 16-bit and 4-bit rows
// Nibbles 0 .. 3 of each half of `w`: as low-byte steps, the odd ones times 16.
__device__ __forceinline__ void code_steps(unsigned w, unsigned (&c)[4]) {
  const unsigned z = w >> 8;
  c[0] = w & 0x000f000fu; c[1] = w & 0x00f000f0u; c[2] = z & 0x000f000fu; c[3] = z & 0x00f000f0u;
}
constexpr float kValueLift = 0x1p70f, kValueDrop = 0x1p63f;  // 2^70 on the weights, 2^-133 on the codes

// Shared memory of a CTA: the warps' rings (4-bit rows), and after the loop their parts of the result.
template <int DB, int NT, bool INT4>
struct AttendSmem {
  static constexpr int kTiles = INT4 && DB * NT <= 2 ? 2 : 1;         // tiles of 16 slots in a step (or stage)
  static constexpr int kStages = 2;  // 3 and 4 stages leave room for fewer warps: 1 % and 12 % slower
  static constexpr int kRowBytes = DB * 32 + 16;                       // largest distance of 4-bit rows
  static constexpr int kScaleBytes = DB * 8;                           // largest scales of a slot
  static constexpr int kStageBytes = 16 * kTiles * 2 * (kRowBytes + kScaleBytes);
  static constexpr int kRing = INT4 ? kAttendWarps * kStages * kStageBytes : 0;
  static constexpr int kPartRow = DB * 64 + 4;                         // floats
  static constexpr int kParts = kAttendWarps * NT * 8 * kPartRow * 4;
  static constexpr int kBytes = kRing > kParts ? kRing : kParts;
};

// DB: blocks of 64 columns; NT: blocks of 8 query heads; FULL: head_dim is
// 64 DB, so that row offsets are constants and no column is checked; ONE: one
// query head a key head, so that the odd columns of S^T are not computed on.
template <typename T, int DB, int NT, bool INT4, bool FULL, bool ONE>
__global__ void __launch_bounds__(kAttendThreads, DB * NT == 1 ? (INT4 ? 7 : 6) : INT4 && DB == 2 && NT == 1 ? 3 : 1)
    k_attend_mma(const AttendArgs a) {
  constexpr int J = 2 * DB;   // 16-bit: 16-byte pieces of a key row a lane holds
  using Smem = AttendSmem<DB, NT, INT4>;
  constexpr int TS = Smem::kTiles;
  constexpr int X = ONE ? 1 : 2;  // query heads a lane has of each block: 8 n + 2 t + x
  using PT = typename std::conditional<INT4, __nv_bfloat16, T>::type;  // operands of the second product
  constexpr float kLift = std::is_same<PT, __half>::value ? 10.f : 0.f;
  constexpr bool kTwo = INT4 && std::is_same<T, __half>::value;  // 4-bit: a weight is two bf16
  extern __shared__ uint4 dynamic[];
  float(*sh_o)[NT * 8][Smem::kPartRow] = reinterpret_cast<float(*)[NT * 8][Smem::kPartRow]>(dynamic);
  __shared__ float sh_m[kAttendWarps][NT * 8], sh_l[kAttendWarps][NT * 8];
  const int split = blockIdx.x, kv = blockIdx.y / a.blocks, block = blockIdx.y % a.blocks, stream = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (a.splits > 1) let_next_kernel_start();
  const int seen = slots_seen(a.positions[stream], a.slots);
  int first, last;
  split_slots(seen, 16 * TS * kAttendWarps, split, a.splits, first, last);
  const int head0 = kv * a.group + block * NT * 8;                          // first query head of the block
  const int nheads = min(NT * 8, a.group - block * NT * 8);

  const long long row0 = stream * a.stream_stride + kv * a.head_stride;
  const int dim = FULL ? DB * 64 : a.head_dim, groups = dim / 32, row_bytes = INT4 ? dim / 2 : dim * 2;
  constexpr int kStep = 16 * TS * kAttendWarps;
  int slot0 = first + warp * 16 * TS;
  constexpr int SW = INT4 ? J : 1;

  // 4-bit rows: this warp's ring. A stage: key rows, value rows, key scales, value scales of kSlots slots.
  constexpr int kSlots = 16 * TS;
  const int row_apart = row_bytes + (row_bytes / 16 % 2 ? 0 : 16), scale_bytes = groups * 4;
  char* const ring = reinterpret_cast<char*>(dynamic) + warp * Smem::kStages * Smem::kStageBytes;
  const char* const k4 = static_cast<const char*>(a.keys) + row0 * row_bytes;
  const char* const v4 = static_cast<const char*>(a.values) + row0 * row_bytes;
  const char* const ks4 = reinterpret_cast<const char*>(a.key_scales) + row0 * scale_bytes;
  const char* const vs4 = reinterpret_cast<const char*>(a.value_scales) + row0 * scale_bytes;
  auto fill = [&](int stage, int at) {
    if (at < last) {
      char* to = ring + stage * Smem::kStageBytes;
      const int chunks = row_bytes / 16;
      const long long off = (long long)at * row_bytes;
      auto rows = [&](int c) {
        const int row = FULL ? c / (2 * DB) : c / chunks, col = FULL ? c % (2 * DB) : c - row * chunks;
        const bool in = at + row < last;
        copy_async<16>(to + row * row_apart + col * 16, k4 + (in ? off + c * 16 : 0), in);
        copy_async<16>(to + (kSlots + row) * row_apart + col * 16, v4 + (in ? off + c * 16 : 0), in);
      };
      if constexpr (FULL) {
#pragma unroll
        for (int c = 0; c < kSlots * 2 * DB; c += 32) rows(c + lane);
      } else {
        for (int c = lane; c < kSlots * chunks; c += 32) rows(c);
      }
      to += 2 * kSlots * row_apart;
      const long long soff = (long long)at * scale_bytes;
      // lanes take slots: 32 of each side, or 16 of both
      const int slot = TS == 2 ? lane : lane & 15;
      const bool in = at + slot < last;
#pragma unroll
      for (int side = 0; side < TS; ++side) {
        const bool value = TS == 2 ? side == 1 : lane >= 16;
        const char* from = (value ? vs4 : ks4) + (in ? soff + slot * scale_bytes : 0);
        char* dst = to + (value ? kSlots * scale_bytes : 0) + slot * scale_bytes;
        if constexpr (FULL) {
          constexpr int N = DB == 1 ? 8 : 16;
#pragma unroll
          for (int i = 0; i < 8 * DB; i += N) copy_async<N>(dst + i, from + i, in);
        } else {
          for (int i = 0; i < scale_bytes; i += 4) copy_async<4>(dst + i, from + i, in);
        }
      }
    }
    copy_commit();
  };
  // scales of slot `slot` of a stage's side
  auto read_scales = [&](const char* p, int slot, unsigned(&f)[SW]) {
    p += slot * scale_bytes;
    if constexpr (FULL && J == 2) {
      const uint2 w = *reinterpret_cast<const uint2*>(p);
      f[0] = w.x; f[1] = w.y;
    } else if constexpr (FULL && INT4) {
#pragma unroll
      for (int j = 0; j < J; j += 4) {
        const uint4 w = *reinterpret_cast<const uint4*>(p + 4 * j);
        f[j] = w.x; f[j + 1] = w.y; f[j + 2] = w.z; f[j + 3] = w.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < SW; ++j) f[j] = j < groups ? *reinterpret_cast<const unsigned*>(p + 4 * j) : 0u;
    }
  };

  // 16-bit rows: one tile in registers, loaded a step ahead of its use. This lane's first addresses:
  const char* kp = static_cast<const char*>(a.keys) + (row0 + slot0 + g) * row_bytes + t * 16;
  const char* vp = static_cast<const char*>(a.values) + (row0 + slot0 + 2 * t) * row_bytes + g * 16;
  unsigned kf[2][J * 4], vf[4][DB * 4];
  // Slots past `last` load nothing and count as zeros, so that no value there matters; `whole`: the step has none.
  auto load_k = [&](int at, bool whole) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const bool in = whole || at + g + 8 * r < last;
      const char* p = kp + 8 * r * row_bytes;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const uint4 w = in && (FULL || j * 32 + t * 8 < dim) ? ld_row16(p + j * 64) : make_uint4(0, 0, 0, 0);
        kf[r][4 * j] = w.x; kf[r][4 * j + 1] = w.y; kf[r][4 * j + 2] = w.z; kf[r][4 * j + 3] = w.w;
      }
    }
  };
  auto load_v = [&](int at, bool whole) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int ahead = (r & 1) + 8 * (r >> 1);
      const bool in = whole || at + 2 * t + ahead < last;
      const char* p = vp + ahead * row_bytes;
#pragma unroll
      for (int i = 0; i < DB; ++i) {
        const uint4 w = in && (FULL || i * 64 + g * 8 < dim) ? ld_row16(p + i * 128) : make_uint4(0, 0, 0, 0);
        vf[r][4 * i] = w.x; vf[r][4 * i + 1] = w.y; vf[r][4 * i + 2] = w.z; vf[r][4 * i + 3] = w.w;
      }
    }
  };
  auto fetch_k = [&](int at) {
    if (at + 16 <= last) load_k(at, true);
    else load_k(at, false);
    kp += (long long)kStep * row_bytes;
  };
  auto fetch_v = [&](int at) {
    if (at + 16 <= last) load_v(at, true);
    else load_v(at, false);
    vp += (long long)kStep * row_bytes;
  };
  if constexpr (INT4) {
#pragma unroll
    for (int i = 0; i < Smem::kStages - 1; ++i) fill(i, slot0 + i * kStep);
  } else if (slot0 < last) {
    fetch_k(slot0);
    fetch_v(slot0);
  }

  // query fragments: the columns of this lane's key words, head 8 n + g
  unsigned qf[NT][J][4];
  float qsum[NT][INT4 ? J : 1][X], scale2[NT][X];  // 4-bit, heads 8 n + 2 t + x: sum of a group's columns; units of S
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const bool head_on = n * 8 + g < nheads;
    const T* qp = static_cast<const T*>(a.q) + stream * a.q_row + (long long)(head0 + n * 8 + g) * a.q_head;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      uint4 w = make_uint4(0, 0, 0, 0);
      if (head_on && j * 32 + t * 8 < dim) w = *reinterpret_cast<const uint4*>(qp + j * 32 + t * 8);
      qf[n][j][0] = w.x; qf[n][j][1] = w.y; qf[n][j][2] = w.z; qf[n][j][3] = w.w;
    }
#pragma unroll
    for (int x = 0; x < X; ++x) scale2[n][x] = a.scale2;
    if constexpr (INT4) {
      // the largest exponent of the head, within limits that leave both factors normal numbers
      constexpr int kTop = std::is_same<T, __half>::value ? 10 : 100, kStep = std::is_same<T, __half>::value ? 24 : 133;
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float f[8];
        load8(reinterpret_cast<const T*>(qf[n][j]), f);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(f[i]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = min(max((int)(__float_as_uint(top) >> 23), 107), 220);
      const float up = __uint_as_float((unsigned)(254 + kTop - e) << 23);                // 2^kTop / 2^(e - 127)
      const float unit = __uint_as_float((unsigned)(254 + kTop - kStep - e) << 23);      // up * 2^-kStep
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float f[8], sum = 0.f;
        load8(reinterpret_cast<const T*>(qf[n][j]), f);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += f[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // columns i and i + 4 meet a word's nibbles i and i + 4
          const float by = i & 1 ? up * 0.0625f : up;
          qf[n][j][i] = pack2((T*)nullptr, f[i] * by, f[i + 4] * by);
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
        for (int x = 0; x < X; ++x) qsum[n][j][x] = __shfl_sync(0xffffffffu, sum * unit, (2 * t + x) * 4);
      }
#pragma unroll
      for (int x = 0; x < X; ++x) scale2[n][x] = a.scale2 / __shfl_sync(0xffffffffu, unit, (2 * t + x) * 4);
    }
  }

  float o[NT][DB][4][4] = {};        // [head block][column block][m-tile]
  float olow[NT][INT4 ? J : 1][X] = {};  // 4-bit: the fp32 part, over this lane's slots
  float m[NT][X], l[NT][X];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int x = 0; x < X; ++x) m[n][x] = -INFINITY, l[n][x] = 0.f;

  int stage = 0;
  for (; slot0 < last; slot0 += kStep) {
    const char* tile = ring + stage * Smem::kStageBytes;  // this step's stage
    if constexpr (INT4) {
      copy_wait<Smem::kStages - 2>();
      __syncwarp();  // everybody's copies have landed, and nobody reads the stage before this one any more
      fill(stage == 0 ? Smem::kStages - 1 : stage - 1, slot0 + (Smem::kStages - 1) * kStep);
      stage = stage + 1 == Smem::kStages ? 0 : stage + 1;
    }
    // S^T: slots g (c0, c1) and g + 8 (c2, c3) of each tile, heads 8 n + 2 t, + 1
    float s[TS][NT][4] = {};
#pragma unroll
    for (int u = 0; u < TS; ++u) {
      unsigned ks[2][SW];
      if constexpr (INT4)
#pragma unroll
        for (int r = 0; r < 2; ++r) read_scales(tile + 2 * kSlots * row_apart, 16 * u + 8 * r + g, ks[r]);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if constexpr (INT4) {
          if (!FULL && j >= groups) break;
          unsigned c[2][4];
#pragma unroll
          for (int r = 0; r < 2; ++r)
            code_steps(*reinterpret_cast<const unsigned*>(tile + (16 * u + 8 * r + g) * row_apart + j * 16 + t * 4), c[r]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            mma<T>(acc, c[0][0], c[1][0], c[0][1], c[1][1], qf[n][j][0], qf[n][j][1]);
            mma<T>(acc, c[0][2], c[1][2], c[0][3], c[1][3], qf[n][j][2], qf[n][j][3]);
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int x = 0; x < X; ++x)
                s[u][n][2 * r + x] = fmaf(acc[2 * r + x], group_scale(ks[r][j]),
                                          fmaf(group_lowest(ks[r][j]), qsum[n][j][x], s[u][n][2 * r + x]));
          }
        } else {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma<T>(s[u][n], kf[0][4 * j], kf[1][4 * j], kf[0][4 * j + 1], kf[1][4 * j + 1], qf[n][j][0], qf[n][j][1]);
            mma<T>(s[u][n], kf[0][4 * j + 2], kf[1][4 * j + 2], kf[0][4 * j + 3], kf[1][4 * j + 3], qf[n][j][2],
                   qf[n][j][3]);
          }
        }
      }
    }
    const int next = slot0 + kStep;
    if constexpr (!INT4)
      if (next < last) fetch_k(next);

    unsigned pf[TS][NT][SW][kTwo ? 4 : 2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float p[TS][2][X], top[X];
#pragma unroll
      for (int x = 0; x < X; ++x) {
        top[x] = -INFINITY;
#pragma unroll
        for (int u = 0; u < TS; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            p[u][r][x] = slot0 + g + 16 * u + 8 * r < last ? s[u][n][2 * r + x] * scale2[n][x] : -INFINITY;
            top[x] = fmaxf(top[x], p[u][r][x]);
          }
#pragma unroll
        for (int d = 4; d < 32; d *= 2) top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], d));
      }
      if (__any_sync(0xffffffffu, top[0] > m[n][0] || top[X - 1] > m[n][X - 1])) {
#pragma unroll
        for (int x = 0; x < X; ++x) {
          top[x] = fmaxf(top[x], m[n][x]);
          const float keep = top[x] == -INFINITY ? 1.f : exp2_fast(m[n][x] - top[x]);
          m[n][x] = top[x];
          l[n][x] *= keep;
#pragma unroll
          for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              o[n][i][w][x] *= keep;
              o[n][i][w][2 + x] *= keep;
            }
          if constexpr (INT4)
#pragma unroll
            for (int j = 0; j < J; ++j) olow[n][j][x] *= keep;
        }
      }
#pragma unroll
      for (int u = 0; u < TS; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          unsigned vs[SW];
          if constexpr (INT4)
            read_scales(tile + 2 * kSlots * row_apart + kSlots * scale_bytes, 16 * u + 8 * r + g, vs);
#pragma unroll
          for (int x = 0; x < X; ++x) {
            const float ref = m[n][x] == -INFINITY ? 0.f : m[n][x] - kLift;
            p[u][r][x] = exp2_fast(p[u][r][x] - ref);
            l[n][x] += p[u][r][x];
          }
          if constexpr (INT4) {
#pragma unroll
            for (int j = 0; j < J; ++j) {
              const float scale = group_scale(vs[j]), middle = fmaf(7.5f, scale, group_lowest(vs[j]));
              const unsigned w = pack2((PT*)nullptr, p[u][r][0] * (scale * kValueLift),
                                       ONE ? 0.f : p[u][r][X - 1] * (scale * kValueLift));
              pf[u][n][j][r] = transpose8x8(w);
              unsigned rest = 0;
              if constexpr (kTwo) {
                rest = pack2((PT*)nullptr, fmaf(p[u][r][0], scale * kValueLift, -group_scale(w)),
                             ONE ? 0.f : fmaf(p[u][r][X - 1], scale * kValueLift, -group_lowest(w)));
                pf[u][n][j][2 + r] = transpose8x8(rest);
              }
#pragma unroll
              for (int x = 0; x < X; ++x) {
                float rounded = x ? group_lowest(w) : group_scale(w);  // the halves of a word of two bf16
                if constexpr (kTwo) rounded += x ? group_lowest(rest) : group_scale(rest);
                olow[n][j][x] = fmaf(p[u][r][x], middle, fmaf(rounded, -7.5f / kValueLift, olow[n][j][x]));
              }
            }
          } else {
            pf[u][n][0][r] = transpose8x8(pack2((PT*)nullptr, p[u][r][0], ONE ? 0.f : p[u][r][X - 1]));
          }
        }
    }

    // O^T += V^T P^T
#pragma unroll
    for (int u = 0; u < TS; ++u) {
      if constexpr (INT4) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          // slots (2 t, 2 t + 1) and (2 t + 8, 2 t + 9) side by side; rows g and g + 8 of an m-tile: an even and an
          // odd nibble
          if (!FULL && j >= groups) break;
          const char* p = tile + (kSlots + 16 * u + 2 * t) * row_apart + j * 16 + g * 2;
          auto half = [&](int ahead) { return (unsigned)*reinterpret_cast<const unsigned short*>(p + ahead * row_apart); };
          unsigned c0[4], c1[4];
          code_steps(__byte_perm(half(0), half(1), 0x5410), c0);
          code_steps(__byte_perm(half(8), half(9), 0x5410), c1);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              mma<PT>(o[n][j / 2][2 * (j & 1) + w], c0[2 * w], c0[2 * w + 1], c1[2 * w], c1[2 * w + 1], pf[u][n][j][0],
                      pf[u][n][j][1]);
              if constexpr (kTwo)
                mma<PT>(o[n][j / 2][2 * (j & 1) + w], c0[2 * w], c0[2 * w + 1], c1[2 * w], c1[2 * w + 1], pf[u][n][j][2],
                        pf[u][n][j][3]);
            }
        }
      } else {
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            unsigned c[4];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              c[2 * r] = __byte_perm(vf[2 * r][4 * i + w], vf[2 * r + 1][4 * i + w], 0x5410);
              c[2 * r + 1] = __byte_perm(vf[2 * r][4 * i + w], vf[2 * r + 1][4 * i + w], 0x7632);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) mma<PT>(o[n][i][w], c[0], c[1], c[2], c[3], pf[u][n][0][0], pf[u][n][0][1]);
          }
      }
    }
    if constexpr (!INT4)
      if (next < last) fetch_v(next);
  }

  // this warp's part into shared memory, columns in their own order (its own ring lies elsewhere than its part)
  if constexpr (INT4) {
    copy_wait<0>();
    __syncthreads();
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int x = 0; x < X; ++x) {
      const int h = n * 8 + 2 * t + x;
      float sum = l[n][x];
#pragma unroll
      for (int d = 4; d < 32; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if constexpr (INT4)
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int d = 4; d < 32; d *= 2) olow[n][j][x] += __shfl_xor_sync(0xffffffffu, olow[n][j][x], d);
      if (h >= nheads) continue;
      if (g == 0) {
        sh_m[warp][h] = m[n][x];
        sh_l[warp][h] = sum;
      }
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          float2 v = make_float2(o[n][i][w][x], o[n][i][w][2 + x]);
          int d = i * 64 + g * 8 + 2 * w;
          if constexpr (INT4) {  // group 2 i + w / 2, columns 4 g + 2 (w % 2), + 1 (an odd nibble: 16 times as large)
            const float low = olow[n][2 * i + w / 2][x];
            v = make_float2(fmaf(v.x, kValueDrop, low), fmaf(v.y, kValueDrop * 0.0625f, low));
            d = i * 64 + (w / 2) * 32 + g * 4 + 2 * (w & 1);
          }
          *reinterpret_cast<float2*>(&sh_o[warp][h][d]) = v;
        }
    }
  __syncthreads();
  for (int e = threadIdx.x; e < nheads * dim; e += kAttendThreads) {
    const int h = e / dim, d = e - h * dim;
    float top = -INFINITY, sum = 0.f, out = 0.f;
#pragma unroll
    for (int w = 0; w < kAttendWarps; ++w) top = fmaxf(top, sh_m[w][h]);
#pragma unroll
    for (int w = 0; w < kAttendWarps; ++w) {
      const float f = sh_m[w][h] == -INFINITY ? 1.f : exp2_fast(sh_m[w][h] - top);  // an empty part is all zeros, or NaN
      sum = fmaf(sh_l[w][h], f, sum);
      out = fmaf(sh_o[w][h][d], f, out);
    }
    put_result<T>(a, stream, head0 + h, split, d, top, sum, out, seen);
  }
}

// ---------------------------------------------------------------- fp32 rows
// A group of lanes takes a slot, 8 columns a lane; GT query heads share the rows. There is no fp32 tensor
// product, and at GT = 4 the multiply-adds still fit beside the loads.
template <int LANES, int GT>
__global__ void __launch_bounds__(kAttendThreads) k_attend_fp32(const AttendArgs a) {
  constexpr int kGroups = kAttendThreads / LANES;
  __shared__ float sh_m[GT][kGroups], sh_l[GT][kGroups], sh_o[GT][kGroups][LANES * 8];
  const int split = blockIdx.x, kv = blockIdx.y / a.blocks, block = blockIdx.y % a.blocks, stream = blockIdx.z;
  const int group = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  if (a.splits > 1) let_next_kernel_start();
  const bool on = lane * 8 < a.head_dim;
  const int seen = slots_seen(a.positions[stream], a.slots);
  int first, last;
  split_slots(seen, kGroups, split, a.splits, first, last);
  const int head0 = kv * a.group + block * GT, nheads = min(GT, a.group - block * GT);
  float q[GT][8] = {}, o[GT][8] = {}, m[GT], l[GT];
#pragma unroll
  for (int h = 0; h < GT; ++h) {
    m[h] = -INFINITY;
    l[h] = 0.f;
    if (on && h < nheads) load8(static_cast<const float*>(a.q) + stream * a.q_row + (head0 + h) * a.q_head + lane * 8, q[h]);
#pragma unroll
    for (int i = 0; i < 8; ++i) q[h][i] *= a.scale2;
  }
  const long long row0 = stream * a.stream_stride + kv * a.head_stride;
  const float* kp = static_cast<const float*>(a.keys) + row0 * a.head_dim + lane * 8;
  const float* vp = static_cast<const float*>(a.values) + row0 * a.head_dim + lane * 8;
  constexpr int U = GT == 1 ? 4 : 2;   // slots a group loads before it uses them; 4 at GT 2: 31 -> 40 us at 256 streams
  for (int base = first; base < last; base += kGroups * U) {
    float k[U][8] = {}, v[U][8] = {};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long slot = base + u * kGroups + group;
      if (on && slot < last) {
        load8(kp + slot * a.head_dim, k[u]);
        load8(vp + slot * a.head_dim, v[u]);
      }
    }
#pragma unroll
    for (int h = 0; h < GT; ++h) {
      float dot[U] = {};
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < 8; ++i) dot[u] = fmaf(q[h][i], k[u][i], dot[u]);
#pragma unroll
        for (int d = 1; d < LANES; d *= 2) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], d);
        if (base + u * kGroups + group >= last) dot[u] = -INFINITY;
      }
      float top = m[h];
#pragma unroll
      for (int u = 0; u < U; ++u) top = fmaxf(top, dot[u]);
      const float ref = top == -INFINITY ? 0.f : top, keep = exp2_fast(m[h] - ref);
      m[h] = top;
      l[h] *= keep;
      float p[U];
#pragma unroll
      for (int u = 0; u < U; ++u) l[h] += p[u] = exp2_fast(dot[u] - ref);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        o[h][i] *= keep;
#pragma unroll
        for (int u = 0; u < U; ++u) o[h][i] = fmaf(p[u], v[u][i], o[h][i]);
      }
    }
  }
#pragma unroll
  for (int h = 0; h < GT; ++h) {
    if (lane == 0) {
      sh_m[h][group] = m[h];
      sh_l[h][group] = l[h];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sh_o[h][group][lane * 8 + i] = o[h][i];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < nheads * a.head_dim; e += kAttendThreads) {
    const int h = e / a.head_dim, d = e - h * a.head_dim;
    float top = -INFINITY, sum = 0.f, out = 0.f;
    for (int w = 0; w < kGroups; ++w) top = fmaxf(top, sh_m[h][w]);
    for (int w = 0; w < kGroups; ++w) {
      const float f = sh_m[h][w] == -INFINITY ? 1.f : exp2_fast(sh_m[h][w] - top);
      sum = fmaf(sh_l[h][w], f, sum);
      out = fmaf(sh_o[h][w][d], f, out);
    }
    put_result<float>(a, stream, head0 + h, split, d, top, sum, out, seen);
  }
}

// ---------------------------------------------------------------- parts of several CTAs
// One CTA joins one head of one stream: 8 warps take every eighth part, 4
// columns a lane, and meet in shared memory in warp order.
constexpr int kMergeWarps = 8;
constexpr int kMaxSplits = 1024;

template <typename T>
__global__ void __launch_bounds__(32 * kMergeWarps) k_merge(const AttendArgs a) {
  __shared__ float sh_f[kMaxSplits], sh_w[2][kMergeWarps];
  __shared__ float4 sh_o[kMergeWarps][ST_CACHE_MAX_HEAD_DIM / 4];
  const int h = blockIdx.x, stream = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seen = slots_seen(a.positions[stream], a.slots);
  const long long at = ((long long)stream * a.heads + h) * a.splits;
  const float2* ml = reinterpret_cast<const float2*>(a.parts) + at;
  const float4* part = reinterpret_cast<const float4*>(a.parts + a.sums_at + at * a.head_dim);
  const int quads = a.head_dim / 4;
  wait_for_previous_kernel();
  float top = -INFINITY, sum = 0.f;
  for (int s = threadIdx.x; s < a.splits; s += 32 * kMergeWarps) top = fmaxf(top, ml[s].x);
#pragma unroll
  for (int d = 1; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (lane == 0) sh_w[0][warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kMergeWarps; ++w) top = fmaxf(top, sh_w[0][w]);
  for (int s = threadIdx.x; s < a.splits; s += 32 * kMergeWarps) {
    const float2 p = ml[s];
    const float f = p.x == -INFINITY ? 1.f : exp2_fast(p.x - top);  // an empty part is all zeros, or NaN
    sh_f[s] = f;
    sum = fmaf(p.y, f, sum);
  }
#pragma unroll
  for (int d = 1; d < 32; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) sh_w[1][warp] = sum;
  __syncthreads();
  for (int c = lane; c < quads; c += 32) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = warp; s < a.splits; s += kMergeWarps) {
      const float4 v = __ldcg(part + (long long)s * quads + c);
      const float f = sh_f[s];
      o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
    }
    sh_o[warp][c] = o;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < a.head_dim; d += 32 * kMergeWarps) {
    float l = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) {
      l += sh_w[1][w];
      o += reinterpret_cast<const float*>(sh_o[w])[d];
    }
    static_cast<T*>(a.out)[stream * a.o_row + h * a.o_head + d] = static_cast<T>(seen ? o / l : 0.f);
  }
}

// ---------------------------------------------------------------- host
// Query heads that one CTA takes.
int heads_per_block(const st_cache* c, int heads) {
  const int group = heads / c->heads;
  if (c->type == ST_MODE_FP32) return group <= 1 ? 1 : group <= 2 ? 2 : 4;
  return group <= 8 || c->head_dim > 128 ? 8 : 16;
}

// CTAs that share the slots of one key head. One for each SM while each still has
// 64 slots, if that makes at least 6 of them; whole steps are dealt, of 64 slots
// (128 of narrow 4-bit rows), so that some parts can stay empty: 504 slots in 7
// parts are 8 steps, 2 each for 4 of them (the join costs 1.5 us: one stream of
// 16 heads, 260 slots, takes 4.6 us whole and 5.2 in 4 parts, with 504 slots 6.2
// whole and 5.2 in 7); up to 12 for each SM while each has 512, so that streams of
// uneven lengths even out (6, 8 and 12 for each SM: 64, 60 and 61 us at fp16, 129,
// 123 and 117 at 4 bits; one stream of 131076 slots 88, 92 and 93).
int splits_of(const st_cache* c, int heads) {
  const int per = heads_per_block(c, heads), group = heads / c->heads, slots = c->sinks + c->window;
  const long long ctas = (long long)c->streams * c->heads * ((group + per - 1) / per), sms = sm_count(c->device);
  long long fill = std::min<long long>(sms / ctas, slots / 64);
  if (fill < 6) fill = 1;
  const long long even = std::min<long long>(12 * sms / ctas, slots / 512);
  return (int)std::min<long long>(std::max<long long>({fill, even, 1}), kMaxSplits);
}

template <typename T, int DB, int NT, bool INT4, bool FULL, bool ONE>
void launch_one(const AttendArgs& a, dim3 grid, cudaStream_t s) {
  constexpr int kBytes = AttendSmem<DB, NT, INT4>::kBytes;
  if (kBytes > 40 * 1024)  // above what a launch may ask for by itself, with the static arrays
    cudaFuncSetAttribute(k_attend_mma<T, DB, NT, INT4, FULL, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
  k_attend_mma<T, DB, NT, INT4, FULL, ONE><<<grid, kAttendThreads, kBytes, s>>>(a);
}
template <typename T, int DB, bool INT4, bool FULL>
void launch_mma(const AttendArgs& a, int per, dim3 grid, cudaStream_t s) {
  if (a.group == 1) launch_one<T, DB, 1, INT4, FULL, true>(a, grid, s);
  else if (per == 8) launch_one<T, DB, 1, INT4, FULL, false>(a, grid, s);
  else if constexpr (DB < 4) launch_one<T, DB, 2, INT4, FULL, false>(a, grid, s);
}
template <typename T, bool INT4>
void launch_mma(const AttendArgs& a, int per, dim3 grid, cudaStream_t s) {
  if (a.head_dim == 64) launch_mma<T, 1, INT4, true>(a, per, grid, s);
  else if (a.head_dim < 64) launch_mma<T, 1, INT4, false>(a, per, grid, s);
  else if (a.head_dim == 128) launch_mma<T, 2, INT4, true>(a, per, grid, s);
  else if (a.head_dim < 128) launch_mma<T, 2, INT4, false>(a, per, grid, s);
  else if (a.head_dim == 256) launch_mma<T, 4, INT4, true>(a, per, grid, s);
  else launch_mma<T, 4, INT4, false>(a, per, grid, s);
}

template <int LANES>
void launch_fp32(const AttendArgs& a, int per, dim3 grid, cudaStream_t s) {
  if (per == 1) k_attend_fp32<LANES, 1><<<grid, kAttendThreads, 0, s>>>(a);
  else if (per == 2) k_attend_fp32<LANES, 2><<<grid, kAttendThreads, 0, s>>>(a);
  else k_attend_fp32<LANES, 4><<<grid, kAttendThreads, 0, s>>>(a);
}

template <typename T>
cudaError_t launch_merge(const AttendArgs& a, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.heads, a.streams);
  cfg.blockDim = dim3(32 * kMergeWarps);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;  // its launch overlaps the parts' kernel
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_merge<T>, a);
}

int check_heads(const st_cache* c, int heads) {
  return heads < 1 || heads > 65535 || heads % c->heads
             ? cache_fail(ST_ERR_INVALID, "query heads are a multiple of the cache's heads, up to 65535") : ST_OK;
}

// Floats of the parts' statistics, up to the 16 bytes on which their sums start.
long long statistics_floats(const st_cache* c, int heads, int splits) {
  return ((long long)c->streams * heads * splits * 2 + 3) / 4 * 4;
}
size_t workspace_bytes(const st_cache* c, int heads, int splits) {
  return splits == 1 ? 0 : (statistics_floats(c, heads, splits) + (size_t)c->streams * heads * splits * c->head_dim) * sizeof(float);
}

}  // namespace
}  // namespace st

using namespace st;

extern "C" {

int st_cache_attention_workspace(const st_cache* c, int heads, size_t* bytes) {
  int rc = check_cache(c, false);
  if (rc != ST_OK || (rc = check_heads(c, heads)) != ST_OK) return rc;
  if (!bytes) return cache_fail(ST_ERR_INVALID, "null pointer");
  *bytes = workspace_bytes(c, heads, splits_of(c, heads));
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
  if ((rc = check_aligned(p->positions, "positions", 8)) != ST_OK) return rc;
  if (!(fabsf(p->scale) <= 0x1p64f)) return cache_fail(ST_ERR_INVALID, "scale must be within 2^64");
  DeviceScope scope(c->device);
  if (scope.status() != ST_OK) return scope.status();
  const int splits = splits_of(c, p->heads);
  const size_t need = workspace_bytes(c, p->heads, splits);
  if (need && (!p->workspace || p->workspace_bytes < need || reinterpret_cast<uintptr_t>(p->workspace) % 256))
    return cache_fail(ST_ERR_INVALID, "the workspace is too small or not on a 256-byte boundary");
  const int per = heads_per_block(c, p->heads);
  AttendArgs a{};
  a.q = p->q.data; a.out = p->out.data;
  a.q_row = p->q.row_stride; a.q_head = p->q.head_stride;
  a.o_row = p->out.row_stride; a.o_head = p->out.head_stride;
  a.keys = c->keys; a.values = c->values;
  a.key_scales = static_cast<const unsigned*>(c->key_scales);
  a.value_scales = static_cast<const unsigned*>(c->value_scales);
  a.stream_stride = c->stream_stride; a.head_stride = c->head_stride;
  a.positions = reinterpret_cast<const long long*>(p->positions);
  a.parts = static_cast<float*>(p->workspace);
  a.sums_at = statistics_floats(c, p->heads, splits);
  a.streams = c->streams; a.heads = p->heads; a.kv_heads = c->heads; a.group = p->heads / c->heads;
  a.head_dim = c->head_dim; a.slots = c->sinks + c->window; a.splits = splits;
  a.blocks = (a.group + per - 1) / per;
  a.scale2 = p->scale * kLog2e;
  const long long blocks = (long long)c->heads * a.blocks;
  if (blocks > 65535) return cache_fail(ST_ERR_INVALID, "query heads are a multiple of the cache's heads, up to 65535");
  const dim3 grid(splits, (unsigned)blocks, c->streams);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool four = c->type == ST_CACHE_INT4;
  if (p->mode == ST_MODE_FP32) {
    switch (lanes_per_row(c->head_dim)) {
      case 1: launch_fp32<1>(a, per, grid, s); break;
      case 2: launch_fp32<2>(a, per, grid, s); break;
      case 4: launch_fp32<4>(a, per, grid, s); break;
      case 8: launch_fp32<8>(a, per, grid, s); break;
      case 16: launch_fp32<16>(a, per, grid, s); break;
      default: launch_fp32<32>(a, per, grid, s); break;
    }
  } else if (p->mode == ST_MODE_FP16) {
    four ? launch_mma<__half, true>(a, per, grid, s) : launch_mma<__half, false>(a, per, grid, s);
  } else {
    four ? launch_mma<__nv_bfloat16, true>(a, per, grid, s) : launch_mma<__nv_bfloat16, false>(a, per, grid, s);
  }
  rc = cache_cuda(cudaGetLastError(), "cache attention launch: ");
  if (rc != ST_OK || splits == 1) return rc;
  const cudaError_t e = p->mode == ST_MODE_FP32   ? launch_merge<float>(a, s)
                        : p->mode == ST_MODE_FP16 ? launch_merge<__half>(a, s)
                                                  : launch_merge<__nv_bfloat16>(a, s);
  if (e != cudaSuccess) {
    cudaGetLastError();  // reported here, so not left pending
    return cache_cuda(e, "cache attention merge launch: ");
  }
  return ST_OK;
}

}  // extern "C"
