// st_cache_attention.cu -- one query row per stream over its cache
// (st_cache_attention).
//
// The bound is memory: every seen key and value row is read once, and each
// byte of a 16-bit row meets one multiply-add per query head of its group. A
// kernel for a head alone would read the rows once per head, so a CTA takes all
// query heads of a key head (in blocks of 8 or 16), and 16-bit and 4-bit rows
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
// 4-bit rows: codes 0..15 are exact 16-bit operands. Within a group of 32
// columns sum q k = scale * sum q code + lowest * sum q, so the product runs on
// the codes and the group's scale and lowest value enter in fp32 once per slot
// and head. For values the scale is folded into the weight before its one
// rounding (to bf16: its range holds any scale), and sum p * lowest is kept in
// fp32 beside the product.
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
  float* parts;   // [stream][head][split]{m, l}, then [stream][head][split][head_dim]
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
__device__ __forceinline__ uint2 ld_row8(const void* p) {
  uint2 r;
  asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ unsigned ld_row4(const void* p) {
  unsigned r;
  asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(r) : "l"(p));
  return r;
}

// Nibbles i and i + 4 of `w` as a pair of exact 16-bit numbers: the nibble in
// the low mantissa bits of 2^10 (fp16) or 2^7 (bf16), which is taken off again.
template <typename T>
__device__ __forceinline__ unsigned code_pair(unsigned w, int i) {
  if constexpr (std::is_same<T, __half>::value) {
    unsigned x = ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u;
    const unsigned base = 0x64006400u;
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&base));
    return *reinterpret_cast<const unsigned*>(&y);
  } else {
    unsigned x = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
    const unsigned base = 0x43004300u;
    const __nv_bfloat162 y =
        __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&base));
    return *reinterpret_cast<const unsigned*>(&y);
  }
}

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
  a.parts[(long long)a.streams * a.heads * a.splits * 2 + at * a.head_dim + d] = o;
}

__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---------------------------------------------------------------- 16-bit and 4-bit rows
// DB: blocks of 64 columns; NT: blocks of 8 query heads; FULL: head_dim is 64 DB, so that row offsets are constants
// and no column is checked.
template <typename T, int DB, int NT, bool INT4, bool FULL>
__global__ void __launch_bounds__(kAttendThreads) k_attend_mma(const AttendArgs a) {
  constexpr int J = 2 * DB;   // pieces of 32 columns
  constexpr float kLift = std::is_same<T, __half>::value && !INT4 ? 10.f : 0.f;
  using PT = typename std::conditional<INT4, __nv_bfloat16, T>::type;  // type of the second product
  __shared__ float sh_o[kAttendWarps][NT * 8][DB * 64 + 4];
  __shared__ float sh_m[kAttendWarps][NT * 8], sh_l[kAttendWarps][NT * 8];
  const int split = blockIdx.x, kv = blockIdx.y / a.blocks, block = blockIdx.y % a.blocks, stream = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (a.splits > 1) let_next_kernel_start();
  const int seen = slots_seen(a.positions[stream], a.slots);
  int first, last;
  split_slots(seen, 16 * kAttendWarps, split, a.splits, first, last);
  const int head0 = kv * a.group + block * NT * 8;                          // first query head of the block
  const int nheads = min(NT * 8, a.group - block * NT * 8);

  // query fragments: columns 32 j + 8 t of head 8 n + g (4-bit: pairs (i, i + 4) of the 8 columns)
  unsigned qf[NT][J][4];
  float qsum[NT][J][2];  // 4-bit: sum of the group's columns for heads 8 n + 2 t, + 1
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const bool head_on = n * 8 + g < nheads;
    const T* qp = static_cast<const T*>(a.q) + stream * a.q_row + (long long)(head0 + n * 8 + g) * a.q_head;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      uint4 u = make_uint4(0, 0, 0, 0);
      // 4-bit: the group's 8-column words reach lanes 0 .. 3 in the order 0, 2, 1, 3 (see the exchange below)
      const int col = j * 32 + (INT4 ? (t & 1) * 16 + (t >> 1) * 8 : t * 8);
      if (head_on && col < a.head_dim) u = *reinterpret_cast<const uint4*>(qp + col);
      if (INT4) {
        qf[n][j][0] = __byte_perm(u.x, u.z, 0x5410);  // columns 0, 4
        qf[n][j][1] = __byte_perm(u.x, u.z, 0x7632);  // 1, 5
        qf[n][j][2] = __byte_perm(u.y, u.w, 0x5410);  // 2, 6
        qf[n][j][3] = __byte_perm(u.y, u.w, 0x7632);  // 3, 7
        float f[8], s = 0.f;
        load8(reinterpret_cast<const T*>(&u), f);
#pragma unroll
        for (int i = 0; i < 8; ++i) s += f[i];
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        qsum[n][j][0] = __shfl_sync(0xffffffffu, s, (2 * t) * 4);
        qsum[n][j][1] = __shfl_sync(0xffffffffu, s, (2 * t + 1) * 4);
      } else {
        qf[n][j][0] = u.x; qf[n][j][1] = u.y; qf[n][j][2] = u.z; qf[n][j][3] = u.w;
      }
    }
  }

  float o[NT][DB][4][4] = {};        // [head block][column block][m-tile]
  float olow[NT][J][2] = {};         // 4-bit: sum of weight * lowest, this lane's slots
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;

  const long long row0 = stream * a.stream_stride + kv * a.head_stride;
  const int dim = FULL ? DB * 64 : a.head_dim, groups = dim / 32, row_bytes = INT4 ? dim / 2 : dim * 2;
  const int step = 16 * kAttendWarps;
  int slot0 = first + warp * 16;
  // this lane's first addresses of the tile to load next
  const char* kp = static_cast<const char*>(a.keys) + (row0 + slot0 + g) * row_bytes + t * (INT4 ? 8 : 16);
  const char* vp = static_cast<const char*>(a.values) + (row0 + slot0 + 2 * t) * row_bytes + g * (INT4 ? 4 : 16);
  const unsigned* ksp = a.key_scales + (row0 + slot0 + g) * groups;
  const unsigned* vsp = a.value_scales + (row0 + slot0 + g) * groups;

  // one tile in registers: loaded a step ahead of its use
  constexpr int KW = INT4 ? DB * 2 : J * 4, VW = INT4 ? DB : DB * 4;
  unsigned kf[2][KW], vf[4][VW], ks[2][INT4 ? J : 1], vs[2][INT4 ? J : 1];

  auto load_scales = [&](unsigned(&f)[2][INT4 ? J : 1], const unsigned* sp, int at, bool whole) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const bool in = whole || at + g + 8 * r < last;
      const unsigned* p = sp + 8 * r * groups;
      if constexpr (FULL && J % 4 == 0) {
#pragma unroll
        for (int j = 0; j < J; j += 4) {
          const uint4 u = in ? ld_row16(p + j) : make_uint4(0, 0, 0, 0);
          f[r][j] = u.x; f[r][j + 1] = u.y; f[r][j + 2] = u.z; f[r][j + 3] = u.w;
        }
      } else if constexpr (FULL) {
        const uint2 u = in ? ld_row8(p) : make_uint2(0, 0);
        f[r][0] = u.x; f[r][1] = u.y;
      } else {
#pragma unroll
        for (int j = 0; j < J; ++j) f[r][j] = in && j < groups ? ld_row4(p + j) : 0u;
      }
    }
  };
  // Slots past `last` load nothing and count as zeros, so that no value there matters; `whole`: the tile has none.
  auto load_k = [&](int at, bool whole) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const bool in = whole || at + g + 8 * r < last;
      const char* p = kp + 8 * r * row_bytes;
      if constexpr (INT4) {
#pragma unroll
        for (int i = 0; i < DB; ++i) {  // 16 columns: 64 i + 16 t
          const uint2 u = in && (FULL || i * 64 + t * 16 < dim) ? ld_row8(p + i * 32) : make_uint2(0, 0);
          kf[r][2 * i] = u.x; kf[r][2 * i + 1] = u.y;
        }
      } else {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const uint4 u = in && (FULL || j * 32 + t * 8 < dim) ? ld_row16(p + j * 64) : make_uint4(0, 0, 0, 0);
          kf[r][4 * j] = u.x; kf[r][4 * j + 1] = u.y; kf[r][4 * j + 2] = u.z; kf[r][4 * j + 3] = u.w;
        }
      }
    }
    if constexpr (INT4) load_scales(ks, ksp, at, whole);
  };
  auto load_v = [&](int at, bool whole) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int ahead = (r & 1) + 8 * (r >> 1);
      const bool in = whole || at + 2 * t + ahead < last;
      const char* p = vp + ahead * row_bytes;
#pragma unroll
      for (int i = 0; i < DB; ++i) {
        const bool on = in && (FULL || i * 64 + g * 8 < dim);
        if constexpr (INT4) {
          vf[r][i] = on ? ld_row4(p + i * 32) : 0u;
        } else {
          const uint4 u = on ? ld_row16(p + i * 128) : make_uint4(0, 0, 0, 0);
          vf[r][4 * i] = u.x; vf[r][4 * i + 1] = u.y; vf[r][4 * i + 2] = u.z; vf[r][4 * i + 3] = u.w;
        }
      }
    }
    if constexpr (INT4) load_scales(vs, vsp, at, whole);
  };
  auto fetch_k = [&](int at) {
    if (at + 16 <= last) load_k(at, true);
    else load_k(at, false);
    kp += (long long)step * row_bytes;
    if (INT4) ksp += step * groups;
  };
  auto fetch_v = [&](int at) {
    if (at + 16 <= last) load_v(at, true);
    else load_v(at, false);
    vp += (long long)step * row_bytes;
    if (INT4) vsp += step * groups;
  };

  if (slot0 < last) {
    fetch_k(slot0);
    fetch_v(slot0);
  }
  for (; slot0 < last; slot0 += step) {
    // S^T: slots g (c0, c1) and g + 8 (c2, c3), heads 8 n + 2 t, + 1
    float s[NT][4];
    if constexpr (INT4) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int i = 0; i < DB; ++i) {
        // lanes t = 0, 1 hold 16 columns of group 2 i, lanes 2, 3 of group 2 i + 1: swap one word, so that every
        // lane has 8 columns of each; the group's 4 words come in the order of lanes 0, 2, 1, 3
        unsigned w[2][2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const unsigned give = t < 2 ? kf[r][2 * i + 1] : kf[r][2 * i], keep = t < 2 ? kf[r][2 * i] : kf[r][2 * i + 1];
          const unsigned got = __shfl_xor_sync(0xffffffffu, give, 2);
          w[r][0] = t < 2 ? keep : got;
          w[r][1] = t < 2 ? got : keep;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = 2 * i + e;
          unsigned c[2][4];
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int x = 0; x < 4; ++x) c[r][x] = code_pair<T>(w[r][e], x);
          const float s0 = group_scale(ks[0][j]), l0 = group_lowest(ks[0][j]);
          const float s1 = group_scale(ks[1][j]), l1 = group_lowest(ks[1][j]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            mma<T>(acc, c[0][0], c[1][0], c[0][1], c[1][1], qf[n][j][0], qf[n][j][1]);
            mma<T>(acc, c[0][2], c[1][2], c[0][3], c[1][3], qf[n][j][2], qf[n][j][3]);
            s[n][0] = fmaf(acc[0], s0, fmaf(l0, qsum[n][j][0], s[n][0]));
            s[n][1] = fmaf(acc[1], s0, fmaf(l0, qsum[n][j][1], s[n][1]));
            s[n][2] = fmaf(acc[2], s1, fmaf(l1, qsum[n][j][0], s[n][2]));
            s[n][3] = fmaf(acc[3], s1, fmaf(l1, qsum[n][j][1], s[n][3]));
          }
        }
      }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          mma<T>(s[n], kf[0][4 * j], kf[1][4 * j], kf[0][4 * j + 1], kf[1][4 * j + 1], qf[n][j][0], qf[n][j][1]);
          mma<T>(s[n], kf[0][4 * j + 2], kf[1][4 * j + 2], kf[0][4 * j + 3], kf[1][4 * j + 3], qf[n][j][2], qf[n][j][3]);
        }
      }
    }
    const int next = slot0 + step;
    if (next < last) fetch_k(next);

    const bool in0 = slot0 + g < last, in1 = slot0 + g + 8 < last;
    unsigned pf[NT][INT4 ? J : 1][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float p[4], top[2];
#pragma unroll
      for (int x = 0; x < 4; ++x) p[x] = (x < 2 ? in0 : in1) ? s[n][x] * a.scale2 : -INFINITY;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        top[x] = fmaxf(p[x], p[2 + x]);
#pragma unroll
        for (int d = 4; d < 32; d *= 2) top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], d));
      }
      if (__any_sync(0xffffffffu, top[0] > m[n][0] || top[1] > m[n][1])) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
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
          if (INT4)
#pragma unroll
            for (int j = 0; j < J; ++j) olow[n][j][x] *= keep;
        }
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float ref = m[n][x & 1] == -INFINITY ? 0.f : m[n][x & 1] - kLift;
        p[x] = exp2_fast(p[x] - ref);
        l[n][x & 1] += p[x];
      }
      if constexpr (INT4) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const float s0 = group_scale(vs[0][j]), l0 = group_lowest(vs[0][j]);
          const float s1 = group_scale(vs[1][j]), l1 = group_lowest(vs[1][j]);
          olow[n][j][0] = fmaf(p[0], l0, fmaf(p[2], l1, olow[n][j][0]));
          olow[n][j][1] = fmaf(p[1], l0, fmaf(p[3], l1, olow[n][j][1]));
          pf[n][j][0] = transpose8x8(pack2((PT*)nullptr, p[0] * s0, p[1] * s0));
          pf[n][j][1] = transpose8x8(pack2((PT*)nullptr, p[2] * s1, p[3] * s1));
        }
      } else {
        pf[n][0][0] = transpose8x8(pack2((PT*)nullptr, p[0], p[1]));
        pf[n][0][1] = transpose8x8(pack2((PT*)nullptr, p[2], p[3]));
      }
    }

    // O^T += V^T P^T
#pragma unroll
    for (int i = 0; i < DB; ++i) {
      if constexpr (INT4) {
        // lanes g < 4 hold 8 columns of group 2 i, g >= 4 of group 2 i + 1: swap halves with lane g ^ 4, so that
        // every lane has 4 columns of each (low half: group 2 i)
        unsigned w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const unsigned got = __shfl_xor_sync(0xffffffffu, vf[r][i], 16);
          w[r] = __byte_perm(vf[r][i], got, g < 4 ? 0x5410 : 0x3276);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // slots (2 t, 2 t + 1) and (2 t + 8, 2 t + 9) side by side: nibble c of both halves is column c's pair
          const unsigned x0 = __byte_perm(w[0], w[1], e ? 0x7632 : 0x5410);
          const unsigned x1 = __byte_perm(w[2], w[3], e ? 0x7632 : 0x5410);
          unsigned c0[4], c1[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) c0[c] = code_pair<PT>(x0, c), c1[c] = code_pair<PT>(x1, c);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c)
              mma<PT>(o[n][i][2 * e + c], c0[2 * c], c0[2 * c + 1], c1[2 * c], c1[2 * c + 1], pf[n][2 * i + e][0],
                      pf[n][2 * i + e][1]);
        }
      } else {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const unsigned a0 = __byte_perm(vf[0][4 * i + w], vf[1][4 * i + w], 0x5410);
          const unsigned a1 = __byte_perm(vf[0][4 * i + w], vf[1][4 * i + w], 0x7632);
          const unsigned a2 = __byte_perm(vf[2][4 * i + w], vf[3][4 * i + w], 0x5410);
          const unsigned a3 = __byte_perm(vf[2][4 * i + w], vf[3][4 * i + w], 0x7632);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma<PT>(o[n][i][w], a0, a1, a2, a3, pf[n][0][0], pf[n][0][1]);
        }
      }
    }
    if (next < last) fetch_v(next);
  }

  // this warp's part into shared memory, columns in their own order
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int h = n * 8 + 2 * t + x;
      float sum = l[n][x];
#pragma unroll
      for (int d = 4; d < 32; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (g == 0) {
        sh_m[warp][h] = m[n][x];
        sh_l[warp][h] = sum;
      }
      if (INT4)
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int d = 4; d < 32; d *= 2) olow[n][j][x] += __shfl_xor_sync(0xffffffffu, olow[n][j][x], d);
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if (INT4) {
              // m-tile w: group 2 i + w / 2; this lane's 4 columns of it are 8 (g % 4) + (g < 4 ? 0 : 4)
              const int c = i * 64 + (w / 2) * 32 + (g & 3) * 8 + (g < 4 ? 0 : 4) + (w & 1) * 2 + r;
              sh_o[warp][h][c] = o[n][i][w][2 * r + x] + olow[n][2 * i + w / 2][x];
            } else {
              sh_o[warp][h][i * 64 + g * 8 + w * 2 + r] = o[n][i][w][2 * r + x];
            }
          }
    }
  __syncthreads();
  for (int e = threadIdx.x; e < nheads * a.head_dim; e += kAttendThreads) {
    const int h = e / a.head_dim, d = e - h * a.head_dim;
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
  constexpr int U = 2;   // slots a group loads before it uses them
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
template <typename T>
__global__ void __launch_bounds__(kAttendThreads) k_merge(const AttendArgs a) {
  __shared__ float sh_f[kAttendThreads];
  const int h = blockIdx.x, stream = blockIdx.y;
  const int seen = slots_seen(a.positions[stream], a.slots);
  const long long at = ((long long)stream * a.heads + h) * a.splits;
  const float2* ml = reinterpret_cast<const float2*>(a.parts) + at;
  const float* part = a.parts + (long long)a.streams * a.heads * a.splits * 2 + at * a.head_dim;
  wait_for_previous_kernel();
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ml[s].x);
  float sum = 0.f, o[2] = {};
  for (int base = 0; base < a.splits; base += kAttendThreads) {
    const int n = min(kAttendThreads, a.splits - base);
    __syncthreads();
    if ((int)threadIdx.x < n) {
      const float m = ml[base + threadIdx.x].x;
      sh_f[threadIdx.x] = m == -INFINITY ? 1.f : exp2_fast(m - top);
    }
    __syncthreads();
    for (int s = 0; s < n; ++s) {
      sum = fmaf(ml[base + s].y, sh_f[s], sum);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int d = threadIdx.x + r * kAttendThreads;
        if (d < a.head_dim) o[r] = fmaf(part[(long long)(base + s) * a.head_dim + d], sh_f[s], o[r]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int d = threadIdx.x + r * kAttendThreads;
    if (d < a.head_dim)
      static_cast<T*>(a.out)[stream * a.o_row + h * a.o_head + d] = static_cast<T>(seen ? o[r] / sum : 0.f);
  }
}

// ---------------------------------------------------------------- host
// Query heads that one CTA takes.
int heads_per_block(const st_cache* c, int heads) {
  const int group = heads / c->heads;
  if (c->type == ST_MODE_FP32) return group <= 1 ? 1 : group <= 2 ? 2 : 4;
  return group <= 8 || c->head_dim > 128 ? 8 : 16;
}

// CTAs that share the slots of one key head.
int splits_of(const st_cache* c, int heads) {
  const int per = heads_per_block(c, heads), group = heads / c->heads;
  const long long ctas = (long long)c->streams * c->heads * ((group + per - 1) / per);
  const int slots = c->sinks + c->window;
  const long long want = (8ll * sm_count(c->device) + ctas - 1) / ctas;  // 4 resident CTAs an SM, twice over
  const long long most = (slots + 255) / 256;                             // at least 256 slots each
  const long long n = want < most ? want : most;
  return n < 1 ? 1 : n > 1024 ? 1024 : (int)n;
}

template <typename T, bool INT4, bool FULL>
void launch_mma(const AttendArgs& a, int per, dim3 grid, cudaStream_t s) {
  if (a.head_dim <= 64) {
    if (per == 8) k_attend_mma<T, 1, 1, INT4, FULL><<<grid, kAttendThreads, 0, s>>>(a);
    else k_attend_mma<T, 1, 2, INT4, FULL><<<grid, kAttendThreads, 0, s>>>(a);
  } else if (a.head_dim <= 128) {
    if (per == 8) k_attend_mma<T, 2, 1, INT4, FULL><<<grid, kAttendThreads, 0, s>>>(a);
    else k_attend_mma<T, 2, 2, INT4, FULL><<<grid, kAttendThreads, 0, s>>>(a);
  } else {
    k_attend_mma<T, 4, 1, INT4, FULL><<<grid, kAttendThreads, 0, s>>>(a);
  }
}
template <typename T, bool INT4>
void launch_mma(const AttendArgs& a, int per, dim3 grid, cudaStream_t s) {
  if (a.head_dim == 64 || a.head_dim == 128 || a.head_dim == 256) launch_mma<T, INT4, true>(a, per, grid, s);
  else launch_mma<T, INT4, false>(a, per, grid, s);
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
  cfg.blockDim = dim3(kAttendThreads);
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

size_t workspace_bytes(const st_cache* c, int heads, int splits) {
  return splits == 1 ? 0 : (size_t)c->streams * heads * splits * (2 + c->head_dim) * sizeof(float);
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
  if (!(p->scale > -1.0e38f && p->scale < 1.0e38f)) return cache_fail(ST_ERR_INVALID, "scale must be finite");
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
