// st_window.cu -- causal attention of packed sequences with a sliding window
// and sinks (st_window_attention).
//
// Three kernels. k_window_tiles: 16-bit rows, on tcgen05.
// k_window_fp32: fp32 rows of up to 128 columns, tiled for the fp32 units (there
// is no fp32 tensor product). k_window_rows: a few lanes walk the keys that one
// query row of one head sees; it serves the rest (wider fp32 rows, 16-bit rows
// with a scale that is not positive, calls of a few rows).
//
// k_window_tiles. A CTA takes two tiles of 128 query rows, one TMEM lane a row,
// that share their keys: two heads of one key head, or where a key head has an
// odd number of them two neighbouring tiles of one head (one tile: past 128 columns,
// and then up to 64, see launch_tiles). Rows may belong to
// several sequences: the keys that are needed are those from the first row's
// window on, which covers every sequence that begins behind it, and the sinks of
// the first row's sequence. They are walked in blocks of 32 rows (sinks first,
// then the window from exactly its first key), several blocks to a key tile:
//   S = Q K^T          one MMA per 16 columns, both operands in shared memory, S in TMEM
//   P = 2^(c S - m)    one thread a row; m, and the sum l, in fp32
//   O += P V           P from TMEM (written over S), V as it lies in memory (N contiguous)
// While the four warps of one tile are in their exponentials, the products of
// the other run, and the copies of the next key tile: with one tile a CTA and
// room for one key tile, the waits for its copy and for the products set the pace
// (8192 rows, window 4096, 32 heads of 128: 529 us, now 465, 0.53 of the measured
// dense rate; what bounds it is the chain S, softmax, O of each query tile, 3700
// cycles a key tile where exponentials and products take 2050 each; the rest has
// not been measured). O is rescaled only when a row's maximum
// has grown by more than 2^8 since the last time; P then stays below 2^8, which
// both 16-bit types hold, and l and O share the reference, so the quotient is
// exact.
//
// A warp masks only the blocks at an edge of one of its rows' windows, and skips
// those that none of its rows sees. A masked weight is 0, but 0 times an infinite
// or NaN value is NaN: when a result of the tile is not finite (only then), the
// CTA does its rows again with the row kernel's code, which never reads what a
// row does not see. k_window_fp32 does the same.
//
// Every wait has a limit; a CTA that ran into one writes NaN.
#include <cuda.h>

#include <atomic>

#include "st_cache_host.h"
#include "st_umma.cuh"
#include "st_cache.cuh"

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
// `end`, if given: the first row behind that sequence.
__device__ int sequence_start(const WindowArgs& a, int row, int* end = nullptr) {
  if (end) *end = a.rows;
  if (!a.starts) return 0;
  int lo = 0, hi = a.sequences;  // the first sequence that ends behind the row
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;  // the sum of both passes 2^31 from 2^30 sequences on
    if (a.starts[mid + 1] <= row) lo = mid + 1;
    else hi = mid;
  }
  if (lo == a.sequences) return -1;
  if (end) *end = clamp_row(a.starts[lo + 1], a.rows);
  const int first = clamp_row(a.starts[lo], a.rows);
  return first <= row ? first : -1;
}

// One query row of one head by a group of LANES lanes (`mask`: those lanes of the warp).
// KEYS at a time: 2 where that is all a kernel does (201 fp32 rows of 256 columns 27.5 -> 18.5 us, bf16 9 % less; 4 take
// more registers: 17 % more), 1 where another kernel falls back on it.
template <typename T, int LANES, int KEYS = 1>
__device__ __forceinline__ void window_row(const WindowArgs& a, int row, int start, int h, int lane, unsigned mask) {
  const int kv = h / (a.heads / a.kv_heads);
  const bool on = lane * 8 < a.head_dim;
  float q[8] = {}, acc[8] = {}, m = -INFINITY, l = 0.f;
  if (on) load8(static_cast<const T*>(a.q) + row * a.q_row + h * a.q_head + lane * 8, q);
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] *= a.scale;
  const T* kp = static_cast<const T*>(a.k) + kv * a.k_head + lane * 8;
  const T* vp = static_cast<const T*>(a.v) + kv * a.v_head + lane * 8;
  const int low = (int)max((long long)start, (long long)row - a.window + 1);  // first row of the window
  const long long sinks = (long long)start + a.sinks;                         // first row behind the sinks
  int j = start < low && a.sinks > 0 ? start : low;
  while (j <= row) {
    float k[KEYS][8] = {}, v[KEYS][8] = {}, dot[KEYS] = {};
    bool seen[KEYS];
#pragma unroll
    for (int u = 0; u < KEYS; ++u) {
      seen[u] = j <= row;
      if (seen[u] && on) {
        load8(kp + j * a.k_row, k[u]);
        load8(vp + j * a.v_row, v[u]);
      }
      ++j;
      if (j < low && j >= sinks) j = low;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int u = 0; u < KEYS; ++u) dot[u] = fmaf(q[i], k[u][i], dot[u]);
#pragma unroll
    for (int o = 1; o < LANES; o *= 2)
#pragma unroll
      for (int u = 0; u < KEYS; ++u) dot[u] += __shfl_xor_sync(mask, dot[u], o);
    float top = m;
#pragma unroll
    for (int u = 0; u < KEYS; ++u) top = seen[u] ? fmaxf(top, dot[u]) : top;
    const float ref = top == -INFINITY ? 0.f : top, keep = top == -INFINITY ? 1.f : __expf(m - top);
    m = top;
    l *= keep;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] *= keep;
#pragma unroll
    for (int u = 0; u < KEYS; ++u) {
      const float p = seen[u] ? __expf(dot[u] - ref) : 0.f;  // a NaN stays one
      l += p;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = fmaf(p, v[u][i], acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] /= l;
  if (on) store8(static_cast<T*>(a.out) + row * a.o_row + h * a.o_head + lane * 8, acc);
}

template <int LANES>
__device__ __forceinline__ unsigned row_mask() {
  return LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u) << ((threadIdx.x & 31) / LANES * LANES);
}

template <typename T, int LANES>
__global__ void __launch_bounds__(kWindowThreads) k_window_rows(const WindowArgs a) {
  const long long row = (long long)blockIdx.x * (kWindowThreads / LANES) + threadIdx.x / LANES;
  if (row >= a.rows) return;
  const int start = sequence_start(a, (int)row);
  if (start < 0) return;
  window_row<T, LANES, 2>(a, (int)row, start, blockIdx.y, threadIdx.x % LANES, row_mask<LANES>());
}

// ---------------------------------------------------------------- tcgen05
constexpr int kTileRows = 128;      // query rows of a CTA: TMEM lanes
constexpr int kBlockRows = 32;      // key rows of one copy
constexpr int kWaitTries = 1 << 26;  // a second or two

// Whether a phase of `bar` completed within the limit. It polls: a try_wait that suspends the thread costs more to
// wake from than most of these waits last (8192 rows, window 4096: 641 us with it, 557 without).
__device__ __forceinline__ bool wait_phase(unsigned long long* bar, unsigned parity) {
#pragma unroll 1
  for (int i = 0; i < kWaitTries; ++i)
    if (mbar_test_wait(bar, parity)) return true;
  return false;
}

// DP: columns, padded to 64, 128 or 256 with zeros by the copies; SUBS: query tiles of a CTA. S and O take DP TMEM
// columns each for each query tile, so that one CTA of 128 or 256 columns, or two (four of one query tile) of 64, fill an
// SM's TMEM. Key tiles are DP rows, of 256 columns 64: shared memory holds no more (2 sequences of 4000 rows, window 4000,
// 16 heads of 256: 550 us, 622 TFLOP/s).
template <int DP, int SUBS>
struct Tiles {
  static constexpr int kKeys = DP == 256 ? 64 : DP, kBlocks = kKeys / kBlockRows, kPanels = DP / 64;
  static constexpr int kQBytes = kPanels * kTileRows * 128, kKvBytes = kPanels * kKeys * 128;
  // 4 warps of rows for each tile, one that copies, one that issues products; at 128 columns two more, which make the
  // last four a warpgroup that hands registers to the others
  static constexpr int kCopyWarp = 4 * SUBS, kIssueWarp = kCopyWarp + 1;
  static constexpr int kThreads = DP == 128 ? 384 : kIssueWarp * 32 + 32, kCtas = DP == 64 ? 4 / SUBS : 1;
  // One ring for K and V tiles in the order of their use: two are being read, the others are on their way. With two
  // slots each (one ahead) the products waited for the copies.
  static constexpr int kSlots = DP == 128 ? 5 : 4 * SUBS;
  static constexpr int kSmem = SUBS * kQBytes + kSlots * kKvBytes + 1024;
};

struct TileMaps {
  CUtensorMap q, k, v;
};

// Shared-memory matrix descriptors, 128-byte swizzle (layout type 2), version 1. K-major (Q, K): 8-row groups 1024
// bytes apart. MN-major (V): the same groups along K, 64-column panels `panel` bytes apart.
__device__ __forceinline__ unsigned long long swizzled_desc(const void* smem, unsigned panel) {
  return (unsigned long long)((smem_addr(smem) & 0x3FFFFu) >> 4) | ((unsigned long long)(panel >> 4) << 16) |
         ((unsigned long long)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// Box at (column, head, row) of a row tensor.
__device__ __forceinline__ void copy_box(void* dst, const CUtensorMap* map, int col, int head, int row,
                                         unsigned long long* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      :: "r"(smem_addr(dst)), "l"(map), "r"(col), "r"(head), "r"(row), "r"(smem_addr(bar)) : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  unsigned yes;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(yes));
  return yes != 0;
}

// A from TMEM, B by descriptor.
__device__ __forceinline__ void umma_f16_ts(unsigned d, unsigned at, unsigned long long bdesc, unsigned idesc,
                                            unsigned accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(at), "l"(bdesc), "r"(idesc),
      "r"(accumulate)
      : "memory");
}

// 32 lanes x 32 or 64 columns between registers and TMEM. The wait belongs to the load's own statement: its registers
// have no value before it, and nothing may move them.
__device__ __forceinline__ void tmem_ld32(unsigned addr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31"
      "}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld64(unsigned addr, float (&v)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
      "}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]),
        "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]),
        "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]),
        "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]),
        "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(unsigned addr, const float (&v)[32]) {
  unsigned r[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(v[i]);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
      "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
      "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(unsigned addr, const unsigned (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long x, y, z, d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(z) : "f"(c.x), "f"(c.y));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(x), "l"(y), "l"(z));
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(d));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long x, y, d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(x), "l"(y));
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(d));
  return r;
}

// Bits lo .. hi of a 32-bit word (either end may lie outside it).
__device__ __forceinline__ unsigned bit_range(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 31);
  return lo > hi ? 0u : (0xffffffffu >> (31 - hi)) & (0xffffffffu << lo);
}

// What a CTA's tile of rows needs: its rows inside sequences, and its key blocks.
struct TileKeys {
  int r0, r1;              // first and last row inside a sequence
  int start;               // first row of r0's sequence
  bool one;                // r1 is in that sequence too
  int sink_end;            // sinks walked apart: rows start .. sink_end - 1
  int low;                 // first row of the window blocks
  int sink_blocks, blocks;
  __device__ int base(int block) const {  // first row of a block
    return block < sink_blocks ? start + block * kBlockRows : low + (block - sink_blocks) * kBlockRows;
  }
};
__device__ __forceinline__ bool tile_keys(const WindowArgs& a, long long first, int rows, TileKeys& t) {
  if (first >= a.rows) return false;
  t.r0 = (int)first;
  t.r1 = (int)min((long long)a.rows, first + rows) - 1;
  if (a.starts) {
    t.r0 = max(t.r0, clamp_row(a.starts[0], a.rows));
    t.r1 = min(t.r1, clamp_row(a.starts[a.sequences], a.rows) - 1);
  }
  if (t.r0 > t.r1) return false;
  int end;
  t.start = sequence_start(a, t.r0, &end);
  t.one = end > t.r1;
  if (t.start < 0) t.start = t.r0;  // only with starts that decrease
  t.low = (int)max((long long)t.start, (long long)t.r0 - a.window + 1);
  t.sink_end = (int)min((long long)t.low, (long long)t.start + a.sinks);
  t.sink_blocks = (t.sink_end - t.start + kBlockRows - 1) / kBlockRows;
  t.blocks = t.sink_blocks + (t.r1 - t.low + kBlockRows) / kBlockRows;
  return true;
}

// The keys one row sees, as bits of a block of 32 key rows.
struct RowLimits {
  int row, start, low, sink_last;  // start -1: none
  __device__ void set(const WindowArgs& a, const TileKeys& t, int r) {
    row = r;
    start = r < t.r0 || r > t.r1 ? -1 : t.one ? t.start : sequence_start(a, r);
    low = (int)max((long long)start, (long long)r - a.window + 1);
    sink_last = (int)min((long long)r, (long long)start + a.sinks - 1);
  }
  __device__ unsigned bits(const TileKeys& t, int block) const {
    if (start < 0 || block >= t.blocks) return 0;
    const int base = t.base(block);
    if (block < t.sink_blocks) return start == t.start ? bit_range(0, min(sink_last, t.sink_end - 1) - base) : 0u;
    return bit_range(low - base, row - base) | bit_range(start - base, sink_last - base);
  }
};
// First row that is inside the window of every row up to r1 of r1's sequence.
__device__ __forceinline__ int common_low(const WindowArgs& a, const TileKeys& t, int r1) {
  return (int)max((long long)(t.one ? t.start : sequence_start(a, r1)), (long long)r1 - a.window + 1);
}

// One of a CTA's two tiles: which key blocks any of its rows can see, and which all of them do.
struct SubTile {
  int r0, r1, start, low, sink_end, all_low;
  bool any;
  __device__ void set(const WindowArgs& a, const TileKeys& t, long long first) {
    any = first <= t.r1;
    if (!any) return;
    r0 = max((int)first, t.r0);
    r1 = (int)min((long long)t.r1, first + kTileRows - 1);
    any = r0 <= r1;
    if (!any) return;
    start = t.one ? t.start : max(sequence_start(a, r0), 0);
    low = (int)max((long long)start, (long long)r0 - a.window + 1);
    sink_end = (int)min((long long)r0, (long long)start + a.sinks);
    all_low = common_low(a, t, r1);
  }
  __device__ bool needs(const TileKeys& t, int b0, int nb) const {
    if (!any) return false;
    if (b0 < t.sink_blocks) return start == t.start || b0 + nb > t.sink_blocks;
    const int first = t.base(b0), last = t.base(b0 + nb - 1) + kBlockRows - 1;
    return (last >= low && first <= r1) || (last >= start && first < sink_end);
  }
  __device__ bool sees_all(const TileKeys& t, int b0, int nb) const {
    return b0 >= t.sink_blocks && t.base(b0) >= all_low && t.base(b0 + nb - 1) + kBlockRows - 1 <= r0;
  }
};

template <typename T, int DP, int SUBS>
__global__ void __launch_bounds__(Tiles<DP, SUBS>::kThreads, Tiles<DP, SUBS>::kCtas)
    k_window_tiles(const WindowArgs a, const __grid_constant__ TileMaps maps) {
  using G = Tiles<DP, SUBS>;
  extern __shared__ unsigned char raw[];
  __shared__ unsigned long long q_full, full[G::kSlots], free[G::kSlots], s_full[SUBS], p_full[SUBS], o_full[SUBS];
  __shared__ unsigned tmem_base;
  __shared__ int sh_slow, sh_dead;
  const int warp = threadIdx.x >> 5;
  // one query tile, or two: two heads of one tile of rows, or two tiles of one head; those with most keys first
  const bool two_heads = SUBS == 2 && (a.heads / a.kv_heads) % 2 == 0;
  const int per_row = two_heads ? a.heads / 2 : a.heads, row_tiles = two_heads ? 1 : SUBS;
  const int h0 = two_heads ? blockIdx.x % per_row * 2 : blockIdx.x % per_row;
  const long long pair_row = (long long)(gridDim.x / per_row - 1 - blockIdx.x / per_row) * row_tiles * kTileRows;
  auto head_of = [&](int s) { return two_heads ? h0 + s : h0; };
  auto first_row = [&](int s) { return pair_row + (two_heads ? 0 : s * kTileRows); };
  TileKeys keys;
  if (!tile_keys(a, pair_row, row_tiles * kTileRows, keys)) return;
  unsigned char* smem = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);
  unsigned char *sq = smem, *ring = sq + SUBS * G::kQBytes;  // ring item 2 i: K of key tile i, 2 i + 1: V
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    for (int s = 0; s < G::kSlots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&free[s], 1);
    }
    for (int s = 0; s < SUBS; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4);
      mbar_init(&o_full[s], 1);
    }
    fence_mbar_init();
    sh_slow = sh_dead = 0;
  }
  if (warp == G::kIssueWarp) {
    tmem_alloc(&tmem_base, 2 * SUBS * DP);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // TMEM: S of both tiles, then O of both
  const unsigned tmem = tmem_base;
  const int tiles = (keys.blocks + G::kBlocks - 1) / G::kBlocks;
  // A wait that runs out ends its role; the others' waits then run out as well.
  auto wait = [&](unsigned long long* bar, int use) -> bool {
    if (wait_phase(bar, use & 1)) return true;
    *(volatile int*)&sh_dead = 1;
    return false;
  };

  if (warp >= G::kCopyWarp) {
    // 384 threads start with 168 registers each: 2 * 128 * 208 + 128 * 88 is as many
    if constexpr (DP == 128) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    // Both warps run as a whole, and one lane issues: what an instruction takes then stays in uniform registers. The
    // products' issue is on the critical path (by one lane alone, with descriptors built for each, 8192 rows, window
    // 4096: 557 us, so 489).
    if (warp == G::kCopyWarp) {
      const bool lead = elect_one();
      const int kv = h0 / (a.heads / a.kv_heads);
      if (lead) {
        mbar_expect_tx(&q_full, SUBS * G::kQBytes);
        for (int s = 0; s < SUBS; ++s)
          for (int p = 0; p < G::kPanels; ++p)
            copy_box(sq + s * G::kQBytes + p * kTileRows * 128, &maps.q, p * 64, head_of(s), (int)first_row(s), &q_full);
      }
      int item = 0, slot = 0, use = 0;
      for (; item < 2 * tiles; ++item) {
        const int b0 = item / 2 * G::kBlocks, nb = min(G::kBlocks, keys.blocks - b0);
        if (use > 0 && !wait(&free[slot], use - 1)) break;
        if (lead) {
          mbar_expect_tx(&full[slot], nb * G::kPanels * kBlockRows * 128);
          unsigned char* to = ring + slot * G::kKvBytes;
          const CUtensorMap* map = item & 1 ? &maps.v : &maps.k;
          for (int b = 0; b < nb; ++b, to += kBlockRows * 128) {
            const int row = keys.base(b0 + b);
#pragma unroll
            for (int p = 0; p < G::kPanels; ++p) copy_box(to + p * G::kKeys * 128, map, p * 64, kv, row, &full[slot]);
          }
        }
        if (++slot == G::kSlots) slot = 0, ++use;
      }
      if (*(volatile int*)&sh_dead) {  // no copy may land after the CTA has left
        wait_phase(&q_full, 0);
        for (int i = max(0, item - G::kSlots); i < item; ++i) wait_phase(&full[i % G::kSlots], (i / G::kSlots) & 1);
      }
    } else if (warp == G::kIssueWarp) {
      const bool lead = elect_one();
      SubTile sub[SUBS];
      for (int s = 0; s < SUBS; ++s) sub[s].set(a, keys, first_row(s));
      const int ksteps = (a.head_dim + 15) / 16;
      const unsigned idesc_s = umma_idesc<T>(kTileRows, G::kKeys);
      const unsigned idesc_o = umma_idesc<T>(kTileRows, ksteps * 16) | (1u << 16);  // V: N contiguous
      const unsigned long long dq = swizzled_desc(sq, 0), dk = swizzled_desc(ring, 0), dv = swizzled_desc(ring, G::kKeys * 128);
      constexpr unsigned kSlotStep = G::kKvBytes >> 4;
      int done[SUBS] = {};  // second products issued
      auto needs = [&](int s, int i) {
        return i < tiles && sub[s].needs(keys, i * G::kBlocks, min(G::kBlocks, keys.blocks - i * G::kBlocks));
      };
      // S of a key tile, once P of the last one, under it, has been read
      auto first_product = [&](int s, int slot, int nb) -> bool {
        if (done[s] > 0 && !wait(&o_full[s], done[s] - 1)) return false;
        tc_fence_after();
        const unsigned idesc = nb == G::kBlocks ? idesc_s : umma_idesc<T>(kTileRows, nb * kBlockRows);
        const unsigned long long q = dq + s * (G::kQBytes >> 4), k = dk + slot * kSlotStep;
        if (lead) {
#pragma unroll
          for (int e = 0; e < DP / 16; ++e)
            if (e < ksteps)
              umma_f16(tmem + s * DP, q + (e / 4) * (kTileRows * 128 >> 4) + (e % 4) * 2,
                       k + (e / 4) * (G::kKeys * 128 >> 4) + (e % 4) * 2, idesc, e > 0);
          umma_commit(&s_full[s]);
        }
        __syncwarp();
        return true;
      };
      auto second_product = [&](int s, int slot, int nb) -> bool {
        if (!wait(&p_full[s], done[s])) return false;
        tc_fence_after();
        const unsigned long long v = dv + slot * kSlotStep;
        if (lead) {
#pragma unroll
          for (int e = 0; e < G::kBlocks * 2; ++e)
            if (e < nb * 2)
              umma_f16_ts(tmem + (SUBS + s) * DP, tmem + s * DP + e * 8, v + e * (2048 >> 4), idesc_o, e > 0 || done[s] > 0);
          umma_commit(&o_full[s]);
        }
        __syncwarp();
        ++done[s];
        return true;
      };
      int slot = 0, use = 0;   // of the next ring item
      auto here = [&]() { return wait(&full[slot], use); };
      auto advance = [&]() {
        const int was = slot;
        if (++slot == G::kSlots) slot = 0, ++use;
        return was;
      };
      auto release = [&](int which) {
        if (lead) umma_commit(&free[which]);
        __syncwarp();
      };
      int nb = min(G::kBlocks, keys.blocks);
      constexpr int kLast = SUBS - 1;
      bool need0 = needs(0, 0), need1 = kLast && needs(kLast, 0);  // one query tile: the second is never needed
      bool ok = wait(&q_full, 0) && here();
      if (ok) {
        const int k = advance();
        ok = (!need0 || first_product(0, k, nb)) && (!need1 || first_product(kLast, k, nb));
        if (ok) release(k);
      }
      for (int i = 0; i < tiles && ok; ++i) {
        const bool next0 = needs(0, i + 1), next1 = kLast && needs(kLast, i + 1), more = i + 1 < tiles;
        const int next_nb = min(G::kBlocks, keys.blocks - (i + 1) * G::kBlocks);
        if (!(ok = here())) break;
        const int v = advance();
        if (need0 && !(ok = second_product(0, v, nb))) break;
        int k = 0;
        if (more) {
          if (!(ok = here())) break;
          k = advance();
          if (next0 && !(ok = first_product(0, k, next_nb))) break;
        }
        if (need1 && !(ok = second_product(kLast, v, nb))) break;
        release(v);
        if (more) {
          if (next1 && !(ok = first_product(kLast, k, next_nb))) break;
          release(k);
        }
        need0 = next0;
        need1 = next1;
        nb = next_nb;
      }
    }
  } else {
    if constexpr (DP == 128) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int side = warp >> 2, h = head_of(side), lane = threadIdx.x & 31;
    SubTile sub;
    sub.set(a, keys, first_row(side));
    const long long row = first_row(side) + (threadIdx.x & 127);
    const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
    const unsigned my_s = tmem + side * DP + lanes, my_o = tmem + (SUBS + side) * DP + lanes;
    RowLimits limits;
    limits.set(a, keys, (int)min(row, (long long)INT32_MAX));
    const bool inside = limits.start >= 0;
    const float c = a.scale * 1.4426950408889634f;
    float m = -INFINITY, l = 0.f;  // m: reference of the weights, in units of S
    bool ok = true;
    int n = 0;                     // key tiles of this side so far
    for (int i = 0; i < tiles && ok; ++i) {
      const int b0 = i * G::kBlocks, nb = min(G::kBlocks, keys.blocks - b0);
      if (!sub.needs(keys, b0, nb)) continue;
      // the blocks: bits of the keys this row sees; a block that no row of the warp sees is left out
      const bool plain = nb == G::kBlocks && sub.sees_all(keys, b0, nb);
      unsigned seen[G::kBlocks];
      bool some[G::kBlocks], edge[G::kBlocks];
#pragma unroll
      for (int b = 0; b < G::kBlocks; ++b) {
        seen[b] = plain ? ~0u : b < nb ? limits.bits(keys, b0 + b) : 0u;
        some[b] = plain || __any_sync(0xffffffffu, seen[b] != 0u);
        edge[b] = !plain && __any_sync(0xffffffffu, seen[b] != ~0u);
      }
      if (!(ok = wait(&s_full[side], n))) break;
      tc_fence_after();
      // At 128 columns the registers hold the tile between the passes, else it is read again.
      constexpr bool kKeep = DP == 128;
      float x[kKeep ? 2 : 1][kKeep ? 64 : 32], tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // for latency
      auto mask = [&](int b, auto& y, int from) {
        if (edge[b])
#pragma unroll
          for (int e = 0; e < 32; ++e) y[from + e] = (seen[b] >> e) & 1u ? y[from + e] : -INFINITY;
      };
      auto look = [&](auto& y, int from) {
#pragma unroll
        for (int e = 0; e < 32; e += 2) tops[e / 2 % 4] = max3(tops[e / 2 % 4], y[from + e], y[from + e + 1]);
      };
      if constexpr (kKeep) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
          if (some[2 * half] || some[2 * half + 1]) {
            tmem_ld64(my_s + half * 64, x[half]);
#pragma unroll
            for (int b = 0; b < 2; ++b)
              if (some[2 * half + b]) {
                mask(2 * half + b, x[half], b * 32);
                look(x[half], b * 32);
              }
          }
      } else {
#pragma unroll
        for (int b = 0; b < G::kBlocks; ++b)
          if (some[b]) {
            tmem_ld32(my_s + b * 32, x[0]);
            mask(b, x[0], 0);
            look(x[0], 0);
          }
      }
      const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
      // a new reference only when the old one is too low; exp2(8) is the most a weight can be
      const bool grow = top > m && !((top - m) * c <= 8.f);
      if (__any_sync(0xffffffffu, grow)) {
        const float next = grow ? top : m;
        const float keep = next == -INFINITY ? 1.f : exp2_fast((m - next) * c);
        m = next;
        l *= keep;
        if (n > 0) {
#pragma unroll
          for (int d = 0; d < DP; d += 32) {
            float o[32];
            tmem_ld32(my_o + d, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= keep;
            tmem_st32(my_o + d, o);
          }
        }
      }
      // fp16 weights 2^7 higher, up to 2^15, away from its denormals
      const float ref = m == -INFINITY ? 0.f : m * c - (std::is_same<T, __half>::value ? 7.f : 0.f);
      const float2 c2 = make_float2(c, c), ref2 = make_float2(-ref, -ref);
      float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int b = 0; b < G::kBlocks; ++b) {
        if (b >= nb) break;
        unsigned p[16];
        if (some[b]) {
          if constexpr (!kKeep) {
            tmem_ld32(my_s + b * 32, x[0]);
            mask(b, x[0], 0);
          }
          auto& y = x[kKeep ? b / 2 : 0];
          const int from = kKeep ? b % 2 * 32 : 0;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float2 w = fma2(make_float2(y[from + 2 * e], y[from + 2 * e + 1]), c2, ref2);
            w = make_float2(exp2_fast(w.x), exp2_fast(w.y));
            sums[e & 1] = add2(sums[e & 1], w);
            p[e] = pack2((T*)nullptr, w.x, w.y);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) p[e] = 0u;
        }
        tmem_st16(my_s + b * 16, p);
      }
      l += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[side]);
      ++n;
    }
    if (ok && n > 0) ok = wait(&o_full[side], n - 1);
    tc_fence_after();
    const bool good = __all_sync(0xffffffffu, ok && n > 0);
    T* const out = static_cast<T*>(a.out) + h * a.o_head;
    if (good) {
      // through this tile's place of the queries, which are done with: a row a thread in, whole lines out (8192
      // rows, window 512: 147 us, with 16-byte pieces straight from the threads, each to a line of its own, 151). Pieces
      // are exchanged by row, so that neither way meets in a bank.
      constexpr int kPieces = DP / 8, kRowBytes = DP * 2;
      unsigned char* mine = sq + side * G::kQBytes + (warp & 3) * 32 * kRowBytes;
      const float inv = 1.f / l;
      float finite = 0.f;  // NaN once a result is not finite
#pragma unroll
      for (int d = 0; d < DP; d += 32) {
        float o[32];
        tmem_ld32(my_o + d, o);
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          float r[8];
#pragma unroll
          for (int w = 0; w < 8; ++w) {
            r[w] = o[e + w] * inv;
            if (d + e < a.head_dim) finite = fmaf(r[w], 0.f, finite);
          }
          store8(reinterpret_cast<T*>(mine + lane * kRowBytes + (((d + e) / 8) ^ (lane & 7)) * 16), r);
        }
      }
      if (inside && finite != finite) sh_slow = 1;
      const unsigned rows_inside = __ballot_sync(0xffffffffu, inside);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int r = i * (32 / kPieces) + lane / kPieces, piece = lane % kPieces;
        if ((rows_inside >> r & 1u) && piece * 8 < a.head_dim)
          *reinterpret_cast<uint4*>(out + (row - lane + r) * a.o_row + piece * 8) =
              *reinterpret_cast<const uint4*>(mine + r * kRowBytes + (piece ^ (r & 7)) * 16);
      }
    } else if (inside) {
      for (int d = 0; d < a.head_dim; ++d) out[row * a.o_row + d] = static_cast<T>(NAN);
    }
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == G::kIssueWarp) tmem_dealloc(tmem, 2 * SUBS * DP);
  if (sh_slow && !sh_dead && warp < G::kCopyWarp) {
    constexpr int kLanes = DP / 8;
    const int side = warp >> 2;
    SubTile sub;
    sub.set(a, keys, first_row(side));
    if (sub.any)
      for (int r = sub.r0 + (threadIdx.x & 127) / kLanes; r <= sub.r1; r += 128 / kLanes) {
        const int start = sequence_start(a, r);
        if (start >= 0) window_row<T, kLanes>(a, r, start, head_of(side), threadIdx.x % kLanes, row_mask<kLanes>());
      }
  }
}

// ---------------------------------------------------------------- fp32 tiles
// 8 RT query rows of one head by 128 threads; thread (ty, tx) of 8 x 16 has rows
// RT ty .. + RT - 1 of everything, keys tx + 16 i of a 64-key tile in S, columns
// 64 i + 4 tx .. + 3 of O. With RT = 4 that is 16 multiply-adds for each 32 bytes
// read from shared memory; rows are padded by 16 bytes against bank conflicts. Key
// rows of the next tile load under the second product, value rows under the first.
// RT = 8 reads less and was slower, with half the warps an SM (2500 rows, window
// 300, 32 heads of 64: 269 us against 226, a third of the fp32 rate).
constexpr int kFp32Keys = 64, kFp32Threads = 128;

template <int DP, int RT>
struct Fp32Tiles {
  static constexpr int kRows = 8 * RT, kRow = DP + 4, kPRow = kFp32Keys + 4;
  static constexpr int kFloats = (kRows + 2 * kFp32Keys) * kRow + kRows * kPRow;
  static constexpr int kSmem = kFloats * 4;
};

__device__ __forceinline__ void copy16(float* dst, const float* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(in ? 16 : 0) : "memory");
}

template <int DP, int RT>
__global__ void __launch_bounds__(kFp32Threads) k_window_fp32(const WindowArgs a) {
  using G = Fp32Tiles<DP, RT>;
  extern __shared__ float4 dynamic[];
  float* sq = reinterpret_cast<float*>(dynamic);
  float *sk = sq + G::kRows * G::kRow, *sv = sk + kFp32Keys * G::kRow, *sp = sv + kFp32Keys * G::kRow;
  __shared__ int sh_slow;
  const int h = blockIdx.x % a.heads, tile = gridDim.x / a.heads - 1 - blockIdx.x / a.heads, kv = h / (a.heads / a.kv_heads);
  TileKeys keys;
  if (!tile_keys(a, (long long)tile * G::kRows, G::kRows, keys)) return;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  if (threadIdx.x == 0) sh_slow = 0;
  // A thread copies one column piece of every kStep-th row. Rows past the input, blocks past the tile's last and
  // columns past head_dim are zeros.
  constexpr int kPieces = DP / 4, kStep = kFp32Threads / kPieces;
  const int piece = threadIdx.x % kPieces * 4, my_row = threadIdx.x / kPieces;
  const bool on = piece < a.head_dim;
  auto copy_rows = [&](float* dst, const float* src, long long stride, long long row, int count, int most) {
    const float* p = src + (row + my_row) * stride + piece;
    dst += my_row * G::kRow + piece;
#pragma unroll
    for (int r = my_row; r < count; r += kStep, dst += kStep * G::kRow, p += kStep * stride) {
      const bool in = on && r < most;
      copy16(dst, in ? p : src, in);
    }
  };
  auto copy_tile = [&](float* dst, const void* src, long long stride, long long head, int block0) {
    const float* p = static_cast<const float*>(src) + head;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int block = block0 + b, row = block < keys.blocks ? keys.base(block) : 0;
      copy_rows(dst + b * kBlockRows * G::kRow, p, stride, row, kBlockRows,
                block < keys.blocks ? min(kBlockRows, a.rows - row) : 0);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  copy_rows(sq, static_cast<const float*>(a.q) + h * a.q_head, a.q_row, (long long)tile * G::kRows, G::kRows,
            (int)min((long long)G::kRows, a.rows - (long long)tile * G::kRows));
  copy_tile(sk, a.k, a.k_row, kv * a.k_head, 0);
  copy_tile(sv, a.v, a.v_row, kv * a.v_head, 0);

  RowLimits limits[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) limits[r].set(a, keys, tile * G::kRows + ty * RT + r);
  const int all_low = common_low(a, keys, keys.r1);
  const float c = a.scale * 1.4426950408889634f;
  float o[RT][DP / 64][4] = {}, m[RT], l[RT] = {};
#pragma unroll
  for (int r = 0; r < RT; ++r) m[r] = -INFINITY;
  for (int b0 = 0; b0 < keys.blocks; b0 += 2) {
    const bool more = b0 + 2 < keys.blocks;
    const bool plain = b0 >= keys.sink_blocks && b0 + 1 < keys.blocks && keys.base(b0) >= all_low &&
                       keys.base(b0 + 1) + kBlockRows - 1 <= keys.r0;
    asm volatile("cp.async.wait_group 1;" ::: "memory");  // queries and keys; the values may still be on their way
    __syncthreads();
    float s[RT][4] = {};
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
      float4 k[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) k[i] = *reinterpret_cast<const float4*>(sk + (tx + 16 * i) * G::kRow + d);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const float4 q = *reinterpret_cast<const float4*>(sq + (ty * RT + r) * G::kRow + d);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[r][i] = fmaf(q.x, k[i].x, s[r][i]);
          s[r][i] = fmaf(q.y, k[i].y, s[r][i]);
          s[r][i] = fmaf(q.z, k[i].z, s[r][i]);
          s[r][i] = fmaf(q.w, k[i].w, s[r][i]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const unsigned b[2] = {plain ? ~0u : limits[r].bits(keys, b0), plain ? ~0u : limits[r].bits(keys, b0 + 1)};
      float top = m[r];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[r][i] = (b[i / 2] >> (tx + 16 * (i & 1))) & 1u ? s[r][i] * c : -INFINITY;
        top = fmaxf(top, s[r][i]);
      }
#pragma unroll
      for (int d = 1; d < 16; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float ref = top == -INFINITY ? 0.f : top, keep = m[r] == -INFINITY ? 0.f : exp2_fast(m[r] - ref);
      m[r] = top;
      l[r] *= keep;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[r][i] = exp2_fast(s[r][i] - ref);
        l[r] += s[r][i];
        sp[(ty * RT + r) * G::kPRow + tx + 16 * i] = s[r][i];
      }
#pragma unroll
      for (int i = 0; i < DP / 64; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[r][i][e] *= keep;
    }
    __syncthreads();  // everybody is done with the keys
    if (more) copy_tile(sk, a.k, a.k_row, kv * a.k_head, b0 + 2);
    if (more) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // values and weights are there
#pragma unroll 2
    for (int j = 0; j < kFp32Keys; j += 4) {
      float4 v[4][DP / 64];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < DP / 64; ++i)
          v[e][i] = *reinterpret_cast<const float4*>(sv + (j + e) * G::kRow + i * 64 + tx * 4);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const float4 p = *reinterpret_cast<const float4*>(sp + (ty * RT + r) * G::kPRow + j);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float w = e == 0 ? p.x : e == 1 ? p.y : e == 2 ? p.z : p.w;
#pragma unroll
          for (int i = 0; i < DP / 64; ++i) {
            o[r][i][0] = fmaf(w, v[e][i].x, o[r][i][0]);
            o[r][i][1] = fmaf(w, v[e][i].y, o[r][i][1]);
            o[r][i][2] = fmaf(w, v[e][i].z, o[r][i][2]);
            o[r][i][3] = fmaf(w, v[e][i].w, o[r][i][3]);
          }
        }
      }
    }
    __syncthreads();  // everybody is done with the values and weights
    if (more) copy_tile(sv, a.v, a.v_row, kv * a.v_head, b0 + 2);
  }
  bool odd = false;  // a result that is not finite
#pragma unroll
  for (int r = 0; r < RT; ++r) {
#pragma unroll
    for (int d = 1; d < 16; d *= 2) l[r] += __shfl_xor_sync(0xffffffffu, l[r], d);
    if (limits[r].start < 0) continue;
    float* to = static_cast<float*>(a.out) + (long long)limits[r].row * a.o_row + h * a.o_head;
#pragma unroll
    for (int i = 0; i < DP / 64; ++i)
      if (i * 64 + tx * 4 < a.head_dim) {
        const float4 v = make_float4(o[r][i][0] / l[r], o[r][i][1] / l[r], o[r][i][2] / l[r], o[r][i][3] / l[r]);
        odd |= !(fabsf(v.x) < INFINITY && fabsf(v.y) < INFINITY && fabsf(v.z) < INFINITY && fabsf(v.w) < INFINITY);
        *reinterpret_cast<float4*>(to + i * 64 + tx * 4) = v;
      }
  }
  if (odd) sh_slow = 1;
  __syncthreads();
  if (sh_slow) {
    constexpr int kLanes = DP / 8;
    for (int r = keys.r0 + threadIdx.x / kLanes; r <= keys.r1; r += kFp32Threads / kLanes) {
      const int start = sequence_start(a, r);
      if (start >= 0) window_row<float, kLanes>(a, r, start, h, threadIdx.x % kLanes, row_mask<kLanes>());
    }
  }
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

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static std::atomic<EncodeTiled> fn{nullptr};
  EncodeTiled f = fn.load(std::memory_order_acquire);
  if (!f) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found{};
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess) {
      cudaGetLastError();  // the caller reports it
      return nullptr;
    }
    if (found != cudaDriverEntryPointSuccess) return nullptr;
    f = reinterpret_cast<EncodeTiled>(p);
    fn.store(f, std::memory_order_release);
  }
  return f;
}

// [rows][heads][head_dim] as a tensor whose boxes are 64 columns of `box_rows` rows of one head. Columns past
// head_dim and rows past `rows` read as zeros. A stride of 0 repeats its row or head; along a dimension of one element
// it is never used, whatever it is.
bool encode_rows(CUtensorMap* map, const st_rows& r, int mode, long long rows, int heads, int head_dim, int box_rows) {
  const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? r.head_stride : head_dim) * 2, (cuuint64_t)r.row_stride * 2};
  const cuuint32_t box[3] = {64, 1, (cuuint32_t)box_rows}, step[3] = {1, 1, 1};
  const EncodeTiled encode = encode_tiled();
  return encode && encode(map, mode == ST_MODE_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                          r.data, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP, int RT>
cudaError_t launch_fp32(const WindowArgs& a, cudaStream_t s) {
  using G = Fp32Tiles<DP, RT>;
  const cudaError_t e = cudaFuncSetAttribute(k_window_fp32<DP, RT>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem);
  if (e != cudaSuccess) return e;
  const unsigned tiles = (unsigned)((a.rows + G::kRows - 1ll) / G::kRows);
  k_window_fp32<DP, RT><<<tiles * a.heads, kFp32Threads, G::kSmem, s>>>(a);
  return cudaSuccess;
}
// Few rows are dealt to more CTAs, 1 or 2 a thread: as long as those of 1 find an SM each, and those of 2 a place (4
// heads of 64, window 64: 201 rows 6.6 us with 1, 7.7 with 2, 10.9 with 4; 400 rows 9.0, 7.7, 10.9; 1400 rows 17.1,
// 13.8, 14.8; 2000 rows 25.1, 16.4, 15.0. Of 128: 400 rows 15.4, 11.4, 16.0; 1000 rows 36.9, 17.5, 16.3).
template <int DP>
cudaError_t launch_fp32(const WindowArgs& a, cudaStream_t s) {
  constexpr long long kSms = 148;
  if ((a.rows + 7ll) / 8 * a.heads <= kSms) return launch_fp32<DP, 1>(a, s);
  if ((a.rows + 15ll) / 16 * a.heads <= kSms * (DP == 64 ? 3 : 1)) return launch_fp32<DP, 2>(a, s);
  return launch_fp32<DP, 4>(a, s);
}

template <typename T, int DP, int SUBS>
cudaError_t launch_tiles(const WindowArgs& a, const TileMaps& maps, cudaStream_t s) {
  using G = Tiles<DP, SUBS>;
  const cudaError_t e =
      cudaFuncSetAttribute(k_window_tiles<T, DP, SUBS>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem);
  if (e != cudaSuccess) return e;
  const unsigned tiles = (unsigned)((a.rows + kTileRows - 1ll) / kTileRows);
  const unsigned ctas =
      SUBS == 2 && a.heads / a.kv_heads % 2 == 0 ? tiles * (a.heads / 2) : (tiles + SUBS - 1) / SUBS * a.heads;
  k_window_tiles<T, DP, SUBS><<<ctas, G::kThreads, G::kSmem, s>>>(a, maps);
  return cudaSuccess;
}

// Up to 64 columns four CTAs of one query tile fit an SM. That is faster where no two heads share their keys (16 uneven
// backlogs, 16 heads of 64, window 256: 41.0 us, with two tiles a CTA 42.6; 200 rows 8.9 and 10.0) and slower where
// they do, as the keys then come twice (4 key heads of 16: 41.0 and 39.2; 8192 rows, 8 of 32, window 512: 97 and 94).
template <typename T>
cudaError_t launch_tiles(const WindowArgs& a, const TileMaps& maps, cudaStream_t s) {
  if (a.head_dim > 128) return launch_tiles<T, 256, 1>(a, maps, s);
  if (a.head_dim > 64) return launch_tiles<T, 128, 2>(a, maps, s);
  return a.heads / a.kv_heads % 2 == 0 ? launch_tiles<T, 64, 2>(a, maps, s) : launch_tiles<T, 64, 1>(a, maps, s);
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
  if (p->rows < 0 || p->rows > (1 << 30)) return cache_fail(ST_ERR_INVALID, "rows are 0 to 2^30");
  if (p->window < 1 || p->sinks < 0) return cache_fail(ST_ERR_INVALID, "window is at least 1 and sinks at least 0");
  if (p->starts ? p->sequences < 0 : p->sequences != 1)
    return cache_fail(ST_ERR_INVALID, "without starts there is one sequence");
  if (!(fabsf(p->scale) <= 0x1p64f)) return cache_fail(ST_ERR_INVALID, "scale must be within 2^64");
  if (p->rows == 0 || p->sequences == 0) return ST_OK;
  int rc;
  if ((rc = check_rows(p->q, "q", p->mode, p->rows, p->heads, p->head_dim, false)) != ST_OK ||
      (rc = check_rows(p->k, "k", p->mode, p->rows, p->kv_heads, p->head_dim, false)) != ST_OK ||
      (rc = check_rows(p->v, "v", p->mode, p->rows, p->kv_heads, p->head_dim, false)) != ST_OK ||
      (rc = check_rows(p->out, "out", p->mode, p->rows, p->heads, p->head_dim, true)) != ST_OK)
    return rc;
  if ((rc = check_aligned(p->starts, "starts", 4)) != ST_OK) return rc;
  const struct { const st_rows* rows; int heads; const char* name; } inputs[] = {
      {&p->q, p->heads, "q"}, {&p->k, p->kv_heads, "k"}, {&p->v, p->kv_heads, "v"}};
  for (const auto& x : inputs)  // what a tensor map takes
    if (p->mode != ST_MODE_FP32 && ((p->rows > 1 && x.rows->row_stride >= (int64_t)1 << 39) ||
                                    (x.heads > 1 && x.rows->head_stride >= (int64_t)1 << 39)))
      return cache_fail(ST_ERR_INVALID, ": strides of 16-bit rows are below 2^40 bytes", x.name);
  if (p->out.data == p->q.data || p->out.data == p->k.data || p->out.data == p->v.data)
    return cache_fail(ST_ERR_INVALID, "out may not be an input");
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
  // So few rows see so few keys that walking them one by one ends before a tile has been set up (bf16, 1 row: 2.2 us,
  // in tiles 4.6 at 64 columns and 6.3 at 128; 4 rows: 3.2 to 3.6, and 4.6 and 6.6; 16: 7.6 to 7.9, and 4.9 and 6.7).
  const bool few = p->rows <= 6;
  if (!few && p->mode == ST_MODE_FP32 && p->head_dim <= 128 && (p->rows + 31) / 32 * p->heads <= INT32_MAX) {
    if ((rc = cache_cuda(p->head_dim <= 64 ? launch_fp32<64>(a, s) : launch_fp32<128>(a, s), "window attention: ")) != ST_OK) {
      cudaGetLastError();  // reported here, so not left pending
      return rc;
    }
    return cache_cuda(cudaGetLastError(), "window attention launch: ");
  }
  TileMaps maps;
  const long long ctas = (p->rows + kTileRows - 1) / kTileRows * p->heads;
  if (!few && p->mode != ST_MODE_FP32 && p->scale > 0.f && ctas <= INT32_MAX) {
    if (!encode_rows(&maps.q, p->q, p->mode, p->rows, p->heads, p->head_dim, kTileRows) ||
        !encode_rows(&maps.k, p->k, p->mode, p->rows, p->kv_heads, p->head_dim, kBlockRows) ||
        !encode_rows(&maps.v, p->v, p->mode, p->rows, p->kv_heads, p->head_dim, kBlockRows))
      return cache_fail(ST_ERR_CUDA, "window attention: the driver takes no tensor map of the rows");
    const cudaError_t e = p->mode == ST_MODE_FP16 ? launch_tiles<__half>(a, maps, s) : launch_tiles<__nv_bfloat16>(a, maps, s);
    if (e != cudaSuccess) {
      cudaGetLastError();  // reported here, so not left pending
      return cache_cuda(e, "window attention: ");
    }
  } else if (p->mode == ST_MODE_FP32) {
    launch_window<float>(a, s);
  } else if (p->mode == ST_MODE_FP16) {
    launch_window<__half>(a, s);
  } else {
    launch_window<__nv_bfloat16>(a, s);
  }
  return cache_cuda(cudaGetLastError(), "window attention launch: ");
}
