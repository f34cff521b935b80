// Low-rank adapters of many requests beside a shared projection: with e the adapter of token t,
//   out[t] = base[t] + scale[e] b[e] (a[e] x[t]),   a (n, r, H), b (n, N, r);   out[t] = base[t] where t has none
// (base NULL: zeros).  Tokens are sorted by adapter, e's rows starting at a multiple of `align` (smoe_token_permutation), so that a tile of 16
// to `align` rows has one adapter.  x, base and out are met once each: between 20 and 200 operations for a byte of them, so that
// memory is the floor of all of this.  The kernels do not reach it: what holds each of them up is written there.
//
// The inner product is fp32: every warp's part by the tensor core's fp32 sums, the parts added in the same order every time.  s = scale[e] (a x) goes on
// as two 16-bit numbers, its leading bits and the rest (16 bits of s for bf16; 22 for fp16, after a row of s was multiplied by a power of two,
// which keeps it in range), and the second product takes both: rounding s to 16 bits alone would make the error of out half as large
// again where base is small.  out is rounded once.
//
// The blocks of a cluster share a tile of rows: each has a part of the columns of x and a, they add their products over distributed shared memory, and
// each computes a part of the columns of out.
//   few_kernel     (adapters.cu) tiles of 16 rows, clusters of eight; the warps of a block share the columns, and weights go straight from memory to
//                  registers: for few tokens, or few to an adapter, where weights are everything and latency counts
//   tile_kernel    (adapters_tile.cu) tiles of 32 to 128 rows of one adapter, a warp for 16 of them; the warps share the weights in shared memory
//   tensor_kernel  (adapters_tile.cu) tiles of 128 rows by tcgen05.mma, where rows of x, a and b are whole 16-byte pieces
//
// What the kernels share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/sonicmoe_b200.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace smoe {
namespace adapters {

constexpr int kMaxAdapters = 4096, kMaxRank = 128, kMaxRows = 0x7fff0000;
constexpr int kCluster = 8, kWarps = 8;   // of few_kernel; warps of a tile's blocks at most
constexpr int kGroup = 32;                // columns of out that a warp has at a time

struct Params {
  const char* x; long long x_ld;          // distances in bytes
  const char* a;
  const char* b;
  const float* scale;                     // (n) or nullptr
  const char* base; long long base_ld;    // or nullptr
  char* out; long long out_ld;
  const int* off;                         // (n + 1) first row of each adapter, ascending
  const int* count;                       // (n) its rows that have tokens
  const int* gather;                      // (rows) token of each row
  const int* reverse;                     // (T) row of each token
  int T, rows, H, N, n, r;
  int tiles;                              // at most
  int cluster;                            // blocks that share a tile
  int sparse;                             // few_kernel: most tiles of 16 rows may be empty, its tiles are the others
  int others;                             // tokens of a warp, of those that see to tokens without an adapter; 0: out is base, which holds them
  int* status;                            // tensor_kernel: set where a wait was given up, or nullptr
};

// ----------------------------------------------------------------------------------------------
// what the kernels share
// ----------------------------------------------------------------------------------------------
// c += a b: 16 rows of a, 8 columns of b, 16 products each.  Lane 4 g + t holds a[g][2t, 2t+1], a[g+8][..], a[g][2t+8, ..], a[g+8][..], b[2t, ..][g],
// b[2t+8, ..][g] and c[g][2t, 2t+1], c[g+8][..].
template <class T>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight 16-bit values that begin `o` bytes into v, at its beginning; those from the `left`-th on are zeros.
__device__ __forceinline__ void shift_down(uint32_t (&v)[8], int o, int left) {
#pragma unroll
  for (int i = 0; i < 6; ++i) v[i] = o & 8 ? v[i + 2] : v[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) v[i] = o & 4 ? v[i + 1] : v[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __funnelshift_r(v[i], v[i + 1], 8 * (o & 2));
  if (left < 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = left <= 2 * i ? 0u : left == 2 * i + 1 ? v[i] & 0xFFFFu : v[i];
  }
}

// Eight 16-bit values of a row from column `col` on (a multiple of 8), zeros behind its last column.  ALIGNED: rows start on 16-byte boundaries and
// have whole eights.  Otherwise the one or two 16-byte blocks that hold them are loaded, none that holds nothing of the row.
template <bool ALIGNED>
__device__ __forceinline__ uint4 load8(const char* row, int col, int cols) {
  if (col >= cols) return make_uint4(0u, 0u, 0u, 0u);
  if (ALIGNED) return *reinterpret_cast<const uint4*>(row + 2ll * col);
  const int o = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15);
  const char* p = row + 2ll * col - o;
  const uint4 q = *reinterpret_cast<const uint4*>(p);
  uint4 r = make_uint4(0u, 0u, 0u, 0u);
  if (o != 0 && 2 * (cols - col) + o > 16) r = *reinterpret_cast<const uint4*>(p + 16);
  uint32_t v[8] = {q.x, q.y, q.z, q.w, r.x, r.y, r.z, r.w};
  shift_down(v, o, cols - col);
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// load8 in two steps, so that many loads are on their way before the first is looked at.
template <bool ALIGNED>
struct Raw8 {
  uint4 q, r;
  __device__ __forceinline__ void load(const char* row, int col, int cols) {
    const int o = ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15);
    const char* p = row + 2ll * col - o;
    q = make_uint4(0u, 0u, 0u, 0u);
    if (col < cols) q = *reinterpret_cast<const uint4*>(p);
    if (!ALIGNED) {
      r = make_uint4(0u, 0u, 0u, 0u);
      if (o != 0 && 2ll * (cols - col) + o > 16) r = *reinterpret_cast<const uint4*>(p + 16);
    }
  }
  __device__ __forceinline__ uint4 get(const char* row, int col, int cols) const {
    if (ALIGNED) return q;
    uint32_t v[8] = {q.x, q.y, q.z, q.w, r.x, r.y, r.z, r.w};
    shift_down(v, static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15), cols - col);
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
};

// The same from a copy of the row's 16-byte blocks: eight values `o` bytes behind `p`, of which `left` belong to the row.
__device__ __forceinline__ uint4 in_place8(const char* p, int o, int left) {
  const uint4 q = *reinterpret_cast<const uint4*>(p), r = *reinterpret_cast<const uint4*>(p + 16);
  uint32_t v[8] = {q.x, q.y, q.z, q.w, r.x, r.y, r.z, r.w};
  shift_down(v, o, left);
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// The adapter of row `row` (all lanes of the warp): the last whose first row is not behind it.
__device__ __forceinline__ int adapter_of(const Params& p, int row) {
  const int lane = threadIdx.x & 31;
  int count = 0;
  for (int i = lane; i < p.n; i += 32) count += p.off[i] <= row;
  count = static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(count)));
  return min(max(count - 1, 0), p.n - 1);
}
// Whether rows from `row` on may have tokens.
__device__ __forceinline__ bool within(const Params& p, int row) { return row < min(p.off[p.n], p.rows); }
// The token of a row, or -1.  It is the row's if `reverse` says so too: a pair may have been dropped after the sort, in `reverse` alone.
__device__ __forceinline__ int gathered_of(const Params& p, int row) {
  if (row >= p.rows) return -1;
  const int t = p.gather[row];
  return static_cast<unsigned>(t) < static_cast<unsigned>(p.T) ? t : -1;
}

// The `tile`-th tile's adapter, first row and end, adapters in their order (all lanes of the warp); adapter -1 behind the last.  Each lane counts
// the tiles of a run of adapters; then the lanes look at the run that holds the tile.
__device__ __forceinline__ int4 tile_of(const Params& p, int tile, int tile_rows) {
  const int lane = threadIdx.x & 31;
  const auto tiles = [&](int e) { return (max(p.count[e], 0) + tile_rows - 1) / tile_rows; };
  const auto scan = [&](int v) {  // sum over the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int other = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += other;
    }
    return v;
  };
  const int run = (p.n + 31) / 32;
  int mine = 0;
  const int run_end = min(p.n, (lane + 1) * run);
#pragma unroll 4
  for (int e = lane * run; e < run_end; ++e) mine += tiles(e);
  int sum = scan(mine);
  unsigned found = __ballot_sync(0xffffffffu, tile < sum);
  if (found == 0u) return make_int4(-1, 0, 0, 0);
  const int who = __ffs(found) - 1;
  int before = __shfl_sync(0xffffffffu, sum - mine, who);
  const int end = min(p.n, (who + 1) * run);
  for (int e0 = who * run; e0 < end; e0 += 32) {
    const int here = e0 + lane < end ? tiles(e0 + lane) : 0;
    sum = before + scan(here);
    found = __ballot_sync(0xffffffffu, tile < sum);
    if (found != 0u) {
      const int at = __ffs(found) - 1, e = e0 + at;
      const int first = min(max(p.off[e], 0), p.rows);
      const long long row = first + static_cast<long long>(tile - __shfl_sync(0xffffffffu, sum - here, at)) * tile_rows;
      if (row < 0 || row >= p.rows) return make_int4(-1, 0, 0, 0);  // (counts that no sort gave)
      const long long end = min(row + tile_rows, static_cast<long long>(first) + max(p.count[e], 0));
      return make_int4(e, static_cast<int>(row), static_cast<int>(min(end, static_cast<long long>(p.rows))), 0);
    }
    before = __shfl_sync(0xffffffffu, sum, 31);
  }
  return make_int4(-1, 0, 0, 0);
}

// Ranks are padded to 16, 32, 64 or 128.
static inline int padded_rank(int r) { return r <= 16 ? 16 : r <= 32 ? 32 : r <= 64 ? 64 : 128; }

// Rows of tokens that no tile writes: base, or zeros.  A warp sees to tokens first .. end - 1: `begin` looks up the rows of the first 32, `finish` writes
// what no tile has, 16-byte blocks of out, four of a lane on their way together.
struct Others {
  int first, end, row;
  __device__ __forceinline__ void begin(const Params& p, int warp /* of the grid */) {
    first = static_cast<int>(min(static_cast<long long>(warp) * p.others, static_cast<long long>(p.T)));
    end = min(first + min(p.others, p.T - first), p.T);
    const int t = first + static_cast<int>(threadIdx.x & 31);
    row = t < end ? p.reverse[t] : -1;
  }
  __device__ __forceinline__ void finish(const Params& p) const {
    if (first >= end) return;
    const int lane = threadIdx.x & 31, sorted = min(p.off[p.n], p.rows);
    for (int at = first; at < end; at += 32) {
      const int t = at + lane, of = at == first ? row : t < end ? p.reverse[t] : -1;
      bool other = t < end;
      if (other && of >= 0 && of < sorted) other = p.gather[of] != t;
      for (unsigned todo = __ballot_sync(0xffffffffu, other); todo != 0u; todo &= todo - 1u)
        for (int c = 0; c < p.N; c += 1024) copy(p, at + __ffs(todo) - 1, c, min(c + 1024, p.N));
    }
  }
  static __device__ __forceinline__ void copy(const Params& p, int t, int c0, int c1) {
    const int lane = threadIdx.x & 31;
    char* out = p.out + t * p.out_ld;
    const char* base = p.base != nullptr ? p.base + t * p.base_ld : nullptr;
    // columns of the piece in front of out's next 16-byte boundary, and behind its last one, one by one
    const int head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(out + 2ll * c0) & 15)) & 15) / 2, c1 - c0), blocks = (c1 - c0 - head) / 8;
    const int edge = lane < 8 ? (lane < head ? c0 + lane : -1) : lane < 16 && c0 + head + 8 * blocks + lane - 8 < c1 ? c0 + head + 8 * blocks + lane - 8 : -1;
    Raw8<false> v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = lane + 32 * i, c = c0 + head + 8 * k;
      v[i].load(base + 2ll * c, 0, base != nullptr && k < blocks ? 8 : 0);
    }
    const uint16_t one = base != nullptr && edge >= 0 ? reinterpret_cast<const uint16_t*>(base)[edge] : static_cast<uint16_t>(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = lane + 32 * i, c = c0 + head + 8 * k;
      if (k < blocks) *reinterpret_cast<uint4*>(out + 2ll * c) = v[i].get(base + 2ll * c, 0, base != nullptr ? 8 : 0);
    }
    if (edge >= 0) reinterpret_cast<uint16_t*>(out)[edge] = one;
  }
};

// s as leading bits and the rest.  fp16: `factor` is a power of two that takes the row's largest |s| to 2^14; the product is multiplied by its inverse.
template <class T>
__device__ __forceinline__ float factor_of(float most) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return 1.f;
  const int e = static_cast<int>(__float_as_uint(most) >> 23);  // exponent + 127; 255: infinity, NaN
  if (e == 255 || most == 0.f) return 1.f;
  return __int_as_float(min(127 + 14 + 127 - e, 253) << 23);
}
template <class T>
__device__ __forceinline__ float inverse_of(float factor) {  // of a power of two
  return __int_as_float((254 << 23) - __float_as_int(factor));
}
template <class T>
__device__ __forceinline__ void split(float s, uint32_t& lead, uint32_t& rest) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const uint32_t bits = __float_as_uint(s);
    lead = bits >> 16;  // cut, so that it stays finite
    if ((bits & 0x7F800000u) == 0x7F800000u) {
      if ((bits & 0x7FFFFFu) != 0u) lead |= 0x40u;  // NaN stays NaN
      rest = 0u;
    } else {
      rest = __bfloat16_as_ushort(__float2bfloat16_rn(s - __uint_as_float(bits & 0xFFFF0000u)));
    }
  } else {
    const __half h = __float2half_rn(s);
    lead = __half_as_ushort(h);
    rest = (lead & 0x7C00u) == 0x7C00u ? 0u : __half_as_ushort(__float2half_rn(s - __half2float(h)));
  }
}
template <class T>
__device__ __forceinline__ void split2(float x, float y, uint32_t& lead, uint32_t& rest) {
  uint32_t l0, r0, l1, r1;
  split<T>(x, l0, r0);
  split<T>(y, l1, r1);
  lead = l0 | l1 << 16;
  rest = r0 | r1 << 16;
}

template <class T>
__device__ __forceinline__ float2 unpack(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <class T>
__device__ __forceinline__ uint32_t pack(float x, float y) {
  uint32_t w;
  if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(y), "f"(x));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(y), "f"(x));
  return w;
}
template <class T>
__device__ __forceinline__ float value(uint16_t w) { return unpack<T>(w).x; }

// The second product: 16 rows of s by columns n0 .. n0 + 31 of out.  Products are taken in an order that lets a lane load what lies together: of
// RP = 16 columns of s, lane t of a quad has 4t .. 4t + 3 (one step), of 32 it has 8t .. 8t + 7 (two steps).  And column 8 (g / 2) + 2 j + g % 2 of out
// is column g of product j, so that the four products give a lane the eight columns 8t .. 8t + 7 of out.
template <int RP>
struct Steps {
  static constexpr int K = RP / 16;                     // steps of 16
  static constexpr int L = RP == 16 ? 1 : RP / 32;      // loads of a lane for a row
};
// steps 2 l and 2 l + 1 (RP 16: step 0) of a product by one load `w` of a row of b
template <class T, int RP>
__device__ __forceinline__ void step(float (&c)[4], const uint32_t (&lead)[Steps<RP>::K][4], const uint32_t (&rest)[Steps<RP>::K][4], int l, uint4 w) {
  constexpr int two = RP == 16 ? 1 : 2;
#pragma unroll
  for (int k = 0; k < two; ++k) {
    const int i = two * l + k;
    const uint32_t b0 = k == 0 ? w.x : w.z, b1 = k == 0 ? w.y : w.w;
    mma<T>(c, lead[i][0], lead[i][1], lead[i][2], lead[i][3], b0, b1);
    mma<T>(c, rest[i][0], rest[i][1], rest[i][2], rest[i][3], b0, b1);
  }
}
__device__ __forceinline__ int out_column(int g, int j) { return 8 * (g >> 1) + 2 * j + (g & 1); }

// base + c inverse for the rows of tokens t0 (g) and t1 (g + 8), columns n0 + 8 t ..; nothing for a token of -1.  ALIGNED: eight columns at a time,
// else a warp's 16 rows one by one through `stage` (16 x 34 floats).
template <class T>
struct BaseRows {
  uint4 v[2];
  __device__ __forceinline__ void load(const Params& p, int n, int t0, int t1) {
    v[0] = v[1] = make_uint4(0u, 0u, 0u, 0u);
    if (p.base == nullptr || n >= p.N) return;
    if (t0 >= 0) v[0] = __ldcs(reinterpret_cast<const uint4*>(p.base + t0 * p.base_ld + 2ll * n));
    if (t1 >= 0) v[1] = __ldcs(reinterpret_cast<const uint4*>(p.base + t1 * p.base_ld + 2ll * n));
  }
};
// base + c inverse: eight columns of row g (half 0) or g + 8 (half 1)
template <class T>
__device__ __forceinline__ uint4 sum_row(const uint4& base, const float (&c)[4][4], int half, float inverse) {
  const uint32_t b[4] = {base.x, base.y, base.z, base.w};
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = unpack<T>(b[j]);
    o[j] = pack<T>(fmaf(c[j][2 * half], inverse, f.x), fmaf(c[j][2 * half + 1], inverse, f.y));
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}
template <class T>
__device__ __forceinline__ void put_row(const Params& p, int n, int t, const uint4& base, const float (&c)[4][4], int half, float inverse) {
  if (t < 0 || n >= p.N) return;
  __stcs(reinterpret_cast<uint4*>(p.out + t * p.out_ld + 2ll * n), sum_row<T>(base, c, half, inverse));
}
// Results of a row, columns n0 - 8 and on, to a row of out that starts anywhere, `shift` values behind a 16-byte boundary: block k of those from column n0 - shift
// on.  Only columns from `first` to below `end`, which others border on.
__device__ __forceinline__ void put_block(const Params& p, char* out, const char* results, int n0, int k, int shift, int first, int end) {
  const int col = n0 + 8 * k - shift, from = 2 * (8 + 8 * k - shift);
  const uint4 v = in_place8(results + (from & ~15), from & 15, 8);
  if (col >= first && col + 8 <= end) {
    __stcs(reinterpret_cast<uint4*>(out + 2ll * col), v);
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j >= first && col + j < end) reinterpret_cast<uint16_t*>(out)[col + j] = static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1)));
  }
}
// A warp's 16 rows of results, columns n0 - 8 .. n0 + 63: the blocks of out that end at n0 + 64 or before, and what is left of the row where `last`; otherwise
// that waits for the next columns.
__device__ __forceinline__ void put_shifted(const Params& p, const char* results, int pitch, int tokens /* of row `lane` % 16 */, int n0, int first, int end, bool last) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (lane >> 3) + 4 * i, k = lane & 7, token = __shfl_sync(0xffffffffu, tokens, row);
    if (token < 0) continue;
    char* out = p.out + token * p.out_ld;
    const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(out) & 15) / 2;
    put_block(p, out, results + row * pitch, n0, k, shift, first, end);
    if (last && k == 7 && shift > 0) put_block(p, out, results + row * pitch, n0, 8, shift, first, end);
  }
}
// Without whole pieces: a warp's 16 rows one by one, a column to a lane, by way of `stage` (16 x 34 floats).  Their base is fetched at once.
constexpr int kStagePitch = 34;
struct BaseColumn {
  uint16_t v[16];
  __device__ __forceinline__ void load(const Params& p, int n, int tokens /* of row `lane` % 16 */) {
#pragma unroll
    for (int row = 0; row < 16; ++row) {
      const int token = __shfl_sync(0xffffffffu, tokens, row);
      v[row] = p.base != nullptr && token >= 0 && n < p.N ? *reinterpret_cast<const uint16_t*>(p.base + token * p.base_ld + 2ll * n) : static_cast<uint16_t>(0);
    }
  }
};
template <class T>
__device__ __forceinline__ void put_staged(const Params& p, int n0, int tokens, const BaseColumn& base, const float (&c)[4][4], float inverse0, float inverse1, float* stage) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    *reinterpret_cast<float2*>(stage + g * kStagePitch + 8 * t + 2 * j) = make_float2(c[j][0] * inverse0, c[j][1] * inverse0);
    *reinterpret_cast<float2*>(stage + (g + 8) * kStagePitch + 8 * t + 2 * j) = make_float2(c[j][2] * inverse1, c[j][3] * inverse1);
  }
  __syncwarp();
  const int n = n0 + lane;
#pragma unroll
  for (int row = 0; row < 16; ++row) {
    const int token = __shfl_sync(0xffffffffu, tokens, row);
    const float f = stage[row * kStagePitch + lane] + value<T>(base.v[row]);
    if (token >= 0 && n < p.N) *reinterpret_cast<uint16_t*>(p.out + token * p.out_ld + 2ll * n) = static_cast<uint16_t>(pack<T>(f, 0.f));
  }
}

// What a lane needs of b for columns n0 .. n0 + 31 of out, straight from memory.
template <int RP, bool ALIGNED>
struct ColumnWeights {
  static constexpr int L = Steps<RP>::L;
  Raw8<ALIGNED> w[4][L];
  // (a row ends where b has no more)
  static __device__ __forceinline__ void place(const Params& p, const char* b, int n0, int j, int l, const char*& row, int& col, int& cols) {
    const int lane = threadIdx.x & 31, n = n0 + out_column(lane >> 2, j);
    row = b + static_cast<long long>(n) * p.r * 2;
    col = RP == 16 ? 8 * ((lane & 3) >> 1) : 32 * l + 8 * (lane & 3);
    cols = n < p.N ? p.r : 0;
  }
  __device__ __forceinline__ void load(const Params& p, const char* b, int n0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int l = 0; l < L; ++l) {
        const char* row;
        int col, cols;
        place(p, b, n0, j, l, row, col, cols);
        w[j][l].load(row, col, cols);
      }
    }
  }
  template <class T>
  __device__ __forceinline__ void multiply(const Params& p, const char* b, int n0, const uint32_t (&lead)[Steps<RP>::K][4], const uint32_t (&rest)[Steps<RP>::K][4], float (&c)[4][4]) const {
    const bool odd = threadIdx.x & 1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.f;
#pragma unroll
      for (int l = 0; l < L; ++l) {
        const char* row;
        int col, cols;
        place(p, b, n0, j, l, row, col, cols);
        uint4 v = w[j][l].get(row, col, cols);
        if (RP == 16 && odd) v = make_uint4(v.z, v.w, 0u, 0u);  // four of the eight are this lane's
        step<T, RP>(c[j], lead, rest, l, v);
      }
    }
  }
};

__device__ __forceinline__ float4 load_cluster(uint32_t addr) {
  float4 f;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(addr) : "memory");
  return f;
}

// Pitch of the blocks' parts in shared memory, in floats, for lanes that write two at a time in eight rows.
template <int RP>
constexpr int kPartPitch = RP + 8;

// Tiles of 16 `warps` rows, adapters_tile.cu.  wide_in: rows of x, a and b are whole 16-byte pieces; wide_out: those of base and out are.
int launch_tiles(const Params& p, int dtype, bool wide_in, bool wide_out, int warps, long long blocks, cudaStream_t st);

}  // namespace adapters
}  // namespace smoe
