// Low-rank adapters of many requests beside a shared projection: with e the adapter of token t,
//   out[t] = base[t] + scale[e] b[e] (a[e] x[t]),   a (n, r, H), b (n, N, r);   out[t] = base[t] where t has none
// (base NULL: zeros).  Tokens are sorted by adapter, e's rows starting at a multiple of `align` (smoe_token_permutation), so that a tile of 16
// to `align` rows has one adapter.  x, base and out are met once each: between 20 and 200 operations for a byte of them, so that the products
// go by mma.sync from registers and shared memory, whose rate they stay below, and memory bounds all of this.
//
// The inner product is fp32: every warp's part by the tensor core's fp32 sums, the parts added in the same order every time.  s = scale[e] (a x) goes on
// as two 16-bit numbers, its leading bits and the rest (16 bits of s for bf16; 22 for fp16, after a row of s was multiplied by a power of two,
// which keeps it in range), and the second product takes both: rounding s to 16 bits alone would make the error of out half as large
// again where base is small.  out is rounded once.
//
// In both kernels the blocks of a cluster share a tile of rows: each has a part of the columns of x and a, they add their products over distributed
// shared memory, and each computes a part of the columns of out.
//   few_kernel   tiles of 16 rows, clusters of eight; the warps of a block share the columns, and weights go straight from memory to registers: for few
//                tokens, or few to an adapter, where weights are everything and latency counts
//   tile_kernel  tiles of 32 to 128 rows of one adapter, a warp for 16 of them; the warps share the weights in shared memory
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
constexpr int kCluster = 8, kWarps = 8;   // of few_kernel; warps of tile_kernel at most
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
  int tiles;                              // few_kernel: of 16 rows; tile_kernel: at most
  int cluster;                            // tile_kernel: blocks that share a tile
  int copies;                             // pieces of other tokens' rows for a warp
  int sparse;                             // few_kernel: most tiles of 16 rows may be empty, its tiles are the others
  int in_place;                           // out is base
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
__device__ __forceinline__ int token_of(const Params& p, int row) {
  const int t = gathered_of(p, row);
  return t >= 0 && p.reverse[t] == row ? t : -1;
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
      const int at = __ffs(found) - 1, e = e0 + at, first = min(max(p.off[e], 0), p.rows);
      const int row = first + (tile - __shfl_sync(0xffffffffu, sum - here, at)) * tile_rows;
      return make_int4(e, row, min(min(row + tile_rows, first + max(p.count[e], 0)), p.rows), 0);
    }
    before = __shfl_sync(0xffffffffu, sum, 31);
  }
  return make_int4(-1, 0, 0, 0);
}

// Rows of tokens that no tile writes: base, or zeros.  A piece of work is 1024 columns of a token, `pieces` of them to each of `warps` warps, of which
// this is warp `warp` (all its lanes); 16-byte blocks of out, four of a lane on their way together.
constexpr int kCopyCols = 1024;
static long long copy_pieces(int T, int N) { return static_cast<long long>(T) * ((N + kCopyCols - 1) / kCopyCols); }
__device__ __forceinline__ void copy_others(const Params& p, long long warp) {
  const int lane = threadIdx.x & 31;
  const int end = min(p.off[p.n], p.rows), parts = (p.N + kCopyCols - 1) / kCopyCols;
  const long long all = static_cast<long long>(p.T) * parts;
  for (long long piece = warp * p.copies; piece < min((warp + 1) * p.copies, all); ++piece) {
    const int t = static_cast<int>(piece / parts), c0 = static_cast<int>(piece - static_cast<long long>(t) * parts) * kCopyCols, c1 = min(c0 + kCopyCols, p.N);
    const int row = p.reverse[t];
    if (row >= 0 && row < p.rows && row / 16 * 16 < end && p.gather[row] == t) continue;
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
}

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
// A warp's 16 rows of results, columns n0 - 8 .. n0 + 63, to rows of out that start anywhere: the 16-byte blocks of out that end at n0 + 64 or before, what
// is left waits for the next columns.  Columns from `first` on, where others have those before; `end`: of the last columns, whose rest goes
// out too.
__device__ __forceinline__ void put_shifted(const Params& p, const char* results, int pitch, int tokens /* of row `lane` % 16 */, int n0, int first, int end) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (lane >> 3) + 4 * i, token = __shfl_sync(0xffffffffu, tokens, row);
    if (token < 0) continue;
    char* out = p.out + token * p.out_ld;
    const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(out) & 15) / 2;  // values of out's first block in front of the row
    for (int k = lane & 7; k < (end != 0x7fffffff ? 9 : 8); k += 8) {
      const int col = n0 + 8 * k - shift, from = 2 * (8 + 8 * k - shift);
      if (k == 8 && shift == 0) continue;  // nothing is left
      const uint4 v = in_place8(results + row * pitch + (from & ~15), from & 15, 8);
      if (col >= first && col + 8 <= min(end, p.N)) {
        __stcs(reinterpret_cast<uint4*>(out + 2ll * col), v);
      } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (col + j >= first && col + j < min(end, p.N) && 8 * k - shift + j < 64)
            reinterpret_cast<uint16_t*>(out)[col + j] = static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1)));
        }
      }
    }
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

// ----------------------------------------------------------------------------------------------
// few rows
// ----------------------------------------------------------------------------------------------
__device__ __forceinline__ float4 load_cluster(uint32_t addr) {
  float4 f;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(addr) : "memory");
  return f;
}

// Pitches in shared memory, in floats: of parts, which lanes write two at a time in eight rows, and of s, which they read four at a time.
template <int RP>
struct Few {
  static constexpr int kPart = RP + 8, kS = RP + 4;
  static constexpr int kWarp = 16 * (kPart > kStagePitch ? kPart : kStagePitch);  // a warp's part, later its staged rows
  static constexpr size_t kSmem = sizeof(float) * (kWarps * kWarp + 16 * kPart + 16 * kS);
};

// AHEAD: a warp's weights and base for its first columns of out are on their way before the blocks add their parts, those of the next ones before the
// last are done, and more of x and a at a time.  That takes registers, so it is for as many blocks as there is room for at once.
template <class T, int RP, bool ALIGNED, bool AHEAD>
__global__ void __launch_bounds__(32 * kWarps, AHEAD ? 1 : RP == 16 ? (ALIGNED ? 4 : 2) : RP == 32 ? (ALIGNED ? 3 : 2) : RP == 64 && ALIGNED ? 2 : 1) few_kernel(const Params p) {
  release_next();
  wait_for_previous();
  using F = Few<RP>;
  extern __shared__ __align__(16) float smem[];
  float* parts = smem;                       // [warp][16][kPart]
  float* part = smem + kWarps * F::kWarp;    // [16][kPart]
  float* s_all = part + 16 * F::kPart;       // [16][kS]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rank = static_cast<int>(cluster_ctarank()), tile = blockIdx.x / kCluster;
  if (tile >= p.tiles) {
    const long long first = static_cast<long long>(p.tiles) * kCluster;
    copy_others(p, (blockIdx.x - first) * kWarps + warp);
    return;
  }
  // Loads of the row's tokens, of the adapters' rows, and then of all that hangs on them are on their way together; whether a row is still its token's
  // is looked at in the end.
  int row0 = 16 * tile, e;
  bool rows_here = true;
  if (p.sparse) {
    const int4 what = tile_of(p, tile, 16);
    e = max(what.x, 0);
    row0 = what.y;
    rows_here = what.x >= 0;
  } else {
    e = adapter_of(p, row0);
  }
  const int my_row = row0 + (lane & 15);
  const int candidate = gathered_of(p, my_row);
  if (!p.sparse) rows_here = within(p, row0);
  const int gathered = rows_here ? candidate : -1;
  if (__all_sync(0xffffffffu, gathered < 0)) return;  // (the cluster's blocks all see the same)
  const int row_of = gathered >= 0 ? p.reverse[gathered] : -1;
  const int x_t0 = __shfl_sync(0xffffffffu, gathered, g), x_t1 = __shfl_sync(0xffffffffu, gathered, g + 8);
  const int groups = (p.N + kGroup - 1) / kGroup;
  const int n_first = static_cast<int>(static_cast<long long>(groups) * rank / kCluster), n_end = static_cast<int>(static_cast<long long>(groups) * (rank + 1) / kCluster);
  const char* b = p.b + static_cast<long long>(e) * p.N * p.r * 2;
  {  // the L2 fetches the weights of this block's columns of out meanwhile
    const long long first = static_cast<long long>(n_first) * kGroup * p.r * 2, end = min(static_cast<long long>(n_end) * kGroup, static_cast<long long>(p.N)) * p.r * 2;
    for (long long o = first + 128ll * threadIdx.x; o < end; o += 128ll * blockDim.x) asm volatile("prefetch.global.L2 [%0];" ::"l"(b + o));
  }
  // a x over this warp's columns
  constexpr int NT = RP / 8;
  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  {
    const int chunks = (p.H + 31) / 32, parts_of = kCluster * kWarps, mine = rank * kWarps + warp;
    const int first = static_cast<int>(static_cast<long long>(chunks) * mine / parts_of), end = static_cast<int>(static_cast<long long>(chunks) * (mine + 1) / parts_of);
    const char* x0 = p.x + x_t0 * p.x_ld;
    const char* x1 = p.x + x_t1 * p.x_ld;
    const char* a = p.a + (static_cast<long long>(e) * p.r + g) * p.H * 2;
    const int width0 = x_t0 >= 0 ? p.H : 0, width1 = x_t1 >= 0 ? p.H : 0;
    constexpr int U = RP <= 32 || (RP == 64 && ALIGNED && AHEAD) ? 2 : 1;  // chunks whose loads are on their way together
    for (int c = first; c < end; c += U) {
      Raw8<ALIGNED> xa[U][2], w[U][NT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int col = c + u < end ? 32 * (c + u) + 8 * t : p.H;
        xa[u][0].load(x0, col, width0);
        xa[u][1].load(x1, col, width1);
#pragma unroll
        for (int j = 0; j < NT; ++j) w[u][j].load(a + 16ll * j * p.H, col, 8 * j + g < p.r ? p.H : 0);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int col = c + u < end ? 32 * (c + u) + 8 * t : p.H;
        const uint4 v0 = xa[u][0].get(x0, col, width0), v1 = xa[u][1].get(x1, col, width1);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 v = w[u][j].get(a + 16ll * j * p.H, col, 8 * j + g < p.r ? p.H : 0);
          mma<T>(acc[j], v0.x, v1.x, v0.y, v1.y, v.x, v.y);
          mma<T>(acc[j], v0.z, v1.z, v0.w, v1.w, v.z, v.w);
        }
      }
    }
  }
  int group = n_first + warp;
  ColumnWeights<RP, ALIGNED> weights;
  BaseRows<T> base;
  BaseColumn column;
  const auto fetch = [&] {
    if (group >= n_end) return;
    weights.load(p, b, kGroup * group);
    if (ALIGNED) base.load(p, kGroup * group + 8 * t, x_t0, x_t1);
    else column.load(p, kGroup * group + lane, gathered);
  };
  if (AHEAD && RP <= 64) fetch();
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    float* to = parts + warp * F::kWarp + g * F::kPart + 8 * j + 2 * t;
    *reinterpret_cast<float2*>(to) = make_float2(acc[j][0], acc[j][1]);
    *reinterpret_cast<float2*>(to + 8 * F::kPart) = make_float2(acc[j][2], acc[j][3]);
  }
  __syncthreads();
  constexpr int Q = RP / 4;  // fours of a row
#pragma unroll
  for (int i0 = 0; i0 < 16 * Q; i0 += 32 * kWarps) {
    const int i = i0 + threadIdx.x, at = i / Q * F::kPart + 4 * (i % Q);
    if (i >= 16 * Q) continue;
    float4 f = *reinterpret_cast<const float4*>(parts + at);
#pragma unroll
    for (int w = 1; w < kWarps; ++w) {
      const float4 v = *reinterpret_cast<const float4*>(parts + w * F::kWarp + at);
      f.x += v.x; f.y += v.y; f.z += v.z; f.w += v.w;
    }
    *reinterpret_cast<float4*>(part + at) = f;
  }
  cluster_sync_all();
  const float scale = p.scale != nullptr ? p.scale[e] : 1.f;
#pragma unroll
  for (int i0 = 0; i0 < 16 * Q; i0 += 32 * kWarps) {
    const int i = i0 + threadIdx.x;
    if (i >= 16 * Q) continue;
    const uint32_t at = smem_u32(part + i / Q * F::kPart + 4 * (i % Q));
    float4 f[kCluster];
#pragma unroll
    for (int k = 0; k < kCluster; ++k) f[k] = load_cluster(map_to_cta(at, k));
#pragma unroll
    for (int k = 1; k < kCluster; ++k) {
      f[0].x += f[k].x; f[0].y += f[k].y; f[0].z += f[k].z; f[0].w += f[k].w;
    }
    *reinterpret_cast<float4*>(s_all + i / Q * F::kS + 4 * (i % Q)) = make_float4(f[0].x * scale, f[0].y * scale, f[0].z * scale, f[0].w * scale);
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // this block has read the others' parts
  __syncthreads();
  // s in this warp's registers
  constexpr int K = Steps<RP>::K;
  uint32_t lead[K][4], rest[K][4];
  const auto fours = [&](int row, int k) {
    return *reinterpret_cast<const float4*>(s_all + row * F::kS + (RP == 16 ? 4 * t : 32 * (k / 2) + 8 * t + 4 * (k & 1)));
  };
  float f0 = 1.f, f1 = 1.f;
  if (std::is_same<T, __half>::value) {
    float most0 = 0.f, most1 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float4 u = fours(g, k), v = fours(g + 8, k);
      most0 = fmaxf(fmaxf(most0, fmaxf(fabsf(u.x), fabsf(u.y))), fmaxf(fabsf(u.z), fabsf(u.w)));
      most1 = fmaxf(fmaxf(most1, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
    }
#pragma unroll
    for (int o = 1; o < 4; o *= 2) {
      most0 = fmaxf(most0, __shfl_xor_sync(0xffffffffu, most0, o));
      most1 = fmaxf(most1, __shfl_xor_sync(0xffffffffu, most1, o));
    }
    f0 = factor_of<T>(most0);
    f1 = factor_of<T>(most1);
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const float4 u = fours(g, k), v = fours(g + 8, k);
    split2<T>(u.x * f0, u.y * f0, lead[k][0], rest[k][0]);
    split2<T>(v.x * f1, v.y * f1, lead[k][1], rest[k][1]);
    split2<T>(u.z * f0, u.w * f0, lead[k][2], rest[k][2]);
    split2<T>(v.z * f1, v.w * f1, lead[k][3], rest[k][3]);
  }
  const float i0 = inverse_of<T>(f0), i1 = inverse_of<T>(f1);
  const int tokens = row_of == my_row ? gathered : -1;
  const int t0 = __shfl_sync(0xffffffffu, tokens, g), t1 = __shfl_sync(0xffffffffu, tokens, g + 8);
  if (!AHEAD || RP > 64) fetch();
  while (group < n_end) {
    const int n0 = kGroup * group;
    float c[4][4];
    weights.template multiply<T>(p, b, n0, lead, rest, c);
    const BaseRows<T> base_now = base;
    const BaseColumn column_now = column;
    group += kWarps;
    if (AHEAD) fetch();
    if (ALIGNED) {
      put_row<T>(p, n0 + 8 * t, t0, base_now.v[0], c, 0, i0);
      put_row<T>(p, n0 + 8 * t, t1, base_now.v[1], c, 1, i1);
    } else {
      put_staged<T>(p, n0, tokens, column_now, c, i0, i1, parts + warp * F::kWarp);
    }
    if (!AHEAD) fetch();
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ----------------------------------------------------------------------------------------------
// tiles
// ----------------------------------------------------------------------------------------------
// Stages of 64 columns, `kStages` of them in turn: RP rows of a (or 64 of b) for the block, and each warp's 16 rows of x (or base), which it brings in
// itself.  ALIGNED: rows of 128 bytes by asynchronous copies; the halves of odd ones trade places, so that eight lanes of a load meet all
// banks.  Otherwise rows of x and base come in by the nine 16-byte blocks that hold them and are put in place on the way out of shared
// memory, weights on the way in.
template <int RP, bool ALIGNED>
struct Tile {
  static constexpr int kCols = 64, kStages = 3;
  static constexpr int kPitch = ALIGNED ? 128 : 144, kWarpBytes = 16 * kPitch, kWeightBytes = RP * 128;
  static constexpr int kOutPitch = 160;  // of a row of results on its way out: eight columns of the stage before, 64, and what a shifted load may touch
  // of a warp: s (leading bits, the rest), later its results
  static constexpr int kOwnBytes = 64 * RP > 16 * kOutPitch || ALIGNED ? 64 * RP : 16 * kOutPitch;
  static size_t smem(int warps) {
    const size_t stages = kStages * static_cast<size_t>(kWeightBytes + warps * kWarpBytes), part = sizeof(float) * 16 * warps * Few<RP>::kPart;
    return (stages > part ? stages : part) + static_cast<size_t>(warps) * kOwnBytes + sizeof(float) * 16 * warps;
  }
};
// place of the 16-byte block `k` of row `row`
__device__ __forceinline__ int swizzled(int row, int k) { return 16 * (k ^ ((row & 1) << 2)); }
// place of block `k` of row `row` among rows of RP 16-bit values
template <int RP>
__device__ __forceinline__ int weight_place(int row, int k) { return 2 * RP * row + (RP >= 64 ? swizzled(row, k) : 16 * k); }

__device__ __forceinline__ void store_cluster(uint32_t addr, uint2 v) {
  asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(v.x), "r"(v.y) : "memory");
}

// A warp's 16 rows on their way into shared memory: lane l has block l % 8 (and l % 8 = 0 the ninth) of the rows l / 8, + 4, + 8, + 12.
template <bool ALIGNED, int PITCH>
struct RowCopy {
  const char* row[4];  // the row's first block, or nullptr
  long long bytes[4];  // up to the row's end
  __device__ __forceinline__ void set(const char* rows, long long ld, int width, int tokens /* of row `lane` % 16 */) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int token = __shfl_sync(0xffffffffu, tokens, (lane >> 3) + 4 * i);
      const char* p = rows + token * ld;
      const int off = ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
      row[i] = token >= 0 && rows != nullptr ? p - off : nullptr;
      bytes[i] = off + 2ll * width;
    }
  }
  // columns 64 stage and on; zeros behind the row's end
  __device__ __forceinline__ void fetch(char* to, int stage, const void* some /* an address for copies of nothing */) const {
    const int lane = threadIdx.x & 31, k = lane & 7;
    const char* none = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(some) & ~static_cast<uintptr_t>(15));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = (lane >> 3) + 4 * i;
      const long long at = 128ll * stage + 16 * k;
      const bool has = row[i] != nullptr && at < bytes[i];
      cp_async16(smem_u32(to + r * PITCH + (ALIGNED ? swizzled(r, k) : 16 * k)), has ? row[i] + at : none, has ? 16 : 0);
      if (!ALIGNED && k == 0) {
        const bool more = row[i] != nullptr && at + 128 < bytes[i];
        cp_async16(smem_u32(to + r * PITCH + 128), more ? row[i] + at + 128 : none, more ? 16 : 0);
      }
    }
  }
};
// eight columns from 8 k of a stage on, of row `r`, which begins `off` bytes into its first block; `left`: columns of the row from there on
template <bool ALIGNED, int PITCH>
__device__ __forceinline__ uint4 staged_row(const char* from, int r, int k, int off, int left) {
  if (ALIGNED) return *reinterpret_cast<const uint4*>(from + r * PITCH + swizzled(r, k));
  return in_place8(from + r * PITCH + 16 * k, off, left);
}

// One block of rows of weights, RP or 64 of them, 64 or RP columns each, into shared memory by all threads.
template <bool ALIGNED, class Place>
__device__ __forceinline__ void fetch_weights(char* to, const char* from, int width /* of a row in memory */, int rows, int rows_left, int col, int cols, Place place) {
  const int per = cols / 8;
  for (int i = threadIdx.x; i < rows * per; i += blockDim.x) {
    const int row = i / per, k = i % per, c = col + 8 * k;
    const char* p = from + 2ll * width * row;
    const bool has = row < rows_left && c < width;
    if (ALIGNED) cp_async16(smem_u32(to + place(row, k)), has ? p + 2ll * c : from, has ? 16 : 0);
    else *reinterpret_cast<uint4*>(to + place(row, k)) = load8<false>(p, has ? c : width, width);
  }
}

template <class T, int RP, bool ALIGNED>
__global__ void __launch_bounds__(32 * kWarps, RP <= 64 ? 2 : 1) tile_kernel(const Params p) {
  release_next();
  wait_for_previous();
  using Ti = Tile<RP, ALIGNED>;
  extern __shared__ __align__(128) char smem_tile[];
  constexpr int COLS = Ti::kCols, STAGES = Ti::kStages, PITCH = Ti::kPitch, NT = RP / 8, C = COLS / 32, K = Steps<RP>::K, L = Steps<RP>::L;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, warps = blockDim.x / 32, tile_rows = 16 * warps;
  const int tile = blockIdx.x / p.cluster, share = blockIdx.x - tile * p.cluster;
  if (tile >= p.tiles) {
    const long long first = static_cast<long long>(p.tiles) * p.cluster;
    copy_others(p, (blockIdx.x - first) * warps + warp);
    return;
  }
  const int4 what = tile_of(p, tile, tile_rows);
  if (what.x < 0) return;  // (the cluster's blocks all see the same)
  const int e = what.x, my_row = what.y + 16 * warp + (lane & 15);
  const int gathered = my_row < what.z ? gathered_of(p, my_row) : -1;
  const bool any = __any_sync(0xffffffffu, gathered >= 0);
  const int row_of = gathered >= 0 ? p.reverse[gathered] : -1;  // what is read of a token does not wait for the check that the row is still its own
  const int stage_bytes = Ti::kWeightBytes + warps * Ti::kWarpBytes;
  const auto weights_in = [&](int stage) { return smem_tile + stage % STAGES * stage_bytes; };
  const auto rows_in = [&](int stage) { return weights_in(stage) + Ti::kWeightBytes + warp * Ti::kWarpBytes; };
  const size_t ring = max(static_cast<size_t>(STAGES) * stage_bytes, sizeof(float) * tile_rows * Few<RP>::kPart);
  char* own = smem_tile + ring;                                                // [warp][lead: 16 x RP, rest: 16 x RP]
  float* inverses = reinterpret_cast<float*>(own + warps * Ti::kOwnBytes);     // [tile_rows]
  const auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
  const auto range = [&](int all, int& first, int& end) {
    first = static_cast<int>(static_cast<long long>(all) * share / p.cluster);
    end = static_cast<int>(static_cast<long long>(all) * (share + 1) / p.cluster);
  };

  // s, of this block's columns of x
  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  {
    int first, end;
    range((p.H + COLS - 1) / COLS, first, end);
    const char* a = p.a + static_cast<long long>(e) * p.r * p.H * 2;
    RowCopy<ALIGNED, PITCH> x;
    x.set(p.x, p.x_ld, p.H, gathered);
    const auto fetch = [&](int stage) {
      if (stage < end) {
        if (any) x.fetch(rows_in(stage), stage, p.x);
        fetch_weights<ALIGNED>(weights_in(stage), a, p.H, RP, p.r, COLS * stage, COLS, [](int row, int k) { return 128 * row + swizzled(row, k); });
      }
      commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch(first + i);
    const int t0 = __shfl_sync(0xffffffffu, gathered, g), t1 = __shfl_sync(0xffffffffu, gathered, g + 8);
    const int o0 = ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(p.x + t0 * p.x_ld) & 15), o1 = ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(p.x + t1 * p.x_ld) & 15);
    for (int stage = first; stage < end; ++stage) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      __syncthreads();  // the stage is there for all, and the one whose place the next takes has been read
      fetch(stage + STAGES - 1);
      if (!any) continue;
      const char* xs = rows_in(stage);
      const char* ws = weights_in(stage);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int left = p.H - (COLS * stage + 32 * c + 8 * t);
        const uint4 x0 = staged_row<ALIGNED, PITCH>(xs, g, 4 * c + t, o0, left), x1 = staged_row<ALIGNED, PITCH>(xs, g + 8, 4 * c + t, o1, left);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 w = *reinterpret_cast<const uint4*>(ws + 128 * (8 * j + g) + swizzled(g, 4 * c + t));
          mma<T>(acc[j], x0.x, x1.x, x0.y, x1.y, w.x, w.y);
          mma<T>(acc[j], x0.z, x1.z, x0.w, x1.w, w.z, w.w);
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
  }

  // the blocks add their parts, each for a share of the rows, and give all of them the sums
  constexpr int PART = Few<RP>::kPart;
  float* part = reinterpret_cast<float*>(smem_tile);  // [tile_rows][PART]
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    float* to = part + (16 * warp + g) * PART + 8 * j + 2 * t;
    *reinterpret_cast<float2*>(to) = make_float2(acc[j][0], acc[j][1]);
    *reinterpret_cast<float2*>(to + 8 * PART) = make_float2(acc[j][2], acc[j][3]);
  }
  cluster_sync_all();
  {
    const float scale = p.scale != nullptr ? p.scale[e] : 1.f;
    constexpr int Q = RP / 4;  // threads of a row, four columns each
    const int mine = tile_rows / p.cluster;
    for (int first_of = 0; first_of < mine * Q; first_of += blockDim.x) {  // (all threads, for the shuffles)
      const int i = first_of + threadIdx.x;
      const bool live = i < mine * Q;
      const int row = share * mine + (live ? i / Q : 0), q = i % Q;
      float f[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int k = 0; k < p.cluster; ++k) {
        const float4 v = load_cluster(map_to_cta(smem_u32(part + row * PART + 4 * q), k));
        f[0] += v.x; f[1] += v.y; f[2] += v.z; f[3] += v.w;
      }
      float most = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[j] *= scale;
        most = fmaxf(most, fabsf(f[j]));
      }
#pragma unroll
      for (int o = 1; o < Q; o *= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      const float factor = factor_of<T>(most);
      uint2 lead, rest;
      split2<T>(f[0] * factor, f[1] * factor, lead.x, rest.x);
      split2<T>(f[2] * factor, f[3] * factor, lead.y, rest.y);
      if (live) {
        const uint32_t to = smem_u32(own + row / 16 * Ti::kOwnBytes) + weight_place<RP>(row % 16, q / 2) + 8 * (q & 1);
        for (int k = 0; k < p.cluster; ++k) {
          store_cluster(map_to_cta(to, k), lead);
          store_cluster(map_to_cta(to + 32 * RP, k), rest);
          if (std::is_same<T, __half>::value && q == 0)
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(map_to_cta(smem_u32(inverses + row), k)), "f"(inverse_of<T>(factor)) : "memory");
        }
      }
    }
  }
  cluster_sync_all();

  // this block's columns of out
  int first, end;
  range((p.N + COLS - 1) / COLS, first, end);
  const char* b = p.b + static_cast<long long>(e) * p.N * p.r * 2;
  const int tokens = row_of == my_row ? gathered : -1;
  const bool writes = __any_sync(0xffffffffu, tokens >= 0);
  const int t0 = __shfl_sync(0xffffffffu, tokens, g), t1 = __shfl_sync(0xffffffffu, tokens, g + 8);
  RowCopy<ALIGNED, PITCH> base;
  base.set(p.base, p.base_ld, p.N, tokens);
  const auto fetch = [&](int stage) {
    if (stage < end) {
      if (writes && p.base != nullptr) base.fetch(rows_in(stage), stage, p.x);
      fetch_weights<ALIGNED>(weights_in(stage), b + 2ll * COLS * stage * p.r, p.r, COLS, p.N - COLS * stage, 0, RP, weight_place<RP>);
    }
    commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(first + i);
  uint32_t lead[K][4], rest[K][4];
  {
    const char* mine = own + warp * Ti::kOwnBytes;
#pragma unroll
    for (int l = 0; l < L; ++l) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // rows g and g + 8
        if constexpr (RP == 16) {
          const uint2 u = *reinterpret_cast<const uint2*>(mine + weight_place<RP>(g + 8 * h, 0) + 8 * t), v = *reinterpret_cast<const uint2*>(mine + 32 * RP + weight_place<RP>(g + 8 * h, 0) + 8 * t);
          lead[0][h] = u.x; lead[0][2 + h] = u.y;
          rest[0][h] = v.x; rest[0][2 + h] = v.y;
        } else {
          const uint4 u = *reinterpret_cast<const uint4*>(mine + weight_place<RP>(g + 8 * h, 4 * l + t)), v = *reinterpret_cast<const uint4*>(mine + 32 * RP + weight_place<RP>(g + 8 * h, 4 * l + t));
          lead[2 * l][h] = u.x; lead[2 * l][2 + h] = u.y; lead[2 * l + 1][h] = u.z; lead[2 * l + 1][2 + h] = u.w;
          rest[2 * l][h] = v.x; rest[2 * l][2 + h] = v.y; rest[2 * l + 1][h] = v.z; rest[2 * l + 1][2 + h] = v.w;
        }
      }
    }
  }
  const float i0 = std::is_same<T, __half>::value ? inverses[16 * warp + g] : 1.f, i1 = std::is_same<T, __half>::value ? inverses[16 * warp + g + 8] : 1.f;
  const int o0 = ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(p.base + t0 * p.base_ld) & 15), o1 = ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(p.base + t1 * p.base_ld) & 15);
  __syncwarp();  // s has been read: the results may lie there
  char* results = own + warp * Ti::kOwnBytes;
  for (int stage = first; stage < end; ++stage) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncthreads();
    fetch(stage + STAGES - 1);
    if (!writes) continue;
    const char* bs = rows_in(stage);
    const char* ws = weights_in(stage);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int n0 = COLS * stage + kGroup * i;
      float c[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.f;
        const int row = kGroup * i + out_column(g, j);
#pragma unroll
        for (int l = 0; l < L; ++l) {
          uint4 w = make_uint4(0u, 0u, 0u, 0u);
          if constexpr (RP == 16) {
            const uint2 h = *reinterpret_cast<const uint2*>(ws + weight_place<RP>(row, 0) + 8 * t);
            w.x = h.x;
            w.y = h.y;
          } else {
            w = *reinterpret_cast<const uint4*>(ws + weight_place<RP>(row, 4 * l + t));
          }
          step<T, RP>(c[j], lead, rest, l, w);
        }
      }
      uint4 b0 = make_uint4(0u, 0u, 0u, 0u), b1 = b0;
      if (p.base != nullptr) {
        const int left = p.N - (n0 + 8 * t);
        b0 = staged_row<ALIGNED, PITCH>(bs, g, 4 * i + t, o0, left);
        b1 = staged_row<ALIGNED, PITCH>(bs, g + 8, 4 * i + t, o1, left);
      }
      const uint4 r0 = sum_row<T>(b0, c, 0, i0), r1 = sum_row<T>(b1, c, 1, i1);
      if (ALIGNED) {
        const int n = n0 + 8 * t;
        if (t0 >= 0 && n < p.N) __stcs(reinterpret_cast<uint4*>(p.out + t0 * p.out_ld + 2ll * n), r0);
        if (t1 >= 0 && n < p.N) __stcs(reinterpret_cast<uint4*>(p.out + t1 * p.out_ld + 2ll * n), r1);
      } else {
        *reinterpret_cast<uint4*>(results + g * Ti::kOutPitch + 16 + 64 * i + 16 * t) = r0;
        *reinterpret_cast<uint4*>(results + (g + 8) * Ti::kOutPitch + 16 + 64 * i + 16 * t) = r1;
      }
    }
    if (!ALIGNED) {
      __syncwarp();
      put_shifted(p, results, Ti::kOutPitch, tokens, COLS * stage, COLS * first, stage + 1 == end ? min(COLS * end, p.N) : 0x7fffffff);
      __syncwarp();
      if (lane < 16) *reinterpret_cast<uint4*>(results + lane * Ti::kOutPitch) = *reinterpret_cast<const uint4*>(results + lane * Ti::kOutPitch + 128);
      __syncwarp();
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ----------------------------------------------------------------------------------------------
// launches
// ----------------------------------------------------------------------------------------------
static int padded_rank(int r) { return r <= 16 ? 16 : r <= 32 ? 32 : r <= 64 ? 64 : 128; }
// Tiles of `rows` rows, at most: what the adapters' tokens fill, and a part of one more each.
static long long tiles_of(int T, int n, int rows) {
  const long long tiles = T / rows + static_cast<long long>(n < T ? n : T);
  return tiles < T ? tiles : T;
}
static bool by_few_rows(int T, int n, int r) { return tiles_of(T, n, 16) * padded_rank(r) <= 4096; }
// Warps of tile_kernel's blocks, by the tokens that an adapter has on average.
static int warps_of(int T, int n) { return T / n <= 32 ? 2 : T / n <= 64 ? 4 : 8; }
// Blocks of few_kernel with AHEAD that an SM has room for.
template <int RP, bool ALIGNED>
constexpr int kAheadBlocks = RP == 16 ? (ALIGNED ? 3 : 2) : RP == 32 && ALIGNED ? 2 : 1;

template <class T, int RP, bool ALIGNED>
static int launch(Params p, cudaStream_t st) {
  static PerDeviceFlag configured;
  const int dev = current_device();
  if (dev < 0) return SMOE_ERR_DRIVER;
  if (!configured.test(dev)) {
    if (cudaFuncSetAttribute(few_kernel<T, RP, ALIGNED, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Few<RP>::kSmem)) != cudaSuccess ||
        cudaFuncSetAttribute(few_kernel<T, RP, ALIGNED, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Few<RP>::kSmem)) != cudaSuccess ||
        cudaFuncSetAttribute(tile_kernel<T, RP, ALIGNED>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Tile<RP, ALIGNED>::smem(kWarps))) != cudaSuccess)
      return SMOE_ERR_LAUNCH;
    configured.set(dev);
  }
  const bool few = by_few_rows(p.T, p.n, p.r);
  const int warps = few ? kWarps : warps_of(p.T, p.n);
  p.sparse = (p.rows + 15) / 16 > tiles_of(p.T, p.n, 16);
  p.tiles = static_cast<int>(!few ? tiles_of(p.T, p.n, 16 * warps) : p.sparse ? tiles_of(p.T, p.n, 16) : (p.rows + 15) / 16);
  const int full = (p.T + 16 * warps - 1) / (16 * warps);  // tiles, if they were all full
  p.cluster = few ? kCluster : full > 148 ? 1 : full > 74 ? 2 : full > 37 ? 4 : 8;
  // the other tokens: a piece to a warp, or up to eight where that makes more blocks than the device takes at a time
  const long long pieces = p.in_place ? 0 : copy_pieces(p.T, p.N), room = 148 * 4 * kWarps;
  p.copies = static_cast<int>(pieces <= room ? 1 : pieces >= 8 * room ? 8 : pieces / room);
  const long long to_a_cluster = static_cast<long long>(p.copies) * warps * p.cluster;
  const long long blocks = (p.tiles + (pieces + to_a_cluster - 1) / to_a_cluster) * p.cluster;
  if (blocks > 0x7fffffffll) return SMOE_ERR_SHAPE;
  if (blocks == 0) return SMOE_OK;
  const bool ahead = tiles_of(p.T, p.n, 16) * kCluster <= 148 * kAheadBlocks<RP, ALIGNED>;
  return launched(few ? launch_chained(ahead ? few_kernel<T, RP, ALIGNED, true> : few_kernel<T, RP, ALIGNED, false>, dim3(static_cast<unsigned>(blocks)), 32 * warps, Few<RP>::kSmem, st, p.cluster, p)
                      : launch_chained(tile_kernel<T, RP, ALIGNED>, dim3(static_cast<unsigned>(blocks)), 32 * warps, Tile<RP, ALIGNED>::smem(warps), st, p.cluster, p));
}
template <class T, bool ALIGNED>
static int launch(const Params& p, cudaStream_t st) {
  switch (padded_rank(p.r)) {
    case 16: return launch<T, 16, ALIGNED>(p, st);
    case 32: return launch<T, 32, ALIGNED>(p, st);
    case 64: return launch<T, 64, ALIGNED>(p, st);
    default: return launch<T, 128, ALIGNED>(p, st);
  }
}

static long long address(const void* p) { return static_cast<long long>(reinterpret_cast<uintptr_t>(p)); }

}  // namespace adapters
}  // namespace smoe

using namespace smoe;
using namespace smoe::adapters;

extern "C" {

int smoe_adapter_linear(const void* x, long long ld, const void* a, const void* b, const float* scale, const void* base, long long base_ld,
                        void* out, long long out_ld, int dtype, const int* expert_frequency_offset, const int* expert_frequency,
                        const int* x_gather_idx, const int* s_reverse_scatter_idx, int T, long long rows, int H, int N, int n, int r, int align, void* stream) {
  if (dtype != SMOE_BF16 && dtype != SMOE_F16) return SMOE_ERR_DTYPE;
  if (T < 0 || T > kMaxRows || rows < 0 || rows > kMaxRows || H <= 0 || N <= 0 || n <= 0 || n > kMaxAdapters || r <= 0 || r > kMaxRank || align <= 0 ||
      align % 16 != 0 || ld < 0 || base_ld < 0 || out_ld < N)
    return SMOE_ERR_SHAPE;
  if (H > 1 << 28 || N > 1 << 28) return SMOE_ERR_SHAPE;
  if (T == 0) return SMOE_OK;
  if (x == nullptr || a == nullptr || b == nullptr || out == nullptr || expert_frequency_offset == nullptr || expert_frequency == nullptr || s_reverse_scatter_idx == nullptr ||
      (rows > 0 && x_gather_idx == nullptr))
    return SMOE_ERR_SHAPE;
  if ((address(x) | address(a) | address(b) | address(base) | address(out)) % 2 != 0 ||
      (address(scale) | address(expert_frequency_offset) | address(expert_frequency) | address(x_gather_idx) | address(s_reverse_scatter_idx)) % 4 != 0)
    return SMOE_ERR_ALIGNMENT;
  Params p = {};
  p.x = static_cast<const char*>(x); p.x_ld = 2 * ld;
  p.a = static_cast<const char*>(a); p.b = static_cast<const char*>(b); p.scale = scale;
  p.base = static_cast<const char*>(base); p.base_ld = base != nullptr ? 2 * base_ld : 0;
  p.out = static_cast<char*>(out); p.out_ld = 2 * out_ld;
  p.off = expert_frequency_offset; p.count = expert_frequency; p.gather = x_gather_idx; p.reverse = s_reverse_scatter_idx;
  p.T = T; p.rows = static_cast<int>(rows); p.H = H; p.N = N; p.n = n; p.r = r;
  p.in_place = base == out && base_ld == out_ld;
  const bool aligned = (address(x) | address(a) | address(b) | address(base) | address(out) | p.x_ld | p.base_ld | p.out_ld) % 16 == 0 && H % 8 == 0 &&
                       N % 8 == 0 && r % 8 == 0;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == SMOE_BF16) return aligned ? launch<__nv_bfloat16, true>(p, st) : launch<__nv_bfloat16, false>(p, st);
  return aligned ? launch<__half, true>(p, st) : launch<__half, false>(p, st);
}

}  // extern "C"
