// Tokens sorted by expert and back, for experts that are not this library's own GEMMs.
//
//   permutation   row(p) = offset[e_p] + rank of p among the pairs of expert e_p  (stable: by flat slot p = t K + k)
//                 offset[e + 1] = offset[e] + count[e] rounded up to a multiple of `align`
//   spread        rows[row(t, k)] = w[t, k] x[t], zeros in rows without a pair; also the gradient of the combine by its rows,
//                 and with it dw[t, k] = <dout[t], rows[row(t, k)]>
//   collect       out[t] = sum over k of w[t, k] rows[row(t, k)]; also the gradient of the sort by x (w = 1)
//
// A pair whose expert is not in [0, E) is dropped: it has no row (-1), adds nothing and its weight is not read.  So is one whose
// row number is taken out of `row` later on: a row has a pair where `slot` and `row` name one another.  Everything here
// is bound by memory.  The row movers go token by token, not row by row: a token's row is read once for its K places (expert
// by expert the whole of x would be read up to K times), and the sum over k stays in registers, in fp32, in the order of k.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>
#include <type_traits>

#include "../../include/sonicmoe_b200.h"
#include "launch.cuh"
#include "rows16.cuh"

namespace smoe {
namespace permute {

static inline cudaStream_t S(void* s) { return static_cast<cudaStream_t>(s); }

// ----------------------------------------------------------------------------------------------
// the permutation
// ----------------------------------------------------------------------------------------------
constexpr int kMaxExperts = 4096;
constexpr int kMaxBlocks = 256;
constexpr int kWarps = 8, kSteps = 8;                 // warps of a block; groups of 32 pairs that a warp has at a time, at most
constexpr int kScanWarps = 4;
constexpr int kOneWarps = 32;                         // the form with one block
constexpr int kOneMaxPairs = 2048, kOneMaxExperts = 1024;
static_assert(kOneMaxPairs <= kOneWarps * kSteps * 32, "pairs that the block's registers hold");

struct Plan {
  const void* idx;   // (n) int32 or int64
  int wide;          // int64
  int n, K, E, align, rows;
  int* count;        // (E)
  int* offset;       // (E + 1)
  int* token;        // (rows)
  int* slot;         // (rows)
  int* row;          // (n)
  int* hist;         // (E, kMaxBlocks): pairs of each expert in a block's chunk, then in the chunks before
};

// expert of pair p, or -1
__device__ __forceinline__ int expert_of(const Plan& a, int p) {
  if (p >= a.n) return -1;
  const long long e = a.wide ? static_cast<const long long*>(a.idx)[p] : static_cast<const int*>(a.idx)[p];
  return e >= 0 && e < a.E ? static_cast<int>(e) : -1;
}

// Exclusive prefix of v over the block's threads; *total: its sum.  partial: one word per warp.
__device__ __forceinline__ int block_scan(int v, int* partial, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int incl = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 31) partial[warp] = incl;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < warps; ++w) {
    const int s = partial[w];
    if (w < warp) before += s;
    all += s;
  }
  __syncthreads();
  *total = all;
  return before + incl - v;
}

// Rank of every pair of this warp's 32 * steps among the warp's pairs of the same expert; cnt: the warp's counters.
__device__ __forceinline__ void rank_pairs(const Plan& a, int first, int steps, uint16_t* cnt, int (&expert)[kSteps], int (&rank)[kSteps]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) expert[i] = i < steps ? expert_of(a, first + 32 * i + lane) : -1;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    if (i >= steps) break;
    const int e = expert[i];
    const unsigned peers = __match_any_sync(0xffffffffu, e);
    const int before = __popc(peers & ((1u << lane) - 1u));
    const int old = e >= 0 ? cnt[e] : 0;
    __syncwarp();
    if (e >= 0 && before == 0) cnt[e] = static_cast<uint16_t>(old + __popc(peers));
    __syncwarp();
    rank[i] = old + before;
  }
}

// cnt[w][e] -> pairs of expert e in the warps before w; returns their sum over all warps
__device__ __forceinline__ int scan_warps(uint16_t* cnt, int E, int e, int warps) {
  int run = 0;
  for (int w = 0; w < warps; ++w) {
    const int v = cnt[w * E + e];
    cnt[w * E + e] = static_cast<uint16_t>(run);
    run += v;
  }
  return run;
}

__device__ __forceinline__ void place_pairs(const Plan& a, int first, int steps, const uint16_t* cnt, const int* base,
                                            const int (&expert)[kSteps], const int (&rank)[kSteps]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    if (i >= steps) break;
    const int p = first + 32 * i + lane, e = expert[i];
    if (p >= a.n) continue;
    int r = -1;
    if (e >= 0) {
      r = base[e] + cnt[e] + rank[i];
      a.slot[r] = p;
      a.token[r] = p / a.K;
    }
    a.row[p] = r;
  }
}

// Rows behind an expert's pairs (warp by warp) and behind the last expert hold no pair.  Unsigned row numbers: a step behind the last
// row may pass 2^31.
__device__ __forceinline__ void mark_rest(const Plan& a, const int* offset, int block, int blocks) {
  const unsigned lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (a.align > 1) {
    for (int e = block * warps + (threadIdx.x >> 5); e < a.E; e += blocks * warps)
      for (unsigned r = offset[e] + a.count[e] + lane, end = offset[e + 1]; r < end; r += 32) a.slot[r] = a.token[r] = -1;
  }
  for (unsigned r = offset[a.E] + block * blockDim.x + threadIdx.x, end = a.rows; r < end; r += blocks * blockDim.x)
    a.slot[r] = a.token[r] = -1;
}

__device__ __forceinline__ int round_up(int n, int align) { return (n + align - 1) / align * align; }

// Up to kOneMaxPairs pairs: one block does it all from registers and shared memory, one launch instead of three.  512, 1024, 2048
// pairs 4.5, 5.7, 8.0 us; three launches 6.6 for each, and about 4 us more of the host's time.
__global__ void __launch_bounds__(32 * kOneWarps) permutation_one_block_kernel(const Plan a) {
  release_next();
  wait_for_previous();
  extern __shared__ int smem[];
  __shared__ int partial[kOneWarps];
  int* base = smem;                                                // (E + 1)
  uint16_t* cnt = reinterpret_cast<uint16_t*>(smem + a.E + 1);     // (warps, E)
  const int warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < kOneWarps * a.E; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  int expert[kSteps], rank[kSteps];
  const int per_warp = round_up((a.n + kOneWarps - 1) / kOneWarps, 32);  // contiguous pairs of a warp, at most 32 kSteps
  const int first = warp * per_warp;
  Plan mine = a;
  mine.n = min(a.n, first + per_warp);
  rank_pairs(mine, first, per_warp / 32, cnt + warp * a.E, expert, rank);
  __syncthreads();
  const int e = threadIdx.x;
  const int c = e < a.E ? scan_warps(cnt, a.E, e, kOneWarps) : 0;
  int total;
  const int at = block_scan(e < a.E ? round_up(c, a.align) : 0, partial, &total);
  if (e < a.E) {
    base[e] = a.offset[e] = at;
    a.count[e] = c;
  }
  if (e == 0) base[a.E] = a.offset[a.E] = total;
  __syncthreads();
  place_pairs(mine, first, per_warp / 32, cnt + warp * a.E, base, expert, rank);
  mark_rest(a, base, 0, 1);
}

// Chunk of block b: pairs [b * per_block, (b + 1) * per_block).  hist has kMaxBlocks words per expert, so that the scan reads and
// writes whole lines of one expert's blocks.
__global__ void __launch_bounds__(32 * kWarps) permutation_count_kernel(const Plan a, int per_block) {
  release_next();
  wait_for_previous();
  extern __shared__ int smem[];
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) smem[e] = 0;
  __syncthreads();
  const int first = blockIdx.x * per_block, end = min(a.n - first, per_block);
#pragma unroll 8
  for (int i = threadIdx.x; i < end; i += blockDim.x) {
    const int e = expert_of(a, first + i);
    if (e >= 0) atomicAdd(&smem[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) a.hist[e * kMaxBlocks + blockIdx.x] = smem[e];
}

// hist[e][b] -> pairs of expert e in the blocks before b; counts.  A warp has an expert, a lane four of its blocks at a time (the
// ones that do not exist count nothing).
__global__ void __launch_bounds__(32 * kScanWarps) permutation_scan_kernel(const Plan a, int blocks) {
  release_next();
  wait_for_previous();
  constexpr int kQuads = kMaxBlocks / 128;
  static_assert(kMaxBlocks % 128 == 0, "a warp's lanes have four blocks each at a time");
  const int lane = threadIdx.x & 31, e = blockIdx.x * kScanWarps + (threadIdx.x >> 5);
  if (e >= a.E) return;
  int4* words = reinterpret_cast<int4*>(a.hist + e * kMaxBlocks) + lane;
  int4 v[kQuads];
#pragma unroll
  for (int q = 0; q < kQuads; ++q) v[q] = words[32 * q];
  int all = 0;
#pragma unroll
  for (int q = 0; q < kQuads; ++q) {
    const int b = 128 * q + 4 * lane;
    if (b >= blocks) v[q].x = 0;
    if (b + 1 >= blocks) v[q].y = 0;
    if (b + 2 >= blocks) v[q].z = 0;
    if (b + 3 >= blocks) v[q].w = 0;
    const int own = v[q].x + v[q].y + v[q].z + v[q].w;
    int incl = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += o;
    }
    const int before = all + incl - own;
    words[32 * q] = make_int4(before, before + v[q].x, before + v[q].x + v[q].y, before + v[q].x + v[q].y + v[q].z);
    all += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) a.count[e] = all;
}

// steps: groups of 32 pairs of a warp, so that a block has a chunk of 32 * steps * kWarps at a time.
__global__ void __launch_bounds__(32 * kWarps) permutation_place_kernel(const Plan a, int per_block, int steps) {
  release_next();
  wait_for_previous();
  extern __shared__ int smem[];
  __shared__ int partial[kWarps];
  int* offset = smem;                                                // (E + 1)
  int* base = smem + a.E + 1;                                        // (E) next row of every expert
  uint16_t* cnt = reinterpret_cast<uint16_t*>(smem + 2 * a.E + 1);   // (kWarps, E)
  const int warp = threadIdx.x >> 5;
  int before = 0;
  for (int e0 = 0; e0 < a.E; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    const int c = e < a.E ? a.count[e] : 0, in_blocks = e < a.E ? a.hist[e * kMaxBlocks + blockIdx.x] : 0;
    int total;
    const int at = before + block_scan(round_up(c, a.align), partial, &total);
    before += total;
    if (e < a.E) {
      offset[e] = at;
      base[e] = at + in_blocks;
      if (blockIdx.x == 0) a.offset[e] = at;
    }
  }
  if (threadIdx.x == 0) {
    offset[a.E] = before;
    if (blockIdx.x == 0) a.offset[a.E] = before;
  }
  Plan mine = a;
  const long long end = static_cast<long long>(blockIdx.x + 1) * per_block;
  mine.n = end < a.n ? static_cast<int>(end) : a.n;
  for (int first = blockIdx.x * per_block; first < mine.n; first += 32 * kWarps * steps) {
    for (int i = threadIdx.x; i < kWarps * a.E; i += blockDim.x) cnt[i] = 0;
    __syncthreads();
    int expert[kSteps], rank[kSteps];
    const int own = first + warp * (32 * steps);
    rank_pairs(mine, own, steps, cnt + warp * a.E, expert, rank);
    __syncthreads();
    // a chunk's sums are added to the bases only once its pairs have been placed
    int sum[kMaxExperts / (32 * kWarps)];
#pragma unroll
    for (int j = 0; j < kMaxExperts / (32 * kWarps); ++j) {
      const int e = j * 32 * kWarps + threadIdx.x;
      sum[j] = e < a.E ? scan_warps(cnt, a.E, e, kWarps) : 0;
    }
    __syncthreads();
    place_pairs(mine, own, steps, cnt + warp * a.E, base, expert, rank);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kMaxExperts / (32 * kWarps); ++j) {
      const int e = j * 32 * kWarps + threadIdx.x;
      if (e < a.E) base[e] += sum[j];
    }
  }
  __syncthreads();
  mark_rest(a, offset, blockIdx.x, gridDim.x);
}

// ----------------------------------------------------------------------------------------------
// row movers
// ----------------------------------------------------------------------------------------------
// A piece: VEC bytes that one thread moves with one access.
template <int VEC>
struct Piece {
  uint32_t w[VEC >= 4 ? VEC / 4 : 1];  // VEC 2: the low half
};

// STREAM: read once, leaves the L2 first.
template <int VEC, bool STREAM>
__device__ __forceinline__ Piece<VEC> load_piece(const char* p) {
  Piece<VEC> v;
  if constexpr (VEC == 32) {
    if constexpr (STREAM)
      asm volatile("ld.global.L2::evict_first.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
                   : "l"(p)
                   : "memory");
    else
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
                   : "l"(p)
                   : "memory");
  } else if constexpr (VEC == 16) {
    const uint4 q = STREAM ? __ldcs(reinterpret_cast<const uint4*>(p)) : *reinterpret_cast<const uint4*>(p);
    v.w[0] = q.x; v.w[1] = q.y; v.w[2] = q.z; v.w[3] = q.w;
  } else if constexpr (VEC == 4) {
    v.w[0] = STREAM ? __ldcs(reinterpret_cast<const unsigned*>(p)) : *reinterpret_cast<const unsigned*>(p);
  } else {
    v.w[0] = STREAM ? __ldcs(reinterpret_cast<const unsigned short*>(p)) : *reinterpret_cast<const unsigned short*>(p);
  }
  return v;
}

template <int VEC>
__device__ __forceinline__ void store_piece(char* p, const Piece<VEC>& v) {
  if constexpr (VEC == 32) {
    asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(v.w[0]), "r"(v.w[1]), "r"(v.w[2]),
                 "r"(v.w[3]), "r"(v.w[4]), "r"(v.w[5]), "r"(v.w[6]), "r"(v.w[7]), "l"(p)
                 : "memory");
  } else if constexpr (VEC == 16) {
    *reinterpret_cast<uint4*>(p) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
  } else if constexpr (VEC == 4) {
    *reinterpret_cast<uint32_t*>(p) = v.w[0];
  } else {
    *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(v.w[0]);
  }
}

template <class T, int VEC>
constexpr int kElems = VEC / static_cast<int>(sizeof(T));

template <class T>
__device__ __forceinline__ float half_value(uint32_t bits) {
  if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  else return __uint_as_float(bits << 16);
}

template <class T, int VEC>
__device__ __forceinline__ void unpack(const Piece<VEC>& v, float (&f)[kElems<T, VEC>]) {
#pragma unroll
  for (int i = 0; i < kElems<T, VEC>; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = __uint_as_float(v.w[i]);
    } else {
      f[i] = half_value<T>((v.w[i / 2] >> (16 * (i & 1))) & 0xFFFFu);
    }
  }
}

template <class T>
__device__ __forceinline__ uint32_t half_bits(float f) {
  if constexpr (std::is_same<T, __half>::value) return __half_as_ushort(__float2half_rn(f));
  else return __bfloat16_as_ushort(__float2bfloat16_rn(f));
}

template <class T, int VEC>
__device__ __forceinline__ Piece<VEC> pack(const float (&f)[kElems<T, VEC>]) {
  Piece<VEC> v;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < kElems<T, VEC>; ++i) v.w[i] = __float_as_uint(f[i]);
  } else if constexpr (VEC == 2) {
    v.w[0] = half_bits<T>(f[0]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) v.w[i] = half_bits<T>(f[2 * i]) | (half_bits<T>(f[2 * i + 1]) << 16);
  }
  return v;
}

__device__ __forceinline__ float load_weight(const void* w, int dtype, long long i) {
  if (dtype == SMOE_F32) return static_cast<const float*>(w)[i];
  if (dtype == SMOE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
  return __half2float(static_cast<const __half*>(w)[i]);
}

__device__ __forceinline__ void store_weight(void* w, int dtype, long long i, float v) {
  if (dtype == SMOE_F32) static_cast<float*>(w)[i] = v;
  else if (dtype == SMOE_BF16) static_cast<__nv_bfloat16*>(w)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(w)[i] = __float2half_rn(v);
}

// Rows that start anywhere (on a value), by the 16-byte blocks of the row that is written: one store for each, and two loads from a
// row that lies otherwise, shifted together.  The first and the last block are stored value by value.
template <class T>
struct Window {
  static __host__ __device__ __forceinline__ int count(int bytes) { return (bytes + 16 - static_cast<int>(sizeof(T)) + 15) / 16; }
  // offset of block i in the row at `dst`
  static __device__ __forceinline__ int offset(int i, const char* dst) { return 16 * i - static_cast<int>(reinterpret_cast<uintptr_t>(dst) & 15); }
  static __device__ __forceinline__ Piece<16> load(const char* row, int at, int bytes) {
    Piece<16> v;
    load16_around_row<T>(row, at, bytes, v.w);
    return v;
  }
  static __device__ __forceinline__ void store(char* row, int at, int bytes, const Piece<16>& v) {
    if (at >= 0 && at + 16 <= bytes) {
      store_piece<16>(row + at, v);
    } else {
#pragma unroll
      for (int i = 0; i < 16 / static_cast<int>(sizeof(T)); ++i) {
        const int o = at + i * static_cast<int>(sizeof(T));
        if (o < 0 || o >= bytes) continue;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(row + o) = v.w[i];
        else *reinterpret_cast<unsigned short*>(row + o) = static_cast<unsigned short>(v.w[i / 2] >> (16 * (i & 1)));
      }
    }
  }
};

struct Rows {
  const char* token_src;  // spread: (T, H) rows of the tokens, token_ld bytes apart
  long long token_ld;
  const char* row_src;    // collect, dots: (R, H) sorted rows, row_ld bytes apart
  long long row_ld;
  char* out;              // spread: (R, H), collect: (T, H); packed
  const void* weight;     // (T, K) or nullptr = 1
  void* dweight;          // (T, K), the type of weight
  int weight_type;
  const int* row;         // (T, K) sorted row of every pair, or -1
  const int* slot;        // (R) pair of every row, or none (outside of [0, T K))
  int T, K, R, bytes;     // bytes: of one row of H values
};

constexpr int kThreads = 256;
constexpr int kPadRows = 64;  // rows that a block looks through for ones without a pair, eight a warp at a time

// Whether no pair writes row r: none is named, or the one that is has no row or another (a pair dropped after the sort, in `row` alone).
__device__ __forceinline__ bool is_empty(const Rows& a, int r) {
  const int p = a.slot[r];
  return static_cast<unsigned>(p) >= static_cast<unsigned>(a.T * a.K) || a.row[p] != r;
}

// The first blocks of a spread: zeros for the rows without a pair.
template <int VEC>
__device__ __forceinline__ void zero_rows(const Rows& a, int block) {
  const int lane = threadIdx.x & 31;
  Piece<VEC> zero;
#pragma unroll
  for (auto& w : zero.w) w = 0u;
  for (int i = 8 * (threadIdx.x >> 5); i < kPadRows; i += 8 * (blockDim.x >> 5)) {
    const long long first = static_cast<long long>(block) * kPadRows + i;
    const bool empty = lane < 8 && first + lane < a.R && is_empty(a, static_cast<int>(first) + lane);
    unsigned todo = __ballot_sync(0xffffffffu, empty);
    for (; todo != 0u; todo &= todo - 1u) {
      char* dst = a.out + (first + __ffs(todo) - 1) * a.bytes;
      for (int c = lane * VEC; c < a.bytes; c += 32 * VEC) store_piece<VEC>(dst + c, zero);
    }
  }
}

// Pieces of a row per thread, `stride` pieces apart, so that neighbouring threads have neighbouring pieces: rows that allow
// only narrow accesses get several in flight.
constexpr int pieces_per_thread(int vec) { return vec >= 16 ? 1 : 4; }

// rows[row(t, k)] = (w[t, k]) x[t].  WEIGHTED false: the bytes as they are, whatever their type.
template <class T, int VEC, bool WEIGHTED>
__global__ void __launch_bounds__(kThreads) spread_kernel(const Rows a, int pad_blocks) {
  release_next();
  wait_for_previous();
  if (blockIdx.x < pad_blocks) return zero_rows<VEC>(a, blockIdx.x);
  constexpr int U = pieces_per_thread(VEC);
  const int per_row = a.bytes / VEC, stride = (per_row + U - 1) / U;
  const long long g = static_cast<long long>(blockIdx.x - pad_blocks) * kThreads + threadIdx.x;
  if (g >= static_cast<long long>(a.T) * stride) return;
  const int t = static_cast<int>(g / stride), c = static_cast<int>(g - static_cast<long long>(t) * stride);
  const char* src = a.token_src + t * a.token_ld;
  Piece<VEC> v[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (c + u * stride < per_row) v[u] = load_piece<VEC, true>(src + static_cast<long long>(c + u * stride) * VEC);
  const long long p0 = static_cast<long long>(t) * a.K;
  for (int k = 0; k < a.K; ++k) {
    const int r = a.row[p0 + k];
    if (static_cast<unsigned>(r) >= static_cast<unsigned>(a.R)) continue;
    const float w = WEIGHTED ? load_weight(a.weight, a.weight_type, p0 + k) : 1.f;
    char* dst = a.out + static_cast<long long>(r) * a.bytes;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c + u * stride >= per_row) continue;
      char* at = dst + static_cast<long long>(c + u * stride) * VEC;
      if constexpr (WEIGHTED) {
        float f[kElems<T, VEC>];
        unpack<T, VEC>(v[u], f);
#pragma unroll
        for (auto& x : f) x *= w;
        store_piece<VEC>(at, pack<T, VEC>(f));
      } else {
        store_piece<VEC>(at, v[u]);
      }
    }
  }
}

// out[t] = sum over k of (w[t, k]) rows[row(t, k)], fp32 sums in the order of k, one rounding.
template <class T, int VEC>
__global__ void __launch_bounds__(kThreads) collect_kernel(const Rows a) {
  release_next();
  wait_for_previous();
  constexpr int U = pieces_per_thread(VEC), N = kElems<T, VEC>;
  const int per_row = a.bytes / VEC, stride = (per_row + U - 1) / U;
  const long long g = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
  if (g >= static_cast<long long>(a.T) * stride) return;
  const int t = static_cast<int>(g / stride), c = static_cast<int>(g - static_cast<long long>(t) * stride);
  float acc[U][N];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (auto& x : acc[u]) x = 0.f;
  const long long p0 = static_cast<long long>(t) * a.K;
#pragma unroll 4
  for (int k = 0; k < a.K; ++k) {
    const int r = a.row[p0 + k];
    if (static_cast<unsigned>(r) >= static_cast<unsigned>(a.R)) continue;
    const float w = a.weight != nullptr ? load_weight(a.weight, a.weight_type, p0 + k) : 1.f;
    const char* src = a.row_src + r * a.row_ld;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c + u * stride >= per_row) continue;
      float f[N];
      unpack<T, VEC>(load_piece<VEC, true>(src + static_cast<long long>(c + u * stride) * VEC), f);
#pragma unroll
      for (int i = 0; i < N; ++i) acc[u][i] += w * f[i];
    }
  }
  char* dst = a.out + static_cast<long long>(t) * a.bytes;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (c + u * stride < per_row) store_piece<VEC>(dst + static_cast<long long>(c + u * stride) * VEC, pack<T, VEC>(acc[u]));
}

// The two above by windows.  Sides measured (piece by piece / by windows, us): spread, fp32 rows of 1005 values, T 4099, K 6 33 / 22,
// of 2049, T 8192, K 4 84 / 58, bf16 of 3001, T 16384, K 4 125 / 88, but fp16 of 1030, which have 4-byte pieces of two values, T 5003,
// K 3 8.6 / 10.2; collect, in the same order 30.7 / 27.7, 87 / 71, 217 / 128, 18.8 / 11.1.  So a spread goes by windows where a piece
// is one value, a collect where it is less than 16 bytes.  (With the values at the rows' ends loaded one by one a warp with an
// end takes many times as long: 33, 105, 174, 15.8 for the collect.  The gradient of the combine, with a window for each of four
// differently placed rows and their gradients, loses: 212 -> 271 us forward and backward for the rows of 2049.)
template <class T, bool WEIGHTED>
__global__ void __launch_bounds__(kThreads) spread_windows_kernel(const Rows a, int pad_blocks) {
  release_next();
  wait_for_previous();
  if (blockIdx.x < pad_blocks) return zero_rows<sizeof(T)>(a, blockIdx.x);
  using W = Window<T>;
  const int windows = W::count(a.bytes);
  const long long g = static_cast<long long>(blockIdx.x - pad_blocks) * kThreads + threadIdx.x;
  if (g >= static_cast<long long>(a.T) * windows) return;
  const int t = static_cast<int>(g / windows), c = static_cast<int>(g - static_cast<long long>(t) * windows);
  const char* src = a.token_src + t * a.token_ld;
  const long long p0 = static_cast<long long>(t) * a.K;
#pragma unroll 4
  for (int k = 0; k < a.K; ++k) {
    const int r = a.row[p0 + k];
    if (static_cast<unsigned>(r) >= static_cast<unsigned>(a.R)) continue;
    char* dst = a.out + static_cast<long long>(r) * a.bytes;
    const int at = W::offset(c, dst);
    Piece<16> v = W::load(src, at, a.bytes);
    if constexpr (WEIGHTED) {
      const float w = load_weight(a.weight, a.weight_type, p0 + k);
      float f[kElems<T, 16>];
      unpack<T, 16>(v, f);
#pragma unroll
      for (auto& x : f) x *= w;
      v = pack<T, 16>(f);
    }
    W::store(dst, at, a.bytes, v);
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads) collect_windows_kernel(const Rows a) {
  release_next();
  wait_for_previous();
  using W = Window<T>;
  constexpr int N = kElems<T, 16>;
  const int windows = W::count(a.bytes);
  const long long g = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
  if (g >= static_cast<long long>(a.T) * windows) return;
  const int t = static_cast<int>(g / windows), c = static_cast<int>(g - static_cast<long long>(t) * windows);
  char* dst = a.out + static_cast<long long>(t) * a.bytes;
  const int at = W::offset(c, dst);
  float acc[N];
#pragma unroll
  for (auto& x : acc) x = 0.f;
  const long long p0 = static_cast<long long>(t) * a.K;
#pragma unroll 4
  for (int k = 0; k < a.K; ++k) {
    const int r = a.row[p0 + k];
    if (static_cast<unsigned>(r) >= static_cast<unsigned>(a.R)) continue;
    const float w = a.weight != nullptr ? load_weight(a.weight, a.weight_type, p0 + k) : 1.f;
    float f[N];
    unpack<T, 16>(W::load(a.row_src + r * a.row_ld, at, a.bytes), f);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] += w * f[i];
  }
  W::store(dst, at, a.bytes, pack<T, 16>(acc));
}

// The combine's backward pass, one block per token: drows[row(t, k)] = w[t, k] dout[t] and dw[t, k] = <dout[t], rows[row(t, k)]>.
// Four rows of the token are in flight at a time.  A row's dot product is added up piece by piece in a thread, then over the
// lanes of each warp, then over the warps: always in the same order.
constexpr int kDotRows = 4, kDotChunk = 32;

// dot += <f, g> over the one or two values of a word (FULL: both halves of a 16-bit word); returns w g
template <class T, bool FULL>
__device__ __forceinline__ uint32_t dot_word(uint32_t f, uint32_t g, float w, float& dot) {
  if constexpr (sizeof(T) == 4) {
    dot += __uint_as_float(f) * __uint_as_float(g);
    return __float_as_uint(w * __uint_as_float(g));
  } else {
    const float g0 = half_value<T>(g & 0xFFFFu), g1 = half_value<T>(g >> 16);
    dot += half_value<T>(f & 0xFFFFu) * g0;
    if (!FULL) return half_bits<T>(w * g0);
    dot += half_value<T>(f >> 16) * g1;
    return half_bits<T>(w * g0) | (half_bits<T>(w * g1) << 16);
  }
}

template <class T, int VEC>
__global__ void __launch_bounds__(kThreads, 3) spread_dot_kernel(const Rows a, int pad_blocks) {
  release_next();
  wait_for_previous();
  if (blockIdx.x < pad_blocks) return zero_rows<VEC>(a, blockIdx.x);
  constexpr int U = pieces_per_thread(VEC);
  __shared__ float part[kDotChunk][kThreads / 32];
  const int t = blockIdx.x - pad_blocks;
  const int per_row = a.bytes / VEC;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const char* src = a.token_src + t * a.token_ld;
  const long long p0 = static_cast<long long>(t) * a.K;
  for (int kc = 0; kc < a.K; kc += kDotChunk) {
    const int kn = min(kDotChunk, a.K - kc);
    for (int k0 = 0; k0 < kn; k0 += kDotRows) {
      int r[kDotRows];
      float w[kDotRows], dot[kDotRows];
#pragma unroll
      for (int j = 0; j < kDotRows; ++j) {
        r[j] = k0 + j < kn ? a.row[p0 + kc + k0 + j] : -1;
        if (static_cast<unsigned>(r[j]) >= static_cast<unsigned>(a.R)) r[j] = -1;
        w[j] = r[j] >= 0 ? load_weight(a.weight, a.weight_type, p0 + kc + k0 + j) : 0.f;
        dot[j] = 0.f;
      }
      for (int c0 = threadIdx.x; c0 < per_row; c0 += U * blockDim.x) {
        Piece<VEC> y[kDotRows][U], g[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int c = c0 + u * blockDim.x;
          if (c >= per_row) continue;
          const long long at = static_cast<long long>(c) * VEC;
#pragma unroll
          for (int j = 0; j < kDotRows; ++j)
            if (r[j] >= 0) y[j][u] = load_piece<VEC, true>(a.row_src + r[j] * a.row_ld + at);
          g[u] = load_piece<VEC, false>(src + at);
        }
        // word by word, the row's gradient in the place of its values: four rows of 32 bytes fit into 80 registers, and three
        // blocks of 256 threads into an SM (with whole rows unpacked, 120 registers, T 24576, H 1536, K 8 took 223 us, now 196)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int c = c0 + u * blockDim.x;
          if (c >= per_row) continue;
#pragma unroll
          for (int j = 0; j < kDotRows; ++j) {
            if (r[j] < 0) continue;
#pragma unroll
            for (int i = 0; i < (VEC >= 4 ? VEC / 4 : 1); ++i)
              y[j][u].w[i] = dot_word<T, (VEC >= 4)>(y[j][u].w[i], g[u].w[i], w[j], dot[j]);
            store_piece<VEC>(a.out + static_cast<long long>(r[j]) * a.bytes + static_cast<long long>(c) * VEC, y[j][u]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kDotRows; ++j) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], d);
        if (lane == 0 && k0 + j < kn) part[k0 + j][warp] = dot[j];
      }
    }
    __syncthreads();
    if (threadIdx.x < kn) {
      float s = 0.f;
      for (int w = 0; w < warps; ++w) s += part[threadIdx.x][w];
      store_weight(a.dweight, a.weight_type, p0 + kc + threadIdx.x, s);
    }
    __syncthreads();
  }
}

// ----------------------------------------------------------------------------------------------
// host side
// ----------------------------------------------------------------------------------------------
static int type_bytes(int dtype) { return dtype == SMOE_F32 ? 4 : dtype == SMOE_BF16 || dtype == SMOE_F16 ? 2 : 0; }

// The widest access that every row starts on: 32, 16, 4 or 2 bytes.
static int piece_bytes(std::initializer_list<long long> multiples) {
  for (const int vec : {32, 16, 4}) {
    bool fits = true;
    for (const long long m : multiples) fits = fits && m % vec == 0;
    if (fits) return vec;
  }
  return 2;
}
static long long address(const void* p) { return static_cast<long long>(reinterpret_cast<uintptr_t>(p)); }

// LEAST: the narrowest pieces that the kernel has.
template <int LEAST, class F>
static int for_piece(int vec, F&& f) {
  if (vec == 32) return f(std::integral_constant<int, 32>());
  if (vec == 16) return f(std::integral_constant<int, 16>());
  if constexpr (LEAST <= 4) {
    if (vec == 4) return f(std::integral_constant<int, 4>());
  }
  if constexpr (LEAST <= 2) {
    if (vec == 2) return f(std::integral_constant<int, 2>());
  }
  return SMOE_ERR_ALIGNMENT;
}

static long long pad_blocks(int R) { return (static_cast<long long>(R) + kPadRows - 1) / kPadRows; }

static long long flat_blocks(const Rows& a, int vec) {
  const int u = pieces_per_thread(vec);
  const long long stride = (a.bytes / vec + u - 1) / u;
  return (a.T * stride + kThreads - 1) / kThreads;
}

template <class T>
static long long window_blocks(const Rows& a) {
  return (static_cast<long long>(a.T) * Window<T>::count(a.bytes) + kThreads - 1) / kThreads;
}

template <class Kernel, class... Args>
static int launch_blocks(Kernel kernel, long long blocks, unsigned threads, cudaStream_t st, Args... args) {
  if (blocks > 0x7fffffffll) return SMOE_ERR_SHAPE;  // of a grid; less by far than the rows that memory holds, but rows may be broadcast
  return launched(launch_chained(kernel, static_cast<unsigned>(blocks), threads, 0, st, 1, args...));
}

template <class T, bool WEIGHTED>
static int launch_spread(const Rows& a, int vec, cudaStream_t st) {
  const long long pad = pad_blocks(a.R);
  if (vec == static_cast<int>(sizeof(T)))
    return launch_blocks(spread_windows_kernel<T, WEIGHTED>, pad + window_blocks<T>(a), kThreads, st, a, static_cast<int>(pad));
  return for_piece<sizeof(T) == 2 ? 4 : 16>(
      vec, [&](auto v) { return launch_blocks(spread_kernel<T, v, WEIGHTED>, pad + flat_blocks(a, vec), kThreads, st, a, static_cast<int>(pad)); });
}

template <class T>
static int launch_collect(const Rows& a, int vec, cudaStream_t st) {
  if (vec < 16) return launch_blocks(collect_windows_kernel<T>, window_blocks<T>(a), kThreads, st, a);
  return for_piece<16>(vec, [&](auto v) { return launch_blocks(collect_kernel<T, v>, flat_blocks(a, vec), kThreads, st, a); });
}

template <class T>
static int launch_spread_dot(const Rows& a, int vec, cudaStream_t st) {
  return for_piece<static_cast<int>(sizeof(T))>(vec, [&](auto v) {
    const long long pad = pad_blocks(a.R);
    // as few rounds over the row as 256 threads allow, and no more threads than those rounds need
    const int u = pieces_per_thread(vec), pieces = (a.bytes / vec + u - 1) / u, rounds = (pieces + kThreads - 1) / kThreads;
    const unsigned threads = static_cast<unsigned>(((pieces + rounds - 1) / rounds + 31) / 32 * 32);
    return launch_blocks(spread_dot_kernel<T, v>, pad + a.T, threads, st, a, static_cast<int>(pad));
  });
}

template <class F>
static int for_type(int dtype, F&& f) {
  if (dtype == SMOE_F32) return f(float());
  if (dtype == SMOE_BF16) return f(__nv_bfloat16());
  if (dtype == SMOE_F16) return f(__half());
  return SMOE_ERR_DTYPE;
}

static bool bad_rows(int T, int K, int H, long long R, int dtype) {
  return T < 0 || K <= 0 || H <= 0 || R < 0 || R > 0x7fffffffll || static_cast<long long>(T) * K > 0x7fffffffll ||
         static_cast<long long>(H) * type_bytes(dtype) > 0x7fffff00ll;
}

}  // namespace permute
}  // namespace smoe

using namespace smoe;
using namespace smoe::permute;

extern "C" {

long long smoe_token_permutation_rows(long long n, int E, int align) {
  if (n < 0 || E <= 0 || align <= 0) return -1;
  const long long used = n < E ? n : E;
  return (n + used * (align - 1)) / align * align;
}

size_t smoe_token_permutation_workspace_bytes(long long n, int E) {
  if (n <= kOneMaxPairs && E <= kOneMaxExperts) return 0;
  return static_cast<size_t>(kMaxBlocks) * static_cast<size_t>(E > 0 ? E : 1) * sizeof(int);
}

int smoe_token_permutation(const void* expert_idx, int idx_dtype, int T, int K, int E, int align, int* expert_frequency,
                           int* expert_frequency_offset, int* x_gather_idx, int* s_scatter_idx,
                           int* s_reverse_scatter_idx, void* workspace, void* stream) {
  const long long n = static_cast<long long>(T) * K;
  if (T < 0 || K <= 0 || n >= 0x7fff0000ll || E <= 0 || E > kMaxExperts || align <= 0) return SMOE_ERR_SHAPE;
  const long long rows = smoe_token_permutation_rows(n, E, align);
  // the rounded sums of a load stay below rows + E align, whatever the order in which they are added
  if (rows + static_cast<long long>(E) * align > 0x7fffffffll) return SMOE_ERR_SHAPE;
  if (idx_dtype != SMOE_I32 && idx_dtype != SMOE_I64) return SMOE_ERR_DTYPE;
  if (expert_frequency == nullptr || expert_frequency_offset == nullptr) return SMOE_ERR_SHAPE;
  if (n > 0 && (expert_idx == nullptr || x_gather_idx == nullptr || s_scatter_idx == nullptr || s_reverse_scatter_idx == nullptr))
    return SMOE_ERR_SHAPE;
  const size_t ws = smoe_token_permutation_workspace_bytes(n, E);
  if (ws > 0 && workspace == nullptr) return SMOE_ERR_WORKSPACE;
  if (address(expert_idx) % (idx_dtype == SMOE_I64 ? 8 : 4) != 0) return SMOE_ERR_ALIGNMENT;
  if (address(workspace) % 16 != 0) return SMOE_ERR_ALIGNMENT;
  for (const void* p : {static_cast<const void*>(expert_frequency), static_cast<const void*>(expert_frequency_offset),
                        static_cast<const void*>(x_gather_idx), static_cast<const void*>(s_scatter_idx),
                        static_cast<const void*>(s_reverse_scatter_idx)})
    if (address(p) % 4 != 0) return SMOE_ERR_ALIGNMENT;
  const Plan a = {expert_idx, idx_dtype == SMOE_I64, static_cast<int>(n), K, E, align, static_cast<int>(rows),
                  expert_frequency, expert_frequency_offset, x_gather_idx, s_scatter_idx, s_reverse_scatter_idx,
                  static_cast<int*>(workspace)};
  static PerDeviceFlag configured;
  const int dev = current_device();
  if (dev < 0) return SMOE_ERR_DRIVER;
  const auto one_smem = [](int e) { return (e + 1) * 4 + kOneWarps * e * 2; };
  const auto place_smem = [](int e) { return (2 * e + 1) * 4 + kWarps * e * 2; };
  if (!configured.test(dev)) {
    if (cudaFuncSetAttribute(permutation_one_block_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, one_smem(kOneMaxExperts)) != cudaSuccess ||
        cudaFuncSetAttribute(permutation_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, place_smem(kMaxExperts)) != cudaSuccess)
      return SMOE_ERR_LAUNCH;
    configured.set(dev);
  }
  if (ws == 0)
    return launched(launch_chained(permutation_one_block_kernel, 1, 32 * kOneWarps, one_smem(E), S(stream), 1, a));
  // As many blocks as there may be, each with a multiple of 256 pairs: 24594 pairs would be 12 blocks of 2048.  65536 and 262144
  // pairs of 128 experts: at most 128 blocks 8.4 and 19.7 us, 256 blocks 7.8 and 13.9, 512 blocks 8.2 and 15.2.  (One block that
  // scanned all experts made 11.5 and 22.3 of the first.)
  const long long group = 32 * kWarps;
  long long per_block = (n + kMaxBlocks - 1) / kMaxBlocks;
  per_block = per_block > 0 ? (per_block + group - 1) / group * group : group;
  const int steps = per_block / group < kSteps ? static_cast<int>(per_block / group) : kSteps;
  const int blocks = n > 0 ? static_cast<int>((n + per_block - 1) / per_block) : 1;
  const int per = static_cast<int>(per_block);
  cudaError_t rc = launch_chained(permutation_count_kernel, blocks, 32 * kWarps, E * 4, S(stream), 1, a, per);
  if (rc == cudaSuccess) rc = launch_chained(permutation_scan_kernel, (E + kScanWarps - 1) / kScanWarps, 32 * kScanWarps, 0, S(stream), 1, a, blocks);
  if (rc == cudaSuccess) rc = launch_chained(permutation_place_kernel, blocks, 32 * kWarps, place_smem(E), S(stream), 1, a, per, steps);
  return launched(rc, 3);
}

int smoe_permute_rows(const void* x, long long ld, void* rows, int dtype, const void* weights, int weights_dtype,
                      const int* s_reverse_scatter_idx, const int* s_scatter_idx, int T, int K, int H, long long R, void* stream) {
  const int size = type_bytes(dtype);
  if (size == 0 || (weights != nullptr && type_bytes(weights_dtype) == 0)) return SMOE_ERR_DTYPE;
  if (bad_rows(T, K, H, R, dtype)) return SMOE_ERR_SHAPE;
  if (R == 0) return SMOE_OK;
  if (rows == nullptr || s_scatter_idx == nullptr || (T > 0 && (x == nullptr || s_reverse_scatter_idx == nullptr))) return SMOE_ERR_SHAPE;
  if (address(x) % size != 0 || address(rows) % size != 0 || address(s_reverse_scatter_idx) % 4 != 0 || address(s_scatter_idx) % 4 != 0 ||
      (weights != nullptr && address(weights) % type_bytes(weights_dtype) != 0))
    return SMOE_ERR_ALIGNMENT;
  Rows a = {};
  a.token_src = static_cast<const char*>(x); a.token_ld = ld * size;
  a.out = static_cast<char*>(rows);
  a.weight = weights; a.weight_type = weights_dtype;
  a.row = s_reverse_scatter_idx; a.slot = s_scatter_idx;
  a.T = T; a.K = K; a.R = static_cast<int>(R); a.bytes = H * size;
  const int vec = piece_bytes({address(x), a.token_ld, address(rows), a.bytes});
  if (weights == nullptr)
    return size == 4 ? launch_spread<float, false>(a, vec, S(stream)) : launch_spread<__half, false>(a, vec, S(stream));
  return for_type(dtype, [&](auto t) { return launch_spread<decltype(t), true>(a, vec, S(stream)); });
}

int smoe_unpermute_rows(const void* rows, long long ld, void* out, int dtype, const void* weights, int weights_dtype,
                        const int* s_reverse_scatter_idx, int T, int K, int H, long long R, void* stream) {
  const int size = type_bytes(dtype);
  if (size == 0 || (weights != nullptr && type_bytes(weights_dtype) == 0)) return SMOE_ERR_DTYPE;
  if (bad_rows(T, K, H, R, dtype)) return SMOE_ERR_SHAPE;
  if (T == 0) return SMOE_OK;
  if (out == nullptr || s_reverse_scatter_idx == nullptr || (R > 0 && rows == nullptr)) return SMOE_ERR_SHAPE;
  if (address(rows) % size != 0 || address(out) % size != 0 || address(s_reverse_scatter_idx) % 4 != 0 ||
      (weights != nullptr && address(weights) % type_bytes(weights_dtype) != 0))
    return SMOE_ERR_ALIGNMENT;
  Rows a = {};
  a.row_src = static_cast<const char*>(rows); a.row_ld = ld * size;
  a.out = static_cast<char*>(out);
  a.weight = weights; a.weight_type = weights_dtype;
  a.row = s_reverse_scatter_idx;
  a.T = T; a.K = K; a.R = static_cast<int>(R); a.bytes = H * size;
  const int vec = piece_bytes({address(rows), a.row_ld, address(out), a.bytes});
  return for_type(dtype, [&](auto t) { return launch_collect<decltype(t)>(a, vec, S(stream)); });
}

int smoe_unpermute_rows_backward(const void* dout, long long dout_ld, const void* rows, long long ld, void* drows, int dtype,
                                 const void* weights, void* dweights, int weights_dtype, const int* s_reverse_scatter_idx,
                                 const int* s_scatter_idx, int T, int K, int H, long long R, void* stream) {
  const int size = type_bytes(dtype), wsize = type_bytes(weights_dtype);
  if (size == 0 || wsize == 0) return SMOE_ERR_DTYPE;
  if (bad_rows(T, K, H, R, dtype)) return SMOE_ERR_SHAPE;
  if (T == 0 && R == 0) return SMOE_OK;
  if ((R > 0 && (drows == nullptr || rows == nullptr || s_scatter_idx == nullptr)) ||
      (T > 0 && (dout == nullptr || weights == nullptr || dweights == nullptr || s_reverse_scatter_idx == nullptr)))
    return SMOE_ERR_SHAPE;
  if (address(dout) % size != 0 || address(rows) % size != 0 || address(drows) % size != 0 || address(weights) % wsize != 0 ||
      address(dweights) % wsize != 0 || address(s_reverse_scatter_idx) % 4 != 0 || address(s_scatter_idx) % 4 != 0)
    return SMOE_ERR_ALIGNMENT;
  Rows a = {};
  a.token_src = static_cast<const char*>(dout); a.token_ld = dout_ld * size;
  a.row_src = static_cast<const char*>(rows); a.row_ld = ld * size;
  a.out = static_cast<char*>(drows);
  a.weight = weights; a.dweight = dweights; a.weight_type = weights_dtype;
  a.row = s_reverse_scatter_idx; a.slot = s_scatter_idx;
  a.T = T; a.K = K; a.R = static_cast<int>(R); a.bytes = H * size;
  const int vec = piece_bytes({address(dout), a.token_ld, address(rows), a.row_ld, address(drows), a.bytes});
  return for_type(dtype, [&](auto t) { return launch_spread_dot<decltype(t)>(a, vec, S(stream)); });
}

}  // extern "C"
