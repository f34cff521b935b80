// 8-bit integer products: quantisation of rows and the entry points (the formulas are in int8.cuh).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>
#include <type_traits>

#include "../../include/sonicmoe_b200.h"
#include "int8.cuh"
#include "rows16.cuh"

namespace smoe {
namespace i8 {

static inline cudaStream_t S(void* s) { return static_cast<cudaStream_t>(s); }

// ----------------------------------------------------------------------------------------------
// quantisation
// ----------------------------------------------------------------------------------------------
// A row is read once and stays in registers between the maximum and the conversion: PIECES pieces of 16 bytes per thread, `tpr`
// threads (a power of two) per row, and a block of 256 threads (or one row's) has 256 / tpr rows.  Rows that are longer than 1024
// threads hold are read twice.  Bound by memory: what is read is 2 or 4 times what is written.  WIDE: rows start and end on 16-byte
// boundaries.  Otherwise 16-bit values are put together from two loads, 32-bit ones loaded one by one (value by value / by two loads, us:
// 16384 bf16 rows of 3001 69 / 49, fp16 of 1030 28 / 21, but 7888 fp32 rows of 1030 14.7 / 16.8).
template <class T, bool WIDE>
struct Loaded {
  static constexpr int N = 16 / static_cast<int>(sizeof(T));
  uint32_t w[4];
  // piece c of `row`, which has `cols` values
  __device__ __forceinline__ void load(const T* row, int c, int cols) {
    if constexpr (WIDE) {
      const uint4 q = __ldcs(reinterpret_cast<const uint4*>(row + c * N));
      w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = N * c + i < cols ? reinterpret_cast<const uint32_t*>(row)[N * c + i] : 0u;
    } else {
      load16_of_row<T>(reinterpret_cast<const char*>(row), 16 * c, cols * 2, w);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (auto& x : w) x = 0u;
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    return __half2float(__ushort_as_half(static_cast<unsigned short>(w[i / 2] >> (16 * (i & 1)))));
  }
  // the largest magnitude so far, in the type's own bits: magnitudes compare like whole numbers, a NaN above infinity
  __device__ __forceinline__ uint32_t amax_bits(uint32_t m) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) m = max(m, w[i] & 0x7FFFFFFFu);
      else m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
    }
    return m;
  }
  __device__ __forceinline__ void store(const RowScale& s, int8_t* q) const {
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = value(i);
    uint32_t o[N / 4];
    quantize_values<(sizeof(T) == 2)>(s, f, o);
    if constexpr (N == 8) *reinterpret_cast<uint2*>(q) = make_uint2(o[0], o[1]);
    else *reinterpret_cast<uint32_t*>(q) = o[0];
  }
};

// bits of `amax_bits` (two halves for 16-bit types) -> those of the magnitude as fp32
template <class T>
__device__ __forceinline__ uint32_t amax_as_float_bits(uint32_t m) {
  if constexpr (sizeof(T) == 4) return m;
  m = max(m & 0xFFFFu, m >> 16);
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return m << 16;
  return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
}

template <class T, bool WIDE, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 6 : 1) quantize_rows_kernel(const T* x, long long ld, int8_t* q, long long q_ld, float* scale,
                                                             long long rows, int cols, int tpr_log2) {
  release_next();
  wait_for_previous();
  using L = Loaded<T, WIDE>;
  constexpr int PIECES = 4;
  __shared__ uint32_t part[32];
  const int tpr = 1 << tpr_log2, sub = threadIdx.x >> tpr_log2, tid = threadIdx.x & (tpr - 1);
  const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x >> tpr_log2) + sub;
  const bool live = row < rows;
  const int pieces = (cols + L::N - 1) / L::N;
  const T* src = x + (live ? row : 0) * ld;
  const bool kept = pieces <= PIECES * tpr;
  L v[PIECES];
  uint32_t bits = 0u;
  if (kept) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int c = i * tpr + tid;
      if (live && c < pieces) v[i].load(src, c, cols); else v[i].zero();
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) bits = v[i].amax_bits(bits);
  } else if (live) {
    for (int c = tid; c < pieces; c += tpr) {
      v[0].load(src, c, cols);
      bits = v[0].amax_bits(bits);
    }
  }
  bits = amax_as_float_bits<T>(bits);
  bits = __reduce_max_sync(0xffffffffu, bits);  // tpr >= 32
  if (tpr > 32) {
    const int warp = threadIdx.x >> 5, of_row = tpr >> 5;
    if ((threadIdx.x & 31) == 0) part[warp] = bits;
    __syncthreads();
    for (int w = 0; w < of_row; ++w) bits = max(bits, part[sub * of_row + w]);
  }
  if (!live) return;
  const RowScale s = row_scale<(sizeof(T) == 2)>(bits);
  int8_t* dst = q + row * q_ld;
  if (tid == 0) scale[row] = scale_of_row(bits);
  if (kept) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int c = i * tpr + tid;
      if (c < pieces) v[i].store(s, dst + c * L::N);
    }
  } else {
    for (int c = tid; c < pieces; c += tpr) {
      v[0].load(src, c, cols);
      v[0].store(s, dst + c * L::N);
    }
  }
  // columns up to the next multiple of 16 are zeros
  for (int c = pieces * L::N + 4 * tid; c < (cols + 15) / 16 * 16; c += 4 * tpr) *reinterpret_cast<uint32_t*>(dst + c) = 0u;
}

template <class T, bool WIDE>
static cudaError_t launch_quantize(const void* x, long long ld, void* q, long long q_ld, float* scale, long long rows, int cols,
                                   cudaStream_t st) {
  constexpr int N = Loaded<T, WIDE>::N, PIECES = 4;
  const int pieces = (cols + N - 1) / N;
  int log2 = 5;
  while (log2 < 10 && (PIECES << log2) < pieces) ++log2;
  const int tpr = 1 << log2;
  const int threads = tpr > 256 ? tpr : 256;
  const long long blocks = (rows + threads / tpr - 1) / (threads / tpr);
  return launch_chained(threads == 256 ? quantize_rows_kernel<T, WIDE, 256> : quantize_rows_kernel<T, WIDE, 1024>, dim3(static_cast<unsigned>(blocks)), threads, 0, st, 1, static_cast<const T*>(x), ld,
                        static_cast<int8_t*>(q), q_ld, scale, rows, cols, log2);
}

template <class T>
static cudaError_t launch_quantize(const void* x, long long ld, void* q, long long q_ld, float* scale, long long rows, int cols,
                                   cudaStream_t st) {
  const long long size = sizeof(T);
  const bool wide = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld * size % 16 == 0 && cols * size % 16 == 0;
  return wide ? launch_quantize<T, true>(x, ld, q, q_ld, scale, rows, cols, st) : launch_quantize<T, false>(x, ld, q, q_ld, scale, rows, cols, st);
}

static int quantize(const void* x, long long ld, int dtype, void* q, long long q_ld, float* scale, long long rows, int cols,
                    cudaStream_t st) {
  if (dtype == SMOE_F32) return launched(launch_quantize<float>(x, ld, q, q_ld, scale, rows, cols, st));
  if (dtype == SMOE_BF16) return launched(launch_quantize<__nv_bfloat16>(x, ld, q, q_ld, scale, rows, cols, st));
  return launched(launch_quantize<__half>(x, ld, q, q_ld, scale, rows, cols, st));
}

// ----------------------------------------------------------------------------------------------
// product by 4-way integer dot products
// ----------------------------------------------------------------------------------------------
// For up to 8 rows in all, or 32 of several experts, where the weights are everything.  A block takes a unit, up to eight or two (ROWS)
// rows of one expert, and 32 channels, a warp four of those, whose weights its lanes load 16 bytes each, straight from memory and eight
// or four loads ahead (SPLIT: two or four warps take turns with the columns of four channels, and their sums meet in shared memory).
// The rows lie in shared memory, 4096 columns at a time; rows that are not 8-bit yet may be quantised on the way there, by every
// block for itself.  Bound by latency: the first loads of the weights are on their way before x is looked at.
constexpr int kDotRows = 8,  // of a unit, and of a call in which an expert may have them all
    kDotChannels = 4, kDotWarps = 8, kDotThreads = 32 * kDotWarps, kDotChunk = 4096;
constexpr long long kDotWeights = 32ll << 20;  // bytes of one expert's weights up to which they are fetched early
constexpr int kDotMostRows = 32;               // of several experts, in units of two
constexpr int kDotMostBlocks = 2 * 148;        // two to each of a B200's SMs
constexpr int kDotMinCols = 2048;              // that warps share
constexpr int kDotWideN = 2 * 148 * kDotWarps * kDotChannels;  // channels of two blocks on each SM

__device__ __forceinline__ float activate(int act, float x) {
  switch (act) {
    case ACT_SWIGLU: return activate<ACT_SWIGLU>(x);
    case ACT_GEGLU: return activate<ACT_GEGLU>(x);
    case ACT_REGLU: return activate<ACT_REGLU>(x);
    case ACT_RELU_SQ: return activate<ACT_RELU_SQ>(x);
    case ACT_RELU: return activate<ACT_RELU>(x);
    case ACT_GELU: return activate<ACT_GELU>(x);
    case ACT_SILU: return activate<ACT_SILU>(x);
  }
  return x;
}

// TX: int8_t, or the type that x is quantised from.
// ROWS: rows at a time.  Two are for more blocks than two to an SM: with half of the registers, and one round of loads ahead, there are
// four (14336 x 4096, one row 18.0 -> 15.2 us, 12000 x 2512 13.5 -> 10.7, 8 rows of 64 experts, 1536 x 2048, 16.4 -> 14.3; but with
// fewer blocks 4096 x 4096 6.8 -> 7.9).  An expert that has more has several blocks for
// a channel.
template <class TX, bool WIDE, bool SPLIT, int ROWS>
__global__ void __launch_bounds__(kDotThreads, ROWS == kDotRows ? 2 : 4) dot_kernel(const TX* x, long long x_ld, const int8_t* wq, long long w_ld,
                                                          const Params p, const int shares) {
  constexpr bool GIVEN = std::is_same<TX, int8_t>::value;
  constexpr int AHEAD = ROWS == kDotRows ? 2 : 1;
  __shared__ __align__(16) int8_t xs[ROWS][kDotChunk];
  __shared__ uint32_t part[ROWS][kDotWarps];
  __shared__ float row_scales[ROWS];
  __shared__ int where[3];     // expert, first row, rows
  __shared__ int parts[kDotWarps][32];
  __shared__ uint32_t owned;   // rows that an expert has (kDotMostRows at most in all)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int split = SPLIT ? shares : 1;         // warps that share the columns of a channel
  const int share = SPLIT ? warp % split : 0;
  const int n0 = (blockIdx.x * (kDotWarps / split) + warp / split) * kDotChannels;
  const int step = 512 * split;                 // columns that they load at a time
  release_next();
  // One expert: the weights are known.  The L2 fetches them while the previous kernel still runs; nothing is read, so nothing can be
  // stale (4096 x 4096 8.4 -> 7.9 us; but of 14336 x 4096, half of the L2, 18.4 -> 20.1).
  if (p.off == nullptr && static_cast<long long>(p.N) * p.K <= kDotWeights) {
    for (int j = 0; j < kDotChannels && n0 + j < p.N; ++j)
      for (int c = 4096 * share + 128 * lane; c < p.K; c += 4096 * split) asm volatile("prefetch.global.L2 [%0];" ::"l"(wq + (n0 + j) * w_ld + c));
  }
  wait_for_previous();
  // The rows of the blockIdx.y-th unit, and which rows an expert has.  All experts are looked at together (8 rows of 256 experts,
  // 312 x 1600, 10.2 -> 8.2 us); block (0, 0) then clears the rows that no expert has.
  const bool dense = p.off == nullptr;
  if (threadIdx.x == 0) {
    where[0] = 0;
    where[1] = blockIdx.y * ROWS;
    where[2] = dense ? min(p.rows - static_cast<int>(blockIdx.y) * ROWS, ROWS) : 0;
    owned = dense ? 0xFFFFFFFFu : 0u;
  }
  int before = 0;  // units, experts' rows ROWS at a time, so far
  for (int e0 = 0; e0 < p.E && !dense; e0 += kDotThreads) {
    const int e = e0 + threadIdx.x;
    int first = 0, n = 0;
    if (e < p.E) {
      first = first_row(p, e);
      n = end_row(p, e) - first;
    }
    const int units = (max(n, 0) + ROWS - 1) / ROWS;
    int at = units;  // up to this expert, later before it
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, at, d);
      if (lane >= d) at += o;
    }
    __syncthreads();  // the words above, and those of the last round have been read
    if (lane == 31) part[0][warp] = at;
    __syncthreads();
    at += before - units;
#pragma unroll
    for (int w = 0; w < kDotWarps; ++w) {
      const int c = part[0][w];
      if (w < warp) at += c;
      before += c;
    }
    if (n > 0) {
      atomicOr(&owned, (0xFFFFFFFFu >> (32 - n)) << first);
      const int mine = static_cast<int>(blockIdx.y) - at;
      if (mine >= 0 && mine < units) {
        where[0] = e;
        where[1] = first + mine * ROWS;
        where[2] = min(n - mine * ROWS, ROWS);
      }
    }
  }
  __syncthreads();
  const int e = where[0], row0 = where[1], rows = where[2];
  if (rows > 0) {
    const int8_t* w0 = wq + static_cast<long long>(e) * p.N * w_ld + static_cast<long long>(n0) * w_ld;
    // the lane's result, which COPIES neighbours have
    constexpr int COPIES = 32 / (ROWS * kDotChannels);
    const int r_out = lane / COPIES / kDotChannels, n = n0 + lane / COPIES % kDotChannels;
    const bool live = share == 0 && lane % COPIES == 0 && r_out < rows && n < p.N;
    const float ws = live ? p.w_scale[static_cast<long long>(e) * p.N + n] : 0.f;
    const float bias = live && p.bias != nullptr ? load_typed(p.bias, p.bias_type, static_cast<long long>(e) * p.N + n) : 0.f;
    uint4 w[AHEAD][kDotChannels];
    const auto fetch = [&](uint4 (&v)[kDotChannels], int c) {
#pragma unroll
      for (int j = 0; j < kDotChannels; ++j) {
        v[j] = make_uint4(0u, 0u, 0u, 0u);
        if (n0 + j < p.N && c < p.K) v[j] = __ldcs(reinterpret_cast<const uint4*>(w0 + j * w_ld + c));
      }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) fetch(w[i], step * i + 512 * share + 16 * lane);
    if constexpr (!GIVEN) {
      using L = Loaded<TX, WIDE>;
      for (int r = 0; r < rows; ++r) {
        const int s = source_row(p, row0 + r);
        uint32_t bits = 0u;
        if (s >= 0) {
          for (int c = threadIdx.x; c * L::N < p.K; c += kDotThreads) {
            L v;
            v.load(x + s * x_ld, c, p.K);
            bits = v.amax_bits(bits);
          }
        }
        bits = __reduce_max_sync(0xffffffffu, amax_as_float_bits<TX>(bits));
        if (lane == 0) part[r][warp] = bits;
      }
    }
    int acc[ROWS * kDotChannels];
#pragma unroll
    for (auto& a : acc) a = 0;
    for (int k0 = 0; k0 < p.K; k0 += kDotChunk) {
      const int kn = min(kDotChunk, (p.K - k0 + 15) / 16 * 16);
      __syncthreads();
      if constexpr (GIVEN) {
        for (int i = threadIdx.x; i < rows * (kn / 16); i += kDotThreads) {
          const int r = i / (kn / 16), c = i % (kn / 16) * 16;
          const int s = source_row(p, row0 + r);
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (s >= 0) v = *reinterpret_cast<const uint4*>(x + s * x_ld + k0 + c);
          if (k0 + c + 16 > p.K) {  // columns past the last count as zeros, whatever the caller's buffer holds there
            uint32_t* b = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int i2 = 0; i2 < 16; ++i2)
              if (k0 + c + i2 >= p.K) b[i2 / 4] &= ~(0xFFu << (8 * (i2 % 4)));
          }
          *reinterpret_cast<uint4*>(&xs[r][c]) = v;
        }
      } else {
        using L = Loaded<TX, WIDE>;
        for (int r = 0; r < rows; ++r) {
          const int s = source_row(p, row0 + r);
          uint32_t bits = part[r][0];
#pragma unroll
          for (int i = 1; i < kDotWarps; ++i) bits = max(bits, part[r][i]);
          const RowScale sc = row_scale<(sizeof(TX) == 2)>(bits);
          if (threadIdx.x == 0) row_scales[r] = s >= 0 ? scale_of_row(bits) : 0.f;
          for (int c = threadIdx.x; c * L::N < kn; c += kDotThreads) {
            L v;
            v.zero();
            if (s >= 0 && k0 + c * L::N < p.K) v.load(x + s * x_ld, k0 / L::N + c, p.K);
            v.store(sc, &xs[r][c * L::N]);
          }
        }
      }
      __syncthreads();
      for (int c0 = 512 * share + 16 * lane; c0 - 16 * lane < kn; c0 += step * AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const int c = c0 + step * i;
          uint4 v[kDotChannels];
#pragma unroll
          for (int j = 0; j < kDotChannels; ++j) v[j] = w[i][j];
          fetch(w[i], k0 + c + step * AHEAD);
          if (c >= kn) continue;
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            if (r >= rows) break;
            const uint4 q = *reinterpret_cast<const uint4*>(&xs[r][c]);
#pragma unroll
            for (int j = 0; j < kDotChannels; ++j) {
              int& a = acc[r * kDotChannels + j];
              a = __dp4a(static_cast<int>(q.x), static_cast<int>(v[j].x), a);
              a = __dp4a(static_cast<int>(q.y), static_cast<int>(v[j].y), a);
              a = __dp4a(static_cast<int>(q.z), static_cast<int>(v[j].z), a);
              a = __dp4a(static_cast<int>(q.w), static_cast<int>(v[j].w), a);
            }
          }
        }
      }
    }
    // the sums over the lanes: each step halves the sums that a lane has, as long as there are several
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      const int half = d * (ROWS * kDotChannels) / 32;
      if (half > 0) {
        const bool upper = lane & d;
#pragma unroll
        for (int i = 0; i < half; ++i) {
          const int other = __shfl_xor_sync(0xffffffffu, upper ? acc[i] : acc[i + half], d);
          acc[i] = (upper ? acc[i + half] : acc[i]) + other;
        }
      } else {
        acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], d);
      }
    }
    if constexpr (SPLIT) {
      parts[warp][lane] = acc[0];
      __syncthreads();
      if (share == 0)
        for (int i = 1; i < split; ++i) acc[0] += parts[warp + i][lane];
    }
    float y = 0.f;
    if (live) {
      float scale;
      if constexpr (GIVEN) {
        const int s = source_row(p, row0 + r_out);
        scale = s >= 0 ? p.x_scale[s] : 0.f;
      } else {
        scale = row_scales[r_out];
      }
      y = scaled(acc[0], scale, ws);
      if (p.bias != nullptr) y = biased(y, bias);
    }
    const float up = __shfl_down_sync(0xffffffffu, y, COPIES);
    if (is_gated(p.activation)) {
      if (live && (n & 1) == 0)
        store_typed(p.out, p.out_type, static_cast<long long>(row0 + r_out) * (p.N / 2) + n / 2, activate(p.activation, y) * up);
    } else if (live) {
      store_typed(p.out, p.out_type, static_cast<long long>(row0 + r_out) * p.N + n, activate(p.activation, y));
    }
  }
  if (blockIdx.x == 0 && blockIdx.y == 0) {  // rows that no expert has become zeros
    const long long bytes = static_cast<long long>(is_gated(p.activation) ? p.N / 2 : p.N) * (p.out_type == SMOE_F32 ? 4 : 2);
    for (int r = 0; r < p.rows; ++r) {
      if (owned >> r & 1u) continue;
      for (long long c = 2 * threadIdx.x; c < bytes; c += 2 * kDotThreads) *reinterpret_cast<uint16_t*>(static_cast<char*>(p.out) + r * bytes + c) = 0;
    }
  }
}

template <class TX, bool WIDE>
static int launch_dot(const void* x, long long ld, const void* wq, long long w_ld, const Params& p, cudaStream_t st) {
  // Two or four warps share a channel's columns, and a block has fewer channels, while all blocks are on the SMs at once: each warp has
  // eight loads on their way, and with few channels there are too few warps (1 row of bf16, 2048 x 7168 10.4 -> 7.0 us, 1024 x 16384
  // 20.6 -> 10.4, 4096 x 4096 7.7 -> 6.8; with four blocks to an SM 9.7; 8 rows, 1024 x 1024 6.0 -> 6.4).
  const int experts = p.rows < p.E ? p.rows : p.E;  // that can have rows
  const auto blocks = [&](int split) { return (p.N + kDotWarps * kDotChannels / split - 1) / (kDotWarps * kDotChannels / split); };
  int split = 1;
  while (split < 4 && p.K >= kDotMinCols && static_cast<long long>(blocks(2 * split)) * experts <= kDotMostBlocks) split *= 2;
  const bool many = p.rows > kDotRows || (static_cast<long long>(blocks(1)) * experts > kDotMostBlocks && (p.E > 1 || p.rows <= 2));
  const dim3 grid(blocks(many ? 1 : split), many ? (p.rows + experts) / 2 : experts);  // as many units as there may be
  const auto kernel = many ? dot_kernel<TX, WIDE, false, 2> : split > 1 ? dot_kernel<TX, WIDE, true, kDotRows> : dot_kernel<TX, WIDE, false, kDotRows>;
  return launched(launch_chained(kernel, grid, kDotThreads, 0, st, 1, static_cast<const TX*>(x), ld, static_cast<const int8_t*>(wq), w_ld,
                                 p, split));
}

template <class TX>
static int launch_dot_of(const void* x, long long ld, const void* wq, long long w_ld, const Params& p, cudaStream_t st) {
  const long long size = sizeof(TX);
  const bool wide = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld * size % 16 == 0 && p.K * size % 16 == 0;
  return wide ? launch_dot<TX, true>(x, ld, wq, w_ld, p, st) : launch_dot<TX, false>(x, ld, wq, w_ld, p, st);
}

// Whether a product goes by dot products, which read the weights at once but take longer with every row.  8-bit x, 1, 2, 4, 6, 8 rows /
// tiles, us: 1024 x 1024 3.3, 3.5, 3.7, 4.2, 4.4 / 6.8; 7168 x 2048 5.5, 5.8, 6.1, 6.8, 7.7 / 9.4; 4096 x 4096 5.9, 6.3, 7.2, 8.1, 9.0 /
// 10.2; 2048 x 7168 6.0, 6.7, 7.9, 9.3, 10.6 / 12.0; 1024 x 16384 7.8, 9.1, 12.2, 15.0, 18.2 / 19.5; large weights, 4096 x 14336 15.2,
// 16.0, 18.4, 20.9, 24.2 / 20.5.  Four rows of large weights, 8-bit x: 4096 x 14336 16.5 / 18.5, 8448 x 4096 9.9 / 11.4, 7168 x 8192 15.7 /
// 15.6, 14336 x 4096 16.9 / 14.4, 28672 x 4096 29.1 / 24.6: by tiles, which gain more than they lose.  With more than two blocks to an
// SM, bf16, 1, 2, 3 rows: 12000 x 2512 10.7, 11.0, 15.0 / 14.3; 14336 x 4096 15.2, 16.0, 19.7 / 20.5.  Rows of several experts, as a rule one each, are read along with other weights: 8 rows of 128 experts,
// 2048 x 4096, 22.6 us, quantiser and tiles 28.7; of 256, 312 x 1600, 8.2 and 21.5; 16, 24, 32 rows of 128 experts, 2048 x 4096, 32.8, 45.1,
// 55.3 and 43.0, 55.3, 67.6; of 32, 512 x 1024, 6.4, 6.9, 8.7 and 10.2, 10.8, 11.0; all 32
// in one expert 28.7 and 20.5, 7.7 and 9.2.
static bool by_dots(int rows, int N, int cols, int E) {
  if (E > 1) return rows <= kDotRows || (rows <= kDotMostRows && rows <= 2 * E);
  return rows <= (static_cast<long long>(N) * cols > kDotWeights ? 3 : N > kDotWideN ? 2 : kDotRows);
}
// Whether they quantise x themselves: a launch less (about 2 us, and 4 of the host's), but every block works on all of x.  1, 2, 3, 4 rows
// of bf16 inside / with the quantiser: 1024 x 1024 3.7, 4.5, 5.3, 6.1 / 5.2, 5.5, 5.5, 5.6; 7168 x 2048 6.1, 7.2, 8.1, 9.1 / 7.4, 7.7, 8.2,
// 8.4; 4096 x 4096 6.8, 8.2, 10.0, 11.4 / 8.3, 8.8, 9.3, 9.7; 2048 x 7168 7.0, 9.2, 11.4, 13.7 / 8.7, 9.2, 10.0, 10.8; 1024 x 16384 10.4,
// 14.5 / 10.5, 11.9; 512 x 65536 39, 61 / 31, 35.
static bool quantised_inside(int rows, int N, int cols, int E) {
  const bool inside = E > 1 ? cols <= 18432 : rows <= 4 && rows * (cols + 4096) <= 22528;
  return inside && by_dots(rows, N, cols, E);
}

static int type_bytes(int dtype) { return dtype == SMOE_F32 ? 4 : dtype == SMOE_BF16 || dtype == SMOE_F16 ? 2 : 0; }
static bool misaligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }
static long long pitch(int cols) { return (static_cast<long long>(cols) + 15) / 16 * 16; }
static size_t round256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

}  // namespace i8
}  // namespace smoe

using namespace smoe;
using namespace smoe::i8;

extern "C" {

int smoe_int8_quantize_rows(const void* x, long long ld, int dtype, void* q, long long q_ld, float* scale, long long rows, int cols,
                            void* stream) {
  if (type_bytes(dtype) == 0) return SMOE_ERR_DTYPE;
  if (rows < 0 || rows > 0x7fffffffll || cols <= 0 || cols > kMaxCols || q_ld < pitch(cols) || ld < 0) return SMOE_ERR_SHAPE;
  if (rows == 0) return SMOE_OK;
  if (x == nullptr || q == nullptr || scale == nullptr) return SMOE_ERR_SHAPE;
  if (misaligned(x, type_bytes(dtype)) || misaligned(q, 16) || q_ld % 16 != 0 || misaligned(scale, 4)) return SMOE_ERR_ALIGNMENT;
  return quantize(x, ld, dtype, q, q_ld, scale, rows, cols, S(stream));
}

size_t smoe_int8_linear_workspace_bytes(int x_dtype, int x_rows, int rows, int N, int cols, int E) {
  if (x_rows <= 0 || rows <= 0 || N <= 0 || cols <= 0 || E <= 0 || x_dtype == SMOE_I8 || quantised_inside(rows, N, cols, E)) return 0;
  return round256(static_cast<size_t>(x_rows) * pitch(cols)) + round256(static_cast<size_t>(x_rows) * 4);
}

int smoe_int8_linear(const void* x, long long ld, int x_dtype, const float* x_scale, const void* wq, long long w_ld,
                     const float* w_scale, const void* bias, int bias_dtype, void* out, int out_dtype,
                     const int* expert_frequency_offset, const int* expert_frequency, const int* x_gather_idx, int x_rows,
                     int rows, int N, int cols, int E, int activation, void* workspace, int* status, void* stream) {
  if (x_dtype != SMOE_I8 && type_bytes(x_dtype) == 0) return SMOE_ERR_DTYPE;
  if (type_bytes(out_dtype) == 0 || (bias != nullptr && type_bytes(bias_dtype) == 0)) return SMOE_ERR_DTYPE;
  if (x_rows < 0 || x_rows > kMaxRows || rows < 0 || rows > kMaxRows || N <= 0 || cols <= 0 || cols > kMaxCols || E <= 0 || E > kMaxExpertRows || ld < 0 || w_ld < cols)
    return SMOE_ERR_SHAPE;
  if (static_cast<long long>(E) * N > 0x7fffff00ll) return SMOE_ERR_SHAPE;
  if (x_dtype == SMOE_I8 && x_rows > 0 && ld < cols) return SMOE_ERR_SHAPE;
  if (activation < kNoActivation || activation > ACT_SILU || (is_gated(activation) && N % 2 != 0)) return SMOE_ERR_SHAPE;
  if (expert_frequency_offset == nullptr && (E != 1 || expert_frequency != nullptr)) return SMOE_ERR_SHAPE;
  if (x_gather_idx == nullptr && x_rows != rows) return SMOE_ERR_SHAPE;
  if (rows == 0) return SMOE_OK;
  if (x_rows == 0) return SMOE_ERR_SHAPE;
  if (wq == nullptr || w_scale == nullptr || out == nullptr || (x_rows > 0 && x == nullptr)) return SMOE_ERR_SHAPE;
  if (x_dtype == SMOE_I8 ? x_rows > 0 && x_scale == nullptr : x_scale != nullptr) return SMOE_ERR_SHAPE;
  const bool bytes_given = x_dtype == SMOE_I8;
  if (bytes_given ? misaligned(x, 16) || ld % 16 != 0 : misaligned(x, type_bytes(x_dtype))) return SMOE_ERR_ALIGNMENT;
  if (misaligned(wq, 16) || w_ld % 16 != 0 || misaligned(w_scale, 4) || misaligned(x_scale, 4) || misaligned(out, type_bytes(out_dtype)) ||
      (bias != nullptr && misaligned(bias, type_bytes(bias_dtype))) || misaligned(expert_frequency_offset, 4) ||
      misaligned(expert_frequency, 4) || misaligned(x_gather_idx, 4) || misaligned(status, 4))
    return SMOE_ERR_ALIGNMENT;
  const size_t ws = smoe_int8_linear_workspace_bytes(x_dtype, x_rows, rows, N, cols, E);
  if (ws > 0 && workspace == nullptr) return SMOE_ERR_WORKSPACE;
  if (ws > 0 && misaligned(workspace, 256)) return SMOE_ERR_ALIGNMENT;
  const long long out_cols = is_gated(activation) ? N / 2 : N;
  Params p = {};
  p.E = E; p.N = N; p.K = cols; p.rows = rows; p.x_rows = x_rows;
  p.off = expert_frequency_offset; p.count = expert_frequency; p.gather = x_gather_idx;
  p.x_scale = x_scale; p.w_scale = w_scale; p.bias = bias; p.bias_type = bias_dtype;
  p.out = out; p.out_type = out_dtype; p.activation = activation;
  p.wide_out = !misaligned(out, 16) && out_cols * type_bytes(out_dtype) % 16 == 0;
  p.status = status;
  if (!bytes_given && ws == 0) {
    switch (x_dtype) {
      case SMOE_F32: return launch_dot_of<float>(x, ld, wq, w_ld, p, S(stream));
      case SMOE_BF16: return launch_dot_of<__nv_bfloat16>(x, ld, wq, w_ld, p, S(stream));
      default: return launch_dot_of<__half>(x, ld, wq, w_ld, p, S(stream));
    }
  }
  const int8_t* xq = static_cast<const int8_t*>(x);
  if (ws > 0) {
    int8_t* q = static_cast<int8_t*>(workspace);
    float* s = reinterpret_cast<float*>(q + round256(static_cast<size_t>(x_rows) * pitch(cols)));
    const int rc = quantize(x, ld, x_dtype, q, pitch(cols), s, x_rows, cols, S(stream));
    if (rc != SMOE_OK) return rc;
    xq = q; ld = pitch(cols); p.x_scale = s;
  }
  if (by_dots(rows, N, cols, E)) return launch_dot<int8_t, true>(xq, ld, wq, w_ld, p, S(stream));
  return tensor_core_product(xq, ld, static_cast<const int8_t*>(wq), w_ld, p, S(stream));
}

}  // extern "C"
