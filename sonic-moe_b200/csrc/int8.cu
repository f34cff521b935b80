// 8-bit integer products: quantisation of rows and the entry points (the formulas are in int8.cuh).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>
#include <type_traits>

#include "../../include/sonicmoe_b200.h"
#include "int8.cuh"

namespace smoe {
namespace i8 {

static inline cudaStream_t S(void* s) { return static_cast<cudaStream_t>(s); }

// ----------------------------------------------------------------------------------------------
// quantisation
// ----------------------------------------------------------------------------------------------
// A row is read once, PIECES accesses of BYTES bytes per thread, and stays in registers between the maximum and the
// conversion; `tpr` threads (a power of two) share it, and a block of 256 threads (or one row's) has 256 / tpr rows.  Rows that
// are longer than 1024 threads hold are read twice.  Bound by memory.
template <class T, int BYTES>
struct Loaded {
  static constexpr int N = BYTES / static_cast<int>(sizeof(T));
  uint32_t w[BYTES >= 4 ? BYTES / 4 : 1];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (BYTES == 16) {
      const uint4 q = __ldcs(reinterpret_cast<const uint4*>(p));
      w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    } else if constexpr (BYTES == 4) {
      w[0] = __ldcs(reinterpret_cast<const unsigned*>(p));
    } else {
      w[0] = __ldcs(reinterpret_cast<const unsigned short*>(p));
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (auto& x : w) x = 0u;
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    const unsigned short h = static_cast<unsigned short>(w[i / 2] >> (16 * (i & 1)));
    if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(h));
    return __bfloat162float(__ushort_as_bfloat16(h));
  }
  __device__ __forceinline__ uint32_t amax_bits() const {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(value(i)) & 0x7FFFFFFFu);
    return m;
  }
  __device__ __forceinline__ void store(const RowScale& s, int8_t* q) const {
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = value(i);
    uint32_t o[(N + 3) / 4];
    quantize_values<N>(s, f, o);
    if constexpr (N == 8) *reinterpret_cast<uint2*>(q) = make_uint2(o[0], o[1]);
    else if constexpr (N == 4) *reinterpret_cast<uint32_t*>(q) = o[0];
    else if constexpr (N == 2) *reinterpret_cast<uint16_t*>(q) = static_cast<uint16_t>(o[0]);
    else *q = static_cast<int8_t>(o[0]);
  }
};

template <class T, int BYTES>
__global__ void __launch_bounds__(1024) quantize_rows_kernel(const T* x, long long ld, int8_t* q, long long q_ld, float* scale,
                                                             long long rows, int cols, int tpr) {
  release_next();
  wait_for_previous();
  using L = Loaded<T, BYTES>;
  constexpr int PIECES = BYTES == 16 ? 4 : 8;
  __shared__ uint32_t part[32];
  const int per_block = blockDim.x / tpr, sub = threadIdx.x / tpr, tid = threadIdx.x % tpr;
  const long long row = static_cast<long long>(blockIdx.x) * per_block + sub;
  const bool live = row < rows;
  const int pieces = (cols + L::N - 1) / L::N;  // cols is a multiple of N
  const T* src = x + (live ? row : 0) * ld;
  const bool kept = pieces <= PIECES * tpr;
  L v[PIECES];
  uint32_t bits = 0u;
  if (kept) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int c = i * tpr + tid;
      if (live && c < pieces) v[i].load(src + c * L::N); else v[i].zero();
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) bits = max(bits, v[i].amax_bits());
  } else if (live) {
    for (int c = tid; c < pieces; c += tpr) {
      v[0].load(src + c * L::N);
      bits = max(bits, v[0].amax_bits());
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, d));  // tpr >= 32
  if (tpr > 32) {
    const int warp = threadIdx.x >> 5, of_row = tpr >> 5;
    if ((threadIdx.x & 31) == 0) part[warp] = bits;
    __syncthreads();
    for (int w = 0; w < of_row; ++w) bits = max(bits, part[sub * of_row + w]);
  }
  if (!live) return;
  const RowScale s = row_scale(bits);
  int8_t* dst = q + row * q_ld;
  if (tid == 0) scale[row] = s.scale;
  if (kept) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int c = i * tpr + tid;
      if (c < pieces) v[i].store(s, dst + c * L::N);
    }
  } else {
    for (int c = tid; c < pieces; c += tpr) {
      v[0].load(src + c * L::N);
      v[0].store(s, dst + c * L::N);
    }
  }
  for (int c = cols + tid; c < (cols + 15) / 16 * 16; c += tpr) dst[c] = 0;
}

template <class T, int BYTES>
static cudaError_t launch_quantize(const void* x, long long ld, void* q, long long q_ld, float* scale, long long rows, int cols,
                                   cudaStream_t st) {
  constexpr int N = BYTES / static_cast<int>(sizeof(T)), PIECES = BYTES == 16 ? 4 : 8;
  const int pieces = (cols + N - 1) / N;
  int tpr = 32;
  while (tpr < 1024 && tpr * PIECES < pieces) tpr *= 2;
  const int threads = tpr > 256 ? tpr : 256;
  const long long blocks = (rows + threads / tpr - 1) / (threads / tpr);
  return launch_chained(quantize_rows_kernel<T, BYTES>, dim3(static_cast<unsigned>(blocks)), threads, 0, st, 1, static_cast<const T*>(x), ld,
                        static_cast<int8_t*>(q), q_ld, scale, rows, cols, tpr);
}

static int quantize(const void* x, long long ld, int dtype, void* q, long long q_ld, float* scale, long long rows, int cols,
                    cudaStream_t st) {
  const int size = dtype == SMOE_F32 ? 4 : 2;
  const auto fits = [&](int bytes) {
    return reinterpret_cast<uintptr_t>(x) % bytes == 0 && (ld * size) % bytes == 0 && (static_cast<long long>(cols) * size) % bytes == 0;
  };
  cudaError_t rc;
  if (dtype == SMOE_F32)
    rc = fits(16) ? launch_quantize<float, 16>(x, ld, q, q_ld, scale, rows, cols, st) : launch_quantize<float, 4>(x, ld, q, q_ld, scale, rows, cols, st);
  else if (dtype == SMOE_BF16)
    rc = fits(16)  ? launch_quantize<__nv_bfloat16, 16>(x, ld, q, q_ld, scale, rows, cols, st)
         : fits(4) ? launch_quantize<__nv_bfloat16, 4>(x, ld, q, q_ld, scale, rows, cols, st)
                   : launch_quantize<__nv_bfloat16, 2>(x, ld, q, q_ld, scale, rows, cols, st);
  else
    rc = fits(16)  ? launch_quantize<__half, 16>(x, ld, q, q_ld, scale, rows, cols, st)
         : fits(4) ? launch_quantize<__half, 4>(x, ld, q, q_ld, scale, rows, cols, st)
                   : launch_quantize<__half, 2>(x, ld, q, q_ld, scale, rows, cols, st);
  return launched(rc);
}

// ----------------------------------------------------------------------------------------------
// product by 4-way integer dot products
// ----------------------------------------------------------------------------------------------
// A block takes up to 8 rows of one expert and 32 channels: its rows lie in shared memory, 4096 columns at a time; a warp has
// four channels, whose weights its lanes load 16 bytes each, straight from memory.  The weights are read once for 8 rows.
constexpr int kDotMaxRows = 8;
constexpr int kDotRows = 8, kDotChannels = 4, kDotWarps = 8, kDotChunk = 4096;

__global__ void __launch_bounds__(32 * kDotWarps) dot_kernel(const int8_t* xq, long long x_ld, const int8_t* wq, long long w_ld,
                                                             long long w_expert, const Params p) {
  release_next();
  wait_for_previous();
  __shared__ __align__(16) int8_t xs[kDotRows][kDotChunk];
  __shared__ int where[3];  // expert, first row, rows
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp == 0) {  // the expert whose chunks of rows contain blockIdx.y
    int before = 0, e0 = 0, mine = -1;
    for (e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane;
      const int rows = e < p.E ? max(end_row(p, e) - first_row(p, e), 0) : 0;
      int incl = (rows + kDotRows - 1) / kDotRows;
      const int own = incl;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += o;
      }
      const int at = static_cast<int>(blockIdx.y) - (before + incl - own);
      if (at >= 0 && at < own) {
        where[0] = e;
        where[1] = first_row(p, e) + at * kDotRows;
        where[2] = min(kDotRows, rows - at * kDotRows);
        mine = e;
      }
      if (__any_sync(0xffffffffu, mine >= 0)) break;
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (!__any_sync(0xffffffffu, mine >= 0) && lane == 0) where[2] = 0;
  }
  __syncthreads();
  const int e = where[0], row0 = where[1], rows = where[2];
  const int n0 = (blockIdx.x * kDotWarps + warp) * kDotChannels;
  if (rows > 0) {
    int acc[kDotRows * kDotChannels];
#pragma unroll
    for (auto& a : acc) a = 0;
    for (int k0 = 0; k0 < p.K; k0 += kDotChunk) {
      const int kn = min(kDotChunk, (p.K - k0 + 15) / 16 * 16);  // columns up to the next 16 exist, and those of x are zeros
      __syncthreads();
      for (int i = threadIdx.x; i < kDotRows * (kn / 16); i += blockDim.x) {
        const int r = i / (kn / 16), c = i % (kn / 16) * 16;
        const int s = r < rows ? source_row(p, row0 + r) : -1;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (s >= 0) v = *reinterpret_cast<const uint4*>(xq + s * x_ld + k0 + c);
        if (k0 + c + 16 > p.K) {  // columns past the last count as zeros, whatever the caller's buffer holds there
          uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
          for (int b = 0; b < 16; ++b)
            if (k0 + c + b >= p.K) w[b / 4] &= ~(0xFFu << (8 * (b % 4)));
        }
        *reinterpret_cast<uint4*>(&xs[r][c]) = v;
      }
      __syncthreads();
      for (int c = 16 * lane; c < kn; c += 512) {
        uint4 w[kDotChannels];
#pragma unroll
        for (int j = 0; j < kDotChannels; ++j) {
          w[j] = make_uint4(0u, 0u, 0u, 0u);
          if (n0 + j < p.N) w[j] = __ldcs(reinterpret_cast<const uint4*>(wq + e * w_expert + (n0 + j) * w_ld + k0 + c));
        }
#pragma unroll
        for (int r = 0; r < kDotRows; ++r) {
          const uint4 v = *reinterpret_cast<const uint4*>(&xs[r][c]);
#pragma unroll
          for (int j = 0; j < kDotChannels; ++j) {
            int& a = acc[r * kDotChannels + j];
            a = __dp4a(static_cast<int>(v.x), static_cast<int>(w[j].x), a);
            a = __dp4a(static_cast<int>(v.y), static_cast<int>(w[j].y), a);
            a = __dp4a(static_cast<int>(v.z), static_cast<int>(w[j].z), a);
            a = __dp4a(static_cast<int>(v.w), static_cast<int>(w[j].w), a);
          }
        }
      }
    }
    // 32 sums over 32 lanes: afterwards lane l has that of row l / 4, channel l % 4
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      const bool upper = lane & d;
#pragma unroll
      for (int i = 0; i < d; ++i) {
        const int other = __shfl_xor_sync(0xffffffffu, upper ? acc[i] : acc[i + d], d);
        acc[i] = (upper ? acc[i + d] : acc[i]) + other;
      }
    }
    const int r = lane / kDotChannels, n = n0 + lane % kDotChannels;
    const bool live = r < rows && n < p.N;
    float y = 0.f;
    if (live) {
      const int s = source_row(p, row0 + r);
      y = scaled(acc[0], s >= 0 ? p.x_scale[s] : 0.f, p.w_scale[static_cast<long long>(e) * p.N + n]);
      if (p.bias != nullptr) y += load_typed(p.bias, p.bias_type, static_cast<long long>(e) * p.N + n);
    }
    const float up = __shfl_down_sync(0xffffffffu, y, 1);
    if (p.activation >= 0 && act_is_gated(p.activation)) {
      if (live && (n & 1) == 0)
        store_typed(p.out, p.out_type, static_cast<long long>(row0 + r) * (p.N / 2) + n / 2, activate(p.activation, y) * up);
    } else if (live) {
      store_typed(p.out, p.out_type, static_cast<long long>(row0 + r) * p.N + n, activate(p.activation, y));
    }
  }
  zero_other_rows(p, (blockIdx.y * gridDim.x + blockIdx.x) * kDotWarps + warp, gridDim.x * gridDim.y * kDotWarps);
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

size_t smoe_int8_linear_workspace_bytes(int x_dtype, int x_rows, int cols) {
  if (x_rows <= 0 || cols <= 0 || x_dtype == SMOE_I8) return 0;
  return round256(static_cast<size_t>(x_rows) * pitch(cols)) + round256(static_cast<size_t>(x_rows) * 4);
}

int smoe_int8_linear(const void* x, long long ld, int x_dtype, const float* x_scale, const void* wq, long long w_ld,
                     const float* w_scale, const void* bias, int bias_dtype, void* out, int out_dtype,
                     const int* expert_frequency_offset, const int* expert_frequency, const int* x_gather_idx, int x_rows,
                     int rows, int N, int cols, int E, int activation, void* workspace, int* status, void* stream) {
  if (x_dtype != SMOE_I8 && type_bytes(x_dtype) == 0) return SMOE_ERR_DTYPE;
  if (type_bytes(out_dtype) == 0 || (bias != nullptr && type_bytes(bias_dtype) == 0)) return SMOE_ERR_DTYPE;
  if (x_rows < 0 || rows < 0 || N <= 0 || cols <= 0 || cols > kMaxCols || E <= 0 || E > kMaxExpertRows || ld < 0 || w_ld < cols)
    return SMOE_ERR_SHAPE;
  if (static_cast<long long>(E) * N > 0x7fffff00ll) return SMOE_ERR_SHAPE;
  if (x_dtype == SMOE_I8 && x_rows > 0 && ld < cols) return SMOE_ERR_SHAPE;
  if (activation < kNoActivation || activation > ACT_SILU || (activation >= 0 && act_is_gated(activation) && N % 2 != 0)) return SMOE_ERR_SHAPE;
  if (expert_frequency_offset == nullptr && (E != 1 || expert_frequency != nullptr)) return SMOE_ERR_SHAPE;
  if (x_gather_idx == nullptr && x_rows != rows) return SMOE_ERR_SHAPE;
  if (rows == 0) return SMOE_OK;
  if (wq == nullptr || w_scale == nullptr || out == nullptr || (x_rows > 0 && x == nullptr)) return SMOE_ERR_SHAPE;
  if (x_dtype == SMOE_I8 ? x_rows > 0 && x_scale == nullptr : x_scale != nullptr) return SMOE_ERR_SHAPE;
  const bool bytes_given = x_dtype == SMOE_I8;
  if (bytes_given ? misaligned(x, 16) || ld % 16 != 0 : misaligned(x, type_bytes(x_dtype))) return SMOE_ERR_ALIGNMENT;
  if (misaligned(wq, 16) || w_ld % 16 != 0 || misaligned(w_scale, 4) || misaligned(x_scale, 4) || misaligned(out, type_bytes(out_dtype)) ||
      (bias != nullptr && misaligned(bias, type_bytes(bias_dtype))) || misaligned(expert_frequency_offset, 4) ||
      misaligned(expert_frequency, 4) || misaligned(x_gather_idx, 4) || misaligned(status, 4))
    return SMOE_ERR_ALIGNMENT;
  const size_t ws = smoe_int8_linear_workspace_bytes(x_dtype, x_rows, cols);
  if (ws > 0 && workspace == nullptr) return SMOE_ERR_WORKSPACE;
  if (ws > 0 && misaligned(workspace, 256)) return SMOE_ERR_ALIGNMENT;
  const int8_t* xq = static_cast<const int8_t*>(x);
  if (ws > 0) {
    int8_t* q = static_cast<int8_t*>(workspace);
    float* s = reinterpret_cast<float*>(q + round256(static_cast<size_t>(x_rows) * pitch(cols)));
    const int rc = quantize(x, ld, x_dtype, q, pitch(cols), s, x_rows, cols, S(stream));
    if (rc != SMOE_OK) return rc;
    xq = q; ld = pitch(cols); x_scale = s;
  }
  const long long out_cols = activation >= 0 && act_is_gated(activation) ? N / 2 : N;
  Params p = {};
  p.E = E; p.N = N; p.K = cols; p.rows = rows; p.x_rows = x_rows;
  p.off = expert_frequency_offset; p.count = expert_frequency; p.gather = x_gather_idx;
  p.x_scale = x_scale; p.w_scale = w_scale; p.bias = bias; p.bias_type = bias_dtype;
  p.out = out; p.out_type = out_dtype; p.activation = activation;
  p.wide_out = !misaligned(out, 16) && out_cols * type_bytes(out_dtype) % 16 == 0;
  p.status = status;
  if (rows > kDotMaxRows && x_rows > 0) return tensor_core_product(xq, ld, static_cast<const int8_t*>(wq), w_ld, p, S(stream));
  p.zero_others = 1;
  const long long chunks = (static_cast<long long>(rows) + kDotRows - 1) / kDotRows + (E > 1 ? (rows < E ? rows : E) : 0);
  if (chunks > 65535) return SMOE_ERR_SHAPE;  // only without any row of x
  const dim3 grid((N + kDotWarps * kDotChannels - 1) / (kDotWarps * kDotChannels), static_cast<unsigned>(chunks));
  return launched(launch_chained(dot_kernel, grid, 32 * kDotWarps, 0, S(stream), 1, xq, ld, static_cast<const int8_t*>(wq), w_ld,
                                 static_cast<long long>(N) * w_ld, p));
}

}  // extern "C"
