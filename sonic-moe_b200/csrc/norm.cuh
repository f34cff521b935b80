// Root-mean-square norm of rows, with the residual's addition in front and, for the 8-bit products, 8-bit rows behind:
//   h = x + residual, rounded to the rows' type (or h = x);  r = 1 / sqrt(mean(h^2) + eps);  y = h w r
//   scale = max |y| / 127 (1 for a row of zeros);  q = 127 y / max |y| rounded half to even
// and the gradients: with g = dy w
//   dx = dresidual = dh + r (g - h r mean(g h r));  dw = sum over rows of dy h r
// h is what is kept (the residual stream), so it is rounded before it is normalised, and y is the norm of the h that a caller sees.  Everything
// else is fp32: the sum of squares, r, y before its one rounding, and the values that are quantised, which are not rounded to the
// rows' type first (a second rounding, and one step of the type in a row's maximum would move all of its values).
//
// What the kernels share: pieces of rows, and sums over the threads of a row.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>
#include <type_traits>

#include "../../include/sonicmoe_b200.h"
#include "int8.cuh"
#include "launch.cuh"

namespace smoe {
namespace norm {

constexpr int kThreads = 512;  // of a block, and of a row, at most
constexpr int kMaxWidth = 1 << 30;  // so that columns up to the next multiple of a block have 32-bit numbers

static inline cudaStream_t S(void* s) { return static_cast<cudaStream_t>(s); }
static inline long long address(const void* p) { return static_cast<long long>(reinterpret_cast<uintptr_t>(p)); }
static inline int type_bytes(int dtype) { return dtype == SMOE_F32 ? 4 : dtype == SMOE_BF16 || dtype == SMOE_F16 ? 2 : 0; }

template <class T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat162float(v);
  else return __half2float(v);
}
template <class T>
__device__ __forceinline__ T from_float(float f) {
  if constexpr (std::is_same<T, float>::value) return f;
  else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(f);
  else return __float2half_rn(f);
}

// N values that lie on a boundary of their size or 16 bytes: one access, or two.
template <class T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Piece {
  T v[N];
  __device__ __forceinline__ float operator[](int i) const { return to_float(v[i]); }
  __device__ __forceinline__ void set(int i, float f) { v[i] = from_float<T>(f); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = from_float<T>(0.f);
  }
  // of rows, which are read once
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(Piece) == 16) *reinterpret_cast<uint4*>(this) = __ldcs(reinterpret_cast<const uint4*>(p));
    else *this = *reinterpret_cast<const Piece*>(p);
  }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Piece*>(p) = *this; }
  // of the weights, which every row reads
  __device__ __forceinline__ void load_shared(const T* p, bool wide) {
    if (wide) {
      *this = *reinterpret_cast<const Piece*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = p[i];
    }
  }
};

// Sum (and maximum of `bits`) over the 2^log2 threads of a row, the same in all of them and in the same order every time.  part, part_bits:
// a word for each warp of the block.  All threads of the block.
template <bool MAX>
__device__ __forceinline__ void row_reduce(float& sum, uint32_t& bits, int log2, float* part, uint32_t* part_bits) {
  for (int o = min(1 << log2, 32) >> 1; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (MAX) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
  }
  if (log2 <= 5) return;
  const int warp = threadIdx.x >> 5, of_row = 1 << (log2 - 5), first = warp & ~(of_row - 1);
  if ((threadIdx.x & 31) == 0) {
    part[warp] = sum;
    if (MAX) part_bits[warp] = bits;
  }
  __syncthreads();
  sum = 0.f;
  for (int w = 0; w < of_row; ++w) {
    sum += part[first + w];
    if (MAX) bits = max(bits, part_bits[first + w]);
  }
}

// The largest access in bytes, 16 at most, that every one of `sizes` (addresses, distances) is a multiple of.
static inline int access_bytes(std::initializer_list<long long> sizes) {
  long long all = 16;
  for (const long long s : sizes) all |= s;
  return static_cast<int>(all & -all);
}
// Threads of a row as a power of two, `ep` values in each.
static inline int row_threads_log2(int H, int ep) {
  int log2 = 0;
  while ((static_cast<long long>(ep) << log2) < H) ++log2;
  return log2;
}

// go(T(), W()) for rows of type T and weights of type W.
template <class F>
static inline int for_types(int dtype, int weight_dtype, F go) {
  if (dtype == SMOE_F32) return go(float(), float());
  if (dtype == SMOE_BF16) return weight_dtype == SMOE_F32 ? go(__nv_bfloat16(), float()) : go(__nv_bfloat16(), __nv_bfloat16());
  return weight_dtype == SMOE_F32 ? go(__half(), float()) : go(__half(), __half());
}
// go(constant<VE>) with the values of an access: 16 bytes, or 4 or 2 where rows start elsewhere.
template <class T, class F>
static inline auto for_access(int bytes, F go) {
  if (bytes == 16) return go(std::integral_constant<int, 16 / static_cast<int>(sizeof(T))>());
  if constexpr (sizeof(T) == 2) {
    if (bytes >= 4) return go(std::integral_constant<int, 2>());
  }
  return go(std::integral_constant<int, 1>());
}

}  // namespace norm
}  // namespace smoe
