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

#include <type_traits>

#include "../../include/sonicmoe_b200.h"
#include "int8.cuh"
#include "launch.cuh"

namespace smoe {
namespace norm {

constexpr int kThreads = 512;        // of a block, and of a row, at most
constexpr int kMaxWidth = 1 << 28;   // so that bytes of a row have 32-bit numbers

static inline cudaStream_t S(void* s) { return static_cast<cudaStream_t>(s); }
static inline long long address(const void* p) { return static_cast<long long>(reinterpret_cast<uintptr_t>(p)); }
static inline int type_bytes(int dtype) { return dtype == SMOE_F32 ? 4 : dtype == SMOE_BF16 || dtype == SMOE_F16 ? 2 : 0; }

// Two fp32 values that are added and multiplied by one instruction, each rounded as by itself.
struct F2 {
  uint64_t v;
  __device__ __forceinline__ F2() {}
  __device__ __forceinline__ F2(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
  __device__ __forceinline__ void split(float& x, float& y) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
  __device__ __forceinline__ float sum() const {
    float x, y;
    split(x, y);
    return x + y;
  }
};
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// Columns of a row in pieces of 16 bytes of the rows that are written (packed, from a 16-byte boundary on): piece c has the VE columns from
// VE c - shift on, where shift is what the row begins behind its first 16-byte boundary, in values.  ALIGNED: rows of whole pieces,
// all of which start on such a boundary.
template <class T>
constexpr int kValues = 16 / static_cast<int>(sizeof(T));  // VE
template <class T, bool ALIGNED>
struct Columns {
  int H, shift, pieces;
  __device__ __forceinline__ Columns(long long row, int width) : H(width) {
    constexpr int VE = kValues<T>;
    shift = ALIGNED ? 0 : static_cast<int>(static_cast<unsigned>(row) * static_cast<unsigned>(width) & (VE - 1));
    pieces = (H + shift + VE - 1) / VE;
  }
  __device__ __forceinline__ int first(int c) const { return c * kValues<T> - shift; }
  __device__ __forceinline__ bool whole(int c) const { return first(c) >= 0 && first(c) + kValues<T> <= H; }
  // a bit for each value of piece c that lies in the row
  __device__ __forceinline__ uint32_t valid(int c) const {
    constexpr uint32_t all = (1u << kValues<T>) - 1u;
    return (all << max(0, -first(c))) & (all >> max(0, first(c) + kValues<T> - H));
  }
};

// EP values of a row in a thread, in pieces of VE values (of the rows that are written, for weights of another type too), as they are in memory.
template <class T, int EP, int VE>
struct Values {
  static constexpr int P = EP / VE, WORDS = VE * static_cast<int>(sizeof(T)) / 4;  // pieces, words of a piece
  uint32_t w[EP * sizeof(T) / 4];
  __device__ __forceinline__ F2 get(int k) const {
    if constexpr (std::is_same<T, float>::value) return F2(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
    if constexpr (std::is_same<T, __nv_bfloat16>::value) return F2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xFFFF0000u));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[sizeof(T) == 2 ? k : 0]));
    return F2(f.x, f.y);
  }
  __device__ __forceinline__ void set(int k, F2 f) {
    float x, y;
    f.split(x, y);
    if constexpr (std::is_same<T, float>::value) {
      w[2 * k] = __float_as_uint(x);
      w[2 * k + 1] = __float_as_uint(y);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[k]) : "f"(y), "f"(x));
    } else {
      asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[k]) : "f"(y), "f"(x));
    }
  }
  // the sum of two values rounded once
  __device__ __forceinline__ void add(int k, const Values& o) {
    if constexpr (std::is_same<T, float>::value) {
      w[2 * k] = __float_as_uint(__uint_as_float(w[2 * k]) + __uint_as_float(o.w[2 * k]));
      w[2 * k + 1] = __float_as_uint(__uint_as_float(w[2 * k + 1]) + __uint_as_float(o.w[2 * k + 1]));
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(w[k]) : "r"(o.w[k]));
    } else {
      asm("add.rn.f16x2 %0, %0, %1;" : "+r"(w[k]) : "r"(o.w[k]));
    }
  }
  // Keeps the compiler from holding on to 16-bit values as fp32, in twice the registers, from one use to the next.
  __device__ __forceinline__ void forget() {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (auto& x : w) asm volatile("" : "+r"(x));
    }
  }
  __device__ __forceinline__ void clear(int i) {
#pragma unroll
    for (int j = 0; j < WORDS; ++j) w[i * WORDS + j] = 0u;
  }
  // Pieces c0, c0 + step, .. of a row that starts at `row`, zeros where there are none.  WIDE: every piece is whole and starts on a 16-byte
  // boundary.  Otherwise the 16-byte blocks that hold it, one or two, are loaded, with what else they hold, and none that holds nothing
  // of the row.  ONCE: nobody reads them again.
  template <bool WIDE, bool ONCE, class C>
  __device__ __forceinline__ void load(const T* row, const C& columns, int c0, int step) {
    const char* bytes = reinterpret_cast<const char*>(row) - columns.shift * static_cast<int>(sizeof(T));  // of piece 0
    const int off = WIDE ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(bytes) & 15);
    const int begin = columns.shift * static_cast<int>(sizeof(T)), end = begin + columns.H * static_cast<int>(sizeof(T));
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = c0 + i * step;
      if (c >= columns.pieces) {
        clear(i);
        continue;
      }
#pragma unroll
      for (int j = 0; j < WORDS; j += 4) {
        const int at = 4 * (c * WORDS + j) - off;
        const auto block = [&](int o) {
          const uint4* from = reinterpret_cast<const uint4*>(bytes + o);
          if (!WIDE && (o + 16 <= begin || o >= end)) return make_uint4(0u, 0u, 0u, 0u);
          return ONCE ? __ldcs(from) : *from;
        };
        uint4 q = block(at);
        if (!WIDE && off != 0) {
          const uint4 r = block(at + 16);
          uint32_t v[8] = {q.x, q.y, q.z, q.w, r.x, r.y, r.z, r.w};
          if (off & 8) {
#pragma unroll
            for (int k = 0; k < 6; ++k) v[k] = v[k + 2];
          }
          if (off & 4) {
#pragma unroll
            for (int k = 0; k < 5; ++k) v[k] = v[k + 1];
          }
          if (sizeof(T) == 2) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = __funnelshift_r(v[k], v[k + 1], 8 * (off & 2));
          }
          q = make_uint4(v[0], v[1], v[2], v[3]);
        }
        w[i * WORDS + j] = q.x; w[i * WORDS + j + 1] = q.y; w[i * WORDS + j + 2] = q.z; w[i * WORDS + j + 3] = q.w;
      }
    }
  }
  // What `load` brought in from beyond the row's ends becomes zeros.
  template <bool WIDE, class C>
  __device__ __forceinline__ void mask(const C& columns, int c0, int step) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = c0 + i * step;
      if (WIDE || c >= columns.pieces || columns.whole(c)) continue;
      const uint32_t valid = columns.valid(c);
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        if constexpr (sizeof(T) == 4) w[i * WORDS + j] &= valid & (1u << j) ? 0xFFFFFFFFu : 0u;
        else if (j % 2 == 0) w[i * WORDS + j / 2] &= (valid & (1u << j) ? 0x0000FFFFu : 0u) | (valid & (2u << j) ? 0xFFFF0000u : 0u);
      }
    }
  }
  // (to rows of the type that the pieces are of)
  template <bool WIDE, class C>
  __device__ __forceinline__ void store(T* row, const C& columns, int c0, int step) const {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = c0 + i * step;
      if (c >= columns.pieces) continue;
      if (WIDE || columns.whole(c)) {
        *reinterpret_cast<uint4*>(row + columns.first(c)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        continue;
      }
      const uint32_t valid = columns.valid(c);
      char* to = reinterpret_cast<char*>(row) + static_cast<long long>(columns.first(c)) * static_cast<int>(sizeof(T));
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (valid & (1u << j)) *reinterpret_cast<uint32_t*>(to + 4 * j) = w[4 * i + j];
      } else {  // eight, four and two bytes at a time
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const uint32_t mine = valid >> (2 * j);
          if ((mine & 15u) == 15u) {
            *reinterpret_cast<uint2*>(to + 4 * j) = make_uint2(w[4 * i + j], w[4 * i + j + 1]);
            continue;
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t two = mine >> (2 * k) & 3u, word = w[4 * i + j + k];
            if (two == 3u) *reinterpret_cast<uint32_t*>(to + 4 * (j + k)) = word;
            else if (two != 0u) *reinterpret_cast<uint16_t*>(to + 4 * (j + k) + 2 * (two >> 1)) = static_cast<uint16_t>(two == 1u ? word : word >> 16);
          }
        }
      }
    }
  }
};

// How the threads of a block are shared out: `tpr` threads have a row, a power of two up to 32 or whole warps, and a block has `subs` rows at
// a time, of which this thread has a part of row `sub`.
struct Share {
  int tpr, subs, sub, tid;
  __device__ __forceinline__ explicit Share(int threads_of_row) : tpr(threads_of_row), subs(1), sub(0), tid(threadIdx.x) {
    if (blockDim.x != tpr) {
      subs = blockDim.x / tpr;
      sub = threadIdx.x / tpr;
      tid = threadIdx.x - sub * tpr;
    }
  }
};

// The larger magnitude of two and a maximum so far; NaN if one of them is.
__device__ __forceinline__ float max_abs(float m, float x, float y) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(x), "f"(y));
  return r;
}

// Sum (and largest magnitude) over the threads of a row, the same in all of them and in the same order every time.  All threads of the
// block; another array every other time, or a barrier between two calls.
struct Parts {
  float sum[kThreads / 32], most[kThreads / 32];
};
template <bool MAX>
__device__ __forceinline__ void row_reduce(float& sum, float& most, const Share& at, Parts& part) {
  const auto join = [&](int o) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (MAX) {
      const float other = __shfl_xor_sync(0xffffffffu, most, o);
      most = max_abs(most, other, other);
    }
  };
  if (at.tpr >= 32) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) join(o);
  } else {
    for (int o = at.tpr >> 1; o > 0; o >>= 1) join(o);
  }
  if (at.tpr <= 32) return;
  const int warp = threadIdx.x >> 5, of_row = at.tpr >> 5, first = at.sub * of_row;
  if ((threadIdx.x & 31) == 0) {
    part.sum[warp] = sum;
    if (MAX) part.most[warp] = most;
  }
  __syncthreads();
  sum = part.sum[first];
  if (MAX) most = part.most[first];
#pragma unroll 4
  for (int w = 1; w < of_row; ++w) {
    sum += part.sum[first + w];
    if (MAX) most = max_abs(most, part.most[first + w], part.most[first + w]);
  }
}

// 1 / sqrt(x): the hardware's approximation (2 units), corrected by one step of Newton's method for r^-2 = x to within 1 unit; 0 and
// infinity as they come.
__device__ __forceinline__ float inverse_root(float x) {
  float r;
  asm("rsqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  const float better = fmaf(0.5f * r, fmaf(-x * r, r, 1.f), r);
  return r > 0.f && r < __int_as_float(0x7F800000) ? better : r;
}

// Threads of a row of `values` values, `ep` in each, and of a block.
struct Shape {
  int tpr, threads, subs;
};
static inline Shape shape_of(long long values, int ep) {
  Shape s = {};
  const long long need = (values + ep - 1) / ep;
  s.tpr = 1;
  while (s.tpr < 32 && s.tpr < need) s.tpr *= 2;
  if (need > 32) s.tpr = static_cast<int>((need + 31) / 32 * 32);
  s.subs = s.tpr < 256 ? 256 / s.tpr : 1;
  s.threads = s.subs * s.tpr;
  return s;
}

// go(T(), W()) for rows of type T and weights of type W.
template <class F>
static inline int for_types(int dtype, int weight_dtype, F go) {
  if (dtype == SMOE_F32) return go(float(), float());
  if (dtype == SMOE_BF16) return weight_dtype == SMOE_F32 ? go(__nv_bfloat16(), float()) : go(__nv_bfloat16(), __nv_bfloat16());
  return weight_dtype == SMOE_F32 ? go(__half(), float()) : go(__half(), __half());
}

}  // namespace norm
}  // namespace smoe
