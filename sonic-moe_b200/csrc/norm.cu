// Root-mean-square norm, forward (the formulas are in norm.cuh).
#include "norm.cuh"

namespace smoe {
namespace norm {

struct Forward {
  const void* x; long long x_ld;            // values from row to row
  const void* res; long long res_ld;        // or nullptr
  const void* w; int w_wide;                // weights of the columns start on 16-byte boundaries
  void* y;                                  // packed rows, or nullptr
  void* h;                                  // packed rows, or nullptr
  float* rstd;                              // (rows), or nullptr
  int8_t* q; long long q_ld; float* scale;  // or nullptr
  long long rows;
  int H;
  float eps;
};

// VE 8-bit values of b, the `i`-th VE of them.
template <int VE, int N>
__device__ __forceinline__ void store_bytes(int8_t* q, const uint32_t (&b)[N], int i) {
  if constexpr (VE == 8) *reinterpret_cast<uint2*>(q) = make_uint2(b[2 * i], b[2 * i + 1]);
  else if constexpr (VE == 4) *reinterpret_cast<uint32_t*>(q) = b[i];
  else if constexpr (VE == 2) *reinterpret_cast<uint16_t*>(q) = static_cast<uint16_t>(b[i / 2] >> (16 * (i & 1)));
  else *q = static_cast<int8_t>(b[i / 4] >> (8 * (i & 3)));
}

// A row is read once and stays in registers, EP values in each of its 2^log2 threads.  Bound by memory.  y = (h w) r: the maximum of |h w|
// times r is that of |y|, whatever is rounded on the way, so that one reduction serves both.  LONG: rows that a block's threads
// do not hold are read twice, EP values of each thread at a time.
template <class T, class W, int VE, int EP, bool Q, bool LONG>
__global__ void __launch_bounds__(kThreads) forward_kernel(const Forward a, int log2) {
  release_next();
  wait_for_previous();
  constexpr int P = EP / VE;
  __shared__ float part[kThreads / 32];
  __shared__ uint32_t part_bits[kThreads / 32];
  const int tpr = 1 << log2, sub = threadIdx.x >> log2, tid = threadIdx.x & (tpr - 1);
  const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x >> log2) + sub;
  const bool live = row < a.rows;
  const int pieces = live ? a.H / VE : 0;
  const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
  const T* res = static_cast<const T*>(a.res) + row * a.res_ld;
  const W* weight = static_cast<const W*>(a.w);
  Piece<T, VE> h[P];
  Piece<W, VE> w[P];
  // pieces c0, c0 + tpr, ..: h on its way out the first time
  const auto take = [&](int c0, bool first) {
    Piece<T, VE> r[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = c0 + i * tpr;
      if (c < pieces) h[i].load(x + static_cast<long long>(c) * VE); else h[i].zero();
    }
    if (a.res != nullptr) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int c = c0 + i * tpr;
        if (c < pieces) r[i].load(res + static_cast<long long>(c) * VE); else r[i].zero();
      }
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = c0 + i * tpr;
      if (c < pieces) w[i].load_shared(weight + static_cast<long long>(c) * VE, a.w_wide); else w[i].zero();
    }
    if (a.res != nullptr) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int c = c0 + i * tpr;
#pragma unroll
        for (int j = 0; j < VE; ++j) h[i].set(j, h[i][j] + r[i][j]);
        if (first && a.h != nullptr && c < pieces) h[i].store(static_cast<T*>(a.h) + row * a.H + static_cast<long long>(c) * VE);
      }
    }
  };
  float sum = 0.f;
  uint32_t bits = 0u;
  for (int c0 = tid; c0 < (LONG ? pieces : tid + 1); c0 += P * tpr) {
    take(c0, true);
#pragma unroll
    for (int i = 0; i < P; ++i) {
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        sum = fmaf(h[i][j], h[i][j], sum);
        if (Q) bits = max(bits, __float_as_uint(h[i][j] * w[i][j]) & 0x7FFFFFFFu);
      }
    }
  }
  row_reduce<Q>(sum, bits, log2, part, part_bits);
  if (!live) return;
  const float r = __frsqrt_rn(sum / static_cast<float>(a.H) + a.eps);
  if (tid == 0 && a.rstd != nullptr) a.rstd[row] = r;
  i8::RowScale s;
  if (Q) {
    bits = __float_as_uint(__uint_as_float(bits) * r) & 0x7FFFFFFFu;
    s = i8::row_scale<false>(bits);
    if (tid == 0) a.scale[row] = i8::scale_of_row(bits);
  }
  for (int c0 = tid; c0 < (LONG ? pieces : tid + 1); c0 += P * tpr) {
    if (LONG) take(c0, false);
    float f[EP];
#pragma unroll
    for (int i = 0; i < P; ++i) {
#pragma unroll
      for (int j = 0; j < VE; ++j) f[i * VE + j] = h[i][j] * w[i][j] * r;
    }
    if (!Q || a.y != nullptr) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int c = c0 + i * tpr;
        Piece<T, VE> o;
#pragma unroll
        for (int j = 0; j < VE; ++j) o.set(j, f[i * VE + j]);
        if (c < pieces) o.store(static_cast<T*>(a.y) + row * a.H + static_cast<long long>(c) * VE);
      }
    }
    if constexpr (Q) {
      uint32_t b[EP / 4];
      i8::quantize_values<false>(s, f, b);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int c = c0 + i * tpr;
        if (c < pieces) store_bytes<VE>(a.q + row * a.q_ld + static_cast<long long>(c) * VE, b, i);
      }
    }
  }
  if (Q) {  // columns up to the next multiple of 16 are zeros
    for (int c = a.H + tid; c < (a.H + 15) / 16 * 16; c += tpr) a.q[row * a.q_ld + c] = 0;
  }
}

template <class T, class W, int VE, int EP, bool Q, bool LONG>
static cudaError_t launch_forward(const Forward& a, int log2, cudaStream_t st) {
  const int threads = log2 > 8 ? 1 << log2 : 256;
  const long long per = threads >> log2, blocks = (a.rows + per - 1) / per;
  return launch_chained(forward_kernel<T, W, VE, EP, Q, LONG>, dim3(static_cast<unsigned>(blocks)), threads, 0, st, 1, a, log2);
}
template <class T, class W, int VE, bool Q>
static cudaError_t launch_forward(const Forward& a, cudaStream_t st) {
  if (a.H <= 16 * kThreads) return launch_forward<T, W, VE, 16, Q, false>(a, row_threads_log2(a.H, 16), st);
  return launch_forward<T, W, VE, 16, Q, true>(a, 9, st);
}

}  // namespace norm
}  // namespace smoe

using namespace smoe;
using namespace smoe::norm;

extern "C" int smoe_rms_norm(const void* x, long long ld, const void* residual, long long residual_ld, const void* weight,
                             int weight_dtype, void* y, void* h, float* rstd, void* q, long long q_ld, float* scale, int dtype,
                             long long rows, int H, float eps, void* stream) {
  const int size = type_bytes(dtype), wsize = type_bytes(weight_dtype);
  if (size == 0 || wsize == 0 || (weight_dtype != dtype && weight_dtype != SMOE_F32)) return SMOE_ERR_DTYPE;
  if (rows < 0 || rows > 0x7fffffffll || H <= 0 || H > kMaxWidth || ld < 0 || residual_ld < 0 || !(eps >= 0.f)) return SMOE_ERR_SHAPE;
  if (q != nullptr && (H > i8::kMaxCols || q_ld < (H + 15) / 16 * 16)) return SMOE_ERR_SHAPE;
  if (rows == 0) return SMOE_OK;
  if (x == nullptr || weight == nullptr || (y == nullptr && q == nullptr) || (q == nullptr) != (scale == nullptr)) return SMOE_ERR_SHAPE;
  if (h != nullptr && residual == nullptr) return SMOE_ERR_SHAPE;
  if ((address(x) | address(residual) | address(y) | address(h)) % size != 0 || address(weight) % wsize != 0 ||
      (address(rstd) | address(scale)) % 4 != 0 || address(q) % 16 != 0 || (q != nullptr && q_ld % 16 != 0))
    return SMOE_ERR_ALIGNMENT;
  Forward a = {};
  a.x = x; a.x_ld = ld; a.res = residual; a.res_ld = residual != nullptr ? residual_ld : 0;
  a.w = weight; a.w_wide = address(weight) % 16 == 0;
  a.y = y; a.h = h; a.rstd = rstd; a.q = static_cast<int8_t*>(q); a.q_ld = q_ld; a.scale = scale;
  a.rows = rows; a.H = H; a.eps = eps;
  const int bytes = access_bytes({address(x) | address(residual) | address(y) | address(h), ld * size, a.res_ld * size,
                                  static_cast<long long>(H) * size});
  return for_types(dtype, weight_dtype, [&](auto t, auto v) {
    using T = decltype(t);
    using W = decltype(v);
    return launched(for_access<T>(bytes, [&](auto ve) {
      return q != nullptr ? launch_forward<T, W, ve, true>(a, S(stream)) : launch_forward<T, W, ve, false>(a, S(stream));
    }));
  });
}
