// Root-mean-square norm, forward (the formulas are in norm.cuh).
#include "norm.cuh"

namespace smoe {
namespace norm {

struct Forward {
  const void* x; long long x_ld;            // values from row to row
  const void* res; long long res_ld;        // or nullptr
  const void* w; int w_wide;                // starts on a 16-byte boundary
  void* y;                                  // packed rows, or nullptr
  void* h;                                  // packed rows, or nullptr
  float* rstd;                              // (rows), or nullptr
  int8_t* q; long long q_ld; float* scale;  // or nullptr
  long long rows;
  int H;
  float eps, per_value;                     // 1 / H
};

template <class T, class W, int EP, bool ALIGNED, bool MASKED>
__device__ __forceinline__ void take_weights(const Forward& a, const Columns<T, ALIGNED>& columns, int c0, int step, Values<W, EP, kValues<T>>& w) {
  if (ALIGNED && a.w_wide) w.template load<true, false>(static_cast<const W*>(a.w), columns, c0, step);
  else w.template load<false, false>(static_cast<const W*>(a.w), columns, c0, step);
  if (MASKED) w.template mask<ALIGNED>(columns, c0, step);
}
// h, on its way out the first time
template <class T, int EP, bool ALIGNED>
__device__ __forceinline__ void take_rows(const Forward& a, long long row, const Columns<T, ALIGNED>& columns, int c0, int step, bool keep, Values<T, EP, kValues<T>>& h) {
  h.template load<ALIGNED, true>(static_cast<const T*>(a.x) + row * a.x_ld, columns, c0, step);
  if (a.res == nullptr) {
    h.template mask<ALIGNED>(columns, c0, step);
    return;
  }
  Values<T, EP, kValues<T>> r;
  r.template load<ALIGNED, true>(static_cast<const T*>(a.res) + row * a.res_ld, columns, c0, step);
#pragma unroll
  for (int k = 0; k < EP / 2; ++k) h.add(k, r);
  h.template mask<ALIGNED>(columns, c0, step);
  if (keep && a.h != nullptr) h.template store<ALIGNED>(static_cast<T*>(a.h) + row * a.H, columns, c0, step);
}

template <class T, class W, int EP, bool Q>
__device__ __forceinline__ void measure(const Values<T, EP, kValues<T>>& h, const Values<W, EP, kValues<T>>& w, F2& sum, float& most) {
#pragma unroll
  for (int k = 0; k < EP / 2; ++k) {
    const F2 f = h.get(k);
    sum = fma2(f, f, sum);
    if (Q) {
      float x, y;
      (f * w.get(k)).split(x, y);
      most = max_abs(most, x, y);
    }
  }
}

// 8-bit values of fp32 rows are rounded exactly, as quantize_rows rounds them.  Those of 16-bit rows: y, off by some units itself, times 127 /
// max |y| in one fused multiply-add: within 127 * 2^-23 = 1.6e-5 of a step of the half to even of that product (8192 x 4096 with a residual, all of
// the kernel: rounded exactly 55 us, so 45).
template <bool EXACT>
__device__ __forceinline__ void quantise(const i8::RowScale& s, float (&f)[8], uint32_t (&b)[2]) {
  if constexpr (EXACT) {
    i8::quantize_values<false>(s, f, b);
  } else {
    if (s.pre != 1.f) {
#pragma unroll
      for (auto& x : f) x *= s.pre;
    }
    int q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = __float_as_int(fmaf(f[i], s.inv, i8::kRoundMagic));
#pragma unroll
    for (int j = 0; j < 2; ++j)
      b[j] = s.keep & __byte_perm(__byte_perm(q[4 * j], q[4 * j + 1], 0x0040), __byte_perm(q[4 * j + 2], q[4 * j + 3], 0x0040), 0x5410);
  }
}

// What follows the sum of a row's squares and the largest |h w|: r, y = (h w) r, the 8-bit values, the row's scale.  The maximum of |h w|
// times r is that of |y|, whatever is rounded on the way, so that one reduction serves both.
template <class T, class W, int EP, bool ALIGNED, bool Q>
struct Finish {
  static constexpr int VE = kValues<T>;
  float r;
  i8::RowScale s;
  __device__ __forceinline__ Finish(const Forward& a, long long row, float sum, float most, bool writes) {
    r = inverse_root(fmaf(sum, a.per_value, a.eps));
    if (writes && a.rstd != nullptr) a.rstd[row] = r;
    if (Q) {
      const uint32_t bits = __float_as_uint(most * r) & 0x7FFFFFFFu;
      s = i8::row_scale<false>(bits);
      if (writes) a.scale[row] = i8::scale_of_row(bits);
    }
  }
  __device__ __forceinline__ void put(const Forward& a, long long row, const Columns<T, ALIGNED>& columns, int c0, int step,
                                      const Values<T, EP, VE>& h, const Values<W, EP, VE>& w) const {
    if (Q && a.y == nullptr) return;
    const F2 rr(r, r);
    Values<T, EP, VE> y;
#pragma unroll
    for (int k = 0; k < EP / 2; ++k) y.set(k, h.get(k) * w.get(k) * rr);
    y.template store<ALIGNED>(static_cast<T*>(a.y) + row * a.H, columns, c0, step);
  }
  // the 8-bit values, in the order of h's
  __device__ __forceinline__ void quantised(const Values<T, EP, VE>& h, const Values<W, EP, VE>& w, uint32_t (&b)[EP / 4]) const {
    const F2 rr(r, r);
#pragma unroll
    for (int g = 0; g < EP; g += 8) {
      float f[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) (h.get(g / 2 + k) * w.get(g / 2 + k) * rr).split(f[2 * k], f[2 * k + 1]);
      uint32_t two[2];
      quantise<(sizeof(T) == 4)>(s, f, two);
      b[g / 4] = two[0];
      b[g / 4 + 1] = two[1];
    }
  }
};

// A row is read once and stays in registers, EP values in each of its threads.  Bound by memory: bf16 rows of 4096 with a residual 6.8 TB/s at 32768 (158 us,
// 165 as 8-bit rows), 6.4 at 8192 (42; 45 as 8-bit rows), 262144 x 128 5.6 (24); fp32 4099 x 1005 9.5 us, fp16 5003 x 1030 to 8 bits 13 (rows that start
// anywhere); one row of 4096 1.8 us, as 8-bit rows 2.1: latency.
template <class T, class W, int EP, bool ALIGNED, bool Q>
__global__ void __launch_bounds__(kThreads, EP <= 16 ? 2 : 1) forward_kernel(const Forward a, int tpr) {
  release_next();
  wait_for_previous();
  __shared__ Parts part;
  const Share at(tpr);
  const long long row = static_cast<long long>(blockIdx.x) * at.subs + at.sub;
  const bool live = row < a.rows;
  Columns<T, ALIGNED> columns(row, a.H);
  if (!live) columns.pieces = 0;
  Values<T, EP, kValues<T>> h;
  Values<W, EP, kValues<T>> w;
  take_rows<T, EP, ALIGNED>(a, row, columns, at.tid, tpr, true, h);
  take_weights<T, W, EP, ALIGNED, Q>(a, columns, at.tid, tpr, w);
  F2 sums(0.f, 0.f);
  float most = 0.f;
  measure<T, W, EP, Q>(h, w, sums, most);
  float sum = sums.sum();
  row_reduce<Q>(sum, most, at, part);
  h.forget();
  w.forget();
  const Finish<T, W, EP, ALIGNED, Q> finish(a, row, sum, most, live && at.tid == 0);
  finish.put(a, row, columns, at.tid, tpr, h, w);
  if constexpr (Q) {
    // A row of 8-bit values starts on a 16-byte boundary.  Where the pieces do not, the end of a piece and the beginning of the next one
    // make a store; what follows the row are zeros, and so are its columns up to the next multiple of 16.
    constexpr int VE = kValues<T>, P = EP / VE;
    using Bytes = typename std::conditional<VE == 8, uint64_t, uint32_t>::type;
    uint32_t b[EP / 4];
    finish.quantised(h, w, b);
    Bytes v[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if constexpr (VE == 8) v[i] = b[2 * i] | static_cast<uint64_t>(b[2 * i + 1]) << 32;
      else v[i] = b[i];
    }
    if constexpr (!ALIGNED) {
      __shared__ Bytes bytes[EP / VE * kThreads];
#pragma unroll
      for (int i = 0; i < P; ++i) bytes[i * blockDim.x + threadIdx.x] = v[i];
      __syncthreads();
      if (columns.shift > 0) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const bool last = at.tid == tpr - 1;
          const Bytes next = !last ? bytes[i * blockDim.x + threadIdx.x + 1] : i + 1 < P ? bytes[(i + 1) * blockDim.x + threadIdx.x - at.tid] : 0;
          v[i] = (v[i] >> (8 * columns.shift)) | (next << (8 * (VE - columns.shift)));
        }
      }
    }
    const int end = live ? (a.H + 15) / 16 * 16 : 0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = at.tid + i * tpr;
      if (VE * c < end) *reinterpret_cast<Bytes*>(a.q + row * a.q_ld + VE * c) = v[i];
    }
    for (int c = at.tid + P * tpr; VE * c < end; c += tpr) *reinterpret_cast<Bytes*>(a.q + row * a.q_ld + VE * c) = 0;
  }
}

// Rows that a block's threads do not hold: read twice, EP values of each thread at a time, a row to a block.
template <class T, class W, int EP, bool ALIGNED, bool Q>
__global__ void __launch_bounds__(kThreads) forward_long_kernel(const Forward a) {
  release_next();
  wait_for_previous();
  __shared__ Parts part;
  const Share at(kThreads);
  const long long row = blockIdx.x;
  const Columns<T, ALIGNED> columns(row, a.H);
  const int round = EP / kValues<T> * kThreads;
  Values<T, EP, kValues<T>> h;
  Values<W, EP, kValues<T>> w;
  F2 sums(0.f, 0.f);
  float most = 0.f;
  for (int c = 0; c < columns.pieces; c += round) {
    take_rows<T, EP, ALIGNED>(a, row, columns, c + at.tid, kThreads, true, h);
    take_weights<T, W, EP, ALIGNED, Q>(a, columns, c + at.tid, kThreads, w);
    measure<T, W, EP, Q>(h, w, sums, most);
  }
  float sum = sums.sum();
  row_reduce<Q>(sum, most, at, part);
  const Finish<T, W, EP, ALIGNED, Q> finish(a, row, sum, most, at.tid == 0);
  for (int c = 0; c < columns.pieces; c += round) {
    take_rows<T, EP, ALIGNED>(a, row, columns, c + at.tid, kThreads, false, h);
    take_weights<T, W, EP, ALIGNED, Q>(a, columns, c + at.tid, kThreads, w);
    finish.put(a, row, columns, c + at.tid, kThreads, h, w);
    if constexpr (Q) {
      uint32_t b[EP / 4];
      finish.quantised(h, w, b);
#pragma unroll
      for (int i = 0; i < EP; ++i) {
        const int col = columns.first(c + at.tid + i / kValues<T> * kThreads) + i % kValues<T>;
        if (col >= 0 && col < (a.H + 15) / 16 * 16) a.q[row * a.q_ld + col] = static_cast<int8_t>(b[i / 4] >> (8 * (i % 4)));
      }
    }
  }
  if constexpr (Q) {  // zeros up to the next multiple of 16 columns where the rounds' pieces, `shift` columns ahead of them, end before it
    const int covered = columns.first((columns.pieces + round - 1) / round * round);
    if (covered + at.tid < (a.H + 15) / 16 * 16) a.q[row * a.q_ld + covered + at.tid] = 0;
  }
}

template <class T, class W, int EP, bool ALIGNED, bool Q>
static cudaError_t launch_rows(const Forward& a, const Shape& s, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>((a.rows + s.subs - 1) / s.subs));
  return launch_chained(forward_kernel<T, W, EP, ALIGNED, Q>, grid, s.threads, 0, st, 1, a, s.tpr);
}
// Values of a thread.  Whole pieces: 16 with a residual, 32 without one, so that as many loads are on their way (bf16, us: 16384 x 5000 66.5 / 50.1,
// 100000 x 256 18.2 / 17.5; with a residual 32768 x 4096 157.9 / 158.8, as 8-bit rows 163 / 174).  Other rows: whichever of 16, 24 and 32 leaves
// the fewest threads idle (100000 x 257 57.9 / 39.6 / 48.4, 20000 x 2049 with a residual 65.5 / 60.4 / 71.2); of two that leave as many, the
// smaller up to 256 threads a row (5003 x 1030 10.0 / 11.0), the larger above (16384 x 7169 192 / 161).
template <class T, class W, bool ALIGNED, bool Q>
static cudaError_t launch_forward(const Forward& a, cudaStream_t st) {
  const long long values = a.H + (ALIGNED ? 0 : kValues<T> - 1);
  if (values > 32 * kThreads)
    return launch_chained(forward_long_kernel<T, W, 16, ALIGNED, Q>, dim3(static_cast<unsigned>(a.rows)), kThreads, 0, st, 1, a);
  const Shape s16 = shape_of(values, 16), s32 = shape_of(values, 32);
  if constexpr (ALIGNED) {
    if (values <= 16 * kThreads && (a.res != nullptr || values < 64)) return launch_rows<T, W, 16, ALIGNED, Q>(a, s16, st);
    return launch_rows<T, W, 32, ALIGNED, Q>(a, s32, st);
  } else {
    const Shape s24 = shape_of(values, 24);
    const int w16 = 16 * s16.tpr, w24 = 24 * s24.tpr, w32 = 32 * s32.tpr;
    const bool wide = s16.tpr > 256;
    if (s16.tpr <= kThreads && (wide ? w16 < w24 && w16 < w32 : w16 <= w24 && w16 <= w32)) return launch_rows<T, W, 16, ALIGNED, Q>(a, s16, st);
    if (s24.tpr <= kThreads && (wide ? w24 < w32 : w24 <= w32)) return launch_rows<T, W, 24, ALIGNED, Q>(a, s24, st);
    return launch_rows<T, W, 32, ALIGNED, Q>(a, s32, st);
  }
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
  if ((address(x) | address(residual)) % size != 0 || address(weight) % wsize != 0 || (address(y) | address(h) | address(q)) % 16 != 0 ||
      (address(rstd) | address(scale)) % 4 != 0 || (q != nullptr && q_ld % 16 != 0))
    return SMOE_ERR_ALIGNMENT;
  Forward a = {};
  a.x = x; a.x_ld = ld; a.res = residual; a.res_ld = residual != nullptr ? residual_ld : 0;
  a.w = weight; a.w_wide = address(weight) % 16 == 0;
  a.y = y; a.h = h; a.rstd = rstd; a.q = static_cast<int8_t*>(q); a.q_ld = q_ld; a.scale = scale;
  a.rows = rows; a.H = H; a.eps = eps; a.per_value = 1.f / static_cast<float>(H);
  const bool aligned = (address(x) | address(residual) | ld * size | a.res_ld * size | static_cast<long long>(H) * size) % 16 == 0;
  return for_types(dtype, weight_dtype, [&](auto t, auto v) {
    using T = decltype(t);
    using W = decltype(v);
    if (q != nullptr) return launched(aligned ? launch_forward<T, W, true, true>(a, S(stream)) : launch_forward<T, W, false, true>(a, S(stream)));
    return launched(aligned ? launch_forward<T, W, true, false>(a, S(stream)) : launch_forward<T, W, false, false>(a, S(stream)));
  });
}
