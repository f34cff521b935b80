// Products of 8-bit integers with one scale per row and one per output channel:
//   y[r, n] = act( (sum_k xq[s(r), k] wq[e(r), n, k]) x_scale[s(r)] w_scale[e(r), n] + bias[e(r), n] )
// What the kernels share: the argument block, which rows there are, and the arithmetic behind the sum.
//
// The sum is exact in 32-bit integers (at most 131071 products of at most 2^14), so it does not matter how a kernel orders or
// splits it: all of them give the same bits.  It is rounded to fp32 once (2^-24), multiplied by the two scales, the bias is
// added, and the result is rounded to the output's type.
#pragma once
#include <cuda_fp16.h>

#include "epilogue.cuh"
#include "launch.cuh"

namespace smoe {
namespace i8 {

constexpr int kMaxCols = 131071;     // 131071 * 128 * 128 < 2^31
constexpr int kMaxRows = 0x7fff0000; // rows of x and of the output: a tile's last row number fits into 32 bits
constexpr int kMaxExpertRows = 1024; // experts whose offsets the kernels keep in shared memory
constexpr int kNoActivation = -1;

struct Params {
  int E, N, K;           // experts, output channels, columns of x
  int rows;              // rows of the output
  int x_rows;            // rows of x
  const int* off;        // (E + 1) first row of each expert, or nullptr: one expert has all rows
  const int* count;      // (E) rows of each expert, or nullptr: up to the next expert's first
  const int* gather;     // (rows) row of x, or nullptr: the same row; out of range: a row of zeros
  const float* x_scale;  // (x_rows)
  const float* w_scale;  // (E, N)
  const void* bias;      // (E, N) or nullptr
  int bias_type;
  void* out;             // (rows, N), or (rows, N / 2) with a gated activation
  int out_type;
  int activation;        // kNoActivation or smoe::Activation
  int wide_out;          // rows of the output start on 16-byte boundaries
  int* status;
};

__device__ __forceinline__ int first_row(const Params& p, int e) { return p.off != nullptr ? min(max(p.off[e], 0), p.rows) : 0; }
// The row behind the expert's last one.  Offsets that overlap or run past the output are cut, so that no load reaches past it.
__device__ __forceinline__ int end_row(const Params& p, int e) {
  if (p.off == nullptr) return p.rows;
  const int next = min(max(p.off[e + 1], 0), p.rows);
  return p.count != nullptr ? min(next, p.off[e] + max(p.count[e], 0)) : next;
}

// Row of x that output row r takes, or -1.
__device__ __forceinline__ int source_row(const Params& p, int r) {
  const int s = p.gather != nullptr ? p.gather[r] : r;
  return static_cast<unsigned>(s) < static_cast<unsigned>(p.x_rows) ? s : -1;
}

__device__ __forceinline__ float load_typed(const void* v, int dtype, long long i) {
  if (dtype == SMOE_F32) return static_cast<const float*>(v)[i];
  if (dtype == SMOE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(v)[i]);
  return __half2float(static_cast<const __half*>(v)[i]);
}
__device__ __forceinline__ void store_typed(void* v, int dtype, long long i, float f) {
  if (dtype == SMOE_F32) static_cast<float*>(v)[i] = f;
  else if (dtype == SMOE_BF16) static_cast<__nv_bfloat16*>(v)[i] = __float2bfloat16_rn(f);
  else static_cast<__half*>(v)[i] = __float2half_rn(f);
}
__device__ __forceinline__ uint32_t pack_typed(int dtype, float lo, float hi) {
  if (dtype == SMOE_BF16) return pack_bf16(lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// (sum x_scale) w_scale, and + bias, each step rounded by itself: a compiler that fused the last two in one kernel and not in another
// would give other bits.
__device__ __forceinline__ float scaled(int acc, float xs, float ws) { return __fmul_rn(__fmul_rn(__int2float_rn(acc), xs), ws); }
__device__ __forceinline__ float biased(float y, float bias) { return __fadd_rn(y, bias); }

// The activations' values by their definitions.  x sigmoid(x) = x / (1 + exp(-x)) with the fast exponential, off by up to 2 + 1.2 |x|
// units in the last place of its value, and division, 2 units: within (5 + 1.2 |x|) 2^-23 of the value, 2^-20 at x = -2 and 2^-17 at -60;
// below -87, where the value is under 1.5e-36, the division gives zero.  (The hardware tanh that the bf16 epilogues use is off by 2.5e-4
// of x, too much of a small result.)
__device__ __forceinline__ float silu(float x) { return __fdividef(x, 1.f + __expf(-x)); }
template <int ACT>
__device__ __forceinline__ float activate(float x) {
  if constexpr (ACT == ACT_SWIGLU || ACT == ACT_SILU) return silu(x);
  else if constexpr (ACT == ACT_GEGLU || ACT == ACT_GELU) return 0.5f * x * erfcf(x * -0.70710678118654752f);
  else if constexpr (ACT == ACT_RELU_SQ) return x < 0.f ? 0.f : x * x;
  else if constexpr (ACT == ACT_REGLU || ACT == ACT_RELU) return x < 0.f ? 0.f : x;  // NaN stays NaN
  else return x;
}
__host__ __device__ constexpr bool is_gated(int act) { return act >= 0 && act_is_gated(act); }

// Rows that no expert has (between an expert's rows and the next one's, behind the last) become zeros.  Warp `warp` of `warps`,
// all its lanes; a row's expert is found by bisection.
__device__ __forceinline__ void zero_other_rows(const Params& p, int warp, int warps) {
  if (p.off == nullptr) return;
  const int lane = threadIdx.x & 31;
  const int cols = is_gated(p.activation) ? p.N / 2 : p.N;
  const long long bytes = static_cast<long long>(cols) * (p.out_type == SMOE_F32 ? 4 : 2);
  for (long long base = 32ll * warp; base < p.rows; base += 32ll * warps) {
    const int r = static_cast<int>(base) + lane;
    bool other = false;
    if (base + lane < p.rows) {
      int lo = 0, hi = p.E;  // the last expert whose first row is not behind r
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.off[mid] <= r) lo = mid; else hi = mid;
      }
      other = r < first_row(p, lo) || r >= end_row(p, lo);
    }
    for (unsigned todo = __ballot_sync(0xffffffffu, other); todo != 0u; todo &= todo - 1u) {
      char* dst = static_cast<char*>(p.out) + (base + __ffs(todo) - 1) * bytes;
      if (p.wide_out) {
        for (long long c = 16 * lane; c < bytes; c += 512) *reinterpret_cast<uint4*>(dst + c) = make_uint4(0u, 0u, 0u, 0u);
      } else {
        for (long long c = 2 * lane; c < bytes; c += 64) *reinterpret_cast<uint16_t*>(dst + c) = 0;
      }
    }
  }
}

// ----------------------------------------------------------------------------------------------
// quantisation of a row: scale = amax / 127 (1 for a row of zeros), q = 127 x / amax rounded half to even
// ----------------------------------------------------------------------------------------------
// 16-bit values (at most 11 bits).  With significands mx, ma as whole numbers the quotient is 127 mx 2^s / ma, and it lies on a border
// k + 1/2 where 254 mx 2^s = (2k + 1) ma.  Both sides are multiples of min(1, 2^s): a quotient off a border is off by at least 1 / (254
// * 2047) > 2^-19 of its value.  127 divides the left side, so on a border it divides 2k + 1 (which is 127 then, the border 63.5) or ma.
// Multiplied by 127 / amax made larger by 2^-21, values off a border stay on their side and 63.5 goes to 64, which is even: one
// multiply-add rounds right, in every row whose ma is no multiple of 127.  In those that are, the quotient by a reciprocal is corrected
// once by its remainder, which fp32 holds exactly, and so is exact on every border.  (That arithmetic for all rows: 8192 x 4096 bf16 23
// us; a search for borders with remainders behind it 27, with 64-bit divisions 59.)
// fp32 values: one fused multiply-add is within 127 * 2^-24 + 2^-15 = 3.8e-5 of the quotient, as a fixed-point number with 14 fractional
// bits; where that is within a step of a border k + 1/2 (seldom), the remainder 127 x - q amax decides, its products held as sums
// of two.
// Rows whose largest value is below 2^-120 or above 2^120 are multiplied by a power of two first, so that neither 127 / amax nor
// 127 x leaves fp32's range.  Rows that hold an infinity or a NaN get it as their scale, and zeros: every product of theirs is NaN.
struct RowScale {
  float pre;       // power of two for the values
  float amax;      // times pre
  float inv;       // 127 / amax, for 16-bit values times 1 + 2^-21; 0: none
  bool borders;    // 16-bit values: other borders than 63.5
  uint32_t keep;   // 0: zeros
};
// bits: the largest |x| as an integer (a NaN's are above infinity's)
__device__ __forceinline__ float scale_of_row(uint32_t bits) {
  const float amax = __uint_as_float(bits);
  return bits == 0u ? 1.f : bits < 0x7F800000u ? __fdiv_rn(amax, 127.f) : amax;
}
template <bool SHORT>
__device__ __forceinline__ RowScale row_scale(uint32_t bits) {
  RowScale s;
  const bool some = bits != 0u && bits < 0x7F800000u;
  s.pre = !some ? 1.f : bits < (7u << 23) ? 18446744073709551616.f : bits >= (247u << 23) ? 1.f / 18446744073709551616.f : 1.f;  // 2^64
  s.amax = __uint_as_float(bits) * s.pre;
  s.inv = some ? __fdiv_rn(127.f, s.amax) : 0.f;
  if (SHORT) s.inv *= 1.f + 1.f / 2097152.f;
  s.borders = SHORT && some && ((__float_as_uint(s.amax) & 0x7FFFFFu) | 0x800000u) % 127u == 0u;
  s.keep = some ? 0xFFFFFFFFu : 0u;
  return s;
}

constexpr float kRoundMagic = 12582912.f;  // 1.5 * 2^23: adding it leaves the whole number in the low bits
// Adding it leaves t + 1/2 + 2^-14 as a fixed-point number in the low 22 bits of the sum, 14 of them behind the point: bits 14 to
// 21 are t rounded, and the low 14 are at most 2 where t is within a step of a border.
constexpr float kFixedMagic = 768.f + 0.5f + 1.f / 16384.f;

// N values -> N bytes, four per word of w.
template <bool SHORT, int N>
__device__ __forceinline__ void quantize_values(const RowScale& s, float (&f)[N], uint32_t (&w)[N / 4]) {
  static_assert(N % 4 == 0, "whole words");
  if (s.pre != 1.f) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] *= s.pre;
  }
  int q[N];
  if constexpr (SHORT) {
    if (s.borders) {
      const float r = __fdiv_rn(1.f, s.amax);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float x = 127.f * f[i], t = x * r;
        q[i] = __float_as_int(fmaf(fmaf(-t, s.amax, x), r, t) + kRoundMagic);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) q[i] = __float_as_int(fmaf(f[i], s.inv, kRoundMagic));
    }
  } else {
    uint32_t near = 0x3FFFu;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      q[i] = __float_as_int(fmaf(f[i], s.inv, kFixedMagic));
      near = min(near, static_cast<uint32_t>(q[i]) & 0x3FFFu);
      q[i] >>= 14;
    }
    if (near <= 2u) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float whole = static_cast<float>(static_cast<int8_t>(q[i]));
        const float x = 127.f * f[i], x_low = fmaf(127.f, f[i], -x);
        const float p = whole * s.amax, p_low = fmaf(whole, s.amax, -p);
        const float rest = x - p;  // exact: the two are within a factor of two of one another, or p is zero
        const float over = (2.f * fabsf(rest) - s.amax) + 2.f * (rest >= 0.f ? x_low - p_low : p_low - x_low);
        if (over > 0.f || (over == 0.f && (q[i] & 1))) q[i] += rest > 0.f ? 1 : -1;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < N / 4; ++j)
    w[j] = s.keep & __byte_perm(__byte_perm(q[4 * j], q[4 * j + 1], 0x0040), __byte_perm(q[4 * j + 2], q[4 * j + 3], 0x0040), 0x5410);
}

// gemm_int8.cu
int tensor_core_product(const int8_t* xq, long long ld, const int8_t* wq, long long w_ld, const Params& p, cudaStream_t st);

}  // namespace i8
}  // namespace smoe
