// Root-mean-square norm, gradients (the formulas are in norm.cuh).
#include "norm.cuh"

namespace smoe {
namespace norm {

struct Backward {
  const void* dy; long long dy_ld;  // values from row to row
  const void* dh; long long dh_ld;  // or nullptr
  const void* h; long long h_ld;
  const void* w; int w_wide;        // weights of the columns start on 16-byte boundaries
  const float* rstd;
  void* dx;                         // packed rows, or nullptr
  float* partial;                   // (blocks, H): each block's part of the weight's gradient, or nullptr
  long long rows;
  int H;
};

constexpr int kMostBlocks = 4 * 148;  // four to each of a B200's SMs

// Blocks take rows in turn and keep their part of the weight's gradient in registers, EP columns in each thread, until the end.  A row is
// read once.  Bound by memory.  LONG: rows that a block's threads do not hold are read twice, and the part lies in the block's row of
// `partial`, where the same thread adds to the same columns each time.
template <class T, class W, int VE, int EP, bool LONG>
__global__ void __launch_bounds__(kThreads) backward_kernel(const Backward a, int log2) {
  release_next();
  wait_for_previous();
  constexpr int P = EP / VE;
  __shared__ float part[2][kThreads / 32];
  extern __shared__ float sums[];
  const int tpr = 1 << log2, sub = threadIdx.x >> log2, tid = threadIdx.x & (tpr - 1), subs = blockDim.x >> log2;
  const float per_value = 1.f / static_cast<float>(a.H);
  const int all = a.H / VE;
  const W* weight = static_cast<const W*>(a.w);
  float* mine = a.partial + static_cast<long long>(blockIdx.x) * a.H;
  Piece<W, VE> w[P];
  Piece<T, VE> dy[P], h[P], dh[P];
  float acc[EP];
#pragma unroll
  for (int i = 0; i < EP; ++i) acc[i] = 0.f;
  const auto take_weights = [&](int c0) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = c0 + i * tpr;
      if (c < all) w[i].load_shared(weight + static_cast<long long>(c) * VE, a.w_wide); else w[i].zero();
    }
  };
  const auto take = [&](long long row, int c0) {
    const bool live = row < a.rows;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const long long c = c0 + i * tpr;
      if (live && c < all) {
        dy[i].load(static_cast<const T*>(a.dy) + row * a.dy_ld + c * VE);
        h[i].load(static_cast<const T*>(a.h) + row * a.h_ld + c * VE);
        if (a.dh != nullptr) dh[i].load(static_cast<const T*>(a.dh) + row * a.dh_ld + c * VE);
      } else {
        dy[i].zero();
        h[i].zero();
      }
    }
  };
  if (!LONG) take_weights(tid);
  int turn = 0;
  for (long long base = static_cast<long long>(blockIdx.x) * subs; base < a.rows; base += static_cast<long long>(gridDim.x) * subs) {
    const long long row = base + sub;
    const bool live = row < a.rows;
    const float r = live ? a.rstd[row] : 0.f;
    float sum = 0.f;
    for (int c0 = tid; c0 < (LONG ? all : tid + 1); c0 += P * tpr) {
      take(row, c0);
      if (LONG) take_weights(c0);
#pragma unroll
      for (int i = 0; i < P; ++i) {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float t = dy[i][j] * (h[i][j] * r);
          sum = fmaf(t, w[i][j], sum);
          if (!LONG) {
            acc[i * VE + j] += t;
          } else if (a.partial != nullptr && c0 + i * tpr < all) {
            float* d = mine + static_cast<long long>(c0 + i * tpr) * VE + j;
            *d = base == blockIdx.x ? t : *d + t;  // (LONG: a block has a row at a time)
          }
        }
      }
    }
    if (a.dx == nullptr) continue;
    uint32_t none = 0u;
    row_reduce<false>(sum, none, log2, part[turn], nullptr);
    turn ^= 1;  // the next row's sums lie elsewhere: one barrier a row is enough
    const float mean = sum * per_value;
    for (int c0 = tid; c0 < (LONG ? all : tid + 1); c0 += P * tpr) {
      if (LONG) {
        take(row, c0);
        take_weights(c0);
      }
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const long long c = c0 + i * tpr;
        Piece<T, VE> o;
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float g = r * (dy[i][j] * w[i][j] - (h[i][j] * r) * mean);
          o.set(j, a.dh != nullptr ? dh[i][j] + g : g);
        }
        if (live && c < all) o.store(static_cast<T*>(a.dx) + row * a.H + c * VE);
      }
    }
  }
  if (a.partial == nullptr || LONG) return;
  float* to = subs == 1 ? mine : sums + sub * a.H;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = tid + i * tpr;
    if (c < all) {
#pragma unroll
      for (int j = 0; j < VE; ++j) to[c * VE + j] = acc[i * VE + j];
    }
  }
  if (subs == 1) return;
  __syncthreads();
  for (int c = threadIdx.x; c < a.H; c += blockDim.x) {
    float s = 0.f;
    for (int k = 0; k < subs; ++k) s += sums[k * a.H + c];
    mine[c] = s;
  }
}

// dw[c] = sum over the blocks' parts, in the same order every time.
constexpr int kShares = 32;
__global__ void __launch_bounds__(32 * kShares) weight_grad_kernel(const float* partial, int blocks, int H, void* dw, int type) {
  release_next();
  wait_for_previous();
  __shared__ float sums[kShares][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long c = blockIdx.x * 32ll + lane;
  float s = 0.f;
  if (c < H) {
#pragma unroll 4
    for (int b = warp; b < blocks; b += kShares) s += partial[static_cast<long long>(b) * H + c];
  }
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < H) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < kShares; ++k) s += sums[k][lane];
    i8::store_typed(dw, type, c, s);
  }
}

template <class T, class W, int VE, int EP, bool LONG>
static cudaError_t launch_backward(const Backward& a, int log2, int& blocks, cudaStream_t st) {
  const int threads = log2 > 8 ? 1 << log2 : 256, subs = threads >> log2;
  const long long need = (a.rows + subs - 1) / subs;
  blocks = static_cast<int>(need < kMostBlocks ? need : kMostBlocks);
  const size_t smem = subs > 1 ? static_cast<size_t>(subs) * a.H * sizeof(float) : 0;  // subs H <= 256 EP
  return launch_chained(backward_kernel<T, W, VE, EP, LONG>, dim3(static_cast<unsigned>(blocks)), threads, smem, st, 1, a, log2);
}
template <class T, class W, int VE>
static cudaError_t launch_backward(const Backward& a, int& blocks, cudaStream_t st) {
  if (a.H <= 16 * kThreads) return launch_backward<T, W, VE, 16, false>(a, row_threads_log2(a.H, 16), blocks, st);
  return launch_backward<T, W, VE, 16, true>(a, 9, blocks, st);
}

}  // namespace norm
}  // namespace smoe

using namespace smoe;
using namespace smoe::norm;

extern "C" {

size_t smoe_rms_norm_backward_workspace_bytes(long long rows, int H) {
  if (rows <= 0 || H <= 0) return 0;
  return static_cast<size_t>(rows < kMostBlocks ? rows : kMostBlocks) * static_cast<size_t>(H) * sizeof(float);
}

int smoe_rms_norm_backward(const void* dy, long long dy_ld, const void* dh, long long dh_ld, const void* h, long long h_ld,
                           const void* weight, int weight_dtype, const float* rstd, void* dx, void* dweight, int dtype,
                           long long rows, int H, void* workspace, void* stream) {
  const int size = type_bytes(dtype), wsize = type_bytes(weight_dtype);
  if (size == 0 || wsize == 0 || (weight_dtype != dtype && weight_dtype != SMOE_F32)) return SMOE_ERR_DTYPE;
  if (rows < 0 || rows > 0x7fffffffll || H <= 0 || H > kMaxWidth || dy_ld < 0 || dh_ld < 0 || h_ld < 0) return SMOE_ERR_SHAPE;
  if (dx == nullptr && dweight == nullptr) return SMOE_ERR_SHAPE;
  if (rows > 0 && (dy == nullptr || h == nullptr || weight == nullptr || rstd == nullptr)) return SMOE_ERR_SHAPE;
  if ((address(dy) | address(dh) | address(h) | address(dx)) % size != 0 || (address(weight) | address(dweight)) % wsize != 0 ||
      address(rstd) % 4 != 0 || address(workspace) % 16 != 0)
    return SMOE_ERR_ALIGNMENT;
  if (dweight != nullptr && rows > 0 && workspace == nullptr) return SMOE_ERR_WORKSPACE;
  Backward a = {};
  a.dy = dy; a.dy_ld = dy_ld; a.dh = dh; a.dh_ld = dh != nullptr ? dh_ld : 0; a.h = h; a.h_ld = h_ld;
  a.w = weight; a.w_wide = address(weight) % 16 == 0;
  a.rstd = rstd; a.dx = dx; a.partial = dweight != nullptr ? static_cast<float*>(workspace) : nullptr;
  a.rows = rows; a.H = H;
  int blocks = 0, kernels = 0;
  if (rows > 0) {
    const int bytes = access_bytes({address(dy) | address(dh) | address(h) | address(dx), dy_ld * size, h_ld * size, a.dh_ld * size,
                                    static_cast<long long>(H) * size});
    const int rc = for_types(dtype, weight_dtype, [&](auto t, auto v) {
      return launched(for_access<decltype(t)>(bytes, [&](auto ve) { return launch_backward<decltype(t), decltype(v), ve>(a, blocks, S(stream)); }), 0);
    });
    if (rc != SMOE_OK) return rc;
    ++kernels;
  }
  if (dweight == nullptr) return launched(cudaSuccess, kernels);
  return launched(launch_chained(weight_grad_kernel, dim3(static_cast<unsigned>((H + 31ll) / 32)), 32 * kShares, 0, S(stream), 1,
                                 static_cast<const float*>(a.partial), blocks, H, dweight, weight_dtype), kernels + 1);
}

}  // extern "C"
