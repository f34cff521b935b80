// Root-mean-square norm, gradients (the formulas are in norm.cuh).
#include "norm.cuh"

#include <atomic>

namespace smoe {
namespace norm {

struct Backward {
  const void* dy; long long dy_ld;  // values from row to row
  const void* dh; long long dh_ld;  // or nullptr
  const void* h; long long h_ld;
  const void* w; int w_wide;        // starts on a 16-byte boundary
  const float* rstd;
  void* dx;                         // packed rows, or nullptr
  float* partial;                   // (blocks, H): each block's part of the weight's gradient, or nullptr
  long long rows;
  int H;
  float per_value;                  // 1 / H
};

constexpr int kMostBlocks = 4 * 148;  // four to each of a B200's SMs

template <class T, class W, int EP, bool ALIGNED>
__device__ __forceinline__ void take_weights(const Backward& a, const Columns<T, ALIGNED>& columns, int c0, int step, Values<W, EP, kValues<T>>& w) {
  if (ALIGNED && a.w_wide) w.template load<true, false>(static_cast<const W*>(a.w), columns, c0, step);
  else w.template load<false, false>(static_cast<const W*>(a.w), columns, c0, step);
  w.template mask<ALIGNED>(columns, c0, step);
}

// With p = dy w: dx = dh + r (p - h (r mean(p h r))), the sum over a row being r times that of (dy h) w; dw sums (dy h) r.  r^2 is not formed: it leaves fp32's
// range from r = 1.8e19 on (rows of rms below 5e-20 under an eps of 0), where dx is still within it.
template <class T, class W, int EP, int VE>
__device__ __forceinline__ void row_gradient(const Values<T, EP, VE>& dy, const Values<T, EP, VE>& h, const Values<W, EP, VE>& w,
                                             const Values<T, EP, VE>& dh, float r, float mean, Values<T, EP, VE>& dx) {
  const F2 rr(r, r), along(-(r * mean), -(r * mean));
#pragma unroll
  for (int k = 0; k < EP / 2; ++k) dx.set(k, fma2(fma2(h.get(k), along, dy.get(k) * w.get(k)), rr, dh.get(k)));
}

// Blocks take rows in turn and keep the weights and their part of the weights' gradient in registers, EP columns in each thread, until the end: so
// the rows of a thread all have the same shift (Columns), `step` rows apart.  A row is read once.  Bound by memory: bf16 32768 x 4096
// with a residual 171 us, 6.3 TB/s, 8192 x 4096 51; 262144 x 128 36.5, 5.5 TB/s; fp32 4099 x 1005 16.5 us.
template <class T, class W, int EP, bool ALIGNED, int REGISTERS>
__global__ void __maxnreg__(REGISTERS) backward_kernel(const Backward a, int tpr) {
  wait_for_previous();
  constexpr int VE = kValues<T>;
  __shared__ Parts part[2];
  extern __shared__ float sums[];  // (subs, H) where a block has several rows at a time
  const Share at(tpr);
  const long long step = static_cast<long long>(gridDim.x) * at.subs;
  const long long first = static_cast<long long>(blockIdx.x) * at.subs + at.sub;
  const Columns<T, ALIGNED> columns(first, a.H);
  Values<W, EP, VE> w;
  take_weights<T, W, EP, ALIGNED>(a, columns, at.tid, tpr, w);
  F2 acc[EP / 2];
#pragma unroll
  for (int k = 0; k < EP / 2; ++k) acc[k] = F2(0.f, 0.f);
  int turn = 0;
  for (long long row = first; row - at.sub < a.rows; row += step) {
    Columns<T, ALIGNED> mine = columns;
    if (row >= a.rows) mine.pieces = 0;
    const float r = row < a.rows ? a.rstd[row] : 0.f;
    Values<T, EP, VE> dy, h, dh;
    dy.template load<ALIGNED, true>(static_cast<const T*>(a.dy) + row * a.dy_ld, mine, at.tid, tpr);
    h.template load<ALIGNED, true>(static_cast<const T*>(a.h) + row * a.h_ld, mine, at.tid, tpr);
    dy.template mask<ALIGNED>(mine, at.tid, tpr);
    h.template mask<ALIGNED>(mine, at.tid, tpr);
    Columns<T, ALIGNED> upstream = mine;
    if (a.dh == nullptr) upstream.pieces = 0;
    dh.template load<ALIGNED, true>(static_cast<const T*>(a.dh) + row * a.dh_ld, upstream, at.tid, tpr);
    F2 total(0.f, 0.f);
    const F2 rr(r, r);
#pragma unroll
    for (int k = 0; k < EP / 2; ++k) {
      const F2 t = dy.get(k) * h.get(k);
      total = fma2(t, w.get(k), total);
      acc[k] = fma2(t, rr, acc[k]);
    }
    w.forget();
    if (a.dx == nullptr) continue;
    float sum = total.sum(), none = 0.f;
    row_reduce<false>(sum, none, at, part[turn]);
    turn ^= 1;  // the next row's sums lie elsewhere: one barrier a row is enough
    dy.forget();
    h.forget();
    Values<T, EP, VE> dx;
    row_gradient(dy, h, w, dh, r, sum * r * a.per_value, dx);
    dx.template store<ALIGNED>(static_cast<T*>(a.dx) + row * a.H, mine, at.tid, tpr);
    w.forget();
  }
  if (a.partial == nullptr) return;
  float* part_of_block = a.partial + static_cast<long long>(blockIdx.x) * a.H;
  float* to = at.subs > 1 ? sums + at.sub * a.H : part_of_block;
#pragma unroll
  for (int k = 0; k < EP / 2; ++k) {
    float f[2];
    acc[k].split(f[0], f[1]);
#pragma unroll
    for (int i = 2 * k; i < 2 * k + 2; ++i) {
      const int col = columns.first(at.tid + i / VE * tpr) + i % VE;
      if (col >= 0 && col < a.H) to[col] = f[i & 1];
    }
  }
  if (at.subs == 1) return;
  __syncthreads();
  for (int c = threadIdx.x; c < a.H; c += blockDim.x) {
    float s = 0.f;
    for (int k = 0; k < at.subs; ++k) s += sums[k * a.H + c];
    part_of_block[c] = s;
  }
}

// Rows that a block's threads do not hold: read twice, EP values of each thread at a time, a row to a block at a time; the block's part of the
// weights' gradient lies in its row of `partial`, where the same thread adds to the same columns each time (equal shifts here too).
template <class T, class W, int EP, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) backward_long_kernel(const Backward a) {
  wait_for_previous();
  constexpr int VE = kValues<T>;
  __shared__ Parts part[2];
  const Share at(kThreads);
  const Columns<T, ALIGNED> columns(blockIdx.x, a.H);
  const int round = EP / VE * kThreads;
  float* mine = a.partial + static_cast<long long>(blockIdx.x) * a.H;
  Values<W, EP, VE> w;
  Values<T, EP, VE> dy, h;
  int turn = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float r = a.rstd[row];
    const auto take = [&](int c0) {
      dy.template load<ALIGNED, true>(static_cast<const T*>(a.dy) + row * a.dy_ld, columns, c0, kThreads);
      h.template load<ALIGNED, true>(static_cast<const T*>(a.h) + row * a.h_ld, columns, c0, kThreads);
      dy.template mask<ALIGNED>(columns, c0, kThreads);
      h.template mask<ALIGNED>(columns, c0, kThreads);
      take_weights<T, W, EP, ALIGNED>(a, columns, c0, kThreads, w);
    };
    F2 total(0.f, 0.f);
    for (int c0 = at.tid; c0 < columns.pieces; c0 += round) {
      take(c0);
#pragma unroll
      for (int k = 0; k < EP / 2; ++k) {
        const F2 t = dy.get(k) * h.get(k);
        total = fma2(t, w.get(k), total);
        if (a.partial != nullptr) {
          float f[2];
          t.split(f[0], f[1]);
#pragma unroll
          for (int i = 2 * k; i < 2 * k + 2; ++i) {
            const int col = columns.first(c0 + i / VE * kThreads) + i % VE;
            if (col >= 0 && col < a.H) mine[col] = fmaf(f[i & 1], r, row == blockIdx.x ? 0.f : mine[col]);
          }
        }
      }
    }
    if (a.dx == nullptr) continue;
    float sum = total.sum(), none = 0.f;
    row_reduce<false>(sum, none, at, part[turn]);
    turn ^= 1;
    for (int c0 = at.tid; c0 < columns.pieces; c0 += round) {
      take(c0);
      Values<T, EP, VE> dh, dx;
      Columns<T, ALIGNED> upstream = columns;
      if (a.dh == nullptr) upstream.pieces = 0;
      dh.template load<ALIGNED, true>(static_cast<const T*>(a.dh) + row * a.dh_ld, upstream, c0, kThreads);
      row_gradient(dy, h, w, dh, r, sum * r * a.per_value, dx);
      dx.template store<ALIGNED>(static_cast<T*>(a.dx) + row * a.H, columns, c0, kThreads);
    }
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

// Blocks of `kernel`: as many as the device holds at a time, at most one for each `subs` rows, and where rows have different shifts a multiple of
// their number (8 or 4), unless no block has a second row; 0 on failure.  `known`: the last answer of the runtime for this kernel and device.
struct Residency {
  std::atomic<unsigned long long> last[kMaxDevices] = {};  // threads, shared memory, blocks on an SM
};
template <class T, bool ALIGNED, class... Params>
static int blocks_of(void (*kernel)(Params...), int threads, size_t smem, long long rows, int subs, Residency& known) {
  const long long need = (rows + subs - 1) / subs;
  const int sms = num_sms(), dev = current_device();
  if (sms <= 0 || dev < 0) return 0;
  if (need <= sms) return static_cast<int>(need);
  const unsigned long long key = static_cast<unsigned long long>(threads) << 48 | static_cast<unsigned long long>(smem) << 16;
  const unsigned long long last = known.last[dev].load(std::memory_order_relaxed);
  int per = static_cast<int>(last & 0xFFFF);
  if (last >> 16 != key >> 16) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, threads, smem) != cudaSuccess || per <= 0) return 0;
    known.last[dev].store(key | static_cast<unsigned long long>(per), std::memory_order_relaxed);
  }
  long long all = static_cast<long long>(per) * sms;
  if (all > kMostBlocks) all = kMostBlocks;
  if (need <= all) return static_cast<int>(need);
  return static_cast<int>(ALIGNED ? all : all / kValues<T> * kValues<T>);
}

template <class T, class W, int EP, bool ALIGNED, int REGISTERS>
static cudaError_t launch_rows(const Backward& a, const Shape& s, int& blocks, cudaStream_t st) {
  const size_t smem = s.subs > 1 ? static_cast<size_t>(s.subs) * a.H * sizeof(float) : 0;  // subs H <= 256 EP
  static Residency known;
  blocks = blocks_of<T, ALIGNED>(backward_kernel<T, W, EP, ALIGNED, REGISTERS>, s.threads, smem, a.rows, s.subs, known);
  if (blocks == 0) return cudaErrorInvalidConfiguration;
  return launch_chained(backward_kernel<T, W, EP, ALIGNED, REGISTERS>, dim3(static_cast<unsigned>(blocks)), s.threads, smem, st, 1, a, s.tpr);
}
// Values of a thread, and its registers: fp32 rows 16 and 128 (with 80, 8192 x 4096 85.5 / 108 us); 16-bit rows of whole pieces 32 and 128, which
// halves what every thread does for a row (32768 x 4096 with a residual, 32 / 16 values 171 / 179 us, 16384 x 7168 157 / 177, 16384 x 5000 98 / 116),
// but short ones 16 and 80, three blocks to an SM (262144 x 128 40.0 / 36.5; 64 registers 39.8); other rows, whose pieces cost more registers, 16
// up to 256 threads a row (20000 x 2049 126 / 96.5), 32 above (16384 x 7169 245 / 278).
template <class T, class W, bool ALIGNED>
static cudaError_t launch_backward(const Backward& a, int& blocks, cudaStream_t st) {
  const long long values = a.H + (ALIGNED ? 0 : kValues<T> - 1);
  if constexpr (sizeof(T) == 4) {
    if (values <= 16 * kThreads) return launch_rows<T, W, 16, ALIGNED, 128>(a, shape_of(values, 16), blocks, st);
  } else {
    if (ALIGNED ? values < 256 : values <= 16 * 256) return launch_rows<T, W, 16, ALIGNED, 80>(a, shape_of(values, 16), blocks, st);
    if (values <= 32 * kThreads) return launch_rows<T, W, 32, ALIGNED, 128>(a, shape_of(values, 32), blocks, st);
  }
  static Residency known;
  blocks = blocks_of<T, ALIGNED>(backward_long_kernel<T, W, 16, ALIGNED>, kThreads, 0, a.rows, 1, known);
  if (blocks == 0) return cudaErrorInvalidConfiguration;
  return launch_chained(backward_long_kernel<T, W, 16, ALIGNED>, dim3(static_cast<unsigned>(blocks)), kThreads, 0, st, 1, a);
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
  if ((address(dy) | address(dh) | address(h)) % size != 0 || address(dx) % 16 != 0 || (address(weight) | address(dweight)) % wsize != 0 ||
      address(rstd) % 4 != 0 || address(workspace) % 16 != 0)
    return SMOE_ERR_ALIGNMENT;
  if (dweight != nullptr && rows > 0 && workspace == nullptr) return SMOE_ERR_WORKSPACE;
  Backward a = {};
  a.dy = dy; a.dy_ld = dy_ld; a.dh = dh; a.dh_ld = dh != nullptr ? dh_ld : 0; a.h = h; a.h_ld = h_ld;
  a.w = weight; a.w_wide = address(weight) % 16 == 0;
  a.rstd = rstd; a.dx = dx; a.partial = dweight != nullptr ? static_cast<float*>(workspace) : nullptr;
  a.rows = rows; a.H = H; a.per_value = 1.f / static_cast<float>(H);
  int blocks = 0, kernels = 0;
  if (rows > 0) {
    const bool aligned = (address(dy) | address(dh) | address(h) | dy_ld * size | a.dh_ld * size | h_ld * size | static_cast<long long>(H) * size) % 16 == 0;
    const int rc = for_types(dtype, weight_dtype, [&](auto t, auto v) {
      using T = decltype(t);
      using W = decltype(v);
      return launched(aligned ? launch_backward<T, W, true>(a, blocks, S(stream)) : launch_backward<T, W, false>(a, blocks, S(stream)), 0);
    });
    if (rc != SMOE_OK) return rc;
    ++kernels;
  }
  if (dweight == nullptr) return launched(cudaSuccess, kernels);
  return launched(launch_chained(weight_grad_kernel, dim3(static_cast<unsigned>((H + 31ll) / 32)), 32 * kShares, 0, S(stream), 1,
                                 static_cast<const float*>(a.partial), blocks, H, dweight, weight_dtype), kernels + 1);
}

}  // extern "C"
