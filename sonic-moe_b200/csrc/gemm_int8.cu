// Launchers of the tensor-core kernels for 8-bit integer products, and which of them a call takes.
#include "gemm_int8.cuh"

#include <mutex>

#include "../../include/sonicmoe_b200.h"
#include "internal.h"

namespace smoe {
namespace i8 {

static_assert(kMaxExpertRows == kMaxExperts, "the library's limit");

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                   const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn get_encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  });
  return fn;
}

// Rows of `cols` bytes, `pitch` bytes apart; boxes of box_rows x 128 bytes, 128-byte swizzle, zeros outside.
static int encode_rows(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t pitch, uint32_t box_rows) {
  const EncodeTiledFn fn = get_encode_fn();
  if (fn == nullptr) return SMOE_ERR_DRIVER;
  static thread_local bool context_bound = false;  // a thread without any runtime call so far has no current context
  if (!context_bound) {
    if (cudaFree(nullptr) != cudaSuccess) return SMOE_ERR_DRIVER;
    context_bound = true;
  }
  const cuuint64_t dims[2] = {cols, rows};
  const cuuint64_t strides[1] = {pitch};
  const cuuint32_t box[2] = {BK, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? SMOE_OK : SMOE_ERR_TENSORMAP;
}

template <class Kernel>
static int configure(Kernel kernel, PerDeviceFlag& configured, int smem_bytes, bool splits_registers) {
  const int dev = current_device();
  if (dev < 0) return SMOE_ERR_DRIVER;
  if (configured.test(dev)) return SMOE_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes) != cudaSuccess) return SMOE_ERR_LAUNCH;
  if (splits_registers) {  // setmaxnreg 56 / 200 balances only around 128 registers per thread at launch
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, kernel) != cudaSuccess || fa.numRegs != 128) return SMOE_ERR_LAUNCH;
  }
  configured.set(dev);
  return SMOE_OK;
}

template <int MODE>
static int launch_tiles(const CUtensorMap& tmA, const CUtensorMap& tmB, const Params& p, int least, cudaStream_t st) {
  static PerDeviceFlag configured;
  const auto kernel = tiles::int8_tile_kernel<MODE>;
  const int rc = configure(kernel, configured, tiles::SMEM_BYTES, true);
  if (rc != SMOE_OK) return rc;
  const int sms = num_sms();
  if (sms < 2) return SMOE_ERR_DRIVER;
  return launched(launch_chained(kernel, dim3(static_cast<unsigned>(sms & ~1)), tiles::THREADS, tiles::SMEM_BYTES, st, 2, tmA, tmB, p, least));
}

template <int MODE, bool SPLIT>
static int launch_units(const CUtensorMap& tmW, const CUtensorMap& tmX, const Params& p, const int8_t* wq, long long w_ld, int most, int nt, int split, int clusters,
                        cudaStream_t st) {
  static PerDeviceFlag configured;
  const auto kernel = units::int8_unit_kernel<MODE, SPLIT>;
  const int rc = configure(kernel, configured, 227 * 1024, false);
  if (rc != SMOE_OK) return rc;
  const int sms = num_sms();
  if (sms <= 0) return SMOE_ERR_DRIVER;
  const int stages = units::num_stages(nt);
  const unsigned grid = SPLIT ? static_cast<unsigned>(clusters * split) : static_cast<unsigned>(sms);
  return launched(launch_chained(kernel, dim3(grid), units::THREADS, units::smem_bytes(nt, stages), st, static_cast<unsigned>(split), tmW,
                                 tmX, p, wq, w_ld, most, nt, stages, split));
}

// Which kernels take the rows: units of `unit` rows (0: none) for experts with at most `most`, tiles for the others.
struct Choice {
  int unit = 0, most = 0, split = 1, clusters = 0;
};
static Choice choose(const Params& p, int sms) {
  Choice c;
  const long long blocks = (p.N + units::BM - 1) / units::BM;
  const int num_kb = (p.K + BK - 1) / BK;
  const long long used = p.E < p.rows ? p.E : p.rows;  // experts that can have rows
  // the most units of nt rows that any load gives
  const auto bound = [&](int nt) { return (p.E == 1 ? (p.rows + nt - 1) / nt : p.rows / nt + used) * blocks; };
  const double mean = static_cast<double>(p.rows) / p.E;
  if (p.E == 1) {
    // one load only: units where there are at most two per SM and they need fewer rounds than the tiles, which take twice as long
    const long long u = (p.rows + 127ll) / 128 * blocks;
    const long long t = (p.rows + 255ll) / 256 * ((p.N + 255) / 256);
    if (u > 2ll * sms || (u + sms - 1) / sms >= 2 * ((t + sms / 2 - 1) / (sms / 2))) return c;
    c.unit = p.rows <= 32 ? 32 : p.rows <= 64 ? 64 : 128;
    c.most = p.rows;
  } else {
    if (mean > 96) return c;
    const int by_mean = mean <= 12 ? 32 : mean <= 40 ? 64 : units::MAX_NT;
    const bool divide = 1.0 * p.E * p.N * p.K >= 0.5e9;
    const int largest = divide && 2 * by_mean < units::MAX_NT ? 2 * by_mean : units::MAX_NT;
    bool alone = false;
    for (c.unit = by_mean; c.unit <= largest; c.unit *= 2) {
      if ((p.rows + c.unit - 1) / c.unit * blocks <= 2ll * sms) { alone = true; break; }
    }
    if (alone) {
      c.most = p.rows;
    } else {
      c.unit = divide ? by_mean : 0;
      c.most = 2 * by_mean;
      return c;
    }
  }
  const long long most_units = bound(c.unit);
  while (c.split < units::MAX_SPLIT && most_units * 2 * c.split <= sms && 2 * 2 * c.split <= num_kb) c.split *= 2;
  c.clusters = static_cast<int>(most_units);
  return c;
}

template <int MODE>
static int run(const int8_t* xq, long long ld, const int8_t* wq, long long w_ld, Params p, cudaStream_t st) {
  const int sms = num_sms();
  if (sms < 2) return SMOE_ERR_DRIVER;
  const Choice c = choose(p, sms);
  CUtensorMap tmW, tmX;
  int rc = encode_rows(&tmW, wq, static_cast<uint64_t>(p.E) * p.N, p.K, w_ld, 128);
  if (rc != SMOE_OK) return rc;
  static_assert(units::BM == tiles::BN_CTA, "one weight map for both kernels");
  if (c.unit > 0) {
    rc = encode_rows(&tmX, xq, p.x_rows, p.K, ld, p.gather != nullptr ? 1 : units::BOX_ROWS);
    if (rc != SMOE_OK) return rc;
    p.zero_others = 1;
    rc = c.split > 1 ? launch_units<MODE, true>(tmW, tmX, p, wq, w_ld, c.most, c.unit, c.split, c.clusters, st)
                     : launch_units<MODE, false>(tmW, tmX, p, wq, w_ld, c.most, c.unit, 1, 0, st);
    if (rc != SMOE_OK || c.most >= p.rows) return rc;
  }
  rc = encode_rows(&tmX, xq, p.x_rows, p.K, ld, p.gather != nullptr ? 1 : tiles::BM);
  if (rc != SMOE_OK) return rc;
  p.zero_others = c.unit == 0;
  return launch_tiles<MODE>(tmX, tmW, p, c.most, st);
}

int tensor_core_product(const int8_t* xq, long long ld, const int8_t* wq, long long w_ld, const Params& p, cudaStream_t st) {
  if (p.activation == kNoActivation) return run<MODE_PLAIN>(xq, ld, wq, w_ld, p, st);
  if (p.activation == ACT_SWIGLU) return run<MODE_SWIGLU>(xq, ld, wq, w_ld, p, st);
  return run<MODE_ANY>(xq, ld, wq, w_ld, p, st);
}

}  // namespace i8
}  // namespace smoe
