// Launcher of the tensor-core kernel for 8-bit integer products.
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
  if (fn == nullptr || !bind_context()) return SMOE_ERR_DRIVER;
  const cuuint64_t dims[2] = {cols, rows};
  const cuuint64_t strides[1] = {pitch};
  const cuuint32_t box[2] = {BK, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? SMOE_OK : SMOE_ERR_TENSORMAP;
}

template <int ACT, bool NARROW>
static int launch(const CUtensorMap& tmX, const CUtensorMap& tmFew, const CUtensorMap& tmW, const Params& p, int tile_rows, int channels,
                  int sms, cudaStream_t st) {
  static PerDeviceFlag configured;
  const auto kernel = int8_tile_kernel<ACT, NARROW>;
  const int dev = current_device();
  if (dev < 0) return SMOE_ERR_DRIVER;
  if (!configured.test(dev)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess) return SMOE_ERR_LAUNCH;
    cudaFuncAttributes fa;  // setmaxnreg 56 / 200 balances only around 128 registers per thread at launch
    if (cudaFuncGetAttributes(&fa, kernel) != cudaSuccess || fa.numRegs != 128) return SMOE_ERR_LAUNCH;
    configured.set(dev);
  }
  return launched(launch_chained(kernel, dim3(static_cast<unsigned>(sms & ~1)), THREADS, SMEM_BYTES, st, 2, tmX, tmFew, tmW, p, tile_rows, channels));
}

template <int ACT>
static int run(const int8_t* xq, long long ld, const int8_t* wq, long long w_ld, const Params& p, cudaStream_t st) {
  const int sms = num_sms();
  if (sms < 2) return SMOE_ERR_DRIVER;
  // Smaller tiles where even so no pair has two of them, whatever the load, so that pairs which had none load too; a row tile's weights
  // are loaded by each of them, x by each tile of channels.
  const bool gathered = p.gather != nullptr;
  const auto one_each = [&](long long rows, int channels) {
    const long long row_tiles = p.E == 1 ? (p.rows + rows - 1) / rows : p.rows / rows + (p.rows < p.E ? p.rows : p.E);
    return row_tiles * ((p.N + channels - 1) / channels) <= sms / 2;
  };
  int tile_rows = one_each(BM, BN) ? BM : 2 * BM, channels = BN;
  if (!gathered && one_each(128, 128)) tile_rows = channels = 128;
  if (!gathered && one_each(64, 64)) tile_rows = channels = 64;
  CUtensorMap tmX, tmFew, tmW;
  int rc = encode_rows(&tmW, wq, static_cast<uint64_t>(p.E) * p.N, p.K, w_ld, channels / 2);
  if (rc != SMOE_OK) return rc;
  tmX = tmFew = tmW;  // a map that no tile reads is not made
  if (gathered || tile_rows > BM) rc = encode_rows(&tmX, xq, p.x_rows, p.K, ld, gathered ? 1 : BM);
  if (rc == SMOE_OK && !gathered) rc = encode_rows(&tmFew, xq, p.x_rows, p.K, ld, channels < BN ? NARROW_BOX : FEW_BOX);
  if (rc != SMOE_OK) return rc;
  return channels < BN ? launch<ACT, true>(tmX, tmFew, tmW, p, tile_rows, channels, sms, st)
                       : launch<ACT, false>(tmX, tmFew, tmW, p, tile_rows, channels, sms, st);
}

int tensor_core_product(const int8_t* xq, long long ld, const int8_t* wq, long long w_ld, const Params& p, cudaStream_t st) {
  switch (p.activation) {
    case ACT_SWIGLU: return run<ACT_SWIGLU>(xq, ld, wq, w_ld, p, st);
    case ACT_GEGLU: return run<ACT_GEGLU>(xq, ld, wq, w_ld, p, st);
    case ACT_REGLU: return run<ACT_REGLU>(xq, ld, wq, w_ld, p, st);
    case ACT_RELU_SQ: return run<ACT_RELU_SQ>(xq, ld, wq, w_ld, p, st);
    case ACT_RELU: return run<ACT_RELU>(xq, ld, wq, w_ld, p, st);
    case ACT_GELU: return run<ACT_GELU>(xq, ld, wq, w_ld, p, st);
    case ACT_SILU: return run<ACT_SILU>(xq, ld, wq, w_ld, p, st);
    default: return run<kNoActivation>(xq, ld, wq, w_ld, p, st);
  }
}

}  // namespace i8
}  // namespace smoe
