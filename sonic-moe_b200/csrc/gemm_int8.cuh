// 8-bit integer products on the tensor cores (tcgen05.mma.kind::i8: signed bytes, 32-bit integer accumulators in tensor
// memory).  A stage holds 128 columns of an operand row, 128 bytes, so staging, swizzle and descriptors are those of the bf16
// kernels with elements of half the size, and a stage's four MMAs (K 32 each) do twice the work in the same time.
//
// Persistent CTA pairs (cta_group::2), tiles of 256 rows x 256 channels, two accumulators.  An expert's last tile with at most 224
// rows (every tile of a decode step) has the operands in each other's places: its 256 channels are the MMA's rows, and its rows of
// x, up to the next 32, the columns, so that neither rows that do not exist are multiplied nor their stages filled.
//
// Narrow tiles, of 64 rows x 64 channels or 128 x 128, where that many tiles are not more than the pairs (dense products of few
// rows): a stage's bytes hold four or two blocks of 128 columns, so that each of more pairs has as many bytes on their way, which
// is what a short walk waits for, and an MMA has 128 rows, which takes half the time of one with 256.  Channels are the MMA's rows
// here too.  33 rows, 8-bit x: 4096 x 4096 13.1 -> 9.9 us, 2048 x 7168 18.2 -> 12.2, 7168 x 2048 10.5 -> 9.5, 1024 x 1024 7.6 -> 6.9.
// (A block of 64 channels reads 128 bytes each of as many rows again behind its own: sums that no lane takes.)
//
// Warps of a CTA (16): 0 TMA producer (weights; x unless gathered), 1 MMA issuer (leader CTA), 2 and 3 zeros for the rows that no
// expert has, 4..11 epilogue, 12..15 row gather with TMA tile::gather4 (a row that is none reads zeros).  The columns past the
// last are zeros by the tensor maps' extent.
//
// Barriers.  full[s]: leader only; two arrivals, of the two producers, and the bytes of both CTAs.  The other CTA's producer arrives
// although it may have nothing to load (no channels in its half of the tile): a role that a stage does not need could be overtaken
// by the ring twice, and would take an old phase for the one it waits for.  empty[s], acc_full[a]: per CTA, by the leader's commits.
// acc_empty[a]: leader only, one arrival per epilogue warp of both CTAs.  Every wait is bounded (ptx.cuh).
#pragma once
#include <type_traits>

#include "int8.cuh"
#include "ptx.cuh"

namespace smoe {
namespace i8 {

constexpr int BK = 128;  // columns, and bytes, of a stage's row
constexpr int UMMA_K = 32;

__host__ __device__ constexpr uint32_t make_idesc_i8(int M, int N) {
  return (2u << 4)                     // D: 32-bit integers
         | (1u << 7) | (1u << 10)      // A, B: signed bytes, K-major
         | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t"
      "}\n"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void st_shared_word(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_shared_word(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// Where a warp's block of outputs goes: row r of it to base + r * pitch, `valid` bytes from the block's first column to the
// row's end.
struct Block {
  char* base;
  long long pitch;
  int rows;        // rows that exist
  long long valid;
  bool wide;       // 16-byte pieces; otherwise value by value
  bool half;       // 16-bit values
};

// A warp's staged rows (STRIDE bytes apart, BYTES of each, ROWS of them; address of a 16-byte piece by `piece`) go out: whole
// row segments, neighbouring lanes on neighbouring pieces.  All lanes.
template <int ROWS, int BYTES, class Piece>
__device__ __forceinline__ void store_staged(int lane, const Block& b, Piece&& piece) {
  __syncwarp();
  if (b.wide) {
    constexpr int PIECES = BYTES / 16, PER = 32 / PIECES;
#pragma unroll
    for (int i = 0; i < ROWS / PER; ++i) {
      const int r = PER * i + lane / PIECES, q = lane % PIECES;
      const uint4 v = ld_shared_v4(piece(r, q));
      if (r < b.rows && 16 * q < b.valid) *reinterpret_cast<uint4*>(b.base + r * b.pitch + 16 * q) = v;
    }
  } else {
    constexpr int WORDS = BYTES / 4, PER = 32 / WORDS;
    for (int i = 0; i < ROWS / PER; ++i) {
      const int r = PER * i + lane / WORDS, w = lane % WORDS;
      const uint32_t v = ld_shared_word(piece(r, w / 4) + 4 * (w % 4));
      if (r >= b.rows) continue;
      char* dst = b.base + r * b.pitch + 4 * w;
      if (b.half) {
        if (4 * w < b.valid) *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(v);
        if (4 * w + 2 < b.valid) *reinterpret_cast<uint16_t*>(dst + 2) = static_cast<uint16_t>(v >> 16);
      } else if (4 * w < b.valid) {
        *reinterpret_cast<uint32_t*>(dst) = v;
      }
    }
  }
  __syncwarp();
}

// The exclusive prefix of the row tiles of all experts, from their first rows and ends in shared memory.  One warp, all lanes.
template <class Shared>
__device__ __forceinline__ void count_tiles(const Params& p, Shared& ss, int tile_rows, int lane) {
  int running = 0;
  for (int base = 0; base < p.E; base += 32) {
    const int e = base + lane;
    const int v = e < p.E ? max(ss.end[e] - ss.first[e] + tile_rows - 1, 0) / tile_rows : 0;
    int incl = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += o;
    }
    if (e < p.E) ss.tiles_before[e] = running + incl - v;
    running += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) ss.tiles_before[p.E] = running;
}

// Scale and bias of channel f + lane; scale of row row0 + lane.  Loaded before the sums are waited for.
__device__ __forceinline__ void load_channel(const Params& p, int e, int f, int lane, float& ws, float& bias) {
  const bool mine = f + lane < p.N;
  const long long at = static_cast<long long>(e) * p.N + f + lane;
  ws = mine ? p.w_scale[at] : 0.f;
  bias = mine && p.bias != nullptr ? load_typed(p.bias, p.bias_type, at) : 0.f;
}
__device__ __forceinline__ float load_row_scale(const Params& p, int row0, int rows, int lane) {
  if (lane >= rows) return 0.f;
  const int s = source_row(p, row0 + lane);
  return s >= 0 ? p.x_scale[s] : 0.f;
}

// 32 channels (lane l: channel f + l) of up to 32 rows (word j: row row0 + j), of which `rows` exist.  Neighbouring lanes exchange
// half of their values: afterwards word j of an even lane has the channels (l, l + 1) of row 2j and that of an odd one (l - 1, l) of
// row 2j + 1, a gate and its up value, or two values of one 32-bit store.
template <int ACT>
__device__ __forceinline__ void store_rows(const Params& p, uint32_t stage, int lane, int f, int row0, int rows,
                                           const uint32_t (&v)[32], float ws, float bias, float xs) {
  const bool odd = lane & 1;
  constexpr bool gated = is_gated(ACT);
  float lo[16], hi[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    float a = scaled(static_cast<int>(v[2 * j]), __shfl_sync(0xffffffffu, xs, 2 * j), ws);
    float b = scaled(static_cast<int>(v[2 * j + 1]), __shfl_sync(0xffffffffu, xs, 2 * j + 1), ws);
    if (p.bias != nullptr) { a = biased(a, bias); b = biased(b, bias); }
    if constexpr (!gated) { a = activate<ACT>(a); b = activate<ACT>(b); }
    const float other = __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
    lo[j] = odd ? other : a;
    hi[j] = odd ? b : other;
  }
  const long long cols = gated ? p.N / 2 : p.N;
  const int size = p.out_type == SMOE_F32 ? 4 : 2;
  Block b;
  b.pitch = cols * size;
  const long long col = gated ? f / 2 : f;
  b.base = static_cast<char*>(p.out) + row0 * b.pitch + col * size;
  b.rows = rows;
  b.valid = (cols - col) * size;
  b.wide = p.wide_out;
  b.half = size == 2;
  const int pair = lane >> 1;
  const auto at_word = [&](int row, int bytes, int byte) { return stage + row * bytes + byte; };
  if constexpr (gated) {
#pragma unroll
    for (int j = 0; j < 16; ++j) lo[j] = activate<ACT>(lo[j]) * hi[j];
    if (b.half) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const uint32_t h = pack_typed(p.out_type, lo[j], 0.f) & 0xFFFFu;
        asm volatile("st.shared.b16 [%0], %1;" ::"r"(at_word(2 * j + odd, 32, 2 * pair)), "h"(static_cast<unsigned short>(h)) : "memory");
      }
      store_staged<32, 32>(lane, b, [&](int r, int q) { return stage + r * 32 + 16 * q; });
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) st_shared_word(at_word(2 * j + odd, 64, 4 * pair), __float_as_uint(lo[j]));
      store_staged<32, 64>(lane, b, [&](int r, int q) { return stage + r * 64 + 16 * q; });
    }
  } else if (b.half) {
#pragma unroll
    for (int j = 0; j < 16; ++j) st_shared_word(at_word(2 * j + odd, 64, 4 * pair), pack_typed(p.out_type, lo[j], hi[j]));
    store_staged<32, 64>(lane, b, [&](int r, int q) { return stage + r * 64 + 16 * q; });
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // 16 rows of 128 bytes at a time
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        st_shared_word(at_word(2 * j + odd, 128, 8 * pair), __float_as_uint(lo[8 * h + j]));
        st_shared_word(at_word(2 * j + odd, 128, 8 * pair + 4), __float_as_uint(hi[8 * h + j]));
      }
      store_staged<16, 128>(lane, b, [&](int r, int q) { return stage + r * 128 + 16 * q; });
      b.base += 16 * b.pitch;
      b.rows -= 16;
    }
  }
}

constexpr int BM = 128, BN = 256, BN_CTA = 128, STAGES = 6;
constexpr int A_STAGE_BYTES = BM * BK, B_STAGE_BYTES = BN_CTA * BK;
constexpr int THREADS = 512, FIRST_EPI_WARP = 4, EPI_WARPS = 8, FIRST_GATHER_WARP = 12, GATHER_WARPS = 4;
constexpr int COLS_PER_WARP = BN * 4 / EPI_WARPS;
constexpr int FEW_BOX = 16;     // rows per TMA box of a tile with few rows
constexpr int NARROW_BOX = 32;  // of a narrow tile

struct Shared {
  uint64_t full[STAGES];
  uint64_t empty[STAGES];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
  int first[kMaxExpertRows];
  int end[kMaxExpertRows];
  int tiles_before[kMaxExpertRows + 1];
};
constexpr int SMEM_BYTES = 1024 + STAGES * (A_STAGE_BYTES + B_STAGE_BYTES) + ((sizeof(Shared) + 127) & ~127) + EPI_WARPS * (STAGE_ROWS_BYTES + COLS_PER_WARP * 4);
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory per CTA");

// With the operands in each other's places each CTA has its own 128 channels, staged as before, and stages half of the `few` rows of
// x, a multiple of 32.  The sums lie one channel to a lane.  Without it a fifth of the MMAs of 8192 tokens (H 4096, I 1024, E 128, K 8)
// works on rows that do not exist: up projection with its quantisation 450 -> 412 us.  Experts with few rows need no kernel of their
// own either: units of 128 channels x 128 rows per CTA took 231 us for 32 rows per expert of that layer, the tiles take 184.
// Bound by: the weights from memory below some 64 rows per expert (64 tokens of that layer, 1.0 GB in 142 us); above, the MMAs under
// the power cap (8192 x 7168 x 4096 3.4e15 operations/s alone, tensor pipe 80 % busy at 1.5 GHz in the 8192-token load).
struct Tile {
  int e, row0, row_end, n0;  // row0: of this CTA's staged rows
  int first;                 // row of the pair's tile
  int few;                   // 0: rows are the MMA's rows
};
template <bool NARROW>
__device__ __forceinline__ int few_rows(int rows) {
  if (NARROW) return rows <= 64 ? 64 : 128;
  return rows <= 2 * BM - 32 ? (rows + 31) & ~31 : 0;
}

// The tiles of this CTA pair, expert by expert, the channels of a row tile innermost, dealt out round-robin.
template <bool NARROW>
struct Walker {
  const Params& p;
  const Shared& ss;
  const int lane, tile_rows, channels, num_n, total, step_m, step_n;
  int t, mi, ni, e = 0;
  __device__ __forceinline__ Walker(const Params& p_, const Shared& ss_, int lane_, int tile_rows_, int channels_)
      : p(p_), ss(ss_), lane(lane_), tile_rows(tile_rows_), channels(channels_), num_n((p_.N + channels_ - 1) / channels_), total(ss_.tiles_before[p_.E] * num_n),
        step_m(static_cast<int>(gridDim.x >> 1) / num_n), step_n(static_cast<int>(gridDim.x >> 1) % num_n),
        t(blockIdx.x >> 1), mi(t / num_n), ni(t % num_n) {}
  __device__ __forceinline__ void advance() {
    mi += step_m;
    ni += step_n;
    if (ni >= num_n) { ni -= num_n; ++mi; }
    t += gridDim.x >> 1;
  }
  // for one thread, which wants to know Tile::few only
  __device__ __forceinline__ bool next_alone(int& few) {
    if (t >= total) return false;
    while (ss.tiles_before[e + 1] <= mi) ++e;
    few = few_rows<NARROW>(min(ss.end[e] - ss.first[e] - (mi - ss.tiles_before[e]) * tile_rows, tile_rows));
    advance();
    return true;
  }
  __device__ __forceinline__ bool next(uint32_t rank, Tile& tile) {
    if (t >= total) return false;
    while (true) {  // the first expert whose tiles end beyond mi, 32 experts at a time
      const int i = e + 1 + lane;
      const unsigned before = __ballot_sync(0xffffffffu, i <= p.E && ss.tiles_before[i] <= mi);
      e += __popc(before);
      if (before != 0xffffffffu) break;
    }
    tile.e = e;
    tile.first = ss.first[e] + (mi - ss.tiles_before[e]) * tile_rows;
    tile.row_end = min(ss.end[e], tile.first + tile_rows);
    tile.few = few_rows<NARROW>(tile.row_end - tile.first);
    tile.row0 = tile.first + static_cast<int>(rank) * (tile.few != 0 ? tile.few / 2 : BM);
    tile.n0 = ni * channels;
    advance();
    return true;
  }
};

// 32 channels of the warp's 32 rows: lane l has row l's sums in v, and (with a bias) channel n + l's bias; scales: those of the 32
// channels, in shared memory, where they were put before the accumulator was waited for.  With loads of the same words by all
// lanes from memory, asked for in advance or not, a tile waits up to 2.5 kilocycles for each 32 channels: 8192 x 7168 x 1024 took 72
// us, 55 without them.
template <int ACT>
__device__ __forceinline__ void store_columns(const Params& p, uint32_t stage, int lane, int row_base, int row_end, int n,
                                              const uint32_t (&v)[32], float xs, uint32_t scales, float bias) {
  float f[32];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint4 w = ld_shared_v4(scales + 16 * j);
    f[4 * j] = scaled(static_cast<int>(v[4 * j]), xs, __uint_as_float(w.x));
    f[4 * j + 1] = scaled(static_cast<int>(v[4 * j + 1]), xs, __uint_as_float(w.y));
    f[4 * j + 2] = scaled(static_cast<int>(v[4 * j + 2]), xs, __uint_as_float(w.z));
    f[4 * j + 3] = scaled(static_cast<int>(v[4 * j + 3]), xs, __uint_as_float(w.w));
  }
  if (p.bias != nullptr) {
#pragma unroll
    for (int j = 0; j < 32; ++j) f[j] = biased(f[j], __shfl_sync(0xffffffffu, bias, j));
  }
  constexpr bool gated = is_gated(ACT);
  const long long cols = gated ? p.N / 2 : p.N;
  const int size = p.out_type == SMOE_F32 ? 4 : 2;
  Block b;
  b.pitch = cols * size;
  const long long col = gated ? n / 2 : n;
  b.base = static_cast<char*>(p.out) + row_base * b.pitch + col * size;
  b.rows = row_end - row_base;
  b.valid = (cols - col) * size;
  b.wide = p.wide_out;
  b.half = size == 2;
  const auto piece = [&](int r, int q) { return stage_piece(stage, r, q); };
  const auto put = [&](int q, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) { st_shared_v4(piece(lane, q), w0, w1, w2, w3); };
  const auto bits = [&](int j) { return __float_as_uint(f[j]); };
  const auto two = [&](int j) { return pack_typed(p.out_type, f[j], f[j + 1]); };
  if constexpr (gated) {
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j] = activate<ACT>(f[2 * j]) * f[2 * j + 1];
    if (b.half) {
#pragma unroll
      for (int q = 0; q < 2; ++q) put(q, two(8 * q), two(8 * q + 2), two(8 * q + 4), two(8 * q + 6));
      store_staged<32, 32>(lane, b, piece);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) put(q, bits(4 * q), bits(4 * q + 1), bits(4 * q + 2), bits(4 * q + 3));
      store_staged<32, 64>(lane, b, piece);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 32; ++j) f[j] = activate<ACT>(f[j]);
  if (b.half) {
#pragma unroll
    for (int q = 0; q < 4; ++q) put(q, two(8 * q), two(8 * q + 2), two(8 * q + 4), two(8 * q + 6));
    store_staged<32, 64>(lane, b, piece);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int q = 0; q < 4; ++q) put(q, bits(16 * h + 4 * q), bits(16 * h + 4 * q + 1), bits(16 * h + 4 * q + 2), bits(16 * h + 4 * q + 3));
      store_staged<32, 64>(lane, b, piece);
      b.base += 64;
      b.valid -= 64;
    }
  }
}

// ACT: kNoActivation or an Activation (compiled in: with a switch around the element loop's functions GELU took three times as long).
// tmX: rows of x, a box one row high where they are gathered, else BM rows; tmFew: boxes of FEW_BOX rows, unless gathered.
// tile_rows: 256, or 128 where that leaves fewer CTA pairs idle.  NARROW: tile_rows = narrow_channels = 64 or 128, not gathered.
template <int ACT, bool NARROW>
__global__ void __launch_bounds__(THREADS, 1)
int8_tile_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmFew, const __grid_constant__ CUtensorMap tmW,
                 const Params p, const int tile_rows, const int narrow_channels) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_STAGE_BYTES;
  Shared& ss = *reinterpret_cast<Shared*>(smem + STAGES * (A_STAGE_BYTES + B_STAGE_BYTES));
  uint8_t* stage_out = reinterpret_cast<uint8_t*>(&ss) + ((sizeof(Shared) + 127) & ~127);
  const int warp = warp_index();
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  volatile int* abort_flag = &ss.abort_flag;
  const int num_kb = (p.K + BK - 1) / BK;
  const bool gathered = !NARROW && p.gather != nullptr;
  const int channels = NARROW ? narrow_channels : BN, half = channels / 2;
  const int per_stage = NARROW ? BN / channels : 1;  // blocks of BK columns

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&ss.full[s]), 2);
      mbar_init(smem_u32(&ss.empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&ss.acc_full[a]), 1);
      mbar_init(smem_u32(&ss.acc_empty[a]), 2 * EPI_WARPS);
    }
    ss.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmW);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&ss.tmem_base), 2 * BN);
    tmem_relinquish();
  }
  wait_for_previous();
  // All experts at once: one warp by itself waits for the offsets of every 32 experts in turn (64 rows of 256 experts, 312 x 1600,
  // 51.2 -> 50.2 us; of 32 experts, 512 x 1024, 13.3 -> 13.6).
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    ss.first[e] = first_row(p, e);
    ss.end[e] = end_row(p, e);
  }
  __syncthreads();
  if (warp == 2) count_tiles(p, ss, tile_rows, lane);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = ss.tmem_base;

  if (warp < FIRST_EPI_WARP) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      // ---- TMA producer: the weights, and the rows of x where they are not gathered --------------
      const bool elected = elect_one();
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      Tile tile;
      Walker<NARROW> walk(p, ss, lane, tile_rows, channels);
      while (ok && walk.next(rank, tile)) {
        const int staged = tile.few != 0 ? tile.few / 2 : BM;  // rows of x in each CTA
        // channels behind the last are not loaded: the other half of the tile may have none (what it holds then is never stored)
        const int n = tile.n0 + static_cast<int>(rank) * half;
        const bool boxes = NARROW || (!gathered && staged <= BM / 2);  // small ones, or one of BM rows
        constexpr int BOX = NARROW ? NARROW_BOX : FEW_BOX;
        const uint32_t bytes = (2 * (gathered || boxes ? staged : BM) + (tile.n0 + half < p.N ? channels : half)) * BK;
        for (int kb = 0; kb < num_kb; kb += per_stage) {
          if (!mbar_wait_warp(smem_u32(&ss.empty[stage]), phase ^ 1u, abort_flag)) { ok = false; break; }
          if (elected) {
            const int blocks = NARROW ? min(per_stage, num_kb - kb) : 1;
            const uint32_t bar = map_to_cta(smem_u32(&ss.full[stage]), 0);
            if (leader) mbar_arrive_expect_tx(smem_u32(&ss.full[stage]), blocks * bytes);
            else mbar_arrive_cluster_relaxed(bar);
            for (int i = 0; i < blocks; ++i) {
              const uint32_t at = NARROW ? i * half * BK : 0, x_dst = smem_u32(sA + stage * A_STAGE_BYTES) + at;
              const int col = (kb + i) * BK;
              if (!gathered && !boxes) {
                tma_load_2d_pair(&tmX, bar, x_dst, col, tile.row0);
              } else if (boxes) {
                for (int r = 0; r < staged; r += BOX) tma_load_2d_pair(&tmFew, bar, x_dst + r * BK, col, tile.row0 + r);
              }
              if (n < p.N) tma_load_2d_pair(&tmW, bar, smem_u32(sB + stage * B_STAGE_BYTES) + at, col, tile.e * p.N + n);
            }
          }
          __syncwarp();
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok && lane == 0 && p.status) atomicCAS(p.status, ST_OK, ST_TIMEOUT_PRODUCER);
    } else if (warp == 1) {
      // ---- MMA issuer ------------------------------------------------------------------------
      if (leader && elect_one()) {
        int stage = 0, acc = 0, few = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        Walker<NARROW> walk(p, ss, lane, tile_rows, channels);
        while (ok && walk.next_alone(few)) {
          const uint32_t idesc = make_idesc_i8(NARROW ? BM : 2 * BM, few != 0 ? few : BN);
          if (!mbar_wait(smem_u32(&ss.acc_empty[acc]), acc_phase ^ 1u, abort_flag)) { ok = false; break; }
          tc_fence_after();
          for (int kb = 0; kb < num_kb; kb += per_stage) {
            if (!mbar_wait(smem_u32(&ss.full[stage]), phase, abort_flag)) { ok = false; break; }
            tc_fence_after();
            const uint64_t x_desc = make_smem_desc(smem_u32(sA + stage * A_STAGE_BYTES), 16, 1024);
            const uint64_t w_desc = make_smem_desc(smem_u32(sB + stage * B_STAGE_BYTES), 16, 1024);
            uint64_t a_desc = NARROW || few != 0 ? w_desc : x_desc, b_desc = NARROW || few != 0 ? x_desc : w_desc;
            const int blocks = NARROW ? min(per_stage, num_kb - kb) : 1;
            for (int i = 0; i < blocks; ++i) {
#pragma unroll
              for (int k4 = 0; k4 < BK / UMMA_K; ++k4)
                umma_i8_pair(tmem_base + acc * BN, a_desc + ((k4 * UMMA_K) >> 4), b_desc + ((k4 * UMMA_K) >> 4), idesc,
                           (kb > 0 || i > 0 || k4 > 0) ? 1u : 0u);
              if constexpr (NARROW) {
                a_desc += (half * BK) >> 4;
                b_desc += (half * BK) >> 4;
              }
            }
            umma_commit_pair(smem_u32(&ss.empty[stage]), 3);
            if (++stage == STAGES) { stage = 0; phase ^= 1u; }
          }
          if (!ok) break;
          umma_commit_pair(smem_u32(&ss.acc_full[acc]), 3);
          if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
        }
        if (!ok && p.status) atomicCAS(p.status, ST_OK, ST_TIMEOUT_MMA);
      }
    } else {
      zero_other_rows(p, 2 * blockIdx.x + (warp - 2), 2 * gridDim.x);
    }
  } else if (warp >= FIRST_GATHER_WARP) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    // ---- row gather: one thread of each warp issues for 32 rows -------------------------------
    if (gathered) {
      const int gw = warp - FIRST_GATHER_WARP;
      const bool elected = elect_one();
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      Tile tile;
      Walker<NARROW> walk(p, ss, lane, tile_rows, channels);
      while (ok && walk.next(rank, tile)) {
        // Every warp has a quarter of the CTA's rows, 4 at least: a stage is not full without it.  A warp that had none would wait for
        // stages by parity that the others could overtake twice, and take an old phase for the one it waits for.
        const int ops = (tile.few != 0 ? tile.few / 2 : BM) / 16;
        const int r = tile.row0 + 4 * ops * gw + lane;
        int mine = p.x_rows;  // rows that do not exist: zeros
        if (lane < 4 * ops && r < tile.row_end) {
          const int s = source_row(p, r);
          if (s >= 0) mine = s;
        }
        int rows[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) rows[i] = __shfl_sync(0xffffffffu, mine, i);
        if (elected) {
          // all eight operations without a test between them, or up to four or seven
          const auto issue = [&](auto most) {
            constexpr int MOST = decltype(most)::value;
            for (int kb = 0; kb < num_kb; ++kb) {
              if (!mbar_wait(smem_u32(&ss.empty[stage]), phase ^ 1u, abort_flag)) { ok = false; break; }
              const uint32_t bar = map_to_cta(smem_u32(&ss.full[stage]), 0);
              const uint32_t dst = smem_u32(sA + stage * A_STAGE_BYTES) + gw * (MOST == 8 ? 8 : ops) * 512;
#pragma unroll
              for (int q = 0; q < MOST; ++q)
                if (MOST == 8 || q < ops)
                  tma_gather4_pair(&tmX, bar, dst + q * 512, kb * BK, rows[4 * q], rows[4 * q + 1], rows[4 * q + 2], rows[4 * q + 3]);
              if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
          };
          if (ops == 8) issue(std::integral_constant<int, 8>());
          else if (ops <= 4) issue(std::integral_constant<int, 4>());
          else issue(std::integral_constant<int, 7>());
        }
        ok = __all_sync(0xffffffffu, ok);
      }
      if (!ok && lane == 0 && p.status) atomicCAS(p.status, ST_OK, ST_TIMEOUT_PRODUCER);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---- epilogue: a warp has 32 rows x 128 channels -------------------------------------------
    const int quad = warp & 3;
    const int col_half = (warp - FIRST_EPI_WARP) >> 2;
    const uint32_t my_stage = smem_u32(stage_out) + (warp - FIRST_EPI_WARP) * STAGE_ROWS_BYTES;
    const uint32_t my_scales = smem_u32(stage_out) + EPI_WARPS * STAGE_ROWS_BYTES + (warp - FIRST_EPI_WARP) * (COLS_PER_WARP * 4);
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    Tile tile;
    Walker<NARROW> walk(p, ss, lane, tile_rows, channels);
    while (ok && walk.next(rank, tile)) {
      const auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(map_to_cta(smem_u32(&ss.acc_empty[acc]), 0));
      };
      if constexpr (NARROW) {
        // an MMA of 128 rows (64 channels of each CTA): the upper 64 lanes have the second half of the columns
        const int at = (quad & 1) * 32, f = tile.n0 + static_cast<int>(rank) * half + at;
        const int col = 32 * col_half, r = (quad >> 1) * (tile.few / 2) + col, rows = tile.row_end - tile.first - r;
        const bool works = f < p.N && at < half && col < tile.few / 2 && rows > 0;
        float ws = 0.f, bias = 0.f, xs = 0.f;
        if (works) {
          load_channel(p, tile.e, f, lane, ws, bias);
          xs = load_row_scale(p, tile.first + r, rows, lane);
        }
        if (!mbar_wait_warp(smem_u32(&ss.acc_full[acc]), acc_phase, abort_flag)) { ok = false; break; }
        tc_fence_after();
        uint32_t v[32];
        if (works) {
          tmem_ld32(tmem_base + acc * BN + col + (static_cast<uint32_t>(quad * 32) << 16), v);
          tmem_ld_wait();
        }
        release();
        if (works) store_rows<ACT>(p, my_stage, lane, f, tile.first + r, rows, v, ws, bias, xs);
        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
        continue;
      }
      if (tile.few != 0) {
        // lanes are channels: a warp has 32 of them, and every other 32 rows
        const int f = tile.n0 + static_cast<int>(rank) * half + quad * 32, rows = tile.row_end - tile.first;
        const bool works = f < p.N && 32 * col_half < rows;
        float ws = 0.f, bias = 0.f, xs[4] = {0.f, 0.f, 0.f, 0.f};
        if (works) {
          load_channel(p, tile.e, f, lane, ws, bias);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 32 * (col_half + 2 * i);
            xs[i] = load_row_scale(p, tile.first + r, rows - r, lane);
          }
        }
        if (!mbar_wait_warp(smem_u32(&ss.acc_full[acc]), acc_phase, abort_flag)) { ok = false; break; }
        tc_fence_after();
        if (!works) release();
        const uint32_t t_addr = tmem_base + acc * BN + (static_cast<uint32_t>(quad * 32) << 16);
#pragma unroll 1
        for (int c = col_half; works && 32 * c < rows; c += 2) {
          uint32_t v[32];
          tmem_ld32(t_addr + 32 * c, v);
          tmem_ld_wait();
          if (32 * (c + 2) >= rows) release();
          store_rows<ACT>(p, my_stage, lane, f, tile.first + 32 * c, rows - 32 * c, v, ws, bias,
                          c < 4 ? c < 2 ? xs[0] : xs[1] : c < 6 ? xs[2] : xs[3]);
        }
        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
        continue;
      }
      const int row_base = tile.row0 + quad * 32, r = row_base + lane;
      const int n_first = tile.n0 + col_half * COLS_PER_WARP;
      float xs = 0.f;
      if (r < tile.row_end) {
        const int s = source_row(p, r);
        if (s >= 0) xs = p.x_scale[s];
      }
      const bool works = n_first < p.N && row_base < tile.row_end;
      float bias[COLS_PER_WARP / 32];  // of the channels 32 c + lane
#pragma unroll
      for (int c = 0; c < COLS_PER_WARP / 32; ++c) {
        const int n = n_first + 32 * c + lane;
        bias[c] = works && n < p.N && p.bias != nullptr ? load_typed(p.bias, p.bias_type, static_cast<long long>(tile.e) * p.N + n) : 0.f;
      }
#pragma unroll
      for (int c = 0; c < COLS_PER_WARP / 32; ++c) {
        const int n = n_first + 32 * c + lane;
        st_shared_word(my_scales + 4 * (32 * c + lane), __float_as_uint(works && n < p.N ? p.w_scale[static_cast<long long>(tile.e) * p.N + n] : 0.f));
      }
      __syncwarp();
      if (!mbar_wait_warp(smem_u32(&ss.acc_full[acc]), acc_phase, abort_flag)) { ok = false; break; }
      tc_fence_after();
      if (!works) release();
      const uint32_t t_addr = tmem_base + acc * BN + col_half * COLS_PER_WARP + (static_cast<uint32_t>(quad * 32) << 16);
#pragma unroll 1
      for (int c = 0; works && c < COLS_PER_WARP / 32; ++c) {
        const int n = n_first + 32 * c;
        if (n >= p.N) break;
        uint32_t v[32];
        tmem_ld32(t_addr + 32 * c, v);
        const float b = c < 2 ? c < 1 ? bias[0] : bias[1] : c < 3 ? bias[2] : bias[3];
        tmem_ld_wait();
        if (c + 1 == COLS_PER_WARP / 32 || n + 32 >= p.N) release();
        store_columns<ACT>(p, my_stage, lane, row_base, tile.row_end, n, v, xs, my_scales + 128 * c, b);
      }
      if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
    }
    if (!ok && lane == 0 && p.status) atomicCAS(p.status, ST_OK, ST_TIMEOUT_EPILOGUE);
  }

  if (*abort_flag != 0) {
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  // barriers that the lanes of a warp may reach one by one: the MMA role is one lane's
  tc_fence_before();
  block_sync_diverged();
  cluster_sync_diverged();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * BN);
  }
}


}  // namespace i8
}  // namespace smoe
