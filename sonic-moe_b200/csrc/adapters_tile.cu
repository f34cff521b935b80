// Low-rank adapters: the kernels for tiles of rows (the formulas are in adapters.cuh).
#include "adapters.cuh"

namespace smoe {
namespace adapters {

// ----------------------------------------------------------------------------------------------
// tiles
// ----------------------------------------------------------------------------------------------
// Stages of 64 columns, `kStages` of them in turn: RP rows of a (or 64 of b) for the block, and each warp's 16 rows of x (or base), which it brings in
// itself.  ALIGNED: rows of 128 bytes by asynchronous copies; the halves of odd ones trade places, so that eight lanes of a load meet all
// banks.  Otherwise rows of x and base come in by the nine 16-byte blocks that hold them and are put in place on the way out of shared
// memory, weights on the way in.
template <int RP, bool ALIGNED>
struct Tile {
  static constexpr int kCols = 64, kStages = 3;
  static constexpr int kPitch = ALIGNED ? 128 : 144, kWarpBytes = 16 * kPitch, kWeightBytes = RP * 128;
  static constexpr int kOutPitch = 160;  // of a row of results on its way out: eight columns of the stage before, 64, and what a shifted load may touch
  // of a warp: s (leading bits, the rest), later its results
  static constexpr int kOwnBytes = 64 * RP > 16 * kOutPitch || ALIGNED ? 64 * RP : 16 * kOutPitch;
  static size_t smem(int warps) {
    const size_t stages = kStages * static_cast<size_t>(kWeightBytes + warps * kWarpBytes), part = sizeof(float) * 16 * warps * kPartPitch<RP>;
    return (stages > part ? stages : part) + static_cast<size_t>(warps) * kOwnBytes + sizeof(float) * 16 * warps;
  }
};
// place of the 16-byte block `k` of row `row`
__device__ __forceinline__ int swizzled(int row, int k) { return 16 * (k ^ ((row & 1) << 2)); }
// place of block `k` of row `row` among rows of RP 16-bit values
template <int RP>
__device__ __forceinline__ int weight_place(int row, int k) { return 2 * RP * row + (RP >= 64 ? swizzled(row, k) : 16 * k); }

__device__ __forceinline__ void store_cluster(uint32_t addr, uint2 v) {
  asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(v.x), "r"(v.y) : "memory");
}

// A warp's 16 rows on their way into shared memory: lane l has block l % 8 (and l % 8 = 0 the ninth) of the rows l / 8, + 4, + 8, + 12.
template <bool ALIGNED, int PITCH>
struct RowCopy {
  const char* row[4];  // the row's first block, or nullptr
  long long bytes[4];  // up to the row's end
  __device__ __forceinline__ void set(const char* rows, long long ld, int width, int tokens /* of row `lane` % 16 */) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int token = __shfl_sync(0xffffffffu, tokens, (lane >> 3) + 4 * i);
      const char* p = rows + token * ld;
      const int off = ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
      row[i] = token >= 0 && rows != nullptr ? p - off : nullptr;
      bytes[i] = off + 2ll * width;
    }
  }
  // columns 64 stage and on; zeros behind the row's end
  __device__ __forceinline__ void fetch(char* to, int stage, const void* some /* an address for copies of nothing */) const {
    const int lane = threadIdx.x & 31, k = lane & 7;
    const char* none = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(some) & ~static_cast<uintptr_t>(15));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = (lane >> 3) + 4 * i;
      const long long at = 128ll * stage + 16 * k;
      const bool has = row[i] != nullptr && at < bytes[i];
      cp_async16(smem_u32(to + r * PITCH + (ALIGNED ? swizzled(r, k) : 16 * k)), has ? row[i] + at : none, has ? 16 : 0);
      if (!ALIGNED && k == 0) {
        const bool more = row[i] != nullptr && at + 128 < bytes[i];
        cp_async16(smem_u32(to + r * PITCH + 128), more ? row[i] + at + 128 : none, more ? 16 : 0);
      }
    }
  }
};
// eight columns from 8 k of a stage on, of row `r`, which begins `off` bytes into its first block; `left`: columns of the row from there on
template <bool ALIGNED, int PITCH>
__device__ __forceinline__ uint4 staged_row(const char* from, int r, int k, int off, int left) {
  if (ALIGNED) return *reinterpret_cast<const uint4*>(from + r * PITCH + swizzled(r, k));
  return in_place8(from + r * PITCH + 16 * k, off, left);
}

// One block of rows of weights, RP or 64 of them, 64 or RP columns each, into shared memory by all threads.
template <bool ALIGNED, class Place>
__device__ __forceinline__ void fetch_weights(char* to, const char* from, int width /* of a row in memory */, int rows, int rows_left, int col, int cols, Place place) {
  const int per = cols / 8;
  for (int i = threadIdx.x; i < rows * per; i += blockDim.x) {
    const int row = i / per, k = i % per, c = col + 8 * k;
    const char* p = from + 2ll * width * row;
    const bool has = row < rows_left && c < width;
    if (ALIGNED) cp_async16(smem_u32(to + place(row, k)), has ? p + 2ll * c : from, has ? 16 : 0);
    else *reinterpret_cast<uint4*>(to + place(row, k)) = load8<false>(p, has ? c : width, width);
  }
}

// The blocks' parts (`pitch` floats to a row) added, scaled and split, each block's share of the rows, and written to all blocks: columns 4q .. of a row's
// leading bits at `place(row, q)`, the rest `rest` bytes behind them, the inverse of its factor in `inverses`.  Between two meetings of the
// cluster.
template <class T, int RP, int PITCH, class Place>
__device__ __forceinline__ void share_sums(const Params& p, const float* part, int tile_rows, int share, float scale, float* inverses, Place place, uint32_t rest) {
  constexpr int Q = RP / 4;  // threads of a row, four columns each
  const int mine = tile_rows / p.cluster;
  for (int first_of = 0; first_of < mine * Q; first_of += blockDim.x) {  // (all threads, for the shuffles)
    const int i = first_of + threadIdx.x;
    const bool live = i < mine * Q;
    const int row = share * mine + (live ? i / Q : 0), q = i % Q;
    float f[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = 0; k < p.cluster; ++k) {
      const float4 v = load_cluster(map_to_cta(smem_u32(part + row * PITCH + 4 * q), k));
      f[0] += v.x; f[1] += v.y; f[2] += v.z; f[3] += v.w;
    }
    float most = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] *= scale;
      most = fmaxf(most, fabsf(f[j]));
    }
    if (std::is_same<T, __half>::value) {
#pragma unroll
      for (int o = 1; o < Q; o *= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    }
    const float factor = factor_of<T>(most);
    uint2 l, r;
    split2<T>(f[0] * factor, f[1] * factor, l.x, r.x);
    split2<T>(f[2] * factor, f[3] * factor, l.y, r.y);
    if (live) {
      const uint32_t to = place(row, q);
      for (int k = 0; k < p.cluster; ++k) {
        store_cluster(map_to_cta(to, k), l);
        store_cluster(map_to_cta(to + rest, k), r);
        if (std::is_same<T, __half>::value && q == 0)
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(map_to_cta(smem_u32(inverses + row), k)), "f"(inverse_of<T>(factor)) : "memory");
      }
    }
  }
}

// Bound by how a block's rows come and go, 128 bytes at a time in two phases one after the other: 8192 tokens, 4096 x 4096, 8 adapters, bf16 with a base 41 us
// at rank 16 (4.9 TB/s; DRAM 46 % busy in a single cold launch), 47 at rank 32; a kernel that only reads and writes rows in this order (three
// stages of 128 bytes of each, clusters of four) takes 17 + 27 us for the two halves.  Rows that start anywhere: 2048 tokens of 100 adapters, 4097 x 4095, rank 32 66
// us, of 27 on 4096 x 4096: weights go through registers, without the ring's lead.
template <class T, int RP, bool ALIGNED>
__global__ void __launch_bounds__(32 * kWarps, RP <= 64 ? 2 : 1) tile_kernel(const Params p) {
  release_next();
  wait_for_previous();
  using Ti = Tile<RP, ALIGNED>;
  extern __shared__ __align__(128) char smem_tile[];
  constexpr int COLS = Ti::kCols, STAGES = Ti::kStages, PITCH = Ti::kPitch, NT = RP / 8, C = COLS / 32, K = Steps<RP>::K, L = Steps<RP>::L;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, warps = blockDim.x / 32, tile_rows = 16 * warps;
  const int tile = blockIdx.x / p.cluster, share = blockIdx.x - tile * p.cluster;
  Others others;
  others.begin(p, blockIdx.x * (blockDim.x / 32) + warp);
  const int4 what = tile_of(p, tile, tile_rows);
  if (what.x < 0) {  // (the cluster's blocks all see the same)
    others.finish(p);
    return;
  }
  const int e = what.x, my_row = what.y + 16 * warp + (lane & 15);
  const int gathered = my_row < what.z ? gathered_of(p, my_row) : -1;
  const bool any = __any_sync(0xffffffffu, gathered >= 0);
  const int row_of = gathered >= 0 ? p.reverse[gathered] : -1;  // what is read of a token does not wait for the check that the row is still its own
  const int stage_bytes = Ti::kWeightBytes + warps * Ti::kWarpBytes;
  const auto weights_in = [&](int stage) { return smem_tile + stage % STAGES * stage_bytes; };
  const auto rows_in = [&](int stage) { return weights_in(stage) + Ti::kWeightBytes + warp * Ti::kWarpBytes; };
  const size_t ring = max(static_cast<size_t>(STAGES) * stage_bytes, sizeof(float) * tile_rows * kPartPitch<RP>);
  char* own = smem_tile + ring;                                                // [warp][lead: 16 x RP, rest: 16 x RP]
  float* inverses = reinterpret_cast<float*>(own + warps * Ti::kOwnBytes);     // [tile_rows]
  const auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
  const auto range = [&](int all, int& first, int& end) {
    first = static_cast<int>(static_cast<long long>(all) * share / p.cluster);
    end = static_cast<int>(static_cast<long long>(all) * (share + 1) / p.cluster);
  };

  // s, of this block's columns of x
  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  {
    int first, end;
    range((p.H + COLS - 1) / COLS, first, end);
    const char* a = p.a + static_cast<long long>(e) * p.r * p.H * 2;
    RowCopy<ALIGNED, PITCH> x;
    x.set(p.x, p.x_ld, p.H, gathered);
    const auto fetch = [&](int stage) {
      if (stage < end) {
        if (any) x.fetch(rows_in(stage), stage, p.x);
        fetch_weights<ALIGNED>(weights_in(stage), a, p.H, RP, p.r, COLS * stage, COLS, [](int row, int k) { return 128 * row + swizzled(row, k); });
      }
      commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch(first + i);
    const int t0 = __shfl_sync(0xffffffffu, gathered, g), t1 = __shfl_sync(0xffffffffu, gathered, g + 8);
    const int o0 = ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(p.x + t0 * p.x_ld) & 15), o1 = ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(p.x + t1 * p.x_ld) & 15);
    for (int stage = first; stage < end; ++stage) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      __syncthreads();  // the stage is there for all, and the one whose place the next takes has been read
      fetch(stage + STAGES - 1);
      if (!any) continue;
      const char* xs = rows_in(stage);
      const char* ws = weights_in(stage);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int left = p.H - (COLS * stage + 32 * c + 8 * t);
        const uint4 x0 = staged_row<ALIGNED, PITCH>(xs, g, 4 * c + t, o0, left), x1 = staged_row<ALIGNED, PITCH>(xs, g + 8, 4 * c + t, o1, left);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 w = *reinterpret_cast<const uint4*>(ws + 128 * (8 * j + g) + swizzled(g, 4 * c + t));
          mma<T>(acc[j], x0.x, x1.x, x0.y, x1.y, w.x, w.y);
          mma<T>(acc[j], x0.z, x1.z, x0.w, x1.w, w.z, w.w);
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
  }

  // the blocks add their parts, each for a share of the rows, and give all of them the sums
  constexpr int PART = kPartPitch<RP>;
  float* part = reinterpret_cast<float*>(smem_tile);  // [tile_rows][PART]
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    float* to = part + (16 * warp + g) * PART + 8 * j + 2 * t;
    *reinterpret_cast<float2*>(to) = make_float2(acc[j][0], acc[j][1]);
    *reinterpret_cast<float2*>(to + 8 * PART) = make_float2(acc[j][2], acc[j][3]);
  }
  cluster_sync_all();
  share_sums<T, RP, PART>(p, part, tile_rows, share, p.scale != nullptr ? p.scale[e] : 1.f, inverses,
                          [&](int row, int q) { return smem_u32(own + row / 16 * Ti::kOwnBytes) + weight_place<RP>(row % 16, q / 2) + 8 * (q & 1); }, 32 * RP);
  cluster_sync_all();

  // this block's columns of out
  int first, end;
  range((p.N + COLS - 1) / COLS, first, end);
  const char* b = p.b + static_cast<long long>(e) * p.N * p.r * 2;
  const int tokens = row_of == my_row ? gathered : -1;
  const bool writes = __any_sync(0xffffffffu, tokens >= 0);
  const int t0 = __shfl_sync(0xffffffffu, tokens, g), t1 = __shfl_sync(0xffffffffu, tokens, g + 8);
  RowCopy<ALIGNED, PITCH> base;
  base.set(p.base, p.base_ld, p.N, tokens);
  const auto fetch = [&](int stage) {
    if (stage < end) {
      if (writes && p.base != nullptr) base.fetch(rows_in(stage), stage, p.x);
      fetch_weights<ALIGNED>(weights_in(stage), b + 2ll * COLS * stage * p.r, p.r, COLS, p.N - COLS * stage, 0, RP, weight_place<RP>);
    }
    commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(first + i);
  uint32_t lead[K][4], rest[K][4];
  {
    const char* mine = own + warp * Ti::kOwnBytes;
#pragma unroll
    for (int l = 0; l < L; ++l) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // rows g and g + 8
        if constexpr (RP == 16) {
          const uint2 u = *reinterpret_cast<const uint2*>(mine + weight_place<RP>(g + 8 * h, 0) + 8 * t), v = *reinterpret_cast<const uint2*>(mine + 32 * RP + weight_place<RP>(g + 8 * h, 0) + 8 * t);
          lead[0][h] = u.x; lead[0][2 + h] = u.y;
          rest[0][h] = v.x; rest[0][2 + h] = v.y;
        } else {
          const uint4 u = *reinterpret_cast<const uint4*>(mine + weight_place<RP>(g + 8 * h, 4 * l + t)), v = *reinterpret_cast<const uint4*>(mine + 32 * RP + weight_place<RP>(g + 8 * h, 4 * l + t));
          lead[2 * l][h] = u.x; lead[2 * l][2 + h] = u.y; lead[2 * l + 1][h] = u.z; lead[2 * l + 1][2 + h] = u.w;
          rest[2 * l][h] = v.x; rest[2 * l][2 + h] = v.y; rest[2 * l + 1][h] = v.z; rest[2 * l + 1][2 + h] = v.w;
        }
      }
    }
  }
  const float i0 = std::is_same<T, __half>::value ? inverses[16 * warp + g] : 1.f, i1 = std::is_same<T, __half>::value ? inverses[16 * warp + g + 8] : 1.f;
  const int o0 = ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(p.base + t0 * p.base_ld) & 15), o1 = ALIGNED ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(p.base + t1 * p.base_ld) & 15);
  __syncwarp();  // s has been read: the results may lie there
  char* results = own + warp * Ti::kOwnBytes;
  for (int stage = first; stage < end; ++stage) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncthreads();
    fetch(stage + STAGES - 1);
    if (!writes) continue;
    const char* bs = rows_in(stage);
    const char* ws = weights_in(stage);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int n0 = COLS * stage + kGroup * i;
      float c[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.f;
        const int row = kGroup * i + out_column(g, j);
#pragma unroll
        for (int l = 0; l < L; ++l) {
          uint4 w = make_uint4(0u, 0u, 0u, 0u);
          if constexpr (RP == 16) {
            const uint2 h = *reinterpret_cast<const uint2*>(ws + weight_place<RP>(row, 0) + 8 * t);
            w.x = h.x;
            w.y = h.y;
          } else {
            w = *reinterpret_cast<const uint4*>(ws + weight_place<RP>(row, 4 * l + t));
          }
          step<T, RP>(c[j], lead, rest, l, w);
        }
      }
      uint4 b0 = make_uint4(0u, 0u, 0u, 0u), b1 = b0;
      if (p.base != nullptr) {
        const int left = p.N - (n0 + 8 * t);
        b0 = staged_row<ALIGNED, PITCH>(bs, g, 4 * i + t, o0, left);
        b1 = staged_row<ALIGNED, PITCH>(bs, g + 8, 4 * i + t, o1, left);
      }
      const uint4 r0 = sum_row<T>(b0, c, 0, i0), r1 = sum_row<T>(b1, c, 1, i1);
      if (ALIGNED) {
        const int n = n0 + 8 * t;
        if (t0 >= 0 && n < p.N) __stcs(reinterpret_cast<uint4*>(p.out + t0 * p.out_ld + 2ll * n), r0);
        if (t1 >= 0 && n < p.N) __stcs(reinterpret_cast<uint4*>(p.out + t1 * p.out_ld + 2ll * n), r1);
      } else {
        *reinterpret_cast<uint4*>(results + g * Ti::kOutPitch + 16 + 64 * i + 16 * t) = r0;
        *reinterpret_cast<uint4*>(results + (g + 8) * Ti::kOutPitch + 16 + 64 * i + 16 * t) = r1;
      }
    }
    if (!ALIGNED) {
      __syncwarp();
      put_shifted(p, results, Ti::kOutPitch, tokens, COLS * stage, COLS * first, min(COLS * end, p.N), stage + 1 == end);
      __syncwarp();
      if (lane < 16) *reinterpret_cast<uint4*>(results + lane * Ti::kOutPitch) = *reinterpret_cast<const uint4*>(results + lane * Ti::kOutPitch + 128);
      __syncwarp();
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  others.finish(p);
}

// ----------------------------------------------------------------------------------------------
// tiles by tcgen05.mma
// ----------------------------------------------------------------------------------------------
// A tile of 128 rows: s = x a^T in tensor memory, 64 columns of x to a stage; then out's columns, 64 to a stage, the leading bits and the rest of s one after
// the other times the same weights.  All threads bring in what a stage needs by asynchronous copies into the layout that the matrix
// instructions read (rows of 128 bytes, block k of row i in place k ^ (i mod 8)); one thread issues the instructions.  A stage of the second
// product is on the tensor core while the last one's 32 rows by 32 columns of each warp are added to base and go out.
// WIDE: rows of base and out are whole 16-byte pieces.  Otherwise each half of the warps has a run of columns of its own, so that what of a row's results
// does not fill a 16-byte block of out waits in the row's thread for the next ones; base comes in by the blocks that hold it.
// 8192 tokens, 4096 x 4096, 8 adapters, rank 64 56 us (3.7 TB/s, 153 TFLOP/s; DRAM 34 % and the tensor pipe 14 % busy: it is the phases one after the other
// that take the time), 4095 columns of out 83; 32768 tokens 182 us, 4.5 TB/s.
// Of a block's time 30 and 45 thousand cycles are the two products, at the rate at which their rows come and go, 9 the sums' way over the cluster, 5 the
// start.  Rank 128, one block to an SM for its s: 119 us.
template <int RP, bool WIDE>
struct Tensor {
  static constexpr int kAtoms = RP > 64 ? 2 : 1;             // 64 columns of s each
  static constexpr int kWeights = 8192 * kAtoms;             // bytes of a stage's weights: up to 128 rows of a, 64 of b in each atom
  static constexpr int kX = 128 * 128, kS = kAtoms * 16384;  // a stage of x; leading bits of s, or the rest
  static constexpr int kBasePitch = WIDE ? 64 : 80, kBaseWarp = 32 * kBasePitch + (WIDE ? 0 : 16);
  static constexpr int kFirst = 3, kSecond = WIDE ? 3 : 2;   // stages in turn
  static constexpr int kFirstStage = kWeights + kX, kSecondStage = (kWeights + kWarps * kBaseWarp + 1023) / 1024 * 1024;  // on 1024-byte boundaries
  static constexpr int kPart = RP + 4;                       // floats of a row of the block's part, for lanes that write four at a time in rows of their own
  // stages of the second product whose place the part leaves free
  static constexpr int kPartBytes = 128 * kPart * static_cast<int>(sizeof(float));
  static constexpr int kFree = kSecond - (kPartBytes + kSecondStage - 1) / kSecondStage, kEarly = kFree < 0 ? 0 : kFree < kSecond ? kFree : kSecond - 1;
  static constexpr size_t max3(size_t a, size_t b, size_t c) { return a > b ? (a > c ? a : c) : b > c ? b : c; }
  static constexpr size_t kRing = (max3(kFirst * kFirstStage, kSecond * kSecondStage, kPartBytes) + 1023) / 1024 * 1024;
  static constexpr size_t kSmem = kRing + 2 * kS + sizeof(float) * 128 + 1024;  // (1024 for the alignment)
  static_assert(RP * 128 <= kWeights, "a stage of a");
};
template <class T>
__device__ __forceinline__ constexpr uint32_t instruction(int N) {  // 128 rows, N columns, fp32 sums, both operands' columns run along their rows
  return (1u << 4) | (std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u) | (static_cast<uint32_t>(N >> 3) << 17) | (8u << 24);
}

template <class T, int RP, bool WIDE>
__global__ void __launch_bounds__(32 * kWarps, RP <= 64 ? 2 : 1) tensor_kernel(const Params p) {
  wait_for_previous();
  using Te = Tensor<RP, WIDE>;
  extern __shared__ char smem_any[];
  char* smem = smem_any + ((1024 - (smem_u32(smem_any) & 1023)) & 1023);
  char* s_in = smem + Te::kRing;                                        // leading bits, the rest
  float* inverses = reinterpret_cast<float*>(s_in + 2 * Te::kS);        // [128]
  __shared__ __align__(8) uint64_t done_first[Te::kFirst], done_second[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  const int lane = threadIdx.x & 31, warp = warp_index(), quad = warp & 3, half = warp >> 2;
  const int tile = blockIdx.x / p.cluster, share = blockIdx.x - tile * p.cluster;
  Others others;
  others.begin(p, blockIdx.x * (blockDim.x / 32) + warp);
  const int4 what = tile_of(p, tile, 128);
  if (what.x < 0) {  // (the cluster's blocks all see the same)
    others.finish(p);
    return;
  }
  const int e = what.x, row0 = what.y;
  if (threadIdx.x == 0) {
    for (int i = 0; i < Te::kFirst; ++i) mbar_init(smem_u32(&done_first[i]), 1);
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&done_second[i]), 1);
    gave_up = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), 128);
    tmem_relinquish();
  }
  // the row of results that this thread has, and whether it is still its token's
  const int my_row = row0 + 32 * quad + lane;
  const int gathered = my_row < what.z ? gathered_of(p, my_row) : -1;
  const int row_of = gathered >= 0 ? p.reverse[gathered] : -1;
  const auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
  const auto range = [&](int all, int& first, int& end) {
    first = static_cast<int>(static_cast<long long>(all) * share / p.cluster);
    end = static_cast<int>(static_cast<long long>(all) * (share + 1) / p.cluster);
  };
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  release_next();  // not before: a next kernel that waits for this one with all of the tensor memory in hand would leave this block none
  const uint32_t tmem = tmem_slot;
  volatile int* abort_flag = &gave_up;

  // this block's columns of out: of stage i, 32 from `column(0, i)` on and 32 from `column(1, i)` on
  int first, middle, end;  // in groups of 32
  if (WIDE) {
    range((p.N + 63) / 64, first, end);
    first *= 2;
    end *= 2;
    middle = first + (end - first) / 2;
  } else {
    range((p.N + 31) / 32, first, end);
    middle = first + (end - first + 1) / 2;
  }
  const int stages = middle - first;
  const auto column = [&](int of, int i) { return WIDE ? 32 * (first + 2 * i + of) : 32 * ((of == 0 ? first : middle) + i); };
  const auto column_end = [&](int of) { return min(p.N, 32 * (WIDE || of != 0 ? end : middle)); };
  const char* b = p.b + static_cast<long long>(e) * p.N * p.r * 2;
  const int token = row_of == my_row ? gathered : -1;
  const bool writes = __any_sync(0xffffffffu, token >= 0);
  const auto slot = [&](int i) { return smem + (i + Te::kSecond - Te::kEarly) % Te::kSecond * Te::kSecondStage; };
  const auto base_slot = [&](int i) { return slot(i) + Te::kWeights + warp * Te::kBaseWarp; };
  const char* none = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(p.x) & ~static_cast<uintptr_t>(15));
  const int mine_end = column_end(half);
  const auto fetch_second = [&](int i) {
    if (i < stages) {
      char* to = slot(i);
      constexpr int PER = RP / 8;  // blocks of a row
#pragma unroll
      for (int j = 0; j < 64 * PER; j += 32 * kWarps) {
        const int at = j + threadIdx.x, row = at / PER, k = at % PER;
        if (64 * PER < 32 * kWarps && at >= 64 * PER) continue;
        const int n = column(row >> 5, i) + (row & 31);
        const bool has = n < column_end(row >> 5) && 8 * k < p.r;
        cp_async16(smem_u32(to + (k >> 3) * 8192 + row * 128 + (((k & 7) ^ (row & 7)) << 4)), has ? b + 2ll * n * p.r + 16 * k : p.b, has ? 16 : 0);
      }
      if (writes && p.base != nullptr) {
        char* rows = base_slot(i);
        const int c0 = column(half, i);
        if (WIDE) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int row = (lane >> 2) + 8 * j, k = lane & 3, t = __shfl_sync(0xffffffffu, token, row);
            const bool has = t >= 0 && c0 + 8 * k < mine_end;
            cp_async16(smem_u32(rows + row * 64 + ((k ^ (row >> 1 & 3)) << 4)), has ? p.base + t * p.base_ld + 2ll * c0 + 16 * k : none, has ? 16 : 0);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 5; ++j) {
            const int at = lane + 32 * j, row = at / 5, k = at % 5, t = __shfl_sync(0xffffffffu, token, row);
            const char* of = p.base + t * p.base_ld;
            const int off = static_cast<int>(reinterpret_cast<uintptr_t>(of) & 15);
            const bool has = t >= 0 && c0 < mine_end && 2ll * c0 + 16 * k < 2ll * p.N + off;
            cp_async16(smem_u32(rows + row * 80 + 16 * k), has ? of - off + 2ll * c0 + 16 * k : none, has ? 16 : 0);
          }
        }
      }
    }
    commit();
  };

  // s, of this block's columns of x
  {
    int first, end;
    range((p.H + 63) / 64, first, end);
    const char* a = p.a + static_cast<long long>(e) * p.r * p.H * 2;
    // of rows threadIdx / 8, + 32, + 64, + 96 this thread has block threadIdx % 8
    const int k = threadIdx.x & 7, r0 = threadIdx.x >> 3;
    const char* x_row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int token = row0 + r0 + 32 * i < what.z ? gathered_of(p, row0 + r0 + 32 * i) : -1;
      x_row[i] = token >= 0 ? p.x + token * p.x_ld + 16 * k : nullptr;
    }
    const auto slot = [&](int stage) { return smem + (stage - first) % Te::kFirst * Te::kFirstStage; };
    const auto fetch = [&](int stage) {
      if (stage < end) {
        char* to = slot(stage);
        const bool in = 64 * stage + 8 * k < p.H;
        const int place = (k ^ (r0 & 7)) << 4;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          cp_async16(smem_u32(to + Te::kWeights + (r0 + 32 * i) * 128 + place), in && x_row[i] != nullptr ? x_row[i] + 128ll * stage : p.x, in && x_row[i] != nullptr ? 16 : 0);
#pragma unroll
        for (int i = 0; i < (RP + 31) / 32; ++i) {
          const int row = r0 + 32 * i;
          const bool has = in && row < p.r;
          if (row < RP) cp_async16(smem_u32(to + row * 128 + place), has ? a + 2ll * row * p.H + 128ll * stage + 16 * k : p.a, has ? 16 : 0);
        }
      }
      commit();
    };
    for (int i = 0; i < Te::kFirst - 1; ++i) fetch(first + i);
    const bool issues = warp == 0 && elect_one();
    for (int stage = first; stage < end; ++stage) {
      asm volatile("cp.async.wait_group %0;" ::"n"(Te::kFirst - 2) : "memory");
      fence_proxy_async_smem();
      __syncthreads();
      const int i = stage - first;
      if (issues) {
        tc_fence_after();
        const uint64_t w = make_smem_desc(smem_u32(slot(stage)), 16, 1024), x = make_smem_desc(smem_u32(slot(stage) + Te::kWeights), 16, 1024);
#pragma unroll
        for (int step = 0; step < 4; ++step) umma_bf16(tmem, x + 2 * step, w + 2 * step, instruction<T>(RP), i > 0 || step > 0);
        umma_commit(smem_u32(&done_first[i % Te::kFirst]));
      }
      // the stage before has been read: its place is the next one's
      if (i > 0) mbar_wait_warp(smem_u32(&done_first[(i - 1) % Te::kFirst]), (i - 1) / Te::kFirst & 1, abort_flag);
      fetch(stage + Te::kFirst - 1);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    const int last = end - first - 1;
    if (last >= 0) mbar_wait_warp(smem_u32(&done_first[last % Te::kFirst]), last / Te::kFirst & 1, abort_flag);
    tc_fence_after();
    __syncthreads();
    for (int i = 0; i < Te::kEarly; ++i) fetch_second(i);  // on their way while the blocks add their parts
    // this block's part: a row to a thread, the columns in two halves where there are 32 or more
    float* part = reinterpret_cast<float*>(smem);
    constexpr int COLS = RP >= 32 ? RP / 2 : RP;
    if (RP >= 32 || half == 0) {
#pragma unroll
      for (int c = 0; c < COLS; c += 16) {
        uint32_t v[16];
        const int col = half * COLS + c;
        if (last >= 0) {
          tmem_ld16(tmem + col + (static_cast<uint32_t>(quad * 32) << 16), v);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (auto& x : v) x = 0u;
        }
#pragma unroll
        for (int j = 0; j < 16; j += 4)
          *reinterpret_cast<uint4*>(part + (32 * quad + lane) * Te::kPart + col + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
      }
    }
    tc_fence_before();
    cluster_sync_all();
    share_sums<T, RP, Te::kPart>(p, part, 128, share, p.scale != nullptr ? p.scale[e] : 1.f, inverses, [&](int row, int q) {
      return smem_u32(s_in) + (q >> 4) * 16384 + row * 128 + (((q >> 1 & 7) ^ (row & 7)) << 4) + 8 * (q & 1);
    }, Te::kS);
    fence_proxy_async_smem();
    cluster_sync_all();
    fence_proxy_async_smem();
    tc_fence_after();
  }

  for (int i = Te::kEarly; i < Te::kSecond - 1; ++i) fetch_second(i);
  const float inverse = std::is_same<T, __half>::value ? inverses[32 * quad + lane] : 1.f;
  const bool issues = warp == 0 && elect_one();
  uint4 left_over = make_uint4(0u, 0u, 0u, 0u);  // (not WIDE) the row's last eight results
  // the results of stage i, out
  const auto put = [&](int i) {
    mbar_wait_warp(smem_u32(&done_second[i & 1]), i >> 1 & 1, abort_flag);
    tc_fence_after();
    uint32_t v[32];
    tmem_ld32(tmem + 64 * (i & 1) + 32 * half + (static_cast<uint32_t>(quad * 32) << 16), v);
    tmem_ld_wait();
    tc_fence_before();
    const int c0 = column(half, i);
    if (!writes || c0 >= mine_end) return;
    char* rows = base_slot(i);
    char* mine = rows + lane * Te::kBasePitch;
    uint32_t base[20];
#pragma unroll
    for (int k = 0; k < (WIDE ? 4 : 5); ++k) {
      uint4 q = make_uint4(0u, 0u, 0u, 0u);
      if (p.base != nullptr) q = *reinterpret_cast<const uint4*>(mine + (WIDE ? (k ^ (lane >> 1 & 3)) << 4 : 16 * k));
      base[4 * k] = q.x; base[4 * k + 1] = q.y; base[4 * k + 2] = q.z; base[4 * k + 3] = q.w;
    }
    if (!WIDE) {
      const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p.base + token * p.base_ld) & 15);
#pragma unroll
      for (int k = 0; k < 18; ++k) base[k] = off & 8 ? base[k + 2] : base[k];
#pragma unroll
      for (int k = 0; k < 17; ++k) base[k] = off & 4 ? base[k + 1] : base[k];
#pragma unroll
      for (int k = 0; k < 16; ++k) base[k] = __funnelshift_r(base[k], base[k + 1], 8 * (off & 2));
      *reinterpret_cast<uint4*>(mine) = left_over;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack<T>(base[4 * k + j]);
        o[j] = pack<T>(fmaf(__uint_as_float(v[8 * k + 2 * j]), inverse, f.x), fmaf(__uint_as_float(v[8 * k + 2 * j + 1]), inverse, f.y));
      }
      *reinterpret_cast<uint4*>(mine + (WIDE ? (k ^ (lane >> 1 & 3)) << 4 : 16 + 16 * k)) = make_uint4(o[0], o[1], o[2], o[3]);
      if (!WIDE && k == 3) left_over = make_uint4(o[0], o[1], o[2], o[3]);
    }
    __syncwarp();
    const bool last = c0 + 32 >= mine_end;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = (lane >> 2) + 8 * j, k = lane & 3, t = __shfl_sync(0xffffffffu, token, row);
      if (t < 0) continue;
      char* out = p.out + t * p.out_ld;
      if (WIDE) {
        if (c0 + 8 * k < mine_end)
          __stcs(reinterpret_cast<uint4*>(out + 2ll * c0 + 16 * k), *reinterpret_cast<const uint4*>(rows + row * 64 + ((k ^ (row >> 1 & 3)) << 4)));
      } else {
        const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(out) & 15) / 2;  // values of out's first block in front of the row
        put_block(p, out, rows + row * 80, c0, k, shift, column(half, 0), mine_end);
        if (last && k == 3 && shift > 0) put_block(p, out, rows + row * 80, c0, 4, shift, column(half, 0), mine_end);
      }
    }
    __syncwarp();
  };
  for (int i = 0; i < stages; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(Te::kSecond - 2) : "memory");
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    if (issues) {
      tc_fence_after();
      const uint64_t w = make_smem_desc(smem_u32(slot(i)), 16, 1024), s = make_smem_desc(smem_u32(s_in), 16, 1024);
      const uint32_t to = tmem + 64 * (i & 1);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int step = 0; step < RP / 16; ++step)
          umma_bf16(to, s + (h * Te::kS + (step >> 2) * 16384 + (step & 3) * 32) / 16, w + ((step >> 2) * 8192 + (step & 3) * 32) / 16, instruction<T>(64), h > 0 || step > 0);
      }
      umma_commit(smem_u32(&done_second[i & 1]));
    }
    if (i > 0) put(i - 1);
    fetch_second(i + Te::kSecond - 1);
  }
  if (stages > 0) put(stages - 1);
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  others.finish(p);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 128);
  }
  if (threadIdx.x == 0 && gave_up != 0 && p.status != nullptr) atomicCAS(p.status, static_cast<int>(SMOE_ST_OK), static_cast<int>(SMOE_ST_TIMEOUT_MMA));
}

// ----------------------------------------------------------------------------------------------
// launches
// ----------------------------------------------------------------------------------------------
template <class T, int RP, bool WIDE>
static int launch_tile(const Params& p, int warps, long long blocks, cudaStream_t st) {
  static PerDeviceFlag configured;
  const int dev = current_device();
  if (dev < 0) return SMOE_ERR_DRIVER;
  if (!configured.test(dev)) {
    if (cudaFuncSetAttribute(tile_kernel<T, RP, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Tile<RP, WIDE>::smem(kWarps))) != cudaSuccess)
      return SMOE_ERR_LAUNCH;
    configured.set(dev);
  }
  return launched(launch_chained(tile_kernel<T, RP, WIDE>, dim3(static_cast<unsigned>(blocks)), 32 * warps, Tile<RP, WIDE>::smem(warps), st, p.cluster, p));
}
template <class T, int RP, bool WIDE>
static int launch_tensor(const Params& p, long long blocks, cudaStream_t st) {
  static PerDeviceFlag configured;
  const int dev = current_device();
  if (dev < 0) return SMOE_ERR_DRIVER;
  constexpr size_t smem = Tensor<RP, WIDE>::kSmem;
  if (!configured.test(dev)) {
    if (cudaFuncSetAttribute(tensor_kernel<T, RP, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess) return SMOE_ERR_LAUNCH;
    configured.set(dev);
  }
  return launched(launch_chained(tensor_kernel<T, RP, WIDE>, dim3(static_cast<unsigned>(blocks)), 32 * kWarps, smem, st, p.cluster, p));
}
template <class T, int RP>
static int launch_rank(const Params& p, bool wide_in, bool wide_out, int warps, long long blocks, cudaStream_t st) {
  // (tcgen05 / mma.sync, us, 8192 tokens, 4096 x 4096, 8 adapters, rank 16: 59 / 46, 32: 60 / 50, 64: 63.5 / 64, 128: 121 / 129; 4095 columns of out, rank 16:
  // 84 / 86, 64: 88 / 123, 128: 184 / 390; 2048 tokens of one adapter, rank 64: 30 / 36)
  if (wide_in && warps == kWarps) {
    if (!wide_out) return launch_tensor<T, RP, false>(p, blocks, st);
    if constexpr (RP >= 64) return launch_tensor<T, RP, true>(p, blocks, st);
  }
  return wide_in && wide_out ? launch_tile<T, RP, true>(p, warps, blocks, st) : launch_tile<T, RP, false>(p, warps, blocks, st);
}
template <class T>
static int launch_type(const Params& p, bool wide_in, bool wide_out, int warps, long long blocks, cudaStream_t st) {
  switch (padded_rank(p.r)) {
    case 16: return launch_rank<T, 16>(p, wide_in, wide_out, warps, blocks, st);
    case 32: return launch_rank<T, 32>(p, wide_in, wide_out, warps, blocks, st);
    case 64: return launch_rank<T, 64>(p, wide_in, wide_out, warps, blocks, st);
    default: return launch_rank<T, 128>(p, wide_in, wide_out, warps, blocks, st);
  }
}
int launch_tiles(const Params& p, int dtype, bool wide_in, bool wide_out, int warps, long long blocks, cudaStream_t st) {
  return dtype == SMOE_BF16 ? launch_type<__nv_bfloat16>(p, wide_in, wide_out, warps, blocks, st) : launch_type<__half>(p, wide_in, wide_out, warps, blocks, st);
}

}  // namespace adapters
}  // namespace smoe
