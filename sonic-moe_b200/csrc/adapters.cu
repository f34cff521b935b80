// Low-rank adapters: the kernel for few rows, and the entry point (the formulas are in adapters.cuh).
#include "adapters.cuh"

namespace smoe {
namespace adapters {

// ----------------------------------------------------------------------------------------------
// few rows
// ----------------------------------------------------------------------------------------------
// Pitches in shared memory, in floats: of parts, which lanes write two at a time in eight rows, and of s, which they read four at a time.
template <int RP>
struct Few {
  static constexpr int kPart = kPartPitch<RP>, kS = RP + 4;
  static constexpr int kWarp = 16 * (kPart > kStagePitch ? kPart : kStagePitch);  // a warp's part, later its staged rows
  static constexpr size_t kSmem = sizeof(float) * (kWarps * kWarp + 16 * kPart + 16 * kS);
};

// AHEAD: a warp's weights and base for its first columns of out are on their way before the blocks add their parts, those of the next ones before the
// last are done, and more of x and a at a time.  That takes registers, so it is for as many blocks as there is room for at once.
// Latency bounds it (bf16, us): one token, 4096 x 4096, rank 16 4.8 (5.5 without AHEAD); 64 tokens of 64 adapters, 4096 x 2048, rank 16 8.3, rank 64 18
// (1.75 TB/s of weights, x, base and out); 128 tokens of 2, 4096 x 4096, rank 64 8.8 (13 without); 256 of 4, rank 16 6.9.  Clusters: its rows are too
// few to fill the card, so eight blocks share the columns of each 16.
template <class T, int RP, bool ALIGNED, bool AHEAD>
__global__ void __launch_bounds__(32 * kWarps, AHEAD ? 1 : RP == 16 ? (ALIGNED ? 4 : 2) : RP == 32 ? (ALIGNED ? 3 : 2) : RP == 64 && ALIGNED ? 2 : 1) few_kernel(const Params p) {
  release_next();
  wait_for_previous();
  using F = Few<RP>;
  extern __shared__ __align__(16) float smem[];
  float* parts = smem;                       // [warp][16][kPart]
  float* part = smem + kWarps * F::kWarp;    // [16][kPart]
  float* s_all = part + 16 * F::kPart;       // [16][kS]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rank = static_cast<int>(cluster_ctarank()), tile = blockIdx.x / kCluster;
  if (tile >= p.tiles) {
    Others others;
    others.begin(p, (blockIdx.x - p.tiles * kCluster) * kWarps + warp);
    others.finish(p);
    return;
  }
  // Loads of the row's tokens, of the adapters' rows, and then of all that hangs on them are on their way together; whether a row is still its token's
  // is looked at in the end.
  int row0 = 16 * tile, e;
  bool rows_here = true;
  if (p.sparse) {
    const int4 what = tile_of(p, tile, 16);
    e = max(what.x, 0);
    row0 = what.y;
    rows_here = what.x >= 0;
  } else {
    e = adapter_of(p, row0);
  }
  const int my_row = row0 + (lane & 15);
  const int candidate = gathered_of(p, my_row);
  if (!p.sparse) rows_here = within(p, row0);
  const int gathered = rows_here ? candidate : -1;
  if (__all_sync(0xffffffffu, gathered < 0)) return;  // (the cluster's blocks all see the same)
  const int row_of = gathered >= 0 ? p.reverse[gathered] : -1;
  const int x_t0 = __shfl_sync(0xffffffffu, gathered, g), x_t1 = __shfl_sync(0xffffffffu, gathered, g + 8);
  const int groups = (p.N + kGroup - 1) / kGroup;
  const int n_first = static_cast<int>(static_cast<long long>(groups) * rank / kCluster), n_end = static_cast<int>(static_cast<long long>(groups) * (rank + 1) / kCluster);
  const char* b = p.b + static_cast<long long>(e) * p.N * p.r * 2;
  {  // the L2 fetches the weights of this block's columns of out meanwhile
    const long long first = static_cast<long long>(n_first) * kGroup * p.r * 2, end = min(static_cast<long long>(n_end) * kGroup, static_cast<long long>(p.N)) * p.r * 2;
    for (long long o = first + 128ll * threadIdx.x; o < end; o += 128ll * blockDim.x) asm volatile("prefetch.global.L2 [%0];" ::"l"(b + o));
  }
  // a x over this warp's columns
  constexpr int NT = RP / 8;
  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  {
    const int chunks = (p.H + 31) / 32, parts_of = kCluster * kWarps, mine = rank * kWarps + warp;
    const int first = static_cast<int>(static_cast<long long>(chunks) * mine / parts_of), end = static_cast<int>(static_cast<long long>(chunks) * (mine + 1) / parts_of);
    const char* x0 = p.x + x_t0 * p.x_ld;
    const char* x1 = p.x + x_t1 * p.x_ld;
    const char* a = p.a + (static_cast<long long>(e) * p.r + g) * p.H * 2;
    const int width0 = x_t0 >= 0 ? p.H : 0, width1 = x_t1 >= 0 ? p.H : 0;
    constexpr int U = RP <= 32 || (RP == 64 && ALIGNED && AHEAD) ? 2 : 1;  // chunks whose loads are on their way together
    for (int c = first; c < end; c += U) {
      Raw8<ALIGNED> xa[U][2], w[U][NT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int col = c + u < end ? 32 * (c + u) + 8 * t : p.H;
        xa[u][0].load(x0, col, width0);
        xa[u][1].load(x1, col, width1);
#pragma unroll
        for (int j = 0; j < NT; ++j) w[u][j].load(a + 16ll * j * p.H, col, 8 * j + g < p.r ? p.H : 0);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int col = c + u < end ? 32 * (c + u) + 8 * t : p.H;
        const uint4 v0 = xa[u][0].get(x0, col, width0), v1 = xa[u][1].get(x1, col, width1);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint4 v = w[u][j].get(a + 16ll * j * p.H, col, 8 * j + g < p.r ? p.H : 0);
          mma<T>(acc[j], v0.x, v1.x, v0.y, v1.y, v.x, v.y);
          mma<T>(acc[j], v0.z, v1.z, v0.w, v1.w, v.z, v.w);
        }
      }
    }
  }
  int group = n_first + warp;
  ColumnWeights<RP, ALIGNED> weights;
  BaseRows<T> base;
  BaseColumn column;
  const auto fetch = [&] {
    if (group >= n_end) return;
    weights.load(p, b, kGroup * group);
    if (ALIGNED) base.load(p, kGroup * group + 8 * t, x_t0, x_t1);
    else column.load(p, kGroup * group + lane, gathered);
  };
  if (AHEAD && RP <= 64) fetch();
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    float* to = parts + warp * F::kWarp + g * F::kPart + 8 * j + 2 * t;
    *reinterpret_cast<float2*>(to) = make_float2(acc[j][0], acc[j][1]);
    *reinterpret_cast<float2*>(to + 8 * F::kPart) = make_float2(acc[j][2], acc[j][3]);
  }
  __syncthreads();
  constexpr int Q = RP / 4;  // fours of a row
#pragma unroll
  for (int i0 = 0; i0 < 16 * Q; i0 += 32 * kWarps) {
    const int i = i0 + threadIdx.x, at = i / Q * F::kPart + 4 * (i % Q);
    if (i >= 16 * Q) continue;
    float4 f = *reinterpret_cast<const float4*>(parts + at);
#pragma unroll
    for (int w = 1; w < kWarps; ++w) {
      const float4 v = *reinterpret_cast<const float4*>(parts + w * F::kWarp + at);
      f.x += v.x; f.y += v.y; f.z += v.z; f.w += v.w;
    }
    *reinterpret_cast<float4*>(part + at) = f;
  }
  cluster_sync_all();
  const float scale = p.scale != nullptr ? p.scale[e] : 1.f;
#pragma unroll
  for (int i0 = 0; i0 < 16 * Q; i0 += 32 * kWarps) {
    const int i = i0 + threadIdx.x;
    if (i >= 16 * Q) continue;
    const uint32_t at = smem_u32(part + i / Q * F::kPart + 4 * (i % Q));
    float4 f[kCluster];
#pragma unroll
    for (int k = 0; k < kCluster; ++k) f[k] = load_cluster(map_to_cta(at, k));
#pragma unroll
    for (int k = 1; k < kCluster; ++k) {
      f[0].x += f[k].x; f[0].y += f[k].y; f[0].z += f[k].z; f[0].w += f[k].w;
    }
    *reinterpret_cast<float4*>(s_all + i / Q * F::kS + 4 * (i % Q)) = make_float4(f[0].x * scale, f[0].y * scale, f[0].z * scale, f[0].w * scale);
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // this block has read the others' parts
  __syncthreads();
  // s in this warp's registers
  constexpr int K = Steps<RP>::K;
  uint32_t lead[K][4], rest[K][4];
  const auto fours = [&](int row, int k) {
    return *reinterpret_cast<const float4*>(s_all + row * F::kS + (RP == 16 ? 4 * t : 32 * (k / 2) + 8 * t + 4 * (k & 1)));
  };
  float f0 = 1.f, f1 = 1.f;
  if (std::is_same<T, __half>::value) {
    float most0 = 0.f, most1 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float4 u = fours(g, k), v = fours(g + 8, k);
      most0 = fmaxf(fmaxf(most0, fmaxf(fabsf(u.x), fabsf(u.y))), fmaxf(fabsf(u.z), fabsf(u.w)));
      most1 = fmaxf(fmaxf(most1, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
    }
#pragma unroll
    for (int o = 1; o < 4; o *= 2) {
      most0 = fmaxf(most0, __shfl_xor_sync(0xffffffffu, most0, o));
      most1 = fmaxf(most1, __shfl_xor_sync(0xffffffffu, most1, o));
    }
    f0 = factor_of<T>(most0);
    f1 = factor_of<T>(most1);
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const float4 u = fours(g, k), v = fours(g + 8, k);
    split2<T>(u.x * f0, u.y * f0, lead[k][0], rest[k][0]);
    split2<T>(v.x * f1, v.y * f1, lead[k][1], rest[k][1]);
    split2<T>(u.z * f0, u.w * f0, lead[k][2], rest[k][2]);
    split2<T>(v.z * f1, v.w * f1, lead[k][3], rest[k][3]);
  }
  const float i0 = inverse_of<T>(f0), i1 = inverse_of<T>(f1);
  const int tokens = row_of == my_row ? gathered : -1;
  const int t0 = __shfl_sync(0xffffffffu, tokens, g), t1 = __shfl_sync(0xffffffffu, tokens, g + 8);
  if (!AHEAD || RP > 64) fetch();
  while (group < n_end) {
    const int n0 = kGroup * group;
    float c[4][4];
    weights.template multiply<T>(p, b, n0, lead, rest, c);
    const BaseRows<T> base_now = base;
    const BaseColumn column_now = column;
    group += kWarps;
    if (AHEAD) fetch();
    if (ALIGNED) {
      put_row<T>(p, n0 + 8 * t, t0, base_now.v[0], c, 0, i0);
      put_row<T>(p, n0 + 8 * t, t1, base_now.v[1], c, 1, i1);
    } else {
      put_staged<T>(p, n0, tokens, column_now, c, i0, i1, parts + warp * F::kWarp);
    }
    if (!AHEAD) fetch();
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ----------------------------------------------------------------------------------------------
// launches
// ----------------------------------------------------------------------------------------------
// Tiles of `rows` rows, at most: what the adapters' tokens fill, and a part of one more each.
static long long tiles_of(int T, int n, int rows) {
  const long long tiles = T / rows + static_cast<long long>(n < T ? n : T);
  return tiles < T ? tiles : T;
}
// The rules below go by the adapters that there are, since the host does not know how many of them the tokens use: where that is a few of many, they take tiles
// for fewer rows than there are.  8192 tokens of 8 requests, 4096 x 4096, rank 64, 56 / 71 / 109 us with 8 / 64 / 512 adapters to choose from, 2048 tokens
// 30 / 33 / 94; of 12, rank 16, 42 with 8, 63 with 512.
// Tiles of 16 rows and eight blocks each: while few of them are needed, more for wide rows, and where it is the weights of adapters with a few tokens each
// that take the time, which come straight from memory there.  us by few_kernel / by tiles, 4096 x 4096 unless said: 256 tokens of 2 adapters, rank 16,
// 7 / 14; 512 of 8, rank 64, 13 / 20 with 64 tokens each, 20 / 20 drawn at random (37 tiles of eight blocks are what 148 SMs hold at a time at rank 64; the
// tokens then fill 36 to 39); 512 of 4, rank 64, 14 / 21, 1024 x 1024 13 / 12; 2048 of 4, rank 16, 21 / 21, 1024 x 1024 14 / 10; 64 of 64, rank
// 128, 41 / 54, 4097 x 4095 68 / 310; 512 of 100, rank 64, 27 / 31, rank 128, 64 / 56, 4097 x 4095 118 / 346; 4096 of 500, rank 64, 132 / 107, 4097 x
// 4095, rank 128, 524 / 1219; 448 of 160, 342 x 187, rank 16, 31 / 16.
// Of those, the ones with tcgen05.mma need fewer (wide_in, rows of out that start anywhere: 2048 of 100, rank 128, 247 / 121, 512 of 100, rank 64, 65 / 57,
// rank 32, 34 / 49).  Twelve tiles would leave most of the card idle as tiles of more rows: 130 tokens of 2, 1920 x 5917, rank 124, 25 / 55.
static bool by_few_rows(int T, int n, int r, int H, int N, bool wide_in, bool wide_out) {
  const int rank = padded_rank(r);
  const bool tensor = wide_in && !wide_out && rank >= 64;
  const long long tiles = tiles_of(T, n, 16), size = tiles * rank;
  const int most = H + N <= 8000 || tensor ? 1024 : wide_in && wide_out ? 2600 : 2304;
  return tiles <= 12 || size <= most || (T / n < 16 && H + N > 3000 && !tensor && (!wide_out || !wide_in || size <= 8192));
}
// Warps of a tile's blocks otherwise, by the tokens that an adapter has on average: eight where that brings in tcgen05.mma, more for wide weights, which the
// warps fetch together.  us with 2 / 4 / 8: 2048 tokens of 100, 4096 x 4096, rank 32, 27 / 36 / 38, rank 128, 86 / 63 / 82, 4097 x 4095, rank 32, 66 / 89 /
// 85, rank 64, 194 / 133 / 112, rank 128, 533 / 222 / 283, 4096 x 4095, rank 32, 66 / 87 / 65, rank 64, 193 / 133 / 71; 512 of 100, 342 x 187, rank 64, 15 / 19
// / 15; 1024 of 16, 4096 x 4096, rank 128, 56 / 37 / 49.
static int warps_of(int T, int n, int r, bool wide_in, bool wide_out) {
  const int rank = padded_rank(r), tokens = T / n;
  if (wide_in && !wide_out && (rank >= 64 || (rank == 32 && tokens >= 16))) return 8;
  const int two = rank == 128 ? (wide_in ? 16 : 0) : rank == 64 && !wide_in ? 16 : 32;
  return tokens <= two && two > 0 ? 2 : tokens <= 64 ? 4 : 8;
}

// Blocks of few_kernel with AHEAD that an SM has room for.
template <int RP, bool ALIGNED>
constexpr int kAheadBlocks = RP == 16 ? (ALIGNED ? 3 : 2) : RP == 32 && ALIGNED ? 2 : 1;

template <class T, int RP, bool ALIGNED>
static int launch_few(const Params& p, long long blocks, cudaStream_t st) {
  static PerDeviceFlag configured;
  const int dev = current_device();
  if (dev < 0) return SMOE_ERR_DRIVER;
  constexpr int smem = static_cast<int>(Few<RP>::kSmem);
  if (!configured.test(dev)) {
    if (cudaFuncSetAttribute(few_kernel<T, RP, ALIGNED, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
        cudaFuncSetAttribute(few_kernel<T, RP, ALIGNED, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return SMOE_ERR_LAUNCH;
    configured.set(dev);
  }
  const bool ahead = tiles_of(p.T, p.n, 16) * kCluster <= 148 * kAheadBlocks<RP, ALIGNED>;
  return launched(launch_chained(ahead ? few_kernel<T, RP, ALIGNED, true> : few_kernel<T, RP, ALIGNED, false>, dim3(static_cast<unsigned>(blocks)), 32 * kWarps,
                                 smem, st, kCluster, p));
}
template <class T, bool ALIGNED>
static int launch_few(const Params& p, long long blocks, cudaStream_t st) {
  switch (padded_rank(p.r)) {
    case 16: return launch_few<T, 16, ALIGNED>(p, blocks, st);
    case 32: return launch_few<T, 32, ALIGNED>(p, blocks, st);
    case 64: return launch_few<T, 64, ALIGNED>(p, blocks, st);
    default: return launch_few<T, 128, ALIGNED>(p, blocks, st);
  }
}

static long long address(const void* p) { return static_cast<long long>(reinterpret_cast<uintptr_t>(p)); }

}  // namespace adapters
}  // namespace smoe

using namespace smoe;
using namespace smoe::adapters;

extern "C" {

int smoe_adapter_linear(const void* x, long long ld, const void* a, const void* b, const float* scale, const void* base, long long base_ld,
                        void* out, long long out_ld, int dtype, const int* expert_frequency_offset, const int* expert_frequency,
                        const int* x_gather_idx, const int* s_reverse_scatter_idx, int T, long long rows, int H, int N, int n, int r, int align, int* status,
                        void* stream) {
  if (dtype != SMOE_BF16 && dtype != SMOE_F16) return SMOE_ERR_DTYPE;
  if (T < 0 || T > kMaxRows || rows < 0 || rows > kMaxRows || H <= 0 || N <= 0 || n <= 0 || n > kMaxAdapters || r <= 0 || r > kMaxRank || align <= 0 ||
      align % 16 != 0 || ld < 0 || base_ld < 0 || out_ld < N)
    return SMOE_ERR_SHAPE;
  if (H > 1 << 28 || N > 1 << 28) return SMOE_ERR_SHAPE;
  if (T == 0) return SMOE_OK;
  if (x == nullptr || a == nullptr || b == nullptr || out == nullptr || expert_frequency_offset == nullptr || expert_frequency == nullptr || s_reverse_scatter_idx == nullptr ||
      (rows > 0 && x_gather_idx == nullptr))
    return SMOE_ERR_SHAPE;
  if ((address(x) | address(a) | address(b) | address(base) | address(out)) % 2 != 0 ||
      (address(scale) | address(expert_frequency_offset) | address(expert_frequency) | address(x_gather_idx) | address(s_reverse_scatter_idx) | address(status)) % 4 != 0)
    return SMOE_ERR_ALIGNMENT;
  Params p = {};
  p.x = static_cast<const char*>(x); p.x_ld = 2 * ld;
  p.a = static_cast<const char*>(a); p.b = static_cast<const char*>(b); p.scale = scale;
  p.base = static_cast<const char*>(base); p.base_ld = base != nullptr ? 2 * base_ld : 0;
  p.out = static_cast<char*>(out); p.out_ld = 2 * out_ld;
  p.off = expert_frequency_offset; p.count = expert_frequency; p.gather = x_gather_idx; p.reverse = s_reverse_scatter_idx;
  p.T = T; p.rows = static_cast<int>(rows); p.H = H; p.N = N; p.n = n; p.r = r;
  p.status = status;
  const bool wide_in = (address(x) | address(a) | address(b) | p.x_ld) % 16 == 0 && H % 8 == 0 && r % 8 == 0;
  const bool wide_out = (address(base) | address(out) | p.base_ld | p.out_ld) % 16 == 0 && N % 8 == 0;
  const bool few = by_few_rows(T, n, r, H, N, wide_in, wide_out);
  const int warps = few ? kWarps : warps_of(T, n, r, wide_in, wide_out);
  p.sparse = (rows + 15) / 16 > tiles_of(T, n, 16);
  p.tiles = static_cast<int>(few && !p.sparse && rows > 0 ? (rows + 15) / 16 : tiles_of(T, n, few ? 16 : 16 * warps));  // (one at least: its blocks see to the other tokens)
  // Warps of the tiles that there may be, half of the adapters having one that is not full: as many blocks share a tile as let 1200 to 2400 warps, eight
  // to sixteen to an SM, run at a time.  2048 tokens of 100 adapters, 4096 x 1024, rank 32, take 50 / 31 / 23 / 18 us with 1 / 2 / 4 / 8 blocks to a tile
  // of 32 rows; 8192 of 400 110 / 84 / 84 / 85; 8192 of 8, 4096 x 4096, rank 64, 56 us with four to a tile of 128; 32768 of them 183 / 194 / 209 / 244.
  const long long likely = warps * ((T + 16ll * warps - 1) / (16 * warps) + (n < T ? n : T) / 2);
  p.cluster = few ? kCluster : likely > 8 * 148 ? 1 : likely > 4 * 148 ? 2 : likely > 2 * 148 ? 4 : 8;
  // The tokens without an adapter: a warp of clusters behind the tiles' for each, or, with many tokens, some of them for every warp of the tiles (blocks
  // of their own made 8192 tokens that all have adapters wait 13 us for blocks that found nothing).
  long long blocks = static_cast<long long>(p.tiles) * p.cluster;
  if (base != out || base_ld != out_ld) {
    p.others = static_cast<int>(few ? 1 : (T + blocks * warps - 1) / (blocks * warps));
    if (few) blocks += (T + kCluster * kWarps - 1ll) / (kCluster * kWarps) * kCluster;
  }
  if (blocks > 0x7fffffffll) return SMOE_ERR_SHAPE;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!few) return launch_tiles(p, dtype, wide_in, wide_out, warps, blocks, st);
  if (dtype == SMOE_BF16) return wide_in && wide_out ? launch_few<__nv_bfloat16, true>(p, blocks, st) : launch_few<__nv_bfloat16, false>(p, blocks, st);
  return wide_in && wide_out ? launch_few<__half, true>(p, blocks, st) : launch_few<__half, false>(p, blocks, st);
}

}  // extern "C"
