// Kernel choice and launchers of the GEMM, for fp16 (kBf16 = false) and bf16
// operands.  Everything is in an unnamed namespace: b200_gemm.cu instantiates
// the fp16 kernels, b200_gemm_bf16.cu the bf16 ones, each with its own
// workspaces and options.
#pragma once

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <mutex>
#include <type_traits>
#include <utility>

#include "gemm_common.cuh"
#include "gemm_internal.h"
#include "kernel_cta1.cuh"
#include "kernel_cta2.cuh"
#include "kernel_skinny.cuh"
#include "tensor_map.cuh"

namespace b200 {
namespace {

// One GEMM call as the launchers see it (operands already TMA-compatible).
struct GemmArgs {
  const void* A;
  const void* B;
  void* C;
  int M, N, K;
  int64_t lda, ldb, ldc;
  EpiParams scale;
  int sm_count;
  cudaStream_t stream;
  ArgminOut argmin = ArgminOut{};
};

// Width of C's tensor map: the columns the TMA store covers (at least one
// column so the map encodes; when N < 8 it is never used).
inline int c_map_cols(const GemmArgs& g) { return g.scale.n_tma > 0 ? g.scale.n_tma : g.N; }

// Calls fn(row-major B, column-major A) with the two layouts as compile-time
// constants, so every launcher is instantiated for the four combinations.
template <typename Fn>
int with_layouts(bool row_b, bool col_a, Fn&& fn) {
  if (row_b) return col_a ? fn(std::true_type{}, std::true_type{}) : fn(std::true_type{}, std::false_type{});
  return col_a ? fn(std::false_type{}, std::true_type{}) : fn(std::false_type{}, std::false_type{});
}

template <bool kBf16, int BN, int STAGES, bool kBRowMajor, bool kAColMajor>
int launch_tcgen05(const GemmArgs& g, int group_m) {
  using Cfg = TileConfig<BN, STAGES>;
  const void *A = g.A, *B = g.B;
  void* C = g.C;
  const int M = g.M, N = g.N, K = g.K;
  const int64_t lda = g.lda, ldb = g.ldb, ldc = g.ldc;
  const int sm_count = g.sm_count;
  cudaStream_t stream = g.stream;
  CUtensorMap ta, tb, tc;
  int rc = kAColMajor ? make_tmap_2d(&ta, A, K, M, lda, 64, kBK, CU_TENSOR_MAP_L2_PROMOTION_L2_256B)
                      : make_tmap_2d(&ta, A, M, K, lda, kBK, kBM, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (rc) return rc;
  if (kBRowMajor)
    rc = make_tmap_2d(&tb, B, K, N, ldb, 64, kBK, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  else
    rc = make_tmap_2d(&tb, B, N, K, ldb, kBK, BN, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (rc) return rc;
  rc = make_tmap_2d(&tc, C, M, c_map_cols(g), ldc, kEpiCols, kEpiRows, CU_TENSOR_MAP_L2_PROMOTION_NONE);
  if (rc) return rc;

  auto kern = gemm_f16_tcgen05_kernel<BN, STAGES, kBRowMajor, kAColMajor, kBf16>;
  static std::atomic<uint8_t> attr_done[kMaxDevices];
  if (int e = ensure_smem_attr(kern, Cfg::kSmemBytes, attr_done)) return e;
  const long long tiles = (long long)((M + kBM - 1) / kBM) * ((N + BN - 1) / BN);
  const int grid = (int)std::min<long long>(tiles, sm_count);
  const cudaError_t le = launch_gemm(kern, dim3(grid), dim3(kThreads), Cfg::kSmemBytes, stream, ta, tb, tc, M, N, K,
                                     group_m, g.scale);
  return le == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}

// ---- split of the last wave along K (pair kernel, MSUB = 1) ----
// Cost model in SM cycles: a 256 x 256 pair tile spends 1024 cycles per
// 128-deep K stage.  A split tail costs about 8.1k cycles plus 3.4k per K
// range (writing the parts, the arrival, the last unit's read-back and sum),
// fitted to 2560 x 2048 x 8192 at S = 2, 3, 4, 7 (saved time against the
// ideal T (1 - 1/S)).  So only deep K pays: at K = 2048 the split is slower,
// at K = 4096 even, at K = 8192 S = 4 saves 16 %.
constexpr double kPairStageCycles = 1024.0;
constexpr double kSplitFixedCycles = 8100.0;
constexpr double kSplitPartCycles = 3400.0;

// K ranges per tail tile that minimise the last wave's time (1 = no split).
int choose_split(int num_kb, long long smax) {
  // B200_GEMM_SPLIT_S forces the number of K ranges (tuning only).
  static const int forced = [] {
    const char* e = std::getenv("B200_GEMM_SPLIT_S");
    return e ? std::atoi(e) : 0;
  }();
  if (forced >= 1) return (int)std::max<long long>(1, std::min<long long>({(long long)forced, smax, kFixBufs + 1,
                                                                         num_kb / 2}));
  int best = 1;
  double best_cost = num_kb * kPairStageCycles;
  for (int S = 2; S <= smax && S <= kFixBufs + 1 && 2 * S <= num_kb; ++S) {  // fixup holds S - 1 parts
    const double c = num_kb * kPairStageCycles / S + kSplitFixedCycles + kSplitPartCycles * S;
    if (c < best_cost * 0.97) {
      best_cost = c;
      best = S;
    }
  }
  return best;
}

// Last wave's time as a fraction of a whole tile's, with the split the
// launcher would choose.
double pair_tail_fraction(int num_kb, long long tiles, int slots) {
  const long long r = tiles % slots;
  if (r == 0) return 1.0;
  if (tiles < slots) return 1.0;  // a single partial wave is never split
  const int S = choose_split(num_kb, slots / r);
  if (S == 1) return 1.0;
  return (num_kb * kPairStageCycles / S + kSplitFixedCycles + kSplitPartCycles * S) / (num_kb * kPairStageCycles);
}

bool split_enabled() {
  static const bool on = [] {
    const char* e = std::getenv("B200_GEMM_SPLIT");
    return !(e && e[0] == '0');
  }();
  return on;
}

// K ranges the 256 x 256 pair kernel cuts its last wave into (1 = none) for
// `tiles` tiles on `grid_pairs` resident pairs and `num_kb` 128-deep K stages.
int split_ranges_for(long long tiles, int grid_pairs, int num_kb) {
  if (!split_enabled() || grid_pairs <= 0 || tiles <= grid_pairs || tiles % grid_pairs == 0) return 1;
  return choose_split(num_kb, grid_pairs / (tiles % grid_pairs));
}

// One workspace per (device, stream): launches on one stream are ordered, so
// they can share it; other streams get their own.  Allocated on first use
// (never during a stream capture: that launch then runs unsplit).
struct SplitWorkspace {
  int dev;
  cudaStream_t stream;
  float* parts;
  uint32_t* counters;
  int max_parts;
};

std::mutex g_split_mu;
SplitWorkspace g_split_ws[64];
int g_split_n = 0;

bool split_workspace(cudaStream_t stream, int sm_count, SplitTail& st) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  std::lock_guard<std::mutex> lock(g_split_mu);
  SplitWorkspace* w = nullptr;
  for (int i = 0; i < g_split_n; ++i)
    if (g_split_ws[i].dev == dev && g_split_ws[i].stream == stream) w = &g_split_ws[i];
  if (!w) {
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(stream, &cs) != cudaSuccess || cs != cudaStreamCaptureStatusNone) return false;
    if (g_split_n == 64) return false;
    const int max_parts = sm_count;  // R * S <= pairs, two CTAs each
    const size_t part_bytes = (size_t)max_parts * kPartFloats * sizeof(float);
    void* mem = nullptr;
    if (cudaMalloc(&mem, part_bytes + (size_t)max_parts * sizeof(uint32_t)) != cudaSuccess) {
      (void)cudaGetLastError();
      return false;
    }
    uint32_t* ctr = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(mem) + part_bytes);
    if (cudaMemsetAsync(ctr, 0, (size_t)max_parts * sizeof(uint32_t), stream) != cudaSuccess) {
      cudaFree(mem);
      return false;
    }
    w = &g_split_ws[g_split_n++];
    *w = SplitWorkspace{dev, stream, static_cast<float*>(mem), ctr, max_parts};
  }
  st.ws = w->parts;
  st.counters = w->counters;
  return true;  // R * S <= pairs <= sm_count / 2, so the parts always fit
}

// Zeroes the tail counters of every workspace on the current device (after a
// launch that gave up on a bounded wait; the device is idle then).
void reset_split_counters() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return;
  std::lock_guard<std::mutex> lock(g_split_mu);
  for (int i = 0; i < g_split_n; ++i)
    if (g_split_ws[i].dev == dev)
      (void)cudaMemset(g_split_ws[i].counters, 0, (size_t)g_split_ws[i].max_parts * sizeof(uint32_t));
}

// Per-call launch options, set by an entry point for the duration of one
// (host-synchronous) call on this thread.
struct CallOptions {
  bool no_split = false;           // run every tile whole: no split workspace (allocation-free entry)
  uint64_t withhold_fixup_ns = 0;  // fixup-wait self-test (see SplitTail)
  int force_variant = -1;          // >= 0: this variant instead of b200_gemm_set_variant's / auto
  void* split_ws = nullptr;        // kSplitBytes of the caller's memory instead of the stream's own workspace
};
thread_local CallOptions t_call;

struct ScopedCallOptions {
  CallOptions saved;
  explicit ScopedCallOptions(const CallOptions& o) : saved(t_call) { t_call = o; }
  ~ScopedCallOptions() { t_call = saved; }
};

template <bool kBf16, int STAGES, int KSUB, int MSUB, bool kBRowMajor, bool kAColMajor, int BN = 256, bool kDyn = false>
int launch_tcgen05_pair(const GemmArgs& g, int group_m) {
  using Cfg = PairConfig<STAGES, KSUB, MSUB, BN>;
  const void *A = g.A, *B = g.B;
  void* C = g.C;
  const int M = g.M, N = g.N, K = g.K;
  const int64_t lda = g.lda, ldb = g.ldb, ldc = g.ldc;
  const int sm_count = g.sm_count;
  cudaStream_t stream = g.stream;
  CUtensorMap ta, tb, tc;
  int rc = kAColMajor ? make_tmap_2d(&ta, A, K, M, lda, 64, Cfg::kStageK, CU_TENSOR_MAP_L2_PROMOTION_L2_256B)
                      : make_tmap_2d(&ta, A, M, K, lda, kBK, kBM, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (rc) return rc;
  if (kBRowMajor)
    rc = make_tmap_2d(&tb, B, K, N, ldb, 64, Cfg::kStageK, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  else
    rc = make_tmap_2d(&tb, B, N, K, ldb, kBK, Cfg::kHalfN, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (rc) return rc;
  rc = make_tmap_2d(&tc, C, M, c_map_cols(g), ldc, kEpiCols, kEpiRows, CU_TENSOR_MAP_L2_PROMOTION_NONE);
  if (rc) return rc;
  auto kern = gemm_f16_tcgen05_pair_kernel<STAGES, KSUB, MSUB, kBRowMajor, kAColMajor, BN, kDyn, kBf16>;
  static std::atomic<uint8_t> attr_done[kMaxDevices];
  if (int e = ensure_smem_attr(kern, Cfg::kSmemBytes, attr_done)) return e;
  static int pairs_cache[kMaxDevices] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  int pairs = (dev >= 0 && dev < kMaxDevices) ? pairs_cache[dev] : 0;
  if (pairs <= 0) {
    pairs = max_active_pairs(kern, Cfg::kSmemBytes, sm_count);
    if (dev >= 0 && dev < kMaxDevices) pairs_cache[dev] = pairs;
    if (std::getenv("B200_GEMM_DEBUG")) std::fprintf(stderr, "b200_gemm: %d resident 2-CTA clusters\n", pairs);
  }
  const long long tiles = (long long)((M + Cfg::kTileM - 1) / Cfg::kTileM) * ((N + Cfg::kTileN - 1) / Cfg::kTileN);
  // Dynamic tiles launch one cluster per tile (those that have not started
  // when a running pair needs work are cancelled and their tiles taken).
  const int grid_pairs = kDyn ? (int)tiles : (int)std::min<long long>(tiles, pairs);
  if (kDyn && tiles > 0x3fffffffLL) return B200_ERR_TOO_LARGE;
  SplitTail st;
  const int S = (MSUB == 1 && !kDyn && !t_call.no_split)
                    ? split_ranges_for(tiles, grid_pairs, (K + Cfg::kStageK - 1) / Cfg::kStageK)
                    : 1;
  if (S >= 2) {
    const long long r = tiles % grid_pairs;
    SplitTail s2;
    s2.dp_tiles = (int)(tiles - r);
    s2.S = S;
    s2.withhold_fixup_ns = t_call.withhold_fixup_ns;
    if (t_call.split_ws) {
      if (2 * r * S <= kSplitParts) {
        s2.ws = static_cast<float*>(t_call.split_ws);
        s2.counters = reinterpret_cast<uint32_t*>(s2.ws + (size_t)kSplitParts * kPartFloats);
        st = s2;
      }
    } else if (split_workspace(stream, sm_count, s2)) {
      st = s2;
    }
    if (std::getenv("B200_GEMM_DEBUG"))
      std::fprintf(stderr, "b200_gemm: %lld tiles on %d pairs, last %lld tiles split %d ways%s\n", tiles, grid_pairs, r,
                   S, st.S > 1 ? "" : " (no workspace: unsplit)");
  }
  const cudaError_t le = launch_gemm(kern, dim3(2 * grid_pairs), dim3(kThreads), Cfg::kSmemBytes, stream, ta, tb, tc,
                                     M, N, K, group_m, g.scale, st, FusedArgs<kEpiPlain>{});
  return le == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}

// Skinny (K <= 256) B-stationary kernel.  The grid is the largest multiple of
// the number of 256-column N slices that fits the SMs, so every CTA keeps one
// slice of B resident.  Returns B200_ERR_INVALID_ARGUMENT when the shape does
// not qualify (caller falls back to another variant).
template <int A_STAGES, int EPI_BUFS, bool kBRowMajor, bool kAColMajor, bool kArgmin = false, int EPI_W = kEpiWarps>
int launch_skinny(const GemmArgs& g) {
  using Cfg = SkinnyConfig<A_STAGES, EPI_BUFS, EPI_W>;
  const void *A = g.A, *B = g.B;
  void* C = g.C;
  const int M = g.M, N = g.N, K = g.K;
  const int64_t lda = g.lda, ldb = g.ldb, ldc = g.ldc;
  const int sm_count = g.sm_count;
  cudaStream_t stream = g.stream;
  const int num_nb = (N + Cfg::kBN - 1) / Cfg::kBN;
  if (K > Cfg::kMaxKBlocks * kBK || num_nb > sm_count) return B200_ERR_INVALID_ARGUMENT;
  CUtensorMap ta, tb, tc;
  int rc = kAColMajor ? make_tmap_2d(&ta, A, K, M, lda, 64, kBK, CU_TENSOR_MAP_L2_PROMOTION_L2_256B)
                      : make_tmap_2d(&ta, A, M, K, lda, kBK, kBM, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (rc) return rc;
  if (kBRowMajor)
    rc = make_tmap_2d(&tb, B, K, N, ldb, 64, kBK, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  else
    rc = make_tmap_2d(&tb, B, N, K, ldb, kBK, Cfg::kBN, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (rc) return rc;
  if constexpr (kArgmin)
    tc = ta;  // no C: the argmin epilogue writes keys, the map is never used
  else
    rc = make_tmap_2d(&tc, C, M, c_map_cols(g), ldc, kEpiCols, kEpiRows, CU_TENSOR_MAP_L2_PROMOTION_NONE);
  if (rc) return rc;
  auto kern = gemm_f16_skinny_kernel<A_STAGES, EPI_BUFS, kBRowMajor, kAColMajor, kArgmin, EPI_W>;
  static std::atomic<uint8_t> attr_done[kMaxDevices];
  if (int e = ensure_smem_attr(kern, Cfg::kSmemBytes, attr_done)) return e;
  const long long tiles = (long long)((M + kBM - 1) / kBM) * num_nb;
  const int slots = (sm_count / num_nb) * num_nb;
  const int grid = (int)std::min<long long>(tiles, slots);
  const cudaError_t le = launch_gemm(kern, dim3(grid), dim3(skinny_threads(kArgmin, EPI_W)), Cfg::kSmemBytes, stream, ta, tb,
                                     tc, M, N, K, g.scale, g.argmin);
  return le == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}

// Kernel choice for K > 256.  Each persistent variant runs its tiles in waves
// of `slots` concurrent tiles; the last wave is usually partial, so the
// estimate is  waves * (per-SM tile work) / (relative per-SM rate).  Rates are
// measured steady-state throughputs relative to the wide pair (8192^3:
// 1.00 wide pair, 0.96 pair, 0.93 one-CTA); the model reproduces the best
// measured variant on 2048^3 .. 8192^3, 4096 x 8192 x 4096, 8192 x 4096 x 4096,
// 4000 x 6000 x 3000 and 65536 x 8192 x 8192.
// Tile width of the wide pair kernel (256, 224 or 192 columns) for an
// m x n product on `slots` resident pairs.  The MMAs of a narrower tile take
// proportionally less time, but the kernel's stages hold the same bytes
// whatever the width, and measured tile times barely fall with it (4000 x
// 6000 x 3000: 120.4 us at 256 against 122.6 at 224 over the same 3 waves;
// 4096 x 8192 x 4096: 201.6 against 198.6 over 4 waves).  So a narrower tile
// pays only where it needs fewer waves, or within a single wave, where it
// spreads the same work over more SMs (2560 x 2048 x 2048: 23.9-27.0 us with
// 192-wide tiles against 31.5 with 256-wide); other ties keep the widest.
// Returns the width and, in *waves, its wave count.  B200_GEMM_WIDE_BN forces
// one (tuning only).
int wide_pair_bn(int m, int n, int slots, double* waves_out = nullptr) {
  static const int forced = [] {
    const char* e = std::getenv("B200_GEMM_WIDE_BN");
    const int v = e ? std::atoi(e) : 0;
    return (v == 256 || v == 224 || v == 192) ? v : 0;
  }();
  const int cand[3] = {256, 224, 192};
  int best = 256;
  long long best_w = -1;
  for (int bn : cand) {
    if (forced && bn != forced) continue;
    const long long tiles = (long long)((m + 511) / 512) * ((n + bn - 1) / bn);
    const long long w = (tiles + slots - 1) / slots;
    // Fewest waves; among equals the widest tile, except within a single
    // wave, where the narrowest gives each SM the least work.
    if (best_w < 0 || w < best_w || (w == best_w && w == 1 && bn < best)) {
      best_w = w;
      best = bn;
    }
  }
  if (waves_out) *waves_out = (double)best_w;
  return best;
}

int pick_tensor_variant(int m, int n, int k, int sm_count) {
  if (k < 512) return B200_VARIANT_CTA1;  // a pair's prologue is not amortised
  // One wave of 1-CTA tiles of moderate depth: every variant takes about one
  // tile's time and the 1-CTA kernel has the cheapest start (2048^3: 16.4-16.7
  // us against 17.3-17.6 for the pair kernel).  Deeper single-wave shapes go
  // through the model below (1536 x 1280 x 8192: pair 44.7 us against 47.5
  // for the 1-CTA kernel).
  if (k <= 4096 && (long long)((m + 127) / 128) * ((n + 255) / 256) <= sm_count) return B200_VARIANT_CTA1;
  // Cost in SM cycles: waves x one tile's MMA time / relative rate, plus the
  // last tile's accumulator drain (one 256-column block, two for the wide pair).
  struct Opt {
    int variant, tile_m, tile_n, slots, rows_per_sm;
    double rate, drain_cycles;
  };
  const int pairs = sm_count / 2;
  const Opt opts[3] = {
      // Wide pair drain: 3200 cycles since its epilogue releases each
      // accumulator block before storing it (3072^3: one wave of wide tiles
      // 43.0 us against 45.0 for two waves of the pair kernel).
      {B200_VARIANT_PAIR_WIDE, 512, 256, pairs, 256, 1.00, 3200.0},
      {B200_VARIANT_PAIR, 256, 256, pairs, 128, 0.96, 3200.0},
      {B200_VARIANT_CTA1, 128, 256, sm_count, 128, 0.93, 3200.0},
  };
  const double tile128_cycles = 8.0 * k;  // 128 x 256 rows x columns: k / 16 MMAs of 128 cycles
  int best = B200_VARIANT_CTA1;
  double best_cost = 1e300;
  for (const Opt& o : opts) {
    const long long tiles = (long long)((m + o.tile_m - 1) / o.tile_m) * ((n + o.tile_n - 1) / o.tile_n);
    double waves = (double)((tiles + o.slots - 1) / o.slots);
    double width = 1.0;  // tile time relative to a 256-wide tile
    if (o.variant == B200_VARIANT_PAIR_WIDE) {
      const int bn = wide_pair_bn(m, n, o.slots, &waves);  // best tile width's waves
      // In a single wave of moderate depth a narrower tile does finish sooner
      // (2560 x 2048 x 2048: 23.9 us for one wave of 192-wide tiles against
      // 26.0 for the pair kernel's two waves); over several waves it does not.
      if (waves <= 1.0 && k <= 4096) width = bn / 256.0;
    }
    if (o.variant == B200_VARIANT_PAIR && split_enabled() && tiles % o.slots != 0)
      waves = (double)(tiles / o.slots) + pair_tail_fraction((k + 127) / 128, tiles, o.slots);  // split last wave
    const double cost = waves * width * tile128_cycles * (o.rows_per_sm / 128.0) / o.rate + o.drain_cycles;
    if (cost < best_cost * 0.999) {
      best_cost = cost;
      best = o.variant;
    }
  }
  if (best == B200_VARIANT_PAIR_WIDE) {
    const int bn = wide_pair_bn(m, n, pairs);
    if (bn == 224) return B200_VARIANT_PAIR_WIDE_224;
    if (bn == 192) return B200_VARIANT_PAIR_WIDE_192;
  }
  return best;
}

// The kernel the library runs for an m x n x k product when no variant is forced.
int auto_variant(int m, int n, int k, int sm_count) {
  if (k <= 256 && (n + 255) / 256 <= sm_count) {
    // B-stationary pays for its one-off B load once a CTA has several tiles
    // (measured: ahead from ~3 tiles per SM, behind at 1-2).
    const long long tiles = (long long)((m + 127) / 128) * ((n + 255) / 256);
    if (tiles >= 3LL * sm_count) return B200_VARIANT_SKINNY;
  }
  return pick_tensor_variant(m, n, k, sm_count);
}

// Process-wide kernel-variant override (b200_gemm_set_variant).
int g_variant = B200_VARIANT_AUTO;

// Raster band height in tiles; B200_GEMM_GROUP_M overrides it (tuning only).
int group_m_override() {
  static int v = [] {
    const char* e = std::getenv("B200_GEMM_GROUP_M");
    return e ? std::atoi(e) : 0;  // negative: bands of column blocks
  }();
  return v;
}

// Dynamic tile scheduling of the wide pair kernel (cluster launch control),
// used when its tiles take more than one wave: three interleaved rounds at
// 65536 x 8192 x 8192 ran 6341-6459 us against 6461-6506 static, 4000 x 6000
// x 3000 119.2 against 120.3; one-wave shapes have nothing to balance.
// B200_GEMM_DYN=0 turns it off (tuning).
bool dyn_tiles() {
  static const bool on = [] {
    const char* e = std::getenv("B200_GEMM_DYN");
    return !(e && e[0] == '0');
  }();
  return on;
}

// C <- rn(beta * C) for an empty reduction (K == 0) with beta != 0.
template <bool kBf16>
__global__ void scale_c_kernel(uint16_t* C, int64_t ldc, int64_t rows, int64_t cols, float beta) {
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y)
    for (int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; c < cols; c += (int64_t)gridDim.x * blockDim.x) {
      const float v = unpack_16bit<kBf16>(C[r * ldc + c]).x;
      C[r * ldc + c] = static_cast<uint16_t>(pack_16bit_rn<kBf16>(__float_as_uint(beta * v), 0u));
    }
}

// C = alpha * op(A) * op(B) + beta * C on operands that already satisfy TMA's
// alignment rules.
template <bool kBf16>
int gemm_aligned(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb,
                 int64_t ldc, int a_layout, int b_layout, const EpiParams& scale, const DeviceInfo& dev,
                 cudaStream_t stream) {
  if (K == 0) {
    // Empty reduction: C = beta * C (all zeros when beta == 0).
    if (scale.beta == 0.0f)
      return cudaMemset2DAsync(C, ldc * 2, 0, N * 2, M, stream) == cudaSuccess ? B200_OK : B200_ERR_CUDA;
    const unsigned gx = (unsigned)std::min<int64_t>((N + 255) / 256, 64);
    const unsigned gy = (unsigned)std::min<int64_t>(M, 65535);
    scale_c_kernel<kBf16><<<dim3(gx, gy), 256, 0, stream>>>(static_cast<uint16_t*>(C), ldc, M, N, scale.beta);
    return cudaGetLastError() == cudaSuccess ? B200_OK : B200_ERR_CUDA;
  }
  const bool row_b = (b_layout == B200_B_ROW_MAJOR);
  const bool col_a = (a_layout == B200_A_COL_MAJOR);
  const int m = (int)M, n = (int)N, k = (int)K;
  EpiParams ep = scale;
  ep.m = m;
  ep.n = n;
  ep.ldc = ldc;
  ep.c = static_cast<uint16_t*>(C);
  ep.n_tma = n & ~7;  // a TMA store writes whole 16-byte pieces: the partial last one goes by plain stores
  ep.c_evict_first = (dev.l2_bytes > 0 && 2 * M * N > dev.l2_bytes) ? 1 : 0;
  const GemmArgs g{A, B, C, m, n, k, lda, ldb, ldc, ep, dev.sm_count, stream};
  int variant = t_call.force_variant >= 0 ? t_call.force_variant : g_variant;
  if (variant == B200_VARIANT_AUTO) variant = auto_variant(m, n, k, dev.sm_count);
  if constexpr (kBf16) {
    if (variant == B200_VARIANT_SKINNY) variant = B200_VARIANT_CTA1;  // built for fp16 only
  } else if (variant == B200_VARIANT_SKINNY) {
    const int rc = with_layouts(row_b, col_a, [&](auto rb, auto ca) {
      // Measured: 5 A stages with 4 epilogue warps beat 4 stages with 8 warps
      // (the A stream, not the epilogue, then sets the pace) and 4 stages
      // with two staging buffers per warp.
      return launch_skinny<5, 1, decltype(rb)::value, decltype(ca)::value>(g);
    });
    if (rc != B200_ERR_INVALID_ARGUMENT) return rc;
    variant = B200_VARIANT_CTA1;  // shape outside the skinny kernel's range
  }
  const int gm = group_m_override();
  if (variant == B200_VARIANT_PAIR_WIDE || variant == B200_VARIANT_PAIR_WIDE_224 ||
      variant == B200_VARIANT_PAIR_WIDE_192) {
    // Raster: when A is much taller than B is wide, bands of 12 column blocks
    // (65536 x 8192 x 8192 with C stored evict-first, two interleaved rounds:
    // 6435-6465 us against 6452-6482 for bands of 8, 6495-6579 for 16,
    // 6689-6748 for 32 and 6561-6566 for 8-row bands; DRAM reads per launch
    // 8.9 GB against 9.7-11.2 for bands of 8); otherwise bands of 8 row blocks.
    const int group_m = gm ? gm : (m >= 4LL * n ? -12 : 8);
    const int bn = variant == B200_VARIANT_PAIR_WIDE_224 ? 224 : variant == B200_VARIANT_PAIR_WIDE_192 ? 192 : 256;
    return with_layouts(row_b, col_a, [&](auto rb, auto ca) {
      constexpr bool kRb = decltype(rb)::value, kCa = decltype(ca)::value;
      if (bn == 224) return launch_tcgen05_pair<kBf16, 4, 1, 2, kRb, kCa, 224>(g, group_m);
      if (bn == 192) return launch_tcgen05_pair<kBf16, 4, 1, 2, kRb, kCa, 192>(g, group_m);
      if (dyn_tiles() && (long long)((m + 511) / 512) * ((n + 255) / 256) > dev.sm_count / 2)
        return launch_tcgen05_pair<kBf16, 4, 1, 2, kRb, kCa, 256, true>(g, group_m);
      return launch_tcgen05_pair<kBf16, 4, 1, 2, kRb, kCa, 256>(g, group_m);
    });
  }
  if (variant == B200_VARIANT_PAIR) {
    const int group_m = gm ? gm : 8;  // 8 x 256-row bands: fewest DRAM bytes measured at 8192^3
    // Several waves and no split last wave: dynamic tiles, as for the wide pair.
    const long long tiles = (long long)((m + 255) / 256) * ((n + 255) / 256);
    const int pairs = dev.sm_count / 2;
    const bool dyn = dyn_tiles() && tiles > pairs &&
                     (t_call.no_split || split_ranges_for(tiles, pairs, (k + 127) / 128) == 1);
    return with_layouts(row_b, col_a, [&](auto rb, auto ca) {
      constexpr bool kRb = decltype(rb)::value, kCa = decltype(ca)::value;
      if (dyn) return launch_tcgen05_pair<kBf16, 3, 2, 1, kRb, kCa, 256, true>(g, group_m);
      return launch_tcgen05_pair<kBf16, 3, 2, 1, kRb, kCa, 256>(g, group_m);
    });
  }
  const int group_m = gm ? gm : 16;  // 16 x 128-row bands: fewest DRAM bytes measured at 8192^3
  return with_layouts(row_b, col_a, [&](auto rb, auto ca) {
    return launch_tcgen05<kBf16, 256, 4, decltype(rb)::value, decltype(ca)::value>(g, group_m);
  });
}

// See gemm_f16_run() in gemm_internal.h.
template <bool kBf16>
int gemm_run(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb,
             int64_t ldc, int a_layout, int b_layout, void* split_ws, void* stream) {
  static_assert(kSplitPartBytes == kPartFloats * sizeof(float), "a part is one CTA's share of a pair tile");
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  CallOptions opts;
  opts.no_split = split_ws == nullptr;
  opts.force_variant = B200_VARIANT_AUTO;
  opts.split_ws = split_ws;
  ScopedCallOptions scope(opts);
  return gemm_aligned<kBf16>(A, B, C, M, N, K, lda, ldb, ldc, a_layout, b_layout, EpiParams{}, dev,
                             static_cast<cudaStream_t>(stream));
}

// Reads and clears this translation unit's error word (0: none, negative: a CUDA error).
int take_error_word() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_device_error, sizeof(int)) != cudaSuccess) return -1;
  const int zero = 0;
  if (v != 0 && cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) reset_split_counters();  // an aborted launch may have left tail counters counting
  return v;
}

}  // namespace
}  // namespace b200
