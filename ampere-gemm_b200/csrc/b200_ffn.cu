// Gated feed-forward block, forward and backward:
//
//   g = x Wg^T, u = x Wu^T, a = act(g) u, y = a Wo^T          (w_in = [Wg; Wu])
//   da = dy Wo, dg = da u act'(g), du = da act(g)
//   dWo = dy^T a, dx = [dg du] w_in, dw_in = [dg du]^T x
//
// Both input projections, the activation and the product are one GEMM launch
// whose epilogue sees g and u of the same elements (kernel_cta2.cuh,
// epilogue_gate.cuh); da is never written either: its epilogue turns it into
// dg, du and a.  The other products are plain GEMMs on the library's kernels.
// g, u, a, dg and du are kept in the operands' 16-bit type between launches:
// the tensor cores take 16-bit operands, and each such rounding adds about as
// much error as the one rounding of the result.  Their rows are padded to a
// multiple of 8 elements (`hidden_pad`).
//
// Operands that TMA cannot address (rows that do not start on 16 bytes) are
// copied into the workspace by one launch before the products, results that it
// cannot store by one launch after them.
#include <algorithm>
#include <atomic>
#include <cstdint>

#include "gemm_internal.h"
#include "kernel_cta2.cuh"
#include "kernel_rows.cuh"
#include "tensor_map.cuh"

namespace b200 {
namespace {

struct GateShape {
  int rows, hidden, depth;  // of the fused GEMM: M, N (columns of a), K
  int hidden_pad;           // row pitch of a, and of each half of [g u] and [dg du]
};

// Launches the pair kernel with a fused epilogue: 256 x 256 accumulator tiles,
// one cluster per tile, tiles taken dynamically.  A is rows x depth (K-major);
// B is 2 hidden x depth (gate and up) or depth x hidden row-major (backward).
template <bool kBf16, int kEpi>
int launch_gate(const void* A, int64_t lda, const void* B, int64_t ldb, void* C, const GateShape& s,
                const FusedArgs<kEpi>& fx, cudaStream_t stream) {
  constexpr bool kUp = kEpi == kEpiGateUp;
  constexpr int kOutN = kUp ? 128 : 256;
  using Cfg = PairConfig<3, 2, 1>;
  CUtensorMap ta, tb, tc;
  int rc = make_tmap_2d(&ta, A, s.rows, s.depth, lda, kBK, kBM, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (rc) return rc;
  rc = kUp ? make_tmap_2d(&tb, B, 2 * (uint64_t)s.hidden, s.depth, ldb, kBK, Cfg::kHalfN,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B)
           : make_tmap_2d(&tb, B, s.depth, s.hidden, ldb, 64, Cfg::kStageK, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (rc) return rc;
  rc = make_tmap_2d(&tc, C, s.rows, s.hidden_pad, s.hidden_pad, kEpiCols, kEpiRows, CU_TENSOR_MAP_L2_PROMOTION_NONE);
  if (rc) return rc;
  auto kern = gemm_f16_tcgen05_pair_kernel<3, 2, 1, !kUp, false, 256, true, kBf16, kEpi>;
  static std::atomic<uint8_t> attr_done[kMaxDevices];
  if (int e = ensure_smem_attr(kern, Cfg::kSmemBytes, attr_done)) return e;
  const long long tiles =
      (long long)((s.rows + Cfg::kTileM - 1) / Cfg::kTileM) * ((s.hidden + kOutN - 1) / kOutN);
  if (tiles > 0x3fffffffLL) return B200_ERR_TOO_LARGE;
  EpiParams ep;
  ep.m = s.rows;
  ep.n = ep.n_tma = s.hidden_pad;
  ep.ldc = s.hidden_pad;
  ep.c = static_cast<uint16_t*>(C);
  const cudaError_t le = launch_gemm(kern, dim3(2 * (unsigned)tiles), dim3(pair_threads(kEpi)), Cfg::kSmemBytes, stream,
                                     ta, tb, tc, s.rows, s.hidden, s.depth, 8, ep, SplitTail{}, fx);
  return le == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}

// A matrix copied between pitches; columns [cols, dst_cols) of the copy, and
// `zero_rows` rows after it, are zero.
struct CopyJob {
  const uint16_t* src;
  uint16_t* dst;
  int64_t src_ld, dst_ld, rows, zero_rows;
  int64_t cols, dst_cols;
};
constexpr int kMaxJobs = 6;
struct CopyJobs {
  CopyJob job[kMaxJobs];
  int n = 0;
  void add(const void* src, int64_t src_ld, void* dst, int64_t dst_ld, int64_t rows, int64_t cols, int64_t dst_cols,
           int64_t zero_rows = 0) {
    job[n++] = CopyJob{static_cast<const uint16_t*>(src), static_cast<uint16_t*>(dst), src_ld, dst_ld, rows,
                       zero_rows, cols, dst_cols};
  }
};

// blockIdx.y = job, a block a row in turn, a thread eight columns in turn.
__global__ void copy_jobs_kernel(const __grid_constant__ CopyJobs jobs) {
  griddep_wait();
  griddep_launch_dependents();
  const CopyJob& j = jobs.job[blockIdx.y];
  const bool src16 = (reinterpret_cast<uintptr_t>(j.src) & 15u) == 0 && j.src_ld % 8 == 0;
  const bool dst16 = (reinterpret_cast<uintptr_t>(j.dst) & 15u) == 0 && j.dst_ld % 8 == 0;
  for (int64_t r = blockIdx.x; r < j.rows + j.zero_rows; r += gridDim.x) {
    const uint16_t* src = j.src + r * j.src_ld;
    uint16_t* dst = j.dst + r * j.dst_ld;
    const int64_t cols = r < j.rows ? j.cols : 0;
    for (int64_t c = threadIdx.x * 8; c < j.dst_cols; c += blockDim.x * 8) {
      alignas(16) uint16_t v[8] = {};
      if (src16 && c + 8 <= cols) {
        *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(src + c);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < cols) v[e] = src[c + e];
      }
      if (dst16 && c + 8 <= j.dst_cols) {
        *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < j.dst_cols) dst[c + e] = v[e];
      }
    }
  }
}

int run_copies(const CopyJobs& jobs, int sm_count, cudaStream_t stream) {
  if (jobs.n == 0) return B200_OK;
  int64_t rows = 1;
  for (int i = 0; i < jobs.n; ++i) rows = std::max(rows, jobs.job[i].rows + jobs.job[i].zero_rows);
  const cudaError_t e = launch_gemm(copy_jobs_kernel, dim3((unsigned)std::min<int64_t>(rows, 8 * sm_count), jobs.n),
                                    dim3(128), 0, stream, jobs);
  return e == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}

int64_t pad8(int64_t n) { return round_up(n, 8); }

// Bytes of a rows x cols 16-bit matrix with padded rows in a workspace.
int64_t part_bytes(int64_t rows, int64_t cols) { return round_up(rows * pad8(cols) * 2, 256); }

// Takes padded matrices out of a workspace.
struct Carver {
  uint8_t* at;
  uint16_t* take(int64_t rows, int64_t cols) {
    uint16_t* p = reinterpret_cast<uint16_t*>(at);
    at += part_bytes(rows, cols);
    return p;
  }
};

// The operand as TMA can read it: itself, or a copy that `jobs` will make.
const void* readable(const void* p, int64_t& ld, int64_t rows, int64_t cols, Carver& ws, CopyJobs& jobs) {
  if (pitch_ok(p, ld)) return p;
  uint16_t* copy = ws.take(rows, cols);
  jobs.add(p, ld, copy, pad8(cols), rows, cols, pad8(cols));
  ld = pad8(cols);
  return copy;
}
// The result as TMA can store it: itself, or a matrix that `jobs` will copy.
void* writable(void* p, int64_t& ld, int64_t rows, int64_t cols, Carver& ws, CopyJobs& jobs) {
  if (pitch_ok(p, ld)) return p;
  uint16_t* copy = ws.take(rows, cols);
  jobs.add(copy, pad8(cols), p, ld, rows, cols, cols);
  ld = pad8(cols);
  return copy;
}

// ---- few rows of x (kernel_rows.cuh) ----

constexpr int kRowsMaxSmem = 227 * 1024;
// An SM's shared memory, what the system takes of it for each CTA, and its TMEM columns.
constexpr int kSmSmem = 228 * 1024, kCtaSmem = 1024, kSmTmemCols = 512;

// Largest number of S-CTA clusters of the rows kernel resident at once, one
// CTA an SM.
template <typename Kern>
int rows_clusters(Kern kern, int parts, int sm_count) {
  if (parts == 1) return sm_count;
  static std::atomic<int> cache[kMaxDevices][4];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return sm_count / parts;
  std::atomic<int>& slot = cache[dev][parts == 2 ? 1 : parts == 4 ? 2 : 3];
  if (const int n = slot.load(std::memory_order_relaxed)) return n;
  (void)cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsMaxSmem);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sm_count / parts * parts);
  cfg.blockDim = dim3(kRowsThreads);
  cfg.dynamicSmemBytes = kRowsMaxSmem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = parts;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int got = 0;
  if (cudaOccupancyMaxActiveClusters(&got, kern, &cfg) != cudaSuccess || got <= 0) {
    (void)cudaGetLastError();
    got = sm_count / parts;
  }
  got = std::min(got, sm_count / parts);
  slot.store(got, std::memory_order_relaxed);
  return got;
}

// How the rows kernel cuts a product up: CTAs of a cluster, rows of w per
// cluster and rows of x per tile, and the estimated time in cycles.
struct RowsPlan {
  int parts = 0, block = 0, tile = 0;
  double cycles = 0.0;
};

// The least estimated time over cluster sizes, tiles of x and row blocks of w
// (an even share for every cluster, 128 rows or 64).  A CTA's 64-deep block of
// K costs 5.1 cycles a row of w (128 bytes at the 25 bytes a cycle that an SM
// gets of the memory's rate; 2 when another tile brought it into L2), 2 a row
// of x, and its MMAs (4 an accumulator, 42 each or N / 2), which hide loads or
// are hidden in part; a cluster's reduction costs 700, a wave 4500, a row of x
// 16 in the epilogue.  Fitted to sweeps over 512 x 1408 to 4096 x 12288 and 1
// to 128 rows of x (one row block an SM without clusters was 1.3-2.3x slower
// for w_out).
RowsPlan plan_rows(int tokens, int n, int k, int accs, bool w_major_n, const int (&slots_of)[4]) {
  RowsPlan best;
  const int k_blocks = (k + kBK - 1) / kBK;
  const int least_tiles = (tokens + kRowsMaxTokens - 1) / kRowsMaxTokens;
  for (int t_tiles = least_tiles; t_tiles < least_tiles + 3; ++t_tiles) {
    const int tile = (tokens + t_tiles - 1) / t_tiles, pad = (tile + 15) / 16 * 16;
    if (t_tiles > least_tiles && tile < 64) break;
    const double row_cost = (5.1 + 2.0 * (t_tiles - 1)) / t_tiles;
    for (int i = 0, s = 1; s <= kRowsMaxParts && s <= k_blocks; ++i, s *= 2) {
      const int slots = slots_of[i], share = (k_blocks + s - 1) / s;
      for (int choice = 0; choice < 3; ++choice) {
        int block = choice == 0 ? 128 : 64;
        if (choice == 2) {
          if (t_tiles > 1 || w_major_n) continue;  // an even share
          const int even_waves = (n + slots * 128 - 1) / (slots * 128);
          block = (n + slots * even_waves - 1) / (slots * even_waves);
        }
        const long long tiles = (long long)((n + block - 1) / block) * t_tiles;
        const double waves = (double)((tiles + slots - 1) / slots);
        const double mma = accs * 4.0 * std::max(42, pad / 2);
        const double load = row_cost * accs * block + 2.0 * pad;
        const double cycles =
            waves * (share * (std::max(mma, load) + 0.4 * std::min(mma, load)) + 16.0 * accs * pad + 4500.0) +
            (s > 1 ? 700.0 : 0.0);
        if (best.parts == 0 || cycles < best.cycles) best = RowsPlan{s, block, tile, cycles};
      }
    }
  }
  return best;
}

// Estimated cycles of the pair kernel: waves of 256 x 256 accumulator tiles
// (`out_n` columns of the result each), 512 a 64-deep block of K, or 800 where
// w comes from memory and not, for another row of tiles, from L2; and a tile's
// epilogue after the last wave.
double pair_cycles(int tokens, int n, int k, int out_n, int sm_count) {
  const int row_tiles = (tokens + 255) / 256;
  const long long tiles = (long long)row_tiles * ((n + out_n - 1) / out_n);
  const long long waves = (tiles + sm_count / 2 - 1) / (sm_count / 2);
  return (double)waves * (std::max(512.0, 800.0 / row_tiles) * ((k + kBK - 1) / kBK) + 2000.0) + 9000.0;
}

// Shape and shared memory of a launch of the rows kernel.
struct RowsLaunch {
  RowsShape sh;
  int smem = 0, tmem_cols = 0;
};

RowsLaunch rows_launch(int tokens, int n, int n_pad, int k, bool gate, const RowsPlan& plan) {
  RowsLaunch l;
  RowsShape& sh = l.sh;
  const int accs = gate ? 2 : 1;
  sh.tokens = tokens;
  sh.tile = plan.tile;
  sh.tokens_pad = (plan.tile + 15) / 16 * 16;
  sh.n = n;
  sh.n_pad = n_pad;
  sh.n_blocks = (n + plan.block - 1) / plan.block;
  sh.k_blocks = (k + kBK - 1) / kBK;
  sh.block = plan.block;
  sh.block_pad = (sh.block + 7) / 8 * 8;
  const int sub = rows_sub_bytes(sh, gate);
  const int share = (sh.k_blocks + plan.parts - 1) / plan.parts;
  // 48 KB a stage (16 KB: 10-30 % slower, each stage costs its commit) in a
  // ring of 200 KB (94 KB, beside the next launch's: 4-8 % slower).
  constexpr int kStageTarget = 48 * 1024, kRing = 200 * 1024;
  sh.k_sub = std::min(share, std::max(1, kStageTarget / sub));
  const int stage = sub * sh.k_sub;
  sh.stages = std::min({kRing / stage, kRowsMaxStages, (share + sh.k_sub - 1) / sh.k_sub});
  sh.tail = (int)round_up(std::max(0, (128 - sh.block_pad - sh.tokens_pad) * 128), 1024);
  // Tokens of a reduction round: what the stages hold in fp32.
  const int token_bytes = accs * 128 * 4;
  if (sh.stages * stage + sh.tail < 16 * token_bytes) sh.tail = 16 * token_bytes;
  sh.chunk = std::min(sh.tokens_pad, (sh.stages * stage + sh.tail) / token_bytes / 16 * 16);
  l.smem = sh.stages * stage + sh.tail + kRowsBarBytes + 1024;
  l.tmem_cols = rows_tmem_columns(accs, sh.tokens_pad);
  // At least the share of an SM's shared memory that the CTA takes of its
  // TMEM: CTAs that share an SM then find TMEM for all of them.  One that
  // waited for TMEM would hold up its cluster, and clusters that each hold what
  // another one's CTA waits for would never end.  (The whole SM for every CTA of
  // a cluster would do too, but successive launches no longer overlap: 24 x 512
  // x 1408 10.4 -> 12.6 us.)
  l.smem = std::max(l.smem, (int)((int64_t)l.tmem_cols * kSmSmem / kSmTmemCols) - kCtaSmem);
  return l;
}

// One product on the rows kernel; `w` has `n` rows (2 n with kRowsGateUp) of k
// elements, or is stored k x n (kWMajorN).
template <bool kBf16, int kMode, bool kWMajorN>
int launch_rows(const void* x, int64_t ldx, const void* w, int64_t ldw, const RowsOut& io, int tokens, int n, int n_pad,
                int k, int act, bool w_early, const RowsPlan& plan, cudaStream_t stream) {
  auto kern = gemm_rows_kernel<kBf16, kMode, kWMajorN>;
  static std::atomic<uint8_t> attr_done[kMaxDevices];
  if (int e = ensure_smem_attr(kern, kRowsMaxSmem, attr_done)) return e;
  constexpr bool kGate = kMode == kRowsGateUp;
  constexpr int kAccs = kGate ? 2 : 1;
  RowsLaunch l = rows_launch(tokens, n, n_pad, k, kGate, plan);
  RowsShape& sh = l.sh;
  sh.activation = act;
  sh.w_early = w_early ? 1 : 0;
  if (l.smem > kRowsMaxSmem) return B200_ERR_CUDA;
  CUtensorMap tw, tx;
  int rc = kWMajorN ? make_tmap_2d(&tw, w, k, n, ldw, 64, kBK, CU_TENSOR_MAP_L2_PROMOTION_L2_256B)
                    : make_tmap_2d(&tw, w, (uint64_t)kAccs * n, k, ldw, kBK, sh.block,
                                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (rc) return rc;
  rc = make_tmap_2d(&tx, x, tokens, k, ldx, kBK, sh.tokens_pad, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(sh.n_blocks * ((tokens + sh.tile - 1) / sh.tile) * plan.parts));
  cfg.blockDim = dim3(kRowsThreads);
  cfg.dynamicSmemBytes = l.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = plan.parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tw, tx, io, sh);
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}

// Whether a product goes to the rows kernel, and how, with `slots_of[i]`
// clusters of 2^i CTAs resident.  Both ways were measured over 64 to 3000 rows:
// at 4096 x 12288 the block takes 54 us for 1 row and 64 for 128 (pair kernel
// 287 and 131: its loads of a mostly empty tile of x collide), from 300 rows on
// the pair kernel is as fast; at 1000 x 2731 a training step takes 102 us for
// 300 rows (152) and 169 for 1111 (191).
bool rows_wins_on(int tokens, int n, int k, bool gate, bool w_major_n, const int (&slots_of)[4], int sm_count,
                  RowsPlan& plan) {
  if (tokens > 16 * kRowsMaxTokens) return false;
  plan = plan_rows(tokens, n, k, gate ? 2 : 1, w_major_n, slots_of);
  return plan.cycles < pair_cycles(tokens, n, k, gate ? 128 : 256, sm_count);
}
template <bool kBf16, int kMode, bool kWMajorN>
bool rows_wins(int tokens, int n, int k, int sm_count, RowsPlan& plan) {
  auto kern = gemm_rows_kernel<kBf16, kMode, kWMajorN>;
  int slots[4];
  for (int i = 0; i < 4; ++i) slots[i] = rows_clusters(kern, 1 << i, sm_count);
  return rows_wins_on(tokens, n, k, kMode == kRowsGateUp, kWMajorN, slots, sm_count, plan);
}

// Columns [hidden, hidden_pad) of a, g and u hold whatever the tile computed
// there (the up projection's first rows as gates); nothing reads them.
template <bool kBf16>
int gate_up(const void* x, int64_t ldx, const void* w_in, int64_t ldw, uint16_t* a, uint16_t* gate_up, int act,
            const GateShape& s, const DeviceInfo& dev, cudaStream_t stream) {
  RowsPlan plan;
  if (rows_wins<kBf16, kRowsGateUp, false>(s.rows, s.hidden, s.depth, dev.sm_count, plan)) {
    RowsOut io{a, s.hidden_pad};
    if (gate_up) {
      io.g = gate_up;
      io.u = gate_up + s.hidden_pad;
      io.ld_gu = 2 * (int64_t)s.hidden_pad;
    }
    return launch_rows<kBf16, kRowsGateUp, false>(x, ldx, w_in, ldw, io, s.rows, s.hidden, s.hidden_pad, s.depth, act,
                                                  false, plan, stream);
  }
  FusedArgs<kEpiGateUp> fx;
  fx.activation = act;
  fx.save = gate_up != nullptr;
  // Unused maps point at `a`, so that every launch has valid ones.
  const int64_t ld = gate_up ? 2 * (int64_t)s.hidden_pad : s.hidden_pad;
  for (int half = 0; half < 2; ++half)
    if (int rc = make_tmap_2d(half ? &fx.tmap_u : &fx.tmap_g, gate_up ? gate_up + half * s.hidden_pad : a, s.rows,
                              s.hidden_pad, ld, kEpiCols, kEpiRows, CU_TENSOR_MAP_L2_PROMOTION_NONE))
      return rc;
  return launch_gate<kBf16, kEpiGateUp>(x, ldx, w_in, ldw, a, s, fx, stream);
}

template <bool kBf16>
int gate_bwd(const void* dy, int64_t lddy, const void* w_out, int64_t ldw, const uint16_t* gate_up, uint16_t* dgu,
             uint16_t* a, int act, const GateShape& s, const DeviceInfo& dev, cudaStream_t stream) {
  RowsPlan plan;
  if (rows_wins<kBf16, kRowsGateBwd, true>(s.rows, s.hidden, s.depth, dev.sm_count, plan)) {
    RowsOut io{a, s.hidden_pad};
    io.saved_g = gate_up;
    io.saved_u = gate_up + s.hidden_pad;
    io.dg = dgu;
    io.du = dgu + s.hidden_pad;
    io.ld_gu = 2 * (int64_t)s.hidden_pad;
    return launch_rows<kBf16, kRowsGateBwd, true>(dy, lddy, w_out, ldw, io, s.rows, s.hidden, s.hidden_pad, s.depth,
                                                  act, false, plan, stream);
  }
  FusedArgs<kEpiGateBwd> fx;
  fx.activation = act;
  fx.g = gate_up;
  fx.u = gate_up + s.hidden_pad;
  fx.dg = dgu;
  fx.du = dgu + s.hidden_pad;
  fx.a = a;
  fx.ld = 2 * (int64_t)s.hidden_pad;
  fx.ld_a = s.hidden_pad;
  return launch_gate<kBf16, kEpiGateBwd>(dy, lddy, w_out, ldw, a, s, fx, stream);
}

// Whether the GEMM may split the last wave of an M x N x K product along K: all
// those that it would on a device of 64 pairs of SMs or more, by a rule on sizes
// alone, so that a workspace's size does not depend on the device.
bool may_split(int64_t M, int64_t N, int64_t K) {
  return K > 2048 && ((M + 255) / 256) * ((N + 255) / 256) > 64;
}
// Bytes of the workspace that the block's products share for it.
int64_t split_bytes(int64_t rows, int64_t dim, int64_t hidden, int64_t out_dim, bool backward) {
  const bool any = backward ? may_split(rows, dim, 2 * pad8(hidden)) || may_split(2 * hidden, dim, rows) ||
                                  may_split(out_dim, hidden, rows)
                            : may_split(rows, out_dim, hidden);
  return any ? round_up(kSplitBytes, 256) : 0;
}
// Takes it out of the call's workspace, its counters set to zero on `stream`; NULL for none.
int take_split(Carver& ws, int64_t bytes, void** split_ws, cudaStream_t stream) {
  *split_ws = bytes > 0 ? ws.at : nullptr;
  if (bytes == 0) return B200_OK;
  constexpr int64_t kParts = kSplitParts * kSplitPartBytes;
  uint8_t* counters = ws.at + kParts;
  ws.at += bytes;
  return cudaMemsetAsync(counters, 0, kSplitBytes - kParts, stream) == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}

int plain_gemm(bool bf16, const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K, int64_t lda,
               int64_t ldb, int64_t ldc, int a_layout, int b_layout, void* split_ws, void* stream) {
  return (bf16 ? gemm_bf16_run : gemm_f16_run)(A, B, C, M, N, K, lda, ldb, ldc, a_layout, b_layout, split_ws, stream);
}

// C = A B with A rows x k, B stored n x k or k x n (kWMajorN), on the kernel that is faster.
template <bool kBf16, bool kWMajorN>
int product(const void* A, int64_t lda, const void* B, int64_t ldb, void* C, int64_t ldc, int rows, int n, int k,
            bool b_early, const DeviceInfo& dev, void* split_ws, cudaStream_t stream) {
  RowsPlan plan;
  if (rows_wins<kBf16, kRowsPlain, kWMajorN>(rows, n, k, dev.sm_count, plan))
    return launch_rows<kBf16, kRowsPlain, kWMajorN>(A, lda, B, ldb, RowsOut{static_cast<uint16_t*>(C), ldc}, rows, n, n,
                                                    k, 0, b_early, plan, stream);
  return plain_gemm(kBf16, A, B, C, rows, n, k, lda, ldb, ldc, B200_A_ROW_MAJOR,
                    kWMajorN ? B200_B_ROW_MAJOR : B200_B_COL_MAJOR, split_ws, stream);
}

// Dimensions, 2 hidden rounded up among them, are rounded up to tiles and dealt
// out in even shares with 32 bits.
constexpr int64_t kMaxDim = 0x7f000000;
bool too_large(int64_t rows, int64_t dim, int64_t hidden, int64_t out_dim) {
  return rows > kMaxDim || dim > kMaxDim || hidden > kMaxDim / 2 || out_dim > kMaxDim;
}

// Checks shared by the two directions; *empty: some dimension is 0.
int check_ffn(int64_t rows, int64_t dim, int64_t hidden, int64_t out_dim, int activation, int dtype, bool* empty) {
  if (rows < 0 || dim < 0 || hidden < 0 || out_dim < 0) return B200_ERR_INVALID_ARGUMENT;
  if (activation < B200_ACT_SILU || activation > B200_ACT_GELU_TANH) return B200_ERR_INVALID_ARGUMENT;
  if (dtype != B200_DTYPE_F16 && dtype != B200_DTYPE_BF16) return B200_ERR_INVALID_ARGUMENT;
  if (too_large(rows, dim, hidden, out_dim)) return B200_ERR_TOO_LARGE;
  *empty = rows == 0 || dim == 0 || hidden == 0 || out_dim == 0;
  return B200_OK;
}

int zero_rows(void* p, int64_t ld, int64_t rows, int64_t cols, cudaStream_t stream) {
  if (!p || rows == 0 || cols == 0) return B200_OK;
  return cudaMemset2DAsync(p, ld * 2, 0, cols * 2, rows, stream) == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}

bool workspace_ok(const void* ws, int64_t bytes, int64_t need) {
  return need == 0 || (ws && bytes >= need && (reinterpret_cast<uintptr_t>(ws) & 255u) == 0);
}

}  // namespace

int take_error_word_ffn() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_device_error, sizeof(int)) != cudaSuccess) return -1;
  const int zero = 0;
  if (v != 0 && cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int)) != cudaSuccess) return -1;
  return v;
}

}  // namespace b200

extern "C" int64_t b200_gated_ffn_workspace_size(int64_t rows, int64_t dim, int64_t hidden, int64_t out_dim,
                                                 int backward, int unaligned) {
  using namespace b200;
  if (rows < 0 || dim < 0 || hidden < 0 || out_dim < 0) return -B200_ERR_INVALID_ARGUMENT;
  if (too_large(rows, dim, hidden, out_dim)) return -B200_ERR_TOO_LARGE;
  const int64_t hp = pad8(hidden);
  int64_t n = part_bytes(rows, hp) + (backward ? part_bytes(rows, 2 * hp) : 0) +
              split_bytes(rows, dim, hidden, out_dim, backward != 0);
  if (unaligned || hidden % 8 != 0 || dim % 8 != 0 || out_dim % 8 != 0) {
    const int64_t in = part_bytes(rows, dim), w_in = part_bytes(2 * hp, dim), w_out = part_bytes(out_dim, hp),
                  out = part_bytes(rows, out_dim);
    n += in + w_in + w_out + out + (backward ? in + w_in + w_out : 0);
  }
  return n;
}

extern "C" int b200_gated_ffn_plan(int64_t rows, int64_t n, int64_t k, int product, int sm_count, int* ctas,
                                   int* smem_bytes, int* tmem_columns) {
  using namespace b200;
  if (rows <= 0 || n <= 0 || k <= 0 || sm_count < 8 || !ctas || !smem_bytes || !tmem_columns)
    return B200_ERR_INVALID_ARGUMENT;
  if (product < B200_FFN_GATE_UP || product > B200_FFN_IN_GRAD) return B200_ERR_INVALID_ARGUMENT;
  if (rows > kMaxDim || n > kMaxDim || k > kMaxDim) return B200_ERR_TOO_LARGE;
  const bool gate = product == B200_FFN_GATE_UP, w_major_n = product == B200_FFN_GATE_GRAD || product == B200_FFN_IN_GRAD;
  int slots[4];
  for (int i = 0; i < 4; ++i) slots[i] = sm_count >> i;
  RowsPlan plan;
  *ctas = *smem_bytes = *tmem_columns = 0;
  if (!rows_wins_on((int)rows, (int)n, (int)k, gate, w_major_n, slots, sm_count, plan)) return B200_OK;
  const RowsLaunch l = rows_launch((int)rows, (int)n, (int)n, (int)k, gate, plan);
  *ctas = plan.parts;
  *smem_bytes = l.smem;
  *tmem_columns = l.tmem_cols;
  return B200_OK;
}

extern "C" int b200_gated_ffn_fwd(const void* x, const void* w_in, const void* w_out, void* y, void* gate_up,
                                  int64_t rows, int64_t dim, int64_t hidden, int64_t out_dim, int64_t ldx,
                                  int64_t ldw_in, int64_t ldw_out, int64_t ldy, int activation, int dtype,
                                  void* workspace, int64_t workspace_bytes, void* stream_ptr) {
  using namespace b200;
  bool empty = false;
  if (int rc = check_ffn(rows, dim, hidden, out_dim, activation, dtype, &empty)) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  const int64_t hp = pad8(hidden);
  if (empty) {
    if (rows > 0 && out_dim > 0 && (!y || ldy < out_dim)) return B200_ERR_INVALID_ARGUMENT;
    if (int rc = zero_rows(gate_up, 2 * hp, rows, 2 * hp, stream)) return rc;
    return zero_rows(y, ldy, rows, out_dim, stream);
  }
  if (!x || !w_in || !w_out || !y || ldx < dim || ldw_in < dim || ldw_out < hidden || ldy < out_dim)
    return B200_ERR_INVALID_ARGUMENT;
  if ((gate_up && !aligned16(gate_up)) || !aligned_to(2, x, w_in, w_out, y)) return B200_ERR_MISALIGNED;
  const bool copies = !pitch_ok(x, ldx) || !pitch_ok(w_in, ldw_in) || !pitch_ok(w_out, ldw_out) || !pitch_ok(y, ldy);
  if (!workspace_ok(workspace, workspace_bytes, b200_gated_ffn_workspace_size(rows, dim, hidden, out_dim, 0, copies)))
    return B200_ERR_WORKSPACE;
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  if (!dev.sm100) return B200_ERR_UNSUPPORTED_DEVICE;
  const bool bf16 = dtype == B200_DTYPE_BF16;
  Carver ws{static_cast<uint8_t*>(workspace)};
  CopyJobs before, after;
  uint16_t* a = ws.take(rows, hp);
  void* split_ws = nullptr;
  if (int rc = take_split(ws, split_bytes(rows, dim, hidden, out_dim, false), &split_ws, stream)) return rc;
  x = readable(x, ldx, rows, dim, ws, before);
  w_in = readable(w_in, ldw_in, 2 * hidden, dim, ws, before);
  w_out = readable(w_out, ldw_out, out_dim, hidden, ws, before);
  if (int rc = run_copies(before, dev.sm_count, stream)) return rc;
  const GateShape s{(int)rows, (int)hidden, (int)dim, (int)hp};
  int rc = (bf16 ? b200::gate_up<true> : b200::gate_up<false>)(
      x, ldx, w_in, ldw_in, a, static_cast<uint16_t*>(gate_up), activation, s, dev, stream);
  if (rc) return rc;
  y = writable(y, ldy, rows, out_dim, ws, after);
  // w_out was written two kernels ago at the latest: its loads may start early.
  rc = (bf16 ? product<true, false> : product<false, false>)(a, hp, w_out, ldw_out, y, ldy, (int)rows, (int)out_dim,
                                                             (int)hidden, true, dev, split_ws, stream);
  return rc ? rc : run_copies(after, dev.sm_count, stream);
}

extern "C" int b200_gated_ffn_bwd(const void* dy, const void* x, const void* w_in, const void* w_out,
                                  const void* gate_up, void* dx, void* dw_in, void* dw_out, int64_t rows, int64_t dim,
                                  int64_t hidden, int64_t out_dim, int64_t lddy, int64_t ldx, int64_t ldw_in,
                                  int64_t ldw_out, int64_t lddx, int64_t lddw_in, int64_t lddw_out, int activation,
                                  int dtype, void* workspace, int64_t workspace_bytes, void* stream_ptr) {
  using namespace b200;
  bool empty = false;
  if (int rc = check_ffn(rows, dim, hidden, out_dim, activation, dtype, &empty)) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if ((dx && lddx < dim) || (dw_in && lddw_in < dim) || (dw_out && lddw_out < hidden)) return B200_ERR_INVALID_ARGUMENT;
  if (empty) {
    if (int rc = zero_rows(dx, lddx, rows, dim, stream)) return rc;
    if (int rc = zero_rows(dw_in, lddw_in, 2 * hidden, dim, stream)) return rc;
    return zero_rows(dw_out, lddw_out, out_dim, hidden, stream);
  }
  if (!dy || !x || !w_in || !w_out || !gate_up || lddy < out_dim || ldx < dim || ldw_in < dim || ldw_out < hidden)
    return B200_ERR_INVALID_ARGUMENT;
  if (!aligned16(gate_up) || !aligned_to(2, dy, x, w_in, w_out, dx, dw_in, dw_out)) return B200_ERR_MISALIGNED;
  const bool copies = !pitch_ok(dy, lddy) || !pitch_ok(x, ldx) || !pitch_ok(w_in, ldw_in) ||
                      !pitch_ok(w_out, ldw_out) || (dx && !pitch_ok(dx, lddx)) ||
                      (dw_in && !pitch_ok(dw_in, lddw_in)) || (dw_out && !pitch_ok(dw_out, lddw_out));
  if (!workspace_ok(workspace, workspace_bytes, b200_gated_ffn_workspace_size(rows, dim, hidden, out_dim, 1, copies)))
    return B200_ERR_WORKSPACE;
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  if (!dev.sm100) return B200_ERR_UNSUPPORTED_DEVICE;
  const bool bf16 = dtype == B200_DTYPE_BF16;
  const int64_t hp = pad8(hidden);
  Carver ws{static_cast<uint8_t*>(workspace)};
  CopyJobs before, after;
  uint16_t* a = ws.take(rows, hp);
  uint16_t* dgu = ws.take(rows, 2 * hp);
  void* split_ws = nullptr;
  if (int rc = take_split(ws, split_bytes(rows, dim, hidden, out_dim, true), &split_ws, stream)) return rc;
  dy = readable(dy, lddy, rows, out_dim, ws, before);
  w_out = readable(w_out, ldw_out, out_dim, hidden, ws, before);
  if (dw_in) x = readable(x, ldx, rows, dim, ws, before);
  if (dx) {
    if (hidden == hp) {
      w_in = readable(w_in, ldw_in, 2 * hidden, dim, ws, before);
    } else {
      // dx sums over the padded rows of [dg du]: w_in with zero rows in their places.
      uint16_t* copy = ws.take(2 * hp, dim);
      const uint16_t* src = static_cast<const uint16_t*>(w_in);
      for (int half = 0; half < 2; ++half)
        before.add(src + half * hidden * ldw_in, ldw_in, copy + half * hp * pad8(dim), pad8(dim), hidden, dim,
                   pad8(dim), hp - hidden);
      w_in = copy;
      ldw_in = pad8(dim);
    }
  }
  if (int rc = run_copies(before, dev.sm_count, stream)) return rc;
  const GateShape s{(int)rows, (int)hidden, (int)out_dim, (int)hp};
  int rc = (bf16 ? gate_bwd<true> : gate_bwd<false>)(dy, lddy, w_out, ldw_out, static_cast<const uint16_t*>(gate_up),
                                                     dgu, a, activation, s, dev, stream);
  if (rc) return rc;
  if (dx) {
    dx = writable(dx, lddx, rows, dim, ws, after);
    rc = (bf16 ? product<true, true> : product<false, true>)(dgu, 2 * hp, w_in, ldw_in, dx, lddx, (int)rows, (int)dim,
                                                             (int)(2 * hp), true, dev, split_ws, stream);
    if (rc) return rc;
  }
  if (dw_in) {
    uint16_t* out = static_cast<uint16_t*>(writable(dw_in, lddw_in, 2 * hidden, dim, ws, after));
    // One product when the halves of [dg du] follow one another, else one for each.
    const int parts = hidden == hp ? 1 : 2;
    for (int half = 0; half < parts; ++half) {
      rc = plain_gemm(bf16, dgu + half * hp, x, out + half * hidden * lddw_in, 2 * hidden / parts, dim, rows, 2 * hp,
                      ldx, lddw_in, B200_A_COL_MAJOR, B200_B_ROW_MAJOR, split_ws, stream_ptr);
      if (rc) return rc;
    }
  }
  if (dw_out) {
    dw_out = writable(dw_out, lddw_out, out_dim, hidden, ws, after);
    rc = plain_gemm(bf16, dy, a, dw_out, out_dim, hidden, rows, lddy, hp, lddw_out, B200_A_COL_MAJOR,
                    B200_B_ROW_MAJOR, split_ws, stream_ptr);
    if (rc) return rc;
  }
  return run_copies(after, dev.sm_count, stream);
}
