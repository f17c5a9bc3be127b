// GEMM kernel for few to some hundred rows of x: out[t][n] = sum_k x[t][k] w[n][k],
// with the gated feed-forward block's epilogues (see RowsMode).
//
// With few rows such a product is bound by reading w once.  So the operands
// change places: a block of rows of w is the 128-row operand of the MMA (lane =
// row of w) and up to 256 rows of x, rounded up to 16, are its N columns.  Rows
// of w are dealt out evenly: every CTA takes `block` of them (not 128: lanes
// past `block` compute on whatever lies behind the tile in shared memory and
// are never read), so one wave of CTAs streams equal shares of w.  With a
// cluster of S CTAs each takes 1/S of K for S times as many rows, which cuts
// the re-reading of x (all of it, by every cluster) by S and fills the SMs when
// there are few tiles; the S parts are added up through distributed shared
// memory in a fixed order.  More rows of x than one tile holds are split evenly
// over several.
//
//   warp 0      TMA producer; warp 1 MMA issuer; warps 2..9 epilogue, which all
//               ten share once the MMAs are over.
//
// Measured: w of 24576 x 4096 (gate and up) in 42 us, of 4096 x 12288 in 22 us
// for one row of fp16 x: 0.74 and 0.69 of the measured copy bandwidth with the
// launch's start and end, which a short stream cannot hide.
//
// Launched with programmatic stream serialisation.  With `w_early`, w was not
// written by the kernel before this one on the stream: the first stages of w
// are requested before that kernel has finished, only x waits for it.
#pragma once

#include <type_traits>

#include "epilogue_gate.cuh"
#include "gemm_common.cuh"

namespace b200 {

constexpr int kRowsMaxTokens = 256;  // N of one MMA
constexpr int kRowsMaxStages = 16;
constexpr int kRowsMaxParts = 8;     // CTAs of a cluster
constexpr int kRowsThreads = 320;    // producer, issuer and eight epilogue warps

// Epilogues.
enum RowsMode : int {
  kRowsPlain = 0,    // out = the product
  kRowsGateUp = 1,   // w = [Wg; Wu]: out = act(g) u, optionally g and u too
  kRowsGateBwd = 2,  // the product is da: dg, du and out = a from it and the saved g, u
};

struct RowsShape {
  int tokens;      // rows of x
  int tile;        // rows of x per tile
  int tokens_pad;  // `tile` rounded up to 16: N of the MMAs
  int n_blocks;    // row blocks of w
  int n;           // rows of w (of each half with kGate)
  int k_blocks;    // 64-wide blocks of K
  int block;       // rows of w per cluster (of each half), <= 128
  int block_pad;   // rounded up to 8
  int k_sub;       // 64-wide blocks of a stage
  int stages;
  int chunk;       // tokens per reduction round of a cluster
  int activation;
  int w_early;
  int n_pad;       // columns that kRowsGateBwd writes: n, and zeros up to here
  int tail;        // bytes after the stages that an MMA may read: a tile of fewer than 128 rows is read past its end
};

// Where the epilogue writes and reads, row pitches in elements.
struct RowsOut {
  uint16_t* out;
  int64_t ld;
  uint16_t* g = nullptr;  // kRowsGateUp: g and u are stored here unless NULL
  uint16_t* u = nullptr;
  const uint16_t* saved_g = nullptr;  // kRowsGateBwd
  const uint16_t* saved_u = nullptr;
  uint16_t* dg = nullptr;
  uint16_t* du = nullptr;
  int64_t ld_gu = 0;      // of all of these
};

__host__ __device__ inline int rows_sub_bytes(const RowsShape& s, bool gate) {
  return ((gate ? 2 : 1) * s.block_pad + s.tokens_pad) * 128;
}
// TMEM columns of a CTA: a power of two, 32 at least.
__host__ __device__ inline int rows_tmem_columns(int accs, int tokens_pad) {
  int cols = 32;
  while (cols < accs * tokens_pad) cols *= 2;
  return cols;
}
constexpr int kRowsBarBytes = (2 * kRowsMaxStages + 2) * 8 + 16;

__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// wait::ld that names the loaded registers, as tmem_ld_wait_regs.
__device__ __forceinline__ void tmem_ld_wait_regs16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// One lane of a converged warp, as a predicate word for the forms below.  The
// whole warp runs the producer's and the issuer's loops and only the elected
// lane's instruction takes effect: with warp-uniform operands a
// tcgen05.mma.cta_group::1 of N = 16 is issued every 42 cycles, its commit
// costs 150; from a branch that one lane takes they are 71 and 210 (measured).
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p;
}

__device__ __forceinline__ void umma_f16_cta1_if(uint32_t elected, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                                 uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}

__device__ __forceinline__ void umma_commit_cta1_if(uint32_t elected, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(elected)
      : "memory");
}

__device__ __forceinline__ void tma_load_2d_if(uint32_t elected, uint32_t dst, const void* tmap, uint32_t bar,
                                               int32_t x, int32_t y, uint64_t cache_hint) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4}], [%2], %5;\n\t}" ::"r"(dst),
      "l"(tmap), "r"(bar), "r"(x), "r"(y), "l"(cache_hint), "r"(elected)
      : "memory");
}

__device__ __forceinline__ void mbar_expect_tx_if(uint32_t elected, uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t.reg .b64 st;\n\tsetp.ne.b32 q, %2, 0;\n\t"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(bar),
      "r"(bytes), "r"(elected)
      : "memory");
}

__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ float4 ld_shared_cluster_v4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr)
               : "memory");
  return v;
}

__device__ __forceinline__ float gate_value(int activation, float g, float u) {
  if (activation == 0) return activate<0, false>(g).f * u;
  if (activation == 1) return activate<1, false>(g).f * u;
  return activate<2, false>(g).f * u;
}

// dg, du and a of one element.
template <int kAct>
__device__ __forceinline__ float3 gate_grad(float da, float g, float u) {
  const ActValue v = activate<kAct, true>(g);
  return make_float3(da * u * v.slope, da * v.f, v.f * u);
}
__device__ __forceinline__ float3 gate_grads(int activation, float da, float g, float u) {
  if (activation == 0) return gate_grad<0>(da, g, u);
  if (activation == 1) return gate_grad<1>(da, g, u);
  return gate_grad<2>(da, g, u);
}

// The first `n` (<= 4) of four values to 16-bit elements at p, in one store when it is a whole, aligned one.
template <bool kBf16>
__device__ __forceinline__ void store_quad(uint16_t* p, const float (&v)[4], int n) {
  const uint32_t lo = pack_16bit_rn<kBf16>(__float_as_uint(v[0]), __float_as_uint(v[1]));
  const uint32_t hi = pack_16bit_rn<kBf16>(__float_as_uint(v[2]), __float_as_uint(v[3]));
  if (n >= 4 && (reinterpret_cast<uintptr_t>(p) & 7u) == 0) {
    *reinterpret_cast<uint2*>(p) = make_uint2(lo, hi);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n) p[e] = static_cast<uint16_t>((e < 2 ? lo : hi) >> ((e & 1) * 16));
}

// The accumulators' four rows of w of one token, staged at `at` in each of the
// kP CTAs of the cluster: all parts are requested, then added up in order.
template <int kP, int kAccs>
__device__ __forceinline__ void sum_parts(const float* at, int acc_step, float4 (&r)[kAccs]) {
  float4 v[kAccs][kP];
#pragma unroll
  for (int a = 0; a < kAccs; ++a) {
#pragma unroll
    for (int p = 0; p < kP; ++p)
      v[a][p] = kP == 1 ? *reinterpret_cast<const float4*>(at + a * acc_step)
                        : ld_shared_cluster_v4(mapa_shared(smem_u32(at + a * acc_step), p));
  }
#pragma unroll
  for (int a = 0; a < kAccs; ++a) {
    r[a] = v[a][0];
#pragma unroll
    for (int p = 1; p < kP; ++p) {
      r[a].x += v[a][p].x;
      r[a].y += v[a][p].y;
      r[a].z += v[a][p].z;
      r[a].w += v[a][p].w;
    }
  }
}

// kWMajorN: w is stored K x N (N contiguous); `block` is then a multiple of 64.
template <bool kBf16, int kMode, bool kWMajorN>
__global__ void __launch_bounds__(kRowsThreads, 1)
    gemm_rows_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                     const __grid_constant__ RowsOut io, const __grid_constant__ RowsShape sh) {
  constexpr bool kGate = kMode == kRowsGateUp;
  constexpr int kAccs = kGate ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int sub_bytes = rows_sub_bytes(sh, kGate);
  const int stage_bytes = sub_bytes * sh.k_sub;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + sh.stages * stage_bytes + sh.tail);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + kRowsMaxStages;
  uint64_t* done_bar = bars + 2 * kRowsMaxStages;   // accumulators final
  uint64_t* drain_bar = done_bar + 1;               // abort path only
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int parts = static_cast<int>(cluster_nctarank());
  const int rank = static_cast<int>(cluster_ctarank());
  // Row blocks of w are the faster index: the tiles that run together share x.
  const int cluster = static_cast<int>(blockIdx.x) / parts;
  const int n0 = cluster % sh.n_blocks * sh.block;
  const int t_tile = cluster / sh.n_blocks * sh.tile;
  const int tokens = min(sh.tile, sh.tokens - t_tile);
  const int kb0 = static_cast<int>(static_cast<int64_t>(rank) * sh.k_blocks / parts);
  const int kb1 = static_cast<int>(static_cast<int64_t>(rank + 1) * sh.k_blocks / parts);
  const int num_stages = (kb1 - kb0 + sh.k_sub - 1) / sh.k_sub;
  // Every cluster reads all of x.  Clusters start at different places of K and
  // wrap around: in step, they would all ask one L2 slice for the same line.
  const int start = static_cast<int>(static_cast<int64_t>(cluster) * num_stages / (gridDim.x / parts));
  auto k_stage = [&](int it) { return it + start < num_stages ? it + start : it + start - num_stages; };
  auto subs = [&](int it) { return min(sh.k_sub, kb1 - kb0 - k_stage(it) * sh.k_sub); };
  const uint32_t tmem_cols = static_cast<uint32_t>(rows_tmem_columns(kAccs, sh.tokens_pad));

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
    for (int s = 0; s < sh.stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(done_bar, 1);
    mbar_init(drain_bar, 1);
    fence_mbarrier_init();
  }
  if (warp == 1) {
    tmem_alloc<1>(tmem_base_slot, tmem_cols);
    tmem_relinquish_alloc_permit<1>();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_base_slot;
  // The bounded waits below do not run while the kernel before this one does.
  if (warp != 0) griddep_wait();

  if (warp == 0) {
    const uint32_t el = elect_lane();
    // Read once, unless several tiles of x follow one another.
    const uint64_t pol_w = sh.tile < sh.tokens ? policy_evict_normal() : policy_evict_first();
    const uint64_t pol_x = policy_evict_last();   // read by every cluster
    const uint32_t smem0 = smem_u32(smem), full0 = smem_u32(full_bar);
    const uint32_t sub_tx = static_cast<uint32_t>((kAccs * sh.block + sh.tokens_pad) * 128);
    auto load_w = [&](int it, int stage) {
      const int n_sub = subs(it);
      const uint32_t bar = full0 + stage * 8;
      uint32_t dst = smem0 + stage * stage_bytes;
      int k = (kb0 + k_stage(it) * sh.k_sub) * kBK;
      mbar_expect_tx_if(el, bar, static_cast<uint32_t>(n_sub) * sub_tx);
      for (int j = 0; j < n_sub; ++j, dst += sub_bytes, k += kBK) {
        if constexpr (kWMajorN) {
          // Panels of 64 rows of w x 64 of K.
          for (int p = 0; p < sh.block; p += 64) tma_load_2d_if(el, dst + p * 128, &tmap_w, bar, n0 + p, k, pol_w);
        } else {
          tma_load_2d_if(el, dst, &tmap_w, bar, k, n0, pol_w);
        }
        if (kGate) tma_load_2d_if(el, dst + sh.block_pad * 128, &tmap_w, bar, k, sh.n + n0, pol_w);
      }
    };
    auto load_x = [&](int it, int stage) {
      const int n_sub = subs(it);
      const uint32_t bar = full0 + stage * 8;
      uint32_t dst = smem0 + stage * stage_bytes + kAccs * sh.block_pad * 128;
      int k = (kb0 + k_stage(it) * sh.k_sub) * kBK;
      for (int j = 0; j < n_sub; ++j, dst += sub_bytes, k += kBK)
        tma_load_2d_if(el, dst, &tmap_x, bar, k, t_tile, pol_x);
    };
    const int first = min(num_stages, sh.stages);
    if (sh.w_early)
      for (int it = 0; it < first; ++it) load_w(it, it);
    griddep_wait();
    griddep_launch_dependents();
    for (int it = 0; it < first; ++it) {
      if (!sh.w_early) load_w(it, it);
      load_x(it, it);
    }
    int issued = first, stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int it = first; it < num_stages; ++it) {
      ok = __all_sync(0xffffffffu, mbar_wait(&empty_bar[stage], phase, kDevTimeoutProducer));
      if (!ok) break;
      load_w(it, stage);
      load_x(it, stage);
      ++issued;
      if (++stage == sh.stages) { stage = 0; phase ^= 1u; }
    }
    if (lane == 0) {
      // Every load lands before the CTA leaves, also where the issuer has given
      // up and nothing else waits for them.
      for (int it = max(0, issued - sh.stages); it < issued; ++it) {
        uint64_t* bar = &full_bar[it % sh.stages];
        const uint32_t parity = static_cast<uint32_t>(it / sh.stages) & 1u;
        if (!mbar_wait(bar, parity, kDevTimeoutProducer)) mbar_wait_drain(bar, parity);
      }
    }
  } else if (warp == 1) {
    const uint32_t el = elect_lane();
    const uint32_t idesc = make_idesc_f16_f32(128, static_cast<uint32_t>(sh.tokens_pad),
                                              kWMajorN ? Major::kMN : Major::kK,
                                              Major::kK, kBf16);
    // Descriptors advance by adding to their address field (units of 16 bytes;
    // addresses stay below 2^18).
    const uint64_t x_desc0 = make_desc_kmajor_sw128(smem_u32(smem));
    const uint64_t w_desc0 = kWMajorN ? make_desc_mnmajor_sw128(smem_u32(smem), kBK * 128) : x_desc0;
    constexpr uint64_t kWStep = (kWMajorN ? kUmmaK * 128 : kUmmaK * 2) >> 4, kXStep = (kUmmaK * 2) >> 4;
    const uint64_t up_off = static_cast<uint64_t>(sh.block_pad * 128) >> 4;
    const uint64_t x_off = static_cast<uint64_t>(kAccs * sh.block_pad * 128) >> 4;
    const uint64_t sub_off = static_cast<uint64_t>(sub_bytes) >> 4;
    const uint32_t d_up = tmem_base + sh.tokens_pad;
    uint32_t acc = 0;
    bool ok = true;
    int stage = 0;
    uint32_t phase = 0;
    for (int it = 0; it < num_stages; ++it) {
      ok = __all_sync(0xffffffffu, mbar_wait(&full_bar[stage], phase, kDevTimeoutMma));
      if (!ok) break;
      tc_fence_after_sync();
      const int n_sub = subs(it);
      uint64_t at = static_cast<uint64_t>(stage * stage_bytes) >> 4;
      for (int j = 0; j < n_sub; ++j, at += sub_off) {
        const uint64_t wd = w_desc0 + at, xd = x_desc0 + at + x_off;
#pragma unroll
        for (int k = 0; k < kBK / kUmmaK; ++k) {
          umma_f16_cta1_if(el, tmem_base, wd + k * kWStep, xd + k * kXStep, idesc, acc);
          if (kGate) umma_f16_cta1_if(el, d_up, wd + up_off + k * kWStep, xd + k * kXStep, idesc, acc);
          acc = 1;
        }
      }
      umma_commit_cta1_if(el, &empty_bar[stage]);
      if (++stage == sh.stages) { stage = 0; phase ^= 1u; }
    }
    if (ok) {
      umma_commit_cta1_if(el, done_bar);
    } else {
      umma_commit_cta1_if(el, drain_bar);
      if (lane == 0) mbar_wait_drain(drain_bar, 0);
    }
  }
  __syncwarp();

  // ---- epilogue ----
  // Rounds of `chunk` tokens: each CTA stages its accumulators in the idle
  // pipeline stages ([accumulator][token][row of w], fp32; warps 2..9, two to a
  // quarter of the lanes), then takes every S-th token, adds up the S parts and
  // stores.  An item is one token's next four rows of w; items are dealt to all
  // threads, whatever `block` is.
  const uint32_t t_row = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
  bool got = true;
  if (warp >= 2 && lane == 0) got = mbar_wait(done_bar, 0, kDevTimeoutEpilogue);
  got = __shfl_sync(0xffffffffu, got, 0);
  tc_fence_after_sync();
  float* part = reinterpret_cast<float*>(smem);
  const int quads = (min(sh.block, (kMode == kRowsGateBwd ? sh.n_pad : sh.n) - n0) + 3) >> 2;
  const int step_t = kRowsThreads / quads, step_q = kRowsThreads - step_t * quads;
  for (int c0 = 0; c0 < tokens; c0 += sh.chunk) {
    const int c1 = min(sh.tokens_pad, c0 + sh.chunk);
    const int row = (warp & 3) * 32 + lane;
    if (warp >= 2 && (warp & 3) * 32 < sh.block) {
      for (int t0 = c0 + (warp >= 6 ? 16 : 0); t0 < c1; t0 += 32) {
#pragma unroll
        for (int a = 0; a < kAccs; ++a) {
          uint32_t g[16];
          tmem_ld_32x32b_x16(t_row + a * sh.tokens_pad + t0, g);
          tmem_ld_wait_regs16(g);
#pragma unroll
          for (int e = 0; e < 16; ++e) part[(a * sh.chunk + t0 - c0 + e) * 128 + row] = __uint_as_float(g[e]);
        }
      }
    }
    cluster_sync();
    const int share = got ? (min(c1, tokens) - c0 - rank + parts - 1) / parts : 0;  // tokens of this CTA
    int i = threadIdx.x / quads, q = threadIdx.x - i * quads;
    for (; i < share; i += step_t, q += step_q) {
      if (q >= quads) {
        q -= quads;
        if (++i >= share) break;
      }
      const int t = c0 + rank + parts * i;
      const int n = n0 + 4 * q;
      const int64_t row_t = t_tile + t;
      [[maybe_unused]] uint2 sg = make_uint2(0, 0), su = sg;
      if constexpr (kMode == kRowsGateBwd) {
        // Rows of g and u are padded to whole quads (what lies past n counts as 0).
        sg = *reinterpret_cast<const uint2*>(io.saved_g + row_t * io.ld_gu + n);
        su = *reinterpret_cast<const uint2*>(io.saved_u + row_t * io.ld_gu + n);
      }
      float4 r[kAccs];
      const float* at = part + (t - c0) * 128 + 4 * q;
      const int acc_step = sh.chunk * 128;
      switch (parts) {
        case 1: sum_parts<1, kAccs>(at, acc_step, r); break;
        case 2: sum_parts<2, kAccs>(at, acc_step, r); break;
        case 4: sum_parts<4, kAccs>(at, acc_step, r); break;
        default: sum_parts<8, kAccs>(at, acc_step, r); break;
      }
      const float v0[4] = {r[0].x, r[0].y, r[0].z, r[0].w};
      const float v1[4] = {r[kAccs - 1].x, r[kAccs - 1].y, r[kAccs - 1].z, r[kAccs - 1].w};
      const int left = min(sh.block - 4 * q, sh.n - n);  // rows of w from n on
      uint16_t* o = io.out + row_t * io.ld + n;
      if constexpr (kMode == kRowsPlain) {
        store_quad<kBf16>(o, v0, left);
      } else if constexpr (kMode == kRowsGateUp) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = gate_value(sh.activation, v0[e], v1[e]);
        store_quad<kBf16>(o, y, left);
        if (io.g) {
          store_quad<kBf16>(io.g + row_t * io.ld_gu + n, v0, left);
          store_quad<kBf16>(io.u + row_t * io.ld_gu + n, v1, left);
        }
      } else {
        const float2 g0 = unpack_16bit<kBf16>(sg.x), g1 = unpack_16bit<kBf16>(sg.y);
        const float2 u0 = unpack_16bit<kBf16>(su.x), u1 = unpack_16bit<kBf16>(su.y);
        const float g[4] = {g0.x, g0.y, g1.x, g1.y}, u[4] = {u0.x, u0.y, u1.x, u1.y};
        float dg[4], du[4], a[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float3 v = gate_grads(sh.activation, v0[e], g[e], u[e]);
          dg[e] = e < left ? v.x : 0.0f;
          du[e] = e < left ? v.y : 0.0f;
          a[e] = e < left ? v.z : 0.0f;
        }
        const int pad_left = sh.n_pad - n;
        store_quad<kBf16>(io.dg + row_t * io.ld_gu + n, dg, pad_left);
        store_quad<kBf16>(io.du + row_t * io.ld_gu + n, du, pad_left);
        store_quad<kBf16>(o, a, pad_left);
      }
    }
    cluster_sync();
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc<1>(tmem_base, tmem_cols);
  }
}

}  // namespace b200
