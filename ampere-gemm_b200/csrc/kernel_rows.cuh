// GEMM kernel for few rows of x (decoding): out[t][n] = sum_k x[t][k] w[n][k],
// or, with kGate, out[t][n] = act(g) u for w = [Wg; Wu].
//
// Such a product is bound by reading w once.  So the operands change places:
// a block of rows of w is the 128-row operand of the MMA (lane = row of w) and
// all rows of x, rounded up to 16, are its N columns.  Rows of w are dealt out
// evenly: every CTA takes `block` of them (not 128: lanes past `block` compute
// on whatever lies behind the tile in shared memory and are never read), so
// one wave of CTAs streams equal shares of w.  With a cluster of S CTAs each
// takes 1/S of K for S times as many rows, which cuts the re-reading of x (all
// of it, by every cluster) by S; the S parts are added up through distributed
// shared memory in a fixed order.
//
//   warp 0      TMA producer; warp 1 MMA issuer; warps 2..5 epilogue, thread =
//               row of w, so a store instruction writes 32 neighbours of one t.
//
// Launched with programmatic stream serialisation.  With `w_early`, w was not
// written by the kernel before this one on the stream: the first stages of w
// are requested before that kernel has finished, only x waits for it.
#pragma once

#include "epilogue_gate.cuh"
#include "gemm_common.cuh"

namespace b200 {

constexpr int kRowsMaxTokens = 256;  // N of one MMA
constexpr int kRowsMaxStages = 16;

struct RowsShape {
  int tokens;      // rows of x
  int tokens_pad;  // rounded up to 16: N of the MMAs
  int n;           // rows of w (of each half with kGate)
  int k_blocks;    // 64-wide blocks of K
  int block;       // rows of w per cluster (of each half), <= 128
  int block_pad;   // rounded up to 8
  int k_sub;       // 64-wide blocks of a stage
  int stages;
  int chunk;       // tokens per reduction round of a cluster
  int activation;
  int w_early;
  int tail;        // bytes after the stages that an MMA may read: a tile of fewer than 128 rows is read past its end
};

__host__ __device__ inline int rows_sub_bytes(const RowsShape& s, bool gate) {
  return ((gate ? 2 : 1) * s.block_pad + s.tokens_pad) * 128;
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

__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ float ld_shared_cluster_f32(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}

__device__ __forceinline__ float gate_value(int activation, float g, float u) {
  if (activation == 0) return activate<0, false>(g).f * u;
  if (activation == 1) return activate<1, false>(g).f * u;
  return activate<2, false>(g).f * u;
}

template <bool kBf16, bool kGate>
__global__ void __launch_bounds__(kThreads, 2)
    gemm_rows_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                     uint16_t* __restrict__ out, int64_t ld_out, const __grid_constant__ RowsShape sh) {
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
  const int n0 = static_cast<int>(blockIdx.x) / parts * sh.block;
  const int kb0 = static_cast<int>(static_cast<int64_t>(rank) * sh.k_blocks / parts);
  const int kb1 = static_cast<int>(static_cast<int64_t>(rank + 1) * sh.k_blocks / parts);
  const int num_stages = (kb1 - kb0 + sh.k_sub - 1) / sh.k_sub;
  uint32_t tmem_cols = 32;
  while (tmem_cols < static_cast<uint32_t>(kAccs * sh.tokens_pad)) tmem_cols *= 2;

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

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      const uint64_t pol_w = policy_evict_first();   // read once
      const uint64_t pol_x = policy_evict_last();    // read by every cluster
      auto subs = [&](int it) { return min(sh.k_sub, kb1 - kb0 - it * sh.k_sub); };
      auto load_w = [&](int it, int stage) {
        const int n_sub = subs(it);
        mbar_arrive_expect_tx(&full_bar[stage],
                              static_cast<uint32_t>(n_sub * (kAccs * sh.block + sh.tokens_pad) * 128));
        for (int j = 0; j < n_sub; ++j) {
          uint8_t* dst = smem + stage * stage_bytes + j * sub_bytes;
          const int k = (kb0 + it * sh.k_sub + j) * kBK;
          tma_load_2d(dst, &tmap_w, &full_bar[stage], k, n0, pol_w);
          if (kGate) tma_load_2d(dst + sh.block_pad * 128, &tmap_w, &full_bar[stage], k, sh.n + n0, pol_w);
        }
      };
      auto load_x = [&](int it, int stage) {
        const int n_sub = subs(it);
        for (int j = 0; j < n_sub; ++j)
          tma_load_2d(smem + stage * stage_bytes + j * sub_bytes + kAccs * sh.block_pad * 128, &tmap_x,
                      &full_bar[stage], (kb0 + it * sh.k_sub + j) * kBK, 0, pol_x);
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
      int issued = first;
      for (int it = first; it < num_stages; ++it) {
        const int stage = it % sh.stages;
        if (!mbar_wait(&empty_bar[stage], static_cast<uint32_t>(it / sh.stages - 1) & 1u, kDevTimeoutProducer)) {
          ok = false;
          break;
        }
        load_w(it, stage);
        load_x(it, stage);
        ++issued;
      }
      if (!ok) {
        // Let every load still in flight land before the CTA leaves.
        for (int it = max(0, issued - sh.stages); it < issued; ++it)
          mbar_wait_drain(&full_bar[it % sh.stages], static_cast<uint32_t>(it / sh.stages) & 1u);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc =
          make_idesc_f16_f32(128, static_cast<uint32_t>(sh.tokens_pad), Major::kK, Major::kK, kBf16);
      const uint32_t base = smem_u32(smem);
      bool ok = true;
      for (int it = 0; it < num_stages; ++it) {
        const int stage = it % sh.stages;
        ok = mbar_wait(&full_bar[stage], static_cast<uint32_t>(it / sh.stages) & 1u, kDevTimeoutMma);
        if (!ok) break;
        tc_fence_after_sync();
        const int n_sub = min(sh.k_sub, kb1 - kb0 - it * sh.k_sub);
        for (int j = 0; j < n_sub; ++j) {
          const uint32_t w_addr = base + stage * stage_bytes + j * sub_bytes;
          const uint32_t x_addr = w_addr + kAccs * sh.block_pad * 128;
#pragma unroll
          for (int k = 0; k < kBK / kUmmaK; ++k) {
            const uint64_t xd = make_desc_kmajor_sw128(x_addr + k * (kUmmaK * 2));
            const uint32_t acc = (it | j | k) != 0 ? 1u : 0u;
            umma_f16_cta1(tmem_base, make_desc_kmajor_sw128(w_addr + k * (kUmmaK * 2)), xd, idesc, acc);
            if (kGate)
              umma_f16_cta1(tmem_base + sh.tokens_pad,
                            make_desc_kmajor_sw128(w_addr + sh.block_pad * 128 + k * (kUmmaK * 2)), xd, idesc, acc);
          }
        }
        umma_commit_cta1(&empty_bar[stage]);
      }
      if (ok) {
        umma_commit_cta1(done_bar);
      } else {
        umma_commit_cta1(drain_bar);
        mbar_wait_drain(drain_bar, 0);
      }
    }
  }
  __syncwarp();

  // ---- epilogue: warps 2..5, thread = lane `row` of the accumulators ----
  const int row = (warp & 3) * 32 + lane;
  const int n = n0 + row;
  const bool mine = warp >= 2 && row < sh.block && n < sh.n;
  const uint32_t t_row = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
  bool got = true;
  if (warp >= 2) {
    if (lane == 0) got = mbar_wait(done_bar, 0, kDevTimeoutEpilogue);
    got = __shfl_sync(0xffffffffu, got, 0);
    tc_fence_after_sync();
  }
  if (parts == 1) {
    if (warp >= 2 && got) {
      for (int t0 = 0; t0 < sh.tokens; t0 += 16) {
        uint32_t g[16], u[16];
        tmem_ld_32x32b_x16(t_row + t0, g);
        if (kGate) tmem_ld_32x32b_x16(t_row + sh.tokens_pad + t0, u);
        tmem_ld_wait_regs16(g);
        if (kGate) tmem_ld_wait_regs16(u);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float v = __uint_as_float(g[e]);
          if (kGate) v = gate_value(sh.activation, v, __uint_as_float(u[e]));
          if (mine && t0 + e < sh.tokens)
            out[static_cast<int64_t>(t0 + e) * ld_out + n] =
                static_cast<uint16_t>(pack_16bit_rn<kBf16>(__float_as_uint(v), 0u));
        }
      }
    }
  } else {
    // Each round stages `chunk` tokens of the parts in the idle pipeline
    // stages ([accumulator][token][row]) and adds up every S-th of them.
    float* part = reinterpret_cast<float*>(smem);
    for (int c0 = 0; c0 < sh.tokens; c0 += sh.chunk) {
      const int c1 = min(sh.tokens_pad, c0 + sh.chunk);
      if (warp >= 2) {
        for (int t0 = c0; t0 < c1; t0 += 16) {
#pragma unroll
          for (int a = 0; a < kAccs; ++a) {
            uint32_t g[16];
            tmem_ld_32x32b_x16(t_row + a * sh.tokens_pad + t0, g);
            tmem_ld_wait_regs16(g);
#pragma unroll
            for (int e = 0; e < 16; ++e)
              part[(a * sh.chunk + t0 - c0 + e) * 128 + row] = __uint_as_float(g[e]);
          }
        }
      }
      cluster_sync();
      if (mine && got) {
        for (int t = c0 + rank; t < min(c1, sh.tokens); t += parts) {
          float v[kAccs];
#pragma unroll
          for (int a = 0; a < kAccs; ++a) {
            const uint32_t at = smem_u32(part + (a * sh.chunk + t - c0) * 128 + row);
            v[a] = 0.0f;
            for (int p = 0; p < parts; ++p) v[a] += ld_shared_cluster_f32(mapa_shared(at, p));
          }
          const float r = kGate ? gate_value(sh.activation, v[0], v[kAccs - 1]) : v[0];
          out[static_cast<int64_t>(t) * ld_out + n] =
              static_cast<uint16_t>(pack_16bit_rn<kBf16>(__float_as_uint(r), 0u));
        }
      }
      cluster_sync();
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc<1>(tmem_base, tmem_cols);
  }
}

}  // namespace b200
