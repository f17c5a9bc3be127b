// Epilogues of the gated feed-forward block for the 2-CTA GEMM kernel:
//
//   gate and up   g = x Wg^T, u = x Wu^T in one tile;  a = act(g) u
//   backward      da = dy Wo in the accumulator;       a, dg = da u act'(g), du = da act(g)
//
// Activations are computed in fp32 from the fp32 accumulators (forward) or
// from the saved 16-bit g and u (backward).  Both hide behind the MMAs of the
// next tile where the product is deep: 4001 x 4096 x 12288 fp16 forward 538 us
// (0.91 of the measured peak), 8192 x 4096 x 11008 bf16 forward with g and u
// stored 978 us (0.92), backward 607 us (0.74).
#pragma once

#include "gemm_common.cuh"

namespace b200 {

// Epilogues of the pair kernel.
constexpr int kEpiPlain = 0;    // C = alpha * acc + beta * C
constexpr int kEpiGateUp = 1;   // C = act(g) u, optionally g and u too
constexpr int kEpiGateBwd = 2;  // dg, du and a from da and the saved g, u

template <int kEpi>
struct FusedArgs {};

template <>
struct FusedArgs<kEpiGateUp> {
  CUtensorMap tmap_g, tmap_u;  // where g and u are kept for the backward pass
  int activation = 0;          // B200_ACT_*
  int save = 0;                // 0: g and u are not stored
};

template <>
struct FusedArgs<kEpiGateBwd> {
  const uint16_t* g = nullptr;  // the saved g and u, row pitch ld (elements)
  const uint16_t* u = nullptr;
  uint16_t* dg = nullptr;       // their gradients, the same pitch
  uint16_t* du = nullptr;
  uint16_t* a = nullptr;
  int64_t ld = 0, ld_a = 0;
  int activation = 0;
};

// act(g) and act'(g).  The exponentials and quotients are the approximate
// ones: their relative error, a few 2^-22, is far below the 16-bit rounding of
// what they end up in.
struct ActValue {
  float f, slope;
};

__device__ __forceinline__ float exp_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}
// 1 / (1 + exp(-x)); exp(-x) = infinity gives 0.
__device__ __forceinline__ float sigmoid_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + exp_approx(-x)));
  return r;
}

// The normal distribution function Phi(x), from erf(z) = 1 - (a1 t + ... + a5
// t^5) exp(-z^2), t = 1 / (1 + p z), z = |x| / sqrt 2 >= 0 (Abramowitz and
// Stegun 7.1.26, within 1.5e-7); `e` receives exp(-x^2 / 2).  A third of
// erfcf()'s instructions, which the epilogue does not hide altogether (at 4001
// x 4096 x 12288 the gate-and-up product takes 2.16 times the output
// projection's time with erfcf, 1.98 with this, 1.92 with silu).
__device__ __forceinline__ float normal_cdf(float x, float& e) {
  e = exp_approx(-0.5f * x * x);
  float t;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.3275911f * 0.70710678118654752f, fabsf(x), 1.0f)));
  float q = fmaf(1.061405429f, t, -1.453152027f);
  q = fmaf(q, t, 1.421413741f);
  q = fmaf(q, t, -0.284496736f);
  q = fmaf(q, t, 0.254829592f);
  const float tail = 0.5f * q * t * e;  // Phi(-|x|)
  return x < 0.0f ? tail : 1.0f - tail;
}

template <int kAct, bool kSlope>
__device__ __forceinline__ ActValue activate(float g) {
  ActValue r;
  r.slope = 0.0f;
  if constexpr (kAct == 0) {  // silu: g s(g)
    const float s = sigmoid_approx(g);
    r.f = g * s;
    if (kSlope) r.slope = s * (1.0f + g * (1.0f - s));
  } else if constexpr (kAct == 1) {  // gelu: g Phi(g)
    float e;
    const float cdf = normal_cdf(g, e);
    r.f = g * cdf;
    if (kSlope) r.slope = cdf + g * (0.39894228040143268f * e);
  } else {  // gelu with tanh: g (1 + tanh z) / 2 = g s(2z), z = sqrt(2/pi) (g + 0.044715 g^3)
    constexpr float kC = 0.79788456080286536f, kA = 0.044715f;
    const float s = sigmoid_approx(2.0f * kC * g * (1.0f + kA * g * g));
    r.f = g * s;
    // Where g^2 is infinite, s (1 - s) is 0: the bound keeps 0 * infinity out.
    if (kSlope) r.slope = s + g * (2.0f * s * (1.0f - s)) * fminf(kC * (1.0f + 3.0f * kA * g * g), 1.0e30f);
  }
  return r;
}

// Gate and up: the accumulator row holds g in columns [0, 128) and u in
// [128, 256).  Stores a at columns [n0, n0 + 128) of C and, when kept, g and u
// through their own maps.  `release` hands the accumulator back once it is in
// registers.
template <bool kBf16, int kAct, typename Release>
__device__ __forceinline__ void gate_up_chunks(const FusedArgs<kEpiGateUp>& fx, const CUtensorMap& tmap_c,
                                               const EpiParams& sc, uint32_t t_row, uint8_t* epi_buf,
                                               uint32_t epi_addr, int& sbuf, int lane, int n0, int y,
                                               Release&& release) {
#pragma unroll 1
  for (int c = 0; c < 2; ++c) {
    uint32_t pa[32], pg[32], pu[32];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t g[32], u[32];
      tmem_ld_32x32b_x32(t_row + c * kEpiCols + h * 32, g);
      tmem_ld_32x32b_x32(t_row + 128 + c * kEpiCols + h * 32, u);
      tmem_ld_wait_regs(g);
      tmem_ld_wait_regs(u);
      if (c == 1 && h == 1) release();
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float a[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
          a[i] = activate<kAct, false>(__uint_as_float(g[2 * e + i])).f * __uint_as_float(u[2 * e + i]);
        pa[16 * h + e] = pack_16bit_rn<kBf16>(__float_as_uint(a[0]), __float_as_uint(a[1]));
        pg[16 * h + e] = pack_16bit_rn<kBf16>(g[2 * e], g[2 * e + 1]);
        pu[16 * h + e] = pack_16bit_rn<kBf16>(u[2 * e], u[2 * e + 1]);
      }
    }
    const int x = n0 + c * kEpiCols;
    epi_store_block_packed<2>(&tmap_c, epi_buf, epi_addr, sbuf, lane, pa, x, y, sc);
    if (fx.save) {
      epi_store_block_packed<2>(&fx.tmap_g, epi_buf, epi_addr, sbuf, lane, pg, x, y, sc);
      epi_store_block_packed<2>(&fx.tmap_u, epi_buf, epi_addr, sbuf, lane, pu, x, y, sc);
    }
  }
}

template <bool kBf16, typename Release>
__device__ __forceinline__ void gate_up_epilogue(const FusedArgs<kEpiGateUp>& fx, const CUtensorMap& tmap_c,
                                                 const EpiParams& sc, uint32_t t_row, uint8_t* epi_buf,
                                                 uint32_t epi_addr, int& sbuf, int lane, int n0, int y,
                                                 Release&& release) {
  if (fx.activation == 0)
    gate_up_chunks<kBf16, 0>(fx, tmap_c, sc, t_row, epi_buf, epi_addr, sbuf, lane, n0, y, release);
  else if (fx.activation == 1)
    gate_up_chunks<kBf16, 1>(fx, tmap_c, sc, t_row, epi_buf, epi_addr, sbuf, lane, n0, y, release);
  else
    gate_up_chunks<kBf16, 2>(fx, tmap_c, sc, t_row, epi_buf, epi_addr, sbuf, lane, n0, y, release);
}

// Keeps the first `n` of a piece's eight elements (n <= 0: none), zeroes the others.
__device__ __forceinline__ uint4 keep_first(uint4 v, int n) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = n >= 2 * i + 2 ? w[i] : n == 2 * i + 1 ? (w[i] & 0xffffu) : 0u;
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Blocks of 32 rows x 32 columns in the backward epilogue.  In global memory
// lane l handles 16-byte piece l % 4 of rows l / 4, l / 4 + 8, ... (64-byte row
// pieces, eight rows an instruction).  In shared memory row r is at r * 64, its
// piece p at p ^ (r / 2) % 4: neither that mapping nor lane = row conflicts.
constexpr int kGateBlockBytes = 32 * 64;

__device__ __forceinline__ int gate_piece(int row, int piece) {
  return row * 64 + ((piece ^ ((row >> 1) & 3)) << 4);
}

// Reads the blocks of the saved g and u at column x, row y.  Their rows are
// padded to whole pieces; what lies past column N, or in pieces out of range,
// counts as 0.
__device__ __forceinline__ void gate_bwd_fetch(const FusedArgs<kEpiGateBwd>& fx, uint4 (&g)[4], uint4 (&u)[4],
                                               int lane, int x, int y, int M, int N) {
  const int col = x + (lane & 3) * 8;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = y + i * 8 + (lane >> 2);
    g[i] = u[i] = make_uint4(0, 0, 0, 0);
    if (row < M && col < N) {
      const int64_t off = static_cast<int64_t>(row) * fx.ld + col;
      g[i] = *reinterpret_cast<const uint4*>(fx.g + off);
      u[i] = *reinterpret_cast<const uint4*>(fx.u + off);
      if (col + 8 > N) {
        g[i] = keep_first(g[i], N - col);
        u[i] = keep_first(u[i], N - col);
      }
    }
  }
}

// Stores the block staged at `buf` to column x, row y of `out`.
__device__ __forceinline__ void gate_bwd_store(const uint8_t* buf, uint16_t* out, int64_t ld, int lane, int x, int y,
                                               int M, int N) {
  const int col = x + (lane & 3) * 8;
  if (col >= N) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2);
    if (y + r < M)
      *reinterpret_cast<uint4*>(out + static_cast<int64_t>(y + r) * ld + col) =
          *reinterpret_cast<const uint4*>(buf + gate_piece(r, lane & 3));
  }
}

// Backward: the accumulator row holds da at columns [n0, n0 + 128) from t_row
// on.  Per 32 columns, g and u go through the warp's staging buffers into the
// layout of the accumulator (lane = row), dg and du replace them there and
// leave by plain stores (zeros past column N), then a takes the first buffer.
// The next block's g and u are fetched meanwhile.  Eight warps share a tile:
// four took 43000 cycles for it (silu; measured at a depth of 512, where the
// MMAs take 4100), which a depth of 4096 (32800) does not hide.
template <bool kBf16, int kAct, typename Release>
__device__ __forceinline__ void gate_bwd_chunks(const FusedArgs<kEpiGateBwd>& fx, uint4 (&gv)[4], uint4 (&uv)[4],
                                                uint32_t t_row, uint8_t* epi_buf, int lane, int n0, int y, int M,
                                                int N, Release&& release) {
  uint8_t* buf0 = epi_buf;
  uint8_t* buf1 = epi_buf + kGateBlockBytes;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    const int x = n0 + c * 32;
    uint32_t d[32];
    tmem_ld_32x32b_x32(t_row + c * 32, d);
    tmem_ld_wait_regs(d);
    if (c == 3) release();
    if (x >= N) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = gate_piece(i * 8 + (lane >> 2), lane & 3);
      *reinterpret_cast<uint4*>(buf0 + at) = gv[i];
      *reinterpret_cast<uint4*>(buf1 + at) = uv[i];
    }
    __syncwarp();
    if (c < 3) gate_bwd_fetch(fx, gv, uv, lane, x + 32, y, M, N);
    uint32_t pa[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = gate_piece(lane, j);
      const uint4 gq = *reinterpret_cast<const uint4*>(buf0 + at);
      const uint4 uq = *reinterpret_cast<const uint4*>(buf1 + at);
      const uint32_t gw[4] = {gq.x, gq.y, gq.z, gq.w}, uw[4] = {uq.x, uq.y, uq.z, uq.w};
      uint32_t dg[4], du[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 g = unpack_16bit<kBf16>(gw[e]), u = unpack_16bit<kBf16>(uw[e]);
        const ActValue v0 = activate<kAct, true>(g.x), v1 = activate<kAct, true>(g.y);
        const float d0 = __uint_as_float(d[8 * j + 2 * e]), d1 = __uint_as_float(d[8 * j + 2 * e + 1]);
        pa[4 * j + e] = pack_16bit_rn<kBf16>(__float_as_uint(v0.f * u.x), __float_as_uint(v1.f * u.y));
        dg[e] = pack_16bit_rn<kBf16>(__float_as_uint(d0 * u.x * v0.slope), __float_as_uint(d1 * u.y * v1.slope));
        du[e] = pack_16bit_rn<kBf16>(__float_as_uint(d0 * v0.f), __float_as_uint(d1 * v1.f));
      }
      *reinterpret_cast<uint4*>(buf0 + at) = make_uint4(dg[0], dg[1], dg[2], dg[3]);
      *reinterpret_cast<uint4*>(buf1 + at) = make_uint4(du[0], du[1], du[2], du[3]);
    }
    __syncwarp();
    gate_bwd_store(buf0, fx.dg, fx.ld, lane, x, y, M, N);
    gate_bwd_store(buf1, fx.du, fx.ld, lane, x, y, M, N);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<uint4*>(buf0 + gate_piece(lane, j)) =
          make_uint4(pa[4 * j], pa[4 * j + 1], pa[4 * j + 2], pa[4 * j + 3]);
    __syncwarp();
    gate_bwd_store(buf0, fx.a, fx.ld_a, lane, x, y, M, N);
    __syncwarp();
  }
}

template <bool kBf16, typename Release>
__device__ __forceinline__ void gate_bwd_epilogue(const FusedArgs<kEpiGateBwd>& fx, uint4 (&gv)[4], uint4 (&uv)[4],
                                                  uint32_t t_row, uint8_t* epi_buf, int lane, int n0, int y, int M,
                                                  int N, Release&& release) {
  if (fx.activation == 0)
    gate_bwd_chunks<kBf16, 0>(fx, gv, uv, t_row, epi_buf, lane, n0, y, M, N, release);
  else if (fx.activation == 1)
    gate_bwd_chunks<kBf16, 1>(fx, gv, uv, t_row, epi_buf, lane, n0, y, M, N, release);
  else
    gate_bwd_chunks<kBf16, 2>(fx, gv, uv, t_row, epi_buf, lane, n0, y, M, N, release);
}

}  // namespace b200
