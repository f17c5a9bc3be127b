// Layer norm over the last dimension, forward and backward.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r
//   y  = h w + b
//   with q = dy w:  dx = r (q - mean(q) - h mean(q h))
//   dw = sum over rows of dy h,  db = sum over rows of dy
//
// Bound by memory: forward reads x and writes y once, backward reads x and dy
// and writes dx once.  Measured, of the measured copy bandwidth: 20011 x 5120
// bf16 forward 71 us (0.88); 16384 x 4096 bf16 with fp32 weights 49 us forward
// (0.84), 77 + 5 backward (0.75); 8 x 4096 fp16 3.5 us (L2 cold).  What remains is the issue
// of instructions (half the slots) and the wait for a row's sums.  A row stays
// in registers, in its own type, between the passes over it; all sums are in
// fp32 and y, dx, dw and db are rounded once.  Every sum has a fixed order, so
// results do not change from run to run.
#include <algorithm>
#include <cstdint>

#include "elem_types.cuh"
#include "host_common.cuh"

namespace b200 {
namespace {

constexpr int kMaxRowThreads = 512;  // threads of a row that stays in registers: 128 registers each
constexpr int kLongThreads = 1024;   // threads of a longer row

__device__ __forceinline__ void pdl_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the `width` lanes (8, 16 or 32, aligned) that share a row.
__device__ __forceinline__ float lanes_sum(float v, int width) {
  if (width == 32) return warp_sum(v);
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 2);
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  if (width == 16) v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v;
}

// red[0] + ... + red[n - 1], n <= 32, read four at a time by every thread.
__device__ __forceinline__ float sum_of(const float* red, int n) {
  float s = 0.0f;
  for (int i = 0; i < n; i += 4) {
    const float4 r = *reinterpret_cast<const float4*>(red + i);
    s += r.x;
    if (i + 1 < n) s += r.y;
    if (i + 2 < n) s += r.z;
    if (i + 3 < n) s += r.w;
  }
  return s;
}

// Sum over the `tpr` threads of one row: lanes of a warp, or the whole block;
// `red` is then 32 floats that no thread still reads from the sum before the
// last.
__device__ __forceinline__ float row_sum(float v, int tpr, float* red) {
  if (tpr <= 32) return lanes_sum(v, tpr);
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return sum_of(red, tpr >> 5);
}

// The same for N rows at once.
template <int N>
__device__ __forceinline__ void row_sums(float (&v)[N], int tpr, float (*red)[32]) {
  if (tpr <= 32) {
#pragma unroll
    for (int r = 0; r < N; ++r) v[r] = lanes_sum(v[r], tpr);
    return;
  }
#pragma unroll
  for (int r = 0; r < N; ++r) {
    v[r] = warp_sum(v[r]);
    if ((threadIdx.x & 31) == 0) red[r][threadIdx.x >> 5] = v[r];
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < N; ++r) v[r] = sum_of(red[r], tpr >> 5);
}

// Where a thread's packs of a row lie: pack j at (j * threads of the row +
// threadIdx.x) * VEC.  With TPR != 0 the row has TPR threads and exactly
// TPR * NV packs, so offsets are constants and nothing is checked.
template <int VEC, int TPR>
struct Columns {
  int cols;
  __device__ __forceinline__ int at(int j) const {
    return (j * (TPR ? TPR : static_cast<int>(blockDim.x)) + static_cast<int>(threadIdx.x)) * VEC;
  }
  __device__ __forceinline__ bool has(int j) const { return TPR != 0 || at(j) < cols; }
};

// A thread's packs of a row; those past its end (or of no row) are zero.
template <typename T, int VEC, int NV, int TPR>
__device__ __forceinline__ void load_row(Pack<T, VEC> (&v)[NV], const T* row, const Columns<VEC, TPR>& col,
                                         bool active) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    v[j] = Pack<T, VEC>{};
    if (active && col.has(j)) v[j] = load_pack<T, VEC>(row + col.at(j));
  }
}

template <typename T, int VEC, int NV, int TPR>
__device__ __forceinline__ void store_row(T* row, const Pack<T, VEC> (&v)[NV], const Columns<VEC, TPR>& col) {
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (col.has(j)) store_pack<T, VEC>(row + col.at(j), v[j]);
}

// 1 / sqrt(v) for v >= 0: the approximate one after a Newton step (within
// 2^-23 of it); 0 and infinity as they are.
__device__ __forceinline__ float inverse_sqrt(float v) {
  const float r = rsqrtf(v);
  const float s = fmaf(0.5f * r, fmaf(-v * r, r, 1.0f), r);
  return v > 0.0f && v < __builtin_huge_valf() ? s : r;
}

// fn for each pair of a pack's elements (a single one with 0).
template <typename T, int VEC, typename Fn>
__device__ __forceinline__ void for_pairs(const Pack<T, VEC>& p, Fn&& fn) {
  if constexpr (VEC == 1) {
    fn(make_float2(to_f32(p.v), 0.0f));
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) fn(p.pair(i));
  }
}

// Asynchronous copy of 16 bytes into shared memory; a thread's copies are
// counted by its own commit groups.
__device__ __forceinline__ void copy_async_16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src)
               : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Rows that a thread of the forward takes at once: two for 16-bit rows with fp32
// weights, which are most of what the L1 cache delivers, where the row fills its
// threads exactly (16384 x 4096: 59 -> 54 us, 8192 x 8192: 70 -> 64, 20000 x 768:
// 15.4 -> 13.5).  With weights of the row's type one, for twice the blocks (30000
// x 2560: 65 us against 75, 20011 x 5120: 80 against 82).
template <typename T, typename W>
__host__ __device__ constexpr int fwd_rows_at_once(int tpr) {
  return tpr != 0 && sizeof(W) > sizeof(T) ? 2 : 1;
}

// Ring slots of the forward, each of the rows that are taken at once, and their
// bytes of a thread; none where a slot would be more than 128 bytes.  For 16-bit
// rows of two warps or more (us with and without: 20011 x 5120 69, 75; 16384 x
// 4096 with fp32 weights 47, 52; 8192 x 8192 with them 48.5, 58; 4096 x 16384 51,
// 56); rows of a warp and fp32 rows have enough on their way in registers (65536
// x 1024 fp16 46, 43; 8192 x 5120 fp32 56.5, 54).
template <typename T, typename W, int VEC, int NV, int TPR>
struct FwdRing {
  static constexpr int kSlot = fwd_rows_at_once<T, W>(TPR) * NV * 16;
  static constexpr bool kUsed = TPR > 32 && sizeof(T) == 2 && VEC == 8 && kSlot <= 128;
  static constexpr int kSlots = kUsed ? (kSlot > 64 ? 2 : 3) : 0;
  static constexpr size_t kBytes = static_cast<size_t>(kSlots) * kSlot;
};

// Forward.  blockDim = (threads of a row, rows of a block).  The blocks are
// resident and loop over rows.  With FwdRing, rows arrive through a ring in
// shared memory in which every thread reads only what it requested itself.
template <typename T, typename W, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(TPR ? (TPR > 128 ? TPR : 128) : kMaxRowThreads)
    layer_norm_fwd_kernel(const T* __restrict__ x, const W* __restrict__ w, const W* __restrict__ b,
                          T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t rows,
                          int cols, int64_t ldx, int64_t ldy, float eps) {
  constexpr int kRows = fwd_rows_at_once<T, W>(TPR);
  constexpr int kSlots = FwdRing<T, W, VEC, NV, TPR>::kSlots;
  extern __shared__ __align__(16) uint8_t dyn[];  // the ring
  __shared__ __align__(16) float red[2][kRows][32];
  pdl_wait();
  const Columns<VEC, TPR> col{cols};
  const int tpr = TPR ? TPR : static_cast<int>(blockDim.x);
  const float inv_n = 1.0f / static_cast<float>(cols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.y;
  const int64_t x_step = step * ldx, y_step = step * ldy;
  int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const T* xr = x + row * ldx;
  T* yr = y + row * ldy;
  const int threads = tpr * blockDim.y;
  Pack<T, VEC>* ring = reinterpret_cast<Pack<T, VEC>*>(dyn) + threadIdx.y * tpr + threadIdx.x;
  int64_t next = row;  // the row requested next
  const T* xn = xr;
  auto request = [&](int slot) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (next + r * step < rows) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
          copy_async_16(ring + ((slot * kRows + r) * NV + j) * threads, xn + r * x_step + col.at(j));
      }
    }
    copy_async_commit();
    next += kRows * step;
    xn += kRows * x_step;
  };
  int slot = 0;
  if constexpr (kSlots > 0) {
#pragma unroll
    for (int i = 0; i < kSlots - 1; ++i) request(i);
  }
  // The rows of a block take their turns together: row - threadIdx.y is the same for all.
  for (; row - threadIdx.y < rows; row += kRows * step, xr += kRows * x_step, yr += kRows * y_step) {
    bool active[kRows];
    Pack<T, VEC> v[kRows][NV];
    float mu[kRows], rstd[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      active[r] = row + r * step < rows;
      if constexpr (kSlots == 0) load_row<T, VEC, NV>(v[r], xr + r * x_step, col, active[r]);
    }
    if constexpr (kSlots > 0) {
      request(slot == 0 ? kSlots - 1 : slot - 1);
      copy_async_wait<kSlots - 1>();
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          v[r][j] = Pack<T, VEC>{};
          if (active[r]) v[r][j] = ring[((slot * kRows + r) * NV + j) * threads];
        }
      }
      slot = slot == kSlots - 1 ? 0 : slot + 1;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      float2 s2 = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < NV; ++j)
        for_pairs<T, VEC>(v[r][j], [&](float2 f) { s2 = add2(s2, f); });
      mu[r] = s2.x + s2.y;
    }
    row_sums(mu, tpr, red[0]);
    // The centred squares are summed in a second pass over the registers:
    // sum(x^2) - n mu^2 would lose the variance of a row with a large mean.
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      mu[r] *= inv_n;
      const float2 minus_mu = pair_of(-mu[r]);
      float2 q2 = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (col.has(j))
          for_pairs<T, VEC>(v[r][j], [&](float2 f) {
            f = add2(f, minus_mu);
            if (VEC == 1) f.y = 0.0f;
            q2 = fma2(f, f, q2);
          });
      }
      rstd[r] = q2.x + q2.y;
    }
    row_sums(rstd, tpr, red[1]);
#pragma unroll
    for (int r = 0; r < kRows; ++r) rstd[r] = inverse_sqrt(rstd[r] * inv_n + eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!col.has(j)) continue;
      const int c = col.at(j);
      if constexpr (VEC == 1) {
        const float wc = w ? to_f32(w[c]) : 1.0f, bc = b ? to_f32(b[c]) : 0.0f;
#pragma unroll
        for (int r = 0; r < kRows; ++r)
          if (active[r]) yr[r * y_step + c] = from_f32<T>(fmaf((to_f32(v[r][j].v) - mu[r]) * rstd[r], wc, bc));
      } else {
        Pack<W, VEC> pw, pb;
        if (w) pw = load_pack<W, VEC>(w + c);
        if (b) pb = load_pack<W, VEC>(b + c);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float2 minus_mu = pair_of(-mu[r]), r2 = pair_of(rstd[r]);
          Pack<T, VEC> o;
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) {
            float2 f = mul2(add2(v[r][j].pair(i), minus_mu), r2);
            if (w) f = mul2(f, pw.pair(i));
            if (b) f = add2(f, pb.pair(i));
            o.set_pair(i, f);
          }
          if (active[r]) store_pack<T, VEC>(yr + r * y_step + c, o);
        }
      }
    }
    if (threadIdx.x == 0) {
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        if (active[r]) {
          if (mean_out) mean_out[row + r * step] = mu[r];
          if (rstd_out) rstd_out[row + r * step] = rstd[r];
        }
    }
  }
}

// Forward for rows longer than the registers of a block hold: one block a
// row, which is read three times (the second and third from L2).
template <typename T, typename W>
__global__ void __launch_bounds__(kLongThreads)
    layer_norm_fwd_long_kernel(const T* __restrict__ x, const W* __restrict__ w, const W* __restrict__ b,
                               T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                               int64_t rows, int cols, int64_t ldx, int64_t ldy, float eps) {
  __shared__ __align__(16) float red[2][32];
  pdl_wait();
  const float inv_n = 1.0f / static_cast<float>(cols);
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * ldx;
    float s = 0.0f;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) s += to_f32(xr[c]);
    const float mu = row_sum(s, blockDim.x, red[0]) * inv_n;
    float q = 0.0f;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
      const float d = to_f32(xr[c]) - mu;
      q = fmaf(d, d, q);
    }
    const float rstd = inverse_sqrt(row_sum(q, blockDim.x, red[1]) * inv_n + eps);
    for (int c = threadIdx.x; c < cols; c += blockDim.x)
      y[row * ldy + c] = from_f32<T>(
          fmaf((to_f32(xr[c]) - mu) * rstd, w ? to_f32(w[c]) : 1.0f, b ? to_f32(b[c]) : 0.0f));
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[row] = mu;
      if (rstd_out) rstd_out[row] = rstd;
    }
  }
}

template <int N>
__device__ __forceinline__ float element(const float2 (&f)[N], int e) {
  return e & 1 ? f[e / 2].y : f[e / 2].x;
}

constexpr int kBwdThreads = 512;  // of a block, all its rows together
// Rows on their way while one is worked on, with NV packs a thread.
template <int NV>
constexpr int kAhead = NV <= 2 ? 3 : 1;

// Backward.  Threads and packs as in the forward kernel; with several rows in
// a block, each row's threads are whole warps with their own barrier, or lanes
// of a warp.  A thread keeps the same columns for all its rows, so it sums
// their dw and db in registers; a block writes its sums once, as row
// blockIdx.x of `part` (gridDim.x x 2 x cols: dw, then db), and
// layer_norm_bwd_reduce_kernel adds those rows up.  With 16-byte packs, rows
// arrive through a ring in shared memory in which every thread reads only what
// it requested itself: no barrier, and no registers for rows on their way.
// 128 registers a thread also where only 320 threads make a block (8192 x 5120
// fp32: 86 us, against 109 for two blocks an SM, which spill).
template <typename T, typename W, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(kBwdThreads)
    layer_norm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const W* __restrict__ w,
                          const float* __restrict__ mean, const float* __restrict__ rstd_in, T* __restrict__ dx,
                          float* __restrict__ part, int64_t rows, int cols, int64_t lddy, int64_t ldx, int64_t lddx) {
  constexpr bool kAsync = VEC * sizeof(T) == 16;
  constexpr int kSlots = kAhead<NV> + 1;
  __shared__ float2 red[2][kBwdThreads / 32];
  extern __shared__ __align__(16) uint8_t dyn[];  // the ring; after the loop the block's column sums
  pdl_wait();
  const Columns<VEC, TPR> col{cols};
  const int tpr = TPR ? TPR : static_cast<int>(blockDim.x);
  const int tid = threadIdx.y * tpr + threadIdx.x;
  const int threads = tpr * blockDim.y;
  const int warps = tpr >> 5;  // of a row
  const float inv_n = 1.0f / static_cast<float>(cols);
  constexpr int kPairs = VEC * NV / 2;
  float2 dw[kPairs], db[kPairs];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) dw[i] = db[i] = make_float2(0.0f, 0.0f);
  Pack<W, VEC> wv[NV];
  if (w) load_row<W, VEC, NV>(wv, w, col, true);
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.y;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  Pack<T, VEC>* ring = reinterpret_cast<Pack<T, VEC>*>(dyn) + tid;  // [slot][x, dy][j][thread]
  int64_t next = row0;  // the row requested next
  const T* xn = x + next * ldx;
  const T* gn = dy + next * lddy;
  auto request = [&](int slot) {
    if (next < rows) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (col.has(j)) {
          copy_async_16(ring + ((slot * 2 + 0) * NV + j) * threads, xn + col.at(j));
          copy_async_16(ring + ((slot * 2 + 1) * NV + j) * threads, gn + col.at(j));
        }
      }
    }
    copy_async_commit();
    next += step;
    xn += step * ldx;
    gn += step * lddy;
  };
  if (kAsync) {
#pragma unroll
    for (int i = 0; i < kAhead<NV>; ++i) request(i);
  }
  int parity = 0, slot = 0;
  float next_mu = row0 < rows ? mean[row0] : 0.0f, next_rstd = row0 < rows ? rstd_in[row0] : 0.0f;
  T* dr = dx + row0 * lddx;
  for (int64_t row = row0; row - threadIdx.y < rows; row += step, dr += step * lddx) {
    const bool active = row < rows;
    Pack<T, VEC> xv[NV], gv[NV];
    if (kAsync) {
      request(slot == 0 ? kSlots - 1 : slot - 1);
      copy_async_wait<kAhead<NV>>();
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        xv[j] = gv[j] = Pack<T, VEC>{};
        if (active && col.has(j)) {
          xv[j] = ring[((slot * 2 + 0) * NV + j) * threads];
          gv[j] = ring[((slot * 2 + 1) * NV + j) * threads];
        }
      }
      slot = slot == kSlots - 1 ? 0 : slot + 1;
    } else {
      load_row<T, VEC, NV>(xv, x + row * ldx, col, active);
      load_row<T, VEC, NV>(gv, dy + row * lddy, col, active);
    }
    const float mu = next_mu, rstd = next_rstd;
    if (row + step < rows) {
      next_mu = mean[row + step];
      next_rstd = rstd_in[row + step];
    }
    // h and q; elements past the end have x = dy = 0, so all they add is 0.
    float2 h[kPairs], q[kPairs], acc1 = make_float2(0.0f, 0.0f), acc2 = acc1;
    unpack<T, VEC, NV>(xv, h);
    unpack<T, VEC, NV>(gv, q);
    const float2 minus_mu = pair_of(-mu), r2 = pair_of(rstd);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      h[i] = mul2(add2(h[i], minus_mu), r2);
      dw[i] = fma2(q[i], h[i], dw[i]);
      db[i] = add2(db[i], q[i]);
    }
    if (w) {
      float2 c2[kPairs];
      unpack<W, VEC, NV>(wv, c2);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) q[i] = mul2(q[i], c2[i]);
    }
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      acc1 = add2(acc1, q[i]);
      acc2 = fma2(q[i], h[i], acc2);
    }
    float s1 = acc1.x + acc1.y, s2 = acc2.x + acc2.y;
    if (tpr <= 32) {
      s1 = lanes_sum(s1, tpr);
      s2 = lanes_sum(s2, tpr);
    } else {
      // Two buffers in turn: one barrier a row is enough.
      s1 = warp_sum(s1);
      s2 = warp_sum(s2);
      if ((tid & 31) == 0) red[parity][tid >> 5] = make_float2(s1, s2);
      if (blockDim.y == 1)
        __syncthreads();
      else
        asm volatile("bar.sync %0, %1;" ::"r"(threadIdx.y + 1), "r"(tpr) : "memory");
      s1 = s2 = 0.0f;
      const float2* r = red[parity] + threadIdx.y * warps;
      for (int i = 0; i < warps; ++i) {
        s1 += r[i].x;
        s2 += r[i].y;
      }
      parity ^= 1;
    }
    if (active) {
      const float2 m1 = pair_of(-s1 * inv_n), m2 = pair_of(-s2 * inv_n);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) q[i] = mul2(fma2(h[i], m2, add2(q[i], m1)), r2);
      repack<T, VEC, NV>(q, xv);
      store_row<T, VEC, NV>(dr, xv, col);
    }
  }
  if (!part) return;
  float* out = part + static_cast<int64_t>(blockIdx.x) * 2 * cols;
  if (blockDim.y == 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * VEC;
      if (c < cols) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          out[c + e] = element(dw, j * VEC + e);
          out[cols + c + e] = element(db, j * VEC + e);
        }
      }
    }
    return;
  }
  // The block's rows are added up in shared memory, in order.
  float* col_sum = reinterpret_cast<float*>(dyn);  // [2][cols]
  __syncthreads();
  for (int yy = 0; yy < static_cast<int>(blockDim.y); ++yy) {
    if (threadIdx.y == yy) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * blockDim.x + threadIdx.x) * VEC;
        if (c < cols) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            col_sum[c + e] = element(dw, j * VEC + e) + (yy ? col_sum[c + e] : 0.0f);
            col_sum[cols + c + e] = element(db, j * VEC + e) + (yy ? col_sum[cols + c + e] : 0.0f);
          }
        }
      }
    }
    __syncthreads();
  }
  for (int c = tid; c < 2 * cols; c += threads) out[c] = col_sum[c];
}

// dx for rows longer than a block's registers hold: one block a row.
template <typename T, typename W>
__global__ void __launch_bounds__(kLongThreads)
    layer_norm_bwd_long_kernel(const T* __restrict__ dy, const T* __restrict__ x, const W* __restrict__ w,
                               const float* __restrict__ mean, const float* __restrict__ rstd_in, T* __restrict__ dx,
                               int64_t rows, int cols, int64_t lddy, int64_t ldx, int64_t lddx) {
  __shared__ __align__(16) float red[2][32];
  pdl_wait();
  const float inv_n = 1.0f / static_cast<float>(cols);
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * ldx;
    const T* gr = dy + row * lddy;
    const float mu = mean[row], rstd = rstd_in[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
      const float q = to_f32(gr[c]) * (w ? to_f32(w[c]) : 1.0f);
      s1 += q;
      s2 = fmaf(q, (to_f32(xr[c]) - mu) * rstd, s2);
    }
    s1 = row_sum(s1, blockDim.x, red[0]) * inv_n;
    s2 = row_sum(s2, blockDim.x, red[1]) * inv_n;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
      const float q = to_f32(gr[c]) * (w ? to_f32(w[c]) : 1.0f);
      dx[row * lddx + c] = from_f32<T>(rstd * (q - s1 - (to_f32(xr[c]) - mu) * rstd * s2));
    }
  }
}

// Partial dw and db of long rows: thread = column, blockIdx.y = the rows'
// residue modulo gridDim.y; same `part` layout as layer_norm_bwd_kernel.
template <typename T>
__global__ void layer_norm_bwd_columns_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                              const float* __restrict__ mean, const float* __restrict__ rstd,
                                              float* __restrict__ part, int64_t rows, int cols, int64_t lddy,
                                              int64_t ldx) {
  pdl_wait();
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= cols) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float g = to_f32(dy[row * lddy + c]);
    dw = fmaf(g, (to_f32(x[row * ldx + c]) - mean[row]) * rstd[row], dw);
    db += g;
  }
  part[static_cast<int64_t>(blockIdx.y) * 2 * cols + c] = dw;
  part[static_cast<int64_t>(blockIdx.y) * 2 * cols + cols + c] = db;
}

// dw and db: column sums of the `parts` rows of `part`.  32 columns a block,
// blockDim.y threads a column; blockIdx.y = 0 for dw, 1 for db.
template <typename W>
__global__ void layer_norm_bwd_reduce_kernel(const float* __restrict__ part, int parts, int cols, W* __restrict__ dw,
                                             W* __restrict__ db) {
  __shared__ float sums[32][33];
  pdl_wait();
  W* out = blockIdx.y == 0 ? dw : db;
  if (!out) return;
  const int c = blockIdx.x * 32 + threadIdx.x;
  float s = 0.0f;
  if (c < cols)
    for (int p = threadIdx.y; p < parts; p += blockDim.y)
      s += part[(static_cast<int64_t>(p) * 2 + blockIdx.y) * cols + c];
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < cols) {
    for (int i = 1; i < static_cast<int>(blockDim.y); ++i) s += sums[i][threadIdx.x];
    out[c] = from_f32<W>(s);
  }
}

template <int V>
using IntC = std::integral_constant<int, V>;

struct RowPlan {
  int nv = 0;       // packs a thread holds (0: the row does not fit a block's registers)
  int threads = 0;  // threads of a row
  int rows = 1;     // rows of a block
};

// Threads of a row with `nv` packs a thread: 8 or 16 lanes, or whole warps.
int row_threads(int packs, int nv) {
  const int t = (packs + nv - 1) / nv;
  return t <= 8 ? 8 : t <= 16 ? 16 : (t + 31) / 32 * 32;
}

// Packs a thread holds, for which kernels are built.  A 16-byte pack; a pair of
// 16-bit elements, where rows start on 4 bytes only; or one element.
constexpr int kFwdNv[] = {1, 2, 3, 4, 8, 16};
constexpr int kBwdNv[] = {1, 2, 4, 8, 16};
template <int VEC>
constexpr bool fwd_built(int nv) {
  return nv <= (VEC >= 4 ? 8 : 16) && (nv != 3 || VEC == 8);
}
// Two registers a column for dw and db beside the packs of x, dy and w.
template <int VEC>
constexpr bool bwd_built(int nv) {
  return VEC == 8 ? nv <= 4 : VEC == 4 ? nv == 2 || nv == 4 : VEC == 2 ? nv == 4 || nv == 8 : nv == 8 || nv == 16;
}

// Threads of a row for which kernels are built that the row fills exactly, with
// constant offsets and no checks: those bound this kernel otherwise (16384 x
// 4096 bf16 with fp32 weights: forward 58 us against 69, backward 76 against 84).
constexpr bool exact_threads(int t) {
  return t == 32 || t == 64 || t == 96 || t == 128 || t == 160 || t == 192 || t == 256 || t == 320 || t == 512;
}
template <int VEC>
constexpr bool fwd_exact(int nv, int t) {
  // 16 columns a thread for 2560, which 24, 32 and 64 do not divide into whole warps.
  return VEC >= 4 && exact_threads(t) && t <= 256 &&
         (nv * VEC == 24 || nv * VEC == 32 || nv * VEC == 64 || (nv * VEC == 16 && t == 160));
}
template <int VEC>
constexpr bool bwd_exact(int nv, int t) {
  return VEC >= 4 && exact_threads(t) && (nv * VEC == 8 || nv * VEC == 16);
}

// Forward: as many columns a thread as leave 12 warps an SM (a thread's share
// of the reductions and of the addressing is what costs), up to 32, and few
// idle threads.  Rows of a warp or less go 128 threads to a block, longer ones
// take a block each.
template <int VEC>
RowPlan plan_fwd(int packs, int64_t rows, int sm_count) {
  RowPlan best;
  double best_score = 0.0;
  for (int nv : kFwdNv) {
    if (!fwd_built<VEC>(nv)) continue;
    const int t = row_threads(packs, nv);
    if (t > kMaxRowThreads) continue;
    const double fill = std::min(1.0, (double)rows * t / (12.0 * 32 * sm_count));
    const double used = (double)packs / ((double)t * nv);
    double score = fill * used * std::min(1.0, 0.5 + nv * VEC / 64.0);
    if (packs == t * nv && fwd_exact<VEC>(nv, t)) score *= 1.3;
    if (score > best_score) {
      best_score = score;
      best = RowPlan{nv, t, t > 32 ? 1 : 128 / t};
    }
  }
  return best;
}

// Backward: the plan that keeps most of a block's 512 threads busy, of equal
// ones that with the most columns a thread.
template <int VEC>
RowPlan plan_bwd(int packs) {
  RowPlan best;
  double best_score = 0.0;
  for (int nv : kBwdNv) {
    if (!bwd_built<VEC>(nv)) continue;
    const int t = row_threads(packs, nv);
    if (t > kBwdThreads) continue;
    const int rows = kBwdThreads / t;
    // Beyond 16 columns a thread, registers spill.
    double score = (double)packs / ((double)t * nv) * (rows * t) / kBwdThreads * (nv * VEC > 16 ? 0.5 : 1.0);
    if (packs == t * nv && bwd_exact<VEC>(nv, t)) score = 1.2;
    if (score >= 0.97 * best_score) {
      best_score = std::max(score, best_score);
      best = RowPlan{nv, t, rows};
    }
  }
  return best;
}

// fn(threads of a row as a constant) for an exact plan, else fn(0).
template <typename Fn>
int with_tpr(bool exact, int tpr, Fn&& fn) {
  switch (exact ? tpr : 0) {
    case 32: return fn(IntC<32>{});
    case 64: return fn(IntC<64>{});
    case 96: return fn(IntC<96>{});
    case 128: return fn(IntC<128>{});
    case 160: return fn(IntC<160>{});
    case 192: return fn(IntC<192>{});
    case 256: return fn(IntC<256>{});
    case 320: return fn(IntC<320>{});
    case 512: return fn(IntC<512>{});
    default: return fn(IntC<0>{});
  }
}

template <typename Fn>
int with_nv(int nv, Fn&& fn) {
  switch (nv) {
    case 1: return fn(IntC<1>{});
    case 2: return fn(IntC<2>{});
    case 3: return fn(IntC<3>{});
    case 4: return fn(IntC<4>{});
    case 8: return fn(IntC<8>{});
    case 16: return fn(IntC<16>{});
    default: return B200_ERR_INVALID_ARGUMENT;
  }
}

// fn(element type, weight type) for a pair of dtype codes.
template <typename Fn>
int with_types(int dtype, int wdtype, Fn&& fn) {
  if (dtype == B200_DTYPE_F32) return wdtype == B200_DTYPE_F32 ? fn(float{}, float{}) : B200_ERR_INVALID_ARGUMENT;
  if (dtype == B200_DTYPE_F16) {
    if (wdtype == B200_DTYPE_F16) return fn(__half{}, __half{});
    if (wdtype == B200_DTYPE_F32) return fn(__half{}, float{});
  }
  if (dtype == B200_DTYPE_BF16) {
    if (wdtype == B200_DTYPE_BF16) return fn(__nv_bfloat16{}, __nv_bfloat16{});
    if (wdtype == B200_DTYPE_F32) return fn(__nv_bfloat16{}, float{});
  }
  return B200_ERR_INVALID_ARGUMENT;
}

bool dtype_ok(int d) { return d == B200_DTYPE_F16 || d == B200_DTYPE_BF16 || d == B200_DTYPE_F32; }
int dtype_size(int d) { return d == B200_DTYPE_F32 ? 4 : 2; }

// Elements that an access to rows of `cols` elements of `size` bytes at `p`
// (NULL: any) with pitch `ld` may take at once: 16 bytes' worth of the narrower
// of its own and the `other` operand's type, two, or one.
int row_vec(int cols, int size, int other, const void* p, int64_t ld) {
  const int most = 16 / std::min(size, other);
  for (int v = most; v > 1; v = v > 2 ? 2 : 1) {
    const int bytes = std::min(16, v * size);
    if (cols % v == 0 && reinterpret_cast<uintptr_t>(p) % bytes == 0 && ld * size % bytes == 0) return v;
  }
  return 1;
}

// fn(elements of a pack): as many as row_vec() allows.
template <typename T, typename Fn>
int with_vec(int elems, Fn&& fn) {
  if (elems == kVec16<T>) return fn(IntC<kVec16<T>>{});
  if constexpr (sizeof(T) == 2)
    if (elems == 2) return fn(IntC<2>{});
  return fn(IntC<1>{});
}

int cuda_code(cudaError_t e) { return e == cudaSuccess ? B200_OK : B200_ERR_CUDA; }

// Blocks of a kernel resident on the whole device.  Asked once per device and
// block size; `kern` fixes the function, so each instantiation has its own table.
template <auto kern>
int resident_blocks(int threads, size_t smem, int sm_count) {
  static std::atomic<int> table[kMaxDevices][kMaxRowThreads / 8 + 1];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return sm_count;
  std::atomic<int>& slot = table[dev][threads / 8];
  int per_sm = slot.load(std::memory_order_relaxed);
  if (per_sm == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, smem) != cudaSuccess || per_sm <= 0) {
      (void)cudaGetLastError();
      per_sm = 1;
    }
    slot.store(per_sm, std::memory_order_relaxed);
  }
  return per_sm * sm_count;
}

int check_norm_args(int64_t rows, int64_t cols, int dtype, int wdtype) {
  if (rows < 0 || cols < 0 || !dtype_ok(dtype) || !dtype_ok(wdtype)) return B200_ERR_INVALID_ARGUMENT;
  if (wdtype != dtype && wdtype != B200_DTYPE_F32) return B200_ERR_INVALID_ARGUMENT;
  if (cols > 0x3fffffff) return B200_ERR_TOO_LARGE;  // 2 * cols is indexed with 32 bits
  return B200_OK;
}

// Rows of the backward pass's partial sums (its blocks) at most: two blocks an
// SM keep the partials small beside x and dy.
constexpr int kBwdMaxParts = 2 * 160;

}  // namespace
}  // namespace b200

extern "C" int b200_layer_norm_fwd(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd,
                                   int64_t rows, int64_t cols, int64_t ldx, int64_t ldy, int dtype, int wdtype,
                                   float eps, void* stream_ptr) {
  using namespace b200;
  if (int rc = check_norm_args(rows, cols, dtype, wdtype)) return rc;
  if (rows == 0 || cols == 0) return B200_OK;
  if (!x || !y || ldx < cols || ldy < cols) return B200_ERR_INVALID_ARGUMENT;
  if (!aligned_to(dtype_size(dtype), x, y) || !aligned_to(dtype_size(wdtype), w, b) || !aligned_to(4, mean, rstd))
    return B200_ERR_MISALIGNED;
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  if (!dev.sm100) return B200_ERR_UNSUPPORTED_DEVICE;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  const int size = dtype_size(dtype), n = static_cast<int>(cols);
  const int w_size = dtype_size(wdtype);
  const int elems = std::min({row_vec(n, size, w_size, x, ldx), row_vec(n, size, w_size, y, ldy),
                              row_vec(n, w_size, size, w, 0), row_vec(n, w_size, size, b, 0)});
  return with_types(dtype, wdtype, [&](auto t, auto wt) {
    using T = decltype(t);
    using W = decltype(wt);
    return with_vec<T>(elems, [&](auto vc) {
      constexpr int kV = decltype(vc)::value;
      const RowPlan p = plan_fwd<kV>((n + kV - 1) / kV, rows, dev.sm_count);
      if (p.nv == 0) {
        const int grid = (int)std::min<int64_t>(rows, 0x7fffffff);
        return cuda_code(launch_gemm(layer_norm_fwd_long_kernel<T, W>, dim3(grid), dim3(kLongThreads), 0, stream,
                                     static_cast<const T*>(x), static_cast<const W*>(w), static_cast<const W*>(b),
                                     static_cast<T*>(y), mean, rstd, rows, n, ldx, ldy, eps));
      }
      return with_nv(p.nv, [&](auto nvc) {
        constexpr int kNv = decltype(nvc)::value;
        if constexpr (fwd_built<kV>(kNv)) {
          const bool exact = n == p.threads * kV * kNv && fwd_exact<kV>(kNv, p.threads);
          return with_tpr(exact, p.threads, [&](auto tc) {
            constexpr int kT = fwd_exact<kV>(kNv, decltype(tc)::value) ? decltype(tc)::value : 0;
            constexpr auto kern = layer_norm_fwd_kernel<T, W, kV, kNv, kT>;
            const int64_t blocks = (rows + p.rows - 1) / p.rows;
            const size_t smem = FwdRing<T, W, kV, kNv, kT>::kBytes * p.threads * p.rows;
            static std::atomic<uint8_t> attr_done[kMaxDevices];
            if (smem > 0)
              if (int e = ensure_smem_attr(kern, (int)smem, attr_done)) return e;
            const int fit = resident_blocks<kern>(p.threads * p.rows, smem, dev.sm_count);
            const int grid = (int)std::min<int64_t>(blocks, fit);
            return cuda_code(launch_gemm(kern, dim3(grid), dim3(p.threads, p.rows), smem, stream,
                                         static_cast<const T*>(x), static_cast<const W*>(w), static_cast<const W*>(b),
                                         static_cast<T*>(y), mean, rstd, rows, n, ldx, ldy, eps));
          });
        }
        return (int)B200_ERR_INVALID_ARGUMENT;
      });
    });
  });
}

extern "C" int64_t b200_layer_norm_bwd_workspace_size(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return -B200_ERR_INVALID_ARGUMENT;
  if (cols > 0x3fffffff) return -B200_ERR_TOO_LARGE;
  return std::min<int64_t>(rows, b200::kBwdMaxParts) * 2 * cols * 4;
}

extern "C" int b200_layer_norm_bwd(const void* dy, const void* x, const void* w, const float* mean, const float* rstd,
                                   void* dx, void* dw, void* db, int64_t rows, int64_t cols, int64_t lddy, int64_t ldx,
                                   int64_t lddx, int dtype, int wdtype, void* workspace, int64_t workspace_bytes,
                                   void* stream_ptr) {
  using namespace b200;
  if (int rc = check_norm_args(rows, cols, dtype, wdtype)) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (cols == 0) return B200_OK;
  if (!aligned_to(dtype_size(dtype), dy, x, dx) || !aligned_to(dtype_size(wdtype), w, dw, db) ||
      !aligned_to(4, mean, rstd))
    return B200_ERR_MISALIGNED;
  if (rows == 0) {
    const size_t bytes = (size_t)cols * dtype_size(wdtype);
    if (dw && cudaMemsetAsync(dw, 0, bytes, stream) != cudaSuccess) return B200_ERR_CUDA;
    if (db && cudaMemsetAsync(db, 0, bytes, stream) != cudaSuccess) return B200_ERR_CUDA;
    return B200_OK;
  }
  if (!dy || !x || !mean || !rstd || !dx || lddy < cols || ldx < cols || lddx < cols) return B200_ERR_INVALID_ARGUMENT;
  const bool sums = dw || db;
  if (sums && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0 ||
               workspace_bytes < b200_layer_norm_bwd_workspace_size(rows, cols)))
    return B200_ERR_WORKSPACE;
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  if (!dev.sm100) return B200_ERR_UNSUPPORTED_DEVICE;
  const int size = dtype_size(dtype), n = static_cast<int>(cols);
  const int wsize = dtype_size(wdtype);
  const int elems = std::min({row_vec(n, size, wsize, x, ldx), row_vec(n, size, wsize, dy, lddy),
                              row_vec(n, size, wsize, dx, lddx), row_vec(n, wsize, size, w, 0)});
  float* part = sums ? static_cast<float*>(workspace) : nullptr;
  return with_types(dtype, wdtype, [&](auto t, auto wt) {
    using T = decltype(t);
    using W = decltype(wt);
    const T* dyp = static_cast<const T*>(dy);
    const T* xp = static_cast<const T*>(x);
    const W* wp = static_cast<const W*>(w);
    T* dxp = static_cast<T*>(dx);
    int parts = 0;
    int rc = with_vec<T>(elems, [&](auto vc) {
      constexpr int kV = decltype(vc)::value;
      const RowPlan p = plan_bwd<kV>((n + kV - 1) / kV);
      if (p.nv == 0) {
        const int grid = (int)std::min<int64_t>(rows, 0x7fffffff);
        int e = cuda_code(launch_gemm(layer_norm_bwd_long_kernel<T, W>, dim3(grid), dim3(kLongThreads), 0, stream, dyp,
                                      xp, wp, mean, rstd, dxp, rows, n, lddy, ldx, lddx));
        if (e || !sums) return e;
        parts = (int)std::min<int64_t>(rows, 32);
        return cuda_code(launch_gemm(layer_norm_bwd_columns_kernel<T>, dim3((n + 127) / 128, parts), dim3(128), 0,
                                     stream, dyp, xp, mean, rstd, part, rows, n, lddy, ldx));
      }
      return with_nv(p.nv, [&](auto nvc) {
        constexpr int kNv = decltype(nvc)::value;
        if constexpr (bwd_built<kV>(kNv)) {
          const bool exact = n == p.threads * kV * kNv && bwd_exact<kV>(kNv, p.threads);
          return with_tpr(exact, p.threads, [&](auto tc) {
            constexpr int kT = bwd_exact<kV>(kNv, decltype(tc)::value) ? decltype(tc)::value : 0;
            constexpr auto kern = layer_norm_bwd_kernel<T, W, kV, kNv, kT>;
            constexpr size_t kPerThread = kV * sizeof(T) == 16 ? (kAhead<kNv> + 1) * 2 * kNv * 16 : 0;
            constexpr size_t kMost = std::max<size_t>(kPerThread * kBwdThreads, 48 * 1024);
            static std::atomic<uint8_t> attr_done[kMaxDevices];
            if (int e = ensure_smem_attr(kern, (int)kMost, attr_done)) return e;
            const size_t smem = std::max(kPerThread * p.threads * p.rows, p.rows > 1 ? (size_t)2 * n * 4 : 0);
            const int fit = resident_blocks<kern>(p.threads * p.rows, smem, dev.sm_count);
            const int64_t blocks = (rows + p.rows - 1) / p.rows;
            parts = (int)std::min<int64_t>({blocks, (int64_t)fit, (int64_t)kBwdMaxParts});
            return cuda_code(launch_gemm(kern, dim3(parts), dim3(p.threads, p.rows), smem, stream, dyp, xp, wp, mean,
                                         rstd, dxp, part, rows, n, lddy, ldx, lddx));
          });
        }
        return (int)B200_ERR_INVALID_ARGUMENT;
      });
    });
    if (rc || !sums) return rc;
    return cuda_code(launch_gemm(layer_norm_bwd_reduce_kernel<W>, dim3((n + 31) / 32, 2), dim3(32, 16), 0, stream,
                                 static_cast<const float*>(part), parts, n, static_cast<W*>(dw), static_cast<W*>(db)));
  });
}
