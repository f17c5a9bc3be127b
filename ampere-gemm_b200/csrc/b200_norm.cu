// Layer norm over the last dimension, forward and backward.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r
//   y  = h w + b
//   with q = dy w:  dx = r (q - mean(q) - h mean(q h))
//   dw = sum over rows of dy h,  db = sum over rows of dy
//
// Bound by memory: forward reads x and writes y once, backward reads x and dy
// and writes dx once.  A row stays in registers, in its own type, between the
// passes over it; all sums are in fp32 and y, dx, dw and db are rounded once.
// Every sum has a fixed order, so results do not change from run to run.
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

// Sum over the threads of one row.  A row is one warp (each warp of the block
// has its own), or the whole block; `red` is then 32 floats that no thread
// still reads from the sum before the last.
__device__ __forceinline__ float row_sum(float v, bool one_warp, float* red) {
  v = warp_sum(v);
  if (one_warp) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return warp_sum(lane < warps ? red[lane] : 0.0f);
}

// Forward.  blockDim = (threads of a row, rows of a block); a thread holds NV
// packs of VEC elements, pack j at (j * blockDim.x + threadIdx.x) * VEC.
template <typename T, typename W, int VEC, int NV>
__global__ void __launch_bounds__(kMaxRowThreads)
    layer_norm_fwd_kernel(const T* __restrict__ x, const W* __restrict__ w, const W* __restrict__ b,
                                      T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                      int64_t rows, int cols, int64_t ldx, int64_t ldy, float eps) {
  __shared__ float red[2][32];
  pdl_wait();
  const bool one_warp = blockDim.x == 32;
  const float inv_n = 1.0f / static_cast<float>(cols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.y;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; row < rows; row += step) {
    const T* xr = x + row * ldx;
    Pack<T, VEC> v[NV];
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * VEC;
      if (c < cols) v[j] = load_pack<T, VEC>(xr + c);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * VEC;
      if (c < cols) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) s += to_f32(v[j].v[e]);
      }
    }
    const float mu = row_sum(s, one_warp, red[0]) * inv_n;
    // The centred squares are summed in a second pass over the registers:
    // sum(x^2) - n mu^2 would lose the variance of a row with a large mean.
    float q = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * VEC;
      if (c < cols) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float d = to_f32(v[j].v[e]) - mu;
          q = fmaf(d, d, q);
        }
      }
    }
    const float rstd = 1.0f / sqrtf(row_sum(q, one_warp, red[1]) * inv_n + eps);
    T* yr = y + row * ldy;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * VEC;
      if (c < cols) {
        Pack<T, VEC> o;
        Pack<W, VEC> wv, bv;
        if (w) wv = load_pack<W, VEC>(w + c);
        if (b) bv = load_pack<W, VEC>(b + c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float h = (to_f32(v[j].v[e]) - mu) * rstd;
          o.v[e] = from_f32<T>(fmaf(h, w ? to_f32(wv.v[e]) : 1.0f, b ? to_f32(bv.v[e]) : 0.0f));
        }
        store_pack<T, VEC>(yr + c, o);
      }
    }
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[row] = mu;
      if (rstd_out) rstd_out[row] = rstd;
    }
  }
}

// Forward for rows longer than the registers of a block hold: one block a
// row, which is read three times (the second and third from L2).
template <typename T, typename W>
__global__ void __launch_bounds__(kLongThreads) layer_norm_fwd_long_kernel(const T* __restrict__ x, const W* __restrict__ w, const W* __restrict__ b,
                                           T* __restrict__ y, float* __restrict__ mean_out,
                                           float* __restrict__ rstd_out, int64_t rows, int cols, int64_t ldx,
                                           int64_t ldy, float eps) {
  __shared__ float red[2][32];
  pdl_wait();
  const float inv_n = 1.0f / static_cast<float>(cols);
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * ldx;
    float s = 0.0f;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) s += to_f32(xr[c]);
    const float mu = row_sum(s, false, red[0]) * inv_n;
    float q = 0.0f;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
      const float d = to_f32(xr[c]) - mu;
      q = fmaf(d, d, q);
    }
    const float rstd = 1.0f / sqrtf(row_sum(q, false, red[1]) * inv_n + eps);
    for (int c = threadIdx.x; c < cols; c += blockDim.x)
      y[row * ldy + c] = from_f32<T>(
          fmaf((to_f32(xr[c]) - mu) * rstd, w ? to_f32(w[c]) : 1.0f, b ? to_f32(b[c]) : 0.0f));
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[row] = mu;
      if (rstd_out) rstd_out[row] = rstd;
    }
  }
}

// Backward.  Same layout as the forward kernel.  A thread keeps the same
// columns for all its rows, so it sums their dw and db in registers; a block
// writes its sums once, as row blockIdx.x of `part` (gridDim.x x 2 x cols:
// dw, then db), and layer_norm_bwd_reduce_kernel adds those rows up.
template <typename T, typename W, int VEC, int NV>
__global__ void __launch_bounds__(kMaxRowThreads)
    layer_norm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const W* __restrict__ w,
                                      const float* __restrict__ mean, const float* __restrict__ rstd_in,
                                      T* __restrict__ dx, float* __restrict__ part, int64_t rows, int cols,
                                      int64_t lddy, int64_t ldx, int64_t lddx) {
  __shared__ float red[2][2][32];
  extern __shared__ float col_sum[];  // [2][cols], blocks of more than one row
  pdl_wait();
  const bool one_warp = blockDim.x == 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const float inv_n = 1.0f / static_cast<float>(cols);
  float dw[NV][VEC], db[NV][VEC];
  Pack<W, VEC> wv[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * blockDim.x + threadIdx.x) * VEC;
    if (w && c < cols) wv[j] = load_pack<W, VEC>(w + c);
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[j][e] = db[j][e] = 0.0f;
  }
  int parity = 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.y;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y; row < rows; row += step) {
    const T* xr = x + row * ldx;
    const T* gr = dy + row * lddy;
    Pack<T, VEC> xv[NV], gv[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * VEC;
      if (c < cols) {
        xv[j] = load_pack<T, VEC>(xr + c);
        gv[j] = load_pack<T, VEC>(gr + c);
      }
    }
    const float mu = mean[row], rstd = rstd_in[row];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * VEC;
      if (c < cols) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float g = to_f32(gv[j].v[e]);
          const float h = (to_f32(xv[j].v[e]) - mu) * rstd;
          const float q = g * (w ? to_f32(wv[j].v[e]) : 1.0f);
          s1 += q;
          s2 = fmaf(q, h, s2);
          dw[j][e] = fmaf(g, h, dw[j][e]);
          db[j][e] += g;
        }
      }
    }
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if (!one_warp) {
      // Two buffers in turn: one barrier a row is enough.
      if (lane == 0) {
        red[parity][0][warp] = s1;
        red[parity][1][warp] = s2;
      }
      __syncthreads();
      s1 = warp_sum(lane < warps ? red[parity][0][lane] : 0.0f);
      s2 = warp_sum(lane < warps ? red[parity][1][lane] : 0.0f);
      parity ^= 1;
    }
    s1 *= inv_n;
    s2 *= inv_n;
    T* dr = dx + row * lddx;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * VEC;
      if (c < cols) {
        Pack<T, VEC> o;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float h = (to_f32(xv[j].v[e]) - mu) * rstd;
          const float q = to_f32(gv[j].v[e]) * (w ? to_f32(wv[j].v[e]) : 1.0f);
          o.v[e] = from_f32<T>(rstd * (q - s1 - h * s2));
        }
        store_pack<T, VEC>(dr + c, o);
      }
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
          out[c + e] = dw[j][e];
          out[cols + c + e] = db[j][e];
        }
      }
    }
    return;
  }
  // The block's rows are added up in shared memory, in order.
  for (int yy = 0; yy < static_cast<int>(blockDim.y); ++yy) {
    if (threadIdx.y == yy) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * blockDim.x + threadIdx.x) * VEC;
        if (c < cols) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            col_sum[c + e] = dw[j][e] + (yy ? col_sum[c + e] : 0.0f);
            col_sum[cols + c + e] = db[j][e] + (yy ? col_sum[cols + c + e] : 0.0f);
          }
        }
      }
    }
    __syncthreads();
  }
  for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < 2 * cols; c += blockDim.x * blockDim.y) out[c] = col_sum[c];
}

// dx for rows longer than a block's registers hold: one block a row.
template <typename T, typename W>
__global__ void __launch_bounds__(kLongThreads) layer_norm_bwd_long_kernel(const T* __restrict__ dy, const T* __restrict__ x, const W* __restrict__ w,
                                           const float* __restrict__ mean, const float* __restrict__ rstd_in,
                                           T* __restrict__ dx, int64_t rows, int cols, int64_t lddy, int64_t ldx,
                                           int64_t lddx) {
  __shared__ float red[2][32];
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
    s1 = row_sum(s1, false, red[0]) * inv_n;
    s2 = row_sum(s2, false, red[1]) * inv_n;
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

struct RowPlan {
  int nv;       // packs a thread holds (0: the row does not fit a block's registers)
  int threads;  // threads of a row
  int rows;     // rows of a block
};

int round32(int v) { return (v + 31) / 32 * 32; }

// Threads and packs of a row of `packs` packs, at most `max_nv` packs a thread.
// Rows that one warp holds go four to a block; longer ones take a block each
// with as few packs a thread as `threads_wanted` threads allow.
RowPlan plan_rows(int packs, int max_nv, int threads_wanted) {
  for (int nv = 1; nv <= max_nv; nv *= 2) {
    const int t = round32((packs + nv - 1) / nv);
    if (t <= threads_wanted || (nv == max_nv && t <= kMaxRowThreads)) return RowPlan{nv, t, t == 32 ? 4 : 1};
  }
  return RowPlan{0, 0, 1};
}

constexpr int kFwdMaxNv = 8;
// Columns a thread sums dw and db of, in packs: two registers each, beside the
// packs of x, dy and w.
template <int VEC>
constexpr int kBwdMaxNv = VEC == 1 ? 16 : 4;

template <int V>
using IntC = std::integral_constant<int, V>;

template <typename Fn>
int with_nv(int nv, Fn&& fn) {
  switch (nv) {
    case 1: return fn(IntC<1>{});
    case 2: return fn(IntC<2>{});
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

// True when rows at `p` with pitch `ld` elements of `size` bytes all start on 16 bytes.
bool rows_aligned(const void* p, int64_t ld, int size) { return aligned16(p) && (ld * size) % 16 == 0; }

int cuda_code(cudaError_t e) { return e == cudaSuccess ? B200_OK : B200_ERR_CUDA; }

// Blocks of `kern` resident on the whole device.
template <typename Kern>
int resident_blocks(Kern kern, int threads, size_t smem, int sm_count) {
  int per_sm = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, smem) != cudaSuccess || per_sm <= 0) {
    (void)cudaGetLastError();
    per_sm = 1;
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
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  if (!dev.sm100) return B200_ERR_UNSUPPORTED_DEVICE;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  const int size = dtype_size(dtype), n = static_cast<int>(cols);
  const int vec16 = 16 / size;
  const bool vec = n % vec16 == 0 && rows_aligned(x, ldx, size) && rows_aligned(y, ldy, size) &&
                   (!w || aligned16(w)) && (!b || aligned16(b));
  return with_types(dtype, wdtype, [&](auto t, auto wt) {
    using T = decltype(t);
    using W = decltype(wt);
    const RowPlan p = plan_rows(vec ? n / vec16 : n, kFwdMaxNv, rows >= 4 * dev.sm_count ? 128 : kMaxRowThreads);
    auto go = [&](auto vc, auto nvc) {
      auto kern = layer_norm_fwd_kernel<T, W, decltype(vc)::value, decltype(nvc)::value>;
      const int64_t blocks = (rows + p.rows - 1) / p.rows;
      const int grid = (int)std::min<int64_t>(blocks, 0x7fffffff);
      return cuda_code(launch_gemm(kern, dim3(grid), dim3(p.threads, p.rows), 0, stream, static_cast<const T*>(x),
                                   static_cast<const W*>(w), static_cast<const W*>(b), static_cast<T*>(y), mean, rstd,
                                   rows, n, ldx, ldy, eps));
    };
    if (p.nv == 0) {
      const int grid = (int)std::min<int64_t>(rows, 0x7fffffff);
      return cuda_code(launch_gemm(layer_norm_fwd_long_kernel<T, W>, dim3(grid), dim3(kLongThreads), 0, stream,
                                   static_cast<const T*>(x), static_cast<const W*>(w), static_cast<const W*>(b),
                                   static_cast<T*>(y), mean, rstd, rows, n, ldx, ldy, eps));
    }
    return with_nv(p.nv, [&](auto nvc) {
      if constexpr (decltype(nvc)::value <= kFwdMaxNv)
        return vec ? go(IntC<kVec16<T>>{}, nvc) : go(IntC<1>{}, nvc);
      else
        return B200_ERR_INVALID_ARGUMENT;
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
  const int vec16 = 16 / size;
  const bool vec = n % vec16 == 0 && rows_aligned(x, ldx, size) && rows_aligned(dy, lddy, size) &&
                   rows_aligned(dx, lddx, size) && (!w || aligned16(w));
  float* part = sums ? static_cast<float*>(workspace) : nullptr;
  return with_types(dtype, wdtype, [&](auto t, auto wt) {
    using T = decltype(t);
    using W = decltype(wt);
    const T* dyp = static_cast<const T*>(dy);
    const T* xp = static_cast<const T*>(x);
    const W* wp = static_cast<const W*>(w);
    T* dxp = static_cast<T*>(dx);
    int parts = 0;
    int rc;
    const RowPlan p = vec ? plan_rows(n / vec16, kBwdMaxNv<kVec16<T>>, kMaxRowThreads)
                          : plan_rows(n, kBwdMaxNv<1>, kMaxRowThreads);
    if (p.nv == 0) {
      const int grid = (int)std::min<int64_t>(rows, 0x7fffffff);
      rc = cuda_code(launch_gemm(layer_norm_bwd_long_kernel<T, W>, dim3(grid), dim3(kLongThreads), 0, stream, dyp, xp, wp,
                                 mean, rstd, dxp, rows, n, lddy, ldx, lddx));
      if (rc || !sums) return rc;
      parts = (int)std::min<int64_t>(rows, 32);
      rc = cuda_code(launch_gemm(layer_norm_bwd_columns_kernel<T>, dim3((n + 127) / 128, parts), dim3(128), 0, stream,
                                 dyp, xp, mean, rstd, part, rows, n, lddy, ldx));
    } else {
      auto go = [&](auto vc, auto nvc) {
        auto kern = layer_norm_bwd_kernel<T, W, decltype(vc)::value, decltype(nvc)::value>;
        const size_t smem = p.rows > 1 ? (size_t)2 * n * 4 : 0;
        const int fit = resident_blocks(kern, p.threads * p.rows, smem, dev.sm_count);
        const int64_t blocks = (rows + p.rows - 1) / p.rows;
        parts = (int)std::min<int64_t>({blocks, (int64_t)fit, (int64_t)kBwdMaxParts});
        return cuda_code(launch_gemm(kern, dim3(parts), dim3(p.threads, p.rows), smem, stream, dyp, xp, wp, mean, rstd,
                                     dxp, part, rows, n, lddy, ldx, lddx));
      };
      rc = with_nv(p.nv, [&](auto nvc) {
        constexpr int kNv = decltype(nvc)::value;
        if (vec) {
          if constexpr (kNv <= kBwdMaxNv<kVec16<T>>) return go(IntC<kVec16<T>>{}, nvc);
          return (int)B200_ERR_INVALID_ARGUMENT;
        }
        return go(IntC<1>{}, nvc);
      });
    }
    if (rc || !sums) return rc;
    return cuda_code(launch_gemm(layer_norm_bwd_reduce_kernel<W>, dim3((n + 31) / 32, 2), dim3(32, 16), 0, stream,
                                 static_cast<const float*>(part), parts, n, static_cast<W*>(dw), static_cast<W*>(db)));
  });
}
