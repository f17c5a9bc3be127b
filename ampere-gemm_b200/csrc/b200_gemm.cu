// B200 (sm_100a) FP16 GEMM: C[M,N] = A[M,K] * B, fp16 in, fp32 accumulate in
// tensor memory, fp16 out (round-to-nearest-even), behind a C ABI.
//
// Replaces the reference's L4/Ampere kernels (tensorcore_gemm/gemm.cu:1073
// `..._reg_pingpong_256`, :1373 `_colb`, :1811 `_MMA`, :1972 `_colb_MMA`) and
// their launcher `root_gemm_cuda` (tensorcore_gemm/gemm.py:31-154).  The math
// is the same as the reference epilogue `__float2half(alpha * acc)` with
// alpha = 1, beta = 0 (gemm.cu:1360-1361): an fp32 sum of fp16 products,
// rounded once to fp16.
//
// Kernel structure (one persistent CTA per SM, 192 threads, 6 warps):
//   warp 0      TMA producer: loads A (K-major) and B (K-major "colb" or
//               MN-major row-major) k-blocks into a STAGES-deep shared ring.
//   warp 1      allocates TMEM, and one lane issues tcgen05.mma (128 x BN x 16
//               per instruction) into one of two TMEM accumulators.
//   warps 2..5  epilogue: tcgen05.ld -> fp16 -> 128B-swizzled shared tile ->
//               TMA store; releases the accumulator as soon as it is read, so
//               the next tile's mainloop overlaps this tile's stores.
// Out-of-range rows/columns (any M, N, K) are handled by TMA zero fill on
// loads and clipping on stores.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cstring>
#include <cstdio>
#include <cstdlib>
#include <mutex>
#include <type_traits>
#include <utility>

#include "gemm_internal.h"
#include "gemm_launch.cuh"
#include "../../include/b200_gemm.h"

namespace b200 {

// Self-test of the bounded-wait path: one thread waits on an mbarrier that
// nothing ever arrives at, gives up after `limit_ns`, records
// kDevTimeoutSelftest in the device error word and returns.
__global__ void bounded_wait_selftest_kernel(uint64_t limit_ns) {
  __shared__ uint64_t bar;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    fence_mbarrier_init();
    mbar_wait(&bar, 0, kDevTimeoutSelftest, limit_ns);
  }
}

}  // namespace b200

// ===========================================================================
// Host side
// ===========================================================================
// ===========================================================================
// C ABI
// ===========================================================================
namespace b200 {
namespace {

// Arguments common to every entry point.  Returns B200_OK, or an error code;
// sets *nothing_to_do when the output is empty.
int validate_args(const void* C, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb, int64_t ldc,
                  int b_layout, const void* A, const void* B, bool* nothing_to_do, int a_layout = B200_A_ROW_MAJOR) {
  *nothing_to_do = false;
  if (M < 0 || N < 0 || K < 0) return B200_ERR_INVALID_ARGUMENT;
  if (b_layout != B200_B_ROW_MAJOR && b_layout != B200_B_COL_MAJOR) return B200_ERR_INVALID_ARGUMENT;
  if (a_layout != B200_A_ROW_MAJOR && a_layout != B200_A_COL_MAJOR) return B200_ERR_INVALID_ARGUMENT;
  const int64_t kMax = 0x7fffffff;
  if (M > kMax || N > kMax || K > kMax) return B200_ERR_TOO_LARGE;
  if (M == 0 || N == 0) {
    *nothing_to_do = true;
    return B200_OK;
  }
  if (!C || ldc < N) return B200_ERR_INVALID_ARGUMENT;
  if (K > 0) {
    const bool row_b = (b_layout == B200_B_ROW_MAJOR);
    const bool col_a = (a_layout == B200_A_COL_MAJOR);
    if (!A || !B || lda < (col_a ? M : K) || ldb < (row_b ? N : K)) return B200_ERR_INVALID_ARGUMENT;
  }
  return B200_OK;
}

// Copies a rows x cols fp16 matrix between row pitches (elements).
__global__ void pitched_copy_f16_kernel(const uint16_t* __restrict__ src, int64_t src_ld, uint16_t* __restrict__ dst,
                                        int64_t dst_ld, int64_t rows, int64_t cols) {
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y)
    for (int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; c < cols; c += (int64_t)gridDim.x * blockDim.x)
      dst[r * dst_ld + c] = src[r * src_ld + c];
}

int pitched_copy(const void* src, int64_t src_ld, void* dst, int64_t dst_ld, int64_t rows, int64_t cols,
                 cudaStream_t stream) {
  if (rows == 0 || cols == 0) return B200_OK;
  const unsigned gx = (unsigned)std::min<int64_t>((cols + 255) / 256, 64);
  const unsigned gy = (unsigned)std::min<int64_t>(rows, 65535);
  pitched_copy_f16_kernel<<<dim3(gx, gy), 256, 0, stream>>>(static_cast<const uint16_t*>(src), src_ld,
                                                             static_cast<uint16_t*>(dst), dst_ld, rows, cols);
  return cudaGetLastError() == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}

// Workspace plan for operands whose base or row pitch TMA cannot describe:
// each such operand gets a copy with a 16-byte row pitch (pitch rounded up
// to 8 elements) at a 256-byte aligned offset.  Unaligned C is computed into
// its copy and copied back.
struct RepackPlan {
  bool a = false, b = false, c = false;
  int64_t lda2 = 0, ldb2 = 0, ldc2 = 0;
  int64_t off_a = 0, off_b = 0, off_c = 0, bytes = 0;
};

RepackPlan plan_repack(const void* A, const void* B, const void* C, int64_t M, int64_t N, int64_t K, int64_t lda,
                       int64_t ldb, int64_t ldc, int b_layout, int a_layout = B200_A_ROW_MAJOR) {
  RepackPlan p;
  const bool row_b = (b_layout == B200_B_ROW_MAJOR);
  const bool col_a = (a_layout == B200_A_COL_MAJOR);
  if (K > 0) {
    p.a = !pitch_ok(A, lda);
    p.b = !pitch_ok(B, ldb);
  }
  p.c = !pitch_ok(C, ldc);
  int64_t off = 0;
  if (p.a) {
    const int64_t rows = col_a ? K : M, cols = col_a ? M : K;
    p.lda2 = round_up(cols, 8);
    p.off_a = off;
    off = round_up(off + rows * p.lda2 * 2, 256);
  }
  if (p.b) {
    const int64_t rows = row_b ? K : N, cols = row_b ? N : K;
    p.ldb2 = round_up(cols, 8);
    p.off_b = off;
    off = round_up(off + rows * p.ldb2 * 2, 256);
  }
  if (p.c) {
    p.ldc2 = round_up(N, 8);
    p.off_c = off;
    off = round_up(off + M * p.ldc2 * 2, 256);
  }
  p.bytes = off;
  return p;
}

// Repack (as planned), multiply, copy C back; `ws` is device memory of at
// least plan.bytes, 256-byte aligned.
int gemm_repacked(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb,
                  int64_t ldc, int a_layout, int b_layout, const EpiParams& scale, const RepackPlan& p, uint8_t* ws,
                  const DeviceInfo& dev, cudaStream_t stream) {
  const bool row_b = (b_layout == B200_B_ROW_MAJOR);
  const bool col_a = (a_layout == B200_A_COL_MAJOR);
  const void* a = A;
  const void* b = B;
  void* c = C;
  int64_t la = lda, lb = ldb, lc = ldc;
  int rc = B200_OK;
  if (p.a) {
    a = ws + p.off_a;
    la = p.lda2;
    if ((rc = pitched_copy(A, lda, ws + p.off_a, la, col_a ? K : M, col_a ? M : K, stream))) return rc;
  }
  if (p.b) {
    b = ws + p.off_b;
    lb = p.ldb2;
    if ((rc = pitched_copy(B, ldb, ws + p.off_b, lb, row_b ? K : N, row_b ? N : K, stream))) return rc;
  }
  if (p.c) {
    c = ws + p.off_c;
    lc = p.ldc2;
    if (scale.beta != 0.0f && (rc = pitched_copy(C, ldc, c, lc, M, N, stream))) return rc;  // old C is an input
  }
  if ((rc = gemm_aligned<false>(a, b, c, M, N, K, la, lb, lc, a_layout, b_layout, scale, dev, stream))) return rc;
  if (p.c) rc = pitched_copy(c, lc, C, ldc, M, N, stream);
  return rc;
}

}  // namespace
}  // namespace b200

int b200::gemm_f16_run(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K, int64_t lda,
                       int64_t ldb, int64_t ldc, int a_layout, int b_layout, void* split_ws, void* stream) {
  return gemm_run<false>(A, B, C, M, N, K, lda, ldb, ldc, a_layout, b_layout, split_ws, stream);
}

extern "C" int b200_gemm_f16(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K, int64_t lda,
                             int64_t ldb, int64_t ldc, int b_layout, void* stream_ptr) {
  using namespace b200;
  bool done = false;
  if (int rc = validate_args(C, M, N, K, lda, ldb, ldc, b_layout, A, B, &done)) return rc;
  if (done) return B200_OK;
  if (!pitch_ok(C, ldc)) return B200_ERR_MISALIGNED;
  if (K > 0 && (!pitch_ok(A, lda) || !pitch_ok(B, ldb))) return B200_ERR_MISALIGNED;
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  if (!dev.sm100) return B200_ERR_UNSUPPORTED_DEVICE;
  return gemm_aligned<false>(A, B, C, M, N, K, lda, ldb, ldc, B200_A_ROW_MAJOR, b_layout, EpiParams{}, dev,
                      static_cast<cudaStream_t>(stream_ptr));
}

extern "C" int64_t b200_gemm_workspace_size_ex(const void* A, const void* B, const void* C, int64_t M, int64_t N,
                                               int64_t K, int64_t lda, int64_t ldb, int64_t ldc, int a_layout,
                                               int b_layout) {
  using namespace b200;
  bool done = false;
  if (int rc = validate_args(C, M, N, K, lda, ldb, ldc, b_layout, A, B, &done, a_layout)) return -rc;
  if (done) return 0;
  return plan_repack(A, B, C, M, N, K, lda, ldb, ldc, b_layout, a_layout).bytes;
}

extern "C" int64_t b200_gemm_workspace_size(const void* A, const void* B, const void* C, int64_t M, int64_t N,
                                            int64_t K, int64_t lda, int64_t ldb, int64_t ldc, int b_layout) {
  return b200_gemm_workspace_size_ex(A, B, C, M, N, K, lda, ldb, ldc, B200_A_ROW_MAJOR, b_layout);
}

extern "C" int b200_gemm_f16_ex(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K, int64_t lda,
                                int64_t ldb, int64_t ldc, int a_layout, int b_layout, float alpha, float beta,
                                void* workspace, int64_t workspace_bytes, void* stream_ptr) {
  using namespace b200;
  bool done = false;
  if (int rc = validate_args(C, M, N, K, lda, ldb, ldc, b_layout, A, B, &done, a_layout)) return rc;
  if (done) return B200_OK;
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  if (!dev.sm100) return B200_ERR_UNSUPPORTED_DEVICE;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  const EpiParams scale{alpha, beta};
  const RepackPlan p = plan_repack(A, B, C, M, N, K, lda, ldb, ldc, b_layout, a_layout);
  if (p.bytes == 0) return gemm_aligned<false>(A, B, C, M, N, K, lda, ldb, ldc, a_layout, b_layout, scale, dev, stream);
  if (!workspace || workspace_bytes < p.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
    return B200_ERR_WORKSPACE;
  return gemm_repacked(A, B, C, M, N, K, lda, ldb, ldc, a_layout, b_layout, scale, p,
                       static_cast<uint8_t*>(workspace), dev, stream);
}

extern "C" int b200_gemm_f16_ws(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K, int64_t lda,
                                int64_t ldb, int64_t ldc, int b_layout, void* workspace, int64_t workspace_bytes,
                                void* stream_ptr) {
  return b200_gemm_f16_ex(A, B, C, M, N, K, lda, ldb, ldc, B200_A_ROW_MAJOR, b_layout, 1.0f, 0.0f, workspace,
                          workspace_bytes, stream_ptr);
}

extern "C" int b200_gemm_set_variant(int variant) {
  if (variant < B200_VARIANT_AUTO || variant > B200_VARIANT_PAIR_WIDE_192) return B200_ERR_INVALID_ARGUMENT;
  b200::g_variant = variant;
  return B200_OK;
}

extern "C" int b200_gemm_plan(int64_t M, int64_t N, int64_t K, int sm_count, int* variant, int* k_ranges) {
  using namespace b200;
  if (M <= 0 || N <= 0 || K <= 0 || sm_count < 2 || !variant || !k_ranges) return B200_ERR_INVALID_ARGUMENT;
  if (M > 0x7fffffff || N > 0x7fffffff || K > 0x7fffffff) return B200_ERR_TOO_LARGE;
  const int m = (int)M, n = (int)N, k = (int)K;
  int v = g_variant != B200_VARIANT_AUTO ? g_variant : auto_variant(m, n, k, sm_count);
  if (v == B200_VARIANT_SKINNY && (k > 256 || (n + 255) / 256 > sm_count)) v = B200_VARIANT_CTA1;
  int ranges = 1;
  if (v == B200_VARIANT_PAIR) {
    const long long tiles = (long long)((m + 255) / 256) * ((n + 255) / 256);
    ranges = split_ranges_for(tiles, (int)std::min<long long>(tiles, sm_count / 2), (k + 127) / 128);
  }
  *variant = v;
  *k_ranges = ranges;
  return B200_OK;
}

extern "C" const char* b200_gemm_strerror(int code) {
  switch (code) {
    case B200_OK: return "success";
    case B200_ERR_INVALID_ARGUMENT: return "invalid argument (null pointer, negative size, bad layout or leading dimension too small)";
    case B200_ERR_MISALIGNED: return "misaligned operand: base pointers must be 16-byte aligned and leading dimensions multiples of 8 elements";
    case B200_ERR_TOO_LARGE: return "dimension exceeds 2^31 - 1";
    case B200_ERR_CUDA: return "CUDA runtime error or kernel launch failure";
    case B200_ERR_TENSOR_MAP: return "cuTensorMapEncodeTiled unavailable or rejected the tensor map";
    case B200_ERR_DEVICE: return "device error word set: a bounded wait inside the kernel timed out";
    case B200_ERR_UNSUPPORTED_DEVICE: return "current device is not an sm_100 (B200-class) GPU";
    case B200_ERR_WORKSPACE: return "workspace missing, too small, or not 256-byte aligned (see b200_gemm_workspace_size)";
    case B200_ERR_SCRATCH_LIMIT: return "operands need more re-pitch scratch than the 32 MiB built into b200_gemm_f16_noalloc";
    default: return "unknown error code";
  }
}

extern "C" int b200_gemm_last_device_error(void) {
  if (cudaDeviceSynchronize() != cudaSuccess) return -1;
  int first = 0;
  for (int (*take)() : {&b200::take_error_word, &b200::take_error_word_gemm_bf16, &b200::take_error_word_ffn}) {
    const int v = take();
    if (v < 0) return -1;
    if (first == 0) first = v;
  }
  return first;
}

extern "C" int b200_gemm_sm_count(void) {
  b200::DeviceInfo d;
  if (b200::current_device_info(d)) return 0;
  return d.sm_count;
}

extern "C" int b200_gemm_version(void) { return 102; }

#ifdef B200_GEMM_PROFILE
// Copies and clears the per-CTA split-tail step timestamps (profiling builds only).
extern "C" __attribute__((visibility("default"))) int b200_gemm_debug_read_split_profile(unsigned long long* host,
                                                                                       int rows) {
  if (rows > 1024) rows = 1024;
  if (cudaMemcpyFromSymbol(host, b200::g_split_prof, sizeof(unsigned long long) * 8 * rows) != cudaSuccess) return -1;
  static unsigned long long zero[1024][8];
  return cudaMemcpyToSymbol(b200::g_split_prof, zero, sizeof(zero)) == cudaSuccess ? 0 : -1;
}

// Copies and clears the per-CTA wait counters (profiling builds only).
extern "C" __attribute__((visibility("default"))) int b200_gemm_debug_read_profile(unsigned long long* host, int rows) {
  if (rows > 1024) rows = 1024;
  if (cudaDeviceSynchronize() != cudaSuccess) return -1;
  if (cudaMemcpyFromSymbol(host, b200::g_prof, sizeof(unsigned long long) * 8 * rows) != cudaSuccess) return -1;
  static unsigned long long zeros[1024][8];
  return cudaMemcpyToSymbol(b200::g_prof, zeros, sizeof(zeros)) == cudaSuccess ? 0 : -1;
}
#endif

extern "C" int b200_gemm_selftest_bounded_wait(int64_t limit_ns) {
  if (limit_ns <= 0 || limit_ns > 1000000000LL) return -B200_ERR_INVALID_ARGUMENT;
  const int before = b200_gemm_last_device_error();  // clears any earlier word
  if (before < 0) return -B200_ERR_CUDA;
  b200::bounded_wait_selftest_kernel<<<1, 32>>>(static_cast<uint64_t>(limit_ns));
  if (cudaGetLastError() != cudaSuccess) return -B200_ERR_CUDA;
  const int word = b200_gemm_last_device_error();
  return word < 0 ? -B200_ERR_CUDA : word;
}

extern "C" int b200_gemm_selftest_split_fixup(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K,
                                              int64_t limit_ns, void* stream_ptr) {
  using namespace b200;
  if (limit_ns <= 0 || limit_ns > 1000000000LL) return -B200_ERR_INVALID_ARGUMENT;
  bool done = false;
  if (int rc = validate_args(C, M, N, K, K, N, N, B200_B_ROW_MAJOR, A, B, &done)) return -rc;
  if (done || K == 0) return -B200_ERR_INVALID_ARGUMENT;
  if (!pitch_ok(A, K) || !pitch_ok(B, N) || !pitch_ok(C, N)) return -B200_ERR_MISALIGNED;
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return -rc;
  if (!dev.sm100) return -B200_ERR_UNSUPPORTED_DEVICE;
  const long long tiles = ((M + 255) / 256) * ((N + 255) / 256);
  if (split_ranges_for(tiles, (int)std::min<long long>(tiles, dev.sm_count / 2), (int)((K + 127) / 128)) < 2)
    return -B200_ERR_INVALID_ARGUMENT;  // this shape's pair launch has no split last wave
  const int before = b200_gemm_last_device_error();  // clears any earlier word
  if (before < 0) return -B200_ERR_CUDA;
  CallOptions opts;
  opts.withhold_fixup_ns = static_cast<uint64_t>(limit_ns);
  opts.force_variant = B200_VARIANT_PAIR;
  int rc;
  {
    const ScopedCallOptions scoped(opts);
    rc = gemm_aligned<false>(A, B, C, M, N, K, K, N, N, B200_A_ROW_MAJOR, B200_B_ROW_MAJOR, EpiParams{}, dev,
                      static_cast<cudaStream_t>(stream_ptr));
  }
  if (rc) return -rc;
  const int word = b200_gemm_last_device_error();  // synchronises, clears the word, resets the tail counters
  return word < 0 ? -B200_ERR_CUDA : word;
}

// ===========================================================================
// Allocation-free entry point (b200_gemm_f16_noalloc)
//
// Same product as b200_gemm_f16_ws, for callers that may not allocate device
// memory at all: the re-pitch copies live in one fixed scratch array compiled
// into this library.  Every GPU that loads the library holds the array
// (kNoAllocScratchBytes) until the process exits.
// ===========================================================================
namespace b200 {

constexpr int64_t kNoAllocScratchBytes = 32ll << 20;  // 32 MiB

static __device__ __align__(256) uint8_t g_noalloc_scratch[kNoAllocScratchBytes];

namespace {

std::mutex g_noalloc_mu;
uint8_t* g_noalloc_ptr[kMaxDevices] = {};

// The array's name is only a host-side handle; the device address comes from
// cudaGetSymbolAddress, asked once per device with that device current.
int noalloc_scratch(uint8_t** out) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return B200_ERR_CUDA;
  std::lock_guard<std::mutex> lk(g_noalloc_mu);
  if (!g_noalloc_ptr[dev]) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_noalloc_scratch) != cudaSuccess || p == nullptr) {
      cudaGetLastError();
      return B200_ERR_CUDA;
    }
    g_noalloc_ptr[dev] = static_cast<uint8_t*>(p);
  }
  *out = g_noalloc_ptr[dev];
  return B200_OK;
}

}  // namespace
}  // namespace b200

extern "C" int b200_gemm_f16_noalloc(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K,
                                     int64_t lda, int64_t ldb, int64_t ldc, int b_layout, void* stream_ptr) {
  using namespace b200;
  bool done = false;
  if (int rc = validate_args(C, M, N, K, lda, ldb, ldc, b_layout, A, B, &done)) return rc;
  if (done) return B200_OK;
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  if (!dev.sm100) return B200_ERR_UNSUPPORTED_DEVICE;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  // The split last wave of the pair kernel keeps its parts in a per-stream
  // workspace that is allocated on first use; this entry runs every tile whole.
  CallOptions opts;
  opts.no_split = true;
  const ScopedCallOptions scoped(opts);
  const RepackPlan p = plan_repack(A, B, C, M, N, K, lda, ldb, ldc, b_layout);
  if (p.bytes == 0)
    return gemm_aligned<false>(A, B, C, M, N, K, lda, ldb, ldc, B200_A_ROW_MAJOR, b_layout, EpiParams{}, dev, stream);
  if (p.bytes > kNoAllocScratchBytes) return B200_ERR_SCRATCH_LIMIT;
  uint8_t* scratch = nullptr;
  if (int rc = noalloc_scratch(&scratch)) return rc;
  // Nothing in the scratch has to start at zero: the call writes every byte it
  // later reads (the re-pitched operand rows, and all of C's copy) first.
  return gemm_repacked(A, B, C, M, N, K, lda, ldb, ldc, B200_A_ROW_MAJOR, b_layout, EpiParams{}, p, scratch, dev,
                       stream);
}

// ===========================================================================
// K-means assignment (b200_kmeans_assign_f16)
// ===========================================================================
namespace b200 {
namespace {

// ||c_j||^2 in fp32 for each centroid j (column j of a row-major K x N matrix,
// or row j of an N x K one).
__global__ void centroid_norms_kernel(const __half* Cent, int64_t ld, int N, int K, int row_major_kn, float* out) {
  if (row_major_kn) {
    // Column j of K x N: consecutive threads read consecutive columns.
    const int j = blockIdx.x * blockDim.x + threadIdx.x;
    if (j >= N) return;
    float s = 0.0f;
    for (int k = 0; k < K; ++k) {
      const float v = __half2float(Cent[(int64_t)k * ld + j]);
      s = fmaf(v, v, s);
    }
    out[j] = s;
  } else {
    // Row j of N x K: one warp per centroid, lanes stride along the row.
    const int j = (blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (j >= N) return;
    float s = 0.0f;
    for (int k = lane; k < K; k += 32) {
      const float v = __half2float(Cent[(int64_t)j * ld + k]);
      s = fmaf(v, v, s);
    }
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) out[j] = s;
  }
}

__global__ void unpack_keys_kernel(const unsigned long long* keys, int M, int* idx, float* score) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= M) return;
  const unsigned long long k = keys[i];
  idx[i] = (int)(k & 0xffffffffu);
  if (score) score[i] = ordered_to_float((uint32_t)(k >> 32));
}

int64_t kmeans_ws_parts(int64_t M, int64_t N, int64_t* keys_off) {
  *keys_off = round_up(N * 4, 256);
  return *keys_off + round_up(M * 8, 256);
}

}  // namespace
}  // namespace b200

extern "C" int64_t b200_kmeans_workspace_size(int64_t M, int64_t N) {
  if (M < 0 || N < 0) return -B200_ERR_INVALID_ARGUMENT;
  int64_t off = 0;
  return b200::kmeans_ws_parts(M, N, &off);
}

extern "C" int b200_kmeans_assign_f16(const void* X, const void* Cent, int64_t M, int64_t N, int64_t K, int64_t ldx,
                                      int64_t ldcent, int cent_layout, void* workspace, int64_t workspace_bytes,
                                      int32_t* out_idx, float* out_score, void* stream_ptr) {
  using namespace b200;
  if (M < 0 || N <= 0 || K <= 0 || K > 256) return K > 256 ? B200_ERR_TOO_LARGE : B200_ERR_INVALID_ARGUMENT;
  if (cent_layout != B200_B_ROW_MAJOR && cent_layout != B200_B_COL_MAJOR) return B200_ERR_INVALID_ARGUMENT;
  if (M > 0x7fffffff || N > 0x7fffffff) return B200_ERR_TOO_LARGE;
  if (M == 0) return B200_OK;
  const bool row_b = (cent_layout == B200_B_ROW_MAJOR);
  if (!X || !Cent || !out_idx || ldx < K || ldcent < (row_b ? N : K)) return B200_ERR_INVALID_ARGUMENT;
  if (!pitch_ok(X, ldx) || !pitch_ok(Cent, ldcent)) return B200_ERR_MISALIGNED;
  int64_t keys_off = 0;
  const int64_t need = kmeans_ws_parts(M, N, &keys_off);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
    return B200_ERR_WORKSPACE;
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  if (!dev.sm100) return B200_ERR_UNSUPPORTED_DEVICE;
  if ((N + 255) / 256 > dev.sm_count) return B200_ERR_TOO_LARGE;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  float* cnorm = static_cast<float*>(workspace);
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(static_cast<uint8_t*>(workspace) + keys_off);
  const unsigned norm_blocks = row_b ? (unsigned)((N + 127) / 128) : (unsigned)((N * 32 + 127) / 128);
  centroid_norms_kernel<<<norm_blocks, 128, 0, stream>>>(static_cast<const __half*>(Cent), ldcent, (int)N, (int)K,
                                                          row_b ? 1 : 0, cnorm);
  if (cudaGetLastError() != cudaSuccess) return B200_ERR_CUDA;
  if (cudaMemsetAsync(keys, 0xff, M * 8, stream) != cudaSuccess) return B200_ERR_CUDA;
  GemmArgs g{X, Cent, nullptr, (int)M, (int)N, (int)K, ldx, ldcent, 0, EpiParams{}, dev.sm_count, stream};
  g.argmin.cnorm = cnorm;
  g.argmin.keys = keys;
  // The argmin epilogue stages no C, so its staging space is a sixth A stage
  // (measured ~1 % faster than five at 262144 x 1024 x 256).
  // 16 epilogue warps for K <= 128, 8 above (B200_GEMM_KM16=0/1 forces one; tuning only).
  static const int km16_env = [] { const char* e = std::getenv("B200_GEMM_KM16"); return e ? std::atoi(e) : -1; }();
  const bool km16 = km16_env >= 0 ? km16_env == 1 : K <= 128;
  const int rc = km16 ? (row_b ? launch_skinny<6, 0, true, false, true, 16>(g) : launch_skinny<6, 0, false, false, true, 16>(g))
                      : (row_b ? launch_skinny<6, 0, true, false, true>(g) : launch_skinny<6, 0, false, false, true>(g));
  if (rc) return rc;
  unpack_keys_kernel<<<(unsigned)((M + 255) / 256), 256, 0, stream>>>(keys, (int)M, out_idx, out_score);
  return cudaGetLastError() == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}

// ---------------------------------------------------------------------------
// Gathered output (multi-GPU): every rank computes its row shard of C and its
// epilogue writes each finished block both to its own copy of the gathered C
// and, with plain 16-byte stores over NVLink, to every peer's copy, so the
// all-gather of C runs tile by tile under the GEMM instead of after it.  The
// peers' buffers come from this library's IPC helpers (legacy CUDA IPC: one
// cudaMalloc per buffer, no multicast object).  The kernels never wait on a
// peer: completion is the caller's device-side barrier after the launch.
// ---------------------------------------------------------------------------
namespace b200 {

// K == 0 in gathered mode: zero this shard's rows in the local and every peer
// buffer (plain stores, like the epilogue's).
__global__ void zero_rows_kernel(uint16_t* c, const __grid_constant__ EpiParams ep, int64_t rows, int64_t cols) {
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y)
    for (int64_t col = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; col < cols;
         col += (int64_t)gridDim.x * blockDim.x) {
      c[r * ep.ldc + col] = 0;
      for (int p = 0; p < ep.n_peers; ++p) ep.peer[p][r * ep.ldc + col] = 0;
    }
  if (ep.n_peers > 0) __threadfence_system();
}

}  // namespace b200

extern "C" int b200_ipc_handle_size(void) { return (int)sizeof(cudaIpcMemHandle_t); }

extern "C" int b200_ipc_alloc(int64_t bytes, void** ptr, void* handle) {
  if (bytes <= 0 || !ptr || !handle) return B200_ERR_INVALID_ARGUMENT;
  *ptr = nullptr;
  void* p = nullptr;
  if (cudaMalloc(&p, (size_t)bytes) != cudaSuccess) return B200_ERR_CUDA;
  cudaIpcMemHandle_t h;
  if (cudaIpcGetMemHandle(&h, p) != cudaSuccess) {
    cudaFree(p);
    return B200_ERR_CUDA;
  }
  std::memcpy(handle, &h, sizeof(h));
  *ptr = p;
  return B200_OK;
}

extern "C" int b200_ipc_free(void* ptr) {
  if (!ptr) return B200_OK;
  return cudaFree(ptr) == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}

extern "C" int b200_ipc_open(const void* handle, void** ptr) {
  if (!handle || !ptr) return B200_ERR_INVALID_ARGUMENT;
  *ptr = nullptr;
  cudaIpcMemHandle_t h;
  std::memcpy(&h, handle, sizeof(h));
  void* p = nullptr;
  if (cudaIpcOpenMemHandle(&p, h, cudaIpcMemLazyEnablePeerAccess) != cudaSuccess) return B200_ERR_CUDA;
  *ptr = p;
  return B200_OK;
}

extern "C" int b200_ipc_close(void* ptr) {
  if (!ptr) return B200_OK;
  return cudaIpcCloseMemHandle(ptr) == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}

extern "C" int b200_gemm_f16_gather(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K,
                                    int64_t lda, int64_t ldb, int64_t ldc, int b_layout, void* const* peer_c,
                                    int n_peers, void* stream_ptr) {
  using namespace b200;
  if (n_peers < 0 || n_peers > kMaxPeers || (n_peers > 0 && !peer_c)) return B200_ERR_INVALID_ARGUMENT;
  bool done = false;
  if (int rc = validate_args(C, M, N, K, lda, ldb, ldc, b_layout, A, B, &done)) return rc;
  if (done) return B200_OK;
  EpiParams ep;
  ep.n_peers = n_peers;
  ep.m = (int)M;
  ep.n = (int)N;
  ep.ldc = ldc;
  for (int p = 0; p < n_peers; ++p) {
    if (!peer_c[p]) return B200_ERR_INVALID_ARGUMENT;
    if (!aligned16(peer_c[p])) return B200_ERR_MISALIGNED;
    ep.peer[p] = static_cast<uint16_t*>(peer_c[p]);
  }
  DeviceInfo dev;
  if (int rc = current_device_info(dev)) return rc;
  if (!dev.sm100) return B200_ERR_UNSUPPORTED_DEVICE;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (K == 0) {
    const unsigned gx = (unsigned)std::min<int64_t>((N + 255) / 256, 64);
    const unsigned gy = (unsigned)std::min<int64_t>(M, 65535);
    zero_rows_kernel<<<dim3(gx, gy), 256, 0, stream>>>(static_cast<uint16_t*>(C), ep, M, N);
    return cudaGetLastError() == cudaSuccess ? B200_OK : B200_ERR_CUDA;
  }
  // Operands must be TMA-addressable as they are: a re-pitched C would leave
  // the peers' copies unwritten.
  if (plan_repack(A, B, C, M, N, K, lda, ldb, ldc, b_layout, B200_A_ROW_MAJOR).bytes != 0) return B200_ERR_MISALIGNED;
  return gemm_aligned<false>(A, B, C, M, N, K, lda, ldb, ldc, B200_A_ROW_MAJOR, b_layout, ep, dev, stream);
}
