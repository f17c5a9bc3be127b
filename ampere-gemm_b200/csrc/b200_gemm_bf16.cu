// The GEMM kernels for bf16 operands (fp32 accumulate, bf16 out), used by the
// gated feed-forward block; see gemm_launch.cuh.
#include "gemm_internal.h"
#include "gemm_launch.cuh"

namespace b200 {

int gemm_bf16_run(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb,
                  int64_t ldc, int a_layout, int b_layout, void* split_ws, void* stream) {
  return gemm_run<true>(A, B, C, M, N, K, lda, ldb, ldc, a_layout, b_layout, split_ws, stream);
}

int take_error_word_gemm_bf16() { return take_error_word(); }

}  // namespace b200
