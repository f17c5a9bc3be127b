// What the translation units of the library offer each other.
#pragma once

#include <cstdint>

namespace b200 {

// C = A * B (fp32 accumulate, rounded once to the operands' type) on operands
// that satisfy TMA's alignment rules, M and N > 0, on the current device;
// layouts as in b200_gemm_f16_ex.  `stream` is a cudaStream_t.
int gemm_f16_run(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb,
                 int64_t ldc, int a_layout, int b_layout, void* stream);
int gemm_bf16_run(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb,
                  int64_t ldc, int a_layout, int b_layout, void* stream);

// Reads and clears the device error word of another unit's kernels on the
// current device, which must be idle (0: none, negative: a CUDA error).
int take_error_word_gemm_bf16();
int take_error_word_ffn();

}  // namespace b200
