// What the translation units of the library offer each other.
#pragma once

#include <cstdint>

namespace b200 {

// Workspace for the parts of a last wave that is split along K: kSplitParts
// accumulators of 128 x 256 fp32, then as many counters, zero between launches.
constexpr int kSplitParts = 160;
constexpr int64_t kSplitPartBytes = 128 * 256 * 4;
constexpr int64_t kSplitBytes = kSplitParts * kSplitPartBytes + 1024;

// C = A * B (fp32 accumulate, rounded once to the operands' type) on operands
// that satisfy TMA's alignment rules, M and N > 0, on the current device;
// layouts as in b200_gemm_f16_ex.  `split_ws` is kSplitBytes of the caller's
// memory (NULL: every tile runs whole); nothing is allocated, and
// b200_gemm_set_variant does not apply.  `stream` is a cudaStream_t.
int gemm_f16_run(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb,
                 int64_t ldc, int a_layout, int b_layout, void* split_ws, void* stream);
int gemm_bf16_run(const void* A, const void* B, void* C, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb,
                  int64_t ldc, int a_layout, int b_layout, void* split_ws, void* stream);

// Reads and clears the device error word of another unit's kernels on the
// current device, which must be idle (0: none, negative: a CUDA error).
int take_error_word_gemm_bf16();
int take_error_word_ffn();

}  // namespace b200
