// Tensor-map encoding and cluster occupancy for the translation units that
// launch the GEMM kernels (unnamed namespace, as in host_common.cuh).
#pragma once

#include <cuda.h>

#include <cstdio>

#include "gemm_common.cuh"
#include "host_common.cuh"

namespace b200 {
namespace {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn get_encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// 2-D fp16 tensor map over a row-major matrix of `rows` x `cols` (cols
// contiguous, `ld` elements between rows), box `box_cols` x `box_rows`,
// 128-byte swizzle, zero fill out of bounds.
int encode_tmap_2d(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_cols,
                   uint32_t box_rows, CUtensorMapL2promotion promo) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return B200_ERR_TENSOR_MAP;
  // A zero-extent dimension is not encodable; callers never pass one.
  cuuint64_t dims[2] = {cols, rows};
  cuuint64_t strides[1] = {ld * 2};
  cuuint32_t box[2] = {box_cols, box_rows};
  cuuint32_t estr[2] = {1, 1};
  auto encode = [&] {
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, promo, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT) {
    // A thread that has made no runtime call yet (e.g. autograd's device
    // thread) has no current context for this driver call: cudaSetDevice on
    // the current device makes the primary context current, then retry.
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = encode();
  }
  if (r != CUDA_SUCCESS && std::getenv("B200_GEMM_DEBUG"))
    std::fprintf(stderr, "b200_gemm: tensor map rejected (%d): base %p rows %llu cols %llu ld %llu box %u x %u\n",
                 (int)r, base, (unsigned long long)rows, (unsigned long long)cols, (unsigned long long)ld, box_cols,
                 box_rows);
  return r == CUDA_SUCCESS ? B200_OK : B200_ERR_TENSOR_MAP;
}

// Encoding a tensor map is a driver call of about a microsecond; repeated
// GEMMs on the same buffers reuse the encoded map from a small per-thread
// cache keyed by every field that goes into it.
struct TmapKey {
  const void* base;
  uint64_t rows, cols, ld;
  uint32_t box_cols, box_rows, promo;
  bool operator==(const TmapKey& o) const {
    return base == o.base && rows == o.rows && cols == o.cols && ld == o.ld && box_cols == o.box_cols &&
           box_rows == o.box_rows && promo == o.promo;
  }
};

struct TmapCache {
  static constexpr int kEntries = 24;
  TmapKey key[kEntries];
  CUtensorMap map[kEntries];
  bool used[kEntries] = {};
  int next = 0;
};

int make_tmap_2d(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_cols,
                 uint32_t box_rows, CUtensorMapL2promotion promo) {
  static thread_local TmapCache cache;
  const TmapKey k{base, rows, cols, ld, box_cols, box_rows, static_cast<uint32_t>(promo)};
  for (int i = 0; i < TmapCache::kEntries; ++i) {
    if (cache.used[i] && cache.key[i] == k) {
      *map = cache.map[i];
      return B200_OK;
    }
  }
  const int rc = encode_tmap_2d(map, base, rows, cols, ld, box_cols, box_rows, promo);
  if (rc != B200_OK) return rc;
  const int slot = cache.next;
  cache.next = (cache.next + 1) % TmapCache::kEntries;
  cache.key[slot] = k;
  cache.map[slot] = *map;
  cache.used[slot] = true;
  return B200_OK;
}

// Largest number of 2-CTA clusters of `kern` that can be resident at once
// (clusters need both SMs in one GPC, so this can be below sm_count / 2).
template <typename Kern>
int max_active_pairs(Kern kern, int smem_bytes, int sm_count) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (sm_count / 2), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem_bytes;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    n = sm_count / 2;
  }
  return n;
}

}  // namespace
}  // namespace b200
