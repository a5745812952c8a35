// kv_cache.cuh -- the KV cache as the kernels of kv_cache.cu and
// tree_attention.cu see it.
#pragma once

#include "../../include/odi_cuda.h"
#include "common.cuh"

namespace odi_cuda {

// Byte offset of an int8 cache's row scales: after the codes, on the next
// 256-byte boundary.
__host__ __device__ inline int64_t kv_scale_offset(int kv_heads, int hd, int ctx) {
  return ((int64_t)kv_heads * ctx * hd + 255) / 256 * 256;
}

struct KvView {
  void* k;
  void* v;
  int dtype;  // ODI_CUDA_KV_F16 / ODI_CUDA_KV_I8
  int kv_heads, hd, ctx;
  int64_t scale_off;
};

// Checks a caller's cache descriptor; `who` opens the error message.
int kv_view(const odi_cuda_kv_cache* c, KvView* v, const char* who);
// Whether n rows of wa values, lda apart, share memory with n rows of wb, ldb apart.
inline bool rows_overlap(const float* a, int64_t lda, int64_t wa, const float* b, int64_t ldb, int64_t wb, int64_t n) {
  const intptr_t A = (intptr_t)a, B = (intptr_t)b;
  if (n < 1 || A + 4 * ((n - 1) * lda + wa) <= B || B + 4 * ((n - 1) * ldb + wb) <= A) return false;
  for (int64_t i = 0, j = 0; i < n && j < n;) {
    const intptr_t x = A + 4 * i * lda, y = B + 4 * j * ldb;
    if (x + 4 * wa <= y) ++i;
    else if (y + 4 * wb <= x) ++j;
    else return true;
  }
  return false;
}
// A launch's status as the C ABI's.
int kv_launched(cudaError_t e, const char* what);

}  // namespace odi_cuda
