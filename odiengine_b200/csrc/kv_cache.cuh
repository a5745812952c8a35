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
// A launch's status as the C ABI's.
int kv_launched(cudaError_t e, const char* what);

}  // namespace odi_cuda
