// paged_append.cu -- new tokens of several requests into a paged cache: q and k
// normed per head and rotated, k and v stored at the step's slots, q in the
// cache's type.
//
// Per head x of a token at position p: x <- x / sqrt(mean(x^2) + eps) * w (where
// there are weights), then the pairs (i, i + hd/2) turned by p * theta^(-2i/hd).
// The angle is reduced to a fraction of a turn in 64 bits: in fp32 it would be
// off by 6e-3 rad at position 100,000.
//
// One warp takes NH consecutive heads of one token, all loaded before the first
// is used, and its angles serve them all.  Bound by HBM: 4,100 tokens of 64/8 heads
// of 128 dims take 35.3 us, 5.9 TB/s of what they read and write.  Eight tokens take
// 2.0 us: two round trips to memory and a launch.
#include <math.h>

#include "internal.h"
#include "kv_cache.cuh"
#include "paged.cuh"
#include "pdl_launch.cuh"

namespace odi_cuda {
namespace {

// theta^(-2/hd) and its squares: a lane makes its pair's power by its own bits.
struct Turns {
  double r;
  double square[5];
};

template <typename T>
__device__ __forceinline__ T to16(float x);
template <>
__device__ __forceinline__ __half to16<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 to16<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, int PPL>
__device__ __forceinline__ void store16(T* p, const float (&x)[PPL]) {
  if (PPL == 2) {
    const T a[2] = {to16<T>(x[0]), to16<T>(x[PPL - 1])};
    *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(a);
  } else {
    *p = to16<T>(x[0]);
  }
}

template <typename T, int HD, int NH, bool VEC>
__global__ void __launch_bounds__(128) paged_append_kernel(const float* qkv, int64_t ld, const float* __restrict__ q_norm,
                                                           const float* __restrict__ k_norm, float eps, T* q_out,
                                                           int64_t ld_q, PagedView cache, const int* positions,
                                                           const int* slots, int tokens, int heads,
                                                           const __grid_constant__ Turns turns) {
  constexpr int PPL = HD / 64, HALF = HD / 2;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int rows = heads + 2 * cache.kv_heads;
  const int groups = (rows + NH - 1) / NH;
  const int64_t unit = blockIdx.x * 4ll + (threadIdx.x >> 5);
  const int t = (int)(unit / groups), r0 = (int)(unit % groups) * NH;
  if (t >= tokens) return;
  const int slot = __ldcg(slots + t), pos = __ldcg(positions + t);
  const float* src = qkv + t * ld + lane * PPL;
  float lo[NH][PPL], hi[NH][PPL];
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    if (r0 + n >= rows) break;
    const float* p = src + (int64_t)(r0 + n) * HD;
    if (VEC && PPL == 2) {
      const float2 a = __ldcg(reinterpret_cast<const float2*>(p)), b = __ldcg(reinterpret_cast<const float2*>(p + HALF));
      lo[n][0] = a.x, lo[n][PPL - 1] = a.y, hi[n][0] = b.x, hi[n][PPL - 1] = b.y;
    } else {
#pragma unroll
      for (int e = 0; e < PPL; ++e) lo[n][e] = __ldcg(p + e), hi[n][e] = __ldcg(p + HALF + e);
    }
  }
  const int page = slot >> cache.page_shift;
  if (slot < 0 || page >= cache.num_pages) return;  // not a row of the step, or of a request that was refused
  double x = (double)pos * 0.15915494309189533577;  // 1 / (2 pi)
#pragma unroll
  for (int k = 0; k < 5; ++k) x *= (lane >> k) & 1 ? turns.square[k] : 1.0;
  float sn[PPL], cs[PPL];
#pragma unroll
  for (int e = 0; e < PPL; ++e) {
    if (e) x *= turns.r;
    sincospif(2.0f * (float)(x - rint(x)), &sn[e], &cs[e]);
  }
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    const int r = r0 + n;
    if (r >= rows) break;
    const int kind = r < heads ? 0 : r < heads + cache.kv_heads ? 1 : 2;  // q, k, v
    if (kind < 2) {
      const float* w = kind ? k_norm : q_norm;
      if (w) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < PPL; ++e) s += lo[n][e] * lo[n][e] + hi[n][e] * hi[n][e];
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        const float inv = 1.0f / sqrtf(s / (float)HD + eps);
#pragma unroll
        for (int e = 0; e < PPL; ++e) {
          lo[n][e] *= inv * w[lane * PPL + e];
          hi[n][e] *= inv * w[HALF + lane * PPL + e];
        }
      }
#pragma unroll
      for (int e = 0; e < PPL; ++e) {
        const float a = lo[n][e], b = hi[n][e];
        lo[n][e] = a * cs[e] - b * sn[e];
        hi[n][e] = a * sn[e] + b * cs[e];
      }
    }
    T* o;
    if (kind == 0) {
      o = q_out + t * ld_q + (int64_t)r * HD;
    } else {
      const int h = r - heads - (kind - 1) * cache.kv_heads;
      o = static_cast<T*>(kind == 1 ? cache.k : cache.v) +
          ((((int64_t)page * cache.kv_heads + h) << cache.page_shift) + (slot & (cache.page_size - 1))) * HD;
    }
    store16(o + lane * PPL, lo[n]);
    store16(o + HALF + lane * PPL, hi[n]);
  }
}

struct AppendArgs {
  const float* qkv;
  int64_t ld;
  const float *q_norm, *k_norm;
  float eps;
  void* q_out;
  int64_t ld_q;
  PagedView c;
  const int *positions, *slots;
  int tokens, heads;
  Turns turns;
};
template <typename T, int HD, int NH, bool VEC>
cudaError_t launch(const AppendArgs& a, cudaStream_t s) {
  const int groups = (a.heads + 2 * a.c.kv_heads + NH - 1) / NH;
  const dim3 grid((unsigned)(((int64_t)a.tokens * groups + 3) / 4));
  return launch_pdl(paged_append_kernel<T, HD, NH, VEC>, grid, dim3(128), s, a.qkv, a.ld, a.q_norm, a.k_norm, a.eps,
                    static_cast<T*>(a.q_out), a.ld_q, a.c, a.positions, a.slots, a.tokens, a.heads, a.turns);
}
template <typename T, int HD>
cudaError_t launch_hd(const AppendArgs& a, bool many, bool vec, cudaStream_t s) {
  return many ? (vec ? launch<T, HD, 4, true>(a, s) : launch<T, HD, 4, false>(a, s))
              : (vec ? launch<T, HD, 1, true>(a, s) : launch<T, HD, 1, false>(a, s));
}

}  // namespace
}  // namespace odi_cuda

using namespace odi_cuda;

extern "C" {

int odi_cuda_qk_rope_append_paged(const float* d_qkv, int64_t ld_qkv, const float* d_q_norm, const float* d_k_norm,
                                  float eps, void* d_q_out, int64_t ld_q, const odi_cuda_paged_cache* cache,
                                  const odi_cuda_paged_batch* batch, int tokens, int heads, float theta, void* stream) {
  AppendArgs a{};
  PagedGeometry g;
  if (int rc = paged_view(cache, &a.c, "qk_rope_append_paged")) return rc;
  if (int rc = paged_batch_ok(batch, &g, "qk_rope_append_paged")) return rc;
  if (batch->page_size != a.c.page_size)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "qk_rope_append_paged: cache and batch of different page_size");
  if (!d_qkv || !d_q_out) return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "qk_rope_append_paged: null argument");
  if (tokens < 0 || tokens > batch->max_rows || heads < 1 || heads > 65535 || !(theta > 0.f) || !isfinite(theta))
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "qk_rope_append_paged: tokens, heads or theta out of range");
  const int64_t rows = heads + 2ll * a.c.kv_heads;
  if (ld_qkv < rows * a.c.hd || ld_q < (int64_t)heads * a.c.hd || ld_qkv > (1ll << 40) || ld_q > (1ll << 40))
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "qk_rope_append_paged: a row stride is shorter than its row");
  if (((uintptr_t)d_qkv | (uintptr_t)d_q_norm | (uintptr_t)d_k_norm) & 3 || (uintptr_t)d_q_out & 3 || ld_q & 1)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "qk_rope_append_paged: misaligned buffer");
  if ((int64_t)tokens * rows > 0x7fffffffll)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "qk_rope_append_paged: too many rows");
  if (!tokens) return ODI_CUDA_OK;
  if (byte_rows_overlap(d_qkv, 4 * ld_qkv, 4 * rows * a.c.hd, d_q_out, 2 * ld_q, 2ll * heads * a.c.hd, tokens))
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "qk_rope_append_paged: d_q_out overlaps d_qkv");
  const int64_t q_bytes = 2 * ((tokens - 1) * ld_q + (int64_t)heads * a.c.hd), qkv_bytes = 4 * ((tokens - 1) * ld_qkv + rows * a.c.hd);
  for (const void* pool : {a.c.k, a.c.v})
    if (bytes_overlap(d_q_out, q_bytes, pool, a.c.bytes()) || bytes_overlap(d_qkv, qkv_bytes, pool, a.c.bytes()))
      return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "qk_rope_append_paged: d_q_out or d_qkv overlaps the cache");
  a.turns.r = pow((double)theta, -2.0 / a.c.hd);
  double sq = a.c.hd == 128 ? a.turns.r * a.turns.r : a.turns.r;
  for (int k = 0; k < 5; ++k, sq *= sq) a.turns.square[k] = sq;
  a.qkv = d_qkv, a.ld = ld_qkv, a.q_norm = d_q_norm, a.k_norm = d_k_norm, a.eps = eps, a.q_out = d_q_out, a.ld_q = ld_q;
  a.positions = batch->positions, a.slots = batch->slots, a.tokens = tokens, a.heads = heads;
  const bool vec = !((uintptr_t)d_qkv & 7) && !(ld_qkv & 1);
  // Four heads per warp share their angles and are loaded together; with few
  // rows one head per warp spreads the call over more SMs.
  const bool many = (int64_t)tokens * rows >= 148 * 16, bf = a.c.dtype == ODI_CUDA_PAGED_BF16;
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  if (a.c.hd == 128) e = bf ? launch_hd<__nv_bfloat16, 128>(a, many, vec, s) : launch_hd<__half, 128>(a, many, vec, s);
  else e = bf ? launch_hd<__nv_bfloat16, 64>(a, many, vec, s) : launch_hd<__half, 64>(a, many, vec, s);
  return kv_launched(e, "qk_rope_append_paged");
}

}  // extern "C"
