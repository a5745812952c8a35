// kv_cache.cu -- KV caches of several tokens per call: rows written with the
// per-head norm and the rotation in the same pass, read back, and moved.
//
// An fp16 cache is [kv_head][ctx][head_dim] halves, the layout that
// rope_kv_kernel and attn_kernel use.  An int8 cache holds [kv_head][ctx]
// [head_dim] codes and, from the next 256-byte boundary, one fp32 scale per
// row, [kv_head][ctx]: row = code * scale.  One scale per row (not per 32
// values) keeps a row 16-byte aligned for every head_dim, and lets the
// attention multiply the codes as they lie and apply the scale once per score.
#include <math.h>

#include <cstdio>

#include "../../include/odi_cuda.h"
#include "kv_cache.cuh"
#include "internal.h"
#include "pdl_launch.cuh"

namespace odi_cuda {
namespace {

__device__ __forceinline__ float warp_sum_all(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Turns per position of pair i, r^i / (2 pi) with r = theta^(-2/hd), in 64 bits:
// the angle of a far position is a large number of turns, and only its fraction
// matters.  The product is good to about 2^-50 of itself and the whole turns
// are dropped before it becomes fp32, so the angle is good to 2^-24 of a turn up
// to position 2^27 (in fp32 it is off by 6e-3 rad at position 100,000).  A lane
// makes its pair's power from the squares of r, five products by its own bits: a
// table of all pairs as a kernel argument, of which every lane reads another
// entry, serialises in the constant cache (512 tokens of 64/8 heads out of L2:
// 9.6 us, 6.7 this way).
struct Turns {
  double r;          // from one pair to the next
  double square[5];  // PPL pairs on, twice as many, ...
};

// One warp takes NH consecutive heads of one token (of the token's heads + 2
// kv_heads rows of q, k and v), all loaded before the first is used.  Lane l
// holds pairs l * PPL .. + PPL - 1 and their partners head_dim / 2 higher, so
// its angles serve all its heads.  Bound by HBM for many tokens -- 512 tokens
// of 64/8 heads read and write 39.8 MB in 8.8 us, 4.5 TB/s -- and by latency for
// few: one token of 32/8 heads takes 3.3 us.
template <int HD, int NH, bool VEC>
__global__ void __launch_bounds__(128) append_kernel(const float* qkv, int64_t ld, const float* __restrict__ q_norm,
                                                     const float* __restrict__ k_norm, float eps, float* q_out,
                                                     int64_t ld_q, KvView cache, const DecodeState* st,
                                                     const int* __restrict__ depth, int tokens, int heads,
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
  const int pos = __ldcg(&st->pos);
  const int64_t slot = (int64_t)pos + t;
  const bool store = slot >= 0 && slot < cache.ctx;
  const double p = (double)((int64_t)pos + (depth ? __ldcg(depth + t) : t));
  double x = p * 0.15915494309189533577;  // 1 / (2 pi)
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
        const float inv = 1.0f / sqrtf(warp_sum_all(s) / (float)HD + eps);
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
    if (kind == 0) {
      float* o = q_out + t * ld_q + (int64_t)r * HD + lane * PPL;
      if (VEC && PPL == 2) {
        *reinterpret_cast<float2*>(o) = make_float2(lo[n][0], lo[n][PPL - 1]);
        *reinterpret_cast<float2*>(o + HALF) = make_float2(hi[n][0], hi[n][PPL - 1]);
      } else {
#pragma unroll
        for (int e = 0; e < PPL; ++e) o[e] = lo[n][e], o[HALF + e] = hi[n][e];
      }
      continue;
    }
    if (!store) continue;
    const int h = r - heads - (kind - 1) * cache.kv_heads;
    const int64_t row = (int64_t)h * cache.ctx + slot;
    uint8_t* base = static_cast<uint8_t*>(kind == 1 ? cache.k : cache.v);
    if (cache.dtype == ODI_CUDA_KV_F16) {
      __half* o = reinterpret_cast<__half*>(base) + row * HD + lane * PPL;
#pragma unroll
      for (int e = 0; e < PPL; ++e) o[e] = __float2half_rn(lo[n][e]), o[HALF + e] = __float2half_rn(hi[n][e]);
    } else {
      float am = 0.f;
      bool fin = true;
#pragma unroll
      for (int e = 0; e < PPL; ++e) {
        am = fmaxf(am, fmaxf(fabsf(lo[n][e]), fabsf(hi[n][e])));
        fin = fin && isfinite(lo[n][e]) && isfinite(hi[n][e]);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, o));
      fin = __all_sync(0xffffffffu, fin);
      float d = q8_scale(am);
      // a scale below the normal range has no fp32 reciprocal: the row is zero.
      // A row with a value that is not finite reads back as NaN.
      if (!(d >= 1.17549435e-38f)) d = 0.f;
      const float id = fin ? q8_inv(d) : 0.f;
      int8_t* o = reinterpret_cast<int8_t*>(base) + row * HD + lane * PPL;
#pragma unroll
      for (int e = 0; e < PPL; ++e) {
        o[e] = (int8_t)(fin ? q8_round(__fmul_rn(lo[n][e], id)) : 0);
        o[HALF + e] = (int8_t)(fin ? q8_round(__fmul_rn(hi[n][e], id)) : 0);
      }
      if (lane == 0) reinterpret_cast<float*>(base + cache.scale_off)[row] = fin ? d : __int_as_float(0x7fc00000);
    }
  }
}

// Rows start .. start + count of K (blockIdx.z = 0) and V (1) as fp16 or
// fp32, [kv_head][count][hd].  A thread makes one 16-byte piece of the output at
// a time, two 256 pieces apart, so that a warp's stores are whole lines.  HBM
// bound: 32001 int8 positions of 8 heads to fp16 are 199 MB in 31.1 us, 6.4
// TB/s, three quarters of them writes (37.7 with 32 bytes per thread in two
// stores; 38.7, 31.9 and 31.2 with one, two and four pieces and stores that are
// not marked as streaming).  77 positions take 1.3 us.
constexpr int READ_U = 2;
template <bool I8, bool OUT16>
__global__ void __launch_bounds__(256) kv_read_kernel(KvView cache, int start, int count, void* k_out, void* v_out) {
  constexpr int U = READ_U, CH = OUT16 ? 8 : 4;  // pieces per thread, values per piece
  pdl_launch_dependents();
  pdl_wait();
  void* out = blockIdx.z ? v_out : k_out;
  if (!out) return;
  const uint8_t* base = static_cast<const uint8_t*>(blockIdx.z ? cache.v : cache.k);
  const int shift = (cache.hd == 128 ? 7 : 6) - (OUT16 ? 3 : 2);  // pieces per row, log2
  const int64_t total = (int64_t)count << shift;
  const int h = blockIdx.y;
  const int64_t row0 = (int64_t)h * cache.ctx + start;
  const int64_t i0 = (int64_t)blockIdx.x * (256 * U) + threadIdx.x;
  uint32_t raw[U][I8 ? CH / 4 : CH / 2];
  float d[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = i0 + u * 256;
    if (i >= total) break;
    const uint8_t* p = base + ((row0 << shift) + i) * (CH * (I8 ? 1 : 2));
    if constexpr (sizeof raw[u] == 16) {
      const uint4 x = __ldcs(reinterpret_cast<const uint4*>(p));
      raw[u][0] = x.x, raw[u][1] = x.y, raw[u][2] = x.z, raw[u][3] = x.w;
    } else if constexpr (sizeof raw[u] == 8) {
      const uint2 x = __ldcs(reinterpret_cast<const uint2*>(p));
      raw[u][0] = x.x, raw[u][1] = x.y;
    } else {
      raw[u][0] = __ldcs(reinterpret_cast<const unsigned*>(p));
    }
    if (I8) d[u] = __ldcg(reinterpret_cast<const float*>(base + cache.scale_off) + row0 + (i >> shift));
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = i0 + u * 256;
    if (i >= total) break;
    float x[CH];
    if (I8) {
#pragma unroll
      for (int e = 0; e < CH; ++e) x[e] = (float)(int8_t)(raw[u][e / 4] >> (8 * (e % 4))) * d[u];
    } else {
#pragma unroll
      for (int e = 0; e < CH / 2; ++e) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&raw[u][e]));
        x[2 * e] = f.x, x[2 * e + 1] = f.y;
      }
    }
    uint4* dst = reinterpret_cast<uint4*>(out) + h * total + i;
    if constexpr (OUT16) {
      __half2 y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
      __stcs(dst, *reinterpret_cast<uint4*>(y));
    } else {
      __stcs(reinterpret_cast<float4*>(dst), make_float4(x[0], x[1], x[2], x[3]));
    }
  }
}

// Rows src[i] -> dst[i] of one head's K or V.  The columns of a row move
// independently, so a CTA takes 64 bytes of every listed row: it loads them
// all, waits, then stores, which is what makes overlapping lists safe.  With
// n <= 256 rows a thread holds at most four 16-byte pieces.  Latency bound: 5
// rows of 8 heads 2.3 us in a graph, 100 rows of 32 heads 6.9.
__global__ void __launch_bounds__(256) kv_move_kernel(KvView cache, const int* __restrict__ src,
                                                      const int* __restrict__ dst, int n, const DecodeState* st) {
  __shared__ int s_src[ODI_CUDA_KV_MOVE_MAX], s_dst[ODI_CUDA_KV_MOVE_MAX];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t pos = st ? __ldcg(&st->pos) : 0;
  const int tid = threadIdx.x;
  if (tid < n) {
    const int64_t a = pos + __ldcg(src + tid), b = pos + __ldcg(dst + tid);
    const bool ok = a >= 0 && a < cache.ctx && b >= 0 && b < cache.ctx;
    s_src[tid] = ok ? (int)a : -1;
    s_dst[tid] = ok ? (int)b : -1;
  }
  __syncthreads();
  int keep_src = -1, keep_dst = -1;
  if (tid < n && s_dst[tid] >= 0) {  // a destination listed twice takes its last row
    bool last = true;
    for (int j = tid + 1; j < n; ++j) last = last && s_dst[j] != s_dst[tid];
    if (last) keep_src = s_src[tid], keep_dst = s_dst[tid];
  }
  __syncthreads();
  if (tid < n) s_src[tid] = keep_src, s_dst[tid] = keep_dst;
  __syncthreads();
  const int row_bytes = cache.hd * (cache.dtype == ODI_CUDA_KV_F16 ? 2 : 1);
  uint8_t* base = static_cast<uint8_t*>(blockIdx.z ? cache.v : cache.k);
  uint8_t* rows = base + (int64_t)blockIdx.y * cache.ctx * row_bytes + blockIdx.x * 64;
  uint4 v[4];
  float d = 0.f;
  float* scale = reinterpret_cast<float*>(base + cache.scale_off) + (int64_t)blockIdx.y * cache.ctx;
  const bool scales = cache.dtype == ODI_CUDA_KV_I8 && blockIdx.x == 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int i = (tid + u * 256) >> 2;
    if (i < n && s_src[i] >= 0)
      v[u] = __ldcg(reinterpret_cast<const uint4*>(rows + (int64_t)s_src[i] * row_bytes + (tid & 3) * 16));
  }
  if (scales && tid < n && s_src[tid] >= 0) d = __ldcg(scale + s_src[tid]);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int i = (tid + u * 256) >> 2;
    if (i < n && s_src[i] >= 0)
      *reinterpret_cast<uint4*>(rows + (int64_t)s_dst[i] * row_bytes + (tid & 3) * 16) = v[u];
  }
  if (scales && tid < n && s_src[tid] >= 0) scale[s_dst[tid]] = d;
}

template <int HD, int NH>
cudaError_t launch_append(bool vec, const float* qkv, int64_t ld, const float* qn, const float* kn, float eps,
                          float* q_out, int64_t ld_q, const KvView& c, const DecodeState* st, const int* depth,
                          int tokens, int heads, const Turns& turns, cudaStream_t s) {
  const int groups = (heads + 2 * c.kv_heads + NH - 1) / NH;
  const dim3 grid((unsigned)(((int64_t)tokens * groups + 3) / 4));
  return vec ? launch_pdl(append_kernel<HD, NH, true>, grid, dim3(128), s, qkv, ld, qn, kn, eps, q_out, ld_q, c, st,
                          depth, tokens, heads, turns)
             : launch_pdl(append_kernel<HD, NH, false>, grid, dim3(128), s, qkv, ld, qn, kn, eps, q_out, ld_q, c, st,
                          depth, tokens, heads, turns);
}

}  // namespace

int kv_view(const odi_cuda_kv_cache* c, KvView* v, const char* who) {
  char buf[160];
  if (!c || !c->k || !c->v) {
    snprintf(buf, sizeof buf, "%s: null cache", who);
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, buf);
  }
  if (c->dtype != ODI_CUDA_KV_F16 && c->dtype != ODI_CUDA_KV_I8) {
    snprintf(buf, sizeof buf, "%s: cache dtype %d is neither ODI_CUDA_KV_F16 nor ODI_CUDA_KV_I8", who, c->dtype);
    return set_error(ODI_CUDA_ERR_UNSUPPORTED_DTYPE, buf);
  }
  if ((c->head_dim != 64 && c->head_dim != 128) || c->kv_heads < 1 || c->kv_heads > 65535 || c->ctx < 1) {
    snprintf(buf, sizeof buf, "%s: cache of kv_heads %d / head_dim %d / ctx %d", who, c->kv_heads, c->head_dim,
             c->ctx);
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, buf);
  }
  if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) {
    snprintf(buf, sizeof buf, "%s: the cache must be 16-byte aligned", who);
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, buf);
  }
  *v = KvView{c->k, c->v, c->dtype, c->kv_heads, c->head_dim, c->ctx, kv_scale_offset(c->kv_heads, c->head_dim, c->ctx)};
  return ODI_CUDA_OK;
}

int kv_launched(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return ODI_CUDA_OK;
  char buf[256];
  snprintf(buf, sizeof buf, "%s launch: %s (%s)", what, cudaGetErrorString(e), cudaGetErrorName(e));
  return set_error(ODI_CUDA_ERR_OPERATION_FAILED, buf);
}

}  // namespace odi_cuda

using namespace odi_cuda;

extern "C" {

size_t odi_cuda_kv_cache_bytes(int dtype, int kv_heads, int head_dim, int ctx) {
  if (kv_heads < 1 || ctx < 1 || (head_dim != 64 && head_dim != 128)) return 0;
  const int64_t n = (int64_t)kv_heads * ctx;
  if (dtype == ODI_CUDA_KV_F16) return (size_t)(n * head_dim * 2);
  if (dtype == ODI_CUDA_KV_I8) return (size_t)(kv_scale_offset(kv_heads, head_dim, ctx) + n * 4);
  return 0;
}

int odi_cuda_qk_rope_append(const float* d_qkv, int64_t ld_qkv, const float* d_q_norm, const float* d_k_norm,
                            float eps, float* d_q_out, int64_t ld_q, const odi_cuda_kv_cache* cache,
                            const odi_cuda_decode_state* d_state, const int32_t* d_depth, int tokens, int heads,
                            float theta, void* stream) {
  KvView v;
  if (int rc = kv_view(cache, &v, "qk_rope_append")) return rc;
  if (!d_qkv || !d_q_out || !d_state)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "qk_rope_append: null argument");
  if (tokens < 1 || heads < 1 || heads > 65535 || !(theta > 0.f))
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "qk_rope_append: tokens, heads or theta out of range");
  const int64_t rows = heads + 2ll * v.kv_heads;
  if (ld_qkv < rows * v.hd || ld_q < (int64_t)heads * v.hd)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "qk_rope_append: a row stride is shorter than its row");
  if (((uintptr_t)d_qkv | (uintptr_t)d_q_out | (uintptr_t)d_q_norm | (uintptr_t)d_k_norm | (uintptr_t)d_state | (uintptr_t)d_depth) & 3)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "qk_rope_append: misaligned buffer");
  if ((int64_t)tokens * rows > 0x7fffffffll)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "qk_rope_append: too many rows");
  if ((d_q_out != d_qkv || ld_q != ld_qkv) && rows_overlap(d_qkv, ld_qkv, rows * v.hd, d_q_out, ld_q, (int64_t)heads * v.hd, tokens))
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "qk_rope_append: d_q_out overlaps d_qkv and is not d_qkv itself");
  Turns turns;
  turns.r = pow((double)theta, -2.0 / v.hd);
  double sq = v.hd == 128 ? turns.r * turns.r : turns.r;
  for (int k = 0; k < 5; ++k, sq *= sq) turns.square[k] = sq;
  // 8-byte accesses where both buffers and strides allow them
  const bool vec = !(((uintptr_t)d_qkv | (uintptr_t)d_q_out) & 7) && !((ld_qkv | ld_q) & 1);
  const DecodeState* st = reinterpret_cast<const DecodeState*>(d_state);
  cudaStream_t s = (cudaStream_t)stream;
  // Four heads per warp share their angles and are loaded together; with few
  // rows one head per warp spreads the call over more SMs.
  const bool many = (int64_t)tokens * rows >= 148 * 16;
  cudaError_t e;
  if (v.hd == 128)
    e = many ? launch_append<128, 4>(vec, d_qkv, ld_qkv, d_q_norm, d_k_norm, eps, d_q_out, ld_q, v, st, d_depth,
                                     tokens, heads, turns, s)
             : launch_append<128, 1>(vec, d_qkv, ld_qkv, d_q_norm, d_k_norm, eps, d_q_out, ld_q, v, st, d_depth,
                                     tokens, heads, turns, s);
  else
    e = many ? launch_append<64, 4>(vec, d_qkv, ld_qkv, d_q_norm, d_k_norm, eps, d_q_out, ld_q, v, st, d_depth,
                                    tokens, heads, turns, s)
             : launch_append<64, 1>(vec, d_qkv, ld_qkv, d_q_norm, d_k_norm, eps, d_q_out, ld_q, v, st, d_depth,
                                    tokens, heads, turns, s);
  return kv_launched(e, "qk_rope_append");
}

int odi_cuda_kv_read(const odi_cuda_kv_cache* cache, int start, int count, void* d_k_out, void* d_v_out,
                     int out_dtype, void* stream) {
  KvView v;
  if (int rc = kv_view(cache, &v, "kv_read")) return rc;
  if (start < 0 || count < 0 || start > v.ctx - count)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "kv_read: positions outside the cache");
  if (out_dtype != ODI_CUDA_KV_OUT_F16 && out_dtype != ODI_CUDA_KV_OUT_F32)
    return set_error(ODI_CUDA_ERR_UNSUPPORTED_DTYPE, "kv_read: output is ODI_CUDA_KV_OUT_F16 or ODI_CUDA_KV_OUT_F32");
  if (!count) return ODI_CUDA_OK;
  if (!d_k_out && !d_v_out) return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "kv_read: no output");
  if (((uintptr_t)d_k_out | (uintptr_t)d_v_out) & 15)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "kv_read: outputs must be 16-byte aligned");
  // pieces are read and written in no order
  const size_t out_bytes = (size_t)v.kv_heads * count * v.hd * (out_dtype == ODI_CUDA_KV_OUT_F16 ? 2 : 4);
  const size_t cache_bytes = odi_cuda_kv_cache_bytes(v.dtype, v.kv_heads, v.hd, v.ctx);
  const auto clash = [](const void* a, size_t n, const void* b, size_t m) {
    return a && b && (uintptr_t)a < (uintptr_t)b + m && (uintptr_t)b < (uintptr_t)a + n;
  };
  for (const void* o : {d_k_out, d_v_out})
    if (clash(o, out_bytes, v.k, cache_bytes) || clash(o, out_bytes, v.v, cache_bytes))
      return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "kv_read: an output overlaps the cache");
  if (clash(d_k_out, out_bytes, d_v_out, out_bytes))
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "kv_read: the outputs overlap");
  const bool i8 = v.dtype == ODI_CUDA_KV_I8, o16 = out_dtype == ODI_CUDA_KV_OUT_F16;
  const int64_t pieces = (int64_t)count * (v.hd / (o16 ? 8 : 4));
  const dim3 grid((unsigned)((pieces + 256 * READ_U - 1) / (256 * READ_U)), v.kv_heads, 2);
  cudaStream_t s = (cudaStream_t)stream;
  const cudaError_t e = i8 ? (o16 ? launch_pdl(kv_read_kernel<true, true>, grid, dim3(256), s, v, start, count, d_k_out, d_v_out)
                                  : launch_pdl(kv_read_kernel<true, false>, grid, dim3(256), s, v, start, count, d_k_out, d_v_out))
                           : (o16 ? launch_pdl(kv_read_kernel<false, true>, grid, dim3(256), s, v, start, count, d_k_out, d_v_out)
                                  : launch_pdl(kv_read_kernel<false, false>, grid, dim3(256), s, v, start, count, d_k_out, d_v_out));
  return kv_launched(e, "kv_read");
}

int odi_cuda_kv_move(const odi_cuda_kv_cache* cache, const int32_t* d_src, const int32_t* d_dst, int n,
                     const odi_cuda_decode_state* d_state, void* stream) {
  KvView v;
  if (int rc = kv_view(cache, &v, "kv_move")) return rc;
  if (n < 0 || n > ODI_CUDA_KV_MOVE_MAX)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "kv_move: 0 to ODI_CUDA_KV_MOVE_MAX rows per call");
  if (!n) return ODI_CUDA_OK;
  if (!d_src || !d_dst) return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "kv_move: null argument");
  if (((uintptr_t)d_src | (uintptr_t)d_dst | (uintptr_t)d_state) & 3)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "kv_move: misaligned list");
  const int row_bytes = v.hd * (v.dtype == ODI_CUDA_KV_F16 ? 2 : 1);
  const cudaError_t e = launch_pdl(kv_move_kernel, dim3(row_bytes / 64, v.kv_heads, 2), dim3(256), (cudaStream_t)stream,
                                   v, d_src, d_dst, n, reinterpret_cast<const DecodeState*>(d_state));
  return kv_launched(e, "kv_move");
}

}  // extern "C"
