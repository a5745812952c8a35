// tree_attention.cu -- attention of a tree of drafted tokens over a KV cache.
//
// Node t of T drafted nodes is stored in cache slot pos + t.  It sees every
// slot below pos and, of the T tree slots, those whose bit is set in its mask
// row (its ancestors and itself; without a mask, nodes 0..t):
//   s_tj = scale * q_t . k_j,   m_t = max over visible j of s_tj
//   o_t  = sum_j exp(s_tj - m_t) v_j / sum_j exp(s_tj - m_t)
// A node that sees nothing gets zeros.  Slots outside the cache are not seen.
#include <math.h>

#include "../../include/odi_cuda.h"
#include "internal.h"
#include "kv_cache.cuh"
#include "pdl_launch.cuh"

namespace odi_cuda {
namespace {

constexpr int TA_BLOCK = 128;  // cache positions per step
constexpr int TA_SMS = 148;

struct TreeArgs {
  const float* q;
  int64_t ld_q;
  float* out;
  KvView c;
  const unsigned* mask;
  int mask_words;
  const DecodeState* st;
  int tokens, heads, nsplit;
  float scale;
  int* count;   // arrivals per (token, head), zero between launches
  float* part;  // [token][head][split][hd + 2]: running max, sum, accumulator
};

__device__ __forceinline__ float kv_value(const KvView& c, const void* base, int64_t row, int d) {
  if (c.dtype == ODI_CUDA_KV_F16) return __half2float(static_cast<const __half*>(base)[row * c.hd + d]);
  return (float)static_cast<const int8_t*>(base)[row * c.hd + d] *
         reinterpret_cast<const float*>(static_cast<const uint8_t*>(base) + c.scale_off)[row];
}

// One CTA per (head, token, split); a lane scores one position, a warp 32.
template <int HD>
__global__ void __launch_bounds__(128) tree_attn_kernel(const TreeArgs a) {
  __shared__ float qs[HD], fold[4][HD + 2];
  __shared__ int is_last;
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.x, t = blockIdx.y, split = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = h / (a.heads / a.c.kv_heads);
  const int pos = a.st->pos;
  const int64_t len = max((int64_t)0, min((int64_t)a.c.ctx, (int64_t)pos + a.tokens));
  for (int d = threadIdx.x; d < HD; d += 128) qs[d] = a.q[t * a.ld_q + (int64_t)h * HD + d] * a.scale;
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc[HD / 32];
  for (int e = 0; e < HD / 32; ++e) acc[e] = 0.f;
  for (int64_t p0 = (int64_t)split * TA_BLOCK; p0 < len; p0 += (int64_t)a.nsplit * TA_BLOCK) {
    const int64_t p = p0 + warp * 32 + lane;
    bool vis = p < len;
    if (vis && p >= pos) {
      const int j = (int)(p - pos);
      vis = a.mask ? (a.mask[(int64_t)t * a.mask_words + (j >> 5)] >> (j & 31)) & 1u : j <= t;
    }
    float s = -INFINITY;
    const int64_t row = (int64_t)kvh * a.c.ctx + p;
    if (vis) {
      s = 0.f;
      for (int d = 0; d < HD; ++d) s = fmaf(qs[d], kv_value(a.c, a.c.k, row, d), s);
    }
    const unsigned seen = __ballot_sync(0xffffffffu, vis);
    if (!seen) continue;
    float mx = s;
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float mn = fmaxf(m, mx);
    const float corr = m == -INFINITY ? 0.f : expf(m - mn);
    const float pv = vis ? expf(s - mn) : 0.f;
    float ps = pv;
    for (int o = 16; o; o >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
    l = l * corr + ps;
    for (int e = 0; e < HD / 32; ++e) acc[e] *= corr;
    for (int i = 0; i < 32; ++i) {
      const float pi = __shfl_sync(0xffffffffu, pv, i);
      if (!((seen >> i) & 1u)) continue;  // a position that is not seen is not read
      for (int e = 0; e < HD / 32; ++e)
        acc[e] = fmaf(pi, kv_value(a.c, a.c.v, row - lane + i, lane + 32 * e), acc[e]);
    }
    m = mn;
  }
  if (lane == 0) fold[warp][0] = m, fold[warp][1] = l;
  for (int e = 0; e < HD / 32; ++e) fold[warp][2 + lane + 32 * e] = acc[e];
  __syncthreads();
  const int64_t unit = (int64_t)t * a.heads + h;
  float* part = a.part + unit * a.nsplit * (HD + 2);
  auto merge = [&](const float* p, int n, int64_t stride, int d, float* M, float* L) {
    float mm = -INFINITY, ll = 0.f, aa = 0.f;
    for (int i = 0; i < n; ++i) {
      const float mi = __ldcg(p + i * stride);
      if (mi == -INFINITY) continue;
      const float mn = fmaxf(mm, mi), fo = expf(mm - mn), fn = expf(mi - mn);
      ll = ll * fo + p[i * stride + 1] * fn;
      aa = aa * fo + p[i * stride + 2 + d] * fn;
      mm = mn;
    }
    *M = mm, *L = ll;
    return aa;
  };
  for (int d = threadIdx.x; d < HD; d += 128) {
    float mm = -INFINITY, ll = 0.f, aa = 0.f;
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, fold[w][0]);
    for (int w = 0; w < 4; ++w)
      if (fold[w][0] != -INFINITY) {
        const float f = expf(fold[w][0] - mm);
        ll += fold[w][1] * f, aa += fold[w][2 + d] * f;
      }
    float* o = part + split * (HD + 2);
    o[2 + d] = aa;
    if (d == 0) o[0] = mm, o[1] = ll;
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) is_last = atomicAdd(&a.count[unit], 1) == a.nsplit - 1;
  __syncthreads();
  if (!is_last) return;
  __threadfence();
  for (int d = threadIdx.x; d < HD; d += 128) {
    float mm, ll;
    const float aa = merge(part, a.nsplit, HD + 2, d, &mm, &ll);
    a.out[unit * HD + d] = mm == -INFINITY ? 0.f : aa / ll;
  }
  if (threadIdx.x == 0) a.count[unit] = 0;
}

struct TreePlan {
  int nsplit;
  size_t part_off, bytes;
};

TreePlan tree_plan(int tokens, int heads, int kv_heads, int hd, int ctx) {
  TreePlan p;
  const int64_t units = (int64_t)tokens * heads;
  const int64_t blocks = ((int64_t)ctx + TA_BLOCK - 1) / TA_BLOCK;
  int64_t want = TA_SMS * 8 / units;
  want = want < 1 ? 1 : want > 64 ? 64 : want;
  p.nsplit = (int)(want > blocks ? blocks : want);
  p.part_off = (16 + (size_t)units * 4 + 255) / 256 * 256;
  p.bytes = p.part_off + (size_t)units * p.nsplit * (hd + 2) * 4;
  return p;
}

bool tree_shape_ok(int tokens, int heads, int kv_heads, int hd, int ctx) {
  return tokens >= 1 && tokens <= ODI_CUDA_TREE_MAX && heads >= 1 && heads <= 1024 && kv_heads >= 1 &&
         heads % kv_heads == 0 && (hd == 64 || hd == 128) && ctx >= 1;
}

}  // namespace
}  // namespace odi_cuda

using namespace odi_cuda;

extern "C" {

size_t odi_cuda_attention_tree_scratch_bytes(int tokens, int heads, int kv_heads, int head_dim, int ctx) {
  if (!tree_shape_ok(tokens, heads, kv_heads, head_dim, ctx)) return 0;
  return tree_plan(tokens, heads, kv_heads, head_dim, ctx).bytes;
}

int odi_cuda_attention_tree(const float* d_q, int64_t ld_q, const odi_cuda_kv_cache* cache, float* d_out,
                            const uint32_t* d_mask, const odi_cuda_decode_state* d_state, int tokens, int heads,
                            float scale, void* d_scratch, size_t scratch_bytes, void* stream) {
  KvView v;
  if (int rc = kv_view(cache, &v, "attention_tree")) return rc;
  auto bad = [](const char* m) { return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, m); };
  if (!d_q || !d_out || !d_state || !d_scratch) return bad("attention_tree: null argument");
  if (!tree_shape_ok(tokens, heads, v.kv_heads, v.hd, v.ctx))
    return bad("attention_tree: 1 to ODI_CUDA_TREE_MAX tokens, heads (at most 1024) a multiple of kv_heads");
  if (ld_q < (int64_t)heads * v.hd) return bad("attention_tree: the query stride is shorter than its row");
  if (!isfinite(scale)) return bad("attention_tree: the scale must be finite");
  if (((uintptr_t)d_q | (uintptr_t)d_out | (uintptr_t)d_mask) & 3 || ((uintptr_t)d_scratch & 15))
    return bad("attention_tree: misaligned buffer");
  const TreePlan p = tree_plan(tokens, heads, v.kv_heads, v.hd, v.ctx);
  if (scratch_bytes < p.bytes) return bad("attention_tree: scratch too small");
  TreeArgs a{};
  a.q = d_q, a.ld_q = ld_q, a.out = d_out, a.c = v, a.mask = d_mask, a.mask_words = (tokens + 31) / 32;
  a.st = reinterpret_cast<const DecodeState*>(d_state);
  a.tokens = tokens, a.heads = heads, a.nsplit = p.nsplit, a.scale = scale;
  a.count = reinterpret_cast<int*>(static_cast<uint8_t*>(d_scratch) + 16);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(d_scratch) + p.part_off);
  const dim3 grid(heads, tokens, p.nsplit);
  const cudaError_t e = v.hd == 128 ? launch_pdl(tree_attn_kernel<128>, grid, dim3(128), (cudaStream_t)stream, a)
                                    : launch_pdl(tree_attn_kernel<64>, grid, dim3(128), (cudaStream_t)stream, a);
  return kv_launched(e, "attention_tree");
}

}  // extern "C"
