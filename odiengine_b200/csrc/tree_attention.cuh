// tree_attention.cuh -- what the two kernels of tree attention share: their
// arguments, which positions a node sees, and how the shares of the splits
// join.
#pragma once

#include "internal.h"
#include "kv_cache.cuh"

namespace odi_cuda {

constexpr int TA_SMS = 148;
constexpr float TA_NONE = -3.402823466e38f;  // reference of a row that has seen nothing

struct TreeArgs {
  const float* q;
  int64_t ld_q;
  float* out;
  KvView c;
  const unsigned* mask;
  int mask_words;
  const DecodeState* st;
  int tokens, heads, G, R, nsplit;
  unsigned inv_G;    // ceil(2^32 / G): r / G = r * inv_G >> 32 for the rows there are (G > 1)
  float scale_log2;  // scale * log2(e)
  int* count;   // arrivals per (kv head, row tile, cluster rank), zero between launches
  float* part;  // [kv head][tile][cluster][row][hd + 4]: reference, sum, -, -, accumulator
};


__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ uint32_t cluster_nranks() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
__device__ __forceinline__ uint32_t cluster_rank_of() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(n));
  return n;
}
// The barriers' .aligned forms (these, and bar.sync by its number) want whole
// warps, and their callers come from branches of some lanes.
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Rank k's copy of a shared-memory value.
__device__ __forceinline__ float4 peer_f4(const float4* p, int k) {
  uint32_t addr;
  float4 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(k));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 peer_f2(const float2* p, int k) {
  uint32_t addr;
  float2 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(k));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
// The node of row r.
__device__ __forceinline__ int row_node(const TreeArgs& a, int r) {
  return a.G == 1 ? r : (int)__umulhi((unsigned)r, a.inv_G);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126 .. 127
// What a q row of largest value am, brought to 1 .. 1.99, is multiplied by for three
// signed digits; rows past 1.99 * 2^126 can only be brought to 1.99 .. 4.
__device__ __forceinline__ float q_units(float am) { return am > 1.99f * 0x1p126f ? 1048576.f : 4194304.f; }
// scale * inv_unit * 2^ex, in the order that stays in fp32's normal range.
__device__ __forceinline__ float q_factor(float scale, float inv_unit, int ex) {
  return ex > 0 ? scale * pow2(ex) * inv_unit : scale * inv_unit * pow2(ex);
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// Which of positions p0 .. p0 + 31 node t sees (t < 0: a row past the last, none).
__device__ __forceinline__ unsigned seen_bits(const TreeArgs& a, int t, int p0, int pos, int len) {
  if (t < 0) return 0;
  const int words = a.mask_words, j0 = p0 - pos, w0 = j0 >> 5;
  auto word = [&](int w) -> unsigned {
    if (w < 0) return 0xffffffffu;  // below pos: seen by all
    if (w >= words) return 0;
    if (a.mask) return __ldcg(a.mask + (int64_t)t * words + w);
    const int n = t - 32 * w;  // a chain: bits 0 .. t
    return n >= 31 ? 0xffffffffu : n < 0 ? 0u : (2u << n) - 1u;
  };
  const unsigned bits = __funnelshift_r(word(w0), word(w0 + 1), (unsigned)(j0 & 31));
  return len <= p0 ? 0u : len - p0 < 32 ? bits & ((1u << (len - p0)) - 1u) : bits;
}

// Joins the shares of one row tile.  Each CTA's share: reference and sum of
// row n in cta_ml[n], its accumulator in fold[n * HD ..] (both in shared
// memory, not yet synchronised).  Rank k of the cluster takes rows k, k + C,
// ... from every rank's shared memory, in rank order; with several clusters
// the last to arrive joins their shares in cluster order.  Every order is
// fixed, so repeats are bit-identical.  The CTA's other threads meanwhile call
// tree_join_rest, which has the same barriers.
__device__ __forceinline__ void tree_join_rest(int C, int nclusters) {
  if (C > 1) cluster_barrier();
  else __syncthreads();
  if (C > 1) cluster_barrier();
  if (nclusters == 1) return;
  __syncthreads();
  __syncthreads();
}
template <int HD, int ROWS, int THREADS>
__device__ __forceinline__ void tree_join(const TreeArgs& a, int tid, const int* rowt, float2* cta_ml, float* fold, int rows,
                                          int C, int rank, int nclusters) {
  __shared__ int is_last;
  constexpr int V4 = HD / 4;
  float4* fold4 = reinterpret_cast<float4*>(fold);
  const int kvh = blockIdx.x, tile = blockIdx.y, split = blockIdx.z;
  const int64_t unit = (int64_t)kvh * gridDim.y + tile;
  auto add = [](float4& x, const float4& y, float f) {
    x.x = fmaf(y.x, f, x.x), x.y = fmaf(y.y, f, x.y), x.z = fmaf(y.z, f, x.z), x.w = fmaf(y.w, f, x.w);
  };
  auto store = [&](int n, int d4, float4 v, float L) {
    const int r = tile * ROWS + n, t = rowt[n];
    const float inv = L == 0.f ? 0.f : 1.f / L;
    float* out = a.out + ((int64_t)t * a.heads + kvh * a.G + (r - t * a.G)) * HD + d4 * 4;
    if (L == 0.f) v = make_float4(0.f, 0.f, 0.f, 0.f);
    v.x *= inv, v.y *= inv, v.z *= inv, v.w *= inv;
    if (((uintptr_t)out & 15) == 0) *reinterpret_cast<float4*>(out) = v;
    else out[0] = v.x, out[1] = v.y, out[2] = v.z, out[3] = v.w;
  };
  if (C > 1) cluster_barrier();
  else __syncthreads();
  const int mine = rows > rank ? (rows - rank + C - 1) / C : 0;
  constexpr int64_t PS = ROWS * (HD + 4);               // a cluster's share: [row][HD + 4]
  float* part = a.part + unit * (a.nsplit / C) * PS;
  for (int i = tid; i < mine * V4; i += THREADS) {
    const int n = rank + i / V4 * C, d4 = i % V4;
    float2 x[8];
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f), y[8];
    float M = TA_NONE, L = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < C) x[k] = peer_f2(&cta_ml[n], k), y[k] = peer_f4(&fold4[n * V4 + d4], k);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < C) M = fmaxf(M, x[k].x);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < C) {
        const float f = ex2(x[k].x - M);
        L += x[k].y * f;
        add(A, y[k], f);
      }
    if (nclusters == 1) {
      store(n, d4, A, L);
    } else {
      float* p = part + (split / C) * PS + n * (HD + 4);
      *reinterpret_cast<float4*>(p + 4 + d4 * 4) = A;
      if (d4 == 0) *reinterpret_cast<float2*>(p) = make_float2(M, L);
    }
  }
  if (C > 1) cluster_barrier();  // no rank leaves while another reads its memory
  if (nclusters == 1) return;
  __threadfence();
  __syncthreads();
  int* count = a.count + unit * 8 + rank;
  if (tid == 0) is_last = atomicAdd(count, 1) == nclusters - 1;
  __syncthreads();
  if (!is_last) return;
  __threadfence();
  for (int i = tid; i < mine * V4; i += THREADS) {  // the last of the clusters, for this rank's rows
    const int d4 = i % V4, n = rank + i / V4 * C;
    const float* p = part + n * (HD + 4);
    float M = TA_NONE, L = 0.f;
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = 0; k0 < nclusters; k0 += 8) {  // online, eight shares requested together
      float2 x[8];
      float4 y[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float* s = p + (k0 + u) * PS;
        const bool in = k0 + u < nclusters;
        x[u] = in ? __ldcg(reinterpret_cast<const float2*>(s)) : make_float2(TA_NONE, 0.f);
        y[u] = in ? __ldcg(reinterpret_cast<const float4*>(s + 4) + d4) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float top = M;
#pragma unroll
      for (int u = 0; u < 8; ++u) top = fmaxf(top, x[u].x);
      const float f0 = ex2(M - top);
      L *= f0, A.x *= f0, A.y *= f0, A.z *= f0, A.w *= f0;
      M = top;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float f = ex2(x[u].x - M);
        L += x[u].y * f;
        add(A, y[u], f);
      }
    }
    store(n, d4, A, L);
  }
  if (tid == 0) *count = 0;
}

// The tcgen05 kernel (tree_attention_tc.cu): 32 or 64 rows per CTA.
cudaError_t launch_tree_tc(const TreeArgs& a, int rows_per_cta, int tiles, int units, int64_t most, int* err, cudaStream_t s);

// How many clusters of each size a kernel can have resident, by device.
// Clusters live inside one GPC, so sizes differ: with one CTA per SM of 148,
// size 2 fills 148 of them, 4 132, 6 132, 7 105, 8 120.
struct TreeLaunch {
  bool attr_set[64] = {};
  int resident[64][9] = {};  // -1: asked and unknown
};

// Splits each unit's positions over as many CTAs as are resident at once, in
// clusters that join their shares in shared memory: the size that keeps the
// most CTAs busy, or a larger one that loses up to an eighth of them, since the
// clusters of one unit then join through global memory.  (A second wave costs
// as much as the first: 24 clusters of 6 where 22 fit took 41 us, not 21.)
template <typename Launch>
cudaError_t launch_tree_clusters(TreeLaunch& st, const void* kern, TreeArgs& a, int tiles, int units, int64_t room,
                                 int64_t most, int threads, int smem, cudaStream_t s, Launch&& launch) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!st.attr_set[dev]) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    st.attr_set[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  int cluster = 1;
  int64_t best = 1;
  for (int c = 1; c <= 8; ++c) {
    if (!st.resident[dev][c]) {
      cfg.gridDim = dim3(1, 1, c);
      cfg.numAttrs = 1;
      attr[0].val.clusterDim.z = c;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
      }
      st.resident[dev][c] = n > 0 ? n : -1;
    }
    int64_t fit = st.resident[dev][c];
    if (fit * c > room) fit = room / c;
    int64_t n = fit / units;
    if (n * c > most) n = most / c;
    if (n * c * 8 >= best * 7) cluster = c, best = n * c > best ? n * c : best;
    if (cluster == c) a.nsplit = (int)(n * c);
  }
  if (cluster == 1 && a.nsplit < 1) a.nsplit = 1;
  cfg.gridDim = dim3(a.c.kv_heads, tiles, a.nsplit);
  attr[0].val.clusterDim.z = cluster;
  cfg.numAttrs = 2;
  return launch(cfg);
}

}  // namespace odi_cuda
