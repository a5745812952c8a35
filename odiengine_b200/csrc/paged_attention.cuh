// paged_attention.cuh -- what the two kernels of attention over a paged cache
// share: their arguments, how the work is dealt out, and the tensor maps.
//
// The work of a call is the tiles of all (kv head, item) units in a row:
// kv_heads times the batch's list of items.  CTA c takes the share-long run of
// them from c * share on, whatever units it cuts, so that every CTA has the same
// number of tiles however the requests' lengths lie.  A unit inside one run is
// finished there; the pieces of one that is cut go to the scratch, and the last
// CTA to arrive joins them in the order of the positions.  Which pieces there are
// depends on the lengths alone, so repeats are bit-identical.
#pragma once

#include <cuda.h>
#include <math.h>

#include "internal.h"
#include "kv_cache.cuh"
#include "paged.cuh"

namespace odi_cuda {

struct PagedAttnArgs {
  const void* q;
  int64_t ld_q;
  void* out;
  int64_t ld_out;
  int out32;  // out is fp32, not of the cache's type
  PagedView c;
  const int* table;
  int max_pages;
  const int *starts, *lens, *header;
  PagedWork w;
  int G, out_rows;
  unsigned inv_G;    // ceil(2^32 / G): r / G = r * inv_G >> 32 (G > 1)
  float scale_log2;  // scale * log2(e), or scale / cap where there is a cap
  float cap_log2;    // cap * log2(e), or 0
  const float* slopes;
  int vec, vec_out;  // q, out and their strides allow 16-byte accesses
  int least;         // tiles per CTA at least
  float* part;       // [2 * CTAs][rows][HD + 2]
  int* count;        // arrivals per unit, zero between launches
  int* err;
};

constexpr int ERR_PAGED_WAIT = 128, ERR_PAGED_PAGE = 256;

__device__ __forceinline__ float pa_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pa_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh(x) = 1 - 2 / (e^2x + 1): to about 2^-23 of 1, which the cap then scales.
__device__ __forceinline__ float pa_tanh(float x) {
  return fmaf(-2.f, pa_rcp(pa_ex2(x * 2.885390081777927f) + 1.f), 1.f);
}
__device__ __forceinline__ int pa_token(const PagedAttnArgs& a, int r) {
  return a.G == 1 ? r : (int)__umulhi((unsigned)r, a.inv_G);
}

template <typename T>
struct Half16;
template <>
struct Half16<__half> {
  static constexpr uint32_t EXP = 0x7c00u;
  static constexpr bool BF = false;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float up(uint16_t x) { return __half2float(__ushort_as_half(x)); }
};
template <>
struct Half16<__nv_bfloat16> {
  static constexpr uint32_t EXP = 0x7f80u;
  static constexpr bool BF = true;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float up(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
};

__device__ __forceinline__ void pa_tma(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

// A run of tiles, piece by piece.
struct PagedPiece {
  int kvh, item, b, i;  // kv head; item of the batch, its request and place there
  int t0, t1, tn;       // this CTA's tiles of the unit, and all of them
};
struct PagedRun {
  int64_t x, end, share;
  int items, tiles;
  PagedPiece p;
};
// The first unit of the run [x, end): all threads of the CTA, `slot` in shared memory.
__device__ __forceinline__ bool run_begin(const PagedAttnArgs& a, PagedRun& r, int* slot) {
  r.items = __ldcg(a.header + PW_ITEMS);
  r.tiles = __ldcg(a.header + PW_TILES);
  const int64_t all = (int64_t)r.tiles * a.c.kv_heads;
  r.share = max((all + gridDim.x - 1) / gridDim.x, (int64_t)a.least);
  r.x = r.share * blockIdx.x;
  r.end = min(all, r.x + r.share);
  if (r.x >= all) return false;
  r.p.kvh = (int)(r.x / r.tiles);
  const int rem = (int)(r.x - (int64_t)r.p.kvh * r.tiles);
  for (int i = threadIdx.x; i < r.items; i += blockDim.x)
    if (__ldcg(a.w.cum + i) <= rem && rem < __ldcg(a.w.cum + i + 1)) *slot = i;
  __syncthreads();
  r.p.item = *slot;
  return true;
}
// The piece at x, and x moved past it.
__device__ __forceinline__ void run_piece(const PagedAttnArgs& a, PagedRun& r) {
  const int c0 = __ldcg(a.w.cum + r.p.item), c1 = __ldcg(a.w.cum + r.p.item + 1);
  const int2 info = __ldcg(a.w.info + r.p.item);
  r.p.b = info.x, r.p.i = info.y;
  r.p.tn = c1 - c0;
  r.p.t0 = (int)(r.x - (int64_t)r.p.kvh * r.tiles) - c0;
  r.p.t1 = (int)min((int64_t)r.p.tn, r.p.t0 + (r.end - r.x));
  r.x += max(1, r.p.t1 - r.p.t0);
}
__device__ __forceinline__ void run_next(PagedRun& r) {
  if (++r.p.item == r.items) r.p.item = 0, ++r.p.kvh;
}

cudaError_t paged_maps(const PagedView& c, int tile, CUtensorMap* maps);
cudaError_t launch_paged_mma(PagedAttnArgs& a, int mt, bool fancy, cudaStream_t s);
cudaError_t launch_paged_tc(PagedAttnArgs& a, bool fancy, cudaStream_t s);

constexpr int PAGED_SMS = 148, PAGED_ROWS_MAX = 256;
constexpr int paged_ctas(int rows) { return rows <= 32 ? 2 * PAGED_SMS : PAGED_SMS; }

}  // namespace odi_cuda
