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

#include <atomic>

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
  const int* header;  // the batch's work words
  int max_items;
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

// A piece of a unit, as the producer warp hands it on in shared memory.
struct PagedPiece {
  PagedItem it;  // tile0, tiles: the unit's, of all (kv head, item) units' tiles
  int kvh, unit;
  int t0, t1;    // this CTA's tiles of the unit
  int rows;      // of the item, that there are rows of q for
  int least;     // positions below it are seen by every row of the item
  int poison;    // V has values that are not finite where not every row looks
  int last;      // no piece: the run is over
};
// The share of tiles that a CTA takes.
struct PagedRun {
  int64_t x, end, share;
  int items, tiles;
  int kvh, item;
  PagedItem it;  // of `item`
};
struct PagedFound {
  PagedItem it;
  int item;
};
__device__ __forceinline__ PagedItem load_item(const PagedItem* p) {
  const int4 u = __ldcg(reinterpret_cast<const int4*>(p)), v = __ldcg(reinterpret_cast<const int4*>(p) + 1);
  return {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
}
// The first unit of this CTA's run; false (in all threads, before any barrier) if
// there is none.  The list's first items are read along with its length: one round
// trip where the item is among them.
__device__ __forceinline__ bool run_begin(const PagedAttnArgs& a, PagedRun& r, PagedFound* found) {
  const PagedItem* list = paged_items(a.header);
  int i = threadIdx.x;
  PagedItem x{};
  const int2 head = __ldcg(reinterpret_cast<const int2*>(a.header) + PW_ITEMS / 2);
  static_assert(PW_ITEMS == 2 && PW_TILES == 3, "one load");
  if (i < a.max_items) x = load_item(list + i);
  r.items = head.x, r.tiles = head.y;
  const int64_t all = (int64_t)r.tiles * a.c.kv_heads;
  r.share = max((all + gridDim.x - 1) / gridDim.x, (int64_t)a.least);
  r.x = r.share * blockIdx.x;
  r.end = min(all, r.x + r.share);
  if (r.x >= all) return false;
  r.kvh = (int)(r.x / r.tiles);
  const int rem = (int)(r.x - (int64_t)r.kvh * r.tiles);
  while (i < r.items) {
    if (x.tile0 <= rem && rem < x.tile0 + x.tiles) found->it = x, found->item = i;
    i += blockDim.x;
    if (i < r.items) x = load_item(list + i);
  }
  __syncthreads();
  r.it = found->it, r.item = found->item;
  return true;
}
// The piece at x, and x moved past it.
__device__ __forceinline__ PagedPiece run_piece(const PagedAttnArgs& a, PagedRun& r, int rows_per_item) {
  PagedPiece p;
  p.it = r.it;
  p.kvh = r.kvh, p.unit = r.kvh * r.items + r.item;
  p.t0 = (int)(r.x - (int64_t)r.kvh * r.tiles) - r.it.tile0;
  p.t1 = (int)min((int64_t)r.it.tiles, p.t0 + (r.end - r.x));
  p.rows = min(rows_per_item, min(r.it.len - r.it.past, a.out_rows - r.it.start) * a.G - r.it.i * rows_per_item);
  p.least = paged_limit(r.it.past, pa_token(a, r.it.i * rows_per_item), r.it.len, r.it.prefix);
  p.poison = p.last = 0;
  r.x += max(1, p.t1 - p.t0);
  return p;
}
__device__ __forceinline__ void run_next(const PagedAttnArgs& a, PagedRun& r) {
  if (++r.item == r.items) r.item = 0, ++r.kvh;
  r.it = load_item(paged_items(a.header) + r.item);
}
// Where a unit's pieces are: CTA c's first tile is c * share; what begins the unit
// is the CTA's second place, what goes on with one its first.
__device__ __forceinline__ int64_t unit_tile(const PagedRun& r, const PagedPiece& p) {
  return (int64_t)p.kvh * r.tiles + p.it.tile0;
}
__device__ __forceinline__ float* piece_part(const PagedAttnArgs& a, const PagedRun& r, int64_t cta, int64_t ux, int stride) {
  return a.part + (2 * cta + (r.share * cta <= ux ? 1 : 0)) * stride;
}

// Devices whose kernel may take its shared memory; set again by whoever comes twice
// at once, which changes nothing.
struct PagedReady {
  std::atomic<uint64_t> devices{0};
  cudaError_t set(const void* kern, int smem) {
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return e;
    if (dev < 64 && devices.load(std::memory_order_acquire) >> dev & 1) return cudaSuccess;
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return e;
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared))
      return e;
    if (dev < 64) devices.fetch_or(1ull << dev, std::memory_order_release);
    return cudaSuccess;
  }
};

cudaError_t paged_maps(const PagedView& c, int tile, CUtensorMap* maps);
cudaError_t launch_paged_mma(PagedAttnArgs& a, int groups, bool fancy, cudaStream_t s);
cudaError_t launch_paged_tc(PagedAttnArgs& a, bool fancy, cudaStream_t s);

constexpr int PAGED_SMS = 148, PAGED_ROWS_MAX = 256;
// CTAs of a call: two per SM of the narrow kernel, else one
constexpr int paged_ctas(int rows) { return rows <= 16 ? 2 * PAGED_SMS : PAGED_SMS; }

}  // namespace odi_cuda
