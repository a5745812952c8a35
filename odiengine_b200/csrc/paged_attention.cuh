// paged_attention.cuh -- what the two kernels of attention over a paged cache
// share: their arguments, how the work is dealt out, and the tensor maps.
//
// The work of a call is the tiles of all (kv head, item) units in a row:
// kv_heads times the batch's list of items.  CTA c takes the share-long run of
// them from c * share on, whatever units it cuts, so that every CTA has the same
// number of tiles however the requests' lengths lie; an item counts for some more than
// it has, for what its beginning and its end cost.  A unit inside one run is
// finished there; the pieces of one that is cut go to the scratch, and the last
// CTA to arrive joins them in the order of the positions; many pieces first in groups,
// so that no CTA joins more than a few.  Which pieces there are depends on the lengths
// alone, so repeats are bit-identical.
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
  float scale_log2;  // scale * log2(e); with a cap 2 scale / cap * log2(e)
  float cap_log2;    // cap * log2(e), or 0
  const float* slopes;
  int vec, vec_out;  // q, out and their strides allow 16-byte accesses
  int q_boxes;       // Q comes by TMA
  int least;         // tiles per CTA at least
  int extra;         // tiles that an item counts beside its own
  float* part;       // [2 * CTAs][rows][HD + 2]
  int* count;        // arrivals per unit, zero between launches
  int* group;        // arrivals per group of pieces, by its first piece's place
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
// cap * tanh(x), x as 2 x log2(e): cap * (1 - 2 / (e^2x + 1)), to about 2^-23 of the cap.
__device__ __forceinline__ float pa_cap(float x, float cap) { return fmaf(-2.f * cap, pa_rcp(pa_ex2(x) + 1.f), cap); }
__device__ __forceinline__ int pa_token(const PagedAttnArgs& a, int r) {
  return a.G == 1 ? r : (int)__umulhi((unsigned)r, a.inv_G);
}

// log2 of what a weight may reach before the reference moves, and how far below the
// largest score the reference stands when it has moved.  fp16 ends at 2^16 and its steps
// at 2^-24: with the reference 7 lower, weights are up to 2^15, the largest of a row is 2^7
// at least, and one of 2^-21 of that has its 11 bits (2^-14 without), one of 2^-31 some.
constexpr float PAGED_MOVE = 8.f;

template <typename T>
struct Half16;
template <>
struct Half16<__half> {
  static constexpr float BELOW = 7.f;
  static constexpr uint32_t EXP = 0x7c00u;
  static constexpr bool BF = false;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float up(uint16_t x) { return __half2float(__ushort_as_half(x)); }
  // Two weights as a sum of two parts each, to 2^-19 of them (or 2^-23).  The first
  // is cut off, not rounded, and the last bit of the second (2^-20 of the weight at most, or
  // 2^-24, beside half as much for its rounding) is set where the first is not 0: neither
  // is negative, and no part of a weight is 0, or an infinity of V's would become a NaN.
  static constexpr float PARTS = 1.f;  // what the parts' sum is of the weight
  static __device__ __forceinline__ uint32_t split(float2 x, uint32_t& rest) {
    uint32_t y;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(x.y), "f"(x.x));
    const __half2 h = *reinterpret_cast<const __half2*>(&y);
    const float2 r = __ffma2_rn(__half22float2(h), make_float2(-1.f, -1.f), x);
    rest = pack(r.x, r.y) | (__hne2_mask(h, __half2half2(__ushort_as_half(0))) & 0x00010001u);
    return y;
  }
  // Pairs: 0 * x + y, NaN where x is not finite.
  static __device__ __forceinline__ uint32_t times0(uint32_t x, uint32_t y) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0)), *reinterpret_cast<const __half2*>(&y));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};
template <>
struct Half16<__nv_bfloat16> {
  static constexpr float BELOW = 0.f;
  static constexpr uint32_t EXP = 0x7f80u;
  static constexpr bool BF = true;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float up(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
  // To 2^-16 of them; the second part is not 0 because the sum is a little more than the weight.
  static constexpr float PARTS = 1.f + 0x1p-17f;
  static __device__ __forceinline__ uint32_t split(float2 x, uint32_t& rest) {
    uint32_t y;
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(x.y), "f"(x.x));
    const float2 r = __ffma2_rn(x, make_float2(PARTS, PARTS), make_float2(-__uint_as_float(y << 16), -__uint_as_float(y & 0xffff0000u)));
    rest = pack(r.x, r.y);
    return y;
  }
  static __device__ __forceinline__ uint32_t times0(uint32_t x, uint32_t y) {
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x), __bfloat162bfloat162(__ushort_as_bfloat16(0)),
                                     *reinterpret_cast<const __nv_bfloat162*>(&y));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};

__device__ __forceinline__ void pa_tma(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void pa_tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// A piece of a unit, as the producer warp hands it on in shared memory.
struct PagedPiece {
  PagedItem it;  // tile0, tiles: the unit's, of all (kv head, item) units' tiles
  int kvh, unit;
  int t0, t1;    // this CTA's tiles of the unit
  int c0, c1;    // the first and last CTA that have tiles of it
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
// a / b, both below 2^32 but for calls of absurd size.
__device__ __forceinline__ int64_t pa_div(int64_t a, int64_t b) {
  return (a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}
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
  r.share = max(pa_div(all + gridDim.x - 1, gridDim.x), (int64_t)a.least);
  r.x = r.share * blockIdx.x;
  r.end = min(all, r.x + r.share);
  if (r.x >= all) return false;
  r.kvh = (int)pa_div(r.x, r.tiles);
  const int rem = (int)(r.x - (int64_t)r.kvh * r.tiles);
  while (i < r.items) {
    if (x.tile0 <= rem && rem < x.tile0 + x.tiles + a.extra) found->it = x, found->item = i;
    i += blockDim.x;
    if (i < r.items) x = load_item(list + i);
  }
  __syncthreads();
  r.it = found->it, r.item = found->item;
  return true;
}
// The piece at x, and x moved past it.  An item's extra tiles come before its own; a
// run that ends among them has no piece of it (t1 <= t0), and no piece after it.
__device__ __forceinline__ PagedPiece run_piece(const PagedAttnArgs& a, PagedRun& r, int rows_per_item) {
  PagedPiece p;
  p.it = r.it;
  p.kvh = r.kvh, p.unit = r.kvh * r.items + r.item;
  const int64_t ux = (int64_t)r.kvh * r.tiles + r.it.tile0 + a.extra;  // the unit's first tile
  const int64_t next = min(r.end, ux + r.it.tiles);
  p.t0 = (int)max((int64_t)0, r.x - ux);
  p.t1 = (int)(next - ux);
  p.rows = min(rows_per_item, min(r.it.len - r.it.past, a.out_rows - r.it.start) * a.G - r.it.i * rows_per_item);
  p.least = paged_limit(r.it.past, pa_token(a, r.it.i * rows_per_item), r.it.len, r.it.prefix);
  p.poison = p.last = 0;
  p.c0 = p.c1 = blockIdx.x;
  if (p.t0 || p.t1 < r.it.tiles) p.c0 = (int)pa_div(ux, r.share), p.c1 = (int)pa_div(ux + r.it.tiles - 1, r.share);
  r.x = max(r.x + 1, next);
  return p;
}
__device__ __forceinline__ void run_next(const PagedAttnArgs& a, PagedRun& r) {
  if (++r.item == r.items) r.item = 0, ++r.kvh;
  r.it = load_item(paged_items(a.header) + r.item);
}
// The pages of a piece for the producer warp: 32 entries of the table in the warp's
// registers and the next 32 on their way, so that no tile waits for its names (a load
// per tile, even one tile ahead, held a CTA to a tile per round trip: 0.95 us).
struct PagedNames {
  const int* row;
  int step;  // of the blocks: 1, or -1 from the last tile to the first
  int last, block, cur, next;  // entries there are; the 32 at hand
  __device__ __forceinline__ PagedNames(const PagedAttnArgs& a, const PagedPiece& p, int tile, bool down)
      : row(a.table + (int64_t)p.it.b * a.max_pages), step(down ? -1 : 1) {
    // a list made with wider tables than these names pages that they do not have
    last = min((min(p.it.len, p.t1 * tile) + a.c.page_size - 1) >> a.c.page_shift, a.max_pages);
    block = ((down ? p.t1 - 1 : p.t0) * tile >> a.c.page_shift) >> 5;
    cur = load(block), next = load(block + step);
  }
  __device__ __forceinline__ int load(int b) const {
    const int i = b * 32 + (threadIdx.x & 31);
    return i >= 0 && i < last ? __ldcg(row + i) : -1;
  }
  // Entry i, the whole warp asking for entries of one block of 32, at or next to the last's.
  __device__ __forceinline__ int at(int i) {
    const int b = __shfl_sync(0xffffffffu, i, 0) >> 5;
    if (b != block) block = b, cur = next, next = load(b + step);
    return __shfl_sync(0xffffffffu, cur, i & 31);
  }
};
// Where CTA c's piece of the unit is.  A CTA has two places: one for the piece that
// goes on with a unit, one for the piece that begins one, which only c0's can be.
__device__ __forceinline__ float* piece_part(const PagedAttnArgs& a, const PagedPiece& p, int cta, int stride) {
  return a.part + (int64_t)(2 * cta + (cta == p.c0)) * stride;
}

// How a unit's pieces are joined: `n` of them from CTA `first` on, `step` apart, who
// arrive at `counter`; when they are one, the unit is done or its groups are next.
struct PagedJoin {
  int first, step, n;
  int* counter;
  bool final;
};
// Up to `at_once` pieces are joined at once, more of them in groups of about the root
// of their number: 38 pieces of one token of 64/8 heads over 30,000 positions take 36 us
// so, 41 at once; of 16 tokens 55 and 85.
__device__ __forceinline__ PagedJoin join_first(const PagedAttnArgs& a, const PagedPiece& p, int at_once) {
  const int n = p.c1 - p.c0 + 1;
  if (n <= at_once) return {p.c0, 1, n, a.count + p.unit, true};
  const int size = (int)ceilf(sqrtf((float)n)), first = p.c0 + ((int)blockIdx.x - p.c0) / size * size;
  return {first, 1, min(size, p.c1 - first + 1), a.group + 2 * first + (first == p.c0), false};
}
__device__ __forceinline__ PagedJoin join_next(const PagedAttnArgs& a, const PagedPiece& p) {
  const int n = p.c1 - p.c0 + 1, size = (int)ceilf(sqrtf((float)n));
  return {p.c0, size, (n + size - 1) / size, a.count + p.unit, true};
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

cudaError_t paged_maps(const PagedView& c, int tile, bool planes, CUtensorMap* maps);
cudaError_t paged_q_map(const PagedAttnArgs& a, int tokens, CUtensorMap* map);
cudaError_t launch_paged_mma(PagedAttnArgs& a, int groups, bool fancy, cudaStream_t s);
cudaError_t launch_paged_tc(PagedAttnArgs& a, int rows, cudaStream_t s);

constexpr int PAGED_SMS = 148, PAGED_ROWS_MAX = 256;
// CTAs of a call: two per SM of the kernels' narrow forms, else one
constexpr int paged_ctas(int rows) { return rows == 16 || rows == 128 ? 2 * PAGED_SMS : PAGED_SMS; }

}  // namespace odi_cuda
