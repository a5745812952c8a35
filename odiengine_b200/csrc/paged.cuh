// paged.cuh -- several requests over a paged KV cache: what the kernels of
// paged_step.cu, paged_append.cu and paged_attention*.cu share.
//
// A layer's K and V are [num_pages][kv_heads][page_size][head_dim]: one page of
// one kv head is one contiguous run of rows, the shape that the decode step's
// cache has for a whole context, so a box of a tensor map is (part of) a page.
// One block table serves all layers.
#pragma once

#include <cuda_bf16.h>

#include "../../include/odi_cuda.h"
#include "common.cuh"

namespace odi_cuda {

struct PagedView {
  void* k;
  void* v;
  int dtype;  // ODI_CUDA_PAGED_F16 / ODI_CUDA_PAGED_BF16
  int kv_heads, hd, page_size, num_pages;
  int page_shift;
  int64_t bytes() const { return 2ll * num_pages * kv_heads * page_size * hd; }  // of k, and of v
};

// How attention cuts a batch's rows: an item is up to `rows` of the new tokens *
// G rows of one request (row r: token r / G, head r % G of each kv head's
// group), over tiles of `tile` positions.  `extra`: what beginning and ending an item
// costs, in tiles.
struct PagedGeometry {
  int G, rows, tile, extra;
  int64_t max_items;
};

// Words of odi_cuda_paged_batch.work.
constexpr int PW_STATUS = 0, PW_ITEMS = 2, PW_TILES = 3, PW_HEADER = 16;
struct alignas(16) PagedItem {
  int b, i;              // request, item within the request
  int start, past, len;  // its first row; positions before its new ones; all of them
  int prefix;
  int tile0, tiles;      // tiles, and extra ones, of the items before; its own tiles
};
static_assert(sizeof(PagedItem) == 32, "two 16-byte loads");
// PW_ITEMS of them.
inline __host__ __device__ const PagedItem* paged_items(const int* work) {
  return reinterpret_cast<const PagedItem*>(work + PW_HEADER);
}

// Checks of a caller's descriptors; `who` opens the error message.
int paged_view(const odi_cuda_paged_cache* c, PagedView* v, const char* who);
int paged_batch_ok(const odi_cuda_paged_batch* b, PagedGeometry* g, const char* who);
bool paged_geometry(int requests, int max_rows, int max_new, int heads, int kv_heads, PagedGeometry* g);

inline bool page_size_ok(int p) { return p == 16 || p == 32 || p == 64 || p == 128; }
inline int page_shift_of(int p) { return p == 16 ? 4 : p == 32 ? 5 : p == 64 ? 6 : 7; }
// Rows of an item and positions of a tile, by the most rows a request has per kv
// head: the two widths of the mma.sync kernel, and the two of the tcgen05 kernel.
// What an item costs beside its tiles, measured as tiles.  tcgen05: 2048 tokens of
// 64/8 heads alone 93 us with 4, 134 with 0 (a run of short items was 14 of them),
// 105 with 2, 93 with 5; seven prompts of 32/32 heads of 64 dims 91, 87, 88, 91.
// mma.sync: 256 requests of one token over 10 to 600 positions 72.5 us with 2, 75.5
// with 0, 71.5 with 4; 16 requests of 2 to 5 tokens 58.5, 58.5, 60.5.
inline void paged_kind(int64_t most, int* rows, int* tile, int* extra) {
  *rows = most <= 16 ? 16 : most <= 32 ? 32 : most <= 128 ? 128 : 256;
  *tile = 64;
  *extra = *rows <= 32 ? 2 : 4;
}

// Positions of the batch that row r of request b sees: those below the result.
__device__ __forceinline__ int paged_limit(int first, int token, int len, int prefix) {
  return min(len, max(first + token + 1, prefix));
}

}  // namespace odi_cuda
