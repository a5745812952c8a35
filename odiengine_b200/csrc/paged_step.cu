// paged_step.cu -- block tables, slots and attention's work list of one step,
// from the requests' lengths.
//
// Request b keeps keep_b of its positions and takes new_b more.  With P
// positions per page, its pages ceil(keep / P) .. ceil(len / P) - 1 are dropped
// and pages ceil(keep / P) .. ceil((keep + new) / P) - 1 taken.  The free list is
// a stack: all drops go on it before any page is taken, in the order that gives
// the first page dropped back first.  Who gets which page follows from exclusive
// sums over the requests, so a step is the same whatever order the blocks run in.
//
// One CTA for short lists.  Else a cluster: every CTA sums the requests' counts for
// itself (the lists are short), then they share out the requests' pages and the
// step's rows.  One barrier stands between drops and takes; a row on a page that this
// step takes reads the free list, as the table's writer does, so that rows need not
// wait for the table.  Bound by latency: three round trips to memory (lists, dropped
// entries, taken pages) and four sums over the block: 8 requests 3.8 us, 512 requests
// with 16,000 rows 9.0 us.
#include <cstdio>

#include "internal.h"
#include "kv_cache.cuh"
#include "paged.cuh"
#include "pdl_launch.cuh"

namespace odi_cuda {
namespace {

constexpr int MAX_B = ODI_CUDA_PAGED_MAX_REQUESTS;
// what keeps a request from getting its rows
constexpr int REFUSED = ODI_CUDA_PAGED_BAD_NEW | ODI_CUDA_PAGED_TOO_LONG | ODI_CUDA_PAGED_TOO_MANY_ROWS | ODI_CUDA_PAGED_NO_PAGES;

struct StepArgs {
  odi_cuda_page_tables t;
  odi_cuda_paged_batch b;
  const int* keep;
  const int* fresh;
  const int* prefix;
  PagedGeometry g;
  int page_shift;
};

struct Sum2 {
  int a, b;
};
// Exclusive sums over the block's threads; `total` gets the sums of all.  `warps` is
// a buffer that no other sum uses.
template <int WARPS>
__device__ __forceinline__ Sum2 block_scan(Sum2 v, Sum2* total, Sum2* warps) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Sum2 s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, s.a, o), b = __shfl_up_sync(0xffffffffu, s.b, o);
    if (lane >= o) s.a += a, s.b += b;
  }
  if (lane == 31) warps[warp] = s;
  __syncthreads();
  Sum2 w = lane < WARPS ? warps[lane] : Sum2{0, 0};
#pragma unroll
  for (int o = 1; o < WARPS; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, w.a, o), b = __shfl_up_sync(0xffffffffu, w.b, o);
    if (lane >= o) w.a += a, w.b += b;
  }
  *total = {__shfl_sync(0xffffffffu, w.a, WARPS - 1), __shfl_sync(0xffffffffu, w.b, WARPS - 1)};
  const int before = max(warp - 1, 0);
  const Sum2 p = {__shfl_sync(0xffffffffu, w.a, before), __shfl_sync(0xffffffffu, w.b, before)};
  return {s.a - v.a + (warp ? p.a : 0), s.b - v.b + (warp ? p.b : 0)};
}

// The cluster's barrier, an .aligned one, wants whole warps; lanes come to it from a
// loop that they leave at different times.
__device__ __forceinline__ void step_barrier(int C) {
  if (C == 1) {
    __syncthreads();
  } else {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

// The largest i < n with first[i] <= x, the lists being ascending from 0.
__device__ __forceinline__ int last_at_most(const int* first, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// CHUNKS * THREADS requests at most, `CHUNKS` per thread.
template <int THREADS, int CHUNKS>
__global__ void __launch_bounds__(THREADS) paged_step_kernel(const __grid_constant__ StepArgs a) {
  constexpr int WARPS = THREADS / 32, ROOM = CHUNKS * THREADS;
  // per request: positions kept; first row; rank of its first page dropped (later:
  // its first item); rank of its first page taken, or -1 for one that is refused
  __shared__ int s_keep[ROOM], s_row0[ROOM + 1], s_drop0[ROOM], s_take0[ROOM];
  __shared__ Sum2 warps[4][CHUNKS][WARPS], tiles_of[2][WARPS];
  __shared__ int s_status, s_taken;
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  if (tid == 0) s_status = s_taken = 0;
  pdl_wait();
  const int C = gridDim.x, rank = blockIdx.x, B = a.t.requests;
  const int shift = a.page_shift, P = 1 << shift;
  const int cap = (int)min((long long)a.t.max_pages << shift, 0x7fffffffll);
  const int n = min(max(__ldcg(a.t.free_count), 0), a.t.num_pages);
  auto pages = [&](int len) { return (int)(((long long)len + P - 1) >> shift); };
  struct Want {
    int had, keep, rows, takes, bad, row0;
  } w[CHUNKS];
  // ---- what goes, and where rows begin
  Sum2 base = {0, 0};
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int b = c * THREADS + tid;
    w[c] = {};
    if (b < B) {
      const int fresh = __ldcg(a.fresh + b);
      int len = __ldcg(a.t.lens + b), keep = a.keep ? __ldcg(a.keep + b) : len;
      if (len < 0 || len > cap) w[c].bad |= ODI_CUDA_PAGED_BAD_LENGTH, len = min(max(len, 0), cap);
      if (keep < 0 || keep > len) w[c].bad |= a.keep ? ODI_CUDA_PAGED_BAD_KEEP : 0, keep = min(max(keep, 0), len);
      w[c].rows = min(max(fresh, 0), a.b.max_rows);
      if (fresh < 0 || fresh > a.b.max_new) w[c].bad |= ODI_CUDA_PAGED_BAD_NEW;
      else if (fresh > cap - keep) w[c].bad |= ODI_CUDA_PAGED_TOO_LONG;
      w[c].had = pages(len), w[c].keep = keep;
    }
  }
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int b = c * THREADS + tid;
    Sum2 total;
    const Sum2 e = block_scan<WARPS>({b < B ? w[c].had - pages(w[c].keep) : 0, w[c].rows}, &total, warps[0][c]);
    if (b < B) {
      s_keep[b] = w[c].keep;
      s_drop0[b] = base.a + e.a;
      s_row0[b] = w[c].row0 = min(base.b + e.b, a.b.max_rows);
      if (w[c].rows && w[c].row0 + w[c].rows > a.b.max_rows) w[c].bad |= ODI_CUDA_PAGED_TOO_MANY_ROWS;
      w[c].takes = w[c].bad & REFUSED ? 0 : pages(w[c].keep + w[c].rows) - pages(w[c].keep);
    }
    base.a += total.a, base.b += total.b;
  }
  const int drops = base.a, rows = min(base.b, a.b.max_rows);
  const int top = min(n + drops, a.t.num_pages);  // a table that names pages twice cannot push past the list's end
  if (tid == 0) s_row0[B] = rows;
  // ---- what comes.  A request whose pages are not there, and those after it that need
  // some, take none; so the pages that are taken are those of the first ranks.
  base = {0, 0};
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int b = c * THREADS + tid;
    Sum2 total;
    const Sum2 e = block_scan<WARPS>({w[c].takes, 0}, &total, warps[1][c]);
    if (b < B) {
      const int last = base.a + e.a + w[c].takes;
      if (w[c].takes && last > top) w[c].bad |= ODI_CUDA_PAGED_NO_PAGES;
      const bool granted = !(w[c].bad & REFUSED);
      s_take0[b] = granted ? base.a + e.a : -1;
      if (granted && w[c].takes) atomicMax(&s_taken, last);
      if (w[c].bad) atomicOr(&s_status, w[c].bad);
    }
    base.a += total.a;
  }
  __syncthreads();
  // a page dropped per thread, a row per thread
  for (int k = rank * THREADS + tid; k < drops; k += C * THREADS) {
    const int b = last_at_most(s_drop0, B, k), at = n + drops - 1 - k;
    int* entry = a.t.table + (int64_t)b * a.t.max_pages + pages(s_keep[b]) + k - s_drop0[b];
    if (at < a.t.num_pages) a.t.free_pages[at] = __ldcg(entry);
    *entry = -1;
  }
  step_barrier(C);  // drops are on the list, and every CTA has read the lengths
  constexpr int U = THREADS < 1024 ? 1 : 4;  // rows of a thread whose loads overlap
  for (int q = rank * THREADS + tid; q < a.b.max_rows; q += U * C * THREADS) {
    int pos[U], page[U], *entry[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = q + u * C * THREADS;
      pos[u] = page[u] = -1, entry[u] = nullptr;
      if (r >= rows) continue;
      const int b = last_at_most(s_row0, B, r), first = s_take0[b];
      if (first < 0) continue;
      pos[u] = s_keep[b] + r - s_row0[b];
      const int j = pos[u] >> shift, kept = pages(s_keep[b]);
      int* e = a.t.table + (int64_t)b * a.t.max_pages + j;
      if (j < kept) {
        page[u] = __ldcg(e);
      } else {  // a page that the request takes: its first row writes the table
        page[u] = __ldcg(a.t.free_pages + (top - 1 - (first + j - kept)));
        if (!(pos[u] & (P - 1))) entry[u] = e;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = q + u * C * THREADS;
      if (r >= a.b.max_rows) break;
      if (entry[u]) *entry[u] = page[u];
      a.b.positions[r] = pos[u];
      a.b.slots[r] = (unsigned)page[u] < (unsigned)a.t.num_pages ? (page[u] << shift) + (pos[u] & (P - 1)) : -1;
    }
  }
  if (rank == 0) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int b = c * THREADS + tid;
      if (b >= B) break;
      const bool granted = s_take0[b] >= 0;
      const int len = w[c].keep + (granted ? w[c].rows : 0);
      a.t.lens[b] = len;
      a.b.lens[b] = granted ? len : 0;
      a.b.starts[b] = w[c].row0;
    }
    if (tid == 0) {
      a.b.starts[B] = rows;
      *a.t.free_count = top - s_taken;
      a.b.work[PW_STATUS] = s_status;
    }
  }
  if (rank == C - 1) {  // attention's work list, in the order of rows
    PagedItem* list = const_cast<PagedItem*>(paged_items(a.b.work));
    int* s_item0 = s_drop0;  // every warp is past the drops
    base = {0, 0};
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int b = c * THREADS + tid;
      int items = 0;
      if (b < B && s_take0[b] >= 0) items = (int)(((int64_t)w[c].rows * a.g.G + a.g.rows - 1) / a.g.rows);
      Sum2 total;
      const Sum2 e = block_scan<WARPS>({items, 0}, &total, warps[2][c]);
      if (b < B) s_item0[b] = base.a + e.a;
      base.a += total.a;
    }
    const int items = base.a;
    base = {0, 0};
    __syncthreads();
    for (int i0 = 0; i0 < items; i0 += THREADS) {
      const int i = i0 + tid;
      PagedItem x{};
      if (i < items) {
        const int b = last_at_most(s_item0, B, i), k = i - s_item0[b], n_rows = s_row0[b + 1] - s_row0[b];
        const int token = (int)((min((int64_t)n_rows * a.g.G, (int64_t)(k + 1) * a.g.rows) - 1) / a.g.G);
        x.b = b, x.i = k, x.start = s_row0[b], x.past = s_keep[b], x.len = s_keep[b] + n_rows;
        x.prefix = a.prefix ? __ldcg(a.prefix + b) : 0;
        x.tiles = (paged_limit(x.past, token, x.len, x.prefix) + a.g.tile - 1) / a.g.tile;
      }
      Sum2 total;
      const Sum2 e = block_scan<WARPS>({i < items ? x.tiles + a.g.extra : 0, 0}, &total, tiles_of[i0 / THREADS & 1]);
      x.tile0 = base.a + e.a;
      if (i < items) list[i] = x;
      base.a += total.a;
    }
    if (tid == 0) {
      a.b.work[PW_ITEMS] = items;
      a.b.work[PW_TILES] = base.a;
    }
  }
}

}  // namespace

int paged_view(const odi_cuda_paged_cache* c, PagedView* v, const char* who) {
  char msg[160];
  auto bad = [&](int code, const char* what) {
    snprintf(msg, sizeof msg, "%s: %s", who, what);
    return set_error(code, msg);
  };
  if (!c || !c->k || !c->v) return bad(ODI_CUDA_ERR_INVALID_ARGUMENT, "null cache");
  if (c->dtype != ODI_CUDA_PAGED_F16 && c->dtype != ODI_CUDA_PAGED_BF16)
    return bad(ODI_CUDA_ERR_UNSUPPORTED_DTYPE, "cache dtype is ODI_CUDA_PAGED_F16 or ODI_CUDA_PAGED_BF16");
  if (!page_size_ok(c->page_size)) return bad(ODI_CUDA_ERR_INVALID_ARGUMENT, "page_size is 16, 32, 64 or 128");
  if (c->head_dim != 64 && c->head_dim != 128) return bad(ODI_CUDA_ERR_INVALID_ARGUMENT, "head_dim is 64 or 128");
  if (c->kv_heads < 1 || c->kv_heads > 1024 || c->num_pages < 1 ||
      (int64_t)c->num_pages * c->kv_heads * c->page_size > 0x7fffffffll)
    return bad(ODI_CUDA_ERR_INVALID_ARGUMENT, "kv_heads or num_pages out of range");
  if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return bad(ODI_CUDA_ERR_INVALID_ARGUMENT, "cache must be 16-byte aligned");
  const uintptr_t n = (uintptr_t)c->num_pages * c->kv_heads * c->page_size * c->head_dim * 2;
  if ((uintptr_t)c->k < (uintptr_t)c->v + n && (uintptr_t)c->v < (uintptr_t)c->k + n)
    return bad(ODI_CUDA_ERR_INVALID_ARGUMENT, "k and v share memory");
  *v = {c->k, c->v, c->dtype, c->kv_heads, c->head_dim, c->page_size, c->num_pages, page_shift_of(c->page_size)};
  return ODI_CUDA_OK;
}

bool paged_geometry(int requests, int max_rows, int max_new, int heads, int kv_heads, PagedGeometry* g) {
  if (requests < 1 || requests > ODI_CUDA_PAGED_MAX_REQUESTS || max_rows < 1 || max_rows > ODI_CUDA_PAGED_MAX_ROWS ||
      max_new < 1 || max_new > max_rows || kv_heads < 1 || kv_heads > 1024 || heads < kv_heads || heads % kv_heads ||
      heads / kv_heads > 64)
    return false;
  g->G = heads / kv_heads;
  const int64_t most = (int64_t)max_new * g->G;
  paged_kind(most, &g->rows, &g->tile, &g->extra);
  const int64_t by_request = requests * ((most + g->rows - 1) / g->rows),
                by_rows = requests + (int64_t)max_rows * g->G / g->rows;
  g->max_items = by_request < by_rows ? by_request : by_rows;
  return true;
}

int paged_batch_ok(const odi_cuda_paged_batch* b, PagedGeometry* g, const char* who) {
  char msg[160];
  auto bad = [&](const char* what) {
    snprintf(msg, sizeof msg, "%s: %s", who, what);
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, msg);
  };
  if (!b || !b->starts || !b->lens || !b->positions || !b->slots || !b->work) return bad("null batch");
  if (((uintptr_t)b->starts | (uintptr_t)b->lens | (uintptr_t)b->positions | (uintptr_t)b->slots) & 3 || (uintptr_t)b->work & 15)
    return bad("misaligned batch");
  if (!page_size_ok(b->page_size)) return bad("page_size is 16, 32, 64 or 128");
  if (!paged_geometry(b->requests, b->max_rows, b->max_new, b->heads, b->kv_heads, g)) return bad("batch sizes out of range");
  return ODI_CUDA_OK;
}

}  // namespace odi_cuda

using namespace odi_cuda;

extern "C" {

size_t odi_cuda_paged_work_bytes(int requests, int max_rows, int max_new, int heads, int kv_heads) {
  PagedGeometry g;
  if (!paged_geometry(requests, max_rows, max_new, heads, kv_heads, &g)) return 0;
  return 4 * (size_t)PW_HEADER + sizeof(PagedItem) * (size_t)g.max_items;
}

int odi_cuda_paged_step(const odi_cuda_page_tables* t, const odi_cuda_paged_batch* batch, const int32_t* d_keep,
                        const int32_t* d_new, const int32_t* d_prefix, void* stream) {
  StepArgs a{};
  if (!t || !t->table || !t->lens || !t->free_pages || !t->free_count || !d_new)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "paged_step: null argument");
  if (int rc = paged_batch_ok(batch, &a.g, "paged_step")) return rc;
  if (((uintptr_t)t->table | (uintptr_t)t->lens | (uintptr_t)t->free_pages | (uintptr_t)t->free_count | (uintptr_t)d_keep |
       (uintptr_t)d_new | (uintptr_t)d_prefix) & 3)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "paged_step: misaligned list");
  if (t->requests != batch->requests || t->page_size != batch->page_size)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "paged_step: tables and batch do not belong together");
  if (!page_size_ok(t->page_size) || t->num_pages < 1 || t->max_pages < 1 ||
      (int64_t)t->num_pages * t->page_size > 0x7fffffffll || (int64_t)t->requests * t->max_pages > (1 << 30) ||
      (int64_t)t->max_pages * t->page_size > 0x7fffffffll)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "paged_step: page_size, max_pages or num_pages out of range");
  if (a.g.max_items * ((int64_t)t->max_pages * t->page_size / a.g.tile + 1 + a.g.extra) > 0x7fffffffll)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "paged_step: more work than 2^31 tiles");
  // d_keep and d_new are read before lengths and rows are written, d_prefix after;
  // pages are dropped beside all three
  const int64_t B = t->requests, n = 4 * B;
  for (const void* in : {d_keep, d_new, d_prefix})
    if (bytes_overlap(in, n, t->table, n * t->max_pages) || bytes_overlap(in, n, t->free_pages, 4ll * t->num_pages))
      return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "paged_step: d_keep, d_new or d_prefix overlaps the tables");
  if (bytes_overlap(d_prefix, n, t->lens, n) || bytes_overlap(d_prefix, n, t->free_count, 4) || bytes_overlap(d_prefix, n, batch->starts, n + 4) ||
      bytes_overlap(d_prefix, n, batch->lens, n) || bytes_overlap(d_prefix, n, batch->positions, 4ll * batch->max_rows) ||
      bytes_overlap(d_prefix, n, batch->slots, 4ll * batch->max_rows))
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "paged_step: d_prefix overlaps what the step writes");
  a.t = *t, a.b = *batch, a.keep = d_keep, a.fresh = d_new, a.prefix = d_prefix, a.page_shift = page_shift_of(t->page_size);
  // one CTA where its threads see to everything in a few passes; else eight
  const bool small = t->requests <= 256 && batch->max_rows <= 1024;
  const int C = small ? 1 : 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(C);
  cfg.blockDim = dim3(small ? 256 : 1024);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 2 : 1;
  return kv_launched(small ? cudaLaunchKernelEx(&cfg, paged_step_kernel<256, 1>, a)
                           : cudaLaunchKernelEx(&cfg, paged_step_kernel<1024, MAX_B / 1024>, a),
                     "paged_step");
}

}  // extern "C"
