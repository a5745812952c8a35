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
// One cluster: every CTA sums the requests' counts for itself (the lists are
// short), then they share out the requests' pages and the step's rows; two
// cluster barriers stand between drops, takes and the rows' reads of the table.
// Latency bound.
#include <cstdio>

#include "internal.h"
#include "kv_cache.cuh"
#include "paged.cuh"
#include "pdl_launch.cuh"

namespace odi_cuda {
namespace {

constexpr int THREADS = 1024, WARPS = THREADS / 32;
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

struct Sum3 {
  int a, b, c;
};
// Exclusive sums over the block's threads; `total` gets the sums of all.
__device__ __forceinline__ Sum3 block_scan(Sum3 v, Sum3* total, Sum3* warps) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
  Sum3 s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, s.a, o), b = __shfl_up_sync(0xffffffffu, s.b, o),
              c = __shfl_up_sync(0xffffffffu, s.c, o);
    if (lane >= o) s.a += a, s.b += b, s.c += c;
  }
  __syncthreads();  // the last scan's sums have been read
  if (lane == 31) warps[warp] = s;
  __syncthreads();
  Sum3 w = lane < n ? warps[lane] : Sum3{0, 0, 0};
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, w.a, o), b = __shfl_up_sync(0xffffffffu, w.b, o),
              c = __shfl_up_sync(0xffffffffu, w.c, o);
    if (lane >= o) w.a += a, w.b += b, w.c += c;
  }
  *total = {__shfl_sync(0xffffffffu, w.a, 31), __shfl_sync(0xffffffffu, w.b, 31), __shfl_sync(0xffffffffu, w.c, 31)};
  const int before = max(warp - 1, 0);
  const Sum3 p = {__shfl_sync(0xffffffffu, w.a, before), __shfl_sync(0xffffffffu, w.b, before),
                  __shfl_sync(0xffffffffu, w.c, before)};
  return {s.a - v.a + (warp ? p.a : 0), s.b - v.b + (warp ? p.b : 0), s.c - v.c + (warp ? p.c : 0)};
}

__device__ __forceinline__ void step_barrier(int C) {
  if (C == 1) {
    __syncthreads();
  } else {
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

__global__ void __launch_bounds__(THREADS) paged_step_kernel(const __grid_constant__ StepArgs a) {
  // per request: positions kept; first row; rank of its first page dropped (later:
  // its first item); rank of its first page taken, or -1 for one that is refused
  __shared__ int s_keep[MAX_B], s_row0[MAX_B + 1], s_drop0[MAX_B], s_take0[MAX_B];
  __shared__ Sum3 warps[32];
  __shared__ int s_status, s_taken;
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = gridDim.x, rank = blockIdx.x, B = a.t.requests;
  const int shift = a.page_shift, P = 1 << shift;
  const int cap = (int)min((long long)a.t.max_pages << shift, 0x7fffffffll);
  const int n = min(max(__ldcg(a.t.free_count), 0), a.t.num_pages);
  if (tid == 0) s_status = s_taken = 0;
  auto pages = [&](int len) { return (int)(((long long)len + P - 1) >> shift); };
  struct Want {
    int len, keep, rows, drops, takes, bad;
  };
  auto want = [&](int b) {
    Want w{};
    int fresh = __ldcg(a.fresh + b);
    w.len = __ldcg(a.t.lens + b);
    int keep = a.keep ? __ldcg(a.keep + b) : w.len;
    if (w.len < 0 || w.len > cap) w.bad |= ODI_CUDA_PAGED_BAD_LENGTH, w.len = min(max(w.len, 0), cap);
    if (keep < 0 || keep > w.len) w.bad |= a.keep ? ODI_CUDA_PAGED_BAD_KEEP : 0, keep = min(max(keep, 0), w.len);
    w.keep = keep;
    w.rows = min(max(fresh, 0), a.b.max_rows);
    if (fresh < 0 || fresh > a.b.max_new) w.bad |= ODI_CUDA_PAGED_BAD_NEW;
    else if (fresh > cap - keep) w.bad |= ODI_CUDA_PAGED_TOO_LONG;
    w.drops = pages(w.len) - pages(keep);
    w.takes = w.bad & REFUSED ? 0 : pages(keep + w.rows) - pages(keep);
    return w;
  };
  // ---- what goes, and where rows begin
  Sum3 base = {0, 0, 0};
  for (int b0 = 0; b0 < B; b0 += THREADS) {
    const int b = b0 + tid;
    Want w{};
    if (b < B) w = want(b);
    Sum3 total;
    const Sum3 e = block_scan({w.drops, w.rows, 0}, &total, warps);
    if (b < B) {
      s_keep[b] = w.keep;
      s_drop0[b] = base.a + e.a;
      s_row0[b] = min(base.b + e.b, a.b.max_rows);
    }
    base.a += total.a, base.b += total.b;
  }
  const int drops = base.a, rows = min(base.b, a.b.max_rows);
  if (tid == 0) s_row0[B] = rows;
  __syncthreads();
  const int top = min(n + drops, a.t.num_pages);  // a table that names pages twice cannot push past the list's end
  for (int b = rank * WARPS + warp; b < B; b += C * WARPS) {
    const int len = min(max(__ldcg(a.t.lens + b), 0), cap);
    const int j0 = pages(s_keep[b]), j1 = pages(len), r0 = s_drop0[b];
    int* row = a.t.table + (int64_t)b * a.t.max_pages;
    for (int j = j0 + lane; j < j1; j += 32) {
      const int at = n + drops - 1 - (r0 + j - j0);
      if (at < a.t.num_pages) a.t.free_pages[at] = __ldcg(row + j);
      row[j] = -1;
    }
  }
  // ---- what comes: every CTA again for itself, before the lengths change.
  // A request whose pages are not there, and those after it that need some, take
  // none; so the pages that are taken are those of the first ranks.
  base = {0, 0, 0};
  for (int b0 = 0; b0 < B; b0 += THREADS) {
    const int b = b0 + tid;
    Want w{};
    if (b < B) {
      w = want(b);
      if (w.rows && s_row0[b] + w.rows > a.b.max_rows) w.bad |= ODI_CUDA_PAGED_TOO_MANY_ROWS;
      if (w.bad & REFUSED) w.takes = 0;
    }
    Sum3 total;
    const Sum3 e = block_scan({w.takes, 0, 0}, &total, warps);
    if (b < B) {
      const int last = base.a + e.a + w.takes;
      if (w.takes && last > top) w.bad |= ODI_CUDA_PAGED_NO_PAGES;
      const bool granted = !(w.bad & REFUSED);
      s_take0[b] = granted ? base.a + e.a : -1;
      if (granted && w.takes) atomicMax(&s_taken, last);
      if (w.bad) atomicOr(&s_status, w.bad);
    }
    base.a += total.a;
  }
  step_barrier(C);  // drops are on the list, and every CTA has read the lengths
  for (int b = rank * WARPS + warp; b < B; b += C * WARPS) {
    const int r0 = s_take0[b];
    if (r0 < 0) continue;
    const int j0 = pages(s_keep[b]), j1 = pages(s_keep[b] + s_row0[b + 1] - s_row0[b]);
    int* row = a.t.table + (int64_t)b * a.t.max_pages;
    for (int j = j0 + lane; j < j1; j += 32) row[j] = __ldcg(a.t.free_pages + (top - 1 - (r0 + j - j0)));
  }
  if (rank == 0) {
    for (int b = tid; b < B; b += THREADS) {
      const int n_rows = s_row0[b + 1] - s_row0[b], len = s_keep[b] + (s_take0[b] >= 0 ? n_rows : 0);
      a.t.lens[b] = len;
      a.b.lens[b] = s_take0[b] >= 0 ? len : 0;
      a.b.starts[b] = s_row0[b];
    }
    if (tid == 0) {
      a.b.starts[B] = rows;
      *a.t.free_count = top - s_taken;
      a.b.work[PW_STATUS] = s_status;
    }
  }
  if (rank == C - 1) {  // attention's work list, in the order of rows
    PagedItem* list = const_cast<PagedItem*>(paged_items(a.b.work));
    int* s_item0 = s_drop0;
    base = {0, 0, 0};
    for (int b0 = 0; b0 < B; b0 += THREADS) {
      const int b = b0 + tid;
      int items = 0;
      if (b < B && s_take0[b] >= 0) items = (int)(((int64_t)(s_row0[b + 1] - s_row0[b]) * a.g.G + a.g.rows - 1) / a.g.rows);
      Sum3 total;
      const Sum3 e = block_scan({items, 0, 0}, &total, warps);
      if (b < B) s_item0[b] = base.a + e.a;
      base.a += total.a;
    }
    const int items = base.a;
    base = {0, 0, 0};
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
      Sum3 total;
      const Sum3 e = block_scan({x.tiles, 0, 0}, &total, warps);
      x.tile0 = base.a + e.a;
      if (i < items) list[i] = x;
      base.a += total.a;
    }
    if (tid == 0) {
      a.b.work[PW_ITEMS] = items;
      a.b.work[PW_TILES] = base.a;
    }
  }
  step_barrier(C);  // the table is whole
  for (int r = rank * THREADS + tid; r < a.b.max_rows; r += C * THREADS) {
    int pos = -1, slot = -1;
    if (r < rows) {
      const int b = last_at_most(s_row0, B, r);
      if (s_take0[b] >= 0) {
        pos = s_keep[b] + r - s_row0[b];
        const int page = __ldcg(a.t.table + (int64_t)b * a.t.max_pages + (pos >> shift));
        if ((unsigned)page < (unsigned)a.t.num_pages) slot = (page << shift) + (pos & (P - 1));
      }
    }
    a.b.positions[r] = pos;
    a.b.slots[r] = slot;
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
  paged_kind(most, &g->rows, &g->tile);
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
  a.t = *t, a.b = *batch, a.keep = d_keep, a.fresh = d_new, a.prefix = d_prefix, a.page_shift = page_shift_of(t->page_size);
  // one CTA where its threads see to everything at once; else eight
  const int C = batch->max_rows <= 2 * THREADS && t->requests <= 4 * WARPS ? 1 : 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(C);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 2 : 1;
  return kv_launched(cudaLaunchKernelEx(&cfg, paged_step_kernel, a), "paged_step");
}

}  // extern "C"
