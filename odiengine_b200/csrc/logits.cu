// logits.cu -- penalties, biases and grammar masks on rows of logits, and the
// greedy token of each adjusted row.
//
//   l' = (c > 0 ? (l > 0 ? l / r : l * r) : l) - c f - [c > 0] p + b[id]
//   l' = -inf where the mask bit is 0
// with c the id's count in the row's history, r / f / p the repetition,
// frequency and presence penalties, b the sparse biases.  Every step is one
// IEEE fp32 operation in that order (no contraction), so a greedy choice
// between two near values does not depend on how the kernel was compiled.
#include <math.h>

#include "../../include/odi_cuda.h"
#include "internal.h"
#include "kv_cache.cuh"
#include "pdl_launch.cuh"

namespace odi_cuda {
namespace {

// One CTA takes SLICE ids of one row.  Everything it reads is requested at
// once -- its logits and mask words, the first entries of the row's history and
// of the biases -- so a CTA pays one round trip to memory; then the history and
// the biases are sorted into a word per id in shared memory -- the count in the
// low half, the last bias entry + 1 in the high half -- and each id is adjusted
// and stored once.  So the row is read and
// written once whatever the penalties, and the history is re-read (from L2)
// once per slice.  The slice starts on a 16-byte boundary of the row's own
// address, whatever the vocabulary and row stride.  The slices' best ids meet
// in a 64-bit maximum per row: the value's order-preserving image above the
// inverted id, so equal values keep the lowest id and the order in which CTAs
// arrive does not matter.  The row's last CTA writes the token and zeroes the
// row's scratch for the next call.  64 rows of 128259 ids, 67 MB read and
// written, 1000 history ids and 300 biases each: 21 to 24 us (10.3 at the copy
// peak), 11.1 without lists; a CTA's pass over the lists and its barriers are not
// hidden by its neighbours' loads.  One row of 32000: 3.9 us, latency.
constexpr int THREADS = 256;

struct LogitsArgs {
  const float* in;
  float* out;
  int64_t ld_in, ld_out;
  int* tokens;
  const int* history;
  const int* history_len;
  int64_t history_ld;
  int history_max;
  const int* bias_ids;
  const float* bias;
  int bias_count;
  const unsigned* mask;
  int64_t mask_ld;
  float repeat, frequency, presence;
  int64_t V;
  unsigned long long* best;  // [rows]
  unsigned* arrived;         // [rows]
};

// VPT: 16-byte pieces per thread.  Four for many rows; one where the CTAs of
// all rows would not fill the SMs, so that a row spreads over more of them.
// Five CTAs per SM: 24.3 us for those 64 rows, 27.1 with four.
template <int VPT>
__global__ void __launch_bounds__(THREADS, VPT == 4 ? 5 : 1) logits_kernel(const LogitsArgs a) {
  constexpr int SLICE = 4 * THREADS * VPT;
  constexpr int HPT = 4;  // history entries per thread requested ahead
  __shared__ unsigned words[SLICE];
  __shared__ unsigned long long warp_best[THREADS / 32];
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  const bool lists = a.history || a.bias_count;
  if (lists)
#pragma unroll
    for (int u = 0; u < VPT; ++u) reinterpret_cast<uint4*>(words)[u * THREADS + tid] = make_uint4(0, 0, 0, 0);
  pdl_wait();
  const int64_t row = blockIdx.y;
  const float* in = a.in + row * a.ld_in;
  // ids of this slice: first .. first + SLICE - 1, clipped to the vocabulary.
  // Ids, and the ends of a slice past the last, fit 32 bits (V <= 2^31 - 2^16).
  const int V = (int)a.V, shift = (int)(((uintptr_t)in >> 2) & 3);
  const int first = (int)blockIdx.x * SLICE - shift;
  const bool inner = first >= 0 && first <= V - SLICE;  // every id of the slice is a token
  float4 v[VPT];
#pragma unroll
  for (int u = 0; u < VPT; ++u) {
    const int id = first + (u * THREADS + tid) * 4;
    if (inner || (id >= 0 && id < V - 3)) {
      v[u] = __ldcg(reinterpret_cast<const float4*>(in + id));
    } else {
      v[u].x = id >= 0 && id < V ? __ldcg(in + id) : 0.f;
      v[u].y = id + 1 >= 0 && id + 1 < V ? __ldcg(in + id + 1) : 0.f;
      v[u].z = id + 2 >= 0 && id + 2 < V ? __ldcg(in + id + 2) : 0.f;
      v[u].w = id + 3 >= 0 && id + 3 < V ? __ldcg(in + id + 3) : 0.f;
    }
  }
  const unsigned* mask = a.mask ? a.mask + row * a.mask_ld : nullptr;
  unsigned mlo[VPT], mhi[VPT];
#pragma unroll
  for (int u = 0; u < VPT; ++u) {  // the words of four ids from id0 on
    mlo[u] = mhi[u] = 0;
    const int id0 = first + (u * THREADS + tid) * 4;
    if (mask && (inner || (id0 + 3 >= 0 && id0 < V))) {
      mlo[u] = __ldcg(mask + (max(id0, 0) >> 5));
      mhi[u] = __ldcg(mask + (min(id0 + 3, V - 1) >> 5));
    }
  }
  if (lists) {
    const int lo = max(first, 0), span = max(min(first + SLICE, V) - lo, 0);  // the last slice may hold no id
    const int* hist = a.history ? a.history + row * a.history_ld : nullptr;
    int n = !hist ? 0 : a.history_len ? __ldcg(a.history_len + row) : a.history_max;
    int h[HPT];
#pragma unroll
    for (int u = 0; u < HPT; ++u) h[u] = hist && tid + u * THREADS < a.history_max ? __ldcg(hist + tid + u * THREADS) : -1;
    const int b0 = tid < a.bias_count ? __ldcg(a.bias_ids + tid) : -1;
    n = min(n, a.history_max);
    __syncthreads();
    auto mine = [&](int id) { return (unsigned)(id - lo) < (unsigned)span && id >= 0; };
#pragma unroll
    for (int u = 0; u < HPT; ++u)
      if (tid + u * THREADS < n && mine(h[u])) atomicAdd(&words[h[u] - first], 1u);
    for (int i = tid + HPT * THREADS; i < n; i += THREADS) {
      const int id = __ldcg(hist + i);
      if (mine(id)) atomicAdd(&words[id - first], 1u);
    }
    __syncthreads();
    for (int i = tid; i < a.bias_count; i += THREADS) {
      const int id = i == tid ? b0 : __ldcg(a.bias_ids + i);
      if (mine(id)) {  // the low halves no longer change: the maximum is of the entry
        unsigned* w = &words[id - first];
        atomicMax(w, ((unsigned)(i + 1) << 16) | (*(volatile unsigned*)w & 0xffffu));
      }
    }
    if (a.bias_count) __syncthreads();
  }
  float bv = -INFINITY;
  int bi = -1;
  float* out = a.out ? a.out + row * a.ld_out : nullptr;
  const bool out_vec = out && (((uintptr_t)out >> 2) & 3) == (unsigned)shift;
#pragma unroll
  for (int u = 0; u < VPT; ++u) {
    const int slot = (u * THREADS + tid) * 4, id0 = first + slot;
    if (!inner && (id0 + 3 < 0 || id0 >= V)) continue;
    float x[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
    if (lists) {
      const uint4 w4 = *reinterpret_cast<const uint4*>(&words[slot]);
      if (w4.x | w4.y | w4.z | w4.w) {
        const unsigned w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned c = w[e] & 0xffffu, b = w[e] >> 16;
          if (c) {
            x[e] = x[e] > 0.f ? __fdiv_rn(x[e], a.repeat) : __fmul_rn(x[e], a.repeat);
            x[e] = __fsub_rn(x[e], __fmul_rn((float)c, a.frequency));
            x[e] = __fsub_rn(x[e], a.presence);
          }
          if (b) x[e] = __fadd_rn(x[e], __ldcg(a.bias + b - 1));
        }
      }
    }
    if (mask) {  // four bits from id0 on; ids before the row's first have no bits
      const int i0 = max(id0, 0);
      const unsigned bits = __funnelshift_r(mlo[u], mhi[u], (unsigned)(i0 & 31)) << (i0 - id0);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!((bits >> e) & 1u)) x[e] = -INFINITY;
    }
    const bool whole = inner || (id0 >= 0 && id0 < V - 3);
    if (whole) {
      if (out_vec) *reinterpret_cast<float4*>(out + id0) = make_float4(x[0], x[1], x[2], x[3]);
      else if (out) out[id0] = x[0], out[id0 + 1] = x[1], out[id0 + 2] = x[2], out[id0 + 3] = x[3];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in_row = id0 + e >= 0 && id0 + e < V;
        if (out && in_row) out[id0 + e] = x[e];
        if (!in_row) x[e] = -INFINITY;
      }
    }
    const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));  // NaN is passed over
    if (top > bv) {  // ids ascend: the first of equal values stays
      bv = top;
      bi = id0 + (x[0] == top ? 0 : x[1] == top ? 1 : x[2] == top ? 2 : 3);
    }
  }
  if (!a.tokens) return;
  // order-preserving image of the value (-0 as +0); 0: nothing above -inf
  unsigned long long key = 0;
  if (bi >= 0) {
    const unsigned b = __float_as_uint(bv + 0.0f);
    key = ((unsigned long long)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32) | (0xffffffffu - (unsigned)bi);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
    key = other > key ? other : key;
  }
  if ((tid & 31) == 0) warp_best[tid >> 5] = key;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) key = warp_best[w] > key ? warp_best[w] : key;
    if (key) atomicMax(&a.best[row], key);
    __threadfence();
    if (atomicAdd(&a.arrived[row], 1u) == gridDim.x - 1) {
      __threadfence();
      const unsigned long long top = atomicExch(&a.best[row], 0ull);
      a.tokens[row] = top ? (int)(0xffffffffu - (unsigned)(top & 0xffffffffu)) : -1;
      a.arrived[row] = 0;
    }
  }
}

}  // namespace
}  // namespace odi_cuda

using namespace odi_cuda;

extern "C" {

size_t odi_cuda_logits_scratch_bytes(int rows) { return rows > 0 ? (size_t)rows * 16 : 0; }

int odi_cuda_logits_adjust(const float* d_logits, int64_t ld_logits, float* d_out, int64_t ld_out, int32_t* d_tokens,
                           int rows, int64_t V, const odi_cuda_logits_opts* opts, void* d_scratch,
                           size_t scratch_bytes, void* stream) {
  auto bad = [](const char* m) { return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, m); };
  if (!d_logits || (!d_out && !d_tokens)) return bad("logits_adjust: null argument");
  if (rows < 0 || rows > 65535 || V < 1 || V > 0x7fff0000) return bad("logits_adjust: rows or vocabulary out of range");
  if (ld_logits < V || (d_out && ld_out < V)) return bad("logits_adjust: a row stride is shorter than the vocabulary");
  if (((uintptr_t)d_logits | (uintptr_t)d_out | (uintptr_t)d_tokens) & 3) return bad("logits_adjust: misaligned buffer");
  if (d_out && (d_out != d_logits || ld_out != ld_logits) && rows_overlap(d_logits, ld_logits, V, d_out, ld_out, V, rows))
    return bad("logits_adjust: the output overlaps the logits and is not the logits themselves");
  if (d_tokens && (!d_scratch || ((uintptr_t)d_scratch & 7) || scratch_bytes < odi_cuda_logits_scratch_bytes(rows)))
    return bad("logits_adjust: scratch missing, misaligned or too small");
  LogitsArgs a{};
  a.in = d_logits, a.out = d_out, a.ld_in = ld_logits, a.ld_out = ld_out, a.tokens = d_tokens, a.V = V;
  a.repeat = 1.f;
  if (opts) {
    if (!(opts->repeat_penalty > 0.f) || !isfinite(opts->repeat_penalty) || !isfinite(opts->frequency_penalty) ||
        !isfinite(opts->presence_penalty))
      return bad("logits_adjust: penalties must be finite and the repetition penalty positive");
    if (opts->history_max < 0 || opts->history_max > 65535 || opts->bias_count < 0 || opts->bias_count > 65535)
      return bad("logits_adjust: at most 65535 history tokens and biases");
    if (((uintptr_t)opts->history | (uintptr_t)opts->history_len | (uintptr_t)opts->bias_ids | (uintptr_t)opts->bias |
         (uintptr_t)opts->mask) & 3)
      return bad("logits_adjust: misaligned list");
    if (opts->history && opts->history_ld != 0 && opts->history_ld < opts->history_max)
      return bad("logits_adjust: history stride shorter than its row");
    if (opts->bias_count && (!opts->bias_ids || !opts->bias)) return bad("logits_adjust: null biases");
    if (opts->mask && opts->mask_ld != 0 && opts->mask_ld < (V + 31) / 32)
      return bad("logits_adjust: mask stride shorter than its row");
    if (opts->history && opts->history_max > 0) {
      a.history = opts->history, a.history_len = opts->history_len;
      a.history_ld = opts->history_ld, a.history_max = opts->history_max;
    }
    a.bias_ids = opts->bias_ids, a.bias = opts->bias, a.bias_count = opts->bias_count;
    a.mask = opts->mask, a.mask_ld = opts->mask_ld;
    a.repeat = opts->repeat_penalty, a.frequency = opts->frequency_penalty, a.presence = opts->presence_penalty;
  }
  if (!rows) return ODI_CUDA_OK;
  a.best = static_cast<unsigned long long*>(d_scratch);
  a.arrived = reinterpret_cast<unsigned*>(a.best + rows);
  // a row may start up to three ids past a 16-byte boundary
  auto ctas = [&](int vpt) { return (unsigned)((V + 3 + 4 * THREADS * vpt - 1) / (4 * THREADS * vpt)); };
  cudaStream_t s = (cudaStream_t)stream;
  const cudaError_t e = (int64_t)ctas(4) * rows >= 148 * 2 ? launch_pdl(logits_kernel<4>, dim3(ctas(4), rows), dim3(THREADS), s, a)
                                                           : launch_pdl(logits_kernel<1>, dim3(ctas(1), rows), dim3(THREADS), s, a);
  return kv_launched(e, "logits_adjust");
}

}  // extern "C"
