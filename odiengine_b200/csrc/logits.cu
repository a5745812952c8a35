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
// row's scratch for the next call.
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
template <int VPT>
__global__ void __launch_bounds__(THREADS) logits_kernel(const LogitsArgs a) {
  constexpr int SLICE = 4 * THREADS * VPT;
  constexpr int HPT = 4;  // history entries per thread requested ahead
  __shared__ unsigned words[SLICE];
  __shared__ unsigned long long warp_best[THREADS / 32];
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  const bool lists = a.history || a.bias_count;
  if (lists)
    for (int i = tid; i < SLICE / 4; i += THREADS) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
  pdl_wait();
  const int64_t row = blockIdx.y;
  const float* in = a.in + row * a.ld_in;
  // ids of this slice: first .. first + SLICE - 1, clipped to the vocabulary
  const int shift = (int)(((uintptr_t)in >> 2) & 3);
  const int64_t first = (int64_t)blockIdx.x * SLICE - shift;
  float4 v[VPT];
#pragma unroll
  for (int u = 0; u < VPT; ++u) {
    const int64_t id = first + (u * THREADS + tid) * 4;
    if (id >= 0 && id + 3 < a.V) {
      v[u] = __ldcg(reinterpret_cast<const float4*>(in + id));
    } else {
      v[u].x = id >= 0 && id < a.V ? __ldcg(in + id) : 0.f;
      v[u].y = id + 1 >= 0 && id + 1 < a.V ? __ldcg(in + id + 1) : 0.f;
      v[u].z = id + 2 >= 0 && id + 2 < a.V ? __ldcg(in + id + 2) : 0.f;
      v[u].w = id + 3 >= 0 && id + 3 < a.V ? __ldcg(in + id + 3) : 0.f;
    }
  }
  const unsigned* mask = a.mask ? a.mask + row * a.mask_ld : nullptr;
  unsigned mlo[VPT], mhi[VPT];
#pragma unroll
  for (int u = 0; u < VPT; ++u) {  // the words of four ids from id0 on
    mlo[u] = mhi[u] = 0;
    const int64_t id0 = first + (u * THREADS + tid) * 4;
    if (mask && id0 + 3 >= 0 && id0 < a.V) {
      const int64_t i0 = id0 < 0 ? 0 : id0, i3 = id0 + 3 < a.V ? id0 + 3 : a.V - 1;
      mlo[u] = __ldcg(mask + (i0 >> 5));
      mhi[u] = __ldcg(mask + (i3 >> 5));
    }
  }
  if (lists) {
    const int64_t lo = first < 0 ? 0 : first, hi = first + SLICE < a.V ? first + SLICE : a.V;
    const int* hist = a.history ? a.history + row * a.history_ld : nullptr;
    int n = !hist ? 0 : a.history_len ? __ldcg(a.history_len + row) : a.history_max;
    int h[HPT];
#pragma unroll
    for (int u = 0; u < HPT; ++u) h[u] = tid + u * THREADS < a.history_max && hist ? __ldcg(hist + tid + u * THREADS) : -1;
    const int b0 = tid < a.bias_count ? __ldcg(a.bias_ids + tid) : -1;
    n = n < a.history_max ? n : a.history_max;
    __syncthreads();
    auto count = [&](int id) {
      if (id >= lo && id < hi) atomicAdd(&words[id - first], 1u);
    };
#pragma unroll
    for (int u = 0; u < HPT; ++u)
      if (tid + u * THREADS < n) count(h[u]);
    for (int i = tid + HPT * THREADS; i < n; i += THREADS) count(__ldcg(hist + i));
    __syncthreads();
    for (int i = tid; i < a.bias_count; i += THREADS) {
      const int id = i == tid ? b0 : __ldcg(a.bias_ids + i);
      if (id >= lo && id < hi) {  // the low halves no longer change: the maximum is of the entry
        unsigned* w = &words[id - first];
        atomicMax(w, ((unsigned)(i + 1) << 16) | (*(volatile unsigned*)w & 0xffffu));
      }
    }
    if (a.bias_count) __syncthreads();
  }
  float bv = -INFINITY;
  int64_t bi = -1;
  float* out = a.out ? a.out + row * a.ld_out : nullptr;
  const bool out_vec = out && (((uintptr_t)out >> 2) & 3) == (unsigned)shift;
#pragma unroll
  for (int u = 0; u < VPT; ++u) {
    const int slot = (u * THREADS + tid) * 4;
    const int64_t id0 = first + slot;
    if (id0 + 3 < 0 || id0 >= a.V) continue;
    float x[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
    if (lists) {
      const uint4 w4 = *reinterpret_cast<const uint4*>(&words[slot]);
      const unsigned w[4] = {w4.x, w4.y, w4.z, w4.w};
      if (w4.x | w4.y | w4.z | w4.w) {
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
      const int64_t i0 = id0 < 0 ? 0 : id0;
      const unsigned bits = __funnelshift_r(mlo[u], mhi[u], (unsigned)(i0 & 31)) << (int)(i0 - id0);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!((bits >> e) & 1u)) x[e] = -INFINITY;
    }
    const bool whole = id0 >= 0 && id0 + 3 < a.V;
    if (out) {
      if (whole && out_vec) {
        *reinterpret_cast<float4*>(out + id0) = make_float4(x[0], x[1], x[2], x[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (id0 + e >= 0 && id0 + e < a.V) out[id0 + e] = x[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if ((whole || (id0 + e >= 0 && id0 + e < a.V)) && x[e] > bv) bv = x[e], bi = id0 + e;  // ids ascend
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
  if (rows < 0 || rows > 65535 || V < 1 || V > 0x7ffffff0) return bad("logits_adjust: rows or vocabulary out of range");
  if (ld_logits < V || (d_out && ld_out < V)) return bad("logits_adjust: a row stride is shorter than the vocabulary");
  if (d_out == d_logits && ld_out != ld_logits) return bad("logits_adjust: in place needs one row stride");
  if (((uintptr_t)d_logits | (uintptr_t)d_out | (uintptr_t)d_tokens) & 3) return bad("logits_adjust: misaligned buffer");
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
