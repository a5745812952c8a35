// verify.cu -- drafted tokens of several requests against the target's
// probabilities, from given random numbers.
//
//   p_r = softmax(logits_r / T);  the draft x that follows row r is kept iff
//   u_r q_r(x) < p_r(x)
//   at the first row that keeps none, the next token is drawn from
//   max(p - q, 0) (from p where that is nothing), after the last row from p:
//   the first id whose running sum passes u' times the whole
//
// (q: the drafter's probabilities, or 1 at x and 0 elsewhere).  The tokens then
// have the target's distribution.  Everything that a choice hangs on is in 64
// bits: 128,000 ids stand so close that a relative error of 1e-7 would change one
// draw in a hundred.
//
// Two launches.  The first takes 2048 ids of one row per CTA: their largest
// logit, and the sum of exp relative to it.  In the second the CTAs of one
// request each fold its rows' sums, find the row where its drafts end, and add
// up 2048 of that row's weights; the last to arrive finds the token.
#include <math.h>

#include "../../include/odi_cuda.h"
#include "internal.h"
#include "kv_cache.cuh"
#include "pdl_launch.cuh"

namespace odi_cuda {
namespace {

constexpr int THREADS = 256, VPT = 8, SLICE = THREADS * VPT, WARPS = THREADS / 32;
constexpr float TOP = 3.402823466e38f;

struct VerifyArgs {
  const float* logits;
  int64_t ld;
  const int *tokens, *starts;
  const float *probs, *u_accept, *u_next;
  int64_t ld_p;
  int *accepted, *next;
  int requests, rows, slices;
  int64_t V;
  double per_unit;  // 64 / (T ln 2)
  double2* stat;    // [rows][slices]: largest logit, sum
  double2* part;    // [requests][slices]: sums of max(p - q, 0) and of p
  int* count;       // [requests] arrivals, zero between launches
};

// exp(x) for x = t ln2 / 64, t <= 0: 2^(k / 64) from a table, times a Taylor
// polynomial on |t - k| <= 1/2 (the next term is below 2^-54), the table-driven
// method of Tang (1989).  12 operations in 64 bits, which a GPU has few of.
struct Exp64 {
  const double* table;  // [64] in shared memory: 2^(i / 64)
  __device__ __forceinline__ double operator()(double t) const {
    constexpr double c = 0.010830424696249145;  // ln 2 / 64
    t = t < -65000.0 ? -65000.0 : t;            // below 2^-1015: nothing
    const double k = rint(t);
    const int i = (int)k;
    const double r = t - k;
    double p = fma(r, c * c * c * c * c / 120, c * c * c * c / 24);
    p = fma(r, p, c * c * c / 6);
    p = fma(r, p, c * c / 2);
    p = fma(r, p, c);
    p = fma(r, p, 1.0);
    p *= table[i & 63];
    return t <= -65000.0 ? 0.0 : __longlong_as_double(__double_as_longlong(p) + ((long long)(i >> 6) << 52));
  }
};
__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < 64) table[threadIdx.x] = exp2(threadIdx.x / 64.0);
}
__device__ __forceinline__ float load_logit(const float* p) {  // +inf is the largest value there is
  const float x = __ldcg(p);
  return x > TOP ? TOP : x;
}
__device__ __forceinline__ double block_sum(double v, double* s) {
  __syncthreads();
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) t += s[w];
  return t;
}

__global__ void __launch_bounds__(THREADS) verify_stat_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ double table[64], s_sum[WARPS];
  __shared__ float s_max[WARPS];
  pdl_launch_dependents();
  fill_table(table);
  pdl_wait();
  const int row = blockIdx.y, tid = threadIdx.x;
  if (row >= __ldcg(a.starts + a.requests)) return;
  const float* src = a.logits + row * a.ld;
  const int64_t i0 = (int64_t)blockIdx.x * SLICE + tid;
  float x[VPT], m = -INFINITY;
#pragma unroll
  for (int k = 0; k < VPT; ++k) x[k] = i0 + k * THREADS < a.V ? load_logit(src + i0 + k * THREADS) : -INFINITY;
#pragma unroll
  for (int k = 0; k < VPT; ++k) m = fmaxf(m, x[k]);
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((tid & 31) == 0) s_max[tid >> 5] = m;
  __syncthreads();
  for (int w = 0; w < WARPS; ++w) m = fmaxf(m, s_max[w]);
  const Exp64 ex{table};
  const double md = m == -INFINITY ? 0.0 : (double)m;
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < VPT; ++k) sum += x[k] != x[k] ? (double)x[k] : ex(((double)x[k] - md) * a.per_unit);
  sum = block_sum(sum, s_sum);
  if (tid == 0) a.stat[(int64_t)row * a.slices + blockIdx.x] = make_double2(m, sum);
}

__global__ void __launch_bounds__(THREADS) verify_draw_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ double table[64], s_sum[WARPS], s_max[WARPS], s_z[WARPS];
  __shared__ int s_keep[WARPS], s_last;
  pdl_launch_dependents();
  fill_table(table);
  pdl_wait();
  const int b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int start = min(max(__ldcg(a.starts + b), 0), a.rows), end = min(max(__ldcg(a.starts + b + 1), start), a.rows);
  if (start == end) {  // no row: nothing to keep, no token
    if (blockIdx.x == 0 && tid == 0) a.accepted[b] = 0, a.next[b] = -1;
    return;
  }
  __syncthreads();
  const Exp64 ex{table};
  // ---- the row where the drafts end: a warp per row
  int at = end - 1;
  double z = 0.0, m = 0.0;
  for (int r0 = start;; r0 += WARPS) {
    const int r = r0 + warp;
    if (r < end) {
      const double2* st = a.stat + (int64_t)r * a.slices;
      double wm = -INFINITY, wz = 0.0;
      for (int i = lane; i < a.slices; i += 32) wm = fmax(wm, __ldcg(&st[i].x));
#pragma unroll
      for (int o = 16; o; o >>= 1) wm = fmax(wm, __shfl_xor_sync(0xffffffffu, wm, o));
      for (int i = lane; i < a.slices; i += 32) {
        const double2 v = __ldcg(st + i);
        if (v.x > -INFINITY || v.y != v.y) wz += v.y * ex((v.x - wm) * a.per_unit);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) wz += __shfl_xor_sync(0xffffffffu, wz, o);
      if (lane == 0) {
        int keep = 0;
        if (r + 1 < end) {
          const int x = __ldcg(a.tokens + r + 1);
          if (x >= 0 && x < a.V && wz > 0.0) {
            const double e = ex(((double)load_logit(a.logits + r * a.ld + x) - wm) * a.per_unit);
            const double q = a.probs ? (double)__ldcg(a.probs + r * a.ld_p + x) : 1.0;
            keep = (double)__ldcg(a.u_accept + r) * q < e / wz;
          }
        }
        s_keep[warp] = keep, s_z[warp] = wz, s_max[warp] = wm;
      }
    }
    __syncthreads();
    int w = 0;
    while (w < WARPS && r0 + w < end && s_keep[w]) ++w;
    const bool found = w < WARPS && r0 + w < end;
    if (found) at = r0 + w, z = s_z[w], m = s_max[w];
    __syncthreads();
    if (found) break;  // the last row keeps none, so the loop ends
  }
  const bool none = !(z > 0.0);  // no finite logit, or one that is NaN
  const int draft = at + 1 < end ? __ldcg(a.tokens + at + 1) : -1;
  const float *src = a.logits + at * a.ld, *qsrc = a.probs && at + 1 < end ? a.probs + at * a.ld_p : nullptr;
  const double inv = 1.0 / z;
  // (max(p - q, 0), p) of id i
  auto weigh = [&](int64_t i) {
    const double p = ex(((double)load_logit(src + i) - m) * a.per_unit) * inv;
    const double q = qsrc ? (double)__ldcg(qsrc + i) : i == draft && at + 1 < end && !a.probs ? 1.0 : 0.0;
    return make_double2(fmax(p - q, 0.0), p);
  };
  double rest = 0.0, all = 0.0;
  if (!none) {
    const int64_t i0 = (int64_t)blockIdx.x * SLICE + tid;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (i0 + k * THREADS < a.V) {
        const double2 w = weigh(i0 + k * THREADS);
        rest += w.x, all += w.y;
      }
  }
  rest = block_sum(rest, s_sum);
  all = block_sum(all, s_sum);
  if (tid == 0) {
    a.part[(int64_t)b * a.slices + blockIdx.x] = make_double2(rest, all);
    __threadfence();
    s_last = atomicAdd(a.count + b, 1) == a.slices - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  if (tid == 0) a.count[b] = 0, a.accepted[b] = at - start;
  if (none) {
    if (tid == 0) a.next[b] = -1;
    return;
  }
  // ---- the slice, then the id in it
  const double2* part = a.part + (int64_t)b * a.slices;
  __shared__ double s_before, s_target;
  __shared__ int s_slice, s_use, s_token;
  if (warp == 0) {
    double tr = 0.0, tp = 0.0;
    for (int i = lane; i < a.slices; i += 32) {
      const double2 w = __ldcg(part + i);
      tr += w.x, tp += w.y;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) tr += __shfl_xor_sync(0xffffffffu, tr, o), tp += __shfl_xor_sync(0xffffffffu, tp, o);
    const bool use = at + 1 < end && tr > 0.0;  // the rest of p over q
    const double target = (double)__ldcg(a.u_next + b) * (use ? tr : tp);
    double before = 0.0;
    int slice = -1, some = 0;  // the slice, and the last with any weight
    double some_before = 0.0;
    for (int i0 = 0; i0 < a.slices && slice < 0; i0 += 32) {
      const double2 w = i0 + lane < a.slices ? __ldcg(part + i0 + lane) : make_double2(0.0, 0.0);
      const double v = use ? w.x : w.y;
      double s = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
      }
      s += before;
      const double own = s - v;
      const unsigned past = __ballot_sync(0xffffffffu, s > target && v > 0.0), any = __ballot_sync(0xffffffffu, v > 0.0);
      const int pick = past ? __ffs(past) - 1 : any ? 31 - __clz(any) : -1;
      if (pick >= 0) {
        const double pb = __shfl_sync(0xffffffffu, own, pick);
        if (past) slice = i0 + pick, before = pb;
        else some = i0 + pick, some_before = pb;
      }
      if (slice < 0) before = __shfl_sync(0xffffffffu, s, 31);
    }
    if (slice < 0) slice = some, before = some_before;  // rounding left the target past the end
    if (lane == 0) s_before = before, s_target = target, s_slice = slice, s_use = use, s_token = -1;
  }
  __syncthreads();
  const bool use = s_use;
  const int64_t i0 = (int64_t)s_slice * SLICE + tid * VPT;
  double w[VPT], sum = 0.0;
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    w[k] = 0.0;
    if (i0 + k < a.V) {
      const double2 x = weigh(i0 + k);
      w[k] = use ? x.x : x.y;
    }
    sum += w[k];
  }
  double s = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  if (lane == 31) s_sum[warp] = s;
  __syncthreads();
  double run = s_before + (s - sum);
  for (int k = 0; k < warp; ++k) run += s_sum[k];
  // the first id past the target; if rounding leaves none, the last with any weight
  int first = 0x7fffffff, last = -1;
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    run += w[k];
    if (w[k] > 0.0) {
      last = (int)(i0 + k);
      if (run > s_target && first == 0x7fffffff) first = last;
    }
  }
  __shared__ int s_first;
  if (tid == 0) s_first = 0x7fffffff;
  __syncthreads();
  if (first != 0x7fffffff) atomicMin(&s_first, first);
  if (last >= 0) atomicMax(&s_token, last);
  __syncthreads();
  if (tid == 0) a.next[b] = s_first != 0x7fffffff ? s_first : s_token;
}

int64_t slices_of(int64_t V) { return (V + SLICE - 1) / SLICE; }
// The counters have a place of their own, so that calls of other sizes may share a scratch.
constexpr int MAX_REQUESTS = 16384;
constexpr size_t COUNT_BYTES = 4 * MAX_REQUESTS;

}  // namespace
}  // namespace odi_cuda

using namespace odi_cuda;

extern "C" {

size_t odi_cuda_verify_scratch_bytes(int rows, int requests, int64_t V) {
  if (rows < 1 || rows > 65535 || requests < 1 || requests > MAX_REQUESTS || V < 1 || V > 0x7fff0000ll) return 0;
  return COUNT_BYTES + 16 * (size_t)slices_of(V) * ((size_t)rows + requests);
}

int odi_cuda_verify_sampled(const float* d_logits, int64_t ld, const int32_t* d_tokens, const int32_t* d_starts, int rows,
                            int requests, int64_t V, double temperature, const float* d_draft_probs, int64_t ld_probs,
                            const float* d_u_accept, const float* d_u_next, int32_t* d_accepted, int32_t* d_next,
                            void* d_scratch, size_t scratch_bytes, void* stream) {
  if (!d_logits || !d_tokens || !d_starts || !d_u_accept || !d_u_next || !d_accepted || !d_next || !d_scratch)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "verify_sampled: null argument");
  if (rows < 1 || rows > 65535 || requests < 1 || requests > MAX_REQUESTS || V < 1 || V > 0x7fff0000ll)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "verify_sampled: rows, requests or V out of range");
  if (ld < V || ld > (1ll << 40) || (d_draft_probs && (ld_probs < V || ld_probs > (1ll << 40))))
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "verify_sampled: a row stride is shorter than its row");
  if (!(temperature >= 1e-6) || !(temperature <= 1e6))
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "verify_sampled: temperature is 1e-6 to 1e6");
  if (((uintptr_t)d_logits | (uintptr_t)d_tokens | (uintptr_t)d_starts | (uintptr_t)d_draft_probs | (uintptr_t)d_u_accept |
       (uintptr_t)d_u_next | (uintptr_t)d_accepted | (uintptr_t)d_next) & 3 || (uintptr_t)d_scratch & 15)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "verify_sampled: misaligned buffer");
  if (scratch_bytes < odi_cuda_verify_scratch_bytes(rows, requests, V))
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "verify_sampled: scratch too small");
  VerifyArgs a{};
  a.logits = d_logits, a.ld = ld, a.tokens = d_tokens, a.starts = d_starts, a.probs = d_draft_probs, a.ld_p = ld_probs;
  a.u_accept = d_u_accept, a.u_next = d_u_next, a.accepted = d_accepted, a.next = d_next;
  a.requests = requests, a.rows = rows, a.slices = (int)slices_of(V), a.V = V;
  a.per_unit = 92.33248261893241 / temperature;  // 64 / ln 2
  a.count = static_cast<int*>(d_scratch);
  a.stat = reinterpret_cast<double2*>(static_cast<uint8_t*>(d_scratch) + COUNT_BYTES);
  a.part = a.stat + (int64_t)rows * a.slices;
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e = launch_pdl(verify_stat_kernel, dim3(a.slices, rows), dim3(THREADS), s, a);
  if (e == cudaSuccess) e = launch_pdl(verify_draw_kernel, dim3(a.slices, requests), dim3(THREADS), s, a);
  return kv_launched(e, "verify_sampled");
}

}  // extern "C"
