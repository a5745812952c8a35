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
// Two launches.  The first takes 2048 or 8192 ids of one row per CTA: their largest
// logit, and the sum of exp relative to it.  In the second the CTAs of one
// request each fold its rows' sums, find the row where its drafts end, and add
// up as many of that row's weights; the last to arrive finds the token.
//
// 81 rows of 128,259 ids of 16 requests take 31 us, 2.5 TB/s: HBM would let them take
// 11, the 12 operations of 64 bits per id 9, and two launches whose CTAs end with
// joins do the rest.  5 rows of 32,000 ids take 11 us, nearly all of it latency.
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
  int requests, rows, slices, stats;  // pieces of a row: of the draw, of the sums
  int64_t V;
  double unit;      // 256 / (T ln 2)
  double2* stat;    // [rows][stats]: largest logit, sum
  double2* part;    // [requests][slices]: sums of max(p - q, 0) and of p
  int* count;       // [requests] arrivals, zero between launches
};

__constant__ double TWO_TO_256THS[256] = {  // 2^(i / 256)
    1.0, 1.0027112750502025, 1.0054299011128027, 1.0081558981184175,
    1.0108892860517005, 1.0136300849514894, 1.016378314910953, 1.019133996077738,
    1.0218971486541166, 1.0246677928971357, 1.0274459491187637, 1.030231637686041,
    1.0330248790212284, 1.0358256936019572, 1.0386341019613787, 1.041450124688316,
    1.0442737824274138, 1.0471050958792898, 1.0499440858006872, 1.0527907730046264,
    1.0556451783605572, 1.0585073227945128, 1.061377227289262, 1.0642549128844645,
    1.0671404006768237, 1.0700337118202419, 1.0729348675259756, 1.075843889062791,
    1.0787607977571199, 1.0816856149932152, 1.0846183622133092, 1.0875590609177697,
    1.0905077326652577, 1.0934643990728858, 1.0964290818163769, 1.099401802630222,
    1.102382583307841, 1.1053714457017412, 1.1083684117236787, 1.1113735033448175,
    1.1143867425958924, 1.1174081515673693, 1.1204377524096067, 1.12347556733302,
    1.1265216186082418, 1.129575928566288, 1.1326385195987192, 1.1357094141578055,
    1.1387886347566916, 1.1418762039695616, 1.1449721444318042, 1.148076478840179,
    1.1511892299529827, 1.154310420590216, 1.1574400736337511, 1.1605782120274988,
    1.1637248587775775, 1.1668800369524817, 1.1700437696832502, 1.1732160801636373,
    1.1763969916502812, 1.1795865274628758, 1.182784710984341, 1.1859915656609938,
    1.189207115002721, 1.1924313825831512, 1.1956643920398273, 1.1989061670743806,
    1.202156731452703, 1.2054161090051239, 1.2086843236265816, 1.2119613992768012,
    1.215247359980469, 1.2185422298274085, 1.2218460329727576, 1.2251587936371455,
    1.22848053610687, 1.2318112847340759, 1.2351510639369334, 1.2384998981998165,
    1.241857812073484, 1.245224830175258, 1.2486009771892048, 1.2519862778663162,
    1.255380757024691, 1.2587844395497165, 1.2621973503942507, 1.2656195145788063,
    1.2690509571917332, 1.2724917033894028, 1.275941778396392, 1.2794012075056693,
    1.2828700160787783, 1.2863482295460256, 1.2898358734066657, 1.2933329732290895,
    1.2968395546510096, 1.3003556433796506, 1.3038812651919358, 1.3074164459346773,
    1.3109612115247644, 1.3145155879493546, 1.318079601266064, 1.3216532776031575,
    1.3252366431597413, 1.3288297242059544, 1.3324325470831615, 1.3360451382041458,
    1.339667524053303, 1.3432997311868353, 1.3469417862329458, 1.3505937158920345,
    1.3542555469368927, 1.3579273062129011, 1.3616090206382248, 1.365300717204012,
    1.3690024229745905, 1.3727141650876684, 1.3764359707545302, 1.380167867260238,
    1.383909881963832, 1.387662042298529, 1.3914243757719262, 1.3951969099662003,
    1.3989796725383112, 1.4027726912202048, 1.4065759938190154, 1.4103896082172707,
    1.4142135623730951, 1.4180478843204152, 1.4218926021691656, 1.4257477441054942,
    1.42961333839197, 1.433489413367789, 1.4373759974489824, 1.4412731191286257,
    1.4451808069770467, 1.449099089642035, 1.4530279958490526, 1.4569675544014438,
    1.460917794180647, 1.4648787441464057, 1.4688504333369818, 1.4728328908693675,
    1.4768261459394993, 1.4808302278224719, 1.4848451658727524, 1.488870989524397,
    1.4929077282912648, 1.4969554117672355, 1.5010140696264256, 1.5050837316234065,
    1.5091644275934228, 1.5132561874526098, 1.5173590411982147, 1.5214730189088146,
    1.5255981507445384, 1.529734466947287, 1.533881997840956, 1.5380407738316568,
    1.5422108254079407, 1.5463921831410214, 1.550584877685, 1.5547889397770887,
    1.559004400237837, 1.5632312899713576, 1.567469639965553, 1.5717194812923414,
    1.5759808451078865, 1.5802537626528246, 1.5845382652524937, 1.588834384317164,
    1.593142151342267, 1.597461597908627, 1.6017927556826934, 1.606135656416771,
    1.6104903319492543, 1.6148568142048607, 1.6192351351948637, 1.6236253270173289,
    1.6280274218573478, 1.632441451987275, 1.6368674497669644, 1.6413054476440063,
    1.645755478153965, 1.6502175739206177, 1.6546917676561943, 1.6591780921616162,
    1.6636765803267364, 1.6681872651305825, 1.6727101796415966, 1.6772453570178785,
    1.681792830507429, 1.6863526334483934, 1.6909247992693053, 1.6955093614893326,
    1.7001063537185235, 1.7047158096580513, 1.709337763100463, 1.713972247929926,
    1.718619298122478, 1.723278947746274, 1.7279512309618377, 1.732636182022311,
    1.7373338352737062, 1.7420442251551564, 1.746767386199169, 1.7515033530318782,
    1.7562521603732995, 1.761013843037584, 1.7657884359332727, 1.7705759740635547,
    1.7753764925265212, 1.7801900265154245, 1.785016611318935, 1.789856282321401,
    1.7947090750031072, 1.7995750249405351, 1.804454167806624, 1.809346539371032,
    1.8142521755003989, 1.8191711121586085, 1.8241033854070534, 1.8290490314048973,
    1.8340080864093424, 1.8389805867758937, 1.843966568958626, 1.8489660695104508,
    1.8539791250833855, 1.8590057724288205, 1.864046048397789, 1.8690999899412386,
    1.8741676341103, 1.8792490180565602, 1.8843441790323345, 1.8894531543909392,
    1.8945759815869656, 1.8997126981765553, 1.9048633418176741, 1.9100279502703899,
    1.9152065613971474, 1.9203992131630474, 1.925605943636125, 1.930826790987627,
    1.9360617934922943, 1.9413109895286405, 1.9465744175792332, 1.9518521162309783,
    1.9571441241754002, 1.9624504802089273, 1.9677712232331759, 1.9731063922552343,
    1.978456026387951, 1.9838201648502194, 1.9891988469672663, 1.9945921121709402};
// exp of a logit x relative to m, over the temperature: with unit = 256 / (T ln 2),
// t = (x - m) unit is split into a whole k and |t - k| <= 1/2, and the result is
// 2^(k / 256) from a table times a Taylor polynomial (the next term is below 2^-54):
// the table-driven method of Tang (1989).  k is whole by the addition of 1.5 * 2^52,
// whose low word then holds it; conversions and roundings of 64 bits run at a
// quarter of an add's rate.  What is below 2^-1000 counts as that, or as 0: t is
// compared in 64 bits, since fp32 need not have a logit that lies as far below m
// (3e9 has neighbours 256 apart).  12 operations in 64 bits, of which an SM does 64 a
// cycle.
struct Exp64 {
  const double* table;  // in shared memory
  double unit, md;
  __device__ __forceinline__ Exp64(const double* table, const VerifyArgs& a, float m) : table(table), unit(a.unit) {
    md = m == -INFINITY ? 0.0 : (double)m;
  }
  __device__ __forceinline__ double at(double t) const {
    constexpr double c = 0.0027076061740622863, magic = 6755399441055744.0;  // ln 2 / 256
    const double s = t + magic;
    const int i = __double2loint(s);
    const double r = t - (s - magic);
    double p = fma(r, c * c * c * c / 24, c * c * c / 6);
    p = fma(r, p, c * c / 2);
    p = fma(r, p, c);
    p = fma(r, p, 1.0);
    p *= table[i & 255];
    return __hiloint2double(__double2hiint(p) + ((i & ~255) << 12), __double2loint(p));
  }
  static constexpr double LEAST = -256000.0;
  __device__ __forceinline__ double operator()(float x) const {
    const double t = ((double)x - md) * unit;
    return at(t < LEAST ? LEAST : t);  // NaN stays
  }
  __device__ __forceinline__ double or_zero(float x) const {
    const double t = ((double)x - md) * unit;
    return t < LEAST ? 0.0 : at(t);
  }
};
__device__ __forceinline__ void fill_table(double* table) { table[threadIdx.x] = TWO_TO_256THS[threadIdx.x]; }
static_assert(THREADS == 256, "the table");
__device__ __forceinline__ float load_logit(const float* p) {  // +inf is the largest value there is
  const float x = __ldcg(p);
  return x > TOP ? TOP : x;
}
__device__ __forceinline__ float warp_max(float m) {
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}
__device__ __forceinline__ double warp_sum(double s) {
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
// PER values per thread: 8 where the rows' CTAs would not fill the SMs, else 32.
template <int PER>
__global__ void __launch_bounds__(THREADS) verify_stat_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ double table[256];
  __shared__ double2 s_part[WARPS];
  pdl_launch_dependents();
  fill_table(table);
  __syncthreads();
  pdl_wait();
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  if (row >= __ldcg(a.starts + a.requests)) return;
  const float* src = a.logits + row * a.ld;
  const int64_t i0 = (int64_t)blockIdx.x * (THREADS * PER) + tid;
  float x[PER], m = -INFINITY;
  if (((int64_t)blockIdx.x + 1) * (THREADS * PER) <= a.V) {
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] = __ldcg(src + i0 + k * THREADS);
  } else {
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] = i0 + k * THREADS < a.V ? __ldcg(src + i0 + k * THREADS) : -INFINITY;
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) m = fmaxf(m, x[k]);
  m = warp_max(m);  // each warp for itself, so that one barrier is enough
  if (m > TOP) {    // +inf is the largest value there is
    m = TOP;
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] = x[k] > TOP ? TOP : x[k];
  }
  const Exp64 ex(table, a, m);
  double sum[2] = {0.0, 0.0};
#pragma unroll
  for (int k = 0; k < PER; ++k) sum[k & 1] += ex(x[k]);
  const double s = warp_sum(sum[0] + sum[1]);
  if (lane == 0) s_part[tid >> 5] = make_double2(m, m == -INFINITY && s == s ? 0.0 : s);
  __syncthreads();
  if (tid < 32) {
    const double2 v = s_part[lane & (WARPS - 1)];
    const float top = warp_max((float)v.x);
    const double z = warp_sum(lane < WARPS && v.y != 0.0 ? v.y * Exp64(table, a, top)((float)v.x) : 0.0);
    if (tid == 0) a.stat[(int64_t)row * a.stats + blockIdx.x] = make_double2(top, z);
  }
}

template <int PER>
__global__ void __launch_bounds__(THREADS) verify_draw_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ double table[256], s_sum[WARPS], s_max[WARPS], s_z[WARPS];
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
  // ---- the row where the drafts end: a warp per row
  int at = end - 1;
  double z = 0.0, m = 0.0;
  for (int r0 = start;; r0 += WARPS) {
    const int r = r0 + warp;
    if (r < end) {
      // the draft that the row judges, on its way while the sums are folded
      const int x = r + 1 < end ? __ldcg(a.tokens + r + 1) : -1;
      const bool judged = x >= 0 && x < a.V;
      const float lx = judged ? load_logit(a.logits + r * a.ld + x) : 0.f, u = __ldcg(a.u_accept + r);
      const double q = judged && a.probs ? (double)__ldcg(a.probs + r * a.ld_p + x) : 1.0;
      const double2* st = a.stat + (int64_t)r * a.stats;
      float top = -INFINITY;
      double z_all = 0.0;
      for (int i0 = 0; i0 < a.stats; i0 += 32) {
        const double2 v = i0 + lane < a.stats ? __ldcg(st + i0 + lane) : make_double2(-INFINITY, 0.0);
        const float now = fmaxf(top, warp_max((float)v.x));
        const Exp64 ex(table, a, now);
        if (z_all != 0.0 && now != top) z_all *= ex(top);
        z_all += v.y != 0.0 ? v.y * ex((float)v.x) : 0.0;
        top = now;
      }
      const double wz = warp_sum(z_all), wm = top;
      if (lane == 0) {
        const int keep = judged && wz > 0.0 && (double)u * q < Exp64(table, a, top).or_zero(lx) / wz;
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
  const int draft = at + 1 < end && !a.probs ? __ldcg(a.tokens + at + 1) : -1;
  const float *src = a.logits + at * a.ld, *qsrc = a.probs && at + 1 < end ? a.probs + at * a.ld_p : nullptr;
  const double inv = 1.0 / z;
  const Exp64 ex(table, a, (float)m);
  // (max(p - q, 0), p) of an id with logit x and the drafter's probability q
  auto weigh = [&](float x, float q) {
    const double p = ex.or_zero(x > TOP ? TOP : x) * inv;
    return make_double2(fmax(p - (double)q, 0.0), p);
  };
  // the thread's ids of a slice: THREADS apart
  float x[PER], q[PER];
  auto fetch = [&](int slice) {
    const int64_t i0 = (int64_t)slice * (THREADS * PER) + tid;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int64_t i = i0 + k * THREADS;
      x[k] = i < a.V ? __ldcg(src + i) : -INFINITY;
      q[k] = i < a.V && qsrc ? __ldcg(qsrc + i) : i == draft ? 1.f : 0.f;
    }
  };
  double rest = 0.0, all = 0.0;
  if (!none) {
    fetch(blockIdx.x);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const double2 w = weigh(x[k], q[k]);
      rest += w.x, all += w.y;
    }
  }
  rest = warp_sum(rest), all = warp_sum(all);
  if (lane == 0) s_z[warp] = rest, s_max[warp] = all;
  __syncthreads();
  if (tid == 0) {
    rest = all = 0.0;
    for (int w = 0; w < WARPS; ++w) rest += s_z[w], all += s_max[w];
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
  // weights in shared memory, then a run of ids per thread (a place in between, or a
  // warp's runs would start in the same banks)
  __shared__ double s_w[THREADS * (PER + 1)];
  const bool use = s_use;
  fetch(s_slice);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const double2 y = weigh(x[k], q[k]);
    const int at_k = k * THREADS + tid;
    s_w[at_k + at_k / PER] = use ? y.x : y.y;
  }
  __syncthreads();
  const int64_t i0 = (int64_t)s_slice * (THREADS * PER) + tid * PER;
  double w[PER], sum = 0.0;
#pragma unroll
  for (int k = 0; k < PER; ++k) w[k] = s_w[tid * (PER + 1) + k], sum += w[k];
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
  for (int k = 0; k < PER; ++k) {
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
  const int64_t n = 4ll * requests, logit_bytes = 4 * ((rows - 1) * ld + V), prob_bytes = 4 * ((rows - 1) * ld_probs + V);
  for (const void* out : {d_accepted, d_next})
    if (bytes_overlap(out, n, d_tokens, 4ll * rows) || bytes_overlap(out, n, d_starts, n + 4) || bytes_overlap(out, n, d_u_accept, 4ll * rows) ||
        bytes_overlap(out, n, d_u_next, n) || bytes_overlap(out, n, d_logits, logit_bytes) || bytes_overlap(out, n, d_draft_probs, prob_bytes) ||
        bytes_overlap(out, n, d_scratch, (int64_t)scratch_bytes))
      return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "verify_sampled: an output overlaps what the call reads or its scratch");
  if (bytes_overlap(d_accepted, n, d_next, n)) return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "verify_sampled: the outputs overlap");
  VerifyArgs a{};
  a.logits = d_logits, a.ld = ld, a.tokens = d_tokens, a.starts = d_starts, a.probs = d_draft_probs, a.ld_p = ld_probs;
  a.u_accept = d_u_accept, a.u_next = d_u_next, a.accepted = d_accepted, a.next = d_next;
  a.requests = requests, a.rows = rows, a.V = V;
  a.unit = 369.3299304757364 / temperature;  // 256 / ln 2
  a.count = static_cast<int*>(d_scratch);
  a.stat = reinterpret_cast<double2*>(static_cast<uint8_t*>(d_scratch) + COUNT_BYTES);
  a.part = a.stat + (int64_t)rows * slices_of(V);
  cudaStream_t s = (cudaStream_t)stream;
  // more ids of a row per CTA where 2048 would be more CTAs than the SMs hold at once
  auto pieces = [&](int per) { return (int)((V + THREADS * per - 1) / (THREADS * per)); };
  const bool sums = (int64_t)pieces(VPT) * rows > 148 * 8, draws = (int64_t)pieces(VPT) * requests > 148 * 3;
  a.stats = pieces(sums ? 4 * VPT : VPT), a.slices = pieces(draws ? 2 * VPT : VPT);
  cudaError_t e = sums ? launch_pdl(verify_stat_kernel<4 * VPT>, dim3(a.stats, rows), dim3(THREADS), s, a)
                       : launch_pdl(verify_stat_kernel<VPT>, dim3(a.stats, rows), dim3(THREADS), s, a);
  if (e == cudaSuccess)
    e = draws ? launch_pdl(verify_draw_kernel<2 * VPT>, dim3(a.slices, requests), dim3(THREADS), s, a)
              : launch_pdl(verify_draw_kernel<VPT>, dim3(a.slices, requests), dim3(THREADS), s, a);
  return kv_launched(e, "verify_sampled");
}

}  // extern "C"
