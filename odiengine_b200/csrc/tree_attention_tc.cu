// tree_attention_tc.cu -- tree attention for many rows per kv head on the
// sm_100a tensor cores (tcgen05.mma, accumulators in tensor memory).
//
// The same mathematics, row numbering and splits as tree_attention.cu, for
// head_dim 128 and more rows than one warp's tile holds.  A CTA takes 32 or 64 rows
// (two groups of 16 or 32) of one kv head and every nsplit-th block of 128
// positions:
//
//   S^T [128 positions x NT rows] = K . Q^T     positions as M
//   O^T [128 dims x NT rows]     += V^T . P^T   dims as M
//
// With the cache as the M side every instruction is full whatever the number
// of rows, K and V are used as TMA leaves them in shared memory (K as a
// K-major operand, V, the same bytes order, as an MN-major one), and each is
// fetched once for all the CTA's rows.
//
// fp32 results from 16- and 8-bit products, as columns of one instruction:
//  * int8 cache (kind::i8, exact 32-bit integer sums): q is fixed point in
//    three signed digits (3 NT columns), P * (V's row scale) fixed point in four
//    unsigned digits (4 NT columns): an integer up to 2^32 in units of 2^-24 of
//    the largest weight.
//  * fp16 cache (kind::f16): q and P are each the sum of two fp16 values (2 NT
//    columns); the high and low halves' sums are added in fp32.
//
//   warp 0       TMA producer: tiles K0 K1 V0 K2 V1 ... through one ring
//   warps 1, 2   issue the products, one warp for each group of rows; warp 1
//                holds the tensor memory
//   warps 4-7    the first group: thread = position (tensor memory lane) in the
//   warps 8-11   softmax, = dim when O is read; the second group
//
// While one group of rows is in its softmax the tensor core works for the
// other.  As in tree_attention.cu m is a reference that moves only when a
// weight would leave its range; then (and every few blocks, so that integer
// sums cannot overflow and fp32 sums stay short) O moves from tensor memory
// to fp32 registers and starts again.
//
// Every wait is bounded; a wait that gives up sets the error word, all roles
// leave their loops, copies in flight are waited for and the tensor memory is
// released.
#include <cuda.h>
#include <math.h>

#include "tree_attention.cuh"

namespace odi_cuda {
namespace ttc {

constexpr int HD = 128;
constexpr int BK = 128;  // positions per block
constexpr int ERR_TREE_WAIT = 64;

template <bool I8, int NT>
struct Cfg {
  static constexpr int SUBS = 2;
  static constexpr int DQ = I8 ? 3 : 2, DP = I8 ? 4 : 2;  // digits of q and P
  static constexpr int TILE = BK * HD * (I8 ? 1 : 2);     // K or V of one block
  static constexpr int SLOTS = I8 ? 8 : 4;
  static constexpr int QB = DQ * NT * HD * (I8 ? 1 : 2);
  static constexpr int PB = BK * 128;                     // one 128-byte row per position
  static constexpr int Q_OFF = SLOTS * TILE;
  static constexpr int P_OFF = Q_OFF + SUBS * QB;
  static constexpr int SMEM = P_OFF + SUBS * PB + 1024;   // + alignment slack
  static constexpr int THREADS = 128 + 128 * SUBS;
  static constexpr int ROWS = NT * SUBS;
  static constexpr int SCOLS = DQ * NT, OCOL = (I8 ? 4 : 2) * NT, SUBCOLS = 2 * OCOL;
  static constexpr int TMEM_COLS = SUBCOLS * SUBS;
  // blocks between two moves of O to registers: 255 * 127 * 128 * 256 < 2^31;
  // the fp32 accumulator truncates, about 2^-26 of the sum per instruction
  static constexpr int PERIOD = I8 ? 256 : 4;
  static_assert(ROWS * HD * 4 <= SLOTS * TILE, "the joins' shares reuse the ring");
  static_assert(SMEM <= 222 * 1024, "shared memory, beside the static part");
};

// Shared-memory matrix descriptors, 128-byte swizzle.  K-major: rows of 128
// bytes, groups of 8 rows 1024 bytes apart.  MN-major: K rows of 128 bytes of
// the M or N side, groups of 8 K rows 1024 bytes apart, further 128-byte
// pieces of the M side `lbo` bytes apart.
__device__ __forceinline__ uint64_t desc(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
constexpr uint32_t IDESC_M128 = 8u << 24;
__host__ __device__ constexpr uint32_t idesc(bool i8, bool mn, int n) {
  // D: fp32 (1) or s32 (2) | A, B: f16 (0), or A s8 (1) and B s8 (1; P's digits u8: 0) | both MN-major
  return ((i8 ? 2u : 1u) << 4) | (i8 ? 1u << 7 : 0u) | (i8 && !mn ? 1u << 10 : 0u) | (mn ? 3u << 15 : 0u) |
         ((uint32_t)(n >> 3) << 17) | IDESC_M128;
}
template <bool I8>
__device__ __forceinline__ void mma(uint32_t d, uint64_t ad, uint64_t bd, uint32_t id, uint32_t accumulate) {
  if (I8)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(ad), "l"(bd), "r"(id), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(ad), "l"(bd), "r"(id), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}
// 32 lanes x 16 consecutive columns; complete only after ld_wait.
__device__ __forceinline__ void ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
// The registers of the loads before it pass through, so no use moves ahead of it.
template <int N>
__device__ __forceinline__ void ld_wait(uint32_t (&r)[N][16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(r[k][i]));
}
__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void group_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ bool group_any(int id, int n, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
      "bar.red.or.pred p, %2, %3, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "r"(id), "r"(n)
      : "memory");
  return r != 0;
}
// h * 2^16 + m * 2^8 + l of digit sums below 2^22 in size, as fp32.  Each gets
// the exponent of 1.5 * 2^23 by an integer add (the conversion instruction runs
// at an eighth of the rate); m and l are joined first, to a multiple of 2^8:
// 2^-22 of a product of ordinary size, which is 2^29 and more.
__device__ __forceinline__ float join_digits(uint32_t h, uint32_t m, uint32_t l) {
  constexpr float B = 12582912.f;
  const float hf = __uint_as_float(h + 0x4B400000u) - B;
  const float ml = fmaf(__uint_as_float(m + 0x4B400000u), 256.f, __uint_as_float(l + 0x4B400000u)) - B * 257.f;
  return fmaf(hf, 65536.f, ml);
}
// fp32 -> unsigned with the same order
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

template <int SUBS>
struct Bars {
  uint64_t tfull[8], tfree[8];
  uint64_t s_full[SUBS], s_free[SUBS], p_full[SUBS], pv_done[SUBS];
  uint64_t v_clean[2];
};
// What a group's threads share about its rows.
template <int NT>
struct alignas(16) Group {
  float c[NT];    // factor of the scores
  float m[NT];    // reference
  float lv[NT];   // log2 of vs
  float vs[NT];   // factor of the weights (int8: of weight * scale)
  float fo[NT], fl[NT];  // factors of O and of the sums when the reference moves
  uint32_t mx[4][32], dm[4][32], need[4];
  float lv_top;          // the largest lv
  int lv_same;           // all lv are equal
};

template <bool I8, int NT>
__global__ void __launch_bounds__(Cfg<I8, NT>::THREADS, 1)
    tree_tc_kernel(const TreeArgs a, int* err, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap) {
  using F = Cfg<I8, NT>;
  constexpr int SUBS = F::SUBS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ Bars<SUBS> bars;
  __shared__ Group<NT> groups[SUBS];
  __shared__ int rowt[F::ROWS];
  __shared__ float2 cta_ml[F::ROWS];
  __shared__ uint32_t tmem_slot;
  __shared__ int restart[SUBS];
  __shared__ int dead;  // a wait gave up
  __shared__ uint8_t bad_row[2][BK];  // fp16: V rows taken out of the last two tiles that hold tree slots
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = blockIdx.x, tile = blockIdx.y, split = blockIdx.z;
  const int C = (int)cluster_nranks(), rank = (int)cluster_rank_of();

  pdl_launch_dependents();
  if (tid == 0) {
    for (int i = 0; i < 8; ++i) mbar_init(&bars.tfull[i], 1), mbar_init(&bars.tfree[i], SUBS);
    for (int i = 0; i < SUBS; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.s_free[i], 128);
      mbar_init(&bars.p_full[i], 128);
      mbar_init(&bars.pv_done[i], 1);
    }
    mbar_init(&bars.v_clean[0], 128);
    mbar_init(&bars.v_clean[1], 128);
    dead = 0;
    fence_mbar_init();
  }
  pdl_wait();
  const int pos = __ldcg(&a.st->pos);
  const int len = (int)max(0ll, min((long long)a.c.ctx, (long long)pos + a.tokens));
  const int nblocks = (len + BK - 1) / BK;
  // the host splits for a full cache: clusters that the length at hand leaves without a block go
  const int nclusters = max(1, min(a.nsplit / C, (nblocks + C - 1) / C));
  if (split >= nclusters * C) return;
  const int stride = nclusters * C;
  const int nb = nblocks > split ? (nblocks - split + stride - 1) / stride : 0;  // this CTA's blocks
  const int64_t head = (int64_t)kvh * a.c.ctx;
  const int seqs = 2 * nb;                     // tiles K0 K1 V0 K2 V1 ...
  auto vseq = [&](int i) { return min(2 * i + 2, 2 * nb - 1); };
  auto kseq = [&](int i) { return i ? 2 * i - 1 : 0; };

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"(F::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // ---- Q: digits as K-major operand rows n' = digit * 32 + n
  {
    constexpr int NW = F::THREADS / 32, RW = (F::ROWS + NW - 1) / NW;
    float v[RW][4];
    int rt[RW];
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const int n = warp + i * NW, r = tile * F::ROWS + n;
      const bool in = n < F::ROWS && r < a.R;
      rt[i] = in ? r / a.G : -1;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = 0.f;
      if (in) {
        const float* src = a.q + (int64_t)rt[i] * a.ld_q + (int64_t)(kvh * a.G + r - rt[i] * a.G) * HD + lane * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][e] = __ldcg(src + e);
      }
    }
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const int n = warp + i * NW;
      if (n >= F::ROWS) break;
      float am = 0.f;
      bool ok = true;
#pragma unroll
      for (int e = 0; e < 4; ++e) am = fmaxf(am, fabsf(v[i][e])), ok = ok && finite(v[i][e]);
#pragma unroll
      for (int x = 16; x; x >>= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, x));
      ok = __all_sync(0xffffffffu, ok);
      int ex = (int)(__float_as_uint(am) >> 23) - 127;
      if (I8 && am * pow2(-min(max(ex, -100), 126)) > 1.99f) ++ex;
      ex = min(max(ex, -100), 126);
      const float lift = pow2(-ex), up = I8 ? 4194304.f : 8192.f;
      const int sub = n / NT, ln = n % NT;
      if (lane == 0) {
        Group<NT>& gr = groups[sub];
        gr.c[ln] = ok ? a.scale_log2 * (1.f / up) * pow2(ex) : __int_as_float(0x7fc00000);
        gr.m[ln] = TA_NONE;
        gr.lv[ln] = I8 ? 120.f : 4.f;
        gr.vs[ln] = I8 ? TA_VMOST : 16.f;
        gr.fo[ln] = gr.fl[ln] = 1.f;
        if (ln == 0) gr.lv_top = I8 ? 120.f : 4.f, gr.lv_same = 1;
        rowt[n] = rt[i];
      }
      uint8_t* q = smem + F::Q_OFF + sub * F::QB;
      if (I8) {
        int dig[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) dig[e] = ok ? __float2int_rn(v[i][e] * lift * up) : 0;
#pragma unroll
        for (int k = F::DQ - 1; k >= 0; --k) {  // digit 0 the highest
          uint32_t bytes = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int lo = (int)(int8_t)(dig[e] & 255);
            dig[e] = (dig[e] - lo) >> 8;
            bytes |= (uint32_t)(lo & 255) << (8 * e);
          }
          const int row = k * NT + ln;
          *reinterpret_cast<uint32_t*>(q + row * 128 + (((lane >> 2) ^ (row & 7)) << 4) + (lane & 3) * 4) = bytes;
        }
      } else {
        uint32_t w[2][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x0 = ok ? v[i][2 * e] * lift * up : 0.f, x1 = ok ? v[i][2 * e + 1] * lift * up : 0.f;
          const __half2 hi = __floats2half2_rn(x0, x1);
          const float2 back = __half22float2(hi);
          w[0][e] = h2u(hi);
          w[1][e] = h2u(__floats2half2_rn(x0 - back.x, x1 - back.y));
        }
#pragma unroll
        for (int k = 0; k < F::DQ; ++k) {  // two pieces of 64 dims, each [64 rows][128 bytes]
          const int row = k * NT + ln, d = lane * 4;
          *reinterpret_cast<uint2*>(q + (d >> 6) * (F::DQ * NT * 128) + row * 128 + ((((d & 63) >> 3) ^ (row & 7)) << 4) + (d & 7) * 2) =
              make_uint2(w[k][0], w[k][1]);
        }
      }
    }
  }
  fence_proxy_async_smem();
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;

  float facc[NT], l[NT];
  if (warp == 0) {
    // ---------------- producer ----------------
    if (lane == 0) {
      int t = 0;
      for (; t < seqs; ++t) {
        const int slot = t % F::SLOTS;
        if (!mbar_wait(&bars.tfree[slot], ((t / F::SLOTS) & 1) ^ 1, err, ERR_TREE_WAIT)) {
          dead = 1;
          break;
        }
        const bool isk = t == 0 || (t == seqs - 1 ? false : (t & 1));
        const int i = t == 0 ? 0 : isk ? (t + 1) / 2 : t == seqs - 1 ? nb - 1 : t / 2 - 1;
        const int row = (int)(head + (int64_t)(split + i * stride) * BK);
        uint8_t* dst = smem + slot * F::TILE;
        mbar_arrive_expect_tx(&bars.tfull[slot], F::TILE);
        const CUtensorMap* map = isk ? &kmap : &vmap;
        tma_2d(dst, map, 0, row, &bars.tfull[slot]);
        if (!I8) tma_2d(dst + F::TILE / 2, map, 64, row, &bars.tfull[slot]);
      }
      // every issued copy has landed before the CTA can retire
      for (int u = t < F::SLOTS ? 0 : t - F::SLOTS; u < t; ++u)
        mbar_wait(&bars.tfull[u % F::SLOTS], (u / F::SLOTS) & 1, err, ERR_TREE_WAIT);
    }
  } else if (warp <= SUBS) {
    // ---------------- products ----------------
    // The whole warp runs the loop, so that descriptors stay in uniform
    // registers, and one elected thread issues: issued from a lane's branch,
    // with its operands moved there one by one, an instruction took 170 cycles.
    const int u = warp - 1;  // one warp for each group of rows: neither waits for the other's softmax
    const uint32_t q0 = smem_u32(smem + F::Q_OFF + u * F::QB), p0 = smem_u32(smem + F::P_OFF + u * F::PB), t0 = smem_u32(smem);
    const uint64_t qd0 = desc(q0, 16), pd0 = desc(p0, 16), kd0 = desc(t0, 16), vd0 = desc(t0, I8 ? 16 : F::TILE / 2);
    bool ok = true;
    auto wait = [&](uint64_t* bar, int n) {
      ok = ok && mbar_wait(bar, n & 1, err, ERR_TREE_WAIT);
      ok = __all_sync(0xffffffffu, ok);
    };
    auto scores = [&](int i) {
      const int t = kseq(i), slot = t % F::SLOTS;
      wait(&bars.tfull[slot], t / F::SLOTS);
      if (i) wait(&bars.s_free[u], i - 1);
      if (!ok) return;
      fence_after();
      if (elect_one()) {
        const uint64_t kd = kd0 + (uint32_t)(slot * (F::TILE >> 4));
#pragma unroll
        for (int k = 0; k < (I8 ? 4 : 8); ++k)  // 32 bytes of the contraction per instruction
          mma<I8>(tmem + u * F::SUBCOLS, kd + (k >> 2) * (F::TILE / 2 >> 4) + 2 * (k & 3),
                  qd0 + (k >> 2) * (F::DQ * NT * 128 >> 4) + 2 * (k & 3), idesc(I8, false, F::SCOLS), k != 0);
        commit(&bars.s_full[u]);
        commit(&bars.tfree[slot]);
      }
      __syncwarp();
    };
    if (nb) scores(0);
    for (int i = 0; i < nb && ok; ++i) {
      if (i + 1 < nb) scores(i + 1);
      const int t = vseq(i), slot = t % F::SLOTS;
      wait(&bars.tfull[slot], t / F::SLOTS);
      wait(&bars.p_full[u], i);
      if (!ok) break;
      fence_after();
      const uint32_t keep = *reinterpret_cast<volatile int*>(&restart[u]) == 0;
      if (elect_one()) {
        const uint64_t vd = vd0 + (uint32_t)(slot * (F::TILE >> 4));
        constexpr int KS = I8 ? 4 : 8, KB = BK / KS * 128;  // bytes of 32 or 16 positions
#pragma unroll
        for (int k = 0; k < KS; ++k)
          mma<I8>(tmem + u * F::SUBCOLS + F::OCOL, vd + k * (KB >> 4), pd0 + k * (KB >> 4), idesc(I8, true, F::DP * NT),
                  k ? 1u : keep);
        commit(&bars.pv_done[u]);
        commit(&bars.tfree[slot]);
      }
      __syncwarp();
    }
    if (!ok) dead = 1;
  } else if (warp >= 4) {
    // ---------------- softmax ----------------
    const int sub = (warp >> 2) - 1, wq = warp & 3, kl = wq * 32 + lane, bar = 1 + sub;
    Group<NT>& gr = groups[sub];
    const uint32_t s_tm = tmem + sub * F::SUBCOLS + ((uint32_t)(wq * 32) << 16), o_tm = s_tm + F::OCOL;
    uint8_t* prow = smem + F::P_OFF + sub * F::PB + kl * 128;
    const float* ks = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.c.k) + a.c.scale_off) + head;
    const float* vsc = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.c.v) + a.c.scale_off) + head;
    const float nan = __int_as_float(0x7fc00000);
#pragma unroll
    for (int n = 0; n < NT; ++n) facc[n] = 0.f, l[n] = 0.f;
    float dk = 0.f, dv = 0.f, dk_next = 0.f, dv_next = 0.f;
    auto request = [&](int i) {
      const int key = min((split + i * stride) * BK + kl, len - 1);
      dk_next = __ldcg(ks + key), dv_next = __ldcg(vsc + key);
    };
    if (I8 && nb) request(0);
    // O's sums so far, out of tensor memory
    auto flush = [&](int i, bool moved) {
      if (i) {
        if (!mbar_wait(&bars.pv_done[sub], (i - 1) & 1, err, ERR_TREE_WAIT)) dead = 1;
        __syncwarp();
        fence_after();
#pragma unroll
        for (int c0 = 0; c0 < NT; c0 += 16) {
          uint32_t r[F::DP][16];
#pragma unroll
          for (int k = 0; k < F::DP; ++k) ld16(o_tm + k * NT + c0, r[k]);
          ld_wait(r);
#pragma unroll
          for (int n = 0; n < 16; ++n) {
            float x;
            if (I8)  // digit 0 the lowest
              x = fmaf((float)(int)r[F::DP - 1][n], 16777216.f,
                       fmaf((float)(int)r[F::DP - 2][n], 65536.f, fmaf((float)(int)r[1][n], 256.f, (float)(int)r[0][n])));
            else
              x = __uint_as_float(r[0][n]) + __uint_as_float(r[1][n]);
            facc[c0 + n] += x;
          }
        }
        fence_before();
      }
      if (moved)
#pragma unroll
        for (int n = 0; n < NT; ++n) facc[n] *= gr.fo[n], l[n] *= gr.fl[n];
    };
    int since = 0, edges = 0;
    for (int i = 0; i < nb; ++i) {
      const int p0 = (split + i * stride) * BK, key = p0 + kl;
      if (I8) {
        dk = dk_next, dv = dv_next;
        if (i + 1 < nb) request(i + 1);
      }
      bool ok = mbar_wait(&bars.s_full[sub], i & 1, err, ERR_TREE_WAIT);
      __syncwarp();
      fence_after();
      float s[NT];
      // a row whose scale of K or V is not finite gives NaN to who sees it
      const float dkk = finite(dk) && finite(dv) ? dk : nan, dvv = finite(dv) ? dv : 0.f;
#pragma unroll
      for (int c0 = 0; c0 < NT; c0 += 16) {
        uint32_t r[F::DQ][16];
#pragma unroll
        for (int k = 0; k < F::DQ; ++k) ld16(s_tm + k * NT + c0, r[k]);
        ld_wait(r);
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          if (I8)
            s[c0 + n] = join_digits(r[0][n], r[1][n], r[F::DQ - 1][n]) * dkk;
          else
            s[c0 + n] = __uint_as_float(r[0][n]) + __uint_as_float(r[1][n]);
        }
      }
      fence_before();
      mbar_arrive(&bars.s_free[sub]);
      uint32_t vis = 0xffffffffu;  // bit n: row n sees this position
      if (p0 + BK > min(pos, len)) {  // holds tree slots, or ends past the last
        bool bad = false;
        if (!I8) {
          // V rows that are past the end or not finite leave the tile; who
          // sees such a row gets NaN through its score, nobody else meets it.
          // The first group does it and the second waits: two such tiles on, the
          // first is held until the second group's products on this one are done
          // (the tile's slot).
          if (sub == 0) {
            const int t = vseq(i), slot = t % F::SLOTS;
            ok = mbar_wait(&bars.tfull[slot], (t / F::SLOTS) & 1, err, ERR_TREE_WAIT) && ok;
            uint8_t* vrow = smem + slot * F::TILE + kl * 128;
            bad = key >= len;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const uint4 x = *reinterpret_cast<const uint4*>(vrow + (e >> 3) * (F::TILE / 2) + (e & 7) * 16);
              const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int j = 0; j < 4; ++j) bad = bad || (w[j] & 0x7c00u) == 0x7c00u || (w[j] & 0x7c000000u) == 0x7c000000u;
            }
            if (bad)
#pragma unroll
              for (int e = 0; e < 16; ++e)
                *reinterpret_cast<uint4*>(vrow + (e >> 3) * (F::TILE / 2) + (e & 7) * 16) = make_uint4(0, 0, 0, 0);
            bad_row[edges & 1][kl] = bad;
            fence_proxy_async_smem();
            mbar_arrive(&bars.v_clean[edges & 1]);
          } else {
            ok = mbar_wait(&bars.v_clean[edges & 1], (edges >> 1) & 1, err, ERR_TREE_WAIT) && ok;
            bad = bad_row[edges & 1][kl];
          }
          ++edges;
        }
        // lane n: which of the warp's 32 positions row n sees; then its transpose
        const uint32_t rowsee = lane < NT ? seen_bits(a, rowt[sub * NT + lane], p0 + wq * 32, pos, len) : 0u;
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const uint32_t b = __ballot_sync(0xffffffffu, (rowsee >> k) & 1u);
          if (lane == k) vis = b;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (!((vis >> n) & 1u)) s[n] = -INFINITY;
          else if (!I8 && bad) s[n] = nan;
        }
      }
      // does a weight leave its range?  int8: digits hold weight * scale * vs
      // below 2^32 (lv_top is the bound of every row's vs)
      constexpr float TOP = I8 ? 31.f : 11.f;
      const float ldv = I8 ? __log2f(dvv) : 0.f;
      float top = -INFINITY;
#pragma unroll
      for (int n = 0; n < NT; n += 4) {
        const float4 c4 = *reinterpret_cast<const float4*>(&gr.c[n]), m4 = *reinterpret_cast<const float4*>(&gr.m[n]);
        top = fmaxf(top, fmaxf(fmaf(s[n], c4.x, -m4.x), fmaf(s[n + 1], c4.y, -m4.y)));
        top = fmaxf(top, fmaxf(fmaf(s[n + 2], c4.z, -m4.z), fmaf(s[n + 3], c4.w, -m4.w)));
      }
      if (I8) top += fmaxf(-29.f, ldv + gr.lv_top);
      if (!ok) dead = 1;
      bool fresh = i == 0;
      __syncwarp();
      if (group_any(bar, 128, top > TOP || !ok)) {
        if (group_any(bar, 128, *reinterpret_cast<volatile int*>(&dead) != 0)) break;
        uint32_t mx = 0, dm = 0, need = 0;
        const uint32_t dvb = I8 ? __float_as_uint(dvv) : 0u;
#pragma unroll
        for (int n = 0; n < NT; ++n) {  // lane n keeps row n
          const float sn = s[n] * gr.c[n], x = fmaf(s[n], gr.c[n], -gr.m[n]);
          const bool over = (I8 ? x + fmaxf(-29.f, ldv + gr.lv[n]) : x) > TOP;
          const uint32_t hi = __reduce_max_sync(0xffffffffu, sn == sn ? ordered(sn) : 0u);
          const uint32_t dmn = I8 ? __reduce_max_sync(0xffffffffu, (vis >> n) & 1u ? dvb : 0u) : 0u;
          if (__any_sync(0xffffffffu, over)) need |= 1u << n;
          if (lane == n) mx = hi, dm = dmn;
        }
        gr.mx[wq][lane] = mx;
        gr.dm[wq][lane] = dm;
        if (lane == 0) gr.need[wq] = need;
        group_sync(bar, 128);
        if (wq == 0) {
          if (lane < NT) {
            const int n = lane;
            float fo = 1.f, fl = 1.f;
            if (((gr.need[0] | gr.need[1] | gr.need[2] | gr.need[3]) >> n) & 1u) {  // each row by itself
              const float mn = fmaxf(gr.m[n], unordered(max(max(gr.mx[0][n], gr.mx[1][n]), max(gr.mx[2][n], gr.mx[3][n]))));
              fo = fl = ex2(gr.m[n] - mn);
              gr.m[n] = mn;
              if (I8) {
                const uint32_t d = max(max(gr.dm[0][n], gr.dm[1][n]), max(gr.dm[2][n], gr.dm[3][n]));
                const int ex = max((int)(d >> 23) - 126, -96);  // a power of two above the largest scale
                if (d && (float)(24 - ex) < gr.lv[n]) {
                  const float nv = pow2(24 - ex);
                  fo *= nv / gr.vs[n];
                  gr.vs[n] = nv;
                  gr.lv[n] = (float)(24 - ex);
                }
              }
            }
            gr.fo[n] = fo, gr.fl[n] = fl;
          }
          __syncwarp();
          if (I8) {
            float hi = gr.lv[lane % NT], lo = hi;
#pragma unroll
            for (int x = 16; x; x >>= 1) {
              hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, x));
              lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, x));
            }
            if (lane == 0) gr.lv_top = hi, gr.lv_same = hi == lo;
          }
        }
        group_sync(bar, 128);
        flush(i, true);
        fresh = true;
      } else if (since >= F::PERIOD) {
        flush(i, false);
        fresh = true;
      }
      since = fresh ? 1 : since + 1;
      // weights, as digits, into the operand tile
      if (i && !mbar_wait(&bars.pv_done[sub], (i - 1) & 1, err, ERR_TREE_WAIT)) dead = 1;
      if (I8) {
        const float dvs = dvv * gr.vs[0];
        const bool same = gr.lv_same;
#pragma unroll
        for (int c0 = 0; c0 < NT; c0 += 16) {
          uint32_t w[4][4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int n0 = c0 + 4 * q;
            const float4 c4 = *reinterpret_cast<const float4*>(&gr.c[n0]), m4 = *reinterpret_cast<const float4*>(&gr.m[n0]);
            const float cc[4] = {c4.x, c4.y, c4.z, c4.w}, mm[4] = {m4.x, m4.y, m4.z, m4.w};
            float f[4] = {dvs, dvs, dvs, dvs};
            if (!same) {
              const float4 v4 = *reinterpret_cast<const float4*>(&gr.vs[n0]);
              f[0] = dvv * v4.x, f[1] = dvv * v4.y, f[2] = dvv * v4.z, f[3] = dvv * v4.w;
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float p = ex2(fmaf(s[n0 + e], cc[e], -mm[e]));
              l[n0 + e] += p;
              const float x = fmaf(p, f[e], 0.5f);  // 0.5 .. 2^32: its integer part is the weight
              const float h = __fmaf_rz(x, 0x1p-16f, 8388608.f);
              hi[e] = __float_as_uint(h);
              lo[e] = __float_as_uint(__fadd_rz(fmaf(-65536.f, h - 8388608.f, x), 8388608.f));
            }
            const uint32_t l01 = __byte_perm(lo[0], lo[1], 0x5140u), l23 = __byte_perm(lo[2], lo[3], 0x5140u);
            const uint32_t h01 = __byte_perm(hi[0], hi[1], 0x5140u), h23 = __byte_perm(hi[2], hi[3], 0x5140u);
            w[0][q] = __byte_perm(l01, l23, 0x5410u);
            w[1][q] = __byte_perm(l01, l23, 0x7632u);
            w[2][q] = __byte_perm(h01, h23, 0x5410u);
            w[3][q] = __byte_perm(h01, h23, 0x7632u);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *reinterpret_cast<uint4*>(prow + (((k * (NT / 16) + c0 / 16) ^ (kl & 7)) << 4)) =
                make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
        }
      } else {
#pragma unroll
        for (int c0 = 0; c0 < NT; c0 += 8) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int n0 = c0 + 4 * h;
            const float4 c4 = *reinterpret_cast<const float4*>(&gr.c[n0]), m4 = *reinterpret_cast<const float4*>(&gr.m[n0]);
            const float p0 = ex2(fmaf(s[n0], c4.x, -m4.x)), p1 = ex2(fmaf(s[n0 + 1], c4.y, -m4.y));
            const float p2 = ex2(fmaf(s[n0 + 2], c4.z, -m4.z)), p3 = ex2(fmaf(s[n0 + 3], c4.w, -m4.w));
            l[n0] += p0, l[n0 + 1] += p1, l[n0 + 2] += p2, l[n0 + 3] += p3;
            const float x[4] = {p0 * 16.f, p1 * 16.f, p2 * 16.f, p3 * 16.f};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const __half2 t = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
              const float2 back = __half22float2(t);
              hi[2 * h + e] = h2u(t);
              lo[2 * h + e] = h2u(__floats2half2_rn(x[2 * e] - back.x, x[2 * e + 1] - back.y));
            }
          }
          *reinterpret_cast<uint4*>(prow + (((c0 / 8) ^ (kl & 7)) << 4)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(prow + (((NT / 8 + c0 / 8) ^ (kl & 7)) << 4)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
      }
      if (kl == 0) *reinterpret_cast<volatile int*>(&restart[sub]) = fresh;
      fence_proxy_async_smem();
      fence_before();
      mbar_arrive(&bars.p_full[sub]);
    }
    if (nb) flush(nb, false);
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  float* fold = reinterpret_cast<float*>(smem);  // [row][HD]: the ring is idle
  if (warp >= 4) {
    const int sub = (warp >> 2) - 1, wq = warp & 3;
    Group<NT>& gr = groups[sub];
#pragma unroll
    for (int n = 0; n < NT; ++n) fold[(sub * NT + n) * HD + wq * 32 + lane] = facc[n] * (1.f / gr.vs[n]);  // a power of two
    // sums over the group's 128 positions: after the exchanges lane n (and n +
    // 16, of 16 rows) of a warp holds row n's
    if (NT == 16)
#pragma unroll
      for (int n = 0; n < NT; ++n) l[n] += __shfl_xor_sync(0xffffffffu, l[n], 16);
#pragma unroll
    for (int w = NT / 2; w; w >>= 1) {
      const bool up = lane & w;
#pragma unroll
      for (int n = 0; n < w; ++n) {
        const float send = up ? l[n] : l[n + w], keep = up ? l[n + w] : l[n];
        l[n] = keep + __shfl_xor_sync(0xffffffffu, send, w);
      }
    }
    gr.mx[wq][lane] = __float_as_uint(l[0]);
    group_sync(1 + sub, 128);
    if (wq == 0 && lane < NT) {
      float L = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) L += __uint_as_float(gr.mx[k][lane]);
      cta_ml[sub * NT + lane] = make_float2(gr.m[lane], L);
    }
  }
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(F::TMEM_COLS) : "memory");
  tree_join<HD, F::ROWS, F::THREADS>(a, rowt, cta_ml, fold, min(F::ROWS, a.R - tile * F::ROWS), C, rank, nclusters);
}

// cuTensorMapEncodeTiled, from the driver that the runtime already loaded.
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

template <bool I8, int NT>
static cudaError_t launch(TreeArgs a, int tiles, int units, int64_t most, int* err, cudaStream_t s) {
  using F = Cfg<I8, NT>;
  auto kern = tree_tc_kernel<I8, NT>;
  const EncodeFn enc = encode_fn();
  if (!enc) return cudaErrorNotSupported;
  // rows of all heads as one 2-D tensor; a box is one block (fp16: half of its
  // dims).  x is 0 or 64 values: 16-byte boundaries.  Rows past the last are
  // filled with zeros.
  CUtensorMap maps[2];
  const cuuint64_t dims[2] = {(cuuint64_t)HD, (cuuint64_t)a.c.kv_heads * a.c.ctx};
  const cuuint64_t strides[1] = {(cuuint64_t)HD * (I8 ? 1 : 2)};
  const cuuint32_t box[2] = {I8 ? 128u : 64u, (cuuint32_t)BK}, ones[2] = {1, 1};
  for (int i = 0; i < 2; ++i)
    if (enc(&maps[i], I8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, i ? a.c.v : a.c.k, dims,
            strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return cudaErrorInvalidValue;
  static TreeLaunch state;
  return launch_tree_clusters(state, (const void*)kern, a, tiles, units, TA_SMS, most, F::THREADS, F::SMEM, s,
                              [&](const cudaLaunchConfig_t& cfg) {
                                return cudaLaunchKernelEx(&cfg, kern, a, err, maps[0], maps[1]);
                              });
}

}  // namespace ttc

cudaError_t launch_tree_tc(const TreeArgs& a, int rows_per_cta, int tiles, int units, int64_t most, int* err, cudaStream_t s) {
  const bool one = rows_per_cta == 32;
  if (a.c.dtype == ODI_CUDA_KV_I8)
    return one ? ttc::launch<true, 16>(a, tiles, units, most, err, s) : ttc::launch<true, 32>(a, tiles, units, most, err, s);
  return one ? ttc::launch<false, 16>(a, tiles, units, most, err, s) : ttc::launch<false, 32>(a, tiles, units, most, err, s);
}

}  // namespace odi_cuda
