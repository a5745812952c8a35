// tree_attention_tc.cu -- tree attention for many rows per kv head on the
// sm_100a tensor cores (tcgen05.mma, accumulators in tensor memory).
//
// The same mathematics, row numbering and splits as tree_attention.cu, for
// head_dim 128 and more rows per kv head than one 8-row tile.  A CTA takes 32
// or 64 rows (one or two groups of 32) of one kv head and every nsplit-th
// block of 128 positions:
//
//   S^T [128 positions x 32 rows] = K . Q^T     positions as M
//   O^T [128 dims x 32 rows]     += V^T . P^T   dims as M
//
// With the cache as the M side every instruction is full whatever the number
// of rows, K and V are used as TMA leaves them in shared memory (K as a
// K-major operand, V, in the same byte order, as an MN-major one), and each is
// fetched once for all the CTA's rows.
//
// fp32 results from 16- and 8-bit products, as columns of one instruction:
//  * int8 cache (kind::i8, exact 32-bit integer sums): q is fixed point in
//    three signed digits (96 columns), |dq_i| <= 2^-22 max |q|; P * (V's row
//    scale) in four unsigned digits (128 columns), an integer below 2^32.
//  * fp16 cache (kind::f16): q is the sum of two fp16 values (22 bits), P is
//    hi + 2^-11 lo (64 columns each); the two sums are joined in fp32.  With the
//    low half scaled so, a weight of up to 2^15 has 22 bits down to 2^-14 and an
//    absolute error of 2^-37 below.
//
//   warp 0       TMA producer: tiles K0 K1 V0 K2 V1 ... through one ring
//   warps 1, 2   issue the products, one warp for each group of rows; warp 1
//                holds the tensor memory
//   warps 4-11   a warpgroup per group of rows (of one group, one for each half
//                of its rows): thread = position (tensor memory lane) in the
//                softmax, = dim when O is read
//
// While one group of rows is in its softmax the tensor core works for the
// others.  As in tree_attention.cu m is a reference that moves only when a
// weight (int8: weight * scale, what the values enter with) would leave its
// range, by whole powers of two.  Only the row that moves takes its O out of
// tensor memory then, to fp32 registers; all rows do every few blocks, always
// the same ones (integer sums cannot overflow so, and fp32 sums, which truncate,
// stay short): a row's bits do not depend on the rows beside it.
//
// The softmax bounds the kernel: 17 instructions per score (packed fp32 pairs
// where two scores share an operation), of which two warps per scheduler issue
// one every 2.3 cycles.  64 nodes, 64 / 8 heads, 32641 int8 positions: 183 us
// (fp16: 168), where fetching the cache takes 11 and 69 GFLOP at the fp16 rate 41;
// the loop without any products took 176 where the whole took 182.  Smaller shares
// for more warps (16 of 16 rows: 212 us, the work per block that does not depend on
// rows doubles), a vote without a barrier (234 where this took 224), scores one
// block ahead of the weights (200) and V turned into fp16 in shared memory by four
// more warps (220) were slower.
//
// Every wait is bounded; a wait that gives up sets the error word, all roles
// leave their loops, copies in flight are waited for and the tensor memory is
// released.
#include <cuda.h>
#include <math.h>

#include <type_traits>

#include "tree_attention.cuh"

namespace odi_cuda {
namespace ttc {

constexpr int HD = 128;
constexpr int BK = 128;  // positions per block
constexpr int NT = 32;   // rows per group
constexpr int ERR_TREE_WAIT = 64;
constexpr int START_BYTES = 32 * 16;
constexpr float P_LOW = 0x1p-11f;  // fp16: the unit of P's low half, which keeps it from the subnormals

template <bool I8, int SUBS_>
struct Cfg {
  static constexpr int SUBS = SUBS_;                      // groups of rows
  static constexpr int DQ = I8 ? 3 : 2, DP = I8 ? 4 : 2;  // digits of q and P
  static constexpr int TILE = BK * HD * (I8 ? 1 : 2);     // K or V of one block
  static constexpr int SLOTS = I8 ? 8 : 4;
  static constexpr int QB = DQ * NT * HD * (I8 ? 1 : 2);
  static constexpr int PB = BK * 128;                     // one 128-byte row per position
  static constexpr int Q_OFF = SLOTS * TILE;
  static constexpr int P_OFF = Q_OFF + SUBS * QB;
  // int8: what the sums of S start from.  Copied by the tensor core's own
  // instructions in 32-row pieces: 187 us where the softmax threads stored it
  // (54 of their 616 instructions per block), 182 this way, 206 in 128-row pieces
  // (64 nodes over 32641 positions).
  static constexpr int START_OFF = P_OFF + SUBS * PB;
  static constexpr int SMEM = START_OFF + (I8 ? START_BYTES : 0) + 1024;  // + alignment slack
  static constexpr int HALVES = SUBS == 1 ? 2 : 1;        // softmax threads per position and group
  static constexpr int NH = NT / HALVES;                  // rows of a group per softmax thread
  static constexpr int GT = 128 * HALVES;                 // softmax threads of a group
  static constexpr int THREADS = 128 + SUBS * GT;
  // with two groups the launch's registers are shared out anew between the first
  // warpgroup and the softmax's, which holds 96 sums, 32 scores, 32 weights' sums
  // and 32 values of O per thread
  static constexpr int REGS_LAUNCH = 168, REGS_FIRST = 40, REGS_SOFT = 232;
  static_assert(SUBS == 1 || 128 * REGS_FIRST + SUBS * GT * REGS_SOFT <= THREADS * REGS_LAUNCH, "register split");
  static constexpr int ROWS = NT * SUBS;
  static constexpr int SCOLS = DQ * NT, OCOL = (I8 ? 4 : 2) * NT, SUBCOLS = 2 * OCOL;
  static constexpr int TMEM_COLS = SUBCOLS * SUBS;
  // blocks between two moves of all O to registers: 255 * 128 * 128 * 256 < 2^31;
  // the fp32 accumulator truncates, about 2^-26 of the sum per instruction
  static constexpr int PERIOD = I8 ? 256 : 4;
  // Weights in P, log2: what they stay below, and the largest right after a move.
  // int8: an integer below 2^32, so to within 2^-25 of the largest, either way;
  // 64 nodes over 32641 positions 183 us, 198 and 207 with the largest at 2^27 and
  // 2^29, since a block in which a row moves costs two.  fp16: to within 2^-37, which
  // is 2^-44 to 2^-45 of the largest.
  static constexpr float P_TOP = I8 ? 31.9f : 15.f, P_UNIT = I8 ? 26.f : 8.f;
  static_assert(SMEM <= 222 * 1024, "shared memory, beside the static part");
};

// Shared-memory matrix descriptors, 128-byte swizzle.  K-major: rows of 128
// bytes, groups of 8 rows 1024 bytes apart.  MN-major: K rows of 128 bytes of
// the M or N side, groups of 8 K rows 1024 bytes apart, further 128-byte
// pieces of the M side `lbo` bytes apart.
__device__ __forceinline__ uint64_t desc(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// Rows of 16 bytes, groups of 8 rows 128 bytes apart.
__device__ __forceinline__ uint64_t desc_rows16(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (8ull << 16) | (8ull << 32) | (1ull << 46);
}
// 4 columns of tensor memory, the same 32 rows for each warp's lanes, from shared
// memory, before the products that the same thread issues next.
__device__ __forceinline__ void copy_rows16(uint32_t d, uint64_t src) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(d), "l"(src) : "memory");
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
// 32 lanes x N consecutive columns of each digit, `stride` columns apart.  Loads
// and wait are one statement: no use of a register can move ahead of the wait.
#define TA_OUT8(r) "=r"((r)[0]), "=r"((r)[1]), "=r"((r)[2]), "=r"((r)[3]), "=r"((r)[4]), "=r"((r)[5]), "=r"((r)[6]), "=r"((r)[7])
#define TA_OUT16(r) TA_OUT8(r), TA_OUT8((r) + 8)
#define TA_OUT32(r) TA_OUT16(r), TA_OUT16((r) + 16)
__device__ __forceinline__ void ld_digits(uint32_t (&r)[2][8], uint32_t addr, uint32_t stride) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%16];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%17];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : TA_OUT8(r[0]), TA_OUT8(r[1])
      : "r"(addr), "r"(addr + 1 * stride)
      : "memory");
}
__device__ __forceinline__ void ld_digits(uint32_t (&r)[2][16], uint32_t addr, uint32_t stride) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : TA_OUT16(r[0]), TA_OUT16(r[1])
      : "r"(addr), "r"(addr + 1 * stride)
      : "memory");
}
__device__ __forceinline__ void ld_digits(uint32_t (&r)[2][32], uint32_t addr, uint32_t stride) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : TA_OUT32(r[0]), TA_OUT32(r[1])
      : "r"(addr), "r"(addr + 1 * stride)
      : "memory");
}
__device__ __forceinline__ void ld_digits(uint32_t (&r)[3][16], uint32_t addr, uint32_t stride) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%48];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%49];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47}, [%50];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : TA_OUT16(r[0]), TA_OUT16(r[1]), TA_OUT16(r[2])
      : "r"(addr), "r"(addr + 1 * stride), "r"(addr + 2 * stride)
      : "memory");
}
__device__ __forceinline__ void ld_digits(uint32_t (&r)[3][32], uint32_t addr, uint32_t stride) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%96];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%97];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95}, [%98];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : TA_OUT32(r[0]), TA_OUT32(r[1]), TA_OUT32(r[2])
      : "r"(addr), "r"(addr + 1 * stride), "r"(addr + 2 * stride)
      : "memory");
}
__device__ __forceinline__ void st_digits(const uint32_t (&r)[2][8], uint32_t addr, uint32_t stride) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7};\n\t"
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%17], {%8,%9,%10,%11,%12,%13,%14,%15};\n\t"
      "tcgen05.wait::st.sync.aligned;" ::"r"(r[0][0]), "r"(r[0][1]), "r"(r[0][2]), "r"(r[0][3]), "r"(r[0][4]), "r"(r[0][5]),
      "r"(r[0][6]), "r"(r[0][7]), "r"(r[1][0]), "r"(r[1][1]), "r"(r[1][2]), "r"(r[1][3]), "r"(r[1][4]), "r"(r[1][5]),
      "r"(r[1][6]), "r"(r[1][7]), "r"(addr), "r"(addr + 1 * stride)
      : "memory");
}
__device__ __forceinline__ void st_digits(const uint32_t (&r)[2][16], uint32_t addr, uint32_t stride) {
#pragma unroll
  for (int k = 0; k < 2; ++k)
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[k][0]),
        "r"(r[k][1]), "r"(r[k][2]), "r"(r[k][3]), "r"(r[k][4]), "r"(r[k][5]), "r"(r[k][6]), "r"(r[k][7]), "r"(r[k][8]),
        "r"(r[k][9]), "r"(r[k][10]), "r"(r[k][11]), "r"(r[k][12]), "r"(r[k][13]), "r"(r[k][14]), "r"(r[k][15]),
        "r"(addr + k * stride)
        : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void group_sync(int id, int n) {
  __syncwarp();
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory");
}
__device__ __forceinline__ bool group_any(int id, int n, bool v) {
  uint32_t r;
  __syncwarp();
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
      "bar.red.or.pred p, %2, %3, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "r"(id), "r"(n)
      : "memory");
  return r != 0;
}
// The integer sums of S start from the bits of B = 1.5 * 2^23, so that they are
// read back as the fp32 value B + sum (|sum| < 2^22) without a conversion, which
// runs at an eighth of an add's rate.  Two scores at a time: h * 2^16 + m * 2^8 +
// l; m and l are joined first, to a multiple of 2^8, which is 2^-21 of a product
// of ordinary size (2^29 and more); what the Bs add up to leaves with h, exactly.
constexpr uint32_t S_START = 0x4B400000u;
__device__ __forceinline__ float2 f2(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 bits2(uint32_t a, uint32_t b) { return make_float2(__uint_as_float(a), __uint_as_float(b)); }
__device__ __forceinline__ float2 join_digits(float2 h, float2 m, float2 l) {
  constexpr float B = 12582912.f;
  return __fadd2_rn(__ffma2_rn(h, f2(65536.f), f2(-B * 65793.f)), __ffma2_rn(m, f2(256.f), l));
}
// The lane's share of a column-wise maximum: value(n) of N columns on each of 32
// lanes; lane n (N = 16: also n + 16) gets column n's largest.
template <int N, typename V>
__device__ __forceinline__ float lane_max(V&& value) {
  const int lane = threadIdx.x & 31;
  float x[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    x[n] = value(n);
    if (N == 16) x[n] = fmaxf(x[n], __shfl_xor_sync(0xffffffffu, x[n], 16));
  }
#pragma unroll
  for (int w = N / 2; w; w >>= 1) {
    const bool up = lane & w;
#pragma unroll
    for (int n = 0; n < w; ++n) {
      const float send = up ? x[n] : x[n + w], keep = up ? x[n + w] : x[n];
      x[n] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, send, w));
    }
  }
  return x[0];
}

template <int SUBS>
struct Bars {
  uint64_t tfull[8], tfree[8];
  uint64_t s_full[SUBS], s_free[SUBS], p_full[SUBS], pv_done[SUBS];
  uint64_t v_clean[2];
};
// What a group's threads share about its rows.
struct alignas(16) Group {
  float c[NT];      // factor of the scores, positive
  float nm[NT];     // minus the reference, a whole number
  float nx[NT];     // the same, or 0 for a row without one
  float dx[NT];     // how far it moved
  float fo[NT];     // factor of O and of the sums then
  float mx[4][NT];
  unsigned scaled[2];  // rows of each half whose sums it scales
  int none[2];         // some row of the half has no reference yet
};

template <bool I8, int SUBS>
__global__ void __launch_bounds__(Cfg<I8, SUBS>::THREADS, 1)
    tree_tc_kernel(const TreeArgs a, int* err, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap) {
  using F = Cfg<I8, SUBS>;
  constexpr int NH = F::NH, HALVES = F::HALVES, GT = F::GT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ Bars<SUBS> bars;
  __shared__ Group groups[SUBS];
  __shared__ int rowt[F::ROWS];
  __shared__ float2 cta_ml[F::ROWS];
  __shared__ uint32_t tmem_slot;
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
      mbar_init(&bars.s_free[i], GT);
      mbar_init(&bars.p_full[i], GT);
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
  auto request_tile = [&](int t) {  // one thread of warp 0
    const int slot = t % F::SLOTS;
    const bool isk = t == 0 || (t == seqs - 1 ? false : (t & 1));
    const int i = t == 0 ? 0 : isk ? (t + 1) / 2 : t == seqs - 1 ? nb - 1 : t / 2 - 1;
    const int row = (int)(head + (int64_t)(split + i * stride) * BK);
    uint8_t* dst = smem + slot * F::TILE;
    mbar_arrive_expect_tx(&bars.tfull[slot], F::TILE);
    const CUtensorMap* map = isk ? &kmap : &vmap;
    tma_2d(dst, map, 0, row, &bars.tfull[slot]);
    if (!I8) tma_2d(dst + F::TILE / 2, map, 64, row, &bars.tfull[slot]);
  };
  // the first tiles are on their way while the other warps lay out Q
  if (tid == 0)
    for (int t = 0; t < seqs && t < F::SLOTS; ++t) request_tile(t);

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"(F::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // ---- Q: digits as K-major operand rows n' = digit * 32 + n; eight lanes per
  // row, 16 dims each
  if (warp >= 4) {
    constexpr int PASS = F::ROWS / 32;  // 8 warps of 4 rows
    const bool vec = !(((uintptr_t)a.q & 15) | (a.ld_q & 3));
    const int l8 = lane & 7;
    float v[PASS][16];
    int rt[PASS];
#pragma unroll
    for (int i = 0; i < PASS; ++i) {
      const int r = tile * F::ROWS + i * 32 + (warp - 4) * 4 + (lane >> 3);
      rt[i] = r < a.R ? row_node(a, r) : -1;
#pragma unroll
      for (int e = 0; e < 16; ++e) v[i][e] = 0.f;
      if (r < a.R) {
        const float* src = a.q + (int64_t)rt[i] * a.ld_q + (int64_t)(kvh * a.G + r - rt[i] * a.G) * HD + l8 * 16;
        if (vec) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float4 x = __ldcg(reinterpret_cast<const float4*>(src) + e);
            v[i][4 * e] = x.x, v[i][4 * e + 1] = x.y, v[i][4 * e + 2] = x.z, v[i][4 * e + 3] = x.w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) v[i][e] = __ldcg(src + e);
        }
      }
    }
    const float sign = a.scale_log2 < 0.f ? -1.f : a.scale_log2 > 0.f ? 1.f : 0.f;  // the scores' factor stays positive
#pragma unroll
    for (int i = 0; i < PASS; ++i) {
      const int n = i * 32 + (warp - 4) * 4 + (lane >> 3), sub = n / NT, ln = n % NT;
      float am = 0.f, sum = 0.f;  // sum * 0 is 0 only if every value is finite
#pragma unroll
      for (int e = 0; e < 16; ++e) am = fmaxf(am, fabsf(v[i][e])), sum = fmaf(v[i][e], 0.f, sum);
#pragma unroll
      for (int x = 4; x; x >>= 1) {
        am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, x));
        sum += __shfl_xor_sync(0xffffffffu, sum, x);
      }
      const bool ok = sum == 0.f;
      int ex = (int)(__float_as_uint(am) >> 23) - 127;
      if (I8 && am * pow2(-min(max(ex, -100), 126)) > 1.99f) ++ex;
      ex = min(max(ex, -100), 126);
      const float lift = ok ? pow2(-ex) : 0.f, unit = I8 ? q_units(am) : 8192.f, up = unit * sign;
      if (l8 == 0) {
        Group& gr = groups[sub];
        gr.c[ln] = ok ? fmaxf(q_factor(fabsf(a.scale_log2), 1.f / unit, ex), 1e-37f) : __int_as_float(0x7fc00000);
        gr.nm[ln] = ok ? -TA_NONE : 0.f;  // of a row of NaNs any will do
        gr.nx[ln] = 0.f;
        if (ln % NH == 0) gr.none[ln / NH] = 1;
        rowt[n] = rt[i];
      }
      uint8_t* q = smem + F::Q_OFF + sub * F::QB;
      if (I8) {
        int dig[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) dig[e] = ok ? __float2int_rn(v[i][e] * lift * up) : 0;
#pragma unroll
        for (int k = F::DQ - 1; k >= 0; --k) {  // digit 0 the highest
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t bytes = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int lo = (int)(int8_t)(dig[4 * j + e] & 255);
              dig[4 * j + e] = (dig[4 * j + e] - lo) >> 8;
              bytes |= (uint32_t)(lo & 255) << (8 * e);
            }
            w[j] = bytes;
          }
          const int row = k * NT + ln;
          *reinterpret_cast<uint4*>(q + row * 128 + ((l8 ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      } else {  // two pieces of 64 dims, each [64 rows][128 bytes]
        uint8_t* piece = q + (l8 >> 2) * (F::DQ * NT * 128);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x0 = ok ? v[i][8 * j + 2 * e] * lift * up : 0.f, x1 = ok ? v[i][8 * j + 2 * e + 1] * lift * up : 0.f;
            const __half2 h = __floats2half2_rn(x0, x1);
            const float2 back = __half22float2(h);
            hi[e] = h2u(h);
            lo[e] = h2u(__floats2half2_rn(x0 - back.x, x1 - back.y));
          }
          const int ch = (l8 & 3) * 2 + j;
          *reinterpret_cast<uint4*>(piece + ln * 128 + ((ch ^ (ln & 7)) << 4)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(piece + (NT + ln) * 128 + ((ch ^ (ln & 7)) << 4)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
      }
    }
  }
  if (I8 && tid >= 128)
    for (int i = tid - 128; i < START_BYTES / 4; i += SUBS * GT) reinterpret_cast<uint32_t*>(smem + F::START_OFF)[i] = S_START;
  fence_proxy_async_smem();
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp < 4) {
    if (SUBS == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F::REGS_FIRST));
    if (warp == 0) {
      // ---------------- producer ----------------
      if (lane == 0) {
        int t = min(seqs, F::SLOTS);
        for (; t < seqs; ++t) {
          if (!mbar_wait(&bars.tfree[t % F::SLOTS], ((t / F::SLOTS) & 1) ^ 1, err, ERR_TREE_WAIT)) {
            dead = 1;
            break;
          }
          request_tile(t);
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
      const int u = warp - 1;  // one warp for each group: neither waits for the other's softmax
      const uint32_t q0 = smem_u32(smem + F::Q_OFF + u * F::QB), p0 = smem_u32(smem + F::P_OFF + u * F::PB), t0 = smem_u32(smem);
      const uint32_t d0 = tmem + u * F::SUBCOLS;
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
          if (I8)
#pragma unroll
            for (int k = 0; k < F::SCOLS; k += 4) copy_rows16(d0 + k, desc_rows16(smem_u32(smem + F::START_OFF)));
#pragma unroll
          for (int k = 0; k < (I8 ? 4 : 8); ++k)  // 32 bytes of the contraction per instruction
            mma<I8>(d0, kd + (k >> 2) * (F::TILE / 2 >> 4) + 2 * (k & 3), qd0 + (k >> 2) * (F::DQ * NT * 128 >> 4) + 2 * (k & 3),
                    idesc(I8, false, F::SCOLS), I8 || k != 0);
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
        const uint32_t keep = i % F::PERIOD != 0;
        if (elect_one()) {
          const uint64_t vd = vd0 + (uint32_t)(slot * (F::TILE >> 4));
          constexpr int KS = I8 ? 4 : 8, KB = BK / KS * 128;  // bytes of 32 or 16 positions
#pragma unroll
          for (int k = 0; k < KS; ++k)
            mma<I8>(d0 + F::OCOL, vd + k * (KB >> 4), pd0 + k * (KB >> 4), idesc(I8, true, F::DP * NT), k ? 1u : keep);
          commit(&bars.pv_done[u]);
          commit(&bars.tfree[slot]);
        }
        __syncwarp();
      }
      if (!ok) dead = 1;
    }
    tree_join_rest(C, nclusters);
  } else {
    // ---------------- softmax ----------------
    if (SUBS == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F::REGS_SOFT));
    const int sub = HALVES == 2 ? 0 : (warp >> 2) - 1, half = HALVES == 2 ? (warp >> 2) - 1 : 0, wq = warp & 3, kl = wq * 32 + lane, bar = 1 + sub;
    const int h0 = half * NH;  // this thread's rows: h0 .. h0 + NH - 1 of the group
    Group& gr = groups[sub];
    const uint32_t s_tm = tmem + sub * F::SUBCOLS + h0 + ((uint32_t)(wq * 32) << 16), o_tm = s_tm + F::OCOL;
    uint8_t* prow = smem + F::P_OFF + sub * F::PB + kl * 128;
    const int psw = kl & 7;  // swizzle of this row's 16-byte pieces
    const float* ks = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.c.k) + a.c.scale_off) + head;
    const float* vsc = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.c.v) + a.c.scale_off) + head;
    const float nan = __int_as_float(0x7fc00000);
    float facc[NH];
    float2 l2[NH / 2];
#pragma unroll
    for (int n = 0; n < NH; ++n) facc[n] = 0.f;
#pragma unroll
    for (int n = 0; n < NH / 2; ++n) l2[n] = f2(0.f);
    float dk = 0.f, dv = 0.f, dk_next = 0.f, dv_next = 0.f;
    auto request = [&](int i) {
      const int key = min((split + i * stride) * BK + kl, len - 1);
      dk_next = __ldcg(ks + key), dv_next = __ldcg(vsc + key);
    };
    if (I8 && nb) request(0);
    auto wait_pv = [&](int i) {  // O holds the products of the blocks before i
      if (!mbar_wait(&bars.pv_done[sub], (i - 1) & 1, err, ERR_TREE_WAIT)) dead = 1;
      __syncwarp();
      fence_after();
    };
    // O's sums so far of eight rows from c0 on, out of tensor memory.  `only`: of the
    // rows with a bit there (the same for all threads), whose sums then go on from 0.
    auto take = [&](int c0, auto only, unsigned rows) {
      constexpr bool all = !decltype(only)::value;
      if (I8) {  // two low digits of each row, then, 64 columns on, two high ones
        uint32_t r[2][16];
        ld_digits(r, o_tm + h0 + 2 * c0, 2 * NT);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const float x = fmaf((float)(int)r[1][2 * n + 1], 16777216.f,
                               fmaf((float)(int)r[1][2 * n], 65536.f, fmaf((float)(int)r[0][2 * n + 1], 256.f, (float)(int)r[0][2 * n])));
          if (all || ((rows >> n) & 1u)) {
            facc[c0 + n] += x;
            r[0][2 * n] = r[0][2 * n + 1] = r[1][2 * n] = r[1][2 * n + 1] = 0;
          }
        }
        if (!all) st_digits(r, o_tm + h0 + 2 * c0, 2 * NT);
      } else {
        uint32_t r[2][8];
        ld_digits(r, o_tm + c0, NT);
#pragma unroll
        for (int n = 0; n < 8; ++n)
          if (all || ((rows >> n) & 1u)) {
            facc[c0 + n] += fmaf(__uint_as_float(r[1][n]), P_LOW, __uint_as_float(r[0][n]));
            r[0][n] = r[1][n] = 0;
          }
        if (!all) st_digits(r, o_tm + c0, NT);
      }
    };
    auto take_all = [&]() {
#pragma unroll
      for (int c0 = 0; c0 < NH; c0 += 8) take(c0, std::false_type(), 0);
      fence_before();
    };
    // which of the warp's 32 positions lane n's row sees; of this CTA's first
    // block that needs it, asked for now
    auto row_sees = [&](int i) {
      return lane < NH ? seen_bits(a, rowt[sub * NT + h0 + lane], (split + i * stride) * BK + wq * 32, pos, len) : 0u;
    };
    const int b0 = min(pos, len) / BK, first_edge = pos <= 0 || b0 <= split ? 0 : (b0 - split + stride - 1) / stride;
    const uint32_t first_sees = first_edge < nb ? row_sees(first_edge) : 0u;
    // int8: what a weight's integer part is taken after adding; spread over 0 .. 1
    // by the golden ratio from position to position, so that weights below a unit
    // are kept in the mean
    const float dither = (float)((unsigned)kl * 0x9E3779B9u >> 9) * 0x1p-23f;
    int edges = 0;
    for (int i = 0; i < nb; ++i) {
      const int p0 = (split + i * stride) * BK, key = p0 + kl;
      if (I8) {
        dk = dk_next, dv = dv_next;
        if (i + 1 < nb) request(i + 1);
      }
      uint32_t vis = 0xffffffffu;  // bit n: row n sees this position
      bool ok = true, bad = false;
      const bool edge = p0 + BK > min(pos, len);  // holds tree slots, or ends past the last
      if (edge) {  // which of them are seen, while the scores are on their way
        if (!I8) {
          // V rows that are past the end or not finite leave the tile; who
          // sees such a row gets NaN through its score, nobody else meets it.
          // The first half of the first group does it and the others wait: two
          // such tiles on, it is held until everybody's products on this one are
          // done (the tile's slot).
          if (sub == 0 && half == 0) {
            const int t = vseq(i), slot = t % F::SLOTS;
            ok = mbar_wait(&bars.tfull[slot], (t / F::SLOTS) & 1, err, ERR_TREE_WAIT) && ok;
            uint8_t* vrow = smem + slot * F::TILE + kl * 128;
            bad = key >= len;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const uint4 x = *reinterpret_cast<const uint4*>(vrow + (e >> 3) * (F::TILE / 2) + ((e ^ kl) & 7) * 16);  // neighbours on other banks
              const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int j = 0; j < 4; ++j) bad = bad || (w[j] & 0x7c00u) == 0x7c00u || (w[j] & 0x7c000000u) == 0x7c000000u;
            }
            if (bad)
#pragma unroll
              for (int e = 0; e < 16; ++e)
                *reinterpret_cast<uint4*>(vrow + (e >> 3) * (F::TILE / 2) + ((e ^ kl) & 7) * 16) = make_uint4(0, 0, 0, 0);
            bad_row[edges & 1][kl] = bad;
            fence_proxy_async_smem();
            mbar_arrive(&bars.v_clean[edges & 1]);
          } else {
            ok = mbar_wait(&bars.v_clean[edges & 1], (edges >> 1) & 1, err, ERR_TREE_WAIT) && ok;
            bad = bad_row[edges & 1][kl];
          }
          ++edges;
        }
        const uint32_t rowsee = i == first_edge ? first_sees : row_sees(i);
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const uint32_t b = __ballot_sync(0xffffffffu, (rowsee >> k) & 1u);
          if (lane == k) vis = b;
        }
      }
      ok = mbar_wait(&bars.s_full[sub], i & 1, err, ERR_TREE_WAIT) && ok;
      __syncwarp();
      fence_after();
      float2 x2[NH / 2];  // factor * score - reference, base 2
      // a row whose scale of K or V is not finite gives NaN to who sees it
      const float dkk = finite(dk) && finite(dv) ? dk : nan, dvv = finite(dv) ? dv : 0.f;
      {
        uint32_t r[F::DQ][NH];  // all of this thread's sums at once: one latency
        ld_digits(r, s_tm, NT);
#pragma unroll
        for (int n = 0; n < NH / 2; n += 2) {
          const float4 c4 = *reinterpret_cast<const float4*>(&gr.c[h0 + 2 * n]), m4 = *reinterpret_cast<const float4*>(&gr.nx[h0 + 2 * n]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int a0 = 2 * (n + e), a1 = a0 + 1;
            const float2 hi = bits2(r[0][a0], r[0][a1]), lo = bits2(r[1][a0], r[1][a1]);
            float2 s;
            if (I8)
              s = __fmul2_rn(join_digits(hi, lo, bits2(r[F::DQ - 1][a0], r[F::DQ - 1][a1])), f2(dkk));
            else
              s = __fadd2_rn(hi, lo);
            x2[n + e] = __ffma2_rn(s, e ? make_float2(c4.z, c4.w) : make_float2(c4.x, c4.y), e ? make_float2(m4.z, m4.w) : make_float2(m4.x, m4.y));
          }
        }
      }
      fence_before();
      mbar_arrive(&bars.s_free[sub]);
      if (edge) {
#pragma unroll
        for (int n = 0; n < NH; ++n) {
          float& x = n & 1 ? x2[n / 2].y : x2[n / 2].x;
          if (!((vis >> n) & 1u)) x = -INFINITY;
          else if (!I8 && bad) x = nan;
        }
      }
      // does a weight leave its range?  (A scale near 0 stands for 2^-64, so that
      // a key whose values are nothing moves no reference, and overflows none.)
      const float ldv = I8 ? __log2f(fmaxf(dvv, 0x1p-64f)) : 0.f;
      float top = -INFINITY;
#pragma unroll
      for (int n = 0; n < NH / 2; ++n) top = fmaxf(top, fmaxf(x2[n].x, x2[n].y));
      top += ldv;
      if (!ok) dead = 1;
      const bool fresh = i % F::PERIOD == 0;  // O starts again
      bool drained = false;
      if (group_any(bar, GT, top > F::P_TOP || gr.none[half] || !ok)) {
        if (group_any(bar, GT, *reinterpret_cast<volatile int*>(&dead) != 0)) break;
        // Lane n (of 16 rows, and n + 16) gets row n's largest weight among the
        // warp's positions.
        const float mx = lane_max<NH>([&](int n) {
          const float x = (n & 1 ? x2[n / 2].y : x2[n / 2].x) + ldv;
          return x == x ? x : -INFINITY;
        });
        if (lane < NH) gr.mx[wq][h0 + lane] = mx;
        group_sync(bar, GT);
        if (wq == 0) {
          bool scaled = false, none = false;
          if (lane < NH) {
            const int n = h0 + lane;
            const float m = fmaxf(fmaxf(gr.mx[0][n], gr.mx[1][n]), fmaxf(gr.mx[2][n], gr.mx[3][n]));
            float dx = 0.f, fo = 1.f;
            none = gr.nm[n] == -TA_NONE;
            if (m > (none ? -INFINITY : F::P_TOP)) {  // each row by itself
              const float from = none ? 0.f : gr.nm[n], to = from + (F::P_UNIT - ceilf(m));
              dx = to - from;
              scaled = !none;
              if (scaled) fo = dx < -126.f ? 0.f : pow2((int)dx);
              gr.nm[n] = gr.nx[n] = to;
              none = false;
            }
            gr.dx[n] = dx, gr.fo[n] = fo;
          }
          none = __any_sync(0xffffffffu, none);
          const unsigned rows = __ballot_sync(0xffffffffu, scaled);
          if (lane == 0) gr.none[half] = none, gr.scaled[half] = rows;
        }
        group_sync(bar, GT);
#pragma unroll
        for (int n = 0; n < NH / 2; ++n) x2[n] = __fadd2_rn(x2[n], *reinterpret_cast<const float2*>(&gr.dx[h0 + 2 * n]));
        const unsigned rows = gr.scaled[half];
        if (rows) {
          if (i) wait_pv(i);
          if (i && fresh) take_all();
          drained = true;
#pragma unroll
          for (int c0 = 0; c0 < NH; c0 += 8) {
            const unsigned some = (rows >> c0) & 0xffu;
            if (!some) continue;
            if (!fresh) take(c0, std::true_type(), some);
#pragma unroll
            for (int n = 0; n < 8; ++n) {
              const float f = gr.fo[h0 + c0 + n];
              facc[c0 + n] *= f;
              (n & 1 ? l2[(c0 + n) / 2].y : l2[(c0 + n) / 2].x) *= f;
            }
          }
          fence_before();
        }
      }
      if (i && !drained) {
        if (fresh) {
          wait_pv(i);
          take_all();
        } else if (!mbar_wait(&bars.pv_done[sub], (i - 1) & 1, err, ERR_TREE_WAIT)) {
          dead = 1;
        }
      }
      // weights into the operand tile
      if (I8) {
#pragma unroll
        for (int r0 = 0; r0 < NH; r0 += 8) {  // a 16-byte piece of low digits, one of high
          uint32_t lw[4], hw[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int n = r0 / 2 + e;
            const float2 p = make_float2(ex2(x2[n].x), ex2(x2[n].y));
            l2[n] = __fadd2_rn(l2[n], p);
            const float2 y = __ffma2_rn(p, f2(dvv), f2(dither));  // below 2^32: its integer part is the weight
            const float2 hi = __ffma2_rz(y, f2(0x1p-16f), f2(0x1p23f));
            // y - 65536 * (hi - 2^23) + 2^23; all but the last rounding is exact
            const float2 lo = __fadd2_rz(y, __ffma2_rn(hi, f2(-65536.f), f2(0x1p39f + 0x1p23f)));
            lw[e] = __byte_perm(__float_as_uint(lo.x), __float_as_uint(lo.y), 0x5410u);
            hw[e] = __byte_perm(__float_as_uint(hi.x), __float_as_uint(hi.y), 0x5410u);
          }
          *reinterpret_cast<uint4*>(prow + ((((h0 + r0) / 8) ^ psw) << 4)) = make_uint4(lw[0], lw[1], lw[2], lw[3]);
          *reinterpret_cast<uint4*>(prow + (((4 + (h0 + r0) / 8) ^ psw) << 4)) = make_uint4(hw[0], hw[1], hw[2], hw[3]);
        }
      } else {
#pragma unroll
        for (int c0 = 0; c0 < NH / 8; ++c0) {  // eight rows: one 16-byte piece of high halves, one of low
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int n = 4 * c0 + e;
            const float2 p = make_float2(ex2(x2[n].x), ex2(x2[n].y));
            l2[n] = __fadd2_rn(l2[n], p);
            const __half2 t = __floats2half2_rn(p.x, p.y);
            const float2 d = __fmul2_rn(__ffma2_rn(__half22float2(t), f2(-1.f), p), f2(1.f / P_LOW));  // exact
            hi[e] = h2u(t);
            lo[e] = h2u(__floats2half2_rn(d.x, d.y));
          }
          *reinterpret_cast<uint4*>(prow + (((h0 / 8 + c0) ^ psw) << 4)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(prow + (((4 + h0 / 8 + c0) ^ psw) << 4)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
      }
      fence_proxy_async_smem();
      fence_before();
      mbar_arrive(&bars.p_full[sub]);
    }
    if (nb) {
      wait_pv(nb);
      take_all();
    }
    // O and the sums of this group's rows, in its own P tile
    float* fold = reinterpret_cast<float*>(smem + F::P_OFF);  // [row][HD]
    static_assert(F::PB == NT * HD * 4, "a group's rows fill its P tile");
#pragma unroll
    for (int n = 0; n < NH; ++n) fold[(sub * NT + h0 + n) * HD + kl] = facc[n];
    // sums over the group's 128 positions: after the exchanges lane n (of 16
    // rows, and n + 16) of a warp holds row n's
    float l[NH];
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      l[n] = n & 1 ? l2[n / 2].y : l2[n / 2].x;
      if (NH == 16) l[n] += __shfl_xor_sync(0xffffffffu, l[n], 16);
    }
#pragma unroll
    for (int w = NH / 2; w; w >>= 1) {
      const bool up = lane & w;
#pragma unroll
      for (int n = 0; n < w; ++n) {
        const float send = up ? l[n] : l[n + w], keep = up ? l[n + w] : l[n];
        l[n] = keep + __shfl_xor_sync(0xffffffffu, send, w);
      }
    }
    if (lane < NH) gr.mx[wq][h0 + lane] = l[0];
    group_sync(bar, GT);
    if (wq == 0 && lane < NH) {
      float L = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) L += gr.mx[k][h0 + lane];
      cta_ml[sub * NT + h0 + lane] = make_float2(-gr.nm[h0 + lane], L);
    }
    fence_before();
    tree_join<HD, F::ROWS, SUBS * GT>(a, tid - 128, rowt, cta_ml, fold, min(F::ROWS, a.R - tile * F::ROWS), C, rank, nclusters);
  }
  // past the join's barriers nobody reads tensor memory
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(F::TMEM_COLS) : "memory");
  }
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

template <bool I8, int SUBS>
static cudaError_t launch(TreeArgs a, int tiles, int units, int64_t most, int* err, cudaStream_t s) {
  using F = Cfg<I8, SUBS>;
  auto kern = tree_tc_kernel<I8, SUBS>;
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
    return one ? ttc::launch<true, 1>(a, tiles, units, most, err, s) : ttc::launch<true, 2>(a, tiles, units, most, err, s);
  return one ? ttc::launch<false, 1>(a, tiles, units, most, err, s) : ttc::launch<false, 2>(a, tiles, units, most, err, s);
}

}  // namespace odi_cuda
