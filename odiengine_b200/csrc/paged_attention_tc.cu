// paged_attention_tc.cu -- attention of chunks of new tokens over a paged cache on
// the sm_100a tensor cores (tcgen05.mma, accumulators in tensor memory).
//
// An item is up to 128 or 256 rows (new tokens * heads per kv head) of one request
// and kv head, as one half or two halves of 128 whose work alternates (with one half
// the other CTA of the SM alternates with it):
//
//   S [128 rows x 64 positions] = Q K^T     Q and K in shared memory
//   O [128 rows x head_dim]    += P V       P in tensor memory, where S was
//
//   warps 0-3 of a half  softmax: thread = row
//   then four more       the TMA producer (K and V tiles of 64 positions, page by
//                        page); two that issue the products, one a half, of which the
//                        first holds the tensor memory; one that brings Q
//
// Each half has two S, so that the scores of the next tile are there when the
// weights of this one are done.  (One S of 128 positions a half, which leaves the
// tensor core no more than the other half's work during a softmax: 2048 tokens of
// 64/8 heads over 14,001 positions took 3400 cycles per 128 positions.)  The running
// reference of a row moves only when a weight would pass 2^8, so O is rescaled a few
// times per row.
//
// 2048 tokens of 64/8 heads over 14,001 positions: 955 to 980 us, 1.03 to 1.05 PFLOP/s,
// at 1.6 GHz under the 1 kW power cap; 2048 over 4000 301 us, with distance biases 352,
// with a cap 610 (its second exponential and a reciprocal per score).  What bounds it
// is the softmax: a step of 64 positions takes 0.9 to 1.3 us, of which the products
// are half.  An item takes another 4 to 5 us (queries, first scores, epilogue), a
// piece of one that is cut as much again for its join: 2048 tokens alone 90 us, seven
// prompts of 333 to 1200 tokens of 32/32 heads of 64 dims with biases 91, without 67;
// 16 tokens over 30,000 positions 55.
//
// An fp32 output takes the weights as two 16-bit parts, the second where the other half
// of S was, and a second product: 2048 tokens over 14,001 positions 1190 us, 977 with
// one part, alone 112 and 105 (off by 5e-6 of the output's norm, 1.4e-3 with one).
//
// Every wait is bounded; a role whose wait gives up sets the error word and
// leaves its loop, and the CTA ends at one barrier that every role reaches.
#include "paged_attention.cuh"
#include "pdl_launch.cuh"

namespace odi_cuda {
namespace ptc {

constexpr int TILE = 64, HALF_ROWS = 128;
// Of eight pairs of weights one is exponentiated on the FMA pipe.  The loop over 64
// scores of a row, two warps per scheduler: 933 cycles so, 1188 without, 964 with
// three; without the order that the volatile statements keep 1290.
constexpr int ON_FMA = 1;
__device__ __forceinline__ float ex2_here(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// NH: halves of an item.  One: two CTAs per SM; two: one.
template <int HD, int NH>
struct Cfg {
  static constexpr int PLANE = TILE * 128, SLOT = HD / 64 * PLANE;      // K or V of one tile, in planes of 64 dims
  static constexpr int Q_PLANE = HALF_ROWS * 128, Q_HALF = HD / 64 * Q_PLANE;
  static constexpr int ST = (HD == 128 ? 4 : NH == 1 ? 8 : 6) * NH;
  static_assert(ST / 2 < 8, "v_clean");
  static constexpr int Q_OFF = ST * SLOT;
  static constexpr int STAGE_OFF = Q_OFF + NH * Q_HALF, STAGE = HD == 128 ? 32 * 64 : 0;  // of a warp: 64 bytes of 32 rows of the output
  static constexpr int SMEM = STAGE_OFF + 4 * NH * STAGE + 1024;           // + alignment slack
  static constexpr int ROWS = NH * HALF_ROWS, THREADS = NH * 128 + 128, PER_SM = 2 / NH;
  static_assert(PER_SM * (SMEM + 2048) <= 228 * 1024, "shared memory, with 1 KB static and 1 KB of the system's");
  // the launch's registers are shared out anew: a softmax thread holds a tile's scores
  // and weights
  static constexpr int REGS_LAUNCH = NH == 1 ? 128 : 168, REGS_FEW = 72, REGS_SOFT = NH == 1 ? 184 : 216;
  static_assert(128 * REGS_FEW + 128 * NH * REGS_SOFT <= THREADS * REGS_LAUNCH, "register split");
  // tensor memory: two S per half, then an O per half
  static constexpr int O_COL = NH * 128, COLS = NH * 256;
};

__device__ __forceinline__ uint64_t desc(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
template <bool BF>
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn) {
  // D fp32 | A, B f16 (0) or bf16 (1) | B MN-major | N / 8 | M / 16 = 8
  return (1u << 4) | (BF ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}
// Tensor memory of the warp's 32 rows, 16 or 64 columns.  Loads and wait are one
// statement: no use of a register can move ahead of the wait.
#define PT_OUT8(r) "=r"((r)[0]), "=r"((r)[1]), "=r"((r)[2]), "=r"((r)[3]), "=r"((r)[4]), "=r"((r)[5]), "=r"((r)[6]), "=r"((r)[7])
#define PT_OUT32(r) PT_OUT8(r), PT_OUT8((r) + 8), PT_OUT8((r) + 16), PT_OUT8((r) + 24)
#define PT_IN8(r) "r"((r)[0]), "r"((r)[1]), "r"((r)[2]), "r"((r)[3]), "r"((r)[4]), "r"((r)[5]), "r"((r)[6]), "r"((r)[7])
#define PT_IN32(r) PT_IN8(r), PT_IN8((r) + 8), PT_IN8((r) + 16), PT_IN8((r) + 24)
__device__ __forceinline__ void ld16(uint32_t (&r)[16], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : PT_OUT8(r), PT_OUT8((r) + 8)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void st16(const uint32_t* r, uint32_t addr) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::PT_IN8(r),
               PT_IN8((r) + 8), "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ld64(uint32_t (&r)[64], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : PT_OUT32(r), PT_OUT32((r) + 32)
      : "r"(addr), "r"(addr + 32)
      : "memory");
}
__device__ __forceinline__ void st32(const uint32_t* r, uint32_t addr) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::PT_IN32(r),
      "r"(addr)
      : "memory");
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN if one of them is
  float m;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
// 2^x of two scores on the FMA pipe, which has room where the special function unit
// (16 a cycle and SM) has none: x = n + f with n whole and |f| <= 1/2, 2^f as the
// polynomial of degree 5 with the least largest relative error (2^-23.8) among those
// that are 1 at 0, n into the exponent.  Below 2^-126 the result is 0.
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  x.x = fmaxf(x.x, -127.f), x.y = fmaxf(x.y, -127.f);
  constexpr float M = 12582912.f;  // 1.5 * 2^23: adding it rounds to whole numbers
  const float2 t = __fadd2_rn(x, make_float2(M, M));
  const float2 n = __fadd2_rn(t, make_float2(-M, -M));
  const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
  constexpr float C1 = 0.6931465864181519f, C2 = 0.24022166430950165f, C3 = 0.055510472506284714f, C4 = 0.009674952365458012f,
                  C5 = 0.0013202981790527701f;
  float2 p = __ffma2_rn(f, make_float2(C5, C5), make_float2(C4, C4));
  p = __ffma2_rn(p, f, make_float2(C3, C3));
  p = __ffma2_rn(p, f, make_float2(C2, C2));
  p = __ffma2_rn(p, f, make_float2(C1, C1));
  p = __ffma2_rn(p, f, make_float2(1.f, 1.f));
  return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23)),
                     __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23)));
}
// What a score goes through: nothing but the scale; a distance bias; a cap (and a bias).
enum { PLAIN = 0, BIAS = 1, CAP = 2 };

struct Piece {
  PagedPiece p;
  int end[2];  // tiles of the unit that each half of its rows sees
};
struct Bars {
  uint64_t full[12], empty[12];
  uint64_t s_full[2][2], p_full[2][2];  // of a half's two S
  uint64_t q_full[2], q_empty[2], pv_done[2][2];    // in turn too: a half can wait two products ahead
  uint64_t v_clean[8];  // in turn: a half can be ahead of the other by the tiles that the ring holds
  uint64_t d_full[2], d_empty[2], join, drain[2];
};

template <typename T, int HD, int MODE, int NH, bool OUT32>
__global__ void __launch_bounds__(Cfg<HD, NH>::THREADS, Cfg<HD, NH>::PER_SM)
    paged_tc_kernel(const __grid_constant__ PagedAttnArgs a, const __grid_constant__ CUtensorMap kmap,
                    const __grid_constant__ CUtensorMap vmap, const __grid_constant__ CUtensorMap qmap) {
  using F = Cfg<HD, NH>;
  using H = Half16<T>;
  constexpr int ST = F::ST, PLANES = HD / 64, ROWS = F::ROWS;
  constexpr float MOVE = H::BELOW + PAGED_MOVE;
  constexpr int PRODUCER = 4 * NH, PRODUCTS = PRODUCER + 1, LOADER = PRODUCER + 3;  // warps
  // With a distance bias a long piece goes from its last tile to its first: scores
  // only fall that way, and the reference stays where the first tiles put it (2048
  // tokens over 4000 positions 396 us, 492 the other way).  Otherwise the tiles that
  // not every row sees whole come last, when their V is there (seven prompts, of 5 to
  // 19 tiles: 104 us, 116 the other way).
  auto downward = [](const PagedPiece& p) { return MODE == BIAS && p.t1 - p.t0 > 24; };
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ Bars bars;
  __shared__ Piece pieces[2];
  __shared__ uint32_t tmem_slot;
  __shared__ PagedFound found;
  __shared__ int is_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  pdl_launch_dependents();
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) mbar_init(&bars.full[i], 1), mbar_init(&bars.empty[i], NH);
    for (int i = 0; i < 2; ++i) {
      for (int b = 0; b < 2; ++b) mbar_init(&bars.s_full[i][b], 1), mbar_init(&bars.p_full[i][b], 128);
      mbar_init(&bars.q_full[i], 1);
      mbar_init(&bars.q_empty[i], 1);
      mbar_init(&bars.pv_done[i][0], 1), mbar_init(&bars.pv_done[i][1], 1);
      mbar_init(&bars.d_full[i], 1);
      mbar_init(&bars.d_empty[i], 5 * NH + 1);
    }
    for (int i = 0; i < 8; ++i) mbar_init(&bars.v_clean[i], 128);
    mbar_init(&bars.join, 128 * NH);
    mbar_init(&bars.drain[0], 1), mbar_init(&bars.drain[1], 1);
    prefetch_map(&kmap), prefetch_map(&vmap);
    fence_mbar_init();
  }
  if (warp == PRODUCTS) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(F::COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_wait();
  PagedRun run;
  const bool any = run_begin(a, run, &found);  // has a barrier, unless it returns false in all threads
  const int P = a.c.page_size;
  auto wait = [&](uint64_t* bar, int phase) { return mbar_wait(bar, phase & 1, a.err, ERR_PAGED_WAIT); };

  if (warp >= PRODUCER) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F::REGS_FEW));
  if (any && warp == PRODUCER) {
    // ---- producer: K0 K1 V0 K2 V1 ... V of a piece, as the products want them
    const int BR = min(P, TILE), boxes = TILE / BR;
    const int box = lane / PLANES, plane = lane % PLANES;
    const int rows_all = a.c.num_pages * a.c.kv_heads * P;
    int n = 0, k = 0;  // tiles (of K or V) and pieces so far
    bool ok = true;
    while (ok && run.x < run.end) {
      const PagedPiece p = run_piece(a, run, ROWS);
      const int len = p.it.len;
      const bool down = downward(p);
      if (p.t1 <= p.t0) break;
      PagedNames names(a, p, TILE, down);
      if (k >= 2 && !wait(&bars.d_empty[k & 1], k / 2 - 1)) break;
      if (lane == 0) {
        Piece& d = pieces[k & 1];
        d.p = p;
        const int all = min(ROWS, (len - p.it.past) * a.G - p.it.i * ROWS);
        for (int h = 0; h < NH; ++h) {
          const int last_row = p.it.i * ROWS + min(all, (h + 1) * HALF_ROWS) - 1;
          const int tiles = (paged_limit(p.it.past, pa_token(a, last_row), len, p.it.prefix) + TILE - 1) / TILE;
          d.end[h] = all > h * HALF_ROWS ? max(p.t0, min(p.t1, tiles)) : p.t0;
        }
        mbar_arrive(&bars.d_full[k & 1]);
      }
      ++k;
      if (run.x < run.end) run_next(a, run);
      int y_next = 0, live_next = 0;  // of the tile whose K went last, for its V
      const int tiles = p.t1 - p.t0;
      for (int i = 0; ok && i <= tiles; ++i) {
        const int y_v = y_next, live_v = live_next;
        if (i < tiles) {
          const int t = down ? p.t1 - 1 - i : p.t0 + i, pos = t * TILE + box * BR;
          live_next = min(boxes, (len - t * TILE + BR - 1) / BR);
          const int page = names.at(pos >> a.c.page_shift);
          y_next = (int)(((unsigned)page * a.c.kv_heads + p.kvh) * P) + (pos & (P - 1));
          if (box < live_next && (unsigned)page >= (unsigned)a.c.num_pages) {  // names no page: zeros, and the error word
            y_next = rows_all;
            atomicOr(a.err, ERR_PAGED_PAGE);
          }
        }
        for (int v = 0; v < 2; ++v) {
          if (v ? i == 0 : i == tiles) continue;
          const int s = n % ST, live = v ? live_v : live_next, y = v ? y_v : y_next;
          if (n >= ST && !wait(&bars.empty[s], n / ST - 1)) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_arrive_expect_tx(&bars.full[s], live * BR * HD * 2);
          __syncwarp();
          if (box < live)
            pa_tma(smem + s * F::SLOT + plane * F::PLANE + box * BR * 128, v ? &vmap : &kmap, plane * 64, y, &bars.full[s]);
          ++n;
        }
      }
    }
    if (k < 2 || wait(&bars.d_empty[k & 1], k / 2 - 1)) {
      if (lane == 0) {
        pieces[k & 1].p.last = 1;
        mbar_arrive(&bars.d_full[k & 1]);
      }
    }
    for (int i = max(0, n - ST); i < n; ++i) wait(&bars.full[i % ST], i / ST);  // no copy outlives the CTA
  } else if (any && warp >= PRODUCTS && warp < PRODUCTS + NH) {
    // ---- products of one half
    const int h = warp - PRODUCTS;
    const uint32_t ring = smem_u32(smem), q = ring + F::Q_OFF + h * F::Q_HALF, s_col = tmem + h * 128, o_col = tmem + F::O_COL + h * 128;
    constexpr uint32_t ID_S = idesc<H::BF>(TILE, false), ID_O = idesc<H::BF>(HD, true);
    int n = 0, c_clean = 0, c_q = 0, c_s = 0, c_p = 0;  // tiles of the half so far: its S in turn
    bool ok = true;
    for (int k = 0; ok; ++k) {
      if (!wait(&bars.d_full[k & 1], k / 2)) break;
      const Piece& d = pieces[k & 1];
      if (d.p.last) break;
      const int tiles = d.p.t1 - d.p.t0, mine = d.end[h] - d.p.t0;
      const bool down = downward(d.p);
      const int first = down ? tiles - mine : 0, end = down ? tiles : mine;  // the half's tiles in the piece's order
      const int clean = max(0, d.p.t1 - max(d.p.t0, d.p.least / TILE)), c0 = down ? 0 : tiles - clean;  // those that V is checked in
      if (mine > 0) ok = wait(&bars.q_full[h], c_q++);
      // tile i of the piece: K is load 0, 1, 3, 5 ..., V load 2, 4, ... and the last
      for (int i = -2; ok && i < tiles; ++i) {
        const int nk = n + (i + 2 ? 2 * (i + 2) - 1 : 0), nv = n + min(2 * i + 2, 2 * tiles - 1);
        if (i >= first && i < end && i >= 0) {
          const int b = c_p & 1;
          ok = wait(&bars.p_full[h][b], c_p >> 1) && wait(&bars.full[nv % ST], nv / ST);
          const int cc = c_clean + i - c0;
          if (ok && i >= c0 && i < c0 + clean) ok = wait(&bars.v_clean[cc & 7], cc >> 3);
          if (!ok) break;
          ++c_p;
          fence_after();
          if (elect_one()) {
            const uint64_t v = desc(ring + nv % ST * F::SLOT, F::PLANE);
#pragma unroll
            for (int ks = 0; ks < TILE / 16; ++ks) mma_ts(o_col, s_col + b * 64 + ks * 8, v + ks * (2048 >> 4), ID_O, i > first || ks > 0);
            if (OUT32) {
#pragma unroll
              for (int ks = 0; ks < TILE / 16; ++ks) mma_ts(o_col, s_col + b * 64 + 32 + ks * 8, v + ks * (2048 >> 4), ID_O, 1);
            }
            commit(&bars.pv_done[h][b]);
            commit(&bars.empty[nv % ST]);
          }
          __syncwarp();
        } else if (i >= 0) {  // not before it is there: the slot's next tile has a release of its own
          ok = wait(&bars.full[nv % ST], nv / ST);
          if (!ok) break;
          if (lane == 0) mbar_arrive(&bars.empty[nv % ST]);
        }
        if (i + 2 >= tiles) continue;
        ok = wait(&bars.full[nk % ST], nk / ST);
        if (i + 2 >= first && i + 2 < end) {
          // S goes where the P of two tiles before was: an order that nothing but a wait gives
          const int b = c_s & 1;
          if (ok && c_s > 1) ok = wait(&bars.pv_done[h][b], (c_s >> 1) - 1);
          if (!ok) break;
          ++c_s;
          fence_after();
          if (elect_one()) {
            const uint64_t qd = desc(q, 0), kd = desc(ring + nk % ST * F::SLOT, 0);
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks)
              mma_ss(s_col + b * 64, qd + (((ks / 4) * F::Q_PLANE + (ks % 4) * 32) >> 4), kd + (((ks / 4) * F::PLANE + (ks % 4) * 32) >> 4),
                     ID_S, ks > 0);
            commit(&bars.s_full[h][b]);
            commit(&bars.empty[nk % ST]);
            if (i + 3 == end) commit(&bars.q_empty[h]);
          }
          __syncwarp();
        } else if (ok && lane == 0) {
          mbar_arrive(&bars.empty[nk % ST]);
        }
      }
      n += 2 * tiles, c_clean += clean;
      if (lane == 0) mbar_arrive(&bars.d_empty[k & 1]);
    }
    // products in flight end before the tensor memory goes
    if (elect_one()) commit(&bars.drain[h]);
    __syncwarp();
    wait(&bars.drain[h], 0);
  } else if (any && warp == LOADER) {
    // ---- Q of a piece, as soon as the products of the piece before have read theirs.
    // 128 rows are a box of whole tokens where the group divides 128; else 16-byte
    // pieces, HD / 8 to a row (a half of 128 dims takes 4 us so, 1 as boxes).  Rows that
    // there are none of are zero or another request's: nothing of them is kept.
    constexpr int PER = HD / 8;
    const int ch = lane % PER, r0 = lane / PER;
    const T* q = static_cast<const T*>(a.q) + ch * 8;
    int c_q[2] = {0, 0};
    bool ok = true;
    for (int k = 0; ok; ++k) {
      if (!wait(&bars.d_full[k & 1], k / 2)) break;
      const Piece& d = pieces[k & 1];
      const PagedPiece& p = d.p;
      if (p.last) break;
      for (int h = 0; ok && h < NH; ++h) {
        if (d.end[h] <= p.t0) continue;
        if (c_q[h]) ok = wait(&bars.q_empty[h], c_q[h] - 1);
        if (!ok) break;
        ++c_q[h];
        if (a.q_boxes) {
          if (lane == 0) {
            const int token = p.it.start + (p.it.i * ROWS + h * HALF_ROWS) / a.G;
            mbar_arrive_expect_tx(&bars.q_full[h], F::Q_HALF);
#pragma unroll
            for (int pl = 0; pl < PLANES; ++pl)
              pa_tma_3d(smem + F::Q_OFF + h * F::Q_HALF + pl * F::Q_PLANE, &qmap, pl * 64, p.kvh * a.G, token, &bars.q_full[h]);
          }
          continue;
        }
        const uint32_t dst = smem_u32(smem + F::Q_OFF + h * F::Q_HALF + (ch >> 3) * F::Q_PLANE);
        const T* base = q + p.it.start * a.ld_q + (int64_t)p.kvh * a.G * HD;
        const int R0 = p.it.i * ROWS + h * HALF_ROWS, live = p.rows - h * HALF_ROWS;
#pragma unroll 4
        for (int r = r0; r < HALF_ROWS; r += 32 / PER) {
          const int tk = pa_token(a, R0 + r);
          const T* src = r < live ? base + tk * a.ld_q + (R0 + r - tk * a.G) * HD : q;
          const uint32_t to = dst + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
          if (a.vec) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(r < live ? 16 : 0) : "memory");
          } else {
            const unsigned* s4 = reinterpret_cast<const unsigned*>(src);
            uint4 x = make_uint4(0, 0, 0, 0);
            if (r < live) x = make_uint4(__ldcg(s4), __ldcg(s4 + 1), __ldcg(s4 + 2), __ldcg(s4 + 3));
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.q_full[h]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.d_empty[k & 1]);
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F::REGS_SOFT));
    // ---- softmax: thread = row
    const int h = warp >> 2, hr = tid & 127, row = tid;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_addr = tmem + lanes + F::O_COL + h * 128;
    int n = 0, c_s = 0, c_pv = 0, c_clean = 0, joins = 0;
    bool ok = any;
    for (int k = 0; ok; ++k) {
      if (!wait(&bars.d_full[k & 1], k / 2)) break;
      Piece& d = pieces[k & 1];
      if (d.p.last) break;
      const PagedPiece& p = d.p;
      const int rows = p.rows, t0 = p.t0, t1 = p.t1, t_end = d.end[h];
      const bool mine = t_end > t0, down = downward(p);
      const int clean = max(0, t1 - max(t0, p.least / TILE));  // tiles that not every row sees whole
      const int R = p.it.i * ROWS + row, token = pa_token(a, R), head = p.kvh * a.G + R - token * a.G;
      const int lim = row < rows ? paged_limit(p.it.past, token, p.it.len, p.it.prefix) : 0;
      // positions below it are seen by all rows of this half
      const int least_h = paged_limit(p.it.past, pa_token(a, p.it.i * ROWS + h * HALF_ROWS), p.it.len, p.it.prefix);
      const float slope = MODE != PLAIN && a.slopes && row < rows ? __ldg(a.slopes + head) * 1.4426950408889634f : 0.f;
      float ref = -INFINITY;
      float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
      for (int i = 0; i < t_end - t0; ++i) {
        const int t = down ? t_end - 1 - i : t0 + i;
        const int b = c_s & 1;
        const uint32_t s_addr = tmem + lanes + h * 128 + b * 64;
        ok = wait(&bars.s_full[h][b], c_s >> 1);
        ++c_s;
        if (!ok) break;
        __syncwarp();
        fence_after();
        uint32_t s[64];
        ld64(s, s_addr);
        const int col0 = t * TILE;
        if (MODE == CAP) {
#pragma unroll
          for (int c = 0; c < 64; ++c) s[c] = __float_as_uint(pa_cap(__uint_as_float(s[c]) * a.scale_log2, a.cap_log2));
        }
        if (MODE == BIAS || (MODE == CAP && a.slopes)) {
          const int away = p.it.past + token - col0;  // the row's own column
          const float scale = MODE == CAP ? 1.f : a.scale_log2, b0 = -slope * (float)away;
          const float2 sc2 = make_float2(scale, scale);
#pragma unroll
          for (int c = 0; c < 64; c += 2) {
            const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sc2,
                                        make_float2(fmaf(slope, (float)c, b0), fmaf(slope, (float)(c + 1), b0)));
            s[c] = __float_as_uint(x.x), s[c + 1] = __float_as_uint(x.y);
          }
          if (__any_sync(0xffffffffu, lim - col0 > away + 1 && away < 63)) {
            // part of the tile lies behind the row and is seen: it is as far the other way
#pragma unroll
            for (int c = 0; c < 64; ++c)
              if (c > away) s[c] = __float_as_uint(fmaf(-2.f * slope, (float)(c - away), __uint_as_float(s[c])));
          }
        }
        if (col0 + 64 > least_h) {
          const int rel = lim - col0;  // columns that the row sees
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (c >= rel) s[c] = 0xff800000u;
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 64; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) m4[e] = max3(m4[e], __uint_as_float(s[c + 2 * e]), __uint_as_float(s[c + 2 * e + 1]));
        const float scale = MODE == PLAIN ? a.scale_log2 : 1.f;
        const float mx = max3(max3(m4[0], m4[1], m4[2]), m4[3], -INFINITY) * scale;
        const bool move = !(mx <= ref + MOVE) && ref == ref;  // a row that is NaN stays so
        if (__any_sync(0xffffffffu, move)) {
          // a NaN among the scores, or +inf, leaves no weight: the row is NaN from here on
          const float top = !move ? ref : mx == INFINITY ? __int_as_float(0x7fc00000) : mx - H::BELOW;
          const float f = top == ref ? 1.f : pa_ex2(ref - top);
          ref = top;
          sum[0].x *= f, sum[0].y *= f, sum[1].x *= f, sum[1].y *= f;
          if (i > 0) {
            ok = wait(&bars.pv_done[h][(c_pv - 1) & 1], (c_pv - 1) >> 1);
            if (!ok) break;
            __syncwarp();
            fence_after();
#pragma unroll 1
            for (int c = 0; c < HD; c += 16) {
              uint32_t o[16];
              ld16(o, o_addr + c);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              st16(o, o_addr + c);
            }
          }
        }
        const float nref = ref == -INFINITY ? 0.f : -ref;
        const float2 sc2 = make_float2(scale, scale), nr2 = make_float2(nref, nref);
        // eight pairs at a time, sums and packing one group behind
        float2 w[2][8];
        uint32_t rest[OUT32 ? 32 : 1];  // what the rounding of the weights left
#pragma unroll
        for (int g = 0; g <= 4; ++g) {
          if (g < 4) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              w[g & 1][e] = __ffma2_rn(make_float2(__uint_as_float(s[16 * g + 2 * e]), __uint_as_float(s[16 * g + 2 * e + 1])), sc2, nr2);
#pragma unroll
            for (int e = 0; e < 8 - ON_FMA; ++e) w[g & 1][e] = make_float2(ex2_here(w[g & 1][e].x), ex2_here(w[g & 1][e].y));
#pragma unroll
            for (int e = 8 - ON_FMA; e < 8; ++e) w[g & 1][e] = exp2_fma(w[g & 1][e]);
          }
          if (g > 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float2 v = w[(g - 1) & 1][e];
              sum[e & 1] = __fadd2_rn(sum[e & 1], v);
              if constexpr (OUT32) s[8 * (g - 1) + e] = H::split(v, rest[8 * (g - 1) + e]);
              else s[8 * (g - 1) + e] = H::pack(v.x, v.y);
            }
          }
        }
        st32(s, s_addr);
        if constexpr (OUT32) st32(rest, s_addr + 32);
        wait_st();
        if (t >= t1 - clean && (NH == 1 || h == (t < d.end[1] ? 1 : 0))) {
          // the last half at work takes what is not finite out of V: thread = position, half its dims
          const int ip = down ? t1 - 1 - t : t - t0, cc = c_clean + (down ? ip : ip - (t1 - t0 - clean));
          const int iv = n + min(2 * ip + 2, 2 * (t1 - t0) - 1), r = hr & 63, pos = t * TILE + r;
          ok = wait(&bars.full[iv % ST], iv / ST);
          if (!ok) break;
          if (pos >= p.least) {
            uint8_t* v = smem + iv % ST * F::SLOT + r * 128;
            auto at = [&](int e) {
              const int ch = (hr >> 6) * (HD / 16) + e;
              return reinterpret_cast<uint4*>(v + (ch >> 3) * F::PLANE + (((ch & 7) ^ (r & 7)) << 4));
            };
            uint4 z[HD / 16];
#pragma unroll
            for (int e = 0; e < HD / 16; ++e) z[e] = *at(e);
            uint32_t zero = 0;  // 0 times all values: 0 if every one is finite
#pragma unroll
            for (int e = 0; e < HD / 16; ++e) {
              zero = H::times0(z[e].x, zero), zero = H::times0(z[e].y, zero);
              zero = H::times0(z[e].z, zero), zero = H::times0(z[e].w, zero);
            }
            if (zero & 0x7fff7fffu) {
              if (pos < p.it.len) d.p.poison = 1;
#pragma unroll 1
              for (int e = 0; e < HD / 16; ++e) {
                uint32_t* x = reinterpret_cast<uint32_t*>(at(e));
                for (int i = 0; i < 4; ++i) {
                  uint32_t y = x[i];
                  if ((y & H::EXP) == H::EXP) y &= 0xffff0000u;
                  if ((y & (H::EXP << 16)) == H::EXP << 16) y &= 0xffffu;
                  x[i] = y;
                }
              }
            }
          }
          fence_proxy_async_smem();
          mbar_arrive(&bars.v_clean[cc & 7]);
        }
        fence_before();
        mbar_arrive(&bars.p_full[h][b]);
        ++c_pv;
      }
      if (ok && mine) ok = wait(&bars.pv_done[h][(c_pv - 1) & 1], (c_pv - 1) >> 1);
      if (!ok) break;
      __syncwarp();
      fence_after();
      const float L = ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y)) * (OUT32 ? H::PARTS : 1.f);
      const bool whole = t0 == 0 && t1 == p.it.tiles, fix = p.poison != 0;
      constexpr int STRIDE = ROWS * (HD + 2);
      float* part = piece_part(a, p, blockIdx.x, STRIDE);
      // 16 values of the thread's row from dim c on.  A thread's row is far from its
      // neighbours', so rows go through shared memory, 64 bytes at a time, and four lanes
      // write them to a row.
      const int out_row = row < rows ? 1 : 0;
      int64_t out_at = (int64_t)(p.it.start + token) * a.ld_out + (int64_t)head * HD;
      uint8_t* stage = smem + F::STAGE_OFF + warp * F::STAGE;
      auto chunk = [&](int r, int ch) { return reinterpret_cast<uint4*>(stage + r * 64 + ((ch ^ (r >> 1 & 3)) << 4)); };
      auto flush = [&](int c) {  // the staged values are those from dim c on
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = j * 8 + (lane >> 2), ch = lane & 3;
          const int64_t at = __shfl_sync(0xffffffffu, out_at, r) + c;
          const bool some = __shfl_sync(0xffffffffu, out_row, r);
          const uint4 x = *chunk(r, ch);
          uint32_t* y = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.out) + (at << (OUT32 ? 2 : 1))) + ch * 4;
          if (!some) continue;
          if (a.vec_out) *reinterpret_cast<uint4*>(y) = x;
          else y[0] = x.x, y[1] = x.y, y[2] = x.z, y[3] = x.w;
        }
        __syncwarp();
      };
      auto store = [&](const float (&v)[16], int c) {
        if constexpr (F::STAGE == 0) {
          if (row >= rows) return;
          const int64_t at = (int64_t)(p.it.start + token) * a.ld_out + (int64_t)head * HD + c;
          if (OUT32) {
            float* y = static_cast<float*>(a.out) + at;
            if (a.vec_out) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                reinterpret_cast<float4*>(y)[e] = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
            } else {
#pragma unroll
              for (int e = 0; e < 16; ++e) y[e] = v[e];
            }
          } else {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = H::pack(v[2 * e], v[2 * e + 1]);
            uint32_t* y = reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + at);
            if (a.vec_out) {
#pragma unroll
              for (int e = 0; e < 2; ++e)
                reinterpret_cast<uint4*>(y)[e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) y[e] = w[e];
            }
          }
          return;
        }
        if (OUT32) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *chunk(lane, e) = make_uint4(__float_as_uint(v[4 * e]), __float_as_uint(v[4 * e + 1]), __float_as_uint(v[4 * e + 2]),
                                         __float_as_uint(v[4 * e + 3]));
          flush(c);
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            *chunk(lane, (c >> 3 & 2) + e) = make_uint4(H::pack(v[8 * e], v[8 * e + 1]), H::pack(v[8 * e + 2], v[8 * e + 3]),
                                                        H::pack(v[8 * e + 4], v[8 * e + 5]), H::pack(v[8 * e + 6], v[8 * e + 7]));
          if (c & 16) flush(c - 16);
        }
      };
      if (mine) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll 1
        for (int c = 0; c < HD; c += 16) {
          uint32_t o[16];
          __syncwarp();  // lanes part ways below, at what is not finite and where rows end
          ld16(o, o_addr + c);
          float v[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = __uint_as_float(o[e]);
          if (fix)
            for (int j = max(t0 * TILE, p.least); j < min(t1 * TILE, lim) && j >> a.c.page_shift < a.max_pages; ++j) {
              const int page = __ldcg(a.table + (int64_t)p.it.b * a.max_pages + (j >> a.c.page_shift));
              if ((unsigned)page >= (unsigned)a.c.num_pages) continue;
              const unsigned short* src = reinterpret_cast<const unsigned short*>(a.c.v) +
                                          (((int64_t)page * a.c.kv_heads + p.kvh) * P + (j & (P - 1))) * HD + c;
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const float y = H::up(__ldcg(src + e));
                if (!(fabsf(y) <= 3.402823466e38f)) v[e] += y;
              }
            }
          if (whole) {
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = inv == 0.f ? 0.f : v[e] * inv;  // nothing that weighs nothing
            store(v, c);
          } else {
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              *reinterpret_cast<float4*>(part + ((c + e) / 4 * ROWS + row) * 4) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          }
        }
        fence_before();
      }
      if (!whole) {
        const bool warp_rows = (row & ~31) < rows;
        if (warp_rows) *reinterpret_cast<float2*>(part + ROWS * HD + 2 * row) = make_float2(ref, L);
        for (PagedJoin join = join_first(a, p, 8);; join = join_next(a, p)) {
          mbar_arrive(&bars.join);
          ok = wait(&bars.join, joins++);
          if (!ok) break;
          if (tid == 0) {
            __threadfence();
            is_last = atomicAdd(join.counter, 1) == join.n - 1;
            __threadfence();
          }
          mbar_arrive(&bars.join);
          ok = wait(&bars.join, joins++);
          if (!ok || !is_last) break;
          if (warp_rows) {
            auto piece = [&](int q) { return piece_part(a, p, join.first + q * join.step, STRIDE); };
            float* to = piece_part(a, p, join.first, STRIDE);
            float top = -INFINITY, all = 0.f;
#pragma unroll 4
            for (int q = 0; q < join.n; ++q) top = max3(top, __ldcg(reinterpret_cast<const float2*>(piece(q) + ROWS * HD + 2 * row)).x, -INFINITY);
#pragma unroll 1
            for (int d0 = 0; d0 < HD; d0 += 32) {
              float v[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = 0.f;
              all = 0.f;
#pragma unroll 2
              for (int q = 0; q < join.n; ++q) {
                const float* src = piece(q);
                const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + ROWS * HD + 2 * row));
                float4 x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = __ldcg(reinterpret_cast<const float4*>(src + ((d0 / 4 + e) * ROWS + row) * 4));
                // a piece in which the row saw nothing left no sums
                const bool some = !(ml.x == -INFINITY && ml.y == 0.f);
                const float f = ml.x == top ? 1.f : pa_ex2(ml.x - top);
                if (some) {
                  all = fmaf(ml.y, f, all);
#pragma unroll
                  for (int e = 0; e < 8; ++e) {
                    v[4 * e] = fmaf(x[e].x, f, v[4 * e]), v[4 * e + 1] = fmaf(x[e].y, f, v[4 * e + 1]);
                    v[4 * e + 2] = fmaf(x[e].z, f, v[4 * e + 2]), v[4 * e + 3] = fmaf(x[e].w, f, v[4 * e + 3]);
                  }
                }
              }
              if (join.final) {
                const float inv = all == 0.f ? 0.f : 1.f / all;
#pragma unroll
                for (int g = 0; g < 32; g += 16) {
                  float y[16];
#pragma unroll
                  for (int e = 0; e < 16; ++e) y[e] = inv == 0.f ? 0.f : v[g + e] * inv;
                  store(y, d0 + g);
                }
              } else {  // in its first piece's place, whose row no other thread reads
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  *reinterpret_cast<float4*>(to + ((d0 / 4 + e) * ROWS + row) * 4) =
                      make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
              }
            }
            if (!join.final) *reinterpret_cast<float2*>(to + ROWS * HD + 2 * row) = make_float2(top, all);
          }
          if (tid == 0) *join.counter = 0;
          if (join.final) break;
        }
        if (!ok) break;
      }
      n += 2 * (t1 - t0), c_clean += clean;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.d_empty[k & 1]);
    }
  }
  fence_before();
  __syncthreads();
  if (warp == PRODUCTS) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(F::COLS) : "memory");
  }
}

template <typename T, int HD, int MODE, int NH, bool OUT32>
static cudaError_t launch(PagedAttnArgs& a, cudaStream_t s) {
  using F = Cfg<HD, NH>;
  auto kern = paged_tc_kernel<T, HD, MODE, NH, OUT32>;
  CUtensorMap maps[3];
  if (cudaError_t e = paged_maps(a.c, TILE, false, maps)) return e;
  // whole tokens of a group: boxes of 64 dims, G heads, 128 / G tokens
  a.q_boxes = a.vec && HALF_ROWS % a.G == 0;
  maps[2] = maps[0];
  if (a.q_boxes)
    if (cudaError_t e = paged_q_map(a, HALF_ROWS / a.G, &maps[2])) return e;
  static PagedReady ready;
  if (cudaError_t e = ready.set((const void*)kern, F::SMEM)) return e;
  return launch_pdl_smem(kern, dim3(paged_ctas(F::ROWS)), dim3(F::THREADS), F::SMEM, s, a, maps[0], maps[1], maps[2]);
}

}  // namespace ptc

cudaError_t launch_paged_tc(PagedAttnArgs& a, int rows, cudaStream_t s) {
  using namespace ptc;
  static_assert(Cfg<128, 2>::ROWS == PAGED_ROWS_MAX, "the scratch's pieces");
  const int mode = a.cap_log2 != 0.f ? CAP : a.slopes ? BIAS : PLAIN;
  auto by_mode = [&](auto t, auto hd, auto nh, auto out) {
    using T = decltype(t);
    constexpr int HD = decltype(hd)::value, NH = decltype(nh)::value;
    constexpr bool OUT32 = decltype(out)::value;
    return mode == CAP    ? launch<T, HD, CAP, NH, OUT32>(a, s)
           : mode == BIAS ? launch<T, HD, BIAS, NH, OUT32>(a, s)
                          : launch<T, HD, PLAIN, NH, OUT32>(a, s);
  };
  auto by_out = [&](auto t, auto hd, auto nh) {
    return a.out32 ? by_mode(t, hd, nh, std::true_type{}) : by_mode(t, hd, nh, std::false_type{});
  };
  auto by_rows = [&](auto t, auto hd) {
    return rows == HALF_ROWS ? by_out(t, hd, std::integral_constant<int, 1>{}) : by_out(t, hd, std::integral_constant<int, 2>{});
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (a.c.dtype == ODI_CUDA_PAGED_BF16) return a.c.hd == 128 ? by_rows(__nv_bfloat16{}, D128{}) : by_rows(__nv_bfloat16{}, D64{});
  return a.c.hd == 128 ? by_rows(__half{}, D128{}) : by_rows(__half{}, D64{});
}

}  // namespace odi_cuda
