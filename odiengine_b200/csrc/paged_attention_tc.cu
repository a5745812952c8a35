// paged_attention_tc.cu -- attention of chunks of new tokens over a paged cache on
// the sm_100a tensor cores (tcgen05.mma, accumulators in tensor memory).
//
// An item is up to 256 rows (new tokens * heads per kv head) of one request and kv
// head, as two halves of 128 whose work alternates:
//
//   S [128 rows x 128 positions] = Q K^T    Q and K in shared memory
//   O [128 rows x head_dim]     += P V      P in tensor memory, where S was
//
//   warps 0-3, 4-7  softmax of the two halves: thread = row
//   warp 8          TMA producer: K and V tiles of 128 positions, page by page
//   warp 9          issues the products; holds the tensor memory
//   warps 10, 11    only make the warpgroup whole, for its registers
//
// While one half is in its softmax the tensor core works for the other.  The
// running reference of a row moves only when a weight would pass 2^8, so O is
// rescaled a few times per row.
//
// Every wait is bounded; a role whose wait gives up sets the error word and
// leaves its loop, and the CTA ends at one barrier that every role reaches.
#include "paged_attention.cuh"
#include "pdl_launch.cuh"

namespace odi_cuda {
namespace ptc {

constexpr int TILE = 128, ROWS = 256, HALF_ROWS = 128, THREADS = 384;
// The launch's registers are shared out anew: a softmax thread holds a row of 128
// scores, the others next to nothing.
constexpr int REGS_LAUNCH = 168, REGS_FEW = 72, REGS_SOFT = 216;
static_assert(128 * REGS_FEW + 256 * REGS_SOFT <= THREADS * REGS_LAUNCH, "register split");
constexpr float MOVE = 8.f;

template <int HD>
struct Cfg {
  static constexpr int PLANE = 128 * 128;               // 128 rows of 128 bytes: half the dims of head_dim 128
  static constexpr int SLOT = HD / 64 * PLANE;          // K or V of one tile, Q of one half
  static constexpr int ST = HD == 128 ? 4 : 8;
  static constexpr int Q_OFF = ST * SLOT;
  static constexpr int SMEM = Q_OFF + 2 * SLOT + 1024;  // + alignment slack
  static constexpr int S_COL = 0, O_COL = 256, COLS = 512;
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
// Tensor memory of the warp's 32 rows, 32 or 128 columns.  Loads and wait are one
// statement: no use of a register can move ahead of the wait.
#define PT_OUT8(r) "=r"((r)[0]), "=r"((r)[1]), "=r"((r)[2]), "=r"((r)[3]), "=r"((r)[4]), "=r"((r)[5]), "=r"((r)[6]), "=r"((r)[7])
#define PT_OUT32(r) PT_OUT8(r), PT_OUT8((r) + 8), PT_OUT8((r) + 16), PT_OUT8((r) + 24)
#define PT_IN8(r) "r"((r)[0]), "r"((r)[1]), "r"((r)[2]), "r"((r)[3]), "r"((r)[4]), "r"((r)[5]), "r"((r)[6]), "r"((r)[7])
#define PT_IN32(r) PT_IN8(r), PT_IN8((r) + 8), PT_IN8((r) + 16), PT_IN8((r) + 24)
__device__ __forceinline__ void ld32(uint32_t (&r)[32], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : PT_OUT32(r)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void ld128(uint32_t (&r)[128], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%128];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%129];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95}, [%130];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127}, [%131];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : PT_OUT32(r), PT_OUT32((r) + 32), PT_OUT32((r) + 64), PT_OUT32((r) + 96)
      : "r"(addr), "r"(addr + 32), "r"(addr + 64), "r"(addr + 96)
      : "memory");
}
__device__ __forceinline__ void st32(const uint32_t* r, uint32_t addr) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::PT_IN32(r),
      "r"(addr)
      : "memory");
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

struct Piece {
  PagedPiece p;
  int end[2];  // tiles of the unit that each half of its rows sees
};
struct Bars {
  uint64_t full[8], empty[8];
  uint64_t q_full[2], s_full[2], p_full[2], pv_done[2], v_clean;
  uint64_t d_full[2], d_empty[2], join, drain;
};

template <typename T, int HD, bool FANCY>
__global__ void __launch_bounds__(THREADS, 1)
    paged_tc_kernel(const __grid_constant__ PagedAttnArgs a, const __grid_constant__ CUtensorMap kmap,
                    const __grid_constant__ CUtensorMap vmap) {
  using F = Cfg<HD>;
  using H = Half16<T>;
  constexpr int ST = F::ST, PLANES = HD / 64;
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
    for (int i = 0; i < ST; ++i) mbar_init(&bars.full[i], 1), mbar_init(&bars.empty[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.q_full[i], 128);
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], 128);
      mbar_init(&bars.pv_done[i], 1);
      mbar_init(&bars.d_full[i], 1);
      mbar_init(&bars.d_empty[i], 9);
    }
    mbar_init(&bars.v_clean, 128);
    mbar_init(&bars.join, 256);
    mbar_init(&bars.drain, 1);
    fence_mbar_init();
  }
  if (warp == 9) {
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

  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_FEW));
  if (any && warp == 8) {
    // ---- producer
    const int BR = min(P, TILE), boxes = TILE / BR;
    const int box = lane / PLANES, plane = lane % PLANES;
    const int rows_all = a.c.num_pages * a.c.kv_heads * P;
    int n = 0, k = 0;  // tiles (of K or V) and pieces so far
    bool ok = true;
    while (ok && run.x < run.end) {
      const PagedPiece p = run_piece(a, run, ROWS);
      const int len = p.it.len;
      PagedNames names(a, p, TILE);
      if (k >= 2 && !wait(&bars.d_empty[k & 1], k / 2 - 1)) break;
      if (lane == 0) {
        Piece& d = pieces[k & 1];
        d.p = p;
        const int all = min(ROWS, (len - p.it.past) * a.G - p.it.i * ROWS);
        for (int h = 0; h < 2; ++h) {
          const int last_row = p.it.i * ROWS + min(all, (h + 1) * HALF_ROWS) - 1;
          const int tiles = (paged_limit(p.it.past, pa_token(a, last_row), len, p.it.prefix) + TILE - 1) / TILE;
          d.end[h] = all > h * HALF_ROWS ? max(p.t0, min(p.t1, tiles)) : p.t0;
        }
        mbar_arrive(&bars.d_full[k & 1]);
      }
      ++k;
      if (run.x < run.end) run_next(a, run);
      for (int t = p.t0; ok && t < p.t1; ++t) {
        const int pos = t * TILE + box * BR;
        const int live = min(boxes, (len - t * TILE + BR - 1) / BR);
        const int page = names.at(pos >> a.c.page_shift);
        int y = (page * a.c.kv_heads + p.kvh) * P + (pos & (P - 1));
        if (box < live && (unsigned)page >= (unsigned)a.c.num_pages) {  // names no page: zeros, and the error word
          y = rows_all;
          atomicOr(a.err, ERR_PAGED_PAGE);
        }
        for (int v = 0; v < 2; ++v, ++n) {
          const int s = n % ST;
          if (n >= ST && !wait(&bars.empty[s], n / ST - 1)) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_arrive_expect_tx(&bars.full[s], live * BR * HD * 2);
          __syncwarp();
          if (box < live)
            pa_tma(smem + s * F::SLOT + plane * F::PLANE + box * BR * 128, v ? &vmap : &kmap, plane * 64, y, &bars.full[s]);
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
  } else if (any && warp == 9) {
    // ---- products
    const uint32_t ring = smem_u32(smem), q = ring + F::Q_OFF;
    constexpr uint32_t ID_S = idesc<H::BF>(TILE, false), ID_O = idesc<H::BF>(HD, true);
    int n = 0, c_clean = 0, c_q[2] = {0, 0}, c_p[2] = {0, 0};
    auto scores = [&](int h, int s) {  // S of half h from the K tile in slot s
      if (elect_one()) {
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          const uint32_t off = (ks / 4) * F::PLANE + (ks % 4) * 32;
          mma_ss(tmem + F::S_COL + h * 128, desc(q + h * F::SLOT + off, 0), desc(ring + s * F::SLOT + off, 0), ID_S, ks > 0);
        }
        commit(&bars.s_full[h]);
      }
      __syncwarp();
    };
    auto release = [&](int s) {
      if (elect_one()) commit(&bars.empty[s]);
      __syncwarp();
    };
    bool ok = true;
    for (int k = 0; ok; ++k) {
      if (!wait(&bars.d_full[k & 1], k / 2)) break;
      const Piece& d = pieces[k & 1];
      if (d.p.last) break;
      const int t0 = d.p.t0, t1 = d.p.t1, least = d.p.least, end0 = d.end[0], end1 = d.end[1];
      auto end = [&](int h) { return h ? end1 : end0; };
      for (int t = t0 - 1; ok && t < t1; ++t) {
        const int sv = (n + 2 * (t - t0) + 1) % ST, iv = (n + 2 * (t - t0) + 1) / ST;
        const int sk = (n + 2 * (t + 1 - t0)) % ST, ik = (n + 2 * (t + 1 - t0)) / ST;
        if (t >= t0) {
          ok = wait(&bars.full[sv], iv);
          if (ok && (t + 1) * TILE > least) ok = wait(&bars.v_clean, c_clean++);
        }
        bool have_k = false;
        for (int h = 0; ok && h < 2; ++h) {
          if (t >= t0 && t < end(h)) {
            ok = wait(&bars.p_full[h], c_p[h]++);
            if (!ok) break;
            fence_after();
            if (elect_one()) {
#pragma unroll
              for (int ks = 0; ks < TILE / 16; ++ks)
                mma_ts(tmem + F::O_COL + h * 128, tmem + F::S_COL + h * 128 + ks * 8, desc(ring + sv * F::SLOT + ks * 2048, F::PLANE),
                       ID_O, t > t0 || ks > 0);
              commit(&bars.pv_done[h]);
            }
            __syncwarp();
          }
          if (t + 1 < end(h)) {
            if (!have_k) ok = wait(&bars.full[sk], ik), have_k = true;
            if (ok && t < t0) ok = wait(&bars.q_full[h], c_q[h]++);
            if (!ok) break;
            fence_after();
            scores(h, sk);
          }
        }
        if (!ok) break;
        if (t >= t0) release(sv);
        if (t + 1 < t1) release(sk);
      }
      n += 2 * (t1 - t0);
      if (lane == 0) mbar_arrive(&bars.d_empty[k & 1]);
    }
    // products in flight end before the tensor memory goes
    if (elect_one()) commit(&bars.drain);
    __syncwarp();
    wait(&bars.drain, 0);
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFT));
    // ---- softmax: thread = row
    const int h = warp >> 2, row = tid;  // row of the item
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + F::S_COL + h * 128, o_addr = tmem + lanes + F::O_COL + h * 128;
    uint8_t* qs = smem + F::Q_OFF + h * F::SLOT;
    int n = 0, c_s = 0, c_pv = 0, joins = 0;
    bool ok = any;
    for (int k = 0; ok; ++k) {
      if (!wait(&bars.d_full[k & 1], k / 2)) break;
      Piece& d = pieces[k & 1];
      if (d.p.last) break;
      const PagedPiece p = d.p;
      const int start = p.it.start, past = p.it.past, len = p.it.len, rows = p.rows, least = p.least;
      const int t0 = p.t0, t1 = p.t1, t_end = d.end[h], end1 = d.end[1];
      const bool mine = t_end > t0;
      const int R = p.it.i * ROWS + row, token = pa_token(a, R), head = p.kvh * a.G + R - token * a.G;
      const int lim = row < rows ? paged_limit(past, token, len, p.it.prefix) : 0;
      // positions below it are seen by all rows of this half
      const int least_h = paged_limit(past, pa_token(a, p.it.i * ROWS + h * HALF_ROWS), len, p.it.prefix);
      const float slope = FANCY && a.slopes && row < rows ? __ldg(a.slopes + head) * 1.4426950408889634f : 0.f;
      if (mine) {
        // Q: 16-byte pieces, HD / 8 to a row
        constexpr int PER = HD / 8;
        const T* q = static_cast<const T*>(a.q);
#pragma unroll 4
        for (int i = tid & 127; i < HALF_ROWS * PER; i += 128) {
          const int r = i / PER, ch = i % PER;
          uint4 x = make_uint4(0, 0, 0, 0);
          if (h * HALF_ROWS + r < rows) {
            const int RR = p.it.i * ROWS + h * HALF_ROWS + r, tk = pa_token(a, RR);
            const T* src = q + (int64_t)(start + tk) * a.ld_q + (int64_t)(p.kvh * a.G + RR - tk * a.G) * HD + ch * 8;
            if (a.vec) {
              x = __ldcg(reinterpret_cast<const uint4*>(src));
            } else {
              const unsigned* s4 = reinterpret_cast<const unsigned*>(src);
              x = make_uint4(__ldcg(s4), __ldcg(s4 + 1), __ldcg(s4 + 2), __ldcg(s4 + 3));
            }
          }
          *reinterpret_cast<uint4*>(qs + (ch >> 3) * F::PLANE + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = x;
        }
        fence_proxy_async_smem();
        mbar_arrive(&bars.q_full[h]);
      }
      float ref = -INFINITY;
      float2 sum = make_float2(0.f, 0.f);
      for (int t = t0; t < t_end; ++t) {
        ok = wait(&bars.s_full[h], c_s++);
        if (!ok) break;
        fence_after();
        uint32_t s[128];
        ld128(s, s_addr);
        float mx = -INFINITY;
        const int rel = lim - t * TILE;
        if (FANCY) {
          const int away = past + token - t * TILE;
#pragma unroll
          for (int c = 0; c < 128; ++c) {
            float x = __uint_as_float(s[c]) * a.scale_log2;
            if (a.cap_log2 != 0.f) x = a.cap_log2 * pa_tanh(x);
            x = fmaf(-slope, (float)abs(away - c), x);
            s[c] = __float_as_uint(x);
          }
        }
        if ((t + 1) * TILE > least_h) {
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c >= rel) s[c] = 0xff800000u;
        }
#pragma unroll
        for (int c = 0; c < 128; ++c) mx = fmaxf(mx, __uint_as_float(s[c]));
        const float scale = FANCY ? 1.f : a.scale_log2;
        mx *= scale;
        const bool move = mx > ref + MOVE;
        if (__any_sync(0xffffffffu, move)) {
          const float top = move ? mx : ref;
          const float f = top == ref ? 1.f : pa_ex2(ref - top);
          ref = top;
          sum.x *= f, sum.y *= f;
          if (t > t0) {
            ok = wait(&bars.pv_done[h], c_pv - 1);
            if (!ok) break;
            fence_after();
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
              uint32_t o[32];
              ld32(o, o_addr + c);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              st32(o, o_addr + c);
            }
          }
        }
        const float nref = ref == -INFINITY ? 0.f : -ref;
        const float2 sc2 = make_float2(scale, scale), nr2 = make_float2(nref, nref);
#pragma unroll
        for (int c = 0; c < 128; c += 2) {
          const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sc2, nr2);
          const float2 w = make_float2(pa_ex2(x.x), pa_ex2(x.y));
          sum = __fadd2_rn(sum, w);
          s[c / 2] = H::pack(w.x, w.y);
        }
        st32(s, s_addr);
        st32(s + 32, s_addr + 32);
        wait_st();
        if ((t + 1) * TILE > least && h == (t < end1 ? 1 : 0)) {
          // the last half at work takes what is not finite out of V: thread = position
          const int iv = n + 2 * (t - t0) + 1;
          ok = wait(&bars.full[iv % ST], iv / ST);
          if (!ok) break;
          const int r = tid & 127, pos = t * TILE + r;
          if (pos >= least) {
            uint8_t* v = smem + (iv % ST) * F::SLOT + r * 128;
            bool bad = false;
#pragma unroll
            for (int ch = 0; ch < HD / 8; ++ch) {
              uint32_t* x = reinterpret_cast<uint32_t*>(v + (ch >> 3) * F::PLANE + (((ch & 7) ^ (r & 7)) << 4));
              uint4 y = *reinterpret_cast<uint4*>(x);
              uint32_t z[4] = {y.x, y.y, y.z, y.w};
              bool any_bad = false;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if ((z[e] & H::EXP) == H::EXP) z[e] &= 0xffff0000u, any_bad = true;
                if ((z[e] & (H::EXP << 16)) == H::EXP << 16) z[e] &= 0xffffu, any_bad = true;
              }
              if (any_bad) *reinterpret_cast<uint4*>(x) = make_uint4(z[0], z[1], z[2], z[3]);
              bad = bad || any_bad;
            }
            if (bad && pos < len) d.p.poison = 1;
          }
          fence_proxy_async_smem();
          mbar_arrive(&bars.v_clean);
        }
        fence_before();
        mbar_arrive(&bars.p_full[h]);
        ++c_pv;
      }
      if (!ok) break;
      if (mine) {
        ok = wait(&bars.pv_done[h], c_pv - 1);
        if (!ok) break;
        fence_after();
      }
      const float L = sum.x + sum.y;
      const bool whole = t0 == 0 && t1 == p.it.tiles, fix = d.p.poison != 0;
      constexpr int STRIDE = ROWS * (HD + 2);
      float* part = piece_part(a, p, blockIdx.x, STRIDE);
      auto store = [&](const float (&v)[32], int c) {  // 32 values of the row from dim c on
        const int64_t at = (int64_t)(start + token) * a.ld_out + (int64_t)head * HD + c;
        if (a.out32) {
          float* y = static_cast<float*>(a.out) + at;
#pragma unroll
          for (int e = 0; e < 32; ++e) y[e] = v[e];
        } else {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = H::pack(v[2 * e], v[2 * e + 1]);
          uint32_t* y = reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + at);
          if (a.vec_out) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              reinterpret_cast<uint4*>(y)[e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = w[e];
          }
        }
      };
      if (mine) {
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          uint32_t o[32];
          ld32(o, o_addr + c);
          float v[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(o[e]);
          if (fix)
            for (int j = max(t0 * TILE, least); j < min(t1 * TILE, lim); ++j) {
              const int page = __ldcg(a.table + (int64_t)p.it.b * a.max_pages + (j >> a.c.page_shift));
              if ((unsigned)page >= (unsigned)a.c.num_pages) continue;
              const unsigned short* src = reinterpret_cast<const unsigned short*>(a.c.v) +
                                          (((int64_t)page * a.c.kv_heads + p.kvh) * P + (j & (P - 1))) * HD + c;
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const float y = H::up(__ldcg(src + e));
                if (!(fabsf(y) <= 3.402823466e38f)) v[e] += y;
              }
            }
          if (whole) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] *= inv;
            if (row < rows) store(v, c);
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(part + ((c + e) / 4 * ROWS + row) * 4) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          }
        }
        fence_before();
      }
      if (!whole) {
        *reinterpret_cast<float2*>(part + ROWS * HD + 2 * row) = make_float2(ref, L);
        const int c0 = p.c0, c1 = p.c1;
        __threadfence();
        mbar_arrive(&bars.join);
        ok = wait(&bars.join, joins++);
        if (!ok) break;
        if (tid == 0) is_last = atomicAdd(a.count + p.unit, 1) == c1 - c0;
        mbar_arrive(&bars.join);
        ok = wait(&bars.join, joins++);
        if (!ok) break;
        if (is_last) {
          __threadfence();
          auto piece = [&](int c) { return piece_part(a, p, c, STRIDE); };
          float top = -INFINITY, all = 0.f;
          for (int c = c0; c <= c1; ++c)
            top = fmaxf(top, __ldcg(reinterpret_cast<const float2*>(piece(c) + ROWS * HD + 2 * row)).x);
          for (int c = c0; c <= c1; ++c) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(piece(c) + ROWS * HD + 2 * row));
            all += ml.y * (ml.x == top ? 1.f : pa_ex2(ml.x - top));
          }
          const float inv = all == 0.f ? 0.f : 1.f / all;
#pragma unroll 1
          for (int d0 = 0; d0 < HD; d0 += 32) {
            float v[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0.f;
            for (int c = c0; c <= c1; ++c) {
              const float* src = piece(c);
              const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + ROWS * HD + 2 * row));
              if (ml.x == -INFINITY && ml.y == 0.f) continue;  // saw nothing
              const float f = ml.x == top ? 1.f : pa_ex2(ml.x - top);
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                const float4 x = __ldcg(reinterpret_cast<const float4*>(src + ((d0 + e) / 4 * ROWS + row) * 4));
                v[e] = fmaf(x.x, f, v[e]), v[e + 1] = fmaf(x.y, f, v[e + 1]);
                v[e + 2] = fmaf(x.z, f, v[e + 2]), v[e + 3] = fmaf(x.w, f, v[e + 3]);
              }
            }
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] *= inv;
            if (row < rows) store(v, d0);
          }
          if (tid == 0) a.count[p.unit] = 0;
        }
        // nobody sets is_last again before all have read it
        mbar_arrive(&bars.join);
        ok = wait(&bars.join, joins++);
        if (!ok) break;
      }
      n += 2 * (t1 - t0);
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.d_empty[k & 1]);
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 9) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(F::COLS) : "memory");
  }
}

template <typename T, int HD, bool FANCY>
static cudaError_t launch(const PagedAttnArgs& a, cudaStream_t s) {
  using F = Cfg<HD>;
  auto kern = paged_tc_kernel<T, HD, FANCY>;
  CUtensorMap maps[2];
  if (cudaError_t e = paged_maps(a.c, TILE, maps)) return e;
  static PagedReady ready;
  if (cudaError_t e = ready.set((const void*)kern, F::SMEM)) return e;
  return launch_pdl_smem(kern, dim3(paged_ctas(ROWS)), dim3(THREADS), F::SMEM, s, a, maps[0], maps[1]);
}

}  // namespace ptc

cudaError_t launch_paged_tc(PagedAttnArgs& a, bool fancy, cudaStream_t s) {
  using namespace ptc;
  static_assert(ROWS == PAGED_ROWS_MAX, "the scratch's pieces");
  if (a.c.dtype == ODI_CUDA_PAGED_BF16) {
    if (a.c.hd == 128) return fancy ? launch<__nv_bfloat16, 128, true>(a, s) : launch<__nv_bfloat16, 128, false>(a, s);
    return fancy ? launch<__nv_bfloat16, 64, true>(a, s) : launch<__nv_bfloat16, 64, false>(a, s);
  }
  if (a.c.hd == 128) return fancy ? launch<__half, 128, true>(a, s) : launch<__half, 128, false>(a, s);
  return fancy ? launch<__half, 64, true>(a, s) : launch<__half, 64, false>(a, s);
}

}  // namespace odi_cuda
