// paged_attention.cu -- attention of new tokens of several requests over a paged
// cache: the entry point, and the kernel for few rows per kv head.
//
//   s_ij = scale q_i . k_j,  then cap * tanh(s / cap), then - slope_h |i - j|
//   o_i  = sum_j softmax_j(s_ij) v_j  over  j < max(i + 1, prefix)
//
// Up to 32 rows (new tokens * heads per kv head) of a request meet its pages on
// mma.sync, whose 16-row tiles fit so few rows: each row of K and V is read once
// and HBM bounds the kernel.  A producer warp brings tiles of 64 positions, page
// by page, into a ring by TMA; for each 16 rows there are four warps, which take
// 16 positions of a tile each with softmax statistics of their own, so that no
// barrier stands between tiles, and join when a piece ends: three more warps do that
// beside the next piece.
//
// 64 requests of one token, 64/8 heads of 128 dims over 300 to 8,100 positions: 183 us,
// 6.3 TB/s.  Where requests are short or few, latency is the bound: a tile takes a warp
// about 1 us, an item some 2 us beside its tiles (its queries' way from memory, the
// join); 512 such requests over up to 200 positions take 69 us, HBM would 32; one token
// of 32 heads over 518 positions 9.5 us.  17 to 32 rows leave one CTA per SM, whose
// second group of warps has no row where a request has 16 or fewer (the width is the
// batch's): 16 requests of 2 to 5 tokens with a cap 56 us, 52 without, HBM 29.
//
// q . k and o are summed in fp32.  The weights enter the second product rounded
// to the cache's type, relative to a reference that moves only when a weight
// would pass 2^8 of it; their sum is taken before the rounding.  That is half a step of
// the type per weight, independent from weight to weight, so that the sum of many is
// off by less than the rounding of an output of that type.  fp16's steps end: what a
// row's largest weight outweighs 2^31 times has no weight, which is off by 2^-32 of the
// largest per position at most.  For an fp32 output the weights are sums of two parts,
// and the second product is made twice: 64 requests with bf16 caches are off by 5e-6 of
// the output's norm, 1.6e-3 with one part.  Where HBM is the bound that costs nothing;
// 512 short requests take 91 us, 78 with one part, 16 with drafts and a cap 60 and 55.
#include <cstdio>

#include "paged_attention.cuh"
#include "pdl_launch.cuh"

namespace odi_cuda {
namespace pmma {

constexpr int TILE = 64;

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (Half16<T>::BF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// MG: groups of 16 rows.  One group: two CTAs per SM; two: one.
template <int HD, int MG>
struct Cfg {
  static constexpr int SLOT = TILE * HD * 2;  // K or V of one tile
  static constexpr int ST = (HD == 128 ? 5 : 10) * MG;
  static constexpr int FOLD = 4 * 16 * HD * 4;  // a group's sums
  static constexpr int FOLD_OFF = ST * SLOT;
  static constexpr int SMEM = FOLD_OFF + MG * FOLD;
  static constexpr int THREADS = 128 * MG + 128, PER_SM = MG == 1 ? 2 : 1;
  // the launch's registers are shared out anew: a warp at the products holds O (64),
  // Q (32) and operands
  static constexpr int REGS_LAUNCH = MG == 1 ? 128 : 168, REGS_FEW = 104, REGS_MMA = MG == 1 ? 152 : 200;
  static_assert(128 * REGS_FEW + 128 * MG * REGS_MMA <= THREADS * REGS_LAUNCH, "register split");
  static_assert(PER_SM * (SMEM + 2048) <= 228 * 1024, "shared memory, with 1 KB static and 1 KB of the system's");
};
// pieces that the producer may be ahead: those before the one at the products are with the joiners
constexpr int ND = 3;
constexpr int JOINERS = 96;  // threads that join and write out

template <typename T, int HD, int MG, bool FANCY, bool OUT32>
__global__ void __launch_bounds__(Cfg<HD, MG>::THREADS, Cfg<HD, MG>::PER_SM)
    paged_mma_kernel(const __grid_constant__ PagedAttnArgs a, const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap) {
  using F = Cfg<HD, MG>;
  using H = Half16<T>;
  constexpr int KS = HD / 16, ROWS = 16 * MG, ST = F::ST;
  constexpr float MOVE = H::BELOW + PAGED_MOVE;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t full[ST], empty[ST], d_full[ND], d_empty[ND], fold_full, fold_empty, jbar;
  __shared__ PagedPiece pieces[ND];
  __shared__ float2 wml[4 * MG][16];
  __shared__ PagedFound found;
  __shared__ int is_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  pdl_launch_dependents();
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 4 * MG);
    for (int i = 0; i < ND; ++i) mbar_init(&d_full[i], 1), mbar_init(&d_empty[i], 4 * MG + 3);
    mbar_init(&fold_full, 4 * MG);
    mbar_init(&fold_empty, 3);
    mbar_init(&jbar, JOINERS);
    fence_mbar_init();
    prefetch_map(&kmap), prefetch_map(&vmap);
  }
  __syncthreads();
  pdl_wait();
  if (smem_u32(smem) & 1023u) {  // the swizzle counts from there
    if (tid == 0) atomicOr(a.err, ERR_PAGED_WAIT);
    return;
  }
  PagedRun run;
  if (!run_begin(a, run, &found)) return;
  const int P = a.c.page_size, BR = min(P, TILE);  // BR rows to a box, its planes of 64 dims one after the other
  auto wait = [&](uint64_t* bar, int phase) { return mbar_wait(bar, phase & 1, a.err, ERR_PAGED_WAIT); };

  if (warp >= 4 * MG) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F::REGS_FEW));
  if (warp == 4 * MG) {
    // ---- producer: a lane brings one box of K or V
    const int boxes = TILE / BR, box = lane;
    const int rows_all = a.c.num_pages * a.c.kv_heads * P;
    int n = 0, k = 0;
    bool ok = true;
    while (ok && run.x < run.end) {
      const PagedPiece p = run_piece(a, run, ROWS);
      const int len = p.it.len;
      if (p.t1 <= p.t0) break;
      PagedNames names(a, p, TILE, false);
      if (k >= ND && !wait(&d_empty[k % ND], k / ND - 1)) break;
      if (lane == 0) {
        pieces[k % ND] = p;
        mbar_arrive(&d_full[k % ND]);
      }
      ++k;
      if (run.x < run.end) run_next(a, run);
      for (int t = p.t0; ok && t < p.t1; ++t) {
        const int pos = t * TILE + box * BR;
        const int live = min(boxes, (len - t * TILE + BR - 1) / BR);
        const int page = names.at(pos >> a.c.page_shift);
        int y = (int)(((unsigned)page * a.c.kv_heads + p.kvh) * P) + (pos & (P - 1));
        if (box < live && (unsigned)page >= (unsigned)a.c.num_pages) {  // names no page: zeros, and the error word
          y = rows_all;
          atomicOr(a.err, ERR_PAGED_PAGE);
        }
        for (int v = 0; v < 2; ++v, ++n) {
          const int s = n % ST;
          if (n >= ST && !wait(&empty[s], n / ST - 1)) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_arrive_expect_tx(&full[s], live * BR * HD * 2);
          __syncwarp();
          if (box < live) pa_tma_3d(smem + s * F::SLOT + box * BR * HD * 2, v ? &vmap : &kmap, 0, y, 0, &full[s]);
        }
      }
    }
    if (ok && (k < ND || wait(&d_empty[k % ND], k / ND - 1)) && lane == 0) {
      pieces[k % ND].last = 1;
      mbar_arrive(&d_full[k % ND]);
    }
    for (int i = max(0, n - ST); i < n; ++i) wait(&full[i % ST], i / ST);  // no copy outlives the CTA
    return;
  }

  // ---- joins, beside the products of the next piece: the four warps of a group,
  // and the pieces of a unit
  const int jt = tid - (128 * MG + 32);
  const float* folds = reinterpret_cast<const float*>(smem + F::FOLD_OFF);
  int syncs = 0;
  auto sync = [&]() {  // of the joiners, bounded
    mbar_arrive(&jbar);
    return wait(&jbar, syncs++);
  };
  for (int k = 0;; ++k) {
    if (!wait(&d_full[k % ND], k / ND)) return;
    const PagedPiece& p = pieces[k % ND];
    if (p.last) return;
    const int t0 = p.t0, t1 = p.t1, rows = p.rows, least = p.least, len = p.it.len;
    const bool whole = t0 == 0 && t1 == p.it.tiles;
    constexpr int STRIDE = ROWS * (HD + 2);
    float* part = piece_part(a, p, blockIdx.x, STRIDE);
    // a row's value divided by its sum, to where it goes; nothing that weighs nothing
    auto store = [&](int r, int d, float4 v, float inv) {
      if (inv == 0.f) v = make_float4(0.f, 0.f, 0.f, 0.f);
      v.x *= inv, v.y *= inv, v.z *= inv, v.w *= inv;
      const int R = p.it.i * ROWS + r, token = pa_token(a, R);
      const int64_t at = (int64_t)(p.it.start + token) * a.ld_out + (int64_t)(p.kvh * a.G + R - token * a.G) * HD + d;
      if (OUT32) {
        float* y = static_cast<float*>(a.out) + at;
        if (a.vec_out) *reinterpret_cast<float4*>(y) = v;
        else y[0] = v.x, y[1] = v.y, y[2] = v.z, y[3] = v.w;
      } else {
        uint32_t* y = reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + at);
        const uint32_t lo = H::pack(v.x, v.y), hi = H::pack(v.z, v.w);
        if (a.vec_out) *reinterpret_cast<uint2*>(y) = make_uint2(lo, hi);
        else y[0] = lo, y[1] = hi;
      }
    };
    if (!wait(&fold_full, k)) return;
    const bool fix = p.poison;
#pragma unroll 1
    for (int i = jt; i < rows * (HD / 4); i += JOINERS) {
      const int r = i / (HD / 4), d = i % (HD / 4) * 4, mg = r >> 4, fr = r & 15;
      float2 ml[4];
      float top = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) ml[w] = wml[mg * 4 + w][fr], top = fmaxf(top, ml[w].x);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = ml[w].x == top ? 1.f : pa_ex2(ml[w].x - top);
        L += ml[w].y * f;
        const float4 x = *reinterpret_cast<const float4*>(folds + mg * (F::FOLD / 4) + (w * 16 + fr) * HD +
                                                          (((d >> 3) ^ (fr & 7)) & (HD / 8 - 1)) * 8 + (d & 4));
        v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
      }
      if (fix) {
        const int row_lim = paged_limit(p.it.past, pa_token(a, p.it.i * ROWS + r), len, p.it.prefix);
        for (int j = max(t0 * TILE, least); j < min(t1 * TILE, row_lim) && j >> a.c.page_shift < a.max_pages; ++j) {
          const int page = __ldcg(a.table + (int64_t)p.it.b * a.max_pages + (j >> a.c.page_shift));
          if ((unsigned)page >= (unsigned)a.c.num_pages) continue;
          const unsigned short* src = static_cast<const unsigned short*>(a.c.v) +
                                      (((int64_t)page * a.c.kv_heads + p.kvh) * P + (j & (P - 1))) * HD + d;
          float y[4];
          for (int e = 0; e < 4; ++e) {
            y[e] = H::up(__ldcg(src + e));
            if (fabsf(y[e]) <= 3.402823466e38f) y[e] = 0.f;
          }
          v.x += y[0], v.y += y[1], v.z += y[2], v.w += y[3];
        }
      }
      if (whole) {
        store(r, d, v, L == 0.f ? 0.f : 1.f / L);
      } else {
        *reinterpret_cast<float4*>(part + r * HD + d) = v;
        if (d == 0) *reinterpret_cast<float2*>(part + ROWS * HD + 2 * r) = make_float2(top, L);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&fold_empty);
    if (!whole) {
      // the last piece to arrive joins them
      for (PagedJoin join = join_first(a, p, 16);; join = join_next(a, p)) {
        if (!sync()) return;
        if (jt == 0) {
          __threadfence();
          is_last = atomicAdd(join.counter, 1) == join.n - 1;
          __threadfence();
        }
        if (!sync()) return;
        if (!is_last) break;
        // Three places of the unit by four pieces at a time, so that loads overlap; a
        // lane has the factor of one piece for its row, whose LANES lanes share theirs.
        constexpr int LANES = HD / 4;
#pragma unroll 1
        for (int i0 = jt & ~31; i0 < rows * LANES; i0 += 3 * JOINERS) {
          float top[3], L[3];
          float4 v[3];
          int at[3];
#pragma unroll
          for (int u = 0; u < 3; ++u) {
            top[u] = -INFINITY, L[u] = 0.f, v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            at[u] = min(i0 + lane + u * JOINERS, rows * LANES - 1);
          }
#pragma unroll 1
          for (int q0 = 0; q0 < join.n; q0 += LANES) {
            const int q = q0 + lane % LANES, some = min(LANES, join.n - q0);
            float2 ml[3];
            float f[3];
#pragma unroll
            for (int u = 0; u < 3; ++u) {
              ml[u] = make_float2(-INFINITY, 0.f);
              if (q < join.n)
                ml[u] = __ldcg(reinterpret_cast<const float2*>(piece_part(a, p, join.first + q * join.step, STRIDE) + ROWS * HD +
                                                               2 * (at[u] / LANES)));
            }
#pragma unroll
            for (int u = 0; u < 3; ++u) {
              float now = fmaxf(top[u], ml[u].x);
#pragma unroll
              for (int o = LANES / 2; o; o >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, o));
              const float fo = top[u] == now ? 1.f : pa_ex2(top[u] - now);
              f[u] = ml[u].x == now ? 1.f : pa_ex2(ml[u].x - now);
              float l = ml[u].y * f[u];
#pragma unroll
              for (int o = LANES / 2; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
              top[u] = now, L[u] = fmaf(L[u], fo, l);
              v[u].x *= fo, v[u].y *= fo, v[u].z *= fo, v[u].w *= fo;
            }
#pragma unroll 1
            for (int w0 = 0; w0 < some; w0 += 4) {
              float4 x[3][4];
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                const float4* src = reinterpret_cast<const float4*>(
                    piece_part(a, p, join.first + (q0 + min(w0 + w, some - 1)) * join.step, STRIDE));
#pragma unroll
                for (int u = 0; u < 3; ++u) x[u][w] = __ldcg(src + at[u]);
              }
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                if (w0 + w >= some) break;
#pragma unroll
                for (int u = 0; u < 3; ++u) {
                  const float g = __shfl_sync(0xffffffffu, f[u], (lane & ~(LANES - 1)) | (w0 + w));
                  v[u].x = fmaf(x[u][w].x, g, v[u].x), v[u].y = fmaf(x[u][w].y, g, v[u].y);
                  v[u].z = fmaf(x[u][w].z, g, v[u].z), v[u].w = fmaf(x[u][w].w, g, v[u].w);
                }
              }
            }
          }
#pragma unroll
          for (int u = 0; u < 3; ++u) {
            if (i0 + lane + u * JOINERS >= rows * LANES) break;
            const int r = at[u] / LANES, d = at[u] % LANES * 4;
            if (join.final) {
              store(r, d, v[u], L[u] == 0.f ? 0.f : 1.f / L[u]);
            } else {  // in its first piece's place: this warp's lanes alone read that row of it
              float* to = piece_part(a, p, join.first, STRIDE);
              *reinterpret_cast<float4*>(to + r * HD + d) = v[u];
              if (d == 0) *reinterpret_cast<float2*>(to + ROWS * HD + 2 * r) = make_float2(top[u], L[u]);
            }
          }
        }
        if (jt == 0) *join.counter = 0;
        if (join.final) break;
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&d_empty[k % ND]);
  }
  }

  // ---- products: a warp has 16 rows and positions 16 wq .. + 15 of every tile
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F::REGS_MMA));
  const int g = lane >> 2, c = lane & 3, mg = warp >> 2, wq = warp & 3;
  const uint32_t base = smem_u32(smem), plane = BR * 128;
  // where its rows of a slot are: those that the lane addresses of K, and of V
  const int rk = wq * 16 + (lane >> 4) * 8 + (lane & 7), rv = wq * 16 + (lane >> 3 & 1) * 8 + (lane & 7);
  const uint32_t box = (uint32_t)(wq * 16 / BR * BR * HD * 2), in_box = wq * 16 / BR * BR;
  const uint32_t k_at = base + box + (rk - in_box) * 128, v_at = base + box + (rv - in_box) * 128;
  float* fold = reinterpret_cast<float*>(smem + F::FOLD_OFF + mg * F::FOLD);
  int n = 0;
  for (int k = 0;; ++k) {
    if (!wait(&d_full[k % ND], k / ND)) return;
    PagedPiece& p = pieces[k % ND];
    if (p.last) return;
    const int t0 = p.t0, t1 = p.t1, rows = p.rows - mg * 16, least = p.least, len = p.it.len, past = p.it.past;
    const int R0 = p.it.i * ROWS + mg * 16;  // the group's first row of the request
    const bool live_group = rows > 0;
    uint32_t qf[KS][4];
    float o[HD / 8][4], m[2], l[2], slope[2];
    int lim[2];
    float tok[2];
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bool live = e * 8 + g < rows;
      const int R = R0 + (live ? e * 8 + g : 0), token = pa_token(a, R), head = p.kvh * a.G + R - token * a.G;
      tok[e] = (float)token;
      lim[e] = live ? paged_limit(past, token, len, p.it.prefix) : 0;
      slope[e] = FANCY && a.slopes && live ? __ldg(a.slopes + head) * 1.4426950408889634f : 0.f;
      m[e] = -INFINITY, l[e] = 0.f;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q) + (int64_t)(p.it.start + token) * a.ld_q +
                                                              (int64_t)head * HD) + c;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        qf[ks][e] = live ? __ldcg(src + ks * 8) : 0u;
        qf[ks][2 + e] = live ? __ldcg(src + ks * 8 + 4) : 0u;
      }
    }
#pragma unroll
    for (int d = 0; d < HD / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
    for (int t = t0; t < t1; ++t, n += 2) {
      const int sk = n % ST, sv = (n + 1) % ST;
      const int pw = t * TILE + wq * 16;  // the warp's first position
      const bool masked = pw + 16 > least;
      if (!wait(&full[sk], n / ST)) return;
      uint32_t pf[4], pr[4];  // weights, and what their rounding left
      if (live_group) {
        __syncwarp();  // ldmatrix and mma want whole warps, and a wait may let lanes go one by one
        // ---- S = Q K^T
        float sc[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
        const uint32_t ka = k_at + sk * F::SLOT;
#pragma unroll
        for (int k0 = 0; k0 < KS; k0 += 4) {
          uint32_t b[4][4];
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const int chunk = 2 * (k0 + ks) + (lane >> 3 & 1);
            ldsm4(b[ks], ka + (chunk >> 3) * plane + (((chunk & 7) ^ (lane & 7)) << 4));
          }
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            mma<T>(sc[0], qf[k0 + ks], b[ks][0], b[ks][1]);
            mma<T>(sc[1], qf[k0 + ks], b[ks][2], b[ks][3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[sk]);
        // ---- scores, weights
        float mx[2];
        const float at = (float)(pw + 2 * c - past);  // as tok, from the first new token: whole below 2^24, far ones to 2^-24
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[e] = -INFINITY;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x = sc[i >> 1][2 * e + (i & 1)] * a.scale_log2;
            const int j = pw + (i >> 1) * 8 + 2 * c + (i & 1);
            if (FANCY) {
              if (a.cap_log2 != 0.f) x = pa_cap(x, a.cap_log2);
              x = fmaf(-slope[e], fabsf(tok[e] - (at + (float)((i >> 1) * 8 + (i & 1)))), x);
            }
            if (masked && j >= lim[e]) x = -INFINITY;
            sc[i >> 1][2 * e + (i & 1)] = x;
            mx[e] = fmaxf(mx[e], x);
          }
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
        }
        if (__any_sync(0xffffffffu, mx[0] > m[0] + MOVE || mx[1] > m[1] + MOVE)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float top = mx[e] > m[e] + MOVE ? mx[e] - H::BELOW : m[e];
            const float f = m[e] == top ? 1.f : pa_ex2(m[e] - top);
            m[e] = top;
            l[e] *= f;
#pragma unroll
            for (int d = 0; d < HD / 8; ++d) o[d][2 * e] *= f, o[d][2 * e + 1] *= f;
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float ref = m[e] == -INFINITY ? 0.f : m[e];
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w[i] = pa_ex2(sc[i >> 1][2 * e + (i & 1)] - ref);
            l[e] += w[i];
          }
          pf[e] = OUT32 ? H::split(make_float2(w[0], w[1]), pr[e]) : H::pack(w[0], w[1]);
          pf[2 + e] = OUT32 ? H::split(make_float2(w[2], w[3]), pr[2 + e]) : H::pack(w[2], w[3]);
        }
      } else if (lane == 0) {
        mbar_arrive(&empty[sk]);
      }
      if (!wait(&full[sv], (n + 1) / ST)) return;
      if (live_group) {
        __syncwarp();
        // ---- O += P V
        const uint32_t va = v_at + sv * F::SLOT;
        const int j0 = pw + 2 * c;
#pragma unroll
        for (int d0 = 0; d0 < KS; d0 += 4) {
          uint32_t b[4][4];
#pragma unroll
          for (int dt = 0; dt < 4; ++dt) {
            const int chunk = 2 * (d0 + dt) + (lane >> 4);
            ldsm4_t(b[dt], va + (chunk >> 3) * plane + (((chunk & 7) ^ (lane & 7)) << 4));
          }
          if (masked) {
            // What not every row sees must not reach the rows that do not: 0 * NaN is
            // NaN.  Values that are not finite leave here; rows that see them get them
            // when the piece ends.
            uint32_t zero = 0;  // 0 times all values: 0 if every one is finite
#pragma unroll
            for (int dt = 0; dt < 4; ++dt)
#pragma unroll
              for (int i = 0; i < 4; ++i) zero = H::times0(b[dt][i], zero);
            if (__any_sync(0xffffffffu, zero & 0x7fff7fffu)) {
#pragma unroll
              for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const int j = j0 + (i & 1) * 8 + e;
                    const uint32_t ex = H::EXP << (16 * e);
                    if (j >= least && (b[dt][i] & ex) == ex) {
                      b[dt][i] &= ~(0xffffu << (16 * e));
                      bad = bad || j < len;
                    }
                  }
            }
          }
#pragma unroll
          for (int dt = 0; dt < 4; ++dt) {
            mma<T>(o[2 * (d0 + dt)], pf, b[dt][0], b[dt][1]);
            mma<T>(o[2 * (d0 + dt) + 1], pf, b[dt][2], b[dt][3]);
          }
          if (OUT32) {
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) {
              mma<T>(o[2 * (d0 + dt)], pr, b[dt][0], b[dt][1]);
              mma<T>(o[2 * (d0 + dt) + 1], pr, b[dt][2], b[dt][3]);
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (lane == 0) mbar_arrive(&empty[sv]);
    }

    // ---- the piece is over: to the joiners
    if (k > 0 && !wait(&fold_empty, k - 1)) return;
    if (live_group) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
        if (c == 0) wml[warp][e * 8 + g] = make_float2(m[e], OUT32 ? l[e] * H::PARTS : l[e]);
        // 8-dim blocks in an order of the row's own, so that no two rows meet in a bank
#pragma unroll
        for (int d = 0; d < HD / 8; ++d)
          *reinterpret_cast<float2*>(fold + (wq * 16 + e * 8 + g) * HD + ((d ^ g) & (HD / 8 - 1)) * 8 + 2 * c) =
              make_float2(o[d][2 * e], o[d][2 * e + 1]);
      }
      if (bad) p.poison = 1;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&fold_full), mbar_arrive(&d_empty[k % ND]);
  }
}

template <typename T, int HD, int MG, bool FANCY, bool OUT32>
static cudaError_t launch(PagedAttnArgs& a, cudaStream_t s) {
  using F = Cfg<HD, MG>;
  auto kern = paged_mma_kernel<T, HD, MG, FANCY, OUT32>;
  CUtensorMap maps[2];
  if (cudaError_t e = paged_maps(a.c, TILE, true, maps)) return e;
  static PagedReady ready;
  if (cudaError_t e = ready.set((const void*)kern, F::SMEM)) return e;
  return launch_pdl_smem(kern, dim3(paged_ctas(16 * MG)), dim3(F::THREADS), F::SMEM, s, a, maps[0], maps[1]);
}

}  // namespace pmma

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

// K and V as tensors of rows; a box is (part of) one page of one kv head, 64 dims wide,
// in the 128-byte swizzle.  x is 0 or 64 values: 16-byte boundaries.  With `planes` a
// box has all planes of 64 dims, one after the other: half the boxes at 128 dims, which
// with pages of 16 were more than one warp could send (16 requests of 2 to 5 tokens
// 49 us so, 57 with a box per plane).
cudaError_t paged_maps(const PagedView& c, int tile, bool planes, CUtensorMap* maps) {
  const EncodeFn enc = encode_fn();
  if (!enc) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {planes ? 64u : (cuuint64_t)c.hd, (cuuint64_t)c.num_pages * c.kv_heads * c.page_size,
                              (cuuint64_t)c.hd / 64};
  const cuuint64_t strides[2] = {(cuuint64_t)c.hd * 2, 128};
  const cuuint32_t box[3] = {64u, (cuuint32_t)(c.page_size < tile ? c.page_size : tile), (cuuint32_t)c.hd / 64}, ones[3] = {1, 1, 1};
  for (int i = 0; i < 2; ++i)
    if (enc(&maps[i], c.dtype == ODI_CUDA_PAGED_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, planes ? 3 : 2,
            i ? c.v : c.k, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return cudaErrorInvalidValue;
  return cudaSuccess;
}

// q as [token][head][dim], boxes of 64 dims by the heads of a group by some tokens.
cudaError_t paged_q_map(const PagedAttnArgs& a, int tokens, CUtensorMap* map) {
  const EncodeFn enc = encode_fn();
  if (!enc) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {(cuuint64_t)a.c.hd, (cuuint64_t)a.c.kv_heads * a.G, (cuuint64_t)a.out_rows};
  const cuuint64_t strides[2] = {(cuuint64_t)a.c.hd * 2, (cuuint64_t)a.ld_q * 2};
  const cuuint32_t box[3] = {64u, (cuuint32_t)a.G, (cuuint32_t)tokens}, ones[3] = {1, 1, 1};
  return enc(map, a.c.dtype == ODI_CUDA_PAGED_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
             const_cast<void*>(a.q), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? cudaSuccess
             : cudaErrorInvalidValue;
}

cudaError_t launch_paged_mma(PagedAttnArgs& a, int groups, bool fancy, cudaStream_t s) {
  const bool bf = a.c.dtype == ODI_CUDA_PAGED_BF16;
  auto by_out = [&](auto t, auto hd, auto out) {
    using T = decltype(t);
    constexpr int HD = decltype(hd)::value;
    constexpr bool OUT32 = decltype(out)::value;
    if (groups == 1) return fancy ? pmma::launch<T, HD, 1, true, OUT32>(a, s) : pmma::launch<T, HD, 1, false, OUT32>(a, s);
    return fancy ? pmma::launch<T, HD, 2, true, OUT32>(a, s) : pmma::launch<T, HD, 2, false, OUT32>(a, s);
  };
  auto by_rows = [&](auto t, auto hd) { return a.out32 ? by_out(t, hd, std::true_type{}) : by_out(t, hd, std::false_type{}); };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (a.c.hd == 128) return bf ? by_rows(__nv_bfloat16{}, D128{}) : by_rows(__half{}, D128{});
  return bf ? by_rows(__nv_bfloat16{}, D64{}) : by_rows(__half{}, D64{});
}

}  // namespace odi_cuda

using namespace odi_cuda;

extern "C" {

// Error word, pieces, counters of groups of pieces, then a counter per unit.  The
// pieces' place has one size, so that a scratch serves any batch whose counters fit.
constexpr size_t PART_OFF = 256, GROUP_OFF = PART_OFF + (size_t)2 * PAGED_SMS * PAGED_ROWS_MAX * (128 + 2) * 4,
                 COUNT_OFF = GROUP_OFF + 2 * paged_ctas(16) * 4;
static_assert(paged_ctas(16) >= paged_ctas(128) && paged_ctas(16) >= paged_ctas(PAGED_ROWS_MAX), "counters of groups");
static_assert(paged_ctas(16) * 16 <= PAGED_SMS * PAGED_ROWS_MAX && paged_ctas(128) * 128 <= PAGED_SMS * PAGED_ROWS_MAX, "pieces of narrow items");

size_t odi_cuda_attention_paged_scratch_bytes(int requests, int max_rows, int max_new, int heads, int kv_heads, int head_dim) {
  PagedGeometry g;
  if (!paged_geometry(requests, max_rows, max_new, heads, kv_heads, &g) || (head_dim != 64 && head_dim != 128)) return 0;
  return COUNT_OFF + 4 * (size_t)(g.max_items * kv_heads);
}

int odi_cuda_attention_paged(const void* d_q, int64_t ld_q, const odi_cuda_paged_cache* cache,
                             const odi_cuda_page_tables* tables, const odi_cuda_paged_batch* batch, void* d_out,
                             int64_t ld_out, int out_dtype, int tokens, float scale, float softcap, const float* d_slopes,
                             void* d_scratch, size_t scratch_bytes, void* stream) {
  PagedAttnArgs a{};
  PagedGeometry g;
  if (int rc = paged_view(cache, &a.c, "attention_paged")) return rc;
  if (int rc = paged_batch_ok(batch, &g, "attention_paged")) return rc;
  if (!d_q || !d_out || !tables || !tables->table || !d_scratch)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "attention_paged: null argument");
  if (tables->requests != batch->requests || tables->page_size != a.c.page_size || batch->page_size != a.c.page_size ||
      batch->kv_heads != a.c.kv_heads || tables->num_pages != a.c.num_pages || tables->max_pages < 1)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "attention_paged: cache, tables and batch do not belong together");
  if (out_dtype != ODI_CUDA_PAGED_OUT_F32 && out_dtype != ODI_CUDA_PAGED_OUT_CACHE)
    return set_error(ODI_CUDA_ERR_UNSUPPORTED_DTYPE, "attention_paged: output is ODI_CUDA_PAGED_OUT_CACHE or ODI_CUDA_PAGED_OUT_F32");
  if (tokens < 0 || tokens > batch->max_rows)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "attention_paged: more tokens than the batch has rows");
  if (!(scale > 0.f) || !isfinite(scale) || !(softcap >= 0.f) || !isfinite(softcap))
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "attention_paged: scale must be positive, softcap 0 or more");
  // a capped score is off by 2^-21 of the cap at most, which up to here stays below
  // what the rounding of a weight to fp16 costs
  const float scale_log2 = (softcap > 0.f ? 2.f * (scale / softcap) : scale) * 1.4426950408889634f;
  if (softcap > 1024.f || !isfinite(scale_log2))
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "attention_paged: softcap is 1024 at most; scale, or scale / softcap, is out of range");
  const int64_t width = (int64_t)batch->heads * a.c.hd;
  if (ld_q < width || ld_out < width || ld_q > (1ll << 40) || ld_out > (1ll << 40))
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "attention_paged: a row stride is shorter than its row");
  const bool out32 = out_dtype == ODI_CUDA_PAGED_OUT_F32;
  if (((uintptr_t)d_q | (uintptr_t)d_out | (uintptr_t)d_slopes | (uintptr_t)tables->table) & 3 || (ld_q & 1) || (!out32 && (ld_out & 1)) ||
      (uintptr_t)d_scratch & 15)
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "attention_paged: misaligned buffer");
  if (scratch_bytes < odi_cuda_attention_paged_scratch_bytes(batch->requests, batch->max_rows, batch->max_new, batch->heads,
                                                             batch->kv_heads, a.c.hd))
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "attention_paged: scratch too small");
  if (!tokens) return ODI_CUDA_OK;
  const int64_t size = out32 ? 4 : 2;
  if (byte_rows_overlap(d_q, 2 * ld_q, 2 * width, d_out, size * ld_out, size * width, tokens))
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "attention_paged: d_out overlaps d_q");
  const int64_t out_bytes = size * ((tokens - 1) * ld_out + width);
  if (bytes_overlap(d_out, out_bytes, a.c.k, a.c.bytes()) || bytes_overlap(d_out, out_bytes, a.c.v, a.c.bytes()) ||
      bytes_overlap(d_out, out_bytes, d_scratch, (int64_t)scratch_bytes) || bytes_overlap(d_out, out_bytes, d_slopes, 4ll * batch->heads))
    return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "attention_paged: d_out overlaps the cache, the slopes or the scratch");
  a.q = d_q, a.ld_q = ld_q, a.out = d_out, a.ld_out = ld_out, a.out32 = out32;
  a.table = tables->table, a.max_pages = tables->max_pages;
  a.header = batch->work, a.max_items = (int)g.max_items;
  a.extra = g.extra;
  a.G = g.G, a.out_rows = tokens;
  a.inv_G = g.G > 1 ? (unsigned)(((1ull << 32) + g.G - 1) / g.G) : 0;
  a.scale_log2 = scale_log2;
  a.cap_log2 = softcap * 1.4426950408889634f;
  a.slopes = d_slopes;
  a.vec = !((uintptr_t)d_q & 15) && !(ld_q & 7);
  a.vec_out = !((uintptr_t)d_out & 15) && !(ld_out & 7);
  // Tiles that a CTA takes at least: fewer are more pieces to join.  mma.sync, one token
  // of 32 heads over 100, 518 and 2000 positions: 5.5, 9.7 and 13.6 us with two, 7.8, 9.7
  // and 13.5 with one, 5.4, 10.7 and 13.6 with four; tcgen05, 16 tokens of 64/8 heads over
  // 500 and 2000: 16.5 and 22.2 us with four, 17.5 and 24.4 with two, 16.8 and 22.1 with five.
  a.least = g.rows <= 32 ? 2 : 4;
  a.err = static_cast<int*>(d_scratch);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(d_scratch) + PART_OFF);
  a.group = reinterpret_cast<int*>(static_cast<uint8_t*>(d_scratch) + GROUP_OFF);
  a.count = reinterpret_cast<int*>(static_cast<uint8_t*>(d_scratch) + COUNT_OFF);
  const bool fancy = softcap > 0.f || d_slopes;
  cudaStream_t s = (cudaStream_t)stream;
  return kv_launched(g.rows <= 32 ? launch_paged_mma(a, g.rows / 16, fancy, s) : launch_paged_tc(a, g.rows, s), "attention_paged");
}

}  // extern "C"
