// paged_attention.cu -- attention of new tokens of several requests over a paged
// cache: the entry point, and the kernel for few rows per kv head.
//
//   s_ij = scale q_i . k_j,  then cap * tanh(s / cap), then - slope_h |i - j|
//   o_i  = sum_j softmax_j(s_ij) v_j  over  j < max(i + 1, prefix)
//
// Up to 32 rows (new tokens * heads per kv head) of a request meet its pages on
// mma.sync, whose 16-row tiles fit so few rows: each row of K and V is read once
// and HBM bounds the kernel.  A producer warp brings tiles of 64 positions, page
// by page, into a ring by TMA; each of four warps takes 16 positions of a tile
// with softmax statistics of its own, so that no barrier stands between tiles,
// and the four join when a piece ends.
//
// q . k and o are summed in fp32.  The weights enter the second product rounded
// to the cache's type, relative to a reference that moves only when a weight
// would pass 2^8: half a step of that type per weight, independent from weight
// to weight, which is no more than the output's own rounding; their sum is taken
// before the rounding.
#include <cstdio>

#include "paged_attention.cuh"
#include "pdl_launch.cuh"

namespace odi_cuda {
namespace pmma {

constexpr int TILE = 64, ST = 3, THREADS = 160;
constexpr float MOVE = 8.f;  // log2 of what a weight may reach before the reference moves

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

struct Desc {  // what a tile in the ring belongs to
  PagedPiece p;
  int t;  // its place in the unit; -1: the run is over
};

template <int HD>
struct Cfg {
  static constexpr int HALF_BYTES = TILE * 128, TB = HD / 64 * HALF_BYTES, STAGE = 2 * TB;
  static constexpr int FOLD_OFF = ST * STAGE, FOLD = 4 * 16 * 32 * 4;
  static constexpr int SMEM = FOLD_OFF + FOLD + 1024;
};

template <typename T, int HD, int MT, bool FANCY>
__global__ void __launch_bounds__(THREADS, 2)
    paged_mma_kernel(const __grid_constant__ PagedAttnArgs a, const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap) {
  using F = Cfg<HD>;
  using H = Half16<T>;
  constexpr int KS = HD / 16, ROWS = 16 * MT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t full[ST], empty[ST], cbar;
  __shared__ Desc desc[ST];
  __shared__ float2 wml[4][ROWS];
  __shared__ int first_item, poison, is_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  pdl_launch_dependents();
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 4);
    mbar_init(&cbar, 128);
    poison = 0;
    first_item = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  PagedRun run;
  if (!run_begin(a, run, &first_item)) return;
  const int P = a.c.page_size;

  if (warp == 4) {
    // ---- producer: lane l brings box l / (2 halves) of K or V, one half of its dims
    constexpr int PER = 2 * (HD / 64);
    const int BR = min(P, TILE), boxes = TILE / BR;
    const int box = lane / PER, half = lane % (HD / 64), isv = lane / (HD / 64) & 1;
    const int rows_all = a.c.num_pages * a.c.kv_heads * P;
    int n = 0;
    bool ok = true;
    while (ok && run.x < run.end) {
      run_piece(a, run);
      const PagedPiece& p = run.p;
      const int len = __ldcg(a.lens + p.b);
      const int* row = a.table + (int64_t)p.b * a.max_pages;
      auto entry = [&](int t) {
        const int pos = t * TILE + box * BR;
        return box < boxes && t < p.t1 && pos < len ? __ldcg(row + (pos >> a.c.page_shift)) : -1;
      };
      int page = entry(p.t0);
      for (int t = p.t0; t < p.t1; ++t, ++n) {
        const int s = n % ST, pos = t * TILE + box * BR;
        const int next = entry(t + 1);
        if (n >= ST && !mbar_wait(&empty[s], (n / ST - 1) & 1, a.err, ERR_PAGED_WAIT)) {
          ok = false;
          break;
        }
        const int live = min(boxes, (len - t * TILE + BR - 1) / BR);
        if (lane == 0) {
          desc[s].p = p;
          desc[s].t = t;
          mbar_arrive_expect_tx(&full[s], live * BR * HD * 4);
        }
        __syncwarp();
        if (box < live) {
          int y = (page * a.c.kv_heads + p.kvh) * P + (pos & (P - 1));
          if ((unsigned)page >= (unsigned)a.c.num_pages) {  // a table that names no page: zeros, and the error word
            y = rows_all;
            atomicOr(a.err, ERR_PAGED_PAGE);
          }
          pa_tma(smem + s * F::STAGE + isv * F::TB + half * F::HALF_BYTES + box * BR * 128, isv ? &vmap : &kmap, half * 64, y,
                 &full[s]);
        }
        page = next;
      }
      run_next(run);
    }
    if (ok) {
      const int s = n % ST;
      if (n < ST || mbar_wait(&empty[s], (n / ST - 1) & 1, a.err, ERR_PAGED_WAIT)) {
        if (lane == 0) {
          desc[s].t = -1;
          mbar_arrive(&full[s]);
        }
      }
    } else {  // copies in flight land before the CTA leaves
      for (int k = max(0, n - ST); k < n; ++k) mbar_wait(&full[k % ST], (k / ST) & 1, a.err, ERR_PAGED_WAIT);
    }
    return;
  }

  // ---- consumers: warp w has positions 16 w .. + 15 of every tile
  const int g = lane >> 2, c = lane & 3;
  const uint32_t base = smem_u32(smem);
  uint32_t qf[MT][KS][4];
  float o[MT][HD / 8][4], m[MT][2], l[MT][2];
  int lim[MT][2], tok[MT][2];
  float slope[MT][2];
  int len = 0, start = 0, rows = 0, least = 0, past = 0, phase = 0;
  bool bad = false;
  float* fold = reinterpret_cast<float*>(smem + F::FOLD_OFF);
  auto sync = [&]() {  // of the 128 consumers, bounded
    mbar_arrive(&cbar);
    const bool ok = mbar_wait(&cbar, phase & 1, a.err, ERR_PAGED_WAIT);
    ++phase;
    return ok;
  };
  for (int n = 0;; ++n) {
    const int s = n % ST;
    if (!mbar_wait(&full[s], (n / ST) & 1, a.err, ERR_PAGED_WAIT)) return;
    const int t = desc[s].t;
    if (t < 0) return;
    const PagedPiece p = desc[s].p;
    if (t == p.t0) {
      start = __ldcg(a.starts + p.b);
      const int n_new = __ldcg(a.starts + p.b + 1) - start;
      len = __ldcg(a.lens + p.b);
      past = len - n_new;
      const int prefix = __ldcg(a.w.prefix + p.b);
      rows = min(ROWS, min(n_new, a.out_rows - start) * a.G - p.i * ROWS);
      least = paged_limit(past, pa_token(a, p.i * ROWS), len, prefix);
      const T* q = static_cast<const T*>(a.q);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = mt * 16 + e * 8 + g;
          const bool live = r < rows;
          const int R = p.i * ROWS + (live ? r : 0), token = pa_token(a, R), head = p.kvh * a.G + R - token * a.G;
          tok[mt][e] = past + token;
          lim[mt][e] = live ? paged_limit(past, token, len, prefix) : 0;
          if (FANCY) slope[mt][e] = a.slopes ? __ldg(a.slopes + head) * 1.4426950408889634f : 0.f;
          m[mt][e] = -INFINITY, l[mt][e] = 0.f;
          const uint32_t* src = reinterpret_cast<const uint32_t*>(q + (int64_t)(start + token) * a.ld_q + (int64_t)head * HD) + c;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            qf[mt][ks][e] = live ? __ldcg(src + ks * 8) : 0u;
            qf[mt][ks][2 + e] = live ? __ldcg(src + ks * 8 + 4) : 0u;
          }
        }
#pragma unroll
        for (int d = 0; d < HD / 8; ++d) o[mt][d][0] = o[mt][d][1] = o[mt][d][2] = o[mt][d][3] = 0.f;
      }
    }
    const uint32_t kb = base + s * F::STAGE, vb = kb + F::TB;
    const int pw = t * TILE + warp * 16;  // the warp's first position
    const bool masked = pw + 16 > least;
    // ---- S = Q K^T
    float sc[MT][2][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < 2; ++j) sc[mt][j][0] = sc[mt][j][1] = sc[mt][j][2] = sc[mt][j][3] = 0.f;
    {
      const int pr = warp * 16 + (lane >> 4) * 8 + (lane & 7);
      const uint32_t ka = kb + pr * 128;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t b[4];
        const int chunk = 2 * ks + (lane >> 3 & 1);
        ldsm4(b, ka + (chunk >> 3) * F::HALF_BYTES + (((chunk & 7) ^ (pr & 7)) << 4));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma<T>(sc[mt][0], qf[mt][ks], b[0], b[1]);
          mma<T>(sc[mt][1], qf[mt][ks], b[2], b[3]);
        }
      }
    }
    // ---- scores, weights
    uint32_t pf[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float mx[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[e] = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float x = sc[mt][k >> 1][2 * e + (k & 1)] * a.scale_log2;
          const int j = pw + (k >> 1) * 8 + 2 * c + (k & 1);
          if (FANCY) {
            if (a.cap_log2 != 0.f) x = a.cap_log2 * pa_tanh(x);
            x = fmaf(-slope[mt][e], (float)abs(tok[mt][e] - j), x);
          }
          if (masked && j >= lim[mt][e]) x = -INFINITY;
          sc[mt][k >> 1][2 * e + (k & 1)] = x;
          mx[e] = fmaxf(mx[e], x);
        }
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
      }
      const bool up = mx[0] > m[mt][0] + MOVE || mx[1] > m[mt][1] + MOVE;
      if (__any_sync(0xffffffffu, up)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float top = mx[e] > m[mt][e] + MOVE ? mx[e] : m[mt][e];
          const float f = m[mt][e] == top ? 1.f : pa_ex2(m[mt][e] - top);
          m[mt][e] = top;
          l[mt][e] *= f;
#pragma unroll
          for (int d = 0; d < HD / 8; ++d) o[mt][d][2 * e] *= f, o[mt][d][2 * e + 1] *= f;
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float ref = m[mt][e] == -INFINITY ? 0.f : m[mt][e];
        float w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          w[k] = pa_ex2(sc[mt][k >> 1][2 * e + (k & 1)] - ref);
          l[mt][e] += w[k];
        }
        pf[mt][e] = H::pack(w[0], w[1]);
        pf[mt][2 + e] = H::pack(w[2], w[3]);
      }
    }
    // ---- O += P V
    {
      const int pr = warp * 16 + (lane >> 3 & 1) * 8 + (lane & 7);
      const uint32_t va = vb + pr * 128;
      const int j0 = pw + 2 * c;
#pragma unroll
      for (int dt = 0; dt < KS; ++dt) {
        uint32_t b[4];
        const int chunk = 2 * dt + (lane >> 4);
        ldsm4_t(b, va + (chunk >> 3) * F::HALF_BYTES + (((chunk & 7) ^ (pr & 7)) << 4));
        if (masked) {
          // What not every row sees must not reach the rows that do not: 0 * NaN is
          // NaN.  Values that are not finite leave here; rows that see them get them
          // when the piece ends.
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = j0 + (k & 1) * 8 + e;
              const uint32_t ex = H::EXP << (16 * e);
              if (j >= least && (b[k] & ex) == ex) {
                b[k] &= ~(0xffffu << (16 * e));
                bad = bad || j < len;
              }
            }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma<T>(o[mt][2 * dt], pf[mt], b[0], b[1]);
          mma<T>(o[mt][2 * dt + 1], pf[mt], b[2], b[3]);
        }
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[s]);
    if (t != p.t1 - 1) continue;

    // ---- the piece is over: the four warps join
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[mt][e] += __shfl_xor_sync(0xffffffffu, l[mt][e], 1);
        l[mt][e] += __shfl_xor_sync(0xffffffffu, l[mt][e], 2);
        if (c == 0) wml[warp][mt * 16 + e * 8 + g] = make_float2(m[mt][e], l[mt][e]);
      }
    if (bad) poison = 1;
    bad = false;
    if (!sync()) return;
    const bool fix = poison != 0;
    const bool whole = p.t0 == 0 && p.t1 == p.tn;
    const int64_t ux = (int64_t)p.kvh * run.tiles + __ldcg(a.w.cum + p.item);  // the unit's first tile
    const int slot = 2 * blockIdx.x + (run.share * blockIdx.x <= ux ? 1 : 0);
    float* part = a.part + (int64_t)slot * ROWS * (HD + 2);
    const T* vpool = static_cast<const T*>(a.c.v);
    const int fr = tid >> 3, fd = (tid & 7) * 4;  // the row and dims this thread joins
    // what a row's value is divided by, and where it goes
    auto store = [&](int r, int d, float4 v, float L) {
      const float f = L == 0.f ? 0.f : 1.f / L;
      v.x *= f, v.y *= f, v.z *= f, v.w *= f;
      const int R = p.i * ROWS + r, token = pa_token(a, R);
      const int64_t at = (int64_t)(start + token) * a.ld_out + (int64_t)(p.kvh * a.G + R - token * a.G) * HD + d;
      if (a.out32) {
        float* y = static_cast<float*>(a.out) + at;
        y[0] = v.x, y[1] = v.y, y[2] = v.z, y[3] = v.w;
      } else {
        uint32_t* y = reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + at);
        y[0] = H::pack(v.x, v.y), y[1] = H::pack(v.z, v.w);
      }
    };
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float M[2], fw[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = mt * 16 + e * 8 + g;
        M[e] = fmaxf(fmaxf(wml[0][r].x, wml[1][r].x), fmaxf(wml[2][r].x, wml[3][r].x));
        fw[e] = m[mt][e] == M[e] ? 1.f : pa_ex2(m[mt][e] - M[e]);
      }
      const int r = mt * 16 + fr;
      float top = -INFINITY, L = 0.f;
      for (int w = 0; w < 4; ++w) top = fmaxf(top, wml[w][r].x);
      for (int w = 0; w < 4; ++w) L += wml[w][r].y * (wml[w][r].x == top ? 1.f : pa_ex2(wml[w][r].x - top));
      const int R = p.i * ROWS + r;
      const int row_lim = r < rows ? paged_limit(past, pa_token(a, R), len, __ldcg(a.w.prefix + p.b)) : 0;
#pragma unroll
      for (int d0 = 0; d0 < HD; d0 += 32) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            *reinterpret_cast<float2*>(fold + (warp * 16 + e * 8 + g) * 32 + k * 8 + 2 * c) =
                make_float2(o[mt][d0 / 8 + k][2 * e] * fw[e], o[mt][d0 / 8 + k][2 * e + 1] * fw[e]);
        if (!sync()) return;
        if (r < rows) {
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(fold + (w * 16 + fr) * 32 + fd);
            v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
          }
          if (fix)
            for (int j = max(p.t0 * TILE, least); j < min(p.t1 * TILE, row_lim); ++j) {
              const int page = __ldcg(a.table + (int64_t)p.b * a.max_pages + (j >> a.c.page_shift));
              if ((unsigned)page >= (unsigned)a.c.num_pages) continue;
              const T* src = vpool + (((int64_t)page * a.c.kv_heads + p.kvh) * P + (j & (P - 1))) * HD + d0 + fd;
              float y[4];
              for (int e = 0; e < 4; ++e) {
                y[e] = H::up(__ldcg(reinterpret_cast<const unsigned short*>(src) + e));
                if (fabsf(y[e]) <= 3.402823466e38f) y[e] = 0.f;
              }
              v.x += y[0], v.y += y[1], v.z += y[2], v.w += y[3];
            }
          if (whole) store(r, d0 + fd, v, L);
          else *reinterpret_cast<float4*>(part + r * HD + d0 + fd) = v;
        }
        if (!sync()) return;
      }
      if (!whole && (tid & 7) == 0) {
        part[ROWS * HD + 2 * r] = top;
        part[ROWS * HD + 2 * r + 1] = L;
      }
    }
    if (tid == 0) poison = 0;
    if (!whole) {
      // the last piece to arrive joins them all
      const int64_t c_first = ux / run.share, c_last = (ux + p.tn - 1) / run.share;
      const int unit = p.kvh * run.items + p.item;
      __threadfence();
      if (!sync()) return;
      if (tid == 0) is_last = atomicAdd(a.count + unit, 1) == (int)(c_last - c_first);
      if (!sync()) return;
      if (is_last) {
        __threadfence();
        for (int k = tid; k < rows * (HD / 4); k += 128) {
          const int r = k / (HD / 4), d = k % (HD / 4) * 4;
          float top = -INFINITY, L = 0.f;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int64_t q0 = c_first; q0 <= c_last; q0 += 8) {
            float2 ml[8];
            float4 x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const int64_t q = min(q0 + u, c_last);
              const float* src = a.part + (2 * q + (run.share * q <= ux ? 1 : 0)) * ROWS * (HD + 2);
              ml[u] = __ldcg(reinterpret_cast<const float2*>(src + ROWS * HD + 2 * r));
              x[u] = __ldcg(reinterpret_cast<const float4*>(src + r * HD + d));
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              if (q0 + u > c_last) break;
              const float now = fmaxf(top, ml[u].x);
              const float fo = top == now ? 1.f : pa_ex2(top - now), fn = ml[u].x == now ? 1.f : pa_ex2(ml[u].x - now);
              top = now;
              L = L * fo + ml[u].y * fn;
              v.x = v.x * fo + x[u].x * fn, v.y = v.y * fo + x[u].y * fn;
              v.z = v.z * fo + x[u].z * fn, v.w = v.w * fo + x[u].w * fn;
            }
          }
          store(r, d, v, L);
        }
        if (tid == 0) a.count[unit] = 0;
      }
    }
    if (!sync()) return;  // wml, poison and is_last are read
  }
}

template <typename T, int HD, int MT, bool FANCY>
static cudaError_t launch(PagedAttnArgs& a, cudaStream_t s) {
  using F = Cfg<HD>;
  auto kern = paged_mma_kernel<T, HD, MT, FANCY>;
  CUtensorMap maps[2];
  if (cudaError_t e = paged_maps(a.c, TILE, maps)) return e;
  static thread_local uint64_t ready = 0;  // devices whose kernel may take this much shared memory
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  if (dev > 63 || !(ready >> dev & 1)) {
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM)) return e;
    if (dev < 64) ready |= 1ull << dev;
  }
  return launch_pdl_smem(kern, dim3(paged_ctas(16 * MT)), dim3(THREADS), F::SMEM, s, a, maps[0], maps[1]);
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

// K and V as 2-D tensors of rows; a box is (part of) one page of one kv head, 64
// dims wide, in the 128-byte swizzle.  x is 0 or 64 values: 16-byte boundaries.
cudaError_t paged_maps(const PagedView& c, int tile, CUtensorMap* maps) {
  const EncodeFn enc = encode_fn();
  if (!enc) return cudaErrorNotSupported;
  const cuuint64_t dims[2] = {(cuuint64_t)c.hd, (cuuint64_t)c.num_pages * c.kv_heads * c.page_size};
  const cuuint64_t strides[1] = {(cuuint64_t)c.hd * 2};
  const cuuint32_t box[2] = {64u, (cuuint32_t)(c.page_size < tile ? c.page_size : tile)}, ones[2] = {1, 1};
  for (int i = 0; i < 2; ++i)
    if (enc(&maps[i], c.dtype == ODI_CUDA_PAGED_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
            i ? c.v : c.k, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return cudaErrorInvalidValue;
  return cudaSuccess;
}

cudaError_t launch_paged_mma(PagedAttnArgs& a, int mt, bool fancy, cudaStream_t s) {
  const bool bf = a.c.dtype == ODI_CUDA_PAGED_BF16;
  auto by_rows = [&](auto t, auto hd) {
    using T = decltype(t);
    constexpr int HD = decltype(hd)::value;
    if (mt == 1) return fancy ? pmma::launch<T, HD, 1, true>(a, s) : pmma::launch<T, HD, 1, false>(a, s);
    return fancy ? pmma::launch<T, HD, 2, true>(a, s) : pmma::launch<T, HD, 2, false>(a, s);
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (a.c.hd == 128) return bf ? by_rows(__nv_bfloat16{}, D128{}) : by_rows(__half{}, D128{});
  return bf ? by_rows(__nv_bfloat16{}, D64{}) : by_rows(__half{}, D64{});
}

}  // namespace odi_cuda

using namespace odi_cuda;

extern "C" {

// Error word, pieces, then a counter per unit.  The pieces' place has one size,
// so that a scratch serves any batch whose counters fit.
constexpr size_t PART_OFF = 256, COUNT_OFF = PART_OFF + (size_t)2 * PAGED_SMS * PAGED_ROWS_MAX * (128 + 2) * 4;
static_assert(2 * paged_ctas(32) * 32 <= 2 * PAGED_SMS * PAGED_ROWS_MAX, "pieces of the narrow items");

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
  const uintptr_t x = (uintptr_t)d_q, x1 = x + 2 * (uintptr_t)((tokens - 1) * ld_q + width), y = (uintptr_t)d_out,
                  y1 = y + (out32 ? 4 : 2) * (uintptr_t)((tokens - 1) * ld_out + width);
  if (x < y1 && y < x1) return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, "attention_paged: d_out overlaps d_q");
  a.q = d_q, a.ld_q = ld_q, a.out = d_out, a.ld_out = ld_out, a.out32 = out32;
  a.table = tables->table, a.max_pages = tables->max_pages;
  a.starts = batch->starts, a.lens = batch->lens, a.header = batch->work;
  a.w = paged_work(batch->work, batch->requests, g.max_items);
  a.G = g.G, a.out_rows = tokens;
  a.inv_G = g.G > 1 ? (unsigned)(((1ull << 32) + g.G - 1) / g.G) : 0;
  a.scale_log2 = softcap > 0.f ? scale / softcap : scale * 1.4426950408889634f;
  a.cap_log2 = softcap * 1.4426950408889634f;
  a.slopes = d_slopes;
  a.vec = !((uintptr_t)d_q & 15) && !(ld_q & 7);
  a.vec_out = !((uintptr_t)d_out & 15) && !(ld_out & 7);
  a.least = 1;
  a.err = static_cast<int*>(d_scratch);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(d_scratch) + PART_OFF);
  a.count = reinterpret_cast<int*>(static_cast<uint8_t*>(d_scratch) + COUNT_OFF);
  const bool fancy = softcap > 0.f || d_slopes;
  cudaStream_t s = (cudaStream_t)stream;
  return kv_launched(g.rows <= 32 ? launch_paged_mma(a, g.rows / 16, fancy, s) : launch_paged_tc(a, fancy, s), "attention_paged");
}

}  // extern "C"
