// tree_attention.cu -- attention of a tree of drafted tokens over a KV cache.
//
// Node t of T drafted nodes is stored in cache slot pos + t.  It sees every
// slot below pos and, of the T tree slots, those whose bit is set in its mask
// row (its ancestors and itself; without a mask, nodes 0..t):
//   s_tj = scale * q_t . k_j,   m_t = max over visible j of s_tj
//   o_t  = sum_j exp(s_tj - m_t) v_j / sum_j exp(s_tj - m_t)
// A node that sees nothing gets zeros.  Slots outside the cache are not seen.
#include <math.h>

#include "../../include/odi_cuda.h"
#include "internal.h"
#include "kv_cache.cuh"
#include "pdl_launch.cuh"
#include "tree_attention.cuh"

namespace odi_cuda {
namespace {

// Rows of one kv head: r = t * G + g for node t and the g-th of the G query
// heads that share the kv head, R = T * G in all.  A CTA takes NR * 8 of them
// (blockIdx.y) and every nsplit-th share of the cache (blockIdx.z); its four
// warps work alone until the end, each on groups of 16 positions:
//
//   S^T [16 positions x 8 rows] = K . Q^T     (mma.sync, positions as M)
//   O^T [hd x 8 rows]          += V^T . P^T   (mma.sync, dims as M)
//
// With the rows as the narrow side of the product, 8 rows waste nothing, and
// both operands that come from the cache are read straight from global memory
// into the fragments: which dims (or positions) a fragment register holds is
// free as long as both factors agree, so lane (g, c) takes whole 16-byte
// pieces -- K: pieces c, c + 4, ... of rows g and g + 8; V: dims 16 g .. 16 g +
// 15 of positions 2c, 2c + 1, 2c + 8, 2c + 9 -- and no shared memory or barrier
// stands between the cache and the tensor core.  The next group's pieces are
// requested as soon as this group's are used up.
//
// fp32 results from 16- and 8-bit products:
//  * int8 cache: q is fixed point, 24 bits against the row's largest value, in
//    three signed 8-bit digits; the digit products with the codes are exact
//    in 32-bit integers, and joined and scaled in fp32.
//  * fp16 cache: q, scaled by a power of two, is the sum of two fp16 values
//    (22 bits).
//  * P (times the int8 row's scale of V) is the sum of two fp16 values, so
//    the codes, or the fp16 values, of V enter unrounded.
//
// Softmax: m is a reference, not the running maximum: it moves only when a
// weight (int8: weight * scale, what the values enter with) passes 2^15 against
// it, by whole powers of two to where the largest is 2^8 (fp16: 2^12), and the
// sums are scaled; fp16 pairs hold 22 bits of weights from 2^-3 and smaller ones
// to within 2^-25, 2^-33 (2^-37) of the largest.
//
// Bound by the fetch of the cache for long ones: one token, 64 / 8 heads, 131001
// int8 positions 58.5 us, 277 MB at 4.7 TB/s (the copy peak gives 42); 518 fp16
// positions of 32 / 32 heads take 9.6 us, of which the fetch is 1.3: latency of
// launch, first loads and join.
constexpr int TA_WARPS = 4;
constexpr int TA_THREADS = 32 * TA_WARPS;
constexpr int TA_GROUP = 16;
// Rows per kv head above which (head_dim 128) the tcgen05 kernel runs.  32 / 8
// heads, 500 / 4000 / 32000 positions, us here and there: 8 rows of int8 5.9 /
// 11.8 / 20.9 and 7.3 / 10.4 / 23.1, of fp16 6.5 / 13.5 / 33.4 and 8.1 / 11.2 /
// 27.5; 12 rows of int8 8.1 / 13.8 / 29.8 and 7.3 / 10.5 / 23.4, of fp16 8.9 /
// 15.9 / 44.0 and 8.3 / 11.2 / 27.6.  The length is not known on the host.
constexpr int TA_TC_ROWS = 8;
constexpr float TA_TOP = 32768.f;            // a weight past this moves the reference
// log2 of the largest right after that.  An fp16 cache's scales, those of its
// values, are not known: its unit is 2^4 finer.
template <bool I8>
constexpr float TA_UNIT = I8 ? 8.f : 12.f;

__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_h(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 8x8 transpose of 16-bit values held two per lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Loads of what the kernel before this one may have written: from L2, since
// a line of this SM's L1 may be older than the programmatic wait.
__device__ __forceinline__ uint4 ldg16(const void* p) {
  uint4 v;
  asm volatile("ld.global.cg.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ldg8(const void* p) {
  uint2 v;
  asm volatile("ld.global.cg.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
// Fragment registers of one group: KW words of K per row and lane, VW of V per
// position and lane, and the words of Q per lane and row tile.
template <int HD, bool I8>
struct Frag {
  static constexpr int KW = HD * (I8 ? 1 : 2) / 16;  // words of one K row on a lane (4 lanes share a row)
  static constexpr int VW = HD * (I8 ? 1 : 2) / 32;  // words of one V row on a lane (8 lanes share a row)
  static constexpr int DIG = I8 ? 3 : 2;             // digits of q
  static constexpr int QW = KW * DIG;                // words of Q on a lane, per row tile
  static constexpr int MT = HD / 16;                 // 16-dim tiles of O^T
};

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* p, int piece_stride) {
  if (N == 2) {
    const uint2 v = ldg8(p);
    w[0] = v.x, w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = ldg16(p + (int64_t)i * piece_stride);
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  }
}

template <int HD, int NR, bool I8>
struct TreeSmem {
  using F = Frag<HD, I8>;
  static constexpr int Q = NR * F::QW * 32 * 4;
  static constexpr int ROWC = NR * 8 * 8;  // each row's factor of the scores, and its node
  static constexpr int FOLD = TA_WARPS * NR * 8 * HD * 4;
  static constexpr int BYTES = ROWC + (Q > FOLD ? Q : FOLD);
};

template <int HD, int NR, bool I8>
__global__ void __launch_bounds__(TA_THREADS, NR == 1 ? 4 : NR == 2 ? 3 : 2) tree_attn_kernel(const TreeArgs a) {
  using F = Frag<HD, I8>;
  constexpr int KW = F::KW, VW = F::VW, DIG = F::DIG, QW = F::QW, MT = F::MT;
  constexpr int ROWB = HD * (I8 ? 1 : 2);
  extern __shared__ __align__(16) uint8_t ta_smem[];
  float* rowc = reinterpret_cast<float*>(ta_smem);
  int* rowt = reinterpret_cast<int*>(ta_smem) + NR * 8;
  uint32_t* qf = reinterpret_cast<uint32_t*>(ta_smem + TreeSmem<HD, NR, I8>::ROWC);  // [NR][QW / 4][lane][4]
  float* fold = reinterpret_cast<float*>(qf);                                        // [warp][row][HD], at the end
  __shared__ float2 ml[TA_WARPS][NR * 8], cta_ml[NR * 8];                            // reference and sum of each row
  pdl_launch_dependents();
  pdl_wait();
  const int kvh = blockIdx.x, tile = blockIdx.y, split = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int pos = __ldcg(&a.st->pos);
  const int len = (int)max(0ll, min((long long)a.c.ctx, (long long)pos + a.tokens));
  const int ngroups = (len + TA_GROUP - 1) / TA_GROUP;

  // the first group is requested before anything else
  const int64_t head = (int64_t)kvh * a.c.ctx;
  const uint8_t* kb = static_cast<const uint8_t*>(a.c.k) + head * ROWB;
  const uint8_t* vb = static_cast<const uint8_t*>(a.c.v) + head * ROWB;
  const float* ks = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.c.k) + a.c.scale_off) + head;
  const float* vsc = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.c.v) + a.c.scale_off) + head;

  uint32_t kw[2][KW], vw[4][VW];
  float dk[2], dv[2];
  auto load_k = [&](int grp) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = min(grp * TA_GROUP + g + 8 * i, len - 1);  // rows past the end repeat the last: not seen
      load_words<KW>(kw[i], kb + (int64_t)row * ROWB + c * 16, 64);
      if (I8) dk[i] = __ldcg(ks + row), dv[i] = __ldcg(vsc + row);
    }
  };
  auto load_v = [&](int grp) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = min(grp * TA_GROUP + 2 * c + (i & 1) + 8 * (i >> 1), len - 1);
      load_words<VW>(vw[i], vb + (int64_t)row * ROWB + g * (ROWB / 8), 16);
    }
  };
  // The host splits for a full cache: of the clusters that the length at hand
  // does not give two groups per warp, only the first stays.
  const int C = (int)cluster_nranks(), rank = (int)cluster_rank_of();
  const int nclusters = max(1, min(a.nsplit / C, (ngroups + 2 * TA_WARPS * C - 1) / (2 * TA_WARPS * C)));
  if (split >= nclusters * C) return;
  const int step = nclusters * C * TA_WARPS;
  int grp = split * TA_WARPS + warp;
  if (grp < ngroups) {
    load_k(grp);
    load_v(grp);
  }

  // ---- Q: warp w lays out rows w, w + TA_WARPS, ... as digits in fragment
  // order.  Each row is scaled by a power of two: to 2^21 .. 8.35e6 as an
  // integer (three signed digits hold 127 * (2^16 + 2^8 + 1)), or to 2^13 ..
  // 2^14 as fp16 pairs; rowc takes the scale back out.
  {
    constexpr int PL = HD / 32, RW = NR * 8 / TA_WARPS;
    float v[RW][PL];
    int rt[RW];
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const int r = tile * NR * 8 + warp + i * TA_WARPS;
      rt[i] = r < a.R ? row_node(a, r) : -1;
#pragma unroll
      for (int e = 0; e < PL; ++e) v[i][e] = 0.f;
      if (r < a.R) {
        const float* src = a.q + (int64_t)rt[i] * a.ld_q + (int64_t)(kvh * a.G + r - rt[i] * a.G) * HD + lane * PL;
#pragma unroll
        for (int e = 0; e < PL; ++e) v[i][e] = __ldcg(src + e);
      }
    }
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      const int n = warp + i * TA_WARPS;
      float am = 0.f;
      bool ok = true;
#pragma unroll
      for (int e = 0; e < PL; ++e) am = fmaxf(am, fabsf(v[i][e])), ok = ok && finite(v[i][e]);
#pragma unroll
      for (int x = 16; x; x >>= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, x));
      ok = __all_sync(0xffffffffu, ok);
      int ex = (int)(__float_as_uint(am) >> 23) - 127;  // am = 1 .. 2 times 2^ex
      if (I8 && am * pow2(-min(max(ex, -100), 126)) > 1.99f) ++ex;
      ex = min(max(ex, -100), 126);
      const float lift = pow2(-ex), up = I8 ? q_units(am) : 8192.f;
      if (lane == 0) {
        rowc[n] = ok ? q_factor(a.scale_log2, 1.f / up, ex) : __int_as_float(0x7fc00000);
        rowt[n] = rt[i];
      }
      uint8_t* dst = reinterpret_cast<uint8_t*>(qf) + (n >> 3) * QW * 128;
      const int gn = n & 7;
      if (I8) {
        // dims 16 ch + 4 w + b sit in byte b of word w of piece ch on lane ch % 4
        int dig[PL];
#pragma unroll
        for (int e = 0; e < PL; ++e) dig[e] = ok ? __float2int_rn(v[i][e] * lift * up) : 0;
        const int d = lane * PL, ch = d >> 4, w = (d >> 2) & 3, b = d & 3;
#pragma unroll
        for (int k = DIG - 1; k >= 0; --k) {
          uint32_t bytes = 0;
#pragma unroll
          for (int e = 0; e < PL; ++e) {
            const int lo = (int)(int8_t)(dig[e] & 255);
            dig[e] = (dig[e] - lo) >> 8;
            bytes |= (uint32_t)(lo & 255) << (8 * e);
          }
          const int word = k * KW + (ch >> 2) * 4 + w;
          uint8_t* at = dst + ((word >> 2) * 32 + gn * 4 + (ch & 3)) * 16 + (word & 3) * 4 + b;
          if (PL == 4) *reinterpret_cast<uint32_t*>(at) = bytes;
          else *reinterpret_cast<uint16_t*>(at) = (uint16_t)bytes;
        }
      } else {
#pragma unroll
        for (int e = 0; e < PL; e += 2) {
          const int d = lane * PL + e, ch = d >> 3, w = (d >> 1) & 3;
          const float x0 = ok ? v[i][e] * lift * up : 0.f, x1 = ok ? v[i][e + 1] * lift * up : 0.f;
          const __half2 hi = __floats2half2_rn(x0, x1);
          const float2 back = __half22float2(hi);
          const __half2 lo = __floats2half2_rn(x0 - back.x, x1 - back.y);
#pragma unroll
          for (int k = 0; k < DIG; ++k) {
            const int word = k * KW + (ch >> 2) * 4 + w;
            *reinterpret_cast<uint32_t*>(dst + ((word >> 2) * 32 + gn * 4 + (ch & 3)) * 16 + (word & 3) * 4) = h2u(k ? lo : hi);
          }
        }
      }
    }
  }
  __syncthreads();

  float o[NR][MT][4], m[NR][2], l[NR][2], rc[NR][2];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[r][j][e] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) m[r][e] = TA_NONE, l[r][e] = 0.f, rc[r][e] = rowc[r * 8 + 2 * c + e];
  }
  for (; grp < ngroups; grp += step) {
    const int p0 = grp * TA_GROUP;
    const bool edge = p0 + TA_GROUP > min(pos, len);  // holds tree slots, or ends past the last
    unsigned bad = 0;                       // positions of the group whose V is not finite (fp16)
    if (!I8 && edge) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        bool fin = true;
#pragma unroll
        for (int w = 0; w < VW; ++w)
          fin = fin && (vw[i][w] & 0x7c00u) != 0x7c00u && (vw[i][w] & 0x7c000000u) != 0x7c000000u;
        unsigned all = __ballot_sync(0xffffffffu, !fin);
        all |= all >> 16;
        all |= all >> 8;
        all |= all >> 4;
#pragma unroll
        for (int cc = 0; cc < 4; ++cc)
          if ((all >> cc) & 1u) bad |= 1u << (2 * cc + (i & 1) + 8 * (i >> 1));
        // whoever sees such a position gets NaN through its sum; nobody else may meet it
        if ((all >> c) & 1u)
#pragma unroll
          for (int w = 0; w < VW; ++w) vw[i][w] = 0;
      }
    }
    float dvc[2];  // a scale near 0 stands for 2^-64: a key whose values are nothing moves no reference
    if (I8)
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // a row whose scale of K or V is not finite gives NaN to who sees it
        if (!finite(dv[i])) dk[i] = __int_as_float(0x7fc00000), dv[i] = 0.f;
        if (!finite(dk[i])) dk[i] = __int_as_float(0x7fc00000);
        dvc[i] = fmaxf(dv[i], 0x1p-64f);
      }
    uint32_t ph[NR][2], pl[NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float s[4];
      const uint4* qr = reinterpret_cast<const uint4*>(qf) + r * (QW / 4) * 32 + lane;
      if (I8) {
        int acc[DIG][4];
#pragma unroll
        for (int k = 0; k < DIG; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[k][e] = 0;
#pragma unroll
        for (int w = 0; w < KW; w += 4) {
          const uint32_t a0[4] = {kw[0][w], kw[1][w], kw[0][w + 1], kw[1][w + 1]};
          const uint32_t a1[4] = {kw[0][w + 2], kw[1][w + 2], kw[0][w + 3], kw[1][w + 3]};
          uint4 b[DIG];
#pragma unroll
          for (int k = 0; k < DIG; ++k) b[k] = qr[((k * KW + w) >> 2) * 32];
#pragma unroll
          for (int k = 0; k < DIG; ++k) mma_s8(acc[k], a0, b[k].x, b[k].y);
#pragma unroll
          for (int k = 0; k < DIG; ++k) mma_s8(acc[k], a1, b[k].z, b[k].w);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)  // digits joined: |digit sums| < 2^21, so each is exact in fp32
          s[e] = fmaf((float)acc[0][e], 65536.f, fmaf((float)acc[1][e], 256.f, (float)acc[DIG - 1][e])) *
                 dk[e >> 1] * rc[r][e & 1];
      } else {
        float acc[2 * DIG][4];  // high and low halves, two chains of each
#pragma unroll
        for (int k = 0; k < 2 * DIG; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[k][e] = 0.f;
#pragma unroll
        for (int w = 0; w < KW; w += 4) {
          const uint32_t a0[4] = {kw[0][w], kw[1][w], kw[0][w + 1], kw[1][w + 1]};
          const uint32_t a1[4] = {kw[0][w + 2], kw[1][w + 2], kw[0][w + 3], kw[1][w + 3]};
#pragma unroll
          for (int k = 0; k < DIG; ++k) {
            const uint4 b = qr[((k * KW + w) >> 2) * 32];
            mma_h(acc[2 * k], a0, b.x, b.y);
            mma_h(acc[2 * k + 1], a1, b.z, b.w);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = (acc[0][e] + acc[1][e] + (acc[2][e] + acc[3][e])) * rc[r][e & 1];
      }
      if (edge) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const unsigned see = seen_bits(a, rowt[r * 8 + 2 * c + e], p0, pos, len);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (!((see >> (g + 8 * i)) & 1u)) s[2 * i + e] = -INFINITY;
            else if (!I8 && ((bad >> (g + 8 * i)) & 1u)) s[2 * i + e] = __int_as_float(0x7fc00000);
          }
        }
      }
      float p[4], top[2];
      // weights, and each row's largest on this lane
      auto weigh = [&]() {
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = ex2(s[e] - m[r][e & 1]);
#pragma unroll
        for (int e = 0; e < 2; ++e)
          top[e] = I8 ? fmaxf(p[e] * dvc[0], p[2 + e] * dvc[1]) : fmaxf(p[e], p[2 + e]);
      };
      weigh();
      if (__any_sync(0xffffffffu, fmaxf(top[0], top[1]) > TA_TOP)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // each row by itself: a row's result does not depend on its neighbours
          float mx = fmaxf(s[e], s[2 + e]);
          if (I8) mx = fmaxf(s[e] + __log2f(dvc[0]), s[2 + e] + __log2f(dvc[1]));
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) {
            top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], x));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          }
          if (!(top[e] > TA_TOP)) continue;
          const float mn = ceilf(mx) - TA_UNIT<I8>, d = m[r][e] - mn;
          const float corr = d < -126.f ? 0.f : pow2((int)d);
          m[r][e] = mn;
          l[r][e] *= corr;
#pragma unroll
          for (int j = 0; j < MT; ++j) o[r][j][e] *= corr, o[r][j][2 + e] *= corr;
        }
        __syncwarp();  // movmatrix and the products below want the whole warp
        weigh();
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) l[r][e] += p[e] + p[2 + e];
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = I8 ? p[e] * dv[e >> 1] : p[e];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const __half2 hi = __floats2half2_rn(w[2 * i], w[2 * i + 1]);
        const float2 back = __half22float2(hi);
        const __half2 lo = __floats2half2_rn(w[2 * i] - back.x, w[2 * i + 1] - back.y);
        ph[r][i] = transpose8(h2u(hi));
        pl[r][i] = transpose8(h2u(lo));
      }
    }
    if (grp + step < ngroups) load_k(grp + step);
    constexpr int JB = NR == 1 ? 4 : NR == 2 ? 2 : 1;  // independent sums between two products into one
#pragma unroll
    for (int j0 = 0; j0 < MT; j0 += JB) {
      uint32_t af[JB][4];
#pragma unroll
      for (int u = 0; u < JB; ++u) {  // dims 16 g + 2 j (fragment row g) and + 1 (row g + 8)
        const int j = j0 + u;
        if (I8) {
          const int wi = j >> 1;
          const uint32_t sel = (j & 1) ? 0x7362u : 0x5140u;  // bytes 2j, 2j + 1 of two positions
          const uint32_t t0 = __byte_perm(vw[0][wi] ^ 0x80808080u, vw[1][wi] ^ 0x80808080u, sel);
          const uint32_t t1 = __byte_perm(vw[2][wi] ^ 0x80808080u, vw[3][wi] ^ 0x80808080u, sel);
          const __half2 k = __float2half2_rn(1152.f);  // 1024 + (code + 128) in fp16
          af[u][0] = h2u(__hsub2(u2h(__byte_perm(t0, 0x64646464u, 0x4140u)), k));
          af[u][1] = h2u(__hsub2(u2h(__byte_perm(t0, 0x64646464u, 0x4342u)), k));
          af[u][2] = h2u(__hsub2(u2h(__byte_perm(t1, 0x64646464u, 0x4140u)), k));
          af[u][3] = h2u(__hsub2(u2h(__byte_perm(t1, 0x64646464u, 0x4342u)), k));
        } else {
          af[u][0] = __byte_perm(vw[0][j], vw[1][j], 0x5410u);
          af[u][1] = __byte_perm(vw[0][j], vw[1][j], 0x7632u);
          af[u][2] = __byte_perm(vw[2][j], vw[3][j], 0x5410u);
          af[u][3] = __byte_perm(vw[2][j], vw[3][j], 0x7632u);
        }
      }
#pragma unroll
      for (int u = 0; u < JB; ++u)
#pragma unroll
        for (int r = 0; r < NR; ++r) mma_h(o[r][j0 + u], af[u], pl[r][0], pl[r][1]);
#pragma unroll
      for (int u = 0; u < JB; ++u)
#pragma unroll
        for (int r = 0; r < NR; ++r) mma_h(o[r][j0 + u], af[u], ph[r][0], ph[r][1]);
    }
    if (grp + step < ngroups) load_v(grp + step);
  }

  // ---- the warps' shares, then the cluster's, then the clusters'
  __syncthreads();  // every warp is done with the fragments of Q
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = l[r][e];
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      const int n = r * 8 + 2 * c + e;
      float* f = fold + (warp * NR * 8 + n) * HD + MT * 2 * g;
      if (g == 0) ml[warp][n] = make_float2(m[r][e], sum);
#pragma unroll
      for (int j = 0; j < MT; ++j) *reinterpret_cast<float2*>(f + 2 * j) = make_float2(o[r][j][e], o[r][j][2 + e]);
    }
  __syncthreads();
  const int rows = min(NR * 8, a.R - tile * NR * 8);
  constexpr int V4 = HD / 4;
  float4* fold4 = reinterpret_cast<float4*>(fold);
  if (threadIdx.x < NR * 8) {  // each warp's factor, the CTA's reference and sum
    const int n = threadIdx.x;
    float M = TA_NONE, L = 0.f;
#pragma unroll
    for (int w = 0; w < TA_WARPS; ++w) M = fmaxf(M, ml[w][n].x);
#pragma unroll
    for (int w = 0; w < TA_WARPS; ++w) {
      const float f = ex2(ml[w][n].x - M);
      L += ml[w][n].y * f;
      ml[w][n].x = f;
    }
    cta_ml[n] = make_float2(M, L);
  }
  __syncthreads();
  auto add = [](float4& x, const float4& y, float f) {
    x.x = fmaf(y.x, f, x.x), x.y = fmaf(y.y, f, x.y), x.z = fmaf(y.z, f, x.z), x.w = fmaf(y.w, f, x.w);
  };
#pragma unroll 2
  for (int i = threadIdx.x; i < rows * V4; i += TA_THREADS) {
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < TA_WARPS; ++w) add(A, fold4[w * NR * 8 * V4 + i], ml[w][i / V4].x);
    fold4[i] = A;
  }
  tree_join<HD, NR * 8, TA_THREADS>(a, threadIdx.x, rowt, cta_ml, fold, rows, C, rank, nclusters);
}

// Which kernel and how many rows per CTA; room: CTAs resident at once.
struct TreePlan {
  bool tc;  // the tcgen05 kernel
  int rows, tiles, units;
  int64_t room, most;  // most: CTAs that a full cache gives positions to, per unit
  size_t part_off, bytes;
};

TreePlan tree_plan(int tokens, int heads, int kv_heads, int hd, int ctx) {
  TreePlan p;
  const int64_t R = (int64_t)tokens * (heads / kv_heads);
  p.tc = hd == 128 && R > TA_TC_ROWS;
  const int64_t block = p.tc ? 128 : TA_GROUP * TA_WARPS;
  p.most = ((int64_t)ctx + block - 1) / block;
  // A CTA of 32 rows takes 0.98 us per block of 128 positions, one of 64 rows
  // 1.39 and about 3.4 more to start and to join.  32 / 8 heads, us with 32 and
  // with 64 rows, of int8 (fp16): 52 rows per kv head over 4000 positions 13.8 and
  // 15.0 (14.1 and 15.5), 16000 24.6 and 23.7 (25.7 and 23.6), 32000 39.4 and 35.0
  // (41.1 and 35.4); 256 rows over 500 11.2 and 12.5 (11.8 and 13.3), 2000 17.3 and
  // 17.5 (17.6 and 17.7), 4000 24.3 and 22.2 (24.3 and 21.4), 32000 120 and 96.5
  // (128 and 87); 96 rows over 32000 (three tiles against two) 51.1 and 56.9 (51.9
  // and 52.8).
  const int64_t t32 = (R + 31) / 32, t64 = (R + 63) / 64;
  const bool narrow = kv_heads * p.most * (98 * t32 - 139 * t64) < 340 * TA_SMS;
  p.rows = p.tc ? (narrow ? 32 : 64) : R <= 8 ? 8 : R <= 16 ? 16 : 32;
  p.room = TA_SMS * (p.tc ? 1 : p.rows == 8 ? 4 : p.rows == 16 ? 3 : 2);
  p.tiles = (int)((R + p.rows - 1) / p.rows);
  p.units = kv_heads * p.tiles;
  // The scratch is laid out alike whatever the number of tokens, so that calls
  // of any T may share one: counters and shares are used only by units split
  // over several clusters, whose CTAs are all resident -- at most 4 per SM of 8
  // rows, 3 of 16, 2 of 32, 1 of 64.
  p.part_off = (16 + (size_t)TA_SMS * 4 * 8 * 4 + 255) / 256 * 256;
  p.bytes = p.part_off + (size_t)TA_SMS * 64 * (hd + 4) * 4;
  return p;
}

template <int HD, int NR, bool I8>
cudaError_t launch_tree(TreeArgs a, const TreePlan& p, cudaStream_t s) {
  auto kern = tree_attn_kernel<HD, NR, I8>;
  static TreeLaunch state;
  return launch_tree_clusters(state, (const void*)kern, a, p.tiles, p.units, p.room, p.most, TA_THREADS, TreeSmem<HD, NR, I8>::BYTES, s,
                              [&](const cudaLaunchConfig_t& cfg) { return cudaLaunchKernelEx(&cfg, kern, a); });
}

template <int HD>
cudaError_t launch_tree_hd(const TreeArgs& a, const TreePlan& p, cudaStream_t s) {
  if (a.c.dtype == ODI_CUDA_KV_I8)
    return p.rows == 8 ? launch_tree<HD, 1, true>(a, p, s) : p.rows == 16 ? launch_tree<HD, 2, true>(a, p, s)
                                                                          : launch_tree<HD, 4, true>(a, p, s);
  return p.rows == 8 ? launch_tree<HD, 1, false>(a, p, s) : p.rows == 16 ? launch_tree<HD, 2, false>(a, p, s)
                                                                         : launch_tree<HD, 4, false>(a, p, s);
}

bool tree_shape_ok(int tokens, int heads, int kv_heads, int hd, int ctx) {
  return tokens >= 1 && tokens <= ODI_CUDA_TREE_MAX && heads >= 1 && heads <= 1024 && kv_heads >= 1 &&
         heads % kv_heads == 0 && (hd == 64 || hd == 128) && ctx >= 1;
}

}  // namespace
}  // namespace odi_cuda

using namespace odi_cuda;

extern "C" {

size_t odi_cuda_attention_tree_scratch_bytes(int tokens, int heads, int kv_heads, int head_dim, int ctx) {
  if (!tree_shape_ok(tokens, heads, kv_heads, head_dim, ctx)) return 0;
  return tree_plan(tokens, heads, kv_heads, head_dim, ctx).bytes;
}

int odi_cuda_attention_tree(const float* d_q, int64_t ld_q, const odi_cuda_kv_cache* cache, float* d_out,
                            const uint32_t* d_mask, const odi_cuda_decode_state* d_state, int tokens, int heads,
                            float scale, void* d_scratch, size_t scratch_bytes, void* stream) {
  KvView v;
  if (int rc = kv_view(cache, &v, "attention_tree")) return rc;
  auto bad = [](const char* m) { return set_error(ODI_CUDA_ERR_INVALID_ARGUMENT, m); };
  if (!d_q || !d_out || !d_state || !d_scratch) return bad("attention_tree: null argument");
  if (!tree_shape_ok(tokens, heads, v.kv_heads, v.hd, v.ctx))
    return bad("attention_tree: 1 to ODI_CUDA_TREE_MAX tokens, heads (at most 1024) a multiple of kv_heads");
  if (ld_q < (int64_t)heads * v.hd) return bad("attention_tree: the query stride is shorter than its row");
  if (!isfinite(scale)) return bad("attention_tree: the scale must be finite");
  if (((uintptr_t)d_q | (uintptr_t)d_out | (uintptr_t)d_mask | (uintptr_t)d_state) & 3 || ((uintptr_t)d_scratch & 15))
    return bad("attention_tree: misaligned buffer");
  const int64_t width = (int64_t)heads * v.hd;
  if (rows_overlap(d_q, ld_q, width, d_out, width, width, tokens)) return bad("attention_tree: the output overlaps the queries");
  const TreePlan p = tree_plan(tokens, heads, v.kv_heads, v.hd, v.ctx);
  if (scratch_bytes < p.bytes) return bad("attention_tree: scratch too small");
  TreeArgs a{};
  a.q = d_q, a.ld_q = ld_q, a.out = d_out, a.c = v, a.mask = d_mask, a.mask_words = (tokens + 31) / 32;
  a.st = reinterpret_cast<const DecodeState*>(d_state);
  a.tokens = tokens, a.heads = heads, a.G = heads / v.kv_heads, a.R = tokens * a.G;
  a.inv_G = (unsigned)((0x100000000ull + a.G - 1) / a.G);
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  a.count = reinterpret_cast<int*>(static_cast<uint8_t*>(d_scratch) + 16);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(d_scratch) + p.part_off);
  const cudaError_t e = p.tc ? launch_tree_tc(a, p.rows, p.tiles, p.units, p.most, static_cast<int*>(d_scratch), (cudaStream_t)stream)
                        : v.hd == 128 ? launch_tree_hd<128>(a, p, (cudaStream_t)stream)
                                    : launch_tree_hd<64>(a, p, (cudaStream_t)stream);
  return kv_launched(e, "attention_tree");
}

}  // extern "C"
