// mx_attention.hip -- attention of sequences that share a prefix
// (mxs_prefix_attention):
//
//   s[i] = scale q . keys[i],  lse = ln sum_i exp(s[i]),
//   out = sum_i exp(s[i] - lse) values[i],  weight[i] += exp(s[i] - lse)
//
// over the group's prefix and, causally, the row's suffix.
//
// The prefix is read once for all the queries of a group that share a cache head
// (beams x tokens x query heads a cache head), each suffix once for its own.  What
// bounds it is that stream, 4 dim bytes a position and cache head, up to about 300
// queries a cache head; with more, the products (4 dim flops a query and position).
//
// attention_tile_kernel: a workgroup takes a block of queries over a part of the
// positions, 64 at a time, which loads write straight into LDS.  The softmax goes
// along in one pass: scores of a tile, exponentials against a running reference,
// products with the values.  attention_join_kernel joins a query's parts;
// attention_weights_kernel makes the weights from the scores once more: storing the
// scores would write and read 4 bytes a query and position, reading the keys again
// takes 2 dim bytes a position, often still in a cache.  Parts, and not one workgroup
// a cache head, because 8 cache heads of one request would leave 248 of 256 CUs idle.
//
// us a pass, dim 128 and 8 cache heads: 4 beams of 4 heads a cache head on 131072
// positions 96 (at a large copy's 4.92 TB/s the keys and values alone would take 110: a
// stream that is only read is faster); 8 groups of these on up to 4096 positions 31.2
// (24.0), with weights 47.7; 64 sequences of 8 heads on 32768 positions 93: 742 TFLOP/s,
// matrix pipes 34% busy (44 at a large product's rate); one request of 4 beams of 2 heads
// on 512 positions 8.4.
// The 64 sequences step by step: one wave a query 27463; 64 queries a wave, whose sums
// went back and forth between the two kinds of registers, 370; 32 a wave 249; jobs
// spread over the XCDs (a prefix's had been on three of them) 99; two workgroups of four
// waves a CU instead of one of eight 94; the join's first loads early 93.  Tried there and left, us of the tile
// kernel's prefixes: the next tile's scores beside this one's exponentials 84, in a fixed
// order of issue 112, as it is 78; a meeting every second tile 78.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/mx_sampler.h"
#include "mxs_attention_checks.h"
#include "mxs_attention_plan.h"
#include "mxs_ctx.h"
#include "mxs_device.h"

namespace mxs {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct AttArgs {
  const __bf16 *q, *pk, *pv, *k, *v;
  __bf16* out;
  uint64_t qr, qt, qh, pg, ph, pp, kr, kh, kp, orow, ot, oh;   // strides in elements
  const int32_t *plen, *len;
  float *lse, *pw, *w;
  uint32_t W, T, H, KV, D, P, N, per;   // per: query heads a cache head has
  uint32_t g0, ng, b0, wb, t0, nt;      // this launch's groups, rows of each, tokens
  uint32_t nrb, nsb, sp, ss, slots;     // blocks of queries of a prefix and a suffix, parts of either, of a query
  uint32_t np, ns;                      // workgroups of prefixes, of suffixes
  uint32_t NQ;                          // queries: ng * wb * nt * H
  float c;                              // |scale| log2(e)
  uint32_t flip;                        // 0x8000 where the scale is negative: the queries' signs
  float* part;                          // [slots][NQ][DP] sums of a part's exponentials times its values
  float2* stat;                         // [slots][NQ] the part's reference (log2) and sum
  float* ref;                           // [NQ] log2 of a query's whole sum, inf for one that has seen nothing or does not count; NULL: no weights
};

__device__ __forceinline__ uint32_t att_len(const int32_t* len, uint32_t i, uint32_t most) {
  if (!len) return most;
  const int32_t n = len[i];
  return n <= 0 ? 0u : min((uint32_t)n, most);
}
// Suffix positions that token t sees.
__device__ __forceinline__ uint32_t att_seen(uint32_t len, uint32_t T, uint32_t t) {
  const int64_t n = (int64_t)len - T + t + 1;
  return n <= 0 ? 0u : (uint32_t)n;
}

// The largest, or the sum, over the four lanes that hold the same query.
__device__ __forceinline__ float max4(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float sum4(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// 2^(m - to) for the references of two parts; 0 for one that has seen nothing.
__device__ __forceinline__ float share_of(float m, float to) { return m == -INFINITY ? 0.0f : exp2_(m - to); }

__device__ __forceinline__ bf16x8 flipped(bf16x8 v, uint32_t flip) {
  s16x8 b = __builtin_bit_cast(s16x8, v);
  b ^= (short)flip;
  return __builtin_bit_cast(bf16x8, b);
}

// Sixteen bytes a lane into LDS (see mx_linear.hip).
__device__ __forceinline__ void att_load_lds(__bf16* lds, const __bf16* base, uint32_t off, uint32_t at) {
#if defined(__HIP_DEVICE_COMPILE__)
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, -1, 0x27000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, off, at, 0, 0);
#endif
}
// Four rows of a 16-bit array in LDS, transposed: of 16 lanes, lane l gives the
// address of four elements of row l / 4 from column 4 (l % 4) on and gets
// column l of the four rows.
__device__ __forceinline__ s16x4 read_turned(const __bf16* p) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
#else
  return s16x4{};
#endif
}
template <int N>
__device__ __forceinline__ void att_barrier() {   // all but the wave's N newest loads have landed; the workgroup meets
  static_assert(N < 64, "a six-bit counter");
  __asm__ volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);
  __asm__ volatile("s_barrier" ::: "memory");
}

// One job: the queries of a block over positions a..b of one cache head.
struct AttJob {
  const __bf16 *k, *v;      // position 0
  uint64_t stride;          // elements between positions
  uint32_t a, b;
  uint32_t g, kv;           // group within the launch, cache head
  uint32_t m0, m;           // first query of the block, queries of the cache head
  uint32_t row;             // suffix: the row within the group
  uint32_t len;             // suffix: its length
  uint32_t slot;
  bool pre;
};

// Where query m of a job belongs: its row within the group, token and head.
struct AttQuery {
  uint32_t b, t, h;
};
__device__ __forceinline__ AttQuery att_query(const AttArgs& A, const AttJob& J, uint32_t m) {
  uint32_t r = m, hh = 0u, t = 0u;
  if (A.per > 1u) r = m / A.per, hh = m - r * A.per;   // (uniform)
  if (A.nt > 1u) {
    const uint32_t x = r / A.nt;
    t = r - x * A.nt, r = x;
  }
  return {J.pre ? r : J.row, A.t0 + t, J.kv * A.per + hh};
}
__device__ __forceinline__ uint32_t att_id(const AttArgs& A, const AttJob& J, const AttQuery& x) {   // of the launch's queries
  return ((J.g * A.wb + x.b) * A.nt + x.t - A.t0) * A.H + x.h;
}
__device__ __forceinline__ uint64_t att_elements(const AttArgs& A, const AttJob& J, const AttQuery& x) {
  return (uint64_t)((A.g0 + J.g) * A.W + A.b0 + x.b) * A.qr + x.t * A.qt + x.h * A.qh;
}
__device__ __forceinline__ uint32_t att_row(const AttArgs& A, uint32_t row) {   // of the whole call
  return (A.g0 + row / A.wb) * A.W + A.b0 + row % A.wb;
}

struct AttEntry {
  uint32_t id, lim;   // of the launch's queries (~0: none); positions below lim are seen
  uint64_t at;        // its elements
};

// Scores as S^T = K Q^T on v_mfma_f32_16x16x32_bf16 (a lane holds four
// positions of one query), sums as O^T = V^T P^T: a lane's exponentials are the
// second operand as they lie (which positions a product takes together is free, as long
// as both operands agree), so that they never leave the registers; values are
// read transposed from LDS.  The exponentials are rounded to bf16 there, once: a
// second term would cost half as many products again, and its sign would make
// infinite values NaN; the sum and lse keep f32.
// WQ waves take other queries (16 RB each), WP waves other positions of the tile and
// meet at the end: with few queries the four waves split positions, so that LDS is read
// once; 32 queries a wave is what registers hold beside the sums of 128 elements.
template <int DP, int RB, int WQ, int WP, int S>
__device__ __forceinline__ void attention_job(const AttArgs& A, const AttJob& J, __bf16* Ks, __bf16* Vs, float2* stats,
                                              AttEntry* table, uint32_t* odd) {
  constexpr uint32_t PR = DP / 8, LR = 64 / PR;                  // 16-byte pieces of a row, rows a load takes
  constexpr int KS = DP / 32, DB = DP / 16, NW = WQ * WP;
  constexpr int PPW = ATT_TILE / WP, NB = PPW / 16;              // positions a wave takes of a tile, blocks of 16
  constexpr int LD = ATT_TILE / (int)LR / NW;                    // loads a wave issues for keys, and for values
  constexpr uint32_t TE = ATT_TILE * DP;                         // elements of a tile
  static_assert(LD * (int)LR * NW == (int)ATT_TILE, "the loads cover the tile");
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63u, lr = l & 15u, lg = l >> 4;
  const uint32_t wq = w % WQ, wp = w / WQ;

  const uint32_t nt = J.b > J.a ? (J.b - J.a + ATT_TILE - 1u) / ATT_TILE : 0u;
  // A row's pieces lie permuted by its low bits, so that the rows which a read
  // takes fall in different banks.
  auto turn_k = [](uint32_t row) { return PR == 8 ? (row >> 1) & 7u : row & 15u; };
  auto turn_v = [](uint32_t row) { return PR == 8 ? (row >> 1 & 3u) * 2u : (row & 7u) * 2u; };
  auto fetch = [&](uint32_t tile, const __bf16* __restrict__ from, __bf16* __restrict__ to, bool keys) __attribute__((always_inline)) {
    const uint32_t p0 = J.a + tile * ATT_TILE, have = min(ATT_TILE, J.b - p0);
    const __bf16* const base = from + (uint64_t)p0 * J.stride;
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const uint32_t row = (w * LD + i) * LR + l / PR, piece = (l % PR) ^ (keys ? turn_k(row) : turn_v(row));
      if (piece * 8u < A.D)
        att_load_lds(to + (w * LD + i) * LR * DP, base, (min(row, have - 1u) * (uint32_t)J.stride + piece * 8u) * 2u, 0u);
    }
  };
  if (A.D < DP && nt) {   // the keys' elements past dim are never loaded: zero (the values' reach only sums past dim)
    const uint32_t pad = PR - A.D / 8u;
    for (uint32_t i = threadIdx.x; i < S * ATT_TILE * pad; i += NW * 64) {
      const uint32_t row = i / pad, piece = A.D / 8u + i - row * pad;
      reinterpret_cast<bf16x8*>(Ks)[row * PR + (piece ^ turn_k(row % ATT_TILE))] = bf16x8{};
    }
  }
  // The first tiles' loads are under way while the queries are found.
#pragma unroll
  for (uint32_t t = 0; t < (uint32_t)S - 1u; ++t)
    if (t < nt) {
      fetch(t, J.k, Ks + t * TE, true);
      fetch(t, J.v, Vs + t * TE, false);
    }
  // What the block's queries are, worked out once.
  if (threadIdx.x < 16u * RB * WQ) {
    const uint32_t m = J.m0 + threadIdx.x;
    AttEntry e{~0u, 0u, 0ull};
    if (m < J.m) {
      const AttQuery x = att_query(A, J, m);
      e.id = att_id(A, J, x);
      e.lim = J.pre ? J.b : min(J.b, att_seen(J.len, A.T, x.t));
      e.at = att_elements(A, J, x);
    }
    table[threadIdx.x] = e;
  }
  if (threadIdx.x == 0) *odd = 0u;
  att_barrier<63>();

  // the queries, a fragment of each for every 32 elements; and where each one's positions end
  bf16x8 q[RB][KS];
  uint32_t lim[RB], least = J.b;
#pragma unroll
  for (int j = 0; j < RB; ++j) {
    const AttEntry e = table[(wq * RB + j) * 16u + lr];
    lim[j] = e.lim;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[j][s] = *reinterpret_cast<const bf16x8*>(A.q + e.at + min(32u * s + 8u * lg, A.D - 8u));
  }
#pragma unroll
  for (int j = 0; j < RB; ++j)
#pragma unroll
    for (int s = 0; s < KS; ++s) q[j][s] = 32u * s + 8u * lg < A.D ? flipped(q[j][s], A.flip) : bf16x8{};
  if (!J.pre) least = min(J.b, att_seen(J.len, A.T, A.t0));   // (of the launch's first token: none ends earlier)

  f32x4 acc[DB][RB] = {};
  float mc[RB], sum[RB];   // reference (log2) and sum of each query, the sum of this lane's positions
#pragma unroll
  for (int j = 0; j < RB; ++j) mc[j] = -INFINITY, sum[j] = 0.0f;
  const uint32_t kt = turn_k(lr);   // (rows of a fragment: lr more than a multiple of 16)
  const uint32_t vrow = 4u * lg + (lr >> 2), vt = turn_v(vrow);

  const uint32_t at = wp * PPW;   // this wave's first position within a tile
  auto read_k = [&](bf16x8 (&kf)[NB], const __bf16* __restrict__ kb, int ks) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NB; ++i)
      kf[i] = *reinterpret_cast<const bf16x8*>(kb + (at + 16u * i + lr) * DP + ((4u * ks + lg) ^ kt) * 8u);
  };
  auto mul_k = [&](f32x4 (&s)[NB][RB], const bf16x8 (&kf)[NB], int ks) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < RB; ++j)
        s[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[i], q[j][ks], ks ? s[i][j] : f32x4{}, 0, 0, 0);
  };
  auto read_v = [&](s16x4 (&vf)[NB], const __bf16* __restrict__ vb, int d) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NB; ++i)
      vf[i] = read_turned(vb + (at + 16u * i + vrow) * DP + ((2u * d + ((lr & 3u) >> 1)) ^ vt) * 8u + (lr & 1u) * 4u);
  };
  auto mul_v = [&](const s16x4 (&pb)[NB][RB], const s16x4 (&vf)[NB], int d) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NB; i += 2)
#pragma unroll
      for (int j = 0; j < RB; ++j) {
        if constexpr (NB > 1) {
          const s16x8 v8 = __builtin_shufflevector(vf[i], vf[i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
          const s16x8 p8 = __builtin_shufflevector(pb[i][j], pb[i + 1][j], 0, 1, 2, 3, 4, 5, 6, 7);
          acc[d][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v8), __builtin_bit_cast(bf16x8, p8), acc[d][j], 0, 0, 0);
        } else {
          acc[d][j] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(vf[0], pb[0][j], acc[d][j], 0, 0, 0);
        }
      }
  };
  // The exponentials of block i of the positions.
  auto weigh = [&](const f32x4 (&s)[NB][RB], s16x4 (&pb)[NB][RB], int i) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < RB; ++j) {
      const float base = mc[j] == -INFINITY ? 0.0f : mc[j];
      bf16x4 h;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = exp2_(__builtin_fmaf(s[i][j][e], A.c, -base));
        sum[j] += p;
        h[e] = (__bf16)p;
      }
      pb[i][j] = __builtin_bit_cast(s16x4, h);
    }
  };
  auto refer = [&](f32x4 (&s)[NB][RB], uint32_t p0) __attribute__((always_inline)) {
    const uint32_t first = p0 + at + 4u * lg;
    if (p0 + at + 16u * NB > least) {   // uniform: some query sees not all of these
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < RB; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (first + 16u * i + e >= lim[j]) s[i][j][e] = -INFINITY;
    }
    // The reference follows the maximum only where that is 2^8 above it, which
    // the first tiles settle: no exchange between lanes and no rescaling otherwise.
    float top[RB];
    bool grow = false;
#pragma unroll
    for (int j = 0; j < RB; ++j) {
      float t = -INFINITY;
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) t = fmaxf(t, s[i][j][e]);
      top[j] = t;
      grow |= t * A.c > mc[j] + 8.0f;
    }
    if (__builtin_amdgcn_ballot_w64(grow)) {
#pragma unroll
      for (int j = 0; j < RB; ++j) {
        const float m = fmaxf(mc[j], max4(top[j]) * A.c);
        const float f = m == mc[j] ? 1.0f : share_of(mc[j], m);
        mc[j] = m;
        sum[j] *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d][j] *= f;
      }
    }
  };
  // Values that some queries do not see: those past the end become 0, and those
  // that are no numbers too (their weight of 0 would not be 0 times them); the
  // queries that do see these get them at the end.
  auto clean = [&](__bf16* vb, uint32_t p0) {
    const uint32_t have = min(ATT_TILE, J.b - p0);
    const bool look = !J.pre && A.T > 1u;
    for (uint32_t i = (look ? 0u : have * PR) + threadIdx.x; i < ATT_TILE * PR; i += NW * 64) {
      s16x8* const to = reinterpret_cast<s16x8*>(vb) + i;
      s16x8 v = {};
      if (i < have * PR) {
        if (((i % PR) ^ turn_v(i / PR)) * 8u >= A.D) continue;   // (never loaded)
        v = *to;
        bool any = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool bad = (v[e] & 0x7f80) == 0x7f80;
          any |= bad;
          v[e] = bad ? 0 : v[e];
        }
        if (!any) continue;
        *odd = 1u;
      }
      *to = v;
    }
    att_barrier<0>();
  };

  uint32_t cur = 0u, nxt = S - 1u;
  for (uint32_t t = 0; t < nt; ++t) {
    const uint32_t after = nt - 1u - t;   // tiles still in flight, at most S - 2
    if (S > 3 && after >= 2u) att_barrier<4 * LD>();
    else if (S > 2 && after >= 1u) att_barrier<2 * LD>();
    else att_barrier<0>();
    const uint32_t p0 = J.a + t * ATT_TILE;
    if (t + (uint32_t)S - 1u < nt) {
      fetch(t + S - 1u, J.k, Ks + nxt * TE, true);
      fetch(t + S - 1u, J.v, Vs + nxt * TE, false);
    }
    if (p0 + ATT_TILE > least) clean(Vs + cur * TE, p0);
    const __bf16* __restrict__ const kb = Ks + cur * TE;
    const __bf16* __restrict__ const vb = Vs + cur * TE;
    f32x4 s[NB][RB];
    s16x4 pb[NB][RB];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      bf16x8 kf[NB];
      read_k(kf, kb, ks);
      mul_k(s, kf, ks);
    }
    refer(s, p0);
#pragma unroll
    for (int i = 0; i < NB; ++i) weigh(s, pb, i);
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      s16x4 vf[NB];
      read_v(vf, vb, d);
      mul_v(pb, vf, d);
    }
    cur = cur + 1u == (uint32_t)S ? 0u : cur + 1u;
    nxt = nxt + 1u == (uint32_t)S ? 0u : nxt + 1u;
  }
#pragma unroll
  for (int j = 0; j < RB; ++j) sum[j] = sum4(sum[j]);

  auto put = [&](uint32_t id, int d, f32x4 v) { *reinterpret_cast<f32x4*>(A.part + ((uint64_t)J.slot * A.NQ + id) * DP + 16u * d + 4u * lg) = v; };
  auto tell = [&](uint32_t id, float m, float x) {
    if (lg == 0u) A.stat[(uint64_t)J.slot * A.NQ + id] = make_float2(m, x);
  };
  if constexpr (WP > 1) {
    // Waves that took different positions of the same queries meet in LDS; each
    // joins some of the elements.
    static_assert(NW * 16 * RB * DP * 4 <= 2 * S * (int)TE * 2, "the waves' sums fit (Ks and Vs are one array)");
    f32x4* const room = reinterpret_cast<f32x4*>(Ks);
    att_barrier<0>();
#pragma unroll
    for (int j = 0; j < RB; ++j) {
      if (lg == 0u) stats[(w * RB + j) * 16u + lr] = make_float2(mc[j], sum[j]);
#pragma unroll
      for (int d = 0; d < DB; ++d) room[((w * RB + j) * DB + d) * 64u + l] = acc[d][j];
    }
    att_barrier<0>();
#pragma unroll
    for (int j = 0; j < RB; ++j) {
      const uint32_t id = table[(wq * RB + j) * 16u + lr].id;
      float2 st[WP];
      float m = -INFINITY, total = 0.0f;
#pragma unroll
      for (int x = 0; x < WP; ++x) {
        st[x] = stats[((x * WQ + wq) * RB + j) * 16u + lr];
        m = fmaxf(m, st[x].x);
      }
#pragma unroll
      for (int x = 0; x < WP; ++x) {
        const float f = st[x].x == m ? 1.0f : share_of(st[x].x, m);
        total += st[x].y * f;   // (a sum that is NaN stays)
        st[x].x = f;
      }
#pragma unroll
      for (int y = 0; y < DB / WP; ++y) {
        const uint32_t d = wp * (DB / WP) + y;
        f32x4 v = {};
#pragma unroll
        for (int x = 0; x < WP; ++x) v += room[(((x * WQ + wq) * RB + j) * DB + d) * 64u + l] * st[x].x;
        if (id != ~0u) put(id, d, v);
      }
      if (wp == 0u && id != ~0u) tell(id, m, total);
    }
  } else {
#pragma unroll
    for (int j = 0; j < RB; ++j) {
      const uint32_t id = table[(wq * RB + j) * 16u + lr].id;
      if (id == ~0u) continue;
      tell(id, mc[j], sum[j]);
#pragma unroll
      for (int d = 0; d < DB; ++d) put(id, d, acc[d][j]);
    }
  }
  if (!J.pre && A.T > 1u) {
    __syncthreads();
    if (*odd) {
      // Rare: values that are no numbers, times their weights, added where they are
      // seen.  A wave a query: the position's score once more, its weight rounded
      // as `weigh` does.
      constexpr int EL = (DP + 63) / 64;   // elements a lane
      // (the kernel's first argument, read once more: held for this, it cost the loop scalar registers, one short request
      // 8.65 -> 8.83 us)
      const __attribute__((address_space(4))) AttArgs* B = (const __attribute__((address_space(4))) AttArgs*)__builtin_amdgcn_kernarg_segment_ptr();
      __asm__("" : "+s"(B));
      const uint32_t D = B->D, NQ = B->NQ, flip = B->flip;
      const float c = B->c;
      const __bf16* const q = B->q;
      float* const part = B->part;
      const float2* const stat = B->stat;
#pragma unroll 1
      for (uint32_t x = w; x < 16u * RB * WQ; x += NW) {
        const AttEntry e = table[x];
        if (e.id == ~0u) continue;
        const uint64_t entry = (uint64_t)J.slot * NQ + e.id;
        const float ref = stat[entry].x, base = ref == -INFINITY ? 0.0f : ref;
        float add[EL] = {};
#pragma unroll 1
        for (uint32_t p = max(J.a, least & ~(ATT_TILE - 1u)); p < e.lim; ++p) {
          const __bf16* const v = J.v + p * J.stride;
          bool bad = false;
          for (uint32_t d = l; d < D; d += 64u) bad |= !(fabsf((float)v[d]) < INFINITY);
          if (!__builtin_amdgcn_ballot_w64(bad)) continue;
          float s = 0.0f;
          for (uint32_t d = l; d < D; d += 64u) s = __builtin_fmaf((float)q[e.at + d], (float)J.k[p * J.stride + d], s);
          s = wave_sum_f32(s);
          const float weight = (float)(__bf16)exp2_(__builtin_fmaf(flip ? -s : s, c, -base));
#pragma unroll
          for (int y = 0; y < EL; ++y) {
            const float value = 64u * y + l < D ? (float)v[64u * y + l] : 0.0f;
            if (!(fabsf(value) < INFINITY)) add[y] += weight * value;
          }
        }
#pragma unroll
        for (int y = 0; y < EL; ++y)
          if (add[y] != 0.0f) part[entry * DP + 64u * y + l] += add[y];   // (inf or NaN where it is not 0: within dim)
      }
    }
  }
}

template <int DP, int RB, int WQ, int WP, bool SMALL, int S>
__global__ __launch_bounds__(WQ * WP * 64, 2) void attention_tile_kernel(AttArgs A) {
  __shared__ __align__(1024) __bf16 tiles[2][S * ATT_TILE * DP];
  __shared__ float2 stats[WQ * WP * RB * 16];
  __shared__ AttEntry table[16 * RB * WQ < 32 ? 32 : 16 * RB * WQ];
  __shared__ uint32_t odd;
  // XCD x (workgroups go to the XCDs in turn) takes a contiguous range of the
  // prefixes' jobs, then one of the suffixes'.
  const uint32_t xcd = blockIdx.x & 7u, at = blockIdx.x >> 3, pp = (A.np + 7u) / 8u, ps = (A.ns + 7u) / 8u;
  AttJob J;
  J.pre = at < pp;
  const uint32_t job = J.pre ? xcd * pp + at : xcd * ps + at - pp;
  if (job >= (J.pre ? A.np : A.ns)) return;
  if (J.pre) {   // blocks of queries together: they read the same positions
    uint32_t i = job;
    const uint32_t blk = i % A.nrb;
    i /= A.nrb;
    J.slot = i % A.sp;
    i /= A.sp;
    J.kv = i % A.KV;
    J.g = i / A.KV;
    J.m0 = blk * (16u * RB * WQ);
    J.m = A.wb * A.nt * A.per;
    const uint32_t g = A.g0 + J.g, len = att_len(A.plen, g, A.P);
    const uint64_t from = g * A.pg + J.kv * A.ph;
    J.k = A.pk + from, J.v = A.pv + from, J.stride = A.pp;
    const uint32_t tiles_all = (len + ATT_TILE - 1u) / ATT_TILE, each = (tiles_all + A.sp - 1u) / A.sp * ATT_TILE;
    J.a = min(len, J.slot * each), J.b = min(len, J.a + each);
    J.row = 0u, J.len = 0u;
    attention_job<DP, RB, WQ, WP, S>(A, J, tiles[0], tiles[1], stats, table, &odd);
    return;
  }
  uint32_t i = job;
  const uint32_t blk = i % A.nsb;
  i /= A.nsb;
  const uint32_t part = i % A.ss;
  i /= A.ss;
  J.kv = i % A.KV;
  const uint32_t row = i / A.KV;
  J.g = row / A.wb, J.row = row - J.g * A.wb;
  J.slot = A.sp + part;
  J.m0 = blk * (SMALL ? 16u : 16u * RB * WQ);   // (one block, where it is small)
  J.m = A.nt * A.per;
  const uint32_t r = att_row(A, row);
  J.len = att_len(A.len, r, A.N);
  const uint64_t from = r * A.kr + J.kv * A.kh;
  J.k = A.k + from, J.v = A.v + from, J.stride = A.kp;
  const uint32_t end = min(J.len, att_seen(J.len, A.T, A.t0 + A.nt - 1u));   // of the last token here
  const uint32_t tiles_all = (end + ATT_TILE - 1u) / ATT_TILE, each = (tiles_all + A.ss - 1u) / A.ss * ATT_TILE;
  J.a = min(end, part * each), J.b = min(end, J.a + each);
  if constexpr (SMALL) attention_job<DP, 1, WQ * WP / 4, 4, S>(A, J, tiles[0], tiles[1], stats, table, &odd);
  else attention_job<DP, RB, WQ, WP, S>(A, J, tiles[0], tiles[1], stats, table, &odd);
}

// Joins a query's parts: NWV waves a query, each lane four elements of every
// 256 NWV / DP-th part.  Four waves from 17 parts on (128 queries of 64 parts: 4.8 us,
// where one lane an element, part after part, took 56).
template <int DP, int NWV>
__device__ __forceinline__ void attention_join(const AttArgs& A, const uint8_t* counted, uint32_t block, f32x4 (&meet)[4][DP / 4]) {
  constexpr uint32_t LQ = DP / 4, GR = NWV * 64 / LQ;
  const uint32_t w = threadIdx.x >> 6, l = threadIdx.x & 63u;
  const uint32_t id = min(block * (4u / NWV) + w / NWV, A.NQ - 1u);   // (a last workgroup's other waves: the last query once more)
  const uint32_t in = w % NWV * 64u + l, d = in % LQ * 4u, grp = in / LQ;
  // The first parts are on their way while the references are compared.
  constexpr uint32_t AHEAD = 4;
  f32x4 v[AHEAD] = {};
  float at[AHEAD] = {};
  float2 mine = make_float2(-INFINITY, 0.0f);
  if (A.slots) {
    if (l < A.slots) mine = A.stat[(uint64_t)l * A.NQ + id];
#pragma unroll
    for (uint32_t u = 0; u < AHEAD; ++u) {
      const uint64_t s = (uint64_t)min(grp + u * GR, A.slots - 1u) * A.NQ + id;
      v[u] = *reinterpret_cast<const f32x4*>(A.part + s * DP + d);
      at[u] = A.stat[s].x;
    }
  }
  // every wave by itself: the parts' common reference and the whole sum
  float m = mine.x;
  for (uint32_t s = l + 64u; s < A.slots; s += 64u) m = fmaxf(m, A.stat[(uint64_t)s * A.NQ + id].x);
  m = wave_max_f32(m);
  float sum = mine.y * (mine.x == m ? 1.0f : share_of(mine.x, m));   // (a sum that is NaN stays)
  for (uint32_t s = l + 64u; s < A.slots; s += 64u) {
    const float2 x = A.stat[(uint64_t)s * A.NQ + id];
    sum += x.y * (x.x == m ? 1.0f : share_of(x.x, m));
  }
  sum = wave_sum_f32(sum);
  f32x4 o = {};
#pragma unroll
  for (uint32_t u = 0; u < AHEAD; ++u)
    if (grp + u * GR < A.slots) o += v[u] * (at[u] == m ? 1.0f : share_of(at[u], m));
#pragma unroll 4
  for (uint32_t s = grp + AHEAD * GR; s < A.slots; s += GR) {
    const float x = A.stat[(uint64_t)s * A.NQ + id].x;
    o += *reinterpret_cast<const f32x4*>(A.part + ((uint64_t)s * A.NQ + id) * DP + d) * (x == m ? 1.0f : share_of(x, m));
  }
#pragma unroll
  for (uint32_t x = LQ; x < 64u; x <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], x);
  if constexpr (NWV > 1) {
    if (l < LQ) meet[w][l] = o;
    __syncthreads();
    if (w % NWV) return;
#pragma unroll
    for (uint32_t x = 1; x < (uint32_t)NWV; ++x) o += meet[w + x][l % LQ];
  }
  if (l >= LQ) return;
  const uint32_t h = id % A.H, t = A.t0 + id / A.H % A.nt, r = att_row(A, id / A.H / A.nt);
  if (l == 0u) {
    const float ref = m + __log2f(sum);
    if (A.ref) {
      bool none = sum == 0.0f;
      if (counted) none |= counted[r] == 0;
      A.ref[id] = none ? INFINITY : ref;
    }
    if (A.lse) A.lse[((uint64_t)r * A.T + t) * A.H + h] = sum == 0.0f ? -INFINITY : ref * 0.693147181f;
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  if (d < A.D) {
    bf16x4 to;
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = (__bf16)(o[e] * inv);
    *reinterpret_cast<bf16x4*>(A.out + (uint64_t)r * A.orow + t * A.ot + h * A.oh + d) = to;
  }
}

// The sum over 16 lanes of a row, in each of them.
template <int N>
__device__ __forceinline__ float plus_turned(float v) {
  return v + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float row_sum(float v) { return plus_turned<1>(plus_turned<2>(plus_turned<4>(plus_turned<8>(v)))); }

struct AttWeights {
  uint32_t cp, cs;        // chunks of a prefix and of a suffix, 0 where it has no weights
  uint32_t tiles;         // 32 positions each, of a chunk
  uint64_t jobs_p, jobs;  // chunks of all prefixes, of all
};

// The weights of a chunk of positions of a cache head, by one wave: the scores
// once more, 16 MB queries held in registers, the next positions' keys on
// their way.  No two waves write one entry and the sums' order is fixed.  8 groups of 4
// sequences, up to 4096 positions of 8 heads of 128: 17 us (62 MB read); a wave for
// each 32 positions, which found its queries anew, took 26.
template <int DP, int MB, bool SOME>
__device__ __forceinline__ void attention_weights(const AttArgs& A, const AttWeights& G, uint64_t job) {
  constexpr int KS = DP / 32;
  const uint32_t l = threadIdx.x & 63u, lr = l & 15u, lg = l >> 4;
  AttJob J;
  J.pre = job < G.jobs_p;
  uint64_t i = J.pre ? job : job - G.jobs_p;
  const uint32_t chunks = J.pre ? G.cp : G.cs, chunk = (uint32_t)(i % chunks);
  i /= chunks;
  J.kv = (uint32_t)(i % A.KV);
  const uint32_t seg = (uint32_t)(i / A.KV);   // group, or row, within the launch
  J.g = J.pre ? seg : seg / A.wb;
  J.row = J.pre ? 0u : seg - J.g * A.wb;
  const uint32_t r = J.pre ? A.g0 + seg : att_row(A, seg);
  const uint32_t len = J.pre ? att_len(A.plen, r, A.P) : att_len(A.len, r, A.N);
  const uint32_t from = min(len, chunk * G.tiles * 32u), to = min(len, from + G.tiles * 32u);
  if (from >= to) return;
  const uint64_t stride = J.pre ? A.pp : A.kp;
  const __bf16* const kb = J.pre ? A.pk + r * A.pg + J.kv * A.ph : A.k + r * A.kr + J.kv * A.kh;
  float* const out = J.pre ? A.pw + ((uint64_t)r * A.KV + J.kv) * A.P : A.w + ((uint64_t)r * A.KV + J.kv) * A.N;
  const uint32_t mine = 16u * (lr >> 2 & 1u) + 4u * lg + (lr & 3u);   // the position that this lane writes (lr < 8)
  auto load = [&](bf16x8 (&k)[2][KS], uint32_t p0) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const __bf16* const at = kb + (uint64_t)min(p0 + 16u * b + lr, len - 1u) * stride;
#pragma unroll
      for (int s = 0; s < KS; ++s) k[b][s] = *reinterpret_cast<const bf16x8*>(at + min(32u * s + 8u * lg, A.D - 8u));
    }
  };
  const uint32_t M = (J.pre ? A.wb : 1u) * A.nt * A.per;
  for (uint32_t m0 = 0; m0 < M; m0 += 16u * MB) {
    bf16x8 q[MB][KS];
    float ref[MB];
    uint32_t lim[MB];   // positions below it are seen
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      const uint32_t m = m0 + 16u * j + lr;
      const AttQuery x = att_query(A, J, min(m, M - 1u));
      const __bf16* const at = A.q + att_elements(A, J, x);
#pragma unroll
      for (int s = 0; s < KS; ++s) q[j][s] = *reinterpret_cast<const bf16x8*>(at + min(32u * s + 8u * lg, A.D - 8u));
      ref[j] = A.ref[att_id(A, J, x)];
      lim[j] = m >= M ? 0u : J.pre ? len : min(len, att_seen(len, A.T, x.t));
    }
    // (elements past dim: zero in the queries and, lest they be no numbers, in the keys)
#pragma unroll
    for (int j = 0; j < MB; ++j)
#pragma unroll
      for (int s = 0; s < KS; ++s) q[j][s] = 32u * s + 8u * lg < A.D ? flipped(q[j][s], A.flip) : bf16x8{};
    bf16x8 next[2][KS];
    load(next, from);
    if constexpr (SOME) {   // a row that does not count: no weights, of scores that are no numbers neither
#pragma unroll
      for (int j = 0; j < MB; ++j) lim[j] = ref[j] == INFINITY ? 0u : lim[j];
    }
    for (uint32_t p0 = from; p0 < to; p0 += 32u) {
      bf16x8 k[2][KS];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int s = 0; s < KS; ++s) k[b][s] = 32u * s + 8u * lg < A.D ? next[b][s] : bf16x8{};
      const bool write = lr < 8u && p0 + mine < to;
      const float old = write ? out[p0 + mine] : 0.0f;
      if (p0 + 32u < to) load(next, p0 + 32u);
      f32x4 add[2] = {};
#pragma unroll
      for (int j = 0; j < MB; ++j) {
        f32x4 x[2] = {};
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int b = 0; b < 2; ++b) x[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[b][s], q[j][s], x[b], 0, 0, 0);
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = exp2_(__builtin_fmaf(x[b][e], A.c, -ref[j]));
            if (p0 + 16u * b + 4u * lg + e < lim[j]) add[b][e] += p;
          }
      }
      float v = 0.0f;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float all = row_sum(add[b][e]);
          if (lr == 4u * b + e) v = all;
        }
      if (write) out[p0 + mine] = old + v;
    }
  }
}

template <int DP, int NWV>
__global__ __launch_bounds__(256) void attention_join_kernel(AttArgs A, const uint8_t* counted) {   // (rows whose queries add to the weights; NULL: all)
  __shared__ f32x4 meet[4][DP / 4];
  attention_join<DP, NWV>(A, counted, blockIdx.x, meet);
}

template <int DP, int MB, bool SOME>
__global__ __launch_bounds__(256) void attention_weights_kernel(AttArgs A, AttWeights G) {
  for (uint64_t job = (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6); job < G.jobs; job += (uint64_t)gridDim.x * 4u)
    attention_weights<DP, MB, SOME>(A, G, job);
}

size_t attention_scratch_bytes() { return ATT_SCRATCH; }

template <int DP, int RB, int WQ, int WP, int S>
static void att_go(hipStream_t st, const AttArgs& A, bool small) {
  const dim3 grid(((A.np + 7u) / 8u + (A.ns + 7u) / 8u) * 8u), block(WQ * WP * 64);
  // (16 queries a workgroup: all that share a prefix, so that a suffix has no more)
  if (RB * WQ == 1 || small) hipLaunchKernelGGL((attention_tile_kernel<DP, RB, WQ, WP, true, S>), grid, block, 0, st, A);
  else if constexpr (RB * WQ > 1) hipLaunchKernelGGL((attention_tile_kernel<DP, RB, WQ, WP, false, S>), grid, block, 0, st, A);
}

template <int DP>
static void attention_launch(hipStream_t st, const AttArgs& A, const uint8_t* counted, const AttPlan& p) {
  constexpr int S = DP == 64 ? 4 : 2;   // tiles in LDS: 64 KB, or 128 where dim is above 128
  if (A.np + A.ns) {
    if constexpr (DP == 256) {
      if (p.wq == 1u) att_go<DP, 1, 1, 4, S>(st, A, p.small);
      else if (p.wq == 2u) att_go<DP, 1, 2, 2, S>(st, A, p.small);
      else if (p.wq == 4u) att_go<DP, 1, 4, 1, S>(st, A, p.small);
      else att_go<DP, 1, 8, 1, S>(st, A, p.small);
    } else {
      if (p.rb == 1u) att_go<DP, 1, 1, 4, S>(st, A, p.small);
      else if (p.wq == 1u) att_go<DP, 2, 1, 4, S>(st, A, p.small);
      else if (p.wq == 2u) att_go<DP, 2, 2, 2, S>(st, A, p.small);
      else att_go<DP, 2, 4, 1, S>(st, A, p.small);
    }
  }
  if (A.slots > 16u) hipLaunchKernelGGL((attention_join_kernel<DP, 4>), dim3(A.NQ), dim3(256), 0, st, A, counted);
  else hipLaunchKernelGGL((attention_join_kernel<DP, 1>), dim3((A.NQ + 3u) / 4u), dim3(256), 0, st, A, counted);
  if (!A.pw && !A.w) return;
  AttWeights G;
  const uint64_t tp = A.pw ? att_ceil(A.P, 32u) : 0u, ts = A.w ? att_ceil(A.N, 32u) : 0u;
  const uint64_t segs_p = (uint64_t)A.ng * A.KV, segs_s = segs_p * A.wb;
  // so many tiles a wave that the waves fill the chip about once
  const uint64_t each = (segs_p * tp + segs_s * ts) / 2048u;
  G.tiles = each < 1u ? 1u : each > 64u ? 64u : (uint32_t)each;
  G.cp = att_ceil(tp, G.tiles), G.cs = att_ceil(ts, G.tiles);
  G.jobs_p = segs_p * G.cp, G.jobs = G.jobs_p + segs_s * G.cs;
  const uint64_t blocks = (G.jobs + 3u) / 4u;
  const dim3 grid((uint32_t)(blocks < 1u << 20 ? blocks : 1u << 20));
  const uint32_t m = (A.pw ? A.wb : 1u) * A.nt * A.per;
  constexpr int MB = DP == 256 ? 2 : 4;
  // (its own kernels where not all rows count: the test costs the others 0.35 of 27.3 us)
  if (counted) {
    if (m <= 16u) hipLaunchKernelGGL((attention_weights_kernel<DP, 1, true>), grid, dim3(256), 0, st, A, G);
    else hipLaunchKernelGGL((attention_weights_kernel<DP, MB, true>), grid, dim3(256), 0, st, A, G);
  } else {
    if (m <= 16u) hipLaunchKernelGGL((attention_weights_kernel<DP, 1, false>), grid, dim3(256), 0, st, A, G);
    else hipLaunchKernelGGL((attention_weights_kernel<DP, MB, false>), grid, dim3(256), 0, st, A, G);
  }
}

}  // namespace mxs

extern "C" int mxs_prefix_attention(mxs_ctx* ctx, const mxs_attention* attention) {
  return mxs_prefix_attention_counted(ctx, attention, nullptr);
}

extern "C" int mxs_prefix_attention_counted(mxs_ctx* ctx, const mxs_attention* attention, const uint8_t* counted) {
  using namespace mxs;
  if (!ctx) return MXS_EINVAL;
  if (const char* m = attention_check(attention, counted)) return fail(ctx, MXS_EINVAL, m);
  const mxs_attention& a = *attention;
  if (a.groups == 0 || a.beams == 0 || a.tokens == 0) return MXS_OK;
  AttArgs A{};
  A.q = reinterpret_cast<const __bf16*>(a.q);
  A.pk = reinterpret_cast<const __bf16*>(a.prefix_keys);
  A.pv = reinterpret_cast<const __bf16*>(a.prefix_values);
  A.k = reinterpret_cast<const __bf16*>(a.keys);
  A.v = reinterpret_cast<const __bf16*>(a.values);
  A.out = reinterpret_cast<__bf16*>(a.out);
  A.qr = a.q_row, A.qt = a.q_token, A.qh = a.q_head;
  A.pg = a.prefix_group, A.ph = a.prefix_head, A.pp = a.prefix_position;
  A.kr = a.row, A.kh = a.head, A.kp = a.position;
  A.orow = a.out_row, A.ot = a.out_token, A.oh = a.out_head;
  A.plen = a.prefix_lengths, A.len = a.lengths;
  A.lse = a.lse, A.pw = a.prefix_weight, A.w = a.weight;
  A.W = a.beams, A.T = a.tokens, A.H = a.heads, A.KV = a.kv_heads, A.D = a.dim, A.P = a.prefix, A.N = a.suffix;
  A.per = a.heads / a.kv_heads;
  // scale log2(e); 0 becomes the least number above it (at most 5e-7 in a score), since
  // -inf times 0 is no number
  const float c = fabsf(a.scale) * 1.44269504f;
  A.c = c > 0.0f ? c : 1.4013e-45f;
  A.flip = a.scale < 0.0f ? 0x8000u : 0u;
  const AttPlan p = attention_plan(a.groups, a.beams, a.tokens, a.heads, a.kv_heads, a.dim, a.prefix, a.suffix);
  A.sp = p.sp, A.ss = p.ss, A.slots = p.slots;
  int prev = 0;
  (void)hipGetDevice(&prev);
  if (prev != ctx->device) (void)hipSetDevice(ctx->device);
  hipError_t e = hipSuccess;
  for (uint32_t g = 0; g < a.groups && e == hipSuccess; g += p.ng)
    for (uint32_t b = 0; b < a.beams && e == hipSuccess; b += p.wb)
      for (uint32_t t = 0; t < a.tokens && e == hipSuccess; t += p.nt) {
        A.g0 = g, A.ng = a.groups - g < p.ng ? a.groups - g : p.ng;
        A.b0 = b, A.wb = a.beams - b < p.wb ? a.beams - b : p.wb;
        A.t0 = t, A.nt = a.tokens - t < p.nt ? a.tokens - t : p.nt;
        A.NQ = A.ng * A.wb * A.nt * A.H;
        const uint32_t rows = 16u * p.rb * p.wq, ms = A.nt * A.per;
        A.nrb = att_ceil((uint64_t)A.wb * ms, rows), A.nsb = p.small ? 1u : att_ceil(ms, rows);
        A.np = A.ng * A.KV * A.nrb * A.sp;
        A.ns = A.ng * A.wb * A.KV * A.nsb * A.ss;
        A.stat = reinterpret_cast<float2*>(ctx->attention_scratch);
        A.ref = A.pw || A.w ? ctx->attention_scratch + 2ull * A.slots * A.NQ : nullptr;
        A.part = ctx->attention_scratch + ((2ull * A.slots + 1u) * A.NQ + 3u) / 4u * 4u;
        if (p.dp == 64u) attention_launch<64>(ctx->stream, A, counted, p);
        else if (p.dp == 128u) attention_launch<128>(ctx->stream, A, counted, p);
        else attention_launch<256>(ctx->stream, A, counted, p);
        e = hipGetLastError();
      }
  if (prev != ctx->device) (void)hipSetDevice(prev);
  if (e != hipSuccess) return hip_fail(ctx, e, "attention launch");
  return MXS_OK;
}
