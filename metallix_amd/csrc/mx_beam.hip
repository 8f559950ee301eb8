// mx_beam.hip -- beam search: the selection of each group's n best
// continuations over its beams and the vocabulary (mxs_beam_select), and the
// move of the beams' states to their children (mxs_beam_reorder).
//
// The selection.  A live beam b with cumulative score s_b and logits l has
// the candidates (b, v) of score s_b + (l_v - N_b), N_b = ln sum_u exp(l_u); an
// ended beam is one candidate of its own score.  A group keeps the n largest
// by score times the beam's scale.  One launch:
//
// - A row is split into C chunks of T tiles of 4096 tokens, one 256-thread
//   workgroup each (rows that are not live exit).  It streams its chunk once.
//   The weights are summed in f64, relative to a power of two near the first
//   maximum met: with f64's exponent range that unit needs no running maximum
//   (it moves for one 600 nats above).  A weight takes 15 vector instructions
//   (beam_weight), as many as an f32 exponential with a corrected argument
//   and its guards, at 2^-39 instead of 2^-22: beams are ordered by sums of
//   such logarithms over hundreds of steps.
// - Candidates: each thread keeps its largest logit of every tile in LDS.
//   After the chunk (or 8 tiles) a threshold that n of the chunk's threads
//   have reached comes from the threads' maxima (of the waves that have
//   enough of them, where a mask or the row's end leaves some without: 24.7 to
//   22.8 us at 7 x 5 x 151936 bf16 under masks), and only the (thread, tile)
//   pairs that reach it (about n to 1.4 n) look at their 16 logits again, from
//   L2 or the Infinity Cache; a NaN or +inf reaches it too and is found there.
//   Scanning every tile against a running threshold instead took 101 us where
//   this takes 76 (16 x 16 x 262144, n 32).  Near-ties that overflow a wave's
//   256 slots are cut to its n largest, any number of times.
// - The group's last workgroup (arrival counter) merges: the rows' N from
//   their chunks' (unit, sum) in chunk order; a rank that n candidates reach,
//   the best chunk threshold or the n-th largest chunk maximum; the entries
//   at or above it, from the chunks whose maximum is; their order by counting
//   on 32-bit keys.  While more than 2 n + 64 pass, the n-th largest of those
//   kept is a closer threshold (8 x 32 x 151936, n 64, groups at their first
//   step: 475 -> 70 us); more than 1024 equal ranks are taken one by one.
//
// Bound.  16 x 16 x 262144 f32 (221 MB of live rows), n 32: 73 us, 45 at the
// 4.92 TB/s of a large copy; vector instructions (40% of the issue slots over
// the launch) and the tail of the last groups' merges (9 us) keep it off the
// stream.  253 MB are read, 30 of them second looks.  Small calls are a chain
// of latencies: 1 x 4 x 50257, n 8, takes 12.3 us: 3.4 to load and sum, 1.2
// to publish, 1.8 to arrive, 5.4 to merge (statistics 1.1, norms 0.9,
// threshold 1.5, entries 1.0, order and output 0.9).  Also measured, in the first
// shape: 1024 workgroups 83 us and 4096 97 (2048: 76); five workgroups on a
// CU 83 (spills); loads two tiles ahead 78; a polynomial of degree 7 the same.
//
// The move is a copy: reorder_kernel reads each surviving row and writes each
// changed row once, at 4.7 to 5.3 TB/s of both from 64 MB on.

#include <hip/hip_runtime.h>

#include <float.h>
#include <math.h>
#include <stdint.h>

#include <string>
#include <type_traits>

#include "../../include/mx_sampler.h"
#include "mxs_checks.h"
#include "mxs_ctx.h"
#include "mxs_device.h"
#include "mxs_math.h"

namespace mxs {

constexpr int BNT = 256;                  // threads per workgroup
constexpr int BNW = BNT / 64;             // waves
constexpr int BQ = 4;                     // quads per thread and tile
constexpr uint32_t BSL = BNT * 4;         // tokens per slice (one quad per thread)
constexpr uint32_t BTILE = BSL * BQ;      // tokens per tile (4096)
constexpr uint32_t BBT = 8;               // tiles between two looks for candidates
constexpr uint32_t BCAP = 256;            // candidate slots per wave
constexpr uint32_t BLIST = 512;           // entries a chunk publishes at most
constexpr uint32_t BDENSE = 1024;         // entries a group's finisher ranks by counting
constexpr uint32_t BWGS = 2048;           // chunks a call aims at
constexpr uint32_t BGCH = 512;            // chunks per group at most (or one per beam)
static_assert(BLIST >= BNW * MXS_BEAM_N_MAX && BCAP >= MXS_BEAM_N_MAX + 64, "a compacted list fits");

struct BeamStat {
  double ref, sum;      // the chunk's weights: sum of exp(l - ref); ref -inf: no weight
  uint32_t thr;         // order key that n of the chunk's candidates reach (0: fewer than n)
  uint32_t top;         // order key of its largest candidate (0: none)
  uint32_t count;       // entries listed
  uint32_t bad;         // a NaN or +inf among the logits that count
};

struct BeamArgs {
  const void* logits;
  uint64_t stride;
  uint32_t G, W, V, n;
  uint32_t C, T;                          // chunks per row, tiles per chunk
  const double* score;
  const uint8_t* ended;
  const double* scale;
  const uint32_t* mask;
  uint64_t mask_stride;
  uint32_t tok_vocab;
  int32_t end_token;
  int32_t* token;
  int32_t* beam;
  double* oscore;
  uint8_t* oended;
  int32_t* status;
  BeamStat* stat;                         // [G * W * C]
  unsigned long long* list;               // [G * W * C * BLIST]: (order key << 32) | ~token
  uint32_t* ctr;                          // [G * CTR_STRIDE]
};

// What the sum and the candidates are taken over.
enum { BEAM_ALL = 0, BEAM_MASK = 1, BEAM_MASK_NORM = 2 };   // no mask; candidates masked; both masked

__device__ __forceinline__ unsigned long long beam_entry(uint32_t key, uint32_t token) {
  return ((unsigned long long)key << 32) | (unsigned long long)(~token);
}
// The legal ones of the four tokens from e0, from their mask word.
__device__ __forceinline__ uint32_t beam_nibble(uint32_t word, uint32_t e0, uint32_t vm) {
  const uint32_t have = vm > e0 ? vm - e0 : 0u;
  const uint32_t nib = (word >> (e0 & 31u)) & 15u;
  return have < 4u ? nib & ((1u << have) - 1u) : nib;
}
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// 2^(n - n0) e^r for x = n ln 2 + r, |r| <= ln 2 / 2, in f64: `magic` is 1.5
// 2^52 - n0, so the low word of fma(x, log2 e, magic) is n - n0.  e^r by the
// polynomial of degree 8 through its values at the Chebyshev nodes (relative
// error below 2^-39.7).  For |x| <= 2400 the reduction adds 2^-44.
__device__ __forceinline__ double beam_weight(float xf, double magic) {
  const double x = (double)xf;
  const double t = __builtin_fma(x, 1.4426950408889634, magic);
  const double r = __builtin_fma(magic - t, 0.6931471805599453, x);
  double p = 0x1.a15a4f98eb4cep-16;
  p = __builtin_fma(p, r, 0x1.a1aa7f143c63cp-13);
  p = __builtin_fma(p, r, 0x1.6c164df443c8cp-10);
  p = __builtin_fma(p, r, 0x1.111080ae06089p-7);
  p = __builtin_fma(p, r, 0x1.5555557428d91p-5);
  p = __builtin_fma(p, r, 0x1.555555a26dedbp-3);
  p = __builtin_fma(p, r, 0x1.fffffffff71cfp-2);
  p = __builtin_fma(p, r, 0x1.ffffffffd38c1p-1);
  p = __builtin_fma(p, r, 1.0);
  return __builtin_ldexp(p, (int)(uint32_t)__builtin_bit_cast(unsigned long long, t));
}

struct alignas(16) BeamCand {
  double rank;              // score * scale
  unsigned long long tie;   // place among equal ranks (beam_tie)
};

struct alignas(16) BeamSmem {
  union {
    struct {
      unsigned long long cand[BNW][BCAP];                                  // the chunk's candidates, per wave
      float top[BBT][BNT];                                                 // the threads' largest candidate of each tile
      uint16_t hit[BNW][BBT * 64];                                         // (tile, lane) pairs that reach the threshold
    } w;
    struct { double ref[BGCH], sum[BGCH]; } c;                             // the finisher: chunks' weights
    BeamCand d[BDENSE];                                                    // ... and its candidates
  } u;
  double wref[BNW], wsum[BNW];
  uint32_t wthr[2][BNW], whave[2][BNW], wfew[BNW], wcnt[2][BNW], wtop[BNW], wbad[BNW];
  double score[MXS_BEAM_MAX], scale[MXS_BEAM_MAX], norm[MXS_BEAM_MAX];
  uint32_t key[BDENSE];                                                    // beam_key of the finisher's candidates
  uint16_t surv[BGCH], cnt[BGCH];
  uint8_t kind[MXS_BEAM_MAX];                                              // 0: not there, 1: live, 2: ended
  uint32_t flags, nsurv, m, last;
};

__device__ __forceinline__ bool beam_live(const BeamArgs& A, uint32_t row) {
  const double s = A.score[row];
  return s > -INFINITY && !(A.ended && A.ended[row]);
}

// One wave's candidates down to the n largest, sorted; returns how many are
// left and raises `lim` to the n-th.
__device__ __noinline__ uint32_t beam_compact(unsigned long long* c, uint32_t count, uint32_t n, unsigned long long* lim) {
  unsigned long long e[BCAP / 64];
  uint32_t r[BCAP / 64];
#pragma unroll
  for (uint32_t k = 0; k < BCAP / 64u; ++k) {
    e[k] = lane() + 64u * k < count ? c[lane() + 64u * k] : 0ull;
    r[k] = 0u;
  }
  for (uint32_t i = 0; i < count; ++i) {
    const unsigned long long v = c[i];
#pragma unroll
    for (uint32_t k = 0; k < BCAP / 64u; ++k) r[k] += v > e[k] ? 1u : 0u;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (uint32_t k = 0; k < BCAP / 64u; ++k)
    if (lane() + 64u * k < count && r[k] < n) c[r[k]] = e[k];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (count >= n) *lim = max(*lim, c[n - 1u]);
  return min(count, n);
}

// A chunk of one live row: its weights' sum, and a list that holds its n
// largest candidates.
template <typename In, int MODE>
__device__ __forceinline__ void beam_chunk(const BeamArgs& A, BeamSmem& S, uint32_t row, uint32_t chunk) {
  const uint32_t tid = threadIdx.x, V = A.V, n = A.n;
  const uint32_t c0 = chunk * A.T * BTILE, c1 = min(V, c0 + A.T * BTILE);
  const uint32_t tiles = (c1 - c0 + BTILE - 1u) / BTILE;
  const In* src = reinterpret_cast<const In*>(A.logits) + (uint64_t)row * A.stride;
  const uint32_t* mrow = MODE == BEAM_ALL ? nullptr : A.mask + (uint64_t)row * A.mask_stride;
  const uint32_t vm = MODE == BEAM_ALL ? V : min(V, A.tok_vocab);
  typename Quad<In>::Raw cur[BQ], nxt[BQ];
  uint32_t mcur[BQ] = {}, mnxt[BQ] = {};
  // the quad at token e0; nothing past the row is read, what is missing is -inf
  auto load_quad = [&](typename Quad<In>::Raw* raw, uint32_t e0) {
    if (e0 + 4u <= V) {
      *raw = Quad<In>::load(src + e0);
      return;
    }
    In v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = Quad<In>::ninf();
      if (e0 + (uint32_t)e < V) v[e] = src[e0 + (uint32_t)e];
    }
    *raw = Quad<In>::pack(v);
  };
  auto load = [&](typename Quad<In>::Raw (&d)[BQ], uint32_t (&mw)[BQ], uint32_t tile) {
    const uint32_t b = c0 + tile * BTILE;
    if (b + BTILE <= V) {   // uniform
#pragma unroll
      for (int q = 0; q < BQ; ++q) d[q] = Quad<In>::load(src + b + (uint32_t)q * BSL + tid * 4u);
      if (MODE != BEAM_ALL)
#pragma unroll
        for (int q = 0; q < BQ; ++q) mw[q] = mrow[(b + (uint32_t)q * BSL + tid * 4u) >> 5];
    } else {                // the row's last tile
#pragma unroll
      for (int q = 0; q < BQ; ++q) {
        const uint32_t e0 = b + (uint32_t)q * BSL + tid * 4u;
        load_quad(&d[q], e0);
        if (MODE != BEAM_ALL) mw[q] = e0 < V ? mrow[e0 >> 5] : 0u;
      }
    }
  };
  load(cur, mcur, 0u);

  unsigned long long* cand = S.u.w.cand[wave()];
  uint16_t* hit = S.u.w.hit[wave()];
  uint32_t woff = 0u;                 // this wave's candidates (uniform)
  unsigned long long lim = 0ull;      // entries below cannot be among the chunk's n largest
  uint32_t thr = 0u;                  // an order key that n of the chunk's candidates reach
  float lm = -INFINITY;               // this lane's largest candidate
  bool bad = false;
  double sum = 0.0, unit = -INFINITY; // the weights are relative to e^unit
  float ref = -INFINITY, hi = -INFINITY, lo = 0.0f;
  double magic = 0.0;
  bool wide = false;
  uint32_t slot = 0u, held = 0u, hits = 0u;
  // Quad i of the hits (four to a hit): its first token, its raw logits and
  // legal tokens.
  auto hit_load = [&](uint32_t i, uint32_t first, uint32_t* e0, typename Quad<In>::Raw* raw, uint32_t* nib) {
    const uint32_t h = hit[min(i >> 2, hits - 1u)];
    *e0 = c0 + (first + (h >> 6)) * BTILE + (i & 3u) * BSL + (wave() * 64u + (h & 63u)) * 4u;
    static_assert(BQ == 4, "four quads to a hit");
    load_quad(raw, *e0);
    *nib = 0u;
    if (MODE != BEAM_ALL && *e0 < V) *nib = beam_nibble(mrow[*e0 >> 5], *e0, vm);
  };
  for (uint32_t tile = 0; tile < tiles; ++tile) {
    if (tile + 1u < tiles) load(nxt, mnxt, tile + 1u);
    const uint32_t tb = c0 + tile * BTILE + tid * 4u;
    float x[BQ][4], tm;   // the logits weighed, the largest of them
    if (MODE == BEAM_ALL) {
      float qm[BQ];
#pragma unroll
      for (int q = 0; q < BQ; ++q) {
        Quad<In>::unpack(cur[q], x[q]);
        qm[q] = max_nan(max_nan(max_nan(x[q][0], x[q][1]), x[q][2]), x[q][3]);
      }
      tm = max_nan(max_nan(qm[0], qm[1]), max_nan(qm[2], qm[3]));
      S.u.w.top[held][tid] = tm;
      lm = fmaxf(lm, tm);
    } else {
      float ym = -INFINITY;
      tm = -INFINITY;
#pragma unroll
      for (int q = 0; q < BQ; ++q) {
        const uint32_t e0 = tb + (uint32_t)q * BSL, nib = beam_nibble(mcur[q], e0, vm);
        Quad<In>::unpack(cur[q], x[q]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = ((nib >> e) & 1u) ? x[q][e] : -INFINITY;
          ym = max_nan(ym, y);
          if (MODE == BEAM_MASK_NORM) x[q][e] = y;
          else tm = max_nan(tm, x[q][e]);
        }
      }
      if (MODE == BEAM_MASK_NORM) tm = ym;
      else bad |= !(tm < INFINITY);
      S.u.w.top[held][tid] = ym;
      lm = fmaxf(lm, ym);
    }
    ++held;
    const bool look = held == BBT || tile + 1u == tiles;
    const uint32_t first = tile + 1u - held;
    uint32_t he0 = 0u, hnib = 0u;
    typename Quad<In>::Raw hraw{};
    if (look) {
      // A key that at least n of the chunk's lanes have reached, so n of its
      // candidates have: each wave's n/4-th largest lane maximum (0 where
      // fewer lanes hold a candidate), the smallest over the waves, to its
      // upper 18 bits (a few candidates more, 14 ballots less).
      const uint32_t ak = lm > -INFINITY ? okey(lm) : 0u;
      const uint32_t have = (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(ak != 0u));
      auto reached = [&](uint32_t by) {   // by `by` of the wave's lanes
        uint32_t wthr = 0u;
        if (have >= by) {
#pragma unroll
          for (int bit = 31; bit >= 14; --bit) {
            const uint32_t c = wthr | (1u << bit);
            if ((uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(ak >= c)) >= by) wthr = c;
          }
        }
        return wthr;
      };
      const uint32_t wthr = reached((n + (uint32_t)BNW - 1u) / (uint32_t)BNW);
      if (lane() == 0) {
        S.wthr[slot][wave()] = wthr;
        S.whave[slot][wave()] = have;
      }
      lds_barrier();
      uint32_t t = 0xffffffffu;
#pragma unroll
      for (int w = 0; w < BNW; ++w) t = min(t, S.wthr[slot][w]);
      if (t == 0u) {   // uniform: a wave has too few
        // Fewer waves may have enough (a mask's runs, the row's end): the a-th
        // largest of the waves' n/a-th largest.
        uint32_t a = (uint32_t)BNW - 1u;
        for (; a; --a) {
          uint32_t ok = 0u;
#pragma unroll
          for (int w = 0; w < BNW; ++w) ok += S.whave[slot][w] >= (n + a - 1u) / a ? 1u : 0u;
          if (ok >= a) break;
        }
        if (a) {
          const uint32_t w1 = reached((n + a - 1u) / a);
          if (lane() == 0) S.wfew[wave()] = w1;
          lds_barrier();
          uint32_t k[BNW];
#pragma unroll
          for (int w = 0; w < BNW; ++w) k[w] = S.wfew[w];
#pragma unroll
          for (int w = 0; w < BNW; ++w) {
            uint32_t above = 0u;   // those at or above it
#pragma unroll
            for (int v = 0; v < BNW; ++v) above += k[v] >= k[w] ? 1u : 0u;
            if (above >= a) t = max(t, k[w]);
          }
        }
      }
      slot ^= 1u;
      thr = max(thr, t);
      lim = max(lim, (unsigned long long)thr << 32);
      // (a key below the finite ones' is no logit)
      const float fthr = okey_value(max((uint32_t)(lim >> 32), okey(-FLT_MAX)));
      // The few threads whose largest reaches it take a second look at that
      // tile's logits, again from memory (a NaN reaches it too): the loads go
      // out here and are used after the weights.
      hits = 0u;
      for (uint32_t k = 0; k < held; ++k) {
        const bool h = !(S.u.w.top[k][tid] < fthr);
        const uint64_t bal = __builtin_amdgcn_ballot_w64(h);
        if (bal == 0ull) continue;
        if (h) hit[hits + lanes_below(bal)] = (uint16_t)(k * 64u + lane());
        hits += (uint32_t)__builtin_popcountll(bal);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (hits) hit_load(lane(), first, &he0, &hraw, &hnib);
    }
    // The weights, relative to a power of two near the first maximum the wave
    // meets: f64 holds e^-700..e^600 of it, so it moves only for a later
    // maximum 600 above.  (Logits past 1000 in size: for any later maximum. A
    // f32 near 2^33 plus 600 rounds to 1024 above, whose weight f64 does not
    // hold.)
    if (__builtin_amdgcn_ballot_w64(tm > hi)) {
      const float wm = wave_max_f32(tm);
      wide = !(fabsf(wm) <= 1000.0f);
      const double n0 = rint((double)wm * 1.4426950408889634);
      const double u = wide ? (double)wm : n0 * 0.6931471805599453;
      if (ref > -INFINITY) sum *= exp_neg_p(unit - u);
      ref = wm;
      unit = u;
      hi = wide ? wm : wm + 600.0f;
      lo = wm - 700.0f;
      magic = 0x1.8p52 - n0;
    }
    if (ref > -INFINITY) {
      if (!wide) {
#pragma unroll
        for (int q = 0; q < BQ; ++q) {
          double w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = beam_weight(vmax(x[q][e], lo), magic);
          sum += (w[0] + w[1]) + (w[2] + w[3]);
        }
      } else {
#pragma unroll 1
        for (int q = 0; q < BQ; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum += exp_neg_p((double)x[q][e] - unit);
      }
    }
    if (look) {
      for (uint32_t i0 = 0; i0 < 4u * hits; i0 += 64u) {
        if (i0) hit_load(i0 + lane(), first, &he0, &hraw, &hnib);
        const bool in = i0 + lane() < 4u * hits;
        float v[4];
        Quad<In>::unpack(hraw, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool legal = in && (MODE == BEAM_ALL || ((hnib >> e) & 1u));
          const unsigned long long entry = beam_entry(okey(v[e] + 0.0f), he0 + (uint32_t)e);   // -0 as +0
          bad |= legal && !(v[e] < INFINITY);
          bool c = legal && v[e] > -INFINITY && entry >= lim;
          uint64_t bal = __builtin_amdgcn_ballot_w64(c);
          if (bal == 0ull) continue;
          if (woff + (uint32_t)__builtin_popcountll(bal) > BCAP) {
            woff = beam_compact(cand, woff, n, &lim);
            c = c && entry >= lim;
            bal = __builtin_amdgcn_ballot_w64(c);
          }
          if (c) cand[woff + lanes_below(bal)] = entry;
          woff += (uint32_t)__builtin_popcountll(bal);
        }
      }
      held = 0u;
    }
#pragma unroll
    for (int q = 0; q < BQ; ++q) {
      cur[q] = nxt[q];
      mcur[q] = mnxt[q];
    }
  }

  // ---- the chunk's results
  sum = wave_sum_f64(sum);
  const uint32_t top = wave_max_u32(lm > -INFINITY ? okey(lm + 0.0f) : 0u);
  const bool wbad = __builtin_amdgcn_ballot_w64(bad) != 0ull;
  uint32_t kept = 0u;
#pragma unroll
  for (uint32_t k = 0; k < BCAP / 64u; ++k) {
    const uint32_t i = lane() + 64u * k;
    kept += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(i < woff && cand[i < woff ? i : 0u] >= lim));
  }
  if (lane() == 0) {
    S.wsum[wave()] = sum;
    S.wref[wave()] = unit;
    S.wtop[wave()] = top;
    S.wbad[wave()] = wbad ? 1u : 0u;
    S.wcnt[0][wave()] = kept;
  }
  lds_barrier();
  uint32_t before = 0u, total = 0u, ctop = 0u, cbad = 0u;
#pragma unroll
  for (int w = 0; w < BNW; ++w) {
    before += (uint32_t)w < wave() ? S.wcnt[0][w] : 0u;
    total += S.wcnt[0][w];
    ctop = max(ctop, S.wtop[w]);
    cbad |= S.wbad[w];
  }
  if (total > BLIST) {   // near-ties: each wave's n largest
    if (woff > n) woff = beam_compact(cand, woff, n, &lim);
    kept = 0u;
#pragma unroll
    for (uint32_t k = 0; k < BCAP / 64u; ++k) {
      const uint32_t i = lane() + 64u * k;
      kept += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(i < woff && cand[i < woff ? i : 0u] >= lim));
    }
    if (lane() == 0) S.wcnt[1][wave()] = kept;
    lds_barrier();
    before = total = 0u;
#pragma unroll
    for (int w = 0; w < BNW; ++w) {
      before += (uint32_t)w < wave() ? S.wcnt[1][w] : 0u;
      total += S.wcnt[1][w];
    }
  }
  const uint64_t at = (uint64_t)row * A.C + chunk;
#pragma unroll
  for (uint32_t k = 0; k < BCAP / 64u; ++k) {
    const uint32_t i = lane() + 64u * k;
    const unsigned long long e = i < woff ? cand[i] : 0ull;
    const bool c = i < woff && e >= lim;
    const uint64_t bal = __builtin_amdgcn_ballot_w64(c);
    if (c) st_dev(&A.list[at * BLIST + before + lanes_below(bal)], e);
    before += (uint32_t)__builtin_popcountll(bal);
  }
  if (wave() == 0) {   // the waves' sums, each lane one
    const double r = lane() < (uint32_t)BNW ? S.wref[lane()] : -INFINITY;
    const double cr = wave_max_f64(r);
    const double e = r > -INFINITY ? S.wsum[lane()] * exp_neg_p(r - cr) : 0.0;
    const double cs = ((readlane_t(e, 0) + readlane_t(e, 1)) + readlane_t(e, 2)) + readlane_t(e, 3);
    if (lane() == 0) {
      BeamStat* st = &A.stat[at];
      st_dev(&st->ref, cr);
      st_dev(&st->sum, cs);
      st_dev(&st->thr, thr);
      st_dev(&st->top, ctop);
      st_dev(&st->count, total);
      st_dev(&st->bad, cbad);
    }
  }
}

// A candidate's place among equal ranks as one number: lower beam, larger
// logit, lower token.  An ended beam's key is 1, below every logit's.
__device__ __forceinline__ unsigned long long beam_tie(uint32_t beam, uint32_t key, uint32_t token) {
  return ((unsigned long long)(MXS_BEAM_MAX - 1u - beam) << 53) | ((unsigned long long)key << 21) |
         (unsigned long long)(BEAM_MAX_VOCAB - 1u - token);
}
__device__ __forceinline__ double beam_score(const BeamSmem& S, uint32_t b, uint32_t key) {
  return S.kind[b] == 2 ? S.score[b] : S.score[b] + ((double)okey_value(key) - S.norm[b]);
}
__device__ __forceinline__ double beam_rank(const BeamSmem& S, uint32_t b, uint32_t key) {   // of a live beam's candidate
  return (S.score[b] + ((double)okey_value(key) - S.norm[b])) * S.scale[b];
}

// Over each 16 lanes, in all of them.
template <typename F>
__device__ __forceinline__ double row_all_f64(double v, F f) {
  auto turned = [](auto ctrl, double x) {
    return __builtin_bit_cast(double, dpp64<decltype(ctrl)::value>(__builtin_bit_cast(unsigned long long, x)));
  };
  v = f(v, turned(std::integral_constant<int, 0x128>{}, v));   // row_ror:8, 4, 2, 1
  v = f(v, turned(std::integral_constant<int, 0x124>{}, v));
  v = f(v, turned(std::integral_constant<int, 0x122>{}, v));
  return f(v, turned(std::integral_constant<int, 0x121>{}, v));
}

__device__ __forceinline__ bool beam_before(const BeamCand& a, const BeamCand& b) {
  return (a.rank > b.rank) | ((a.rank == b.rank) & (a.tie > b.tie));   // (no branch around the second read)
}

// The upper half of a rank's order key; 0 for none.  (-0 as +0: equal ranks.)
__device__ __forceinline__ uint32_t beam_key(double r) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, r + 0.0);
  return (uint32_t)(((b >> 63) ? ~b : (b | 1ull << 63)) >> 32);
}

// At most the wave's k-th largest of the lanes' ranks (-inf: none), -inf when
// it has fewer: a value near it that k of them reach.
template <int OWN>
__device__ __forceinline__ double beam_wave_nth(const double (&r)[OWN], uint32_t k) {
  uint32_t key[OWN], most = 0u, have = 0u;   // the upper halves of order keys (0: none)
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    key[i] = r[i] > -INFINITY ? beam_key(r[i]) : 0u;
    most = max(most, key[i]);
    have += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(key[i] != 0u));
  }
  if (have < k) return -INFINITY;
  most = wave_max_u32(most);
  uint32_t least = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < OWN; ++i) least = key[i] ? min(least, key[i]) : least;
  least = ~wave_max_u32(~least);
  // twelve bits of the keys' distance from the least: within 2^-11 of their
  // spread (a prefix of the keys themselves says nothing across 2.0, where
  // the exponent's upper bit turns)
#pragma unroll
  for (int i = 0; i < OWN; ++i) key[i] = key[i] ? key[i] - least + 1u : 0u;
  const int first = 31 - __builtin_clz(most - least + 1u);
  uint32_t t = 0u;
  for (int bit = first; bit >= max(0, first - 11); --bit) {
    const uint32_t c = t | (1u << bit);
    uint32_t count = 0u;
#pragma unroll
    for (int i = 0; i < OWN; ++i) count += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(key[i] >= c));
    if (count >= k) t = c;
  }
  t = least + max(t, 1u) - 1u;
  const unsigned long long b = (unsigned long long)t << 32;
  return __builtin_bit_cast(double, (t >> 31) ? b & ~(1ull << 63) : ~b);
}

// The group's n best, by its last workgroup: the rows' norms from their
// chunks, a rank that n candidates reach (the best chunk threshold), the
// entries of the chunks that reach it, their order by counting.
__device__ __forceinline__ void beam_finish(const BeamArgs& A, BeamSmem& S, uint32_t g) {
  const uint32_t tid = threadIdx.x, W = A.W, C = A.C, n = A.n, NC = W * C;
  constexpr int OWN = (int)(BGCH / BNT);
  // (a row's chunks fall to all four waves)
  auto own = [&](int i) { return lane() * (uint32_t)BNW + wave() + (uint32_t)i * BNT; };
  double ref[OWN], sum[OWN];
  uint32_t cthr[OWN], ctop[OWN], ccnt[OWN], cbad[OWN];
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    const uint32_t c = own(i);
    const BeamStat* st = &A.stat[(uint64_t)g * NC + min(c, NC - 1u)];   // (a row that is not live has none: not used)
    ref[i] = ld_dev(&st->ref);
    sum[i] = ld_dev(&st->sum);
    cthr[i] = ld_dev(&st->thr);
    ctop[i] = ld_dev(&st->top);
    ccnt[i] = ld_dev(&st->count);
    cbad[i] = ld_dev(&st->bad);
  }
  if (tid == 0) {
    S.flags = 0u;
    S.nsurv = 0u;
    S.m = 0u;
  }
  uint32_t err = 0u;
  if (tid < W) {
    const uint32_t row = g * W + tid;
    const double s = A.score[row], c = A.scale ? A.scale[row] : 1.0;
    const bool e = A.ended && A.ended[row];
    S.score[tid] = s;
    S.scale[tid] = c;
    S.kind[tid] = !(s > -INFINITY) ? 0 : e ? 2 : 1;
    if (!(s < INFINITY) || !(c > 0.0 && c < INFINITY)) err = 1u;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    const uint32_t c = own(i);
    if (c >= NC || S.kind[c / C] != 1) {
      ccnt[i] = 0u;
      cthr[i] = 0u;
    } else if (cbad[i]) {
      err |= 2u;
    }
    if (c < NC) {
      S.u.c.ref[c] = ref[i];
      S.u.c.sum[c] = sum[i];
      S.cnt[c] = (uint16_t)ccnt[i];
    }
  }
  if (err) atomicOr(&S.flags, err);
  __syncthreads();
  if (S.flags) {   // uniform
    for (uint32_t j = tid; j < n; j += BNT) {
      const uint64_t at = (uint64_t)g * n + j;
      A.token[at] = -1;
      A.beam[at] = -1;
      A.oscore[at] = __builtin_nan("");
      if (A.oended) A.oended[at] = 0;
    }
    if (tid == 0) A.status[g] = (S.flags & 1u) ? MXS_ROW_PROBABILITIES : MXS_ROW_NON_FINITE_LOGIT;
    return;
  }
  // The rows' norms: a row's chunks on 16 lanes or 64, relative to the largest
  // unit, added in an order that the number of chunks alone gives.
  {
    const bool few = C <= 16u || W > (uint32_t)BNW;   // (sixteen rows at once, or one per wave)
    const uint32_t L = few ? 16u : 64u;
    auto whole = [&](double v, auto f) {
      v = row_all_f64(v, f);
      return few ? v : f(f(readlane_t(v, 0), readlane_t(v, 16)), f(readlane_t(v, 32), readlane_t(v, 48)));
    };
    for (uint32_t b0 = wave() * (64u / L); b0 < W; b0 += (uint32_t)BNW * (64u / L)) {
      const uint32_t b = b0 + lane() / L, first = b * C, k0 = lane() % L;
      const bool live = b < W && S.kind[min(b, W - 1u)] == 1;
      double m = -INFINITY, t = 0.0;
      for (uint32_t k = k0; live && k < C; k += L) m = fmax(m, S.u.c.ref[first + k]);
      m = whole(m, [](double x, double y) { return fmax(x, y); });
      for (uint32_t k = k0; live && k < C; k += L) {
        const double r = S.u.c.ref[first + k];
        if (r > -INFINITY) t += S.u.c.sum[first + k] * exp_neg_p(r - m);
      }
      t = whole(t, [](double x, double y) { return x + y; });
      if (live && k0 == 0u) S.norm[b] = m + log(t);   // (a row without weight has no candidates either)
    }
  }
  __syncthreads();
  // A rank that n candidates reach: the best chunk threshold, or the n-th
  // largest of the chunks' largest (by wave: its n/4-th largest, the smallest
  // over the waves), whichever is more.
  double gthr = -INFINITY, ctr[OWN];
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    const uint32_t b = min(own(i), NC - 1u) / C;
    ctr[i] = ccnt[i] ? beam_rank(S, b, ctop[i]) : -INFINITY;
    if (cthr[i]) gthr = fmax(gthr, beam_rank(S, b, max(cthr[i], okey(-FLT_MAX))));
  }
  gthr = wave_max_f64(gthr);
  const double nth = beam_wave_nth(ctr, (n + (uint32_t)BNW - 1u) / (uint32_t)BNW);
  if (lane() == 0) {
    S.wref[wave()] = gthr;
    S.wsum[wave()] = nth;
  }
  __syncthreads();
  double tops = S.wsum[0];
#pragma unroll
  for (int w = 0; w < BNW; ++w) {
    gthr = fmax(gthr, S.wref[w]);
    tops = fmin(tops, S.wsum[w]);
  }
  gthr = fmax(gthr, tops);
  uint32_t ns = 0;
  auto each = [&](auto&& f) {   // every listed entry that reaches gthr, 16 lanes to a chunk
    for (uint32_t k = tid >> 4; k < ns; k += 2u * (BNT / 16u)) {
      double d[2][4];   // (two chunks' loads in flight)
      uint32_t c[2], count[2];
      const double* list[2];
#pragma unroll
      for (uint32_t h = 0; h < 2u; ++h) {
        c[h] = S.surv[min(k + h * (BNT / 16u), ns - 1u)];
        count[h] = k + h * (BNT / 16u) < ns ? S.cnt[c[h]] : 0u;
        list[h] = reinterpret_cast<const double*>(&A.list[((uint64_t)g * NC + c[h]) * BLIST]);
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
          const uint32_t j = (tid & 15u) + 16u * i;
          if (j < count[h]) d[h][i] = ld_dev(&list[h][j]);
        }
      }
#pragma unroll
      for (uint32_t h = 0; h < 2u; ++h) {
        const uint32_t b = c[h] / C;
        const double bs = S.score[b], bn = S.norm[b], bc = S.scale[b];   // (live beams only have lists)
        for (uint32_t j0 = tid & 15u; j0 < count[h]; j0 += 64u) {
          if (j0 >= 64u)
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i)
              if (j0 + 16u * i < count[h]) d[h][i] = ld_dev(&list[h][j0 + 16u * i]);
#pragma unroll
          for (uint32_t i = 0; i < 4u; ++i) {
            if (j0 + 16u * i >= count[h]) continue;
            const unsigned long long e = __builtin_bit_cast(unsigned long long, d[h][i]);
            const uint32_t key = (uint32_t)(e >> 32);
            const double r = (bs + ((double)okey_value(key) - bn)) * bc;
            if (r >= gthr) f(r, beam_tie(b, key, ~(uint32_t)e));
          }
        }
      }
    }
  };
  uint32_t m = 0;
  for (int round = 0;; ++round) {
    // the chunks that reach gthr, the ended beams and the entries that do
#pragma unroll
    for (int i = 0; i < OWN; ++i)
      if (ccnt[i] && ctr[i] >= gthr) S.surv[atomicAdd(&S.nsurv, 1u)] = (uint16_t)own(i);
    auto keep = [&](double r, unsigned long long t) {
      const uint32_t at = atomicAdd(&S.m, 1u);
      if (at < BDENSE) {
        S.u.d[at] = BeamCand{r, t};
        S.key[at] = beam_key(r);
      }
    };
    if (tid < W && S.kind[tid] == 2) {
      const double r = S.score[tid] * S.scale[tid];
      if (r >= gthr) keep(r, beam_tie(tid, 1u, (uint32_t)A.end_token));
    }
    __syncthreads();
    ns = S.nsurv;
    each(keep);
    __syncthreads();
    m = S.m;
    if (m <= 2u * n + 64u || round == 3) break;
    // Many (few chunks or few of them with candidates, so a loose
    // threshold): the n-th largest of those kept,
    // which n candidates reach too, is a closer one.
    double r[BDENSE / BNT];
#pragma unroll
    for (uint32_t i = 0; i < BDENSE / BNT; ++i) {   // (in turn to the waves: neighbours are of one chunk)
      const uint32_t at = (uint32_t)own((int)i);
      r[i] = at < m ? S.u.d[at].rank : -INFINITY;
    }
    const double wnth = beam_wave_nth(r, (n + (uint32_t)BNW - 1u) / (uint32_t)BNW);
    if (lane() == 0) S.wsum[wave()] = wnth;
    __syncthreads();   // (S.m and S.nsurv have been read)
    if (tid == 0) S.m = S.nsurv = 0u;
    double t = S.wsum[0];
#pragma unroll
    for (int w = 1; w < BNW; ++w) t = fmin(t, S.wsum[w]);
    if (!(t > gthr)) break;   // equal ranks: m stands
    gthr = t;
    __syncthreads();
  }
  if (tid < 8u && m + tid < BDENSE) S.key[m + tid] = 0u;
  __syncthreads();
  auto put = [&](uint32_t j, unsigned long long t) {
    const uint64_t at = (uint64_t)g * n + j;
    const uint32_t b = MXS_BEAM_MAX - 1u - (uint32_t)(t >> 53);
    const int32_t token = (int32_t)(BEAM_MAX_VOCAB - 1u - ((uint32_t)t & (BEAM_MAX_VOCAB - 1u)));
    A.token[at] = token;
    A.beam[at] = (int32_t)b;
    A.oscore[at] = beam_score(S, b, (uint32_t)(t >> 21));
    if (A.oended) A.oended[at] = token == A.end_token ? 1 : 0;
  };
  if (m <= BDENSE) {
    // Each one's place by counting, on the upper halves of the ranks' order
    // keys (a 64-bit comparison costs several 32-bit ones); those that share
    // one compare in full.
    for (uint32_t i = tid; i < m; i += BNT) {
      const BeamCand e = S.u.d[i];
      const uint32_t mine = S.key[i];
      uint32_t at = 0, same = 0;
      for (uint32_t k = 0; k < m; k += 8u) {   // (the keys past m are 0)
        const uint4 v0 = *reinterpret_cast<const uint4*>(&S.key[k]), v1 = *reinterpret_cast<const uint4*>(&S.key[k + 4u]);
        const uint32_t v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
        for (uint32_t j = 0; j < 8u; ++j) {
          at += v[j] > mine ? 1u : 0u;
          same += v[j] == mine ? 1u : 0u;
        }
      }
      if (same > 1u)
        for (uint32_t k = 0; k < m; k += 8u) {
          const uint4 v0 = *reinterpret_cast<const uint4*>(&S.key[k]), v1 = *reinterpret_cast<const uint4*>(&S.key[k + 4u]);
          const uint32_t v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
          uint32_t eq = 0u;
#pragma unroll
          for (uint32_t j = 0; j < 8u; ++j) eq |= v[j] == mine ? 1u << j : 0u;
          for (; eq; eq &= eq - 1u) at += beam_before(S.u.d[k + (uint32_t)__builtin_ctz(eq)], e) ? 1u : 0u;
        }
      if (at < n) put(at, e.tie);
    }
  } else {
    // more near-ties than fit: the best after the last one, n times
    BeamCand last{INFINITY, ~0ull};
    for (uint32_t j = 0; j < n; ++j) {
      BeamCand best{-INFINITY, 0ull};
      auto take = [&](double r, unsigned long long t) {
        const BeamCand e{r, t};
        if (beam_before(last, e) && beam_before(e, best)) best = e;
      };
      each(take);
      if (tid < W && S.kind[tid] == 2) take(S.score[tid] * S.scale[tid], beam_tie(tid, 1u, (uint32_t)A.end_token));
      __syncthreads();
      S.u.d[tid] = best;
      __syncthreads();
      for (uint32_t h = BNT / 2; h > 0; h >>= 1) {
        if (tid < h && beam_before(S.u.d[tid + h], S.u.d[tid])) S.u.d[tid] = S.u.d[tid + h];
        __syncthreads();
      }
      last = S.u.d[0];
      if (tid == 0) put(j, last.tie);   // (m > BDENSE >= n candidates: there is always one)
    }
  }
  for (uint32_t j = m + tid; j < n; j += BNT) {
    const uint64_t at = (uint64_t)g * n + j;
    A.token[at] = -1;
    A.beam[at] = -1;
    A.oscore[at] = -INFINITY;
    if (A.oended) A.oended[at] = 0;
  }
  if (tid == 0) A.status[g] = m ? MXS_ROW_OK : MXS_ROW_EMPTY_SUPPORT;
}

template <typename In, int MODE>
__global__ __launch_bounds__(BNT, 4) void beam_kernel(BeamArgs A) {
  __shared__ BeamSmem S;
  const uint32_t row = blockIdx.x / A.C, chunk = blockIdx.x - row * A.C, g = row / A.W;
  if (beam_live(A, row)) beam_chunk<In, MODE>(A, S, row, chunk);
  if (!arrive_last(&A.ctr[g * CTR_STRIDE], A.W * A.C, &S.last)) return;
  beam_finish(A, S, g);
}

// Chunks per row and tiles per chunk: enough workgroups to fill the chip
// (BWGS), no more per group than its finisher's threads hold.
static void beam_layout(uint32_t rows, uint32_t W, uint32_t V, uint32_t* C, uint32_t* T) {
  const uint32_t tiles = (V + BTILE - 1u) / BTILE;
  uint32_t c = BWGS / rows;
  if (c > BGCH / W) c = BGCH / W;
  if (c > tiles) c = tiles;
  if (c < 1u) c = 1u;
  *T = (tiles + c - 1u) / c;
  *C = (tiles + *T - 1u) / *T;
}

size_t beam_scratch_bytes(uint32_t max_rows) {   // rows * C <= BWGS + max_rows
  return ((size_t)BWGS + max_rows) * (sizeof(BeamStat) + BLIST * sizeof(unsigned long long));
}

template <int MODE>
static void beam_go(hipStream_t stream, int32_t dtype, const BeamArgs& A) {
  const dim3 grid(A.G * A.W * A.C);
  if (dtype == MXS_F32) hipLaunchKernelGGL((beam_kernel<float, MODE>), grid, dim3(BNT), 0, stream, A);
  else hipLaunchKernelGGL((beam_kernel<uint16_t, MODE>), grid, dim3(BNT), 0, stream, A);
}

// ---------------------------------------------------------------------------
// The move of the states.
constexpr uint32_t RO_STATES = 64;        // states per launch (their descriptions travel as kernel arguments)
constexpr int RO_NT = 256;

struct ReorderArgs {
  mxs_state st[RO_STATES];
  const int32_t* parent;
  const int32_t* lengths;
  int32_t* status;                        // nullptr: another launch of the call writes it
  uint32_t W, pstride;
};

// Pieces of a row at any alignment (global memory takes unaligned accesses),
// as values in registers.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <typename T>
struct Unaligned { typedef T type __attribute__((aligned(1))); };

// Moves one T at `at` (in row 0 of the group) between the rows.  to[j]: the
// rows that take row j over (uniform over the wave, in LDS).  Row J's value is
// loaded, then the rows' after it, then row J's is stored: all loads before
// all stores.  (A recursion and no array: an array written under conditions
// is kept as one value, and copied whole at each: 222 registers for 8 rows.)
template <typename T, int WMAX, int J>
__device__ __forceinline__ void move_piece(char* at, uint64_t stride, const unsigned long long* to) {
  if constexpr (J < WMAX) {
    typedef typename Unaligned<T>::type U;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)to[J]);
    const uint32_t hi = WMAX > 32 ? __builtin_amdgcn_readfirstlane((uint32_t)(to[J] >> 32)) : 0u;
    T v;
    if (lo | hi) v = *reinterpret_cast<const U*>(at + (uint64_t)J * stride);
    move_piece<T, WMAX, J + 1>(at, stride, to);
    for (uint32_t m = lo; m; m &= m - 1u) *reinterpret_cast<U*>(at + (uint64_t)(uint32_t)__builtin_ctz(m) * stride) = v;
    for (uint32_t m = hi; m; m &= m - 1u) *reinterpret_cast<U*>(at + (uint64_t)(32u + (uint32_t)__builtin_ctz(m)) * stride) = v;
  }
}

// One thread holds the same 16 bytes of all the group's rows: it loads those
// of every row that some other row takes over, then stores them to the rows
// that take them.  No thread reads what another writes, so any permutation
// goes in place, each surviving row read once and each changed row written
// once.  WMAX, the most rows held, is the power of two at or above beams (20,
// 36, 68, 133 and 255 registers).  us, and at 4.92 TB/s: 8 groups x 4 beams x
// 56 states of 8 x 520 x 128 bf16, ragged lengths (1.87 GB) 358-383, 379; 4 x 8
// 432, 433; 2 x 32 of half the length 508, 499; 1 x 64 607, 576; 1 x 4 x 56
// states of 8 x 48 x 128 (28 MB) 7.2, 5.6.
template <int WMAX>
__global__ __launch_bounds__(RO_NT) void reorder_kernel(ReorderArgs A) {
  const mxs_state& s = A.st[blockIdx.z];
  const uint32_t g = blockIdx.y, W = A.W, l = threadIdx.x & 63u;
  const int32_t p = l < W ? A.parent[(uint64_t)g * A.pstride + l] : -1;
  const bool bad = __builtin_amdgcn_ballot_w64(p < -1 || p >= (int32_t)W) != 0ull;
  if (A.status && blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) A.status[g] = bad ? MXS_ROW_INVALID_PARENT : MXS_ROW_OK;
  if (bad) return;
  uint64_t used = s.segment_bytes;
  if (A.lengths && s.position_bytes) {
    const int32_t len = A.lengths[g];
    used = len <= 0 ? 0ull : min(used, (uint64_t)len * s.position_bytes);
  }
  const uint32_t pieces = (uint32_t)((used + 15u) / 16u);   // per segment
  const uint32_t total = pieces * s.segments;               // < 2^31
  if (blockIdx.x * RO_NT >= total) return;                  // the whole workgroup
  __shared__ unsigned long long to[WMAX];
  if (threadIdx.x < 64u) {
    unsigned long long mine = 0ull;   // lane j: the rows that take row j over
    for (uint32_t d = 0; d < W; ++d)
      if ((uint32_t)__builtin_amdgcn_readlane(p, (int)d) == l && d != l) mine |= 1ull << d;
    if (l < (uint32_t)WMAX) to[l] = mine;
  }
  __syncthreads();
  const uint32_t i = blockIdx.x * RO_NT + threadIdx.x;
  if (i >= total) return;
  const uint32_t seg = i / pieces, pc = i - seg * pieces;
  char* at = reinterpret_cast<char*>(s.data) + (uint64_t)g * W * s.row_stride + (uint64_t)seg * s.segment_stride +
             (uint64_t)pc * 16u;
  const uint32_t have = (uint32_t)min((uint64_t)16u, used - (uint64_t)pc * 16u);
  if (have == 16u) {
    move_piece<u32x4, WMAX, 0>(at, s.row_stride, to);
    return;
  }
  // a segment's last bytes
  if (have & 8u) move_piece<u32x2, WMAX, 0>(at, s.row_stride, to);
  at += have & 8u;
  if (have & 4u) move_piece<uint32_t, WMAX, 0>(at, s.row_stride, to);
  at += have & 4u;
  if (have & 2u) move_piece<uint16_t, WMAX, 0>(at, s.row_stride, to);
  at += have & 2u;
  if (have & 1u) move_piece<uint8_t, WMAX, 0>(at, s.row_stride, to);
}

template <int WMAX>
static void reorder_go(hipStream_t stream, dim3 grid, const ReorderArgs& A) {
  hipLaunchKernelGGL(reorder_kernel<WMAX>, grid, dim3(RO_NT), 0, stream, A);
}

}  // namespace mxs

extern "C" int mxs_beam_select(mxs_ctx* ctx, const mxs_beam* beam, const mxs_beam_out* out) {
  using namespace mxs;
  if (!ctx) return MXS_EINVAL;
  if (const char* m = beam_check(beam, out, ctx->max_rows, ctx->max_vocab)) return fail(ctx, MXS_EINVAL, m);
  const mxs_beam& b = *beam;
  if (b.groups == 0) return MXS_OK;
  BeamArgs A{};
  A.logits = b.logits;
  A.stride = b.row_stride;
  A.G = b.groups;
  A.W = b.beams;
  A.V = b.vocab;
  A.n = b.n;
  A.score = b.score;
  A.ended = b.ended;
  A.scale = b.scale;
  A.mask = b.mask_words;
  A.mask_stride = b.mask_stride;
  A.tok_vocab = b.tokenizer_vocab;
  A.end_token = b.end_token;
  A.token = out->token;
  A.beam = out->beam;
  A.oscore = out->score;
  A.oended = out->ended;
  A.status = out->status;
  beam_layout(A.G * A.W, A.W, A.V, &A.C, &A.T);
  A.stat = reinterpret_cast<BeamStat*>(ctx->beam_scratch);
  A.list = reinterpret_cast<unsigned long long*>(A.stat + ((size_t)BWGS + ctx->max_rows));
  A.ctr = ctx->beam_ctr;
  int prev = 0;
  (void)hipGetDevice(&prev);
  if (prev != ctx->device) (void)hipSetDevice(ctx->device);
  if (!b.mask_words) beam_go<BEAM_ALL>(ctx->stream, b.dtype, A);
  else if (!b.legal_norm) beam_go<BEAM_MASK>(ctx->stream, b.dtype, A);
  else beam_go<BEAM_MASK_NORM>(ctx->stream, b.dtype, A);
  const hipError_t e = hipGetLastError();
  if (prev != ctx->device) (void)hipSetDevice(prev);
  if (e != hipSuccess) return hip_fail(ctx, e, "beam launch");
  mask_note_read(ctx, b.mask_words);
  return MXS_OK;
}

extern "C" int mxs_beam_reorder_check(mxs_ctx* ctx, const mxs_reorder* reorder) {
  if (!ctx) return MXS_EINVAL;
  if (const char* m = mxs::reorder_check(reorder)) return fail(ctx, MXS_EINVAL, m);
  return MXS_OK;
}

extern "C" int mxs_beam_reorder(mxs_ctx* ctx, const mxs_reorder* reorder) {
  using namespace mxs;
  if (!ctx) return MXS_EINVAL;
  if (const char* m = reorder_check(reorder)) return fail(ctx, MXS_EINVAL, m);
  const mxs_reorder& r = *reorder;
  if (r.groups == 0) return MXS_OK;
  int prev = 0;
  (void)hipGetDevice(&prev);
  if (prev != ctx->device) (void)hipSetDevice(ctx->device);
  hipError_t e = hipSuccess;
  for (uint32_t first = 0; first < r.count && e == hipSuccess; first += RO_STATES) {
    const uint32_t here = r.count - first < RO_STATES ? r.count - first : RO_STATES;
    ReorderArgs A{};
    A.parent = r.parent;
    A.lengths = r.lengths;
    A.status = first == 0 ? r.status : nullptr;
    A.W = r.beams;
    A.pstride = r.parent_stride;
    uint64_t most = 0;
    for (uint32_t i = 0; i < here; ++i) {
      A.st[i] = r.states[first + i];
      const uint64_t total = (A.st[i].segment_bytes + 15u) / 16u * A.st[i].segments;
      if (total > most) most = total;
    }
    const dim3 grid((uint32_t)((most + RO_NT - 1u) / RO_NT), r.groups, here);
    if (r.beams <= 4) reorder_go<4>(ctx->stream, grid, A);
    else if (r.beams <= 8) reorder_go<8>(ctx->stream, grid, A);
    else if (r.beams <= 16) reorder_go<16>(ctx->stream, grid, A);
    else if (r.beams <= 32) reorder_go<32>(ctx->stream, grid, A);
    else reorder_go<64>(ctx->stream, grid, A);
    e = hipGetLastError();
  }
  if (prev != ctx->device) (void)hipSetDevice(prev);
  if (e != hipSuccess) return hip_fail(ctx, e, "reorder_kernel launch");
  return MXS_OK;
}
