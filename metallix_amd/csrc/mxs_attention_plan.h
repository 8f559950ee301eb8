// mxs_attention_plan.h -- how mxs_prefix_attention splits its work: a pure
// function of the sizes, in plain C++ so that it is checked without a GPU.
#pragma once
#include <stdint.h>

namespace mxs {

constexpr uint32_t ATT_TILE = 64;                  // positions a tile
constexpr uint64_t ATT_SCRATCH = 64ull << 20;      // bytes of a context's scratch for the parts

struct AttPlan {
  uint32_t dp;            // dim rounded up to 64, 128 or 256
  uint32_t rb, wq;        // prefix workgroups: 16 rb queries a wave, wq waves side by side
  bool small;             // suffix workgroups take 16 queries each (else as the prefix's)
  uint32_t sp, ss;        // parts of a prefix and of a suffix
  uint32_t slots;         // of a query: its prefix's parts, then its suffix's
  // One launch takes ng groups of wb rows and nt tokens.
  uint32_t ng, wb, nt;
};

inline uint32_t att_ceil(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1u) / b); }

// Bytes of the parts of so many queries: sums, statistics, and the queries' references.
inline uint64_t att_bytes(uint64_t queries, uint32_t slots, uint32_t dp) { return (queries * (slots * (dp + 2ull) + 1u) + 3u) * 4u; }

// How long `np` workgroups of `a` tiles and then `ns` of `b` take on `places`
// at once, in tiles; starting and ending one takes as long as two.
inline uint64_t att_time(uint64_t np, uint64_t a, uint64_t ns, uint64_t b, uint64_t places) {
  a += 2u, b += 2u;
  const uint64_t rem = np % places;
  uint64_t t = np / places * a;
  if (rem) {   // the others' places take workgroups of the second kind meanwhile
    const uint64_t fit = (places - rem) * (a / b);
    ns = ns > fit ? ns - fit : 0u;
    t += a;
  }
  return t + (ns + places - 1u) / places * b;
}

inline AttPlan attention_plan(uint32_t G, uint32_t W, uint32_t T, uint32_t H, uint32_t KV, uint32_t D, uint32_t P, uint32_t N) {
  AttPlan p{};
  const uint32_t per = H / KV;
  p.dp = D <= 64u ? 64u : D <= 128u ? 128u : 256u;
  const uint32_t least = (P ? 1u : 0u) + (N ? 1u : 0u);   // parts that every query has
  const uint64_t room = (ATT_SCRATCH - 16u) / (((least ? least : 1u) * (p.dp + 2u) + 1u) * 4u);   // queries a launch can hold
  p.ng = G, p.wb = W, p.nt = T;
  if ((uint64_t)G * W * T * H > room) {
    const uint64_t group = (uint64_t)W * T * H, row = (uint64_t)T * H;
    p.ng = group <= room ? (uint32_t)(room / group) : 1u;
    if (group > room) p.wb = row <= room ? (uint32_t)(room / row) : 1u;
    if (row > room) p.nt = (uint32_t)(room / H);
  }
  const uint32_t ms = p.nt * per, m = P ? p.wb * ms : ms;   // queries that share a suffix, a prefix
  p.rb = p.dp == 256u || m <= 16u ? 1u : 2u;
  const uint32_t blocks = att_ceil(m, 16u * p.rb);
  p.wq = blocks <= 1u ? 1u : blocks <= 2u ? 2u : blocks <= 4u || p.dp < 256u ? 4u : 8u;
  p.small = ms <= 16u;
  const uint32_t rows = 16u * p.rb * p.wq, nrb = att_ceil(m, rows), nsb = p.small ? 1u : att_ceil(ms, rows);
  const uint32_t tp = att_ceil(P, ATT_TILE), ts = att_ceil(N, ATT_TILE);
  // Parts: the candidates fill the chip's places once or twice with the prefixes'
  // workgroups, or once with these and the suffixes'.
  const uint64_t jobs_p = (uint64_t)p.ng * KV * nrb, jobs_s = (uint64_t)p.ng * p.wb * KV * nsb;
  const uint64_t places = p.wq == 8u || p.dp == 256u ? 256u : 512u;
  const auto fit = [](uint64_t workgroups, uint64_t jobs, uint32_t tiles) {   // parts, evened out
    if (tiles == 0u) return 0u;
    const uint64_t most = workgroups / jobs;
    const uint32_t n = most < 1u ? 1u : most < tiles ? (uint32_t)most : tiles;
    return att_ceil(tiles, att_ceil(tiles, n));
  };
  uint64_t best = ~0ull;
  for (uint32_t s = 0; s < 3u; ++s) {
    const uint32_t ss = fit(s == 0u ? 0u : places * s / 2u, jobs_s, ts);
    for (uint32_t k = 0; k < 3u; ++k) {
      const uint64_t room_p = k < 2u ? places * (k + 1u) : places > jobs_s * ss ? places - jobs_s * ss : 0u;
      const uint32_t sp = fit(room_p, jobs_p, tp);
      const uint64_t t = att_time(jobs_p * sp, sp ? att_ceil(tp, sp) : 0u, jobs_s * ss, ss ? att_ceil(ts, ss) : 0u, places);
      // (a part more costs its join: a hundredth of a tile's time)
      const uint64_t cost = t * 100u + sp + ss;
      if (cost < best) best = cost, p.sp = sp, p.ss = ss;
    }
  }
  while (att_bytes((uint64_t)p.ng * p.wb * p.nt * H, p.sp + p.ss, p.dp) > ATT_SCRATCH && p.sp + p.ss > least) {
    if (p.sp >= p.ss) p.sp -= (p.sp + 7u) / 8u;   // (1 stays: sp > 1 where it is the larger of more than `least`)
    else p.ss -= (p.ss + 7u) / 8u;
  }
  p.slots = p.sp + p.ss;
  return p;
}

}  // namespace mxs
