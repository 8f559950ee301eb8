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
  p.wq = blocks <= 1u ? 1u : blocks <= 2u ? 2u : blocks <= 4u ? 4u : 8u;
  p.small = ms <= 16u;
  const uint32_t rows = 16u * p.rb * p.wq, nrb = att_ceil(m, rows), nsb = p.small ? 1u : att_ceil(ms, rows);
  const uint32_t tp = att_ceil(P, ATT_TILE), ts = att_ceil(N, ATT_TILE);
  // Tiles of a part: so many that the parts fill the chip about once.
  const uint64_t jobs_p = (uint64_t)p.ng * KV * nrb, jobs_s = (uint64_t)p.ng * p.wb * KV * nsb;
  const uint64_t target = p.wq == 8u || p.dp == 256u ? 256u : 512u;
  uint32_t each = att_ceil(jobs_p * tp + jobs_s * ts, target);
  if (each < 1u) each = 1u;
  for (;; each += each / 8u + 1u) {
    p.sp = att_ceil(tp, each), p.ss = att_ceil(ts, each);
    p.slots = p.sp + p.ss;
    if (each >= tp && each >= ts) break;
    if (att_bytes((uint64_t)p.ng * p.wb * p.nt * H, p.slots, p.dp) <= ATT_SCRATCH) break;
  }
  return p;
}

}  // namespace mxs
