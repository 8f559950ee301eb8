// mx_evict.hip -- caches brought down to a budget of positions
// (mxs_cache_evict): of each (layer, segment, head) the n best slots stay, by
// a key that puts the protected ones first and then goes by weight; those of
// them past n move into the slots before n that became free.
//
// The order of positions is given up for the traffic: a step that frees one slot moves
// one position, where closing the gap would move all behind it.  Sources lie from n on
// and targets below it, so a row's workgroups move their shares without waiting for
// one another; weights and positions go to other arrays, so that all can look at the
// old ones.  What it must do: read 8 bytes a slot, write 8, and read and write the
// positions that move.
//
// The n-th largest key comes digit by digit (11, 11, 10 bits) from counts in LDS, the
// keys in registers up to 32768 slots.  us (at 4.92 TB/s): 28 layers x 8 heads, 1025 to 1024
// slots, 10.5 (0.8: the chain of counts); 8192 to 2048 slots, 94 (82: HBM, 205 MB read and 204
// written); 2 x 8 caches of 131072 to 16384, 94 (55): 24 of it the three launches ahead
// of the moves, 140 without them, 877 when each digit took a look at all slots.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mx_sampler.h"
#include "mxs_attention_checks.h"
#include "mxs_ctx.h"
#include "mxs_device.h"

namespace mxs {

constexpr uint32_t EV_LAYERS = 64;   // layers a launch (their addresses travel as kernel arguments)
constexpr uint32_t EV_LIST = 1024;   // moves listed at a time

struct EvictArgs {
  mxs_cache cache[EV_LAYERS];
  const float* weight;
  const int32_t* index;
  const int32_t* lengths;
  float* weight_out;
  int32_t* index_out;
  int32_t* lengths_out;
  uint64_t ss, hs, ps;       // strides in bytes
  uint32_t S, H, C, bytes;   // segments, heads, capacity, bytes of a position
  uint32_t n, first, recent;
  uint32_t parts, jobs;      // workgroups a row, of all
  uint32_t list;             // entries of the list of slots in question
  // Where several workgroups share a long row, what earlier launches found:
  int32_t* newest;           // [rows * parts]
  uint32_t* counts;          // [rows * parts][EV_BINS] keys by first digit
  struct EvictFound* found;  // [rows]; NULL: nothing was found ahead
  unsigned long long* bits;  // [rows][words] slots with a first digit above the edge's
  uint2* lists;              // [rows][list] slots and keys with the edge's, in any order
};

struct EvictFound {
  uint32_t edge, need, same, count;   // the edge's first digit, how many of those that have it stay, how many there are; listed
};

typedef uint32_t ev_u32x4 __attribute__((ext_vector_type(4)));
typedef ev_u32x4 ev_u32x4_u __attribute__((aligned(1)));
typedef unsigned long long ev_u64_u __attribute__((aligned(1)));
typedef uint32_t ev_u32_u __attribute__((aligned(1)));
typedef uint16_t ev_u16_u __attribute__((aligned(1)));

// Ascending with the weight; NaN lowest, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = w == 0.0f ? 0u : __float_as_uint(w);
  if (w != w) return 0u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr uint32_t EV_BINS = 2048;   // values of a digit

template <int TH>
struct EvictSmem {
  union {
    uint32_t hist[EV_BINS];
    struct {
      uint32_t holes[EV_LIST], late[EV_LIST];
    };
  };
  uint32_t wave[TH / 64];
  uint32_t pick[3];          // the digit, how many are left to take within it, how many have it
};

// Sum over the threads before this one; total: over all.
template <int TH>
__device__ uint32_t before_me(EvictSmem<TH>& S, uint32_t v, uint32_t& total) {
  const uint32_t sc = wave_scan_u32(v), w = threadIdx.x >> 6;
  if ((threadIdx.x & 63u) == 63u) S.wave[w] = sc;
  __syncthreads();
  uint32_t base = 0u;
  total = 0u;
  for (uint32_t i = 0; i < TH / 64u; ++i) {
    if (i < w) base += S.wave[i];
    total += S.wave[i];
  }
  __syncthreads();
  return base + sc - v;
}

// The digit of the `need`-th largest, from the digits' counts; need becomes how
// many to take of those that have it, same how many there are.
template <int TH>
__device__ uint32_t pick_digit(EvictSmem<TH>& S, uint32_t& need, uint32_t& same) {
  constexpr uint32_t B = EV_BINS / TH;
  uint32_t c[B], sum = 0u, total;   // the thread's digits, largest first
#pragma unroll
  for (uint32_t j = 0; j < B; ++j) sum += c[j] = S.hist[EV_BINS - 1u - threadIdx.x * B - j];
  uint32_t before = before_me<TH>(S, sum, total);
#pragma unroll
  for (uint32_t j = 0; j < B; ++j) {
    if (before < need && before + c[j] >= need) {
      S.pick[0] = EV_BINS - 1u - threadIdx.x * B - j;
      S.pick[1] = need - before;
      S.pick[2] = c[j];
    }
    before += c[j];
  }
  __syncthreads();
  need = S.pick[1], same = S.pick[2];
  return S.pick[0];
}

// One digit: f(count) calls count(digit) for each key that is still in question.
template <int TH, typename F>
__device__ uint32_t next_digit(EvictSmem<TH>& S, uint32_t& need, uint32_t& same, F f) {
  for (uint32_t i = threadIdx.x; i < EV_BINS; i += TH) S.hist[i] = 0u;
  __syncthreads();
  f([&](uint32_t digit) { atomicAdd(&S.hist[digit], 1u); });
  __syncthreads();
  return pick_digit<TH>(S, need, same);
}

__device__ __forceinline__ void copy_piece(char* to, const char* from, uint32_t have) {
  if (have >= 16u) {
    *reinterpret_cast<ev_u32x4_u*>(to) = *reinterpret_cast<const ev_u32x4_u*>(from);
    return;
  }
  if (have & 8u) { *reinterpret_cast<ev_u64_u*>(to) = *reinterpret_cast<const ev_u64_u*>(from); to += 8; from += 8; }
  if (have & 4u) { *reinterpret_cast<ev_u32_u*>(to) = *reinterpret_cast<const ev_u32_u*>(from); to += 4; from += 4; }
  if (have & 2u) { *reinterpret_cast<ev_u16_u*>(to) = *reinterpret_cast<const ev_u16_u*>(from); to += 2; from += 2; }
  if (have & 1u) *to = *from;
}

__device__ __forceinline__ uint32_t evict_len(const EvictArgs& A, uint32_t seg) {
  const int32_t n = A.lengths ? A.lengths[seg] : (int32_t)A.C;
  return n <= 0 ? 0u : min((uint32_t)n, A.C);
}
__device__ __forceinline__ uint32_t slot_key(const EvictArgs& A, int32_t recent_from, float w, int32_t p) {
  return p < (int32_t)A.first || p > recent_from ? 0xffffffffu : weight_key(w);
}

// Long rows that several workgroups share would each be looked at whole by all of
// them, three times (131072 slots: 26 us a look).  Instead every workgroup looks
// at its own slots: STEP 0 finds the newest position, 1 counts the keys' first
// digits, 2 marks what lies above the edge's digit and lists what has it.  (Weights
// share few first digits, sign, exponent and two bits of the rest, so that the counts of
// 1 meet in LDS banks: 68% of its LDS cycles, of 7 us.)
template <int STEP>
__global__ __launch_bounds__(1024) void evict_ahead_kernel(EvictArgs A) {
  constexpr uint32_t TH = 1024u;
  extern __shared__ unsigned long long room[];
  __shared__ EvictSmem<1024> S;
  const uint32_t job = (blockIdx.x & 7u) * (gridDim.x / 8u) + (blockIdx.x >> 3), tid = threadIdx.x;
  if (job >= A.jobs) return;
  const uint32_t part = job % A.parts, row = job / A.parts, len = evict_len(A, row / A.H % A.S);
  if (len <= A.n) return;
  const uint32_t span = ((len + A.parts - 1u) / A.parts + 63u) / 64u * 64u, sa = min(len, part * span), sb = min(len, sa + span);
  const uint64_t at = (uint64_t)row * A.C;
  const float* const weight = A.weight + at;
  const int32_t* const index = A.index ? A.index + at : nullptr;
  if (STEP == 0) {
    int32_t newest = -1;
#pragma unroll 8
    for (uint32_t i = sa + tid; i < sb; i += TH) newest = max(newest, index[i]);
    for (int x = 1; x < 64; x <<= 1) newest = max(newest, __shfl_xor(newest, x));
    if ((tid & 63u) == 0u) S.wave[tid >> 6] = (uint32_t)newest;
    __syncthreads();
    if (tid == 0) {
      for (uint32_t i = 1; i < TH / 64u; ++i) newest = max(newest, (int32_t)S.wave[i]);
      A.newest[job] = newest;
    }
    return;
  }
  int32_t recent_from = INT32_MAX;
  if (A.recent) {
    int32_t newest = index ? -1 : (int32_t)len - 1;
    if (index)
      for (uint32_t i = 0; i < A.parts; ++i) newest = max(newest, A.newest[row * A.parts + i]);   // (uniform)
    recent_from = newest - (int32_t)A.recent;
  }
  uint32_t need = A.n, same = 0u, edge = 0u;
  uint2* const list = reinterpret_cast<uint2*>(room);
  for (uint32_t i = tid; i < EV_BINS; i += TH) {
    uint32_t c = 0u;
    if (STEP == 2)
#pragma unroll 8
      for (uint32_t x = 0; x < A.parts; ++x) c += A.counts[(uint64_t)(row * A.parts + x) * EV_BINS + i];
    S.hist[i] = c;
  }
  if (STEP == 1 && part == 0 && tid == 0) A.found[row].count = 0u;
  __syncthreads();
  if (STEP == 2) {
    edge = pick_digit<1024>(S, need, same);
    __syncthreads();
    if (tid == 0) {
      if (part == 0) A.found[row].edge = edge, A.found[row].need = need, A.found[row].same = same;
      S.wave[0] = 0u;
    }
    __syncthreads();
    if (same > A.list) return;   // (more than a list holds: the last launch looks at all of the row)
  }
  constexpr int U = 8;
  for (uint32_t i0 = sa; i0 < sb; i0 += U * TH) {
    float w[U];
    int32_t p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = min(i0 + u * TH + tid, sb - 1u);
      w[u] = weight[i];
      p[u] = index ? index[i] : (int32_t)i;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = i0 + u * TH + tid, k = slot_key(A, recent_from, w[u], p[u]);
      if (STEP == 1) {
        if (i < sb) atomicAdd(&S.hist[k >> 21], 1u);
      } else {
        const unsigned long long b = __builtin_amdgcn_ballot_w64(i < sb && k >> 21 > edge);
        if ((tid & 63u) == 0u && i < sb) A.bits[(uint64_t)row * ((A.C + 63u) / 64u) + (i >> 6)] = b;
        if (i < sb && k >> 21 == edge) list[atomicAdd(&S.wave[0], 1u)] = make_uint2(i, k);
      }
    }
  }
  __syncthreads();
  if (STEP == 1) {
    for (uint32_t i = tid; i < EV_BINS; i += TH) A.counts[(uint64_t)job * EV_BINS + i] = S.hist[i];
    return;
  }
  const uint32_t count = S.wave[0];
  if (tid == 0) S.wave[1] = atomicAdd(&A.found[row].count, count);
  __syncthreads();
  for (uint32_t i = tid; i < count; i += TH) A.lists[(uint64_t)row * A.list + S.wave[1] + i] = list[i];
}

// A row (layer, segment, head) and one of its parts a workgroup; KR: the keys
// a thread holds, 0 where there are more than registers hold and they are worked out
// again for each look.
template <int TH, int KR>
__global__ __launch_bounds__(TH) void evict_kernel(EvictArgs A) {
  extern __shared__ unsigned long long kept[];   // a bit a slot
  __shared__ EvictSmem<TH> S;
  // XCD x (workgroups go to the XCDs in turn) takes a contiguous range of the
  // rows, so that a row's parts read its weights from one L2.
  const uint32_t job = (blockIdx.x & 7u) * (gridDim.x / 8u) + (blockIdx.x >> 3);
  if (job >= A.jobs) return;
  const uint32_t tid = threadIdx.x, part = job % A.parts, row = job / A.parts;
  const uint32_t h = row % A.H, seg = row / A.H % A.S, layer = row / A.H / A.S, n = A.n;
  const uint32_t len = evict_len(A, seg), now = min(len, n);
  const uint64_t at = (uint64_t)row * A.C;
  const float* const weight = A.weight + at;
  const int32_t* const index = A.index ? A.index + at : nullptr;
  float* const weight_out = A.weight_out + at;
  int32_t* const index_out = A.index_out ? A.index_out + at : nullptr;
  if (A.lengths_out && layer == 0 && h == 0 && part == 0 && tid == 0) A.lengths_out[seg] = (int32_t)now;
  // this part's slots
  const uint32_t span = (A.C + A.parts - 1u) / A.parts, sa = part * span, sb = min(A.C, sa + span);
  for (uint32_t i = max(sa, now) + tid; i < sb; i += TH) {
    weight_out[i] = 0.0f;
    if (index_out) index_out[i] = -1;
  }
  if (len <= n) {
    for (uint32_t i = sa + tid; i < min(sb, now); i += TH) {
      weight_out[i] = weight[i];
      if (index_out) index_out[i] = index ? index[i] : (int32_t)i;
    }
    return;
  }
  // The slots' keys: the protected ones above all, then by weight.
  int32_t recent_from = INT32_MAX;   // positions past it are protected (budget < len: 20 bits)
  auto key_of = [&](float w, int32_t p) { return slot_key(A, recent_from, w, p); };
  constexpr int U = KR ? KR : 8;     // slots in flight
  uint32_t keys[U];
  int32_t where[U];
  auto load = [&](uint32_t i0, float (&w)[U], int32_t (&p)[U]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = min(i0 + u * TH + tid, len - 1u);
      w[u] = weight[i];
      p[u] = index ? index[i] : (int32_t)i;
    }
  };
  float held[U];
  if (KR) load(0u, held, where);
  // (a row that was listed ahead is not looked at again)
  const bool ahead = KR == 0 && A.found && A.found[row].same <= A.list;
  if (A.recent && !ahead) {
    int32_t newest = index ? -1 : (int32_t)len - 1;
    if (index) {
      if (KR) {
#pragma unroll
        for (int u = 0; u < U; ++u) newest = max(newest, where[u]);
      } else {
#pragma unroll 8
        for (uint32_t i = tid; i < len; i += TH) newest = max(newest, index[i]);
      }
    }
    for (int x = 1; x < 64; x <<= 1) newest = max(newest, __shfl_xor(newest, x));
    if ((tid & 63u) == 0u) S.wave[tid >> 6] = (uint32_t)newest;
    __syncthreads();
    for (uint32_t i = 0; i < TH / 64u; ++i) newest = max(newest, (int32_t)S.wave[i]);
    __syncthreads();
    recent_from = newest - (int32_t)A.recent;
  }
  if (KR) {
#pragma unroll
    for (int u = 0; u < U; ++u) keys[u] = key_of(held[u], where[u]);
  }
  // f(slot, key, valid) for all slots of a whole number of waves.
  auto each = [&](auto f) __attribute__((always_inline)) {
    if (KR) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if ((uint32_t)u * TH < len) f(u * TH + tid, keys[u], u * TH + tid < len);
    } else {
      for (uint32_t i0 = 0; i0 < len; i0 += U * TH) {
        float w[U];
        int32_t p[U];
        load(i0, w, p);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (i0 + u * TH < len) f(i0 + u * TH + tid, key_of(w[u], p[u]), i0 + u * TH + tid < len);
      }
    }
  };
  // The n-th largest key, 11, 11 and 10 bits at a time, and of the slots that
  // have it the need-th lowest.
  uint32_t need = n, same, edge = 0u, last = ~0u;
  auto round = [&](uint32_t r, auto each_one) {
    const uint32_t shift = r == 0u ? 21u : r == 1u ? 10u : 0u, bits = r == 2u ? 10u : 11u;
    const uint32_t above = shift + bits;   // the digits found so far
    edge |= next_digit<TH>(S, need, same, [&](auto count) {
      each_one([&](uint32_t, uint32_t k, bool valid) {
        if (valid && (above == 32u || k >> above == edge >> above)) count(k >> shift & ((1u << bits) - 1u));
      });
    }) << shift;
  };
  auto settle = [&](auto each_one) {
    if (need >= same) return;
    uint32_t low = 0u;   // of ~slot's 20 bits
#pragma unroll 1
    for (uint32_t r = 0; r < 2u; ++r) {
      const uint32_t shift = r == 0u ? 10u : 0u;
      low |= next_digit<TH>(S, need, same, [&](auto count) {
        each_one([&](uint32_t i, uint32_t k, bool valid) {
          const uint32_t c = ~i & 0xfffffu;
          if (valid && k == edge && (r == 0u || c >> 10 == low >> 10)) count(c >> shift & 0x3ffu);
        });
      }) << shift;
    }
    last = ~low & 0xfffffu;
  };
  if (ahead) {
    edge = A.found[row].edge << 21, need = A.found[row].need, same = A.found[row].same;
  } else {
    round(0u, each);
  }
  if (KR == 0 && same <= A.list) {
    // The slots with the edge's first digit go into a list, and the rest is done
    // on that: two looks at all slots instead of four or more.
    uint2* const list = reinterpret_cast<uint2*>(kept + (A.C + 63u) / 64u);
    uint32_t count = same;
    if (ahead) {
      const uint32_t words = (A.C + 63u) / 64u;
      for (uint32_t i = tid; i < (len + 63u) / 64u; i += TH) kept[i] = A.bits[(uint64_t)row * words + i];
      for (uint32_t i = tid; i < count; i += TH) list[i] = A.lists[(uint64_t)row * A.list + i];
    } else {
      if (tid == 0) S.wave[0] = 0u;
      __syncthreads();
      each([&](uint32_t i, uint32_t k, bool valid) {
        const unsigned long long b = __builtin_amdgcn_ballot_w64(valid && k >> 21 > edge >> 21);
        if ((tid & 63u) == 0u && i < len) kept[i >> 6] = b;
        if (valid && k >> 21 == edge >> 21) list[atomicAdd(&S.wave[0], 1u)] = make_uint2(i, k);
      });
    }
    __syncthreads();
    auto listed = [&](auto f) {
      for (uint32_t x = tid; x < count; x += TH) f(list[x].x, list[x].y, true);
    };
    round(1u, listed);
    round(2u, listed);
    settle(listed);
    listed([&](uint32_t i, uint32_t k, bool) {
      if (k > edge || (k == edge && i <= last)) atomicOr(&kept[i >> 6], 1ull << (i & 63u));
    });
  } else {
    round(1u, each);
    round(2u, each);
    settle(each);
    each([&](uint32_t i, uint32_t k, bool valid) {
      const unsigned long long b = __builtin_amdgcn_ballot_w64(valid && (k > edge || (k == edge && i <= last)));
      if ((tid & 63u) == 0u && i < len) kept[i >> 6] = b;   // (a wave's slots: 64 consecutive ones)
    });
  }
  __syncthreads();
  for (uint32_t i = sa + tid; i < min(sb, n); i += TH)
    if (kept[i >> 6] >> (i & 63u) & 1u) {
      weight_out[i] = weight[i];
      if (index_out) index_out[i] = index ? index[i] : (int32_t)i;
    }
  // Each thread takes some units of 2^us slots; their free slots below n and kept
  // ones from n on, counted.
  uint32_t us = 0u;
  while (us < 6u && (len + (1u << us) - 1u) >> us > TH) ++us;
  const uint32_t units = (len + (1u << us) - 1u) >> us, own = (units + TH - 1u) / TH;
  const uint32_t ua = min(tid * own, units), ub = min(ua + own, units), unit = 1u << us;
  auto bits_of = [&](uint32_t x) { return kept[x << us >> 6] >> (x << us & 63u) & (unit == 64u ? ~0ull : (1ull << unit) - 1ull); };
  auto below = [&](uint32_t x) {   // of the unit's slots those below n
    const uint32_t s = x << us;
    return s >= n ? 0ull : n - s >= unit ? (unit == 64u ? ~0ull : (1ull << unit) - 1ull) : (1ull << (n - s)) - 1ull;
  };
  auto free_of = [&](uint32_t x) { return ~bits_of(x) & below(x); };
  auto late_of = [&](uint32_t x) { return bits_of(x) & ~below(x); };
  uint32_t nf = 0u, nl = 0u, moves, all;
  for (uint32_t x = ua; x < ub; ++x) {
    nf += __builtin_popcountll(free_of(x));
    nl += __builtin_popcountll(late_of(x));
  }
  // (both counts at once where they fit: fewer than 2^16 slots)
  uint32_t f0, m0;
  if (len < 1u << 16) {
    const uint32_t both = before_me<TH>(S, nl << 16 | nf, all);
    f0 = both & 0xffffu, m0 = both >> 16, moves = all >> 16;
  } else {
    f0 = before_me<TH>(S, nf, all);
    m0 = before_me<TH>(S, nl, moves);
  }
  const uint32_t share = (moves + A.parts - 1u) / A.parts, ja = min(moves, part * share), jb = min(moves, ja + share);
  const mxs_cache c = A.cache[layer];
  const uint64_t off = seg * A.ss + h * A.hs;
  char* const ck = reinterpret_cast<char*>(c.keys) + off;
  char* const cv = c.values ? reinterpret_cast<char*>(c.values) + off : nullptr;
  const uint32_t pieces = (A.bytes + 15u) / 16u, both = cv ? 2u * pieces : pieces;
  const uint32_t bb = min(both, (uint32_t)TH), ppi = TH / bb, k0 = tid / bb, p0 = tid - k0 * bb;   // this thread's pairs and piece
  for (uint32_t j = ja; j < jb; j += EV_LIST) {
    const uint32_t m = min(EV_LIST, jb - j);
    auto list = [&](uint32_t rank, uint32_t count, uint32_t* to, auto bits) {
      if (rank >= j + m || rank + count <= j) return;
      for (uint32_t x = ua; x < ub; ++x)
        for (unsigned long long b = bits(x); b; b &= b - 1ull, ++rank)
          if (rank >= j && rank < j + m) to[rank - j] = (x << us) + (uint32_t)__builtin_ctzll(b);
    };
    list(f0, nf, S.holes, free_of);
    list(m0, nl, S.late, late_of);
    __syncthreads();
    for (uint32_t i = tid; i < m; i += TH) {
      const uint32_t to = S.holes[i], from = S.late[i];
      weight_out[to] = weight[from];
      if (index_out) index_out[to] = index ? index[from] : (int32_t)from;
    }
    if (k0 < ppi)
      for (uint32_t p = p0; p < both; p += bb) {
        char* const base = (p < pieces ? ck : cv) + (p < pieces ? p : p - pieces) * 16u;
        const uint32_t have = A.bytes - (p < pieces ? p : p - pieces) * 16u;
        if (have >= 16u) {
          constexpr uint32_t V = 4;   // loads in flight
          for (uint32_t k = k0; k < m; k += V * ppi) {
            ev_u32x4 v[V];
#pragma unroll
            for (uint32_t x = 0; x < V; ++x) v[x] = *reinterpret_cast<const ev_u32x4_u*>(base + S.late[min(k + x * ppi, m - 1u)] * A.ps);
#pragma unroll
            for (uint32_t x = 0; x < V; ++x)
              if (k + x * ppi < m) *reinterpret_cast<ev_u32x4_u*>(base + S.holes[k + x * ppi] * A.ps) = v[x];
          }
        } else {
          for (uint32_t k = k0; k < m; k += ppi) copy_piece(base + S.holes[k] * A.ps, base + S.late[k] * A.ps, have);
        }
      }
    __syncthreads();
  }
}

template <int TH, int KR>
static hipError_t evict_go(mxs_ctx* ctx, uint32_t rows, EvictArgs& A) {
  const hipStream_t st = ctx->stream;
  const uint32_t words = (A.C + 63u) / 64u, room = (148u << 10) - words * 8u;   // (of 160 KB, less the rest)
  A.list = KR ? 0u : room / 8u < 8192u ? room / 8u : 8192u;
  const uint32_t lds = words * 8u + A.list * 8u;
  hipError_t e = hipSuccess;
  if (lds > 32u << 10) e = hipFuncSetAttribute((const void*)evict_kernel<TH, KR>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  if (e != hipSuccess) return e;
  A.parts = rows >= 256u ? 1u : 256u / rows;   // a workgroup a CU
  A.jobs = rows * A.parts;
  const dim3 grid((A.jobs + 7u) / 8u * 8u);
  if (KR == 0 && A.parts > 1u) {
    // (at most 128 rows: 2 MB of counts, 17 MB of bits and 8 MB of lists)
    char* at = reinterpret_cast<char*>(ctx->attention_scratch);
    auto take = [&](uint64_t bytes) {
      char* const p = at;
      at += (bytes + 255u) / 256u * 256u;
      return p;
    };
    A.counts = reinterpret_cast<uint32_t*>(take((uint64_t)A.jobs * EV_BINS * 4u));
    A.newest = reinterpret_cast<int32_t*>(take(A.jobs * 4u));
    A.found = reinterpret_cast<EvictFound*>(take(rows * sizeof(EvictFound)));
    A.bits = reinterpret_cast<unsigned long long*>(take((uint64_t)rows * words * 8u));
    A.lists = reinterpret_cast<uint2*>(take((uint64_t)rows * A.list * 8u));
    if ((uint64_t)(at - reinterpret_cast<char*>(ctx->attention_scratch)) > attention_scratch_bytes()) return hipErrorOutOfMemory;
    const uint32_t lds2 = A.list * 8u;
    e = hipFuncSetAttribute((const void*)evict_ahead_kernel<2>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds2);
    if (e != hipSuccess) return e;
    if (A.index && A.recent) hipLaunchKernelGGL(evict_ahead_kernel<0>, grid, dim3(1024), 0, st, A);
    hipLaunchKernelGGL(evict_ahead_kernel<1>, grid, dim3(1024), 0, st, A);
    hipLaunchKernelGGL(evict_ahead_kernel<2>, grid, dim3(1024), lds2, st, A);
  }
  hipLaunchKernelGGL((evict_kernel<TH, KR>), grid, dim3(TH), lds, st, A);
  return hipGetLastError();
}

}  // namespace mxs

extern "C" int mxs_cache_evict(mxs_ctx* ctx, const mxs_evict* evict) {
  using namespace mxs;
  if (!ctx) return MXS_EINVAL;
  if (const char* m = evict_check(evict)) return fail(ctx, MXS_EINVAL, m);
  const mxs_evict& v = *evict;
  if (v.layers == 0 || v.segments == 0 || v.heads == 0) return MXS_OK;
  int prev = 0;
  (void)hipGetDevice(&prev);
  if (prev != ctx->device) (void)hipSetDevice(ctx->device);
  hipError_t e = hipSuccess;
  const uint64_t a_layer = (uint64_t)v.segments * v.heads;
  for (uint32_t first = 0; first < v.layers && e == hipSuccess; first += EV_LAYERS) {
    const uint32_t here = v.layers - first < EV_LAYERS ? v.layers - first : EV_LAYERS;
    EvictArgs A{};
    for (uint32_t i = 0; i < here; ++i) A.cache[i] = v.caches[first + i];
    const uint64_t skip = first * a_layer * v.capacity;
    A.weight = v.weight + skip;
    A.index = v.index ? v.index + skip : nullptr;
    A.lengths = v.lengths;
    A.weight_out = v.weight_out + skip;
    A.index_out = v.index_out ? v.index_out + skip : nullptr;
    A.lengths_out = first == 0 ? v.lengths_out : nullptr;
    A.ss = v.segment_stride, A.hs = v.head_stride, A.ps = v.position_stride;
    A.S = v.segments, A.H = v.heads, A.C = v.capacity, A.bytes = v.position_bytes;
    A.n = v.budget, A.first = v.keep_first, A.recent = v.keep_recent;
    const uint32_t rows = (uint32_t)(here * a_layer);
    if (A.C <= 2048u) e = evict_go<512, 4>(ctx, rows, A);
    else if (A.C <= 8192u) e = evict_go<1024, 8>(ctx, rows, A);
    else if (A.C <= 32768u) e = evict_go<1024, 32>(ctx, rows, A);
    else e = evict_go<1024, 0>(ctx, rows, A);
  }
  if (prev != ctx->device) (void)hipSetDevice(prev);
  if (e != hipSuccess) return hip_fail(ctx, e, "evict_kernel launch");
  return MXS_OK;
}
