// mx_evict.hip -- caches brought down to a budget of positions
// (mxs_cache_evict): of each (layer, segment, head) the n best slots stay, by
// a key that puts the protected ones first and then goes by weight; those of
// them past n move into the slots before n that became free.
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
  uint32_t parts;            // workgroups a row
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

template <int TH>
struct EvictSmem {
  uint32_t hist[256];
  uint32_t wave[TH / 64];
  uint32_t pick[2];          // the digit, how many are left to take within it
  uint32_t holes[EV_LIST], late[EV_LIST];
};

// The `need`-th largest of f(slot) over the slots, digit by digit from bit
// `top` on down, among the slots where f is true.  f(slot, &key).  On return
// need is how many of the keys equal to the result are among the first `need`.
template <int TH, typename F>
__device__ uint32_t nth_largest(EvictSmem<TH>& S, uint32_t len, uint32_t& need, F f) {
  uint32_t prefix = 0u;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (uint32_t i = threadIdx.x; i < 256u; i += TH) S.hist[i] = 0u;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < len; i += TH) {
      uint32_t key;
      if (!f(i, key)) continue;
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&S.hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 64u) {   // lane l holds digits 255 - 4 l down
      uint32_t c[4], sum = 0u;
      for (int j = 0; j < 4; ++j) sum += c[j] = S.hist[255u - 4u * threadIdx.x - j];
      uint32_t before = wave_scan_u32(sum) - sum;
      for (int j = 0; j < 4; ++j) {
        if (before < need && before + c[j] >= need) {
          S.pick[0] = 255u - 4u * threadIdx.x - j;
          S.pick[1] = need - before;
        }
        before += c[j];
      }
    }
    __syncthreads();
    prefix |= S.pick[0] << shift;
    need = S.pick[1];
    __syncthreads();
  }
  return prefix;
}

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

template <int TH>
__global__ __launch_bounds__(TH) void evict_kernel(EvictArgs A) {
  extern __shared__ unsigned long long kept[];   // a bit a slot
  __shared__ EvictSmem<TH> S;
  const uint32_t tid = threadIdx.x, part = blockIdx.x % A.parts, row = blockIdx.x / A.parts;   // row: (layer, segment, head)
  const uint32_t h = row % A.H, seg = row / A.H % A.S, layer = row / A.H / A.S, n = A.n;
  const int32_t l0 = A.lengths ? A.lengths[seg] : (int32_t)A.C;
  const uint32_t len = l0 <= 0 ? 0u : min((uint32_t)l0, A.C), now = min(len, n);
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
  int64_t recent_from = INT64_MAX;   // positions past it are protected
  if (A.recent) {
    int32_t newest = index ? -1 : (int32_t)len - 1;
    if (index)
      for (uint32_t i = tid; i < len; i += TH) newest = max(newest, index[i]);
    for (int x = 1; x < 64; x <<= 1) newest = max(newest, __shfl_xor(newest, x));
    if ((tid & 63u) == 0u) S.wave[tid >> 6] = (uint32_t)newest;
    __syncthreads();
    for (uint32_t i = 0; i < TH / 64u; ++i) newest = max(newest, (int32_t)S.wave[i]);
    __syncthreads();
    recent_from = (int64_t)newest - A.recent;
  }
  auto key_of = [&](uint32_t i) {
    const int64_t p = index ? index[i] : (int32_t)i;
    if (p < (int64_t)A.first || p > recent_from) return 0xffffffffu;
    return weight_key(weight[i]);
  };
  uint32_t need = n;
  const uint32_t edge = nth_largest<TH>(S, len, need, [&](uint32_t i, uint32_t& k) { k = key_of(i); return true; });
  // of the slots with the edge's key the `need` lowest: down to the need-th largest ~slot
  const uint32_t last = ~nth_largest<TH>(S, len, need, [&](uint32_t i, uint32_t& k) { k = ~i; return key_of(i) == edge; });
  const uint32_t words = (len + 63u) / 64u;
  for (uint32_t i = tid; i < words * 64u; i += TH) {
    const uint32_t k = i < len ? key_of(i) : 0u;
    const unsigned long long b = __builtin_amdgcn_ballot_w64(i < len && (k > edge || (k == edge && i <= last)));
    if ((tid & 63u) == 0u) kept[i >> 6] = b;
  }
  __syncthreads();
  for (uint32_t i = sa + tid; i < min(sb, n); i += TH)
    if (kept[i >> 6] >> (i & 63u) & 1u) {
      weight_out[i] = weight[i];
      if (index_out) index_out[i] = index ? index[i] : (int32_t)i;
    }
  // Each thread takes some words; their free slots below n and kept ones from n on, counted.
  const uint32_t own = (words + TH - 1u) / TH, wa = min(tid * own, words), wb = min(wa + own, words);
  auto free_of = [&](uint32_t w) {
    const uint32_t s = w * 64u;
    return s >= n ? 0ull : ~kept[w] & (n - s >= 64u ? ~0ull : (1ull << (n - s)) - 1ull);
  };
  auto late_of = [&](uint32_t w) {
    const uint32_t s = w * 64u;
    return s + 64u <= n ? 0ull : s >= n ? kept[w] : kept[w] & ~((1ull << (n - s)) - 1ull);
  };
  uint32_t nf = 0u, nl = 0u, moves, same;
  for (uint32_t w = wa; w < wb; ++w) {
    nf += __builtin_popcountll(free_of(w));
    nl += __builtin_popcountll(late_of(w));
  }
  const uint32_t f0 = before_me<TH>(S, nf, same), m0 = before_me<TH>(S, nl, moves);
  const uint32_t share = (moves + A.parts - 1u) / A.parts, ja = part * share, jb = min(moves, ja + share);
  const mxs_cache c = A.cache[layer];
  const uint64_t off = seg * A.ss + h * A.hs;
  char* const ck = reinterpret_cast<char*>(c.keys) + off;
  char* const cv = c.values ? reinterpret_cast<char*>(c.values) + off : nullptr;
  const uint32_t pieces = (A.bytes + 15u) / 16u, both = cv ? 2u * pieces : pieces;
  for (uint32_t j = ja; j < jb; j += EV_LIST) {
    const uint32_t m = min(EV_LIST, jb - j);
    auto list = [&](uint32_t rank, uint32_t count, uint32_t* to, auto bits_of) {
      if (rank >= j + m || rank + count <= j) return;
      for (uint32_t w = wa; w < wb; ++w)
        for (unsigned long long b = bits_of(w); b; b &= b - 1ull, ++rank)
          if (rank >= j && rank < j + m) to[rank - j] = w * 64u + (uint32_t)__builtin_ctzll(b);
    };
    list(f0, nf, S.holes, free_of);
    list(m0, nl, S.late, late_of);
    __syncthreads();
    for (uint32_t i = tid; i < m; i += TH) {
      const uint32_t to = S.holes[i], from = S.late[i];
      weight_out[to] = weight[from];
      if (index_out) index_out[to] = index ? index[from] : (int32_t)from;
    }
    for (uint32_t i = tid; i < m * both; i += TH) {
      const uint32_t k = i / both, p = i - k * both;
      char* const base = p < pieces ? ck : cv;
      const uint32_t pc = (p < pieces ? p : p - pieces) * 16u;
      copy_piece(base + S.holes[k] * A.ps + pc, base + S.late[k] * A.ps + pc, A.bytes - pc);
    }
    __syncthreads();
  }
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
    A.parts = rows >= 256u ? 1u : 256u / rows;
    const uint32_t lds = (A.C + 63u) / 64u * 8u;
    if (lds > 32u << 10)
      e = hipFuncSetAttribute((const void*)evict_kernel<1024>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) break;
    hipLaunchKernelGGL(evict_kernel<1024>, dim3(rows * A.parts), dim3(1024), lds, ctx->stream, A);
    e = hipGetLastError();
  }
  if (prev != ctx->device) (void)hipSetDevice(prev);
  if (e != hipSuccess) return hip_fail(ctx, e, "evict_kernel launch");
  return MXS_OK;
}
