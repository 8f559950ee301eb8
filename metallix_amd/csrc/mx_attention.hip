// mx_attention.hip -- attention of sequences that share a prefix
// (mxs_prefix_attention):
//
//   s[i] = scale q . keys[i],  lse = ln sum_i exp(s[i]),
//   out = sum_i exp(s[i] - lse) values[i],  weight[i] += exp(s[i] - lse)
//
// over the group's prefix and, causally, the row's suffix.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/mx_sampler.h"
#include "mxs_attention_checks.h"
#include "mxs_ctx.h"
#include "mxs_device.h"

namespace mxs {

constexpr size_t ATT_SCRATCH = 64u << 20;

struct AttArgs {
  const __bf16 *q, *pk, *pv, *k, *v;
  __bf16* out;
  uint64_t qr, qt, qh, pg, ph, pp, kr, kh, kp, orow, ot, oh;
  const int32_t *plen, *len;
  float *lse, *pw, *w;
  float* own;                // [rows][tokens][heads] lse of this slice
  uint32_t W, T, H, KV, D, P, N;
  uint32_t r0, nr, t0, nt;   // this slice: rows and tokens
  float scale;
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

// One workgroup a query: each wave takes every fourth position.
__global__ __launch_bounds__(256) void attention_simple_kernel(AttArgs A) {
  __shared__ float sm[4], sl[4], so[4][256];
  const uint32_t w = threadIdx.x >> 6, l = threadIdx.x & 63u;
  const uint32_t h = blockIdx.x % A.H, t = A.t0 + blockIdx.x / A.H % A.nt, r = A.r0 + blockIdx.x / A.H / A.nt;
  const uint32_t g = r / A.W, kv = h / (A.H / A.KV);
  const __bf16* const q = A.q + r * A.qr + t * A.qt + h * A.qh;
  const uint32_t P = att_len(A.plen, g, A.P), N = A.N ? att_seen(att_len(A.len, r, A.N), A.T, t) : 0u;
  const bool in = l * 4u < A.D;
  float qv[4] = {}, o[4] = {}, m = -INFINITY, sum = 0.0f;
  if (in)
    for (int j = 0; j < 4; ++j) qv[j] = (float)q[l * 4u + j];
  for (uint32_t i = w; i < P + N; i += 4u) {
    const bool pre = i < P;
    const uint64_t at = pre ? g * A.pg + kv * A.ph + (uint64_t)i * A.pp : r * A.kr + kv * A.kh + (uint64_t)(i - P) * A.kp;
    const __bf16* const kk = (pre ? A.pk : A.k) + at;
    const __bf16* const vv = (pre ? A.pv : A.v) + at;
    float s = 0.0f;
    if (in)
      for (int j = 0; j < 4; ++j) s += qv[j] * (float)kk[l * 4u + j];
    for (int x = 1; x < 64; x <<= 1) s += __shfl_xor(s, x);
    s *= A.scale;
    const float nm = fmaxf(m, s), base = nm == -INFINITY ? 0.0f : nm;
    const float a = expf(m - base), p = expf(s - base);
    sum = sum * a + p;
    if (in)
      for (int j = 0; j < 4; ++j) o[j] = o[j] * a + (p == 0.0f ? 0.0f : p * (float)vv[l * 4u + j]);
    m = nm;
  }
  if (l == 0) { sm[w] = m; sl[w] = sum; }
  for (int j = 0; j < 4; ++j) so[w][l * 4u + j] = o[j];
  __syncthreads();
  float M = -INFINITY, L = 0.0f;
  for (int x = 0; x < 4; ++x) M = fmaxf(M, sm[x]);
  const float base = M == -INFINITY ? 0.0f : M;
  for (int x = 0; x < 4; ++x) L += sl[x] * expf(sm[x] - base);
  if (threadIdx.x < A.D) {
    float v = 0.0f;
    for (int x = 0; x < 4; ++x) v += so[x][threadIdx.x] * expf(sm[x] - base);
    A.out[r * A.orow + t * A.ot + h * A.oh + threadIdx.x] = (__bf16)(L == 0.0f ? 0.0f : v / L);
  }
  if (threadIdx.x == 0) {
    const float lse = base + logf(L);
    if (A.lse) A.lse[((uint64_t)r * A.T + t) * A.H + h] = lse;
    A.own[blockIdx.x] = lse;
  }
}

// One thread a position.
template <bool PRE>
__global__ __launch_bounds__(256) void attention_weight_kernel(AttArgs A, uint32_t g0, uint32_t ng) {
  const uint32_t n = PRE ? A.P : A.N;
  const uint64_t id = (uint64_t)blockIdx.x * 256u + threadIdx.x;
  const uint32_t i = (uint32_t)(id % n), kv = (uint32_t)(id / n % A.KV), seg = (PRE ? g0 : A.r0) + (uint32_t)(id / n / A.KV);
  if (seg >= (PRE ? g0 + ng : A.r0 + A.nr)) return;
  const uint32_t len = PRE ? att_len(A.plen, seg, A.P) : att_len(A.len, seg, A.N);
  if (i >= len) return;
  const __bf16* const kk = PRE ? A.pk + seg * A.pg + kv * A.ph + (uint64_t)i * A.pp : A.k + seg * A.kr + kv * A.kh + (uint64_t)i * A.kp;
  const uint32_t ra = PRE ? max(seg * A.W, A.r0) : seg, rb = PRE ? min((seg + 1u) * A.W, A.r0 + A.nr) : seg + 1u, per = A.H / A.KV;
  float add = 0.0f;
  for (uint32_t r = ra; r < rb; ++r)
    for (uint32_t t = A.t0; t < A.t0 + A.nt; ++t) {
      if (!PRE && i >= att_seen(len, A.T, t)) continue;
      for (uint32_t h = kv * per; h < (kv + 1u) * per; ++h) {
        const __bf16* const q = A.q + r * A.qr + t * A.qt + h * A.qh;
        float s = 0.0f;
        for (uint32_t d = 0; d < A.D; ++d) s += (float)q[d] * (float)kk[d];
        const float lse = A.own[((uint64_t)(r - A.r0) * A.nt + t - A.t0) * A.H + h];
        s *= A.scale;
        if (lse != -INFINITY) add += expf(s - lse);
      }
    }
  float* const to = PRE ? &A.pw[((uint64_t)seg * A.KV + kv) * A.P + i] : &A.w[((uint64_t)seg * A.KV + kv) * A.N + i];
  *to += add;
}

size_t attention_scratch_bytes() { return ATT_SCRATCH; }

static void attention_slice(hipStream_t st, const AttArgs& A) {
  hipLaunchKernelGGL(attention_simple_kernel, dim3(A.nr * A.nt * A.H), dim3(256), 0, st, A);
  if (A.pw) {
    const uint32_t g0 = A.r0 / A.W, ng = (A.r0 + A.nr - 1u) / A.W + 1u - g0;
    hipLaunchKernelGGL(attention_weight_kernel<true>, dim3((uint32_t)(((uint64_t)ng * A.KV * A.P + 255u) / 256u)), dim3(256), 0, st, A, g0, ng);
  }
  if (A.w)
    hipLaunchKernelGGL(attention_weight_kernel<false>, dim3((uint32_t)(((uint64_t)A.nr * A.KV * A.N + 255u) / 256u)), dim3(256), 0, st, A, 0u, 0u);
}

}  // namespace mxs

extern "C" int mxs_prefix_attention(mxs_ctx* ctx, const mxs_attention* attention) {
  using namespace mxs;
  if (!ctx) return MXS_EINVAL;
  if (const char* m = attention_check(attention)) return fail(ctx, MXS_EINVAL, m);
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
  A.scale = a.scale;
  A.own = ctx->attention_scratch;
  int prev = 0;
  (void)hipGetDevice(&prev);
  if (prev != ctx->device) (void)hipSetDevice(ctx->device);
  // slices of whole rows, or of one row's tokens, whose queries fit the scratch and a launch
  const uint64_t most = 1u << 20;
  const uint32_t rows = a.groups * a.beams;
  const uint32_t nt = (uint32_t)(a.tokens < most / a.heads ? a.tokens : most / a.heads);
  const uint32_t nr = nt < a.tokens ? 1u : (uint32_t)(most / ((uint64_t)nt * a.heads));
  hipError_t e = hipSuccess;
  for (A.r0 = 0; A.r0 < rows && e == hipSuccess; A.r0 += nr)
    for (A.t0 = 0; A.t0 < a.tokens && e == hipSuccess; A.t0 += nt) {
      A.nr = rows - A.r0 < nr ? rows - A.r0 : nr;
      A.nt = a.tokens - A.t0 < nt ? a.tokens - A.t0 : nt;
      attention_slice(ctx->stream, A);
      e = hipGetLastError();
    }
  if (prev != ctx->device) (void)hipSetDevice(prev);
  if (e != hipSuccess) return hip_fail(ctx, e, "attention launch");
  return MXS_OK;
}
