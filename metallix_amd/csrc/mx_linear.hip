// mx_linear.hip -- a bf16 matrix product with bias, activation and residual
// in its epilogue (mxs_linear_bf16):
//
//   out[r][o] = act(sum_k x[r][k] weight[o][k] + bias[o]) + residual[r][o]
//
// Products and sums on v_mfma_f32_16x16x32_bf16 (f32 accumulators), the
// epilogue in f32, one rounding to the output type.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/mx_sampler.h"
#include "mxs_checks.h"
#include "mxs_ctx.h"

namespace mxs {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct LinArgs {
  const __bf16* x;
  const __bf16* w;
  const void* bias;
  const void* res;
  void* out;
  uint64_t xs, ws, rs, os;   // strides in elements
  uint32_t R, K, N;
  int32_t act, out_f32, bias_f32;
  int32_t vec;               // out and residual take 4-element accesses
};

// exp(-y) for the sigmoid, to about 2 ulp: exp2 of fl(-y log2(e)), corrected
// by the argument's rounding.  -y above 89 overflows to inf, the sigmoid's 0.
__device__ __forceinline__ float exp_minus(float y) {
  const float t = -y * 1.44269504f;
  const float r = __builtin_fmaf(t, -0.693147182f, -y);
  const float e = __builtin_amdgcn_exp2f(t);
  return fabsf(t) < 126.0f ? __builtin_fmaf(e, r, e) : e;
}

__device__ __forceinline__ float activate(float y, int32_t act) {
  switch (act) {   // uniform
    case MXS_ACT_RELU: return y < 0.0f ? 0.0f : y;   // (a NaN stays)
    case MXS_ACT_SILU: return y / (1.0f + exp_minus(y));
    case MXS_ACT_GELU: return 0.5f * y * (1.0f + erff(y * 0.707106781f));
    case MXS_ACT_GELU_TANH: {
      // 0.5 (1 + tanh(u)) = 1 / (1 + exp(-2u)), u = sqrt(2/pi) (y + 0.044715 y^3)
      const float u2 = 1.59576912f * __builtin_fmaf(0.044715f * y * y, y, y);
      return y / (1.0f + exp_minus(u2));
    }
    default: return y;
  }
}

__device__ __forceinline__ float ld_elem(const void* p, uint64_t i, int32_t f32) {
  return f32 ? reinterpret_cast<const float*>(p)[i] : (float)reinterpret_cast<const __bf16*>(p)[i];
}

// Four consecutive features o..o+3 of row r (those below N).
__device__ __forceinline__ void epilogue4(const LinArgs& A, uint32_t r, uint32_t o, f32x4 v) {
  const uint32_t have = min(4u, A.N - o);
  const uint64_t at = (uint64_t)r * A.os + o, rat = (uint64_t)r * A.rs + o;
#pragma unroll
  for (uint32_t j = 0; j < 4u; ++j) {
    if (j >= have) break;
    float y = v[j];
    if (A.bias) y += ld_elem(A.bias, o + j, A.bias_f32);
    y = activate(y, A.act);
    if (A.res) y += ld_elem(A.res, rat + j, A.out_f32);
    if (A.out_f32) reinterpret_cast<float*>(A.out)[at + j] = y;
    else reinterpret_cast<__bf16*>(A.out)[at + j] = (__bf16)y;
  }
}

// Sixteen bytes of a row at k, elements from K on as zero.
__device__ __forceinline__ bf16x8 ld_k(const __bf16* row, uint32_t k, uint32_t K) {
  if (k + 8u <= K) return *reinterpret_cast<const bf16x8*>(row + k);
  bf16x8 v = {};
#pragma unroll
  for (uint32_t j = 0; j < 8u; ++j)
    if (k + j < K) v[j] = row[k + j];
  return v;
}

// 64 rows x 64 features per 256-thread workgroup; wave w has 32 x 32 of them
// as 2 x 2 MFMA blocks, operands straight from memory.
__global__ __launch_bounds__(256) void linear_kernel(LinArgs A) {
  const uint32_t w = threadIdx.x >> 6, l = threadIdx.x & 63u, lr = l & 15u, lg = l >> 4;
  const uint32_t o0 = blockIdx.x * 64u + (w & 1u) * 32u, r0 = blockIdx.y * 64u + (w >> 1) * 32u;
  const __bf16* wp[2];
  const __bf16* xp[2];
#pragma unroll
  for (uint32_t i = 0; i < 2u; ++i) {
    wp[i] = A.w + (uint64_t)min(o0 + i * 16u + lr, A.N - 1u) * A.ws;
    xp[i] = A.x + (uint64_t)min(r0 + i * 16u + lr, A.R - 1u) * A.xs;
  }
  f32x4 acc[2][2] = {};
  for (uint32_t k = lg * 8u; k < A.K + lg * 8u; k += 32u) {
    const bf16x8 a0 = ld_k(wp[0], k, A.K), a1 = ld_k(wp[1], k, A.K);
    const bf16x8 b0 = ld_k(xp[0], k, A.K), b1 = ld_k(xp[1], k, A.K);
    acc[0][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, b0, acc[0][0], 0, 0, 0);
    acc[0][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, b1, acc[0][1], 0, 0, 0);
    acc[1][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, b0, acc[1][0], 0, 0, 0);
    acc[1][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, b1, acc[1][1], 0, 0, 0);
  }
#pragma unroll
  for (uint32_t i = 0; i < 2u; ++i)
#pragma unroll
    for (uint32_t j = 0; j < 2u; ++j) {
      const uint32_t o = o0 + i * 16u + lg * 4u, r = r0 + j * 16u + lr;
      if (o < A.N && r < A.R) epilogue4(A, r, o, acc[i][j]);
    }
}

}  // namespace mxs

extern "C" int mxs_linear_bf16(mxs_ctx* ctx, const mxs_linear* linear) {
  using namespace mxs;
  if (!ctx) return MXS_EINVAL;
  if (const char* m = linear_check(linear)) return fail(ctx, MXS_EINVAL, m);
  const mxs_linear& a = *linear;
  if (a.rows == 0) return MXS_OK;
  LinArgs A{};
  A.x = reinterpret_cast<const __bf16*>(a.x);
  A.w = reinterpret_cast<const __bf16*>(a.weight);
  A.bias = a.bias;
  A.res = a.residual;
  A.out = a.out;
  A.xs = a.x_stride;
  A.ws = a.weight_stride;
  A.rs = a.residual_stride;
  A.os = a.out_stride;
  A.R = a.rows;
  A.K = a.in_features;
  A.N = a.out_features;
  A.act = a.act;
  A.out_f32 = a.out_dtype == MXS_F32;
  A.bias_f32 = a.bias_dtype == MXS_F32;
  const uint32_t gx = (a.out_features + 63u) / 64u, gy = (a.rows + 63u) / 64u;
  if (gy > 65535u) return fail(ctx, MXS_EINVAL, "rows must be at most 4194240");
  int prev = 0;
  (void)hipGetDevice(&prev);
  if (prev != ctx->device) (void)hipSetDevice(ctx->device);
  hipLaunchKernelGGL(linear_kernel, dim3(gx, gy), dim3(256), 0, ctx->stream, A);
  const hipError_t e = hipGetLastError();
  if (prev != ctx->device) (void)hipSetDevice(prev);
  if (e != hipSuccess) return hip_fail(ctx, e, "linear_kernel launch");
  return MXS_OK;
}
