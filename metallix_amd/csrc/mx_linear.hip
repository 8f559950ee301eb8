// mx_linear.hip -- a bf16 matrix product with bias, activation and residual
// in its epilogue (mxs_linear_bf16):
//
//   out[r][o] = act(sum_k x[r][k] weight[o][k] + bias[o]) + residual[r][o]
//
// Products and sums on v_mfma_f32_16x16x32_bf16 (f32 accumulators; operand A:
// 16 weight rows, B: 16 rows of x, so that a lane's four results are
// consecutive features of one row), the epilogue in f32, one rounding to the
// output type.  The sums' order depends on the sizes alone.
//
// linear_tile_kernel.  Tiles of 64 k go from memory into LDS without passing
// through registers (buffer_load ... lds), S - 1 tiles ahead, one workgroup
// barrier a tile.  Fragments are read half a tile (32 k) ahead of the products
// that take them, one read after each product, so that neither the reads'
// latency nor the barrier leaves the matrix pipes idle while registers hold
// work.  us at 8192 x 4096 x 14336, step by step: loads into LDS waited for at
// once 1335; restricted pointers (the compiler otherwise waits for the next
// tile's loads before this tile's reads) 1045; fragments ahead and the order
// of issue 803; results through LDS 728 to 746, 1290 to 1321 TFLOP/s (the
// library's product alone 631 us, 1525).  The matrix pipes are busy for 65% of
// the cycles, at the 1.83 GHz the card holds under this load; LDS, 192 KB read
// and 64 written per 2048 cycles of products, is as busy.  Also
// measured there: 32 x 32 x 16 products 905 us; four waves of 128 x 128 991
// (registers spill); wave priorities 826; tiles of 32 k 1127.  No LDS bank
// conflicts.
//
// What the other shapes take (us, floor the larger of bytes at 4.92 TB/s and
// flops at 1587 TFLOP/s): 128 x 1024 x 151936, f32 out, 94 (floor 79: the
// weight stream); 2048 x 4096 x 4096, gelu_tanh and residual, 64 (43); 333 x
// 1000 x 2050, gelu and residual, 10.8 (1.5: 16 dependent steps, the epilogue,
// the launch); 1 x 1024 x 1024 4.1 (0.4: one launch).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/mx_sampler.h"
#include "mxs_checks.h"
#include "mxs_ctx.h"
#include "mxs_device.h"
#include "mxs_linear_choice.h"

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
  uint32_t P, span;          // the sum over k in P parts of `span` k (a multiple of 64) each
  float* part;               // [tiles * P][tile] the parts' sums
  uint32_t* ctr;             // [tiles * CTR_STRIDE] arrivals
};

// exp(-y) for the sigmoid, to about 2 ulp: exp2 of fl(-y log2(e)), corrected
// by the argument's rounding.  -y above 89 overflows to inf, the sigmoid's 0.
__device__ __forceinline__ float exp_minus(float y) {
  const float t = -y * 1.44269504f;
  const float r = __builtin_fmaf(t, -0.693147182f, -y);
  const float e = __builtin_amdgcn_exp2f(t);
  return fabsf(t) < 126.0f ? __builtin_fmaf(e, r, e) : e;
}

// The normal distribution's integral up to y, to 2^-20 relative for y > -3
// (2^-17 further down): erfc(x) = t exp(q(t) - x^2) with x = |y| / sqrt(2), t =
// 1 / (1 + 0.4 x) and q the polynomial of degree 8 through its values at the
// Chebyshev nodes for x in 0..9.3 (1.4e-7).  x^2 = y^2 / 2 in two parts: the
// exponential would turn its rounding into a relative error.  About 25
// instructions, where a wave takes both branches of erff: gelu's share of
// 8192 x 1024 x 4096 went from 35 to 22 us.
__device__ __forceinline__ float normal_cdf(float y) {
  const float a = fminf(fabsf(y), 17.0f);   // (erfc is 0 there)
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.282842712f, a, 1.0f));
  float q = -0.218680516f;
  q = __builtin_fmaf(q, t, 0.978943706f);
  q = __builtin_fmaf(q, t, -1.59774411f);
  q = __builtin_fmaf(q, t, 1.12605083f);
  q = __builtin_fmaf(q, t, -0.530103087f);
  q = __builtin_fmaf(q, t, 0.336691082f);
  q = __builtin_fmaf(q, t, 0.390685141f);
  q = __builtin_fmaf(q, t, 1.00293851f);
  q = __builtin_fmaf(q, t, -1.48878169f);
  const float hi = a * a, lo = __builtin_fmaf(a, a, -hi);
  const float z = __builtin_fmaf(hi, -0.5f, q);
  const float res = __builtin_fmaf(lo, -0.5f, (-0.5f * hi - z) + q);   // what z and hi have lost
  const float yh = z * 1.44269504f;
  const float e = __builtin_amdgcn_exp2f(yh);
  const float h = 0.5f * t * __builtin_fmaf(e, __builtin_fmaf(yh, -0.693147182f, z) + res, e);
  return y < 0.0f ? h : 1.0f - h;
}

__device__ __forceinline__ float activate(float y, int32_t act) {
  switch (act) {   // uniform, or known
    case MXS_ACT_RELU: return y < 0.0f ? 0.0f : y;   // (a NaN stays)
    case MXS_ACT_SILU: return y / (1.0f + exp_minus(y));
    case MXS_ACT_GELU: return y * normal_cdf(y);
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

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_u __attribute__((aligned(4)));     // (global memory takes unaligned accesses)
typedef bf16x4 bf16x4_u __attribute__((aligned(2)));
typedef bf16x8 bf16x8_u __attribute__((aligned(2)));

// Four elements of `have` (1..4, the others 0) at i.
__device__ __forceinline__ f32x4 ld_four(const void* p, uint64_t i, uint32_t have, int32_t f32) {
  if (have == 4u) {
    if (f32) return *reinterpret_cast<const f32x4_u*>(reinterpret_cast<const float*>(p) + i);
    const bf16x4 v = *reinterpret_cast<const bf16x4_u*>(reinterpret_cast<const __bf16*>(p) + i);
    return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
  }
  f32x4 v = {};
#pragma unroll
  for (uint32_t j = 0; j < 3u; ++j)
    if (j < have) v[j] = ld_elem(p, i + j, f32);
  return v;
}
__device__ __forceinline__ void st_four(void* p, uint64_t i, uint32_t have, int32_t f32, f32x4 v) {
  const bf16x4 h{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
  if (have == 4u) {
    if (f32) *reinterpret_cast<f32x4_u*>(reinterpret_cast<float*>(p) + i) = v;
    else *reinterpret_cast<bf16x4_u*>(reinterpret_cast<__bf16*>(p) + i) = h;
    return;
  }
#pragma unroll
  for (uint32_t j = 0; j < 3u; ++j) {
    if (j >= have) continue;
    if (f32) reinterpret_cast<float*>(p)[i + j] = v[j];
    else reinterpret_cast<__bf16*>(p)[i + j] = h[j];
  }
}

// The epilogue of four consecutive features from o in NJ rows, 16 apart from
// r: the residuals' loads go out together.
template <int NJ>
__device__ __forceinline__ void epilogue(const LinArgs& A, int32_t act, uint32_t r, uint32_t o, const f32x4 (&acc)[NJ]) {
  if (o >= A.N) return;
  const uint32_t have = min(4u, A.N - o);
  const f32x4 b = A.bias ? ld_four(A.bias, o, have, A.bias_f32) : f32x4{};
  f32x4 res[NJ];
  if (A.res) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) res[j] = ld_four(A.res, (uint64_t)min(r + 16u * (uint32_t)j, A.R - 1u) * A.rs + o, have, A.out_f32);
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const uint32_t row = r + 16u * (uint32_t)j;
    f32x4 v = acc[j] + b;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = activate(v[e], act);
    if (A.res) v += res[j];
    if (row < A.R) st_four(A.out, (uint64_t)row * A.os + o, have, A.out_f32, v);
  }
}

// The epilogue of a wave's FO x FR blocks, the features from o and rows from
// r on.  A block's lanes hold four features of 16 rows, 32 bytes of a bf16
// row: stored like that the output reached 1.3 TB/s (4096 x 128 x 12288).  So
// 16 rows at a time pass through LDS (the wave's own 16 x 16 FO floats, a row's
// 16-byte pieces permuted by its low bits) and leave as 16 bytes a lane along the rows.  The bias and activation come
// before, the residual, loaded along the rows too, after.
template <int FO, int FR, int ACT, int E>   // E: elements in 16 bytes of output
__device__ __forceinline__ void epilogue_wave(const LinArgs& A, uint32_t r, uint32_t o, const f32x4 (&acc)[FO][FR], float* lds) {
  constexpr uint32_t W = 16u * FO, LPR = W / E, RPP = 64u / LPR, NP = 16u / RPP;   // lanes per row, rows per pass, passes
  const uint32_t l = threadIdx.x & 63u, lr = l & 15u, lg = l >> 4;
  const uint32_t row = l / LPR, col = o + (l % LPR) * E;   // what this lane stores
  f32x4 bias[FO];
#pragma unroll
  for (int i = 0; i < FO; ++i) {
    const uint32_t oi = o + 16u * (uint32_t)i + lg * 4u;
    bias[i] = A.bias && oi < A.N ? ld_four(A.bias, oi, min(4u, A.N - oi), A.bias_f32) : f32x4{};
  }
#pragma unroll
  for (int j = 0; j < FR; ++j) {
    f32x4 res[NP][E / 4];
    if (A.res) {
#pragma unroll
      for (uint32_t p = 0; p < NP; ++p) {
        const uint32_t rr = r + 16u * (uint32_t)j + p * RPP + row;
#pragma unroll
        for (uint32_t q = 0; q < E / 4u; ++q) {
          const uint32_t c = col + 4u * q;
          res[p][q] = rr < A.R && c < A.N ? ld_four(A.res, (uint64_t)rr * A.rs + c, min(4u, A.N - c), E == 4) : f32x4{};
        }
      }
    }
#pragma unroll
    for (int i = 0; i < FO; ++i) {
      f32x4 v = acc[i][j] + bias[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = activate(v[e], ACT);
      *reinterpret_cast<f32x4*>(lds + lr * W + (((uint32_t)i * 4u + lg) ^ (lr & 7u)) * 4u) = v;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (uint32_t p = 0; p < NP; ++p) {
      const uint32_t rr = r + 16u * (uint32_t)j + p * RPP + row;
      f32x4 v[E / 4];
#pragma unroll
      for (uint32_t q = 0; q < E / 4u; ++q) {
        v[q] = *reinterpret_cast<const f32x4*>(lds + (p * RPP + row) * W + (((l % LPR) * (E / 4u) + q) ^ ((p * RPP + row) & 7u)) * 4u);
        if (A.res) v[q] += res[p][q];
      }
      if (rr >= A.R || col >= A.N) continue;
      const uint64_t at = (uint64_t)rr * A.os + col;
      if (E == 8 && col + 8u <= A.N) {
        bf16x8 h;
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) h[e] = (__bf16)v[e / 4u][e & 3u];
        *reinterpret_cast<bf16x8_u*>(reinterpret_cast<__bf16*>(A.out) + at) = h;
      } else {
#pragma unroll
        for (uint32_t q = 0; q < E / 4u; ++q)
          if (col + 4u * q < A.N) st_four(A.out, at + 4u * q, min(4u, A.N - col - 4u * q), E == 4, v[q]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// Sixteen bytes of a row at k, elements from K on as zero.
__device__ __forceinline__ bf16x8 ld_k(const __bf16* row, uint32_t k, uint32_t K) {
  bf16x8 v = {};
  if (k + 8u <= K) v = *reinterpret_cast<const bf16x8*>(row + k);
  if ((K & 7u) && k < K && k + 8u > K) {   // (uniformly not, or one piece of a row)
#pragma unroll
    for (uint32_t j = 0; j < 7u; ++j)
      if (k + j < K) v[j] = row[k + j];
  }
  return v;
}

// At most 16 rows: one MFMA block of 16 features and all rows per workgroup.
// Its waves split the sum over k, 64 at a time in turn (whole 128-byte lines
// of a weight row), operands straight from memory, and their parts meet in
// LDS, added in order.
constexpr int SW = 8;   // waves
__global__ __launch_bounds__(SW * 64) void linear_rows_kernel(LinArgs A) {
  __shared__ f32x4 part[SW][64];
  const uint32_t w = threadIdx.x >> 6, l = threadIdx.x & 63u, lr = l & 15u, lg = l >> 4;
  const uint32_t o0 = blockIdx.x * 16u;
  const __bf16* const wp = A.w + (uint64_t)min(o0 + lr, A.N - 1u) * A.ws;
  const __bf16* const xp = A.x + (uint64_t)min(lr, A.R - 1u) * A.xs;
  f32x4 acc = {};
  const uint32_t whole = A.K / 64u;
  constexpr uint32_t U = 4;   // steps in flight
  uint32_t s = w;
  for (; s + (U - 1u) * SW < whole; s += U * SW) {
    bf16x8 a[U][2], b[U][2];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
#pragma unroll
      for (uint32_t h = 0; h < 2u; ++h) {
        const uint32_t k = (s + u * SW) * 64u + h * 32u + lg * 8u;
        a[u][h] = *reinterpret_cast<const bf16x8*>(wp + k);
        b[u][h] = *reinterpret_cast<const bf16x8*>(xp + k);
      }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
#pragma unroll
      for (uint32_t h = 0; h < 2u; ++h) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[u][h], b[u][h], acc, 0, 0, 0);
  }
  for (; s * 64u < A.K; s += SW) {   // the rest, the last 64 perhaps in part
#pragma unroll
    for (uint32_t h = 0; h < 2u; ++h) {
      const uint32_t k = s * 64u + h * 32u + lg * 8u;
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ld_k(wp, k, A.K), ld_k(xp, k, A.K), acc, 0, 0, 0);
    }
  }
  part[w][l] = acc;
  __syncthreads();
  if (w == 0) {
#pragma unroll
    for (int q = 1; q < SW; ++q) acc += part[q][l];
    const f32x4 one[1] = {acc};
    epilogue<1>(A, A.act, lr, o0 + lg * 4u, one);
  }
}

// Sixteen bytes per lane from base + off + at (off: this lane's, at: the
// wave's) straight into LDS, lane after lane from `lds` on.
__device__ __forceinline__ void load_lds16(__bf16* lds, const __bf16* base, uint32_t off, uint32_t at) {
#if defined(__HIP_DEVICE_COMPILE__)
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, -1, 0x27000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, off, at, 0, 0);
#endif
}
// All but the wave's N newest loads into LDS have landed and its reads are
// done; then the workgroup meets.
template <int N>
__device__ __forceinline__ void tile_barrier() {
  // (the builtin, so that the compiler knows that nothing it tracks is pending)
  static_assert(N < 64, "a six-bit counter");
  __asm__ volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4);   // vmcnt(N) lgkmcnt(0), exports not waited for
  __asm__ volatile("s_barrier" ::: "memory");
}

// The order in which M products and D LDS reads issue: a read after every
// product (or every M / D).
template <int M, int D>
__device__ __forceinline__ void interleave() {
  constexpr int P = M >= D ? M / D : 1;
#pragma unroll
  for (int i = 0; i < D; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, P, 0);
  }
}

// Many rows: BO features x BR rows per workgroup, WO x WR waves.  Tiles of TK
// k pass through S LDS buffers, written there by the loads themselves, S - 1
// tiles ahead; a row's 16-byte pieces are permuted by bits of the row so that
// the 16 rows a fragment takes fall in different banks.
template <int BO, int BR, int WO, int WR, int TK, int S, int ACT, bool SPLIT>
__global__ __launch_bounds__(WO * WR * 64, 2) void linear_tile_kernel(LinArgs A) {
  constexpr int NW = WO * WR, FO = BO / WO / 16, FR = BR / WR / 16;   // waves; 16 x 16 blocks per wave
  constexpr uint32_t PR = TK / 8, LR = 64 / PR;                       // pieces per row, rows per load
  constexpr int LA = BO / (int)LR / NW, LB = BR / (int)LR / NW;       // loads per wave
  static_assert(S <= 5, "the last tiles' waits");
  static_assert(LA * (int)LR * NW == BO && LB * (int)LR * NW == BR, "the loads cover the tile");
  // (two arrays: with one, the compiler waits for every load before a read)
  __shared__ __align__(1024) __bf16 As[S][BO * TK];
  __shared__ __align__(1024) __bf16 Bs[S][BR * TK];
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63u, lr = l & 15u, lg = l >> 4;
  // XCD x (workgroups go to the XCDs in turn) takes a contiguous range of the
  // tiles, in bands of 8 row tiles, so that what it reads is shared in its L2.
  const uint32_t no = (A.N + BO - 1u) / BO, nr = (A.R + BR - 1u) / BR, per = gridDim.x / 8u;
  const uint32_t job = (blockIdx.x & 7u) * per + (blockIdx.x >> 3);
  const uint32_t t = SPLIT ? job / A.P : job, pt = SPLIT ? job - t * A.P : 0u;
  if (t >= no * nr) return;
  const uint32_t band = t / (8u * no), in = t - band * 8u * no, hgt = min(8u, nr - band * 8u);
  const uint32_t o0 = in / hgt * BO, r0 = (band * 8u + in % hgt) * BR;
  auto turn = [](uint32_t row) { return TK == 64 ? row & 7u : (row >> 2) & 3u; };
  const uint32_t ro = l / PR, piece = ((l % PR) ^ turn(ro)) * 8u;   // what this lane loads
  // (32-bit offsets from the tile's first rows: the strides are below 2^22)
  const uint32_t k0 = SPLIT ? pt * A.span : 0u, K = SPLIT ? min(A.K - k0, A.span) : A.K;   // this part's k
  const __bf16* const wt = A.w + (uint64_t)o0 * A.ws + k0;
  const __bf16* const xt = A.x + (uint64_t)r0 * A.xs + k0;
  uint32_t ga[LA], gb[LB];
#pragma unroll
  for (int i = 0; i < LA; ++i) ga[i] = min((w * LA + i) * LR + ro, A.N - 1u - o0) * (uint32_t)A.ws + piece;
#pragma unroll
  for (int i = 0; i < LB; ++i) gb[i] = min((w * LB + i) * LR + ro, A.R - 1u - r0) * (uint32_t)A.xs + piece;
  auto fetch = [&](const __bf16* __restrict__ wk, const __bf16* __restrict__ xk, __bf16* __restrict__ as,
                   __bf16* __restrict__ bs, uint32_t k, int which) __attribute__((always_inline)) {
    if (which == 0) {
#pragma unroll
      for (int i = 0; i < LA; ++i) load_lds16(as + (w * LA + i) * LR * TK, wk, ga[i] * 2u, k * 2u);
    } else {
#pragma unroll
      for (int i = 0; i < LB; ++i) load_lds16(bs + (w * LB + i) * LR * TK, xk, gb[i] * 2u, k * 2u);
    }
  };
  auto fetch_part = [&](uint32_t k, __bf16* as, __bf16* bs) {   // the last k, not a whole tile
    auto rows = [&](auto count, const __bf16* from, uint64_t stride, uint32_t last, __bf16* to) {
      constexpr int C = decltype(count)::value;
      bf16x8 v[C];
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] = ld_k(from + (uint64_t)min((w * C + i) * LR + ro, last) * stride, k + piece, K);
#pragma unroll
      for (int i = 0; i < C; ++i) *reinterpret_cast<bf16x8*>(to + (w * C + i) * LR * TK + l * 8u) = v[i];
    };
    rows(std::integral_constant<int, LA>{}, wt, A.ws, A.N - 1u - o0, as);
    rows(std::integral_constant<int, LB>{}, xt, A.xs, A.R - 1u - r0, bs);
  };
  const uint32_t wo = (w / WR) * (BO / WO), wr = (w % WR) * (BR / WR);
  f32x4 acc[FO][FR] = {};
  const uint32_t whole = K / TK, nk = (K + TK - 1u) / TK;
#pragma unroll
  for (uint32_t k = 0; k < (uint32_t)S - 1u; ++k) {
    if (k < whole) {
      fetch(wt, xt, As[k], Bs[k], k * TK, 0);
      fetch(wt, xt, As[k], Bs[k], k * TK, 1);
    } else if (k < nk) fetch_part(k * TK, As[k], Bs[k]);
  }
  // Fragments are read one half tile ahead of the products that take them, so
  // that the reads' latency passes under the products before; the workgroup
  // meets between the last read of a tile and its last products.
  bf16x8 a0[FO], b0[FR], a1[FO], b1[FR];
  auto read = [&](bf16x8 (&a)[FO], bf16x8 (&b)[FR], const __bf16* __restrict__ ac, const __bf16* __restrict__ bc, uint32_t h)
                  __attribute__((always_inline)) {
    const uint32_t pc = ((h * 4u + lg) ^ turn(lr)) * 8u;
#pragma unroll
    for (int i = 0; i < FO; ++i) a[i] = *reinterpret_cast<const bf16x8*>(ac + (wo + i * 16u + lr) * TK + pc);
#pragma unroll
    for (int j = 0; j < FR; ++j) b[j] = *reinterpret_cast<const bf16x8*>(bc + (wr + j * 16u + lr) * TK + pc);
  };
  auto mul = [&](const bf16x8 (&a)[FO], const bf16x8 (&b)[FR], int from, int to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FO; ++i)
      if (i >= from && i < to) {
#pragma unroll
        for (int j = 0; j < FR; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
      }
  };
  // The restricted pointers tell the compiler that the loads do not write
  // what this tile's reads take, which it would wait for otherwise.  The group
  // barriers have it issue reads and loads between the products.
  auto step = [&](const __bf16* __restrict__ ac, const __bf16* __restrict__ bc, __bf16* __restrict__ an,
                  __bf16* __restrict__ bn, const __bf16* __restrict__ wk, const __bf16* __restrict__ xk, uint32_t kt,
                  auto ahead) __attribute__((always_inline)) {
    constexpr bool AHEAD = decltype(ahead)::value;
    constexpr int HALF = FO / 2 * FR, D = FO + FR;
    if (S == 2) {   // the loads have little time: first
      if (AHEAD) {
        fetch(wk, xk, an, bn, kt * TK, 0);
        fetch(wk, xk, an, bn, kt * TK, 1);
      }
      read(a0, b0, ac, bc, 0u);
      mul(a1, b1, 0, FO);
      interleave<FO * FR, D>();
      __builtin_amdgcn_sched_barrier(0);
    } else {
      read(a0, b0, ac, bc, 0u);
      mul(a1, b1, 0, FO / 2);
      interleave<HALF, D>();
      __builtin_amdgcn_sched_barrier(0);
      if (AHEAD) fetch(wk, xk, an, bn, kt * TK, 0);
      mul(a1, b1, FO / 2, FO * 3 / 4);
      __builtin_amdgcn_sched_barrier(0);
      if (AHEAD) fetch(wk, xk, an, bn, kt * TK, 1);
      mul(a1, b1, FO * 3 / 4, FO);
      __builtin_amdgcn_sched_barrier(0);
    }
    read(a1, b1, ac, bc, 1u);
    mul(a0, b0, 0, FO);
    interleave<FO * FR, D>();
    __builtin_amdgcn_sched_barrier(0);
  };
  static_assert(TK == 64, "two halves to a tile");
#pragma unroll
  for (int i = 0; i < FO; ++i) a1[i] = bf16x8{};
#pragma unroll
  for (int j = 0; j < FR; ++j) b1[j] = bf16x8{};
  uint32_t cur = 0u, nxt = S - 1u, kt = 0u;
  auto turn_buffers = [&] {
    cur = cur + 1u == (uint32_t)S ? 0u : cur + 1u;
    nxt = nxt + 1u == (uint32_t)S ? 0u : nxt + 1u;
  };
  // Tile kt is there when at most the loads of the tiles after it are still
  // in flight.
  for (; kt + (uint32_t)S - 1u < whole; ++kt) {
    tile_barrier<(S - 2) * (LA + LB)>();
    step(As[cur], Bs[cur], As[nxt], Bs[nxt], wt, xt, kt + (uint32_t)S - 1u, std::true_type{});
    turn_buffers();
  }
  for (; kt < nk; ++kt) {
    const uint32_t after = whole > kt + 1u ? whole - 1u - kt : 0u;
    if (S > 4 && after >= 3u) tile_barrier<3 * (LA + LB)>();
    else if (S > 3 && after >= 2u) tile_barrier<2 * (LA + LB)>();
    else if (S > 2 && after >= 1u) tile_barrier<LA + LB>();
    else tile_barrier<0>();
    if (kt + (uint32_t)S - 1u == whole && whole < nk) fetch_part(whole * TK, As[nxt], Bs[nxt]);
    step(As[cur], Bs[cur], As[nxt], Bs[nxt], wt, xt, 0u, std::false_type{});
    turn_buffers();
  }
  mul(a1, b1, 0, FO);
  if (SPLIT) {
    // The parts' sums meet in memory; the tile's last part adds them in order.
    float* mine = A.part + (uint64_t)job * (BO * BR) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < FO; ++i)
#pragma unroll
      for (int j = 0; j < FR; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) st_dev(mine + ((i * FR + j) * 4 + e) * (NW * 64), acc[i][j][e]);
    if (!arrive_last(&A.ctr[t * CTR_STRIDE], A.P, reinterpret_cast<uint32_t*>(&As[0][0]))) return;
    const float* from = A.part + (uint64_t)t * A.P * (BO * BR) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < FO; ++i)
#pragma unroll
      for (int j = 0; j < FR; ++j) acc[i][j] = f32x4{};
    for (uint32_t q = 0; q < A.P; ++q, from += BO * BR) {
#pragma unroll
      for (int i = 0; i < FO; ++i)
#pragma unroll
        for (int j = 0; j < FR; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] += ld_dev(from + ((i * FR + j) * 4 + e) * (NW * 64));
    }
  }
  if constexpr (FO < 4) {   // 64 bytes of a row per wave: straight away (1024 x 1024 x 1024 8.7 us, through LDS 9.7)
#pragma unroll
    for (int i = 0; i < FO; ++i) epilogue<FR>(A, ACT, r0 + wr + lr, o0 + wo + (uint32_t)i * 16u + lg * 4u, acc[i]);
  } else {
    static_assert(sizeof(As) >= NW * 16 * 16 * FO * sizeof(float), "the waves' rows fit");
    __syncthreads();   // the tiles' last reads are done
    float* const rows = reinterpret_cast<float*>(&As[0][0]) + w * (16u * 16u * FO);
    if (A.out_f32) epilogue_wave<FO, FR, ACT, 4>(A, r0 + wr, o0 + wo, acc, rows);
    else epilogue_wave<FO, FR, ACT, 8>(A, r0 + wr, o0 + wo, acc, rows);
  }
}

template <int BO, int BR, int WO, int WR, int S, bool SPLIT>
static void tile_go(hipStream_t st, const LinArgs& A) {
  const uint64_t jobs = (uint64_t)((A.N + BO - 1u) / BO) * ((A.R + BR - 1u) / BR) * (SPLIT ? A.P : 1u);
  const dim3 grid((uint32_t)((jobs + 7u) / 8u * 8u)), block(WO * WR * 64);
  switch (A.act) {
    case MXS_ACT_NONE: hipLaunchKernelGGL((linear_tile_kernel<BO, BR, WO, WR, 64, S, MXS_ACT_NONE, SPLIT>), grid, block, 0, st, A); break;
    case MXS_ACT_RELU: hipLaunchKernelGGL((linear_tile_kernel<BO, BR, WO, WR, 64, S, MXS_ACT_RELU, SPLIT>), grid, block, 0, st, A); break;
    case MXS_ACT_SILU: hipLaunchKernelGGL((linear_tile_kernel<BO, BR, WO, WR, 64, S, MXS_ACT_SILU, SPLIT>), grid, block, 0, st, A); break;
    case MXS_ACT_GELU: hipLaunchKernelGGL((linear_tile_kernel<BO, BR, WO, WR, 64, S, MXS_ACT_GELU, SPLIT>), grid, block, 0, st, A); break;
    default: hipLaunchKernelGGL((linear_tile_kernel<BO, BR, WO, WR, 64, S, MXS_ACT_GELU_TANH, SPLIT>), grid, block, 0, st, A); break;
  }
}

size_t linear_scratch_bytes() { return (size_t)LIN_JOBS * 64u * 64u * sizeof(float); }
size_t linear_ctr_words() { return (size_t)LIN_JOBS * CTR_STRIDE; }

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
  int prev = 0;
  (void)hipGetDevice(&prev);
  if (prev != ctx->device) (void)hipSetDevice(ctx->device);
  A.part = ctx->linear_scratch;
  A.ctr = ctx->linear_ctr;
  const LinChoice c = linear_choice(A.R, A.K, A.N, A.act);
  A.P = c.parts;
  A.span = c.span;
  switch (c.kernel) {
    case LIN_ROWS: hipLaunchKernelGGL(linear_rows_kernel, dim3((A.N + 15u) / 16u), dim3(SW * 64), 0, ctx->stream, A); break;
    case LIN_SPLIT: tile_go<64, 64, 2, 2, 3, true>(ctx->stream, A); break;
    case LIN_SPLIT_LONG: tile_go<64, 64, 2, 2, 5, true>(ctx->stream, A); break;
    case LIN_64_LONG: tile_go<64, 64, 2, 2, 5, false>(ctx->stream, A); break;
    case LIN_64: tile_go<64, 64, 2, 2, 3, false>(ctx->stream, A); break;
    case LIN_128: tile_go<128, 128, 2, 4, 3, false>(ctx->stream, A); break;
    case LIN_128_256: tile_go<128, 256, 2, 4, 3, false>(ctx->stream, A); break;
    case LIN_256: tile_go<256, 256, 2, 4, 2, false>(ctx->stream, A); break;
  }
  const hipError_t e = hipGetLastError();
  if (prev != ctx->device) (void)hipSetDevice(prev);
  if (e != hipSuccess) return hip_fail(ctx, e, "linear_kernel launch");
  return MXS_OK;
}
