// mx_beam.hip -- beam search: the selection of each group's n best
// continuations over its beams and the vocabulary (mxs_beam_select), and the
// move of the beams' states to their children (mxs_beam_reorder).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <string>

#include "../../include/mx_sampler.h"
#include "mxs_checks.h"
#include "mxs_ctx.h"
#include "mxs_device.h"
#include "mxs_math.h"

namespace mxs {

constexpr int BNT = 256;                  // threads per workgroup
constexpr int BNW = BNT / 64;

struct BeamRow {
  double norm;          // ln sum exp of the row's logits that count
  uint32_t bad;         // a NaN or +inf among them
  uint32_t pad;
};

struct BeamArgs {
  const void* logits;
  uint64_t stride;
  uint32_t G, W, V, n;
  const double* score;
  const uint8_t* ended;
  const double* scale;
  const uint32_t* mask;
  uint64_t mask_stride;
  uint32_t tok_vocab, legal_norm;
  int32_t end_token;
  int32_t* token;
  int32_t* beam;
  double* oscore;
  uint8_t* oended;
  int32_t* status;
  BeamRow* rows;
};

__device__ __forceinline__ bool beam_legal(const BeamArgs& A, uint32_t row, uint32_t v) {
  if (!A.mask) return true;
  return v < A.tok_vocab && ((A.mask[(uint64_t)row * A.mask_stride + (v >> 5)] >> (v & 31u)) & 1u);
}

__device__ __forceinline__ bool beam_live(const BeamArgs& A, uint32_t row) {
  const double s = A.score[row];
  return s > -INFINITY && !(A.ended && A.ended[row]);
}

template <typename In>
__global__ __launch_bounds__(BNT) void beam_norm_kernel(BeamArgs A) {
  __shared__ double red[BNW];
  __shared__ float redf[BNW];
  __shared__ uint32_t redu[BNW];
  const uint32_t row = blockIdx.x;
  if (!beam_live(A, row)) return;
  const In* src = reinterpret_cast<const In*>(A.logits) + (uint64_t)row * A.stride;
  float m = -INFINITY;
  uint32_t bad = 0;
  for (uint32_t v = threadIdx.x; v < A.V; v += BNT) {
    if (A.legal_norm && !beam_legal(A, row, v)) continue;
    const float x = Quad<In>::one(src + v);
    bad |= !(x < INFINITY);
    m = fmaxf(m, x);
  }
  m = wave_max_f32(m);
  bad = wave_or_u32(bad);
  if (lane() == 0) { redf[wave()] = m; redu[wave()] = bad; }
  __syncthreads();
  for (int w = 0; w < BNW; ++w) { m = fmaxf(m, redf[w]); bad |= redu[w]; }
  double sum = 0.0;
  if (m > -INFINITY && !bad)
    for (uint32_t v = threadIdx.x; v < A.V; v += BNT) {
      if (A.legal_norm && !beam_legal(A, row, v)) continue;
      sum += exp_neg_p((double)Quad<In>::one(src + v) - (double)m);
    }
  sum = wave_sum_f64(sum);
  if (lane() == 0) red[wave()] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
    for (int w = 0; w < BNW; ++w) sum += red[w];
    A.rows[row].norm = (double)m + log(sum);
    A.rows[row].bad = bad;
  }
}

// A candidate and its place in the order: larger rank, lower beam, larger
// logit, lower token.
struct BeamCand {
  double rank;
  double score;
  uint32_t beam, key, token;
};
__device__ __forceinline__ bool before(const BeamCand& a, const BeamCand& b) {
  if (a.rank != b.rank) return a.rank > b.rank;
  if (a.beam != b.beam) return a.beam < b.beam;
  if (a.key != b.key) return a.key > b.key;
  return a.token < b.token;
}

template <typename In>
__global__ __launch_bounds__(BNT) void beam_pick_kernel(BeamArgs A) {
  __shared__ BeamCand best[BNT];
  const uint32_t g = blockIdx.x, W = A.W, n = A.n;
  uint32_t st = 0;
  for (uint32_t b = 0; b < W; ++b) {
    const uint32_t row = g * W + b;
    const double s = A.score[row], c = A.scale ? A.scale[row] : 1.0;
    if (!(s < INFINITY) || !(c > 0.0 && c < INFINITY)) st |= 1u;
    else if (beam_live(A, row) && A.rows[row].bad) st |= 2u;
  }
  __syncthreads();   // the inputs are read before an output that shares their array is written
  if (st) {
    for (uint32_t j = threadIdx.x; j < n; j += BNT) {
      A.token[g * n + j] = -1;
      A.beam[g * n + j] = -1;
      A.oscore[g * n + j] = __builtin_nan("");
      if (A.oended) A.oended[g * n + j] = 0;
    }
    if (threadIdx.x == 0) A.status[g] = (st & 1u) ? MXS_ROW_PROBABILITIES : MXS_ROW_NON_FINITE_LOGIT;
    return;
  }
  const BeamCand none{-INFINITY, -INFINITY, 0xffffffffu, 0u, 0xffffffffu};
  BeamCand last{INFINITY, 0.0, 0u, 0xffffffffu, 0u};
  BeamCand keep = none;   // thread j holds candidate j
  uint32_t count = 0;
  for (uint32_t j = 0; j < n; ++j) {
    BeamCand mine = none;
    for (uint32_t b = 0; b < W; ++b) {
      const uint32_t row = g * W + b;
      const double s = A.score[row], c = A.scale ? A.scale[row] : 1.0;
      if (!(s > -INFINITY)) continue;
      if (A.ended && A.ended[row]) {
        const BeamCand e{s * c, s, b, 0u, (uint32_t)A.end_token};
        if (threadIdx.x == 0 && (j == 0 || before(last, e)) && before(e, mine)) mine = e;
        continue;
      }
      const In* src = reinterpret_cast<const In*>(A.logits) + (uint64_t)row * A.stride;
      const double norm = A.rows[row].norm;
      for (uint32_t v = threadIdx.x; v < A.V; v += BNT) {
        const float x = Quad<In>::one(src + v) + 0.0f;   // -0 and +0 are equal logits
        if (!(x > -INFINITY) || !beam_legal(A, row, v)) continue;
        const double sc = s + ((double)x - norm);
        const BeamCand e{sc * c, sc, b, okey(x), v};
        if ((j == 0 || before(last, e)) && before(e, mine)) mine = e;
      }
    }
    best[threadIdx.x] = mine;
    __syncthreads();
    for (uint32_t h = BNT / 2; h > 0; h >>= 1) {
      if (threadIdx.x < h && before(best[threadIdx.x + h], best[threadIdx.x])) best[threadIdx.x] = best[threadIdx.x + h];
      __syncthreads();
    }
    last = best[0];
    __syncthreads();
    if (last.beam == 0xffffffffu) break;
    if (threadIdx.x == j) keep = last;
    ++count;
  }
  if (threadIdx.x < n) {
    const uint32_t j = threadIdx.x;
    const bool there = j < count;
    const uint64_t at = (uint64_t)g * n + j;
    A.token[at] = there ? (int32_t)keep.token : -1;
    A.beam[at] = there ? (int32_t)keep.beam : -1;
    A.oscore[at] = there ? keep.score : -INFINITY;
    if (A.oended) A.oended[at] = there && (int32_t)keep.token == A.end_token ? 1 : 0;
  }
  if (threadIdx.x == 0) A.status[g] = count ? 0 : MXS_ROW_EMPTY_SUPPORT;
}

size_t beam_scratch_bytes(uint32_t max_rows) { return (size_t)max_rows * sizeof(BeamRow); }

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

// Sixteen bytes at any alignment (global memory takes unaligned accesses).
struct __attribute__((packed, aligned(1))) Piece16 { uint32_t w[4]; };
struct __attribute__((packed, aligned(1))) Piece8 { uint32_t w[2]; };
struct __attribute__((packed, aligned(1))) Piece4 { uint32_t w; };
struct __attribute__((packed, aligned(1))) Piece2 { uint16_t w; };
struct __attribute__((packed, aligned(1))) Piece1 { uint8_t w; };

// Moves one T at `at` (offset `at` of row 0 of the group) between the rows,
// in the lanes where `act`.  p: lane j holds row j's parent.  Every lane of
// the wave comes here, so that the ballots see all parents.
template <typename T, int WMAX>
__device__ __forceinline__ void move_piece(char* at, uint64_t stride, int32_t p, bool act) {
  const uint32_t l = threadIdx.x & 63u;
  T v[WMAX];
#pragma unroll
  for (int j = 0; j < WMAX; ++j) {
    const uint64_t to = __builtin_amdgcn_ballot_w64(p == j && l != (uint32_t)j);
    if (to && act) v[j] = *reinterpret_cast<const T*>(at + (uint64_t)j * stride);
  }
#pragma unroll
  for (int j = 0; j < WMAX; ++j) {
    uint64_t to = __builtin_amdgcn_ballot_w64(p == j && l != (uint32_t)j);
    while (to) {
      const uint32_t d = (uint32_t)__builtin_ctzll(to);
      to &= to - 1u;
      if (act) *reinterpret_cast<T*>(at + (uint64_t)d * stride) = v[j];
    }
  }
}

// One thread holds the same 16 bytes of all the group's rows: it loads those
// of every row that some other row takes over, then stores them to the rows
// that take them.  No thread reads what another writes, so any permutation
// goes in place, each surviving row read once and each changed row written
// once.  WMAX, the most rows held, is the power of two at or above beams.
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
  const uint32_t i = min(blockIdx.x * RO_NT + threadIdx.x, total - 1u);
  const bool in = blockIdx.x * RO_NT + threadIdx.x < total;
  const uint32_t seg = i / pieces, pc = i - seg * pieces;
  char* at = reinterpret_cast<char*>(s.data) + (uint64_t)g * W * s.row_stride + (uint64_t)seg * s.segment_stride +
             (uint64_t)pc * 16u;
  const uint32_t have = !in ? 0u : (uint32_t)min((uint64_t)16u, used - (uint64_t)pc * 16u);
  move_piece<Piece16, WMAX>(at, s.row_stride, p, have == 16u);
  if (__builtin_amdgcn_ballot_w64(have & 15u)) {   // a segment's last bytes
    move_piece<Piece8, WMAX>(at, s.row_stride, p, (have & 8u) != 0u);
    at += have & 8u;
    move_piece<Piece4, WMAX>(at, s.row_stride, p, (have & 4u) != 0u);
    at += have & 4u;
    move_piece<Piece2, WMAX>(at, s.row_stride, p, (have & 2u) != 0u);
    at += have & 2u;
    move_piece<Piece1, WMAX>(at, s.row_stride, p, (have & 1u) != 0u);
  }
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
  A.legal_norm = b.mask_words ? b.legal_norm : 0u;
  A.end_token = b.end_token;
  A.token = out->token;
  A.beam = out->beam;
  A.oscore = out->score;
  A.oended = out->ended;
  A.status = out->status;
  A.rows = reinterpret_cast<BeamRow*>(ctx->beam_scratch);
  int prev = 0;
  (void)hipGetDevice(&prev);
  if (prev != ctx->device) (void)hipSetDevice(ctx->device);
  if (b.dtype == MXS_F32) {
    hipLaunchKernelGGL(beam_norm_kernel<float>, dim3(A.G * A.W), dim3(BNT), 0, ctx->stream, A);
    hipLaunchKernelGGL(beam_pick_kernel<float>, dim3(A.G), dim3(BNT), 0, ctx->stream, A);
  } else {
    hipLaunchKernelGGL(beam_norm_kernel<uint16_t>, dim3(A.G * A.W), dim3(BNT), 0, ctx->stream, A);
    hipLaunchKernelGGL(beam_pick_kernel<uint16_t>, dim3(A.G), dim3(BNT), 0, ctx->stream, A);
  }
  const hipError_t e = hipGetLastError();
  if (prev != ctx->device) (void)hipSetDevice(prev);
  if (e != hipSuccess) return hip_fail(ctx, e, "beam launch");
  mask_note_read(ctx, b.mask_words);
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
