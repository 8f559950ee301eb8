// mxs_checks.h -- the argument checks of the beam and linear entry points:
// each returns what is wrong with a call, or nullptr.  Plain C++, so that
// they are checked without a GPU.
#pragma once
#include <stdint.h>

#include "../../include/mx_sampler.h"

namespace mxs {

constexpr uint32_t BEAM_MAX_VOCAB = 2u << 20;   // tokens per row of mxs_beam_select

inline bool ranges_meet(const void* a, uint64_t na, const void* b, uint64_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x < y + nb && y < x + na;
}

inline const char* beam_check(const mxs_beam* b, const mxs_beam_out* o, uint32_t max_rows, uint32_t max_vocab) {
  if (!b || !o) return "beam and out are required";
  if (b->groups == 0) return nullptr;
  if (!b->logits || !b->score) return "logits and score are required";
  if (!o->token || !o->beam || !o->score || !o->status) return "token, beam, score and status are required";
  if (b->dtype != MXS_F32 && b->dtype != MXS_BF16) return "dtype must be MXS_F32 or MXS_BF16";
  if (b->beams == 0 || b->beams > MXS_BEAM_MAX) return "beams must be in 1..64";
  if (b->n == 0 || b->n > MXS_BEAM_N_MAX) return "n must be in 1..128";
  if (b->vocab == 0) return "vocab must be positive";
  if ((uint64_t)b->groups * b->beams > max_rows || b->vocab > max_vocab || b->vocab > BEAM_MAX_VOCAB)
    return "batch exceeds the context's max_rows/max_vocab";
  if (b->row_stride < b->vocab || (b->row_stride & 3u)) return "row_stride must be >= vocab and a multiple of 4";
  if (b->row_stride >= 1ull << 40 || (b->mask_words && b->mask_stride >= 1ull << 40)) return "strides are out of range";
  if ((uintptr_t)b->logits % (b->dtype == MXS_F32 ? 16u : 8u)) return "logits must be 16-byte (f32) or 8-byte (bf16) aligned";
  if (b->end_token < -1 || (b->end_token >= 0 && (uint32_t)b->end_token >= b->vocab))
    return "end_token must be -1 or a token of the vocabulary";
  if (b->ended && b->end_token < 0) return "ended beams need an end_token";
  if (b->mask_words) {
    if (b->mask_stride < (b->vocab + 31u) / 32u) return "mask_stride must be >= ceil(vocab / 32)";
  } else if (b->legal_norm) {
    return "legal_norm needs mask_words";
  }
  if (((const void*)o->score == (const void*)b->score || (o->ended && o->ended == b->ended)) && b->n != b->beams)
    return "out may share the input's score and ended arrays only when n == beams";
  // A group's results are written while other groups' inputs are still read,
  // so nothing else may meet.
  struct Range { const void* p; uint64_t bytes; };
  const uint64_t rows = (uint64_t)b->groups * b->beams, items = (uint64_t)b->groups * b->n;
  const Range outs[5] = {{o->token, items * 4u}, {o->beam, items * 4u}, {o->score, items * 8u}, {o->ended, items},
                         {o->status, b->groups * 4ull}};
  const Range ins[5] = {{b->logits, ((rows - 1) * b->row_stride + b->vocab) * (b->dtype == MXS_F32 ? 4u : 2u)},
                        {b->score, rows * 8u}, {b->ended, rows}, {b->scale, rows * 8u},
                        {b->mask_words, ((rows - 1) * b->mask_stride + (b->vocab + 31u) / 32u) * 4u}};
  for (int i = 0; i < 5; ++i) {
    if (!outs[i].p) continue;
    for (int j = 0; j < 5; ++j) {
      const bool own = (i == 2 && j == 1) || (i == 3 && j == 2);   // (checked above)
      if (ins[j].p && !(own && outs[i].p == ins[j].p) && ranges_meet(outs[i].p, outs[i].bytes, ins[j].p, ins[j].bytes))
        return "out overlaps an input";
    }
    for (int j = 0; j < i; ++j)
      if (outs[j].p && ranges_meet(outs[i].p, outs[i].bytes, outs[j].p, outs[j].bytes)) return "the outputs overlap";
  }
  return nullptr;
}

inline const char* reorder_check(const mxs_reorder* r) {
  if (!r) return "reorder is required";
  if (r->groups == 0) return nullptr;
  if (!r->parent || !r->status) return "parent and status are required";
  if (r->count == 0 || !r->states) return "at least one state is required";
  if (r->beams == 0 || r->beams > MXS_BEAM_MAX) return "beams must be in 1..64";
  if (r->groups > 65535u) return "groups must be at most 65535";
  if (r->parent_stride < r->beams) return "parent_stride must be >= beams";
  // A group's status is written while others' parents and lengths are read.
  const uint64_t nst = r->groups * 4ull, npar = ((r->groups - 1ull) * r->parent_stride + r->beams) * 4u;
  if (ranges_meet(r->status, nst, r->parent, npar) || (r->lengths && ranges_meet(r->status, nst, r->lengths, nst)))
    return "status overlaps parent or lengths";
  const uint64_t rows = (uint64_t)r->groups * r->beams;
  for (uint32_t i = 0; i < r->count; ++i) {
    const mxs_state& s = r->states[i];
    if (!s.data) return "a state's data is null";
    if (s.segments == 0 || s.segment_bytes == 0) return "a state's segments and segment_bytes must be positive";
    if (s.segment_bytes >= 1ull << 35 || (s.segment_bytes + 15u) / 16u * s.segments >= 1ull << 31)
      return "a state's row must be below 32 GiB";
    if (s.position_bytes >= 1ull << 32) return "a state's position_bytes must be below 4 GiB";   // (times a length: 63 bits)
    if (s.position_bytes > s.segment_bytes) return "a state's position_bytes must be at most segment_bytes";
    // segments within a row, rows within a state: apart, or interleaved the other way round
    // (all below 2^48 from the first byte, so that no sum wraps)
    if ((s.segments > 1 && s.segment_stride >= (1ull << 48) / (s.segments - 1u)) || (rows > 1 && s.row_stride >= (1ull << 48) / (rows - 1)))
      return "a state's strides are out of range";
    const uint64_t one = s.segment_bytes;
    const bool seg_apart = s.segments == 1 || s.segment_stride >= one;
    const uint64_t row_span = (s.segments - 1ull) * s.segment_stride + one;
    const uint64_t col_span = (rows - 1) * s.row_stride + one;
    const bool nested = rows == 1 || s.row_stride >= row_span;                               // [rows][segments]
    const bool crossed = s.row_stride >= one && (s.segments == 1 || s.segment_stride >= col_span);   // [segments][rows]
    if (!seg_apart || !(nested || crossed)) return "a state's rows or segments overlap";
  }
  return nullptr;
}

inline const char* linear_check(const mxs_linear* a) {
  if (!a) return "linear is required";
  if (a->rows == 0) return nullptr;
  if (!a->x || !a->weight || !a->out) return "x, weight and out are required";
  if (a->in_features == 0 || a->out_features == 0) return "in_features and out_features must be positive";
  if (a->in_features > 1u << 30 || a->out_features > 1u << 30 || a->rows > 1u << 30) return "rows and features must be at most 2^30";
  if ((a->rows + 63ull) / 64u * ((a->out_features + 63ull) / 64u) >= 1ull << 23)   // (a launch holds below 2^32 threads)
    return "rows x out_features must be below 2^35 (counted in whole blocks of 64 x 64)";
  if (a->act < MXS_ACT_NONE || a->act > MXS_ACT_GELU_TANH) return "act must be one of MXS_ACT_*";
  if (a->out_dtype != MXS_F32 && a->out_dtype != MXS_BF16) return "out_dtype must be MXS_F32 or MXS_BF16";
  if (a->bias && a->bias_dtype != MXS_F32 && a->bias_dtype != MXS_BF16) return "bias_dtype must be MXS_F32 or MXS_BF16";
  if (a->x_stride < a->in_features || a->x_stride % 8u || a->weight_stride < a->in_features || a->weight_stride % 8u)
    return "x_stride and weight_stride must be multiples of 8 and >= in_features";
  if (a->out_stride < a->out_features || (a->residual && a->residual_stride < a->out_features))
    return "out_stride and residual_stride must be >= out_features";
  if (a->x_stride >= 1ull << 22 || a->weight_stride >= 1ull << 22) return "x_stride and weight_stride must be below 2^22: out of range";
  if (a->out_stride >= 1ull << 40 || a->residual_stride >= 1ull << 40) return "strides are out of range";
  if (((uintptr_t)a->x | (uintptr_t)a->weight) % 16u) return "x and weight must be 16-byte aligned";
  const uint64_t es = a->out_dtype == MXS_F32 ? 4u : 2u, bs = a->bias_dtype == MXS_F32 ? 4u : 2u;
  if ((uintptr_t)a->out % es || (uintptr_t)a->residual % es || (a->bias && (uintptr_t)a->bias % bs))
    return "out, residual and bias must be aligned to their elements";
  const uint64_t r1 = a->rows - 1ull, ob = (r1 * a->out_stride + a->out_features) * es;
  if (ranges_meet(a->out, ob, a->x, (r1 * a->x_stride + a->in_features) * 2u) ||
      ranges_meet(a->out, ob, a->weight, ((a->out_features - 1ull) * a->weight_stride + a->in_features) * 2u) ||
      (a->bias && ranges_meet(a->out, ob, a->bias, a->out_features * bs)))
    return "out overlaps an input";
  if (a->residual && !(a->residual == a->out && a->residual_stride == a->out_stride) &&
      ranges_meet(a->out, ob, a->residual, (r1 * a->residual_stride + a->out_features) * es))
    return "residual must be out itself or apart from it";
  return nullptr;
}

}  // namespace mxs
