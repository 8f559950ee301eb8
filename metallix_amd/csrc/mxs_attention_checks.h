// mxs_attention_checks.h -- the argument checks of the attention and eviction
// entry points: each returns what is wrong with a call, or nullptr.  Plain
// C++, so that they are checked without a GPU.
#pragma once
#include <math.h>
#include <stdint.h>

#include "../../include/mx_sampler.h"
#include "mxs_checks.h"

namespace mxs {

// Bytes from the first to past the last element of [n0][n1][n2] rows of
// `row` bytes, strides in bytes.
inline uint64_t span3(uint64_t n0, uint64_t s0, uint64_t n1, uint64_t s1, uint64_t n2, uint64_t s2, uint64_t row) {
  return (n0 - 1) * s0 + (n1 - 1) * s1 + (n2 - 1) * s2 + row;
}

struct MemRange { const void* p; uint64_t bytes; };

// What is wrong where one of the outputs meets an input or another output.
template <int NO, int NI>
inline const char* outputs_apart(const MemRange (&outs)[NO], const MemRange (&ins)[NI]) {
  for (int i = 0; i < NO; ++i) {
    if (!outs[i].p) continue;
    for (int j = 0; j < NI; ++j)
      if (ins[j].p && ranges_meet(outs[i].p, outs[i].bytes, ins[j].p, ins[j].bytes)) return "an output overlaps an input";
    for (int j = 0; j < i; ++j)
      if (outs[j].p && ranges_meet(outs[i].p, outs[i].bytes, outs[j].p, outs[j].bytes)) return "the outputs overlap";
  }
  return nullptr;
}

// Whether [n0][n1][n2] rows of `row` elements at these strides lie apart,
// whatever the order of their dimensions in memory.
inline bool rows_apart(uint64_t n0, uint64_t s0, uint64_t n1, uint64_t s1, uint64_t n2, uint64_t s2, uint64_t row) {
  uint64_t n[3] = {n0, n1, n2}, s[3] = {s0, s1, s2};
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 3; ++j)
      if (s[j] < s[i]) {
        const uint64_t a = n[i], b = s[i];
        n[i] = n[j]; s[i] = s[j];
        n[j] = a; s[j] = b;
      }
  uint64_t need = row;
  for (int i = 0; i < 3; ++i) {
    if (n[i] == 1) continue;   // (its stride says nothing)
    if (s[i] < need) return false;
    need += (n[i] - 1) * s[i];
  }
  return true;
}

inline const char* attention_check(const mxs_attention* a, const uint8_t* counted = nullptr) {
  if (!a) return "attention is required";
  if (a->groups == 0 || a->beams == 0 || a->tokens == 0) return nullptr;
  if (!a->q || !a->out) return "q and out are required";
  if (a->heads == 0 || a->kv_heads == 0 || a->heads % a->kv_heads) return "heads must be a multiple of kv_heads";
  if (a->heads > 4096u) return "heads must be at most 4096";
  if (a->dim == 0 || a->dim > 256 || a->dim % 8u) return "dim must be a multiple of 8 in 8..256";
  if (a->prefix > 1u << 30 || a->suffix > 1u << 30) return "prefix and suffix must be at most 2^30";
  const uint64_t rows = (uint64_t)a->groups * a->beams;
  if (rows >= 1ull << 31 || rows * a->tokens >= 1ull << 31 || rows * a->tokens * a->heads >= 1ull << 31)
    return "groups x beams x tokens x heads must be below 2^31";
  if (a->prefix && (!a->prefix_keys || !a->prefix_values)) return "a prefix needs its keys and values";
  if (a->suffix && (!a->keys || !a->values)) return "a suffix needs its keys and values";
  if (a->prefix_weight && !a->prefix) return "prefix_weight needs a prefix";
  if (a->weight && !a->suffix) return "weight needs a suffix";
  if (!(fabsf(a->scale) <= 2.0e38f)) return "scale must be a number of at most 2e38";   // (times log2(e): finite)
  const uint64_t st[12] = {a->q_row, a->q_token, a->q_head, a->out_row, a->out_token, a->out_head,
                           a->prefix_group, a->prefix_head, a->prefix_position, a->row, a->head, a->position};
  const int used = 6 + (a->prefix ? 3 : 0);
  for (int i = 0; i < 12; ++i) {
    if (i >= used && !(a->suffix && i >= 9)) continue;
    if (st[i] % 8u) return "strides must be multiples of 8";
    if (st[i] >= 1ull << 40) return "strides are out of range";
  }
  if ((a->prefix && a->prefix_position >= 1ull << 22) || (a->suffix && a->position >= 1ull << 22))
    return "the positions' strides must be below 2^22";
  if (((uintptr_t)a->q | (uintptr_t)a->out | (uintptr_t)(a->prefix ? a->prefix_keys : nullptr) |
       (uintptr_t)(a->prefix ? a->prefix_values : nullptr) | (uintptr_t)(a->suffix ? a->keys : nullptr) |
       (uintptr_t)(a->suffix ? a->values : nullptr)) % 16u)
    return "q, out and the caches must be 16-byte aligned";
  if (((uintptr_t)a->lse | (uintptr_t)a->prefix_weight | (uintptr_t)a->weight | (uintptr_t)a->prefix_lengths |
       (uintptr_t)a->lengths) % 4u)
    return "lse, weights and lengths must be aligned to their elements";
  // (spans below 2^50, so that no sum wraps)
  const auto wide = [](uint64_t n, uint64_t stride) { return stride >= (1ull << 48) / n; };
  if (wide(rows, a->out_row) || wide(rows, a->q_row) || wide(a->tokens, a->out_token) || wide(a->tokens, a->q_token) ||
      wide(a->heads, a->out_head) || wide(a->heads, a->q_head) ||
      (a->prefix && (wide(a->groups, a->prefix_group) || wide(a->kv_heads, a->prefix_head))) ||
      (a->suffix && (wide(rows, a->row) || wide(a->kv_heads, a->head))))
    return "strides are out of range";
  if (!rows_apart(rows, a->out_row, a->tokens, a->out_token, a->heads, a->out_head, a->dim)) return "out's rows overlap";
  const uint64_t D2 = a->dim * 2ull;
  const uint64_t pre = a->prefix ? span3(a->groups, a->prefix_group * 2u, a->kv_heads, a->prefix_head * 2u, a->prefix, a->prefix_position * 2u, D2) : 0u;
  const uint64_t suf = a->suffix ? span3(rows, a->row * 2u, a->kv_heads, a->head * 2u, a->suffix, a->position * 2u, D2) : 0u;
  const uint64_t queries = rows * a->tokens * a->heads;
  const MemRange outs[4] = {{a->out, span3(rows, a->out_row * 2u, a->tokens, a->out_token * 2u, a->heads, a->out_head * 2u, D2)},
                            {a->lse, queries * 4u},
                            {a->prefix_weight, (uint64_t)a->groups * a->kv_heads * a->prefix * 4u},
                            {a->weight, rows * a->kv_heads * a->suffix * 4u}};
  const MemRange ins[8] = {{a->q, span3(rows, a->q_row * 2u, a->tokens, a->q_token * 2u, a->heads, a->q_head * 2u, D2)},
                           {a->prefix ? a->prefix_keys : nullptr, pre}, {a->prefix ? a->prefix_values : nullptr, pre},
                           {a->suffix ? a->keys : nullptr, suf}, {a->suffix ? a->values : nullptr, suf},
                           {a->prefix_lengths, a->groups * 4ull}, {a->lengths, rows * 4u}, {counted, rows}};
  return outputs_apart(outs, ins);
}

inline const char* evict_check(const mxs_evict* e) {
  if (!e) return "evict is required";
  if (e->layers == 0 || e->segments == 0 || e->heads == 0) return nullptr;
  if (!e->caches || !e->weight || !e->weight_out) return "caches, weight and weight_out are required";
  if (e->capacity == 0 || e->capacity > MXS_EVICT_MAX_CAPACITY) return "capacity must be in 1..2^20";
  const uint64_t sh = (uint64_t)e->segments * e->heads;
  if (sh >= 1ull << 21 || sh * e->layers >= 1ull << 21) return "layers x segments x heads must be below 2^21";
  if (e->budget == 0) return "budget must be positive";
  if (e->keep_first > e->budget || e->keep_recent > e->budget - e->keep_first) return "keep_first + keep_recent must be at most budget";
  if (e->position_bytes == 0 || e->position_bytes > 65536u) return "position_bytes must be in 1..65536";
  if (e->segment_stride >= (1ull << 48) / e->segments || e->head_stride >= (1ull << 48) / e->heads || e->position_stride >= 1ull << 28)
    return "strides are out of range";
  if (!rows_apart(e->segments, e->segment_stride, e->heads, e->head_stride, e->capacity, e->position_stride, e->position_bytes))
    return "a cache's positions overlap";
  if (((uintptr_t)e->weight | (uintptr_t)e->index | (uintptr_t)e->lengths | (uintptr_t)e->weight_out | (uintptr_t)e->index_out |
       (uintptr_t)e->lengths_out) % 4u)
    return "weight, index and lengths must be aligned to their elements";
  for (uint32_t l = 0; l < e->layers; ++l)
    if (!e->caches[l].keys) return "a layer's keys are null";
  const uint64_t n = sh * e->layers * e->capacity * 4u, ns = e->segments * 4ull;
  const MemRange outs[3] = {{e->weight_out, n}, {e->index_out, n}, {e->lengths_out, ns}};
  const MemRange ins[3] = {{e->weight, n}, {e->index, n}, {e->lengths, ns}};
  return outputs_apart(outs, ins);
}

}  // namespace mxs
