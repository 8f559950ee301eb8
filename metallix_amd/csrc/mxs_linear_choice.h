// mxs_linear_choice.h -- which kernel a product of mxs_linear_bf16 takes, by
// its sizes and activation.  Plain C++, so that the choice is checked without
// a GPU.
#pragma once
#include <math.h>
#include <stdint.h>

#include "../../include/mx_sampler.h"

namespace mxs {

constexpr uint32_t LIN_JOBS = 288;   // workgroups of a split sum, at most

enum LinKernel { LIN_ROWS, LIN_SPLIT, LIN_SPLIT_LONG, LIN_64, LIN_64_LONG, LIN_128, LIN_128_256, LIN_256 };
struct LinChoice {
  LinKernel kernel;
  uint32_t parts, span;   // a split sum's parts, of `span` k each
};
inline LinChoice linear_choice(uint32_t R, uint32_t K, uint32_t N, int32_t activation) {
  auto tiles = [&](uint32_t bo, uint32_t br) { return (uint64_t)((N + bo - 1u) / bo) * ((R + br - 1u) / br); };
  const uint32_t steps = (K + 63u) / 64u;
  // Up to 16 rows against weights of moderate size, or up to 4 rows against
  // up to 16384 features, are latency: no LDS tiles.  us, this kernel / tiles
  // of 64 (split): 16 x 1024 x 1024 4.1 / 6.0, 16 x 4096 x 4096 9.8 / 11.9,
  // 4 x 4096 x 14336 26.1 / 30.4; but 16 x 8192 x 1024 16.3 / 11.4, 16 x 4096
  // x 14336 36.3 / 31.1, 4 x 1024 x 151936 72 / 58.
  if ((R <= 16u && N <= 4096u && K <= 4096u) || (R <= 4u && N <= 16384u)) return {LIN_ROWS, 0u, 0u};
  // One workgroup on a CU and a long sum: four tiles of loads ahead, not two,
  // for 0.4 us more to begin with.  us, two / four: 256 x 4096 x 4096 19.0 /
  // 16.4, 256 x 14336 x 4096 83.5 / 68.2, 256 x 1280 x 4096 9.7 / 9.2, 16 x
  // 14336 x 4096 (in parts) 30.3 / 25.3; but 256 x 1024 x 1024 6.7 / 7.1, and
  // with two on a CU 512 x 4096 x 4096 26.2 / 26.7, 100 x 11272 x 1025 23.3 / 24.3.
  constexpr uint32_t LONG = 20;   // steps of 64 k
  // Few tiles of 64 and a long sum: at least 10 steps of 64 k to a part, up to
  // 8 parts.  us, whole / split: 64 x 8192 x 1024 31.4 / 12.4, 256 x 4096 x
  // 1024 18.5 / 11.3, 2197 x 7797 x 31 35.1 / 17.4; but 256 x 1024 x 1024 6.9
  // / 7.8, and 64 x 4096 x 4096 12.4 in 256 jobs, 14.6 in 512.
  const uint64_t t64 = tiles(64, 64);
  uint32_t parts = steps / 10u;
  if (parts > 8u) parts = 8u;
  if (parts > LIN_JOBS / t64) parts = (uint32_t)(LIN_JOBS / t64);
  if (parts >= 2u) {
    const uint32_t span = (steps + parts - 1u) / parts * 64u, P = (K + span - 1u) / span;
    return {span >= LONG * 64u && t64 * P <= 256u ? LIN_SPLIT_LONG : LIN_SPLIT, P, span};
  }
  // Otherwise the tile with the least time: rounds of workgroups over 256 CUs
  // (three of 64 x 64 share one) times what a step of 64 k takes in each, a
  // tile's first loads and stores, and its activations (us; from 8192 x 8192 x
  // 8192, 512 x 4096 x 4096, 4096 x 128 x 12288 and 8192 x 1024 x 4096).  us
  // with tiles of 64 / 128 / 128 x 256 / 256: 8192 x 8192 x 8192 1601 / 1187 /
  // 902 / 785, 2048 x 4096 x 4096 100 / 77 / 64 / 95, 128 x 1024 x 151936 118 /
  // 98 / 112 / 120, 512 x 4096 x 4096 26 / 29 / 46 / 83.
  const double act = activation == MXS_ACT_NONE || activation == MXS_ACT_RELU ? 0.0 : activation == MXS_ACT_GELU ? 11.0 : 8.0;   // of 256 x 256
  auto rounds = [](uint64_t t, uint64_t per) { return (double)((t + per - 1u) / per); };
  const double left = rounds(t64 % 768u, 256);
  const double at64 = (double)(t64 / 768u) * (0.565 * steps + 2.6 + act * 0.19) +
                      (left > 0.0 ? (0.36 + 0.08 * left) * steps + 2.0 + act * 0.0625 * left : 0.0);
  const double at128 = rounds(tiles(128, 128), 256) * (0.56 * steps + 2.7 + act * 0.25);
  const double at128_256 = rounds(tiles(128, 256), 256) * (0.85 * steps + 4.2 + act * 0.5);
  const double at256 = rounds(tiles(256, 256), 256) * (1.46 * steps + 9.0 + act);
  const double least = fmin(fmin(at64, at128), fmin(at128_256, at256));
  const LinKernel best = least == at256 ? LIN_256 : least == at128_256 ? LIN_128_256 : least == at128 ? LIN_128 :
                         t64 <= 256u && steps >= LONG ? LIN_64_LONG : LIN_64;
  return {best, 0u, 0u};
}

}  // namespace mxs
