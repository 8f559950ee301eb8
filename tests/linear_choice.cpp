// Which kernel a linear product takes, for a test without a GPU (built with
// the host compiler).
#include "../metallix_amd/csrc/mxs_linear_choice.h"

extern "C" int choose(uint32_t rows, uint32_t k, uint32_t n, int32_t act, uint32_t* parts, uint32_t* span) {
  const mxs::LinChoice c = mxs::linear_choice(rows, k, n, act);
  *parts = c.parts;
  *span = c.span;
  return c.kernel;
}
