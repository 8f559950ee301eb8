// The argument checks of the beam and linear entry points, for a test
// without a GPU (built with the host compiler).
#include "../metallix_amd/csrc/mxs_checks.h"

extern "C" const char* check_beam(const mxs_beam* b, const mxs_beam_out* o, uint32_t rows, uint32_t vocab) {
  return mxs::beam_check(b, o, rows, vocab);
}
extern "C" const char* check_reorder(const mxs_reorder* r) { return mxs::reorder_check(r); }
extern "C" const char* check_linear(const mxs_linear* a) { return mxs::linear_check(a); }
