// The argument check of attention where only some rows' weights count, for a test without a GPU.
#include "../metallix_amd/csrc/mxs_attention_checks.h"

extern "C" const char* check(const mxs_attention* a, const uint8_t* counted) { return mxs::attention_check(a, counted); }
