// The attention and eviction argument checks, for a test without a GPU.
#include "../metallix_amd/csrc/mxs_attention_checks.h"

extern "C" const char* check_attention(const mxs_attention* a) { return mxs::attention_check(a); }
extern "C" const char* check_evict(const mxs_evict* e) { return mxs::evict_check(e); }
