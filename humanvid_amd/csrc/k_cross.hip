// k_cross.hip -- translation unit for hv_cross_attention.h (see hv_kernels.h)
#include "hv_cross_attention.h"
#include "hv_kernels.h"

int hvk_cross_attention(const hv_cross_attention_params& p, hipStream_t s) { return hv_cross_attention_launch(p, s); }
long hvk_cross_attention_workspace(const hv_cross_attention_params& p) { return hv_cross_attention_workspace_of(p); }
