// The tensor-core form of the attention over the 8-bit MLA latent cache (mla_cache_attn_tc.cu), as
// mla_cache_attn.cu dispatches to it.
#pragma once
#include "kernels.h"

namespace kimi {

bool mla_attn_tc_supported(int dtype, const MlaCacheAttnArgs& a);
int64_t mla_attn_tc_workspace(int dtype, const MlaCacheAttnArgs& a);  // floats of a.part_acc
cudaError_t mla_attn_tc(int dtype, const MlaCacheAttnArgs& a, cudaStream_t s);

}  // namespace kimi
