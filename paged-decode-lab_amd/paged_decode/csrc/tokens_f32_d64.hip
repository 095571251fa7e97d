// Attention of several tokens for FP32 q, head_dim 64: one translation unit of the gfx950 decode
// library (see token_kernels.h).
#include "token_launch.h"

namespace pd {

int launch_tokens_f32_d64(const TokenParams& p, const TokenPlan& plan, int kv_dtype, hipStream_t stream) {
    return launch_tokens<float, 64>(p, plan, kv_dtype, stream);
}

}  // namespace pd
