// Attention of several tokens for BF16 q (BF16 or FP8 K/V), head_dim 64: one translation unit of the gfx950 decode
// library (see token_kernels.h).
#include "token_launch.h"

namespace pd {

int launch_tokens_bf16_d64(const TokenParams& p, const TokenPlan& plan, int kv_dtype, hipStream_t stream) {
    return launch_tokens<__bf16, 64>(p, plan, kv_dtype, stream);
}

}  // namespace pd
