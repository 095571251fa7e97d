// Attention of several tokens for FP16 q (FP16 or FP8 K/V), head_dim 128: one translation unit of the gfx950 decode
// library (see token_kernels.h).
#include "token_launch.h"

namespace pd {

int launch_tokens_f16_d128(const TokenParams& p, const TokenPlan& plan, int kv_dtype, hipStream_t stream) {
    return launch_tokens<_Float16, 128>(p, plan, kv_dtype, stream);
}

}  // namespace pd
