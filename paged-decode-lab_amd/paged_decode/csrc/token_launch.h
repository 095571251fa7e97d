// Launches of the attention of several tokens, for one q format and head dimension.
#ifndef PAGED_DECODE_TOKEN_LAUNCH_H
#define PAGED_DECODE_TOKEN_LAUNCH_H

#include "token_kernels.h"

namespace pd {

int launch_tokens_f32_d64(const TokenParams&, const TokenPlan&, int kv_dtype, hipStream_t);
int launch_tokens_f32_d128(const TokenParams&, const TokenPlan&, int kv_dtype, hipStream_t);
int launch_tokens_f16_d64(const TokenParams&, const TokenPlan&, int kv_dtype, hipStream_t);
int launch_tokens_f16_d128(const TokenParams&, const TokenPlan&, int kv_dtype, hipStream_t);
int launch_tokens_bf16_d64(const TokenParams&, const TokenPlan&, int kv_dtype, hipStream_t);
int launch_tokens_bf16_d128(const TokenParams&, const TokenPlan&, int kv_dtype, hipStream_t);

// Splits of a sequence, on average, up to which a wave merges a row (16 of them: 21.6 us of a call with one, 22.6 with four; 32:
// 20.5 with one, 20.1 with four).
constexpr int kMergeWaveSplits = 24;

template <typename QT, int D>
int merge_tokens(const TokenParams& p, hipStream_t stream) {
    if (p.split != kTokenWhole) {
        const int64_t rows = static_cast<int64_t>(p.batch) * p.tokens * p.query_heads;
        // Four waves for a row of many splits, where one would read them in turns.
        if (p.items > kMergeWaveSplits * p.batch) {
            hipLaunchKernelGGL((token_merge_kernel<QT, D, 4>), dim3(static_cast<uint32_t>(rows)), dim3(256), 0, stream, p);
        } else {
            hipLaunchKernelGGL((token_merge_kernel<QT, D, 1>), dim3(static_cast<uint32_t>((rows + 3) / 4)), dim3(256), 0, stream, p);
        }
    }
    return hipGetLastError() == hipSuccess ? PD_OK : PD_ERR_LAUNCH;
}

template <typename QT, int KVF, int D>
int launch_tokens_format(const TokenParams& p, const TokenPlan& plan, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(token_workgroups(plan, p.kv_heads)));
    constexpr int KT = sizeof(QT) == 4 ? 32 : 64;
    if (plan.stream) {
        constexpr int WAVES = sizeof(QT) == 4 && D == 128 ? kStreamWaves / 2 : kStreamWaves;
        const dim3 threads(WAVES * kWave);
        if (plan.tile_rows == 16) {
            if (plan.once) hipLaunchKernelGGL((token_stream_kernel<QT, KVF, D, 1, WAVES, true>), grid, threads, 0, stream, p);
            else hipLaunchKernelGGL((token_stream_kernel<QT, KVF, D, 1, WAVES, false>), grid, threads, 0, stream, p);
        } else {
            if (plan.once) hipLaunchKernelGGL((token_stream_kernel<QT, KVF, D, 2, WAVES, true>), grid, threads, 0, stream, p);
            else hipLaunchKernelGGL((token_stream_kernel<QT, KVF, D, 2, WAVES, false>), grid, threads, 0, stream, p);
        }
    } else {
        const dim3 threads(4 * kWave * plan.groups);
        if (plan.tile_rows == 64) {
            if (plan.groups == 2) hipLaunchKernelGGL((token_kernel<QT, KVF, D, 1, 4, KT, 2, false>), grid, threads, 0, stream, p);
            else hipLaunchKernelGGL((token_kernel<QT, KVF, D, 1, 4, KT, 1, false>), grid, threads, 0, stream, p);
        } else if constexpr (!(sizeof(QT) == 4 && D == 128)) {
            if (D == 128 && plan.products_first) {
                hipLaunchKernelGGL((token_kernel<QT, KVF, D, 2, 4, KT, 1, D == 128>), grid, threads, 0, stream, p);
            } else {
                hipLaunchKernelGGL((token_kernel<QT, KVF, D, 2, 4, KT, 1, false>), grid, threads, 0, stream, p);
            }
        }
    }
    return merge_tokens<QT, D>(p, stream);
}

template <typename QT, int D>
int launch_tokens(const TokenParams& p, const TokenPlan& plan, int kv_dtype, hipStream_t stream) {
    if constexpr (sizeof(QT) == 2) {
        if (kv_dtype == PD_DTYPE_FP8_E4M3) return launch_tokens_format<QT, PD_DTYPE_FP8_E4M3, D>(p, plan, stream);
        if (kv_dtype == PD_DTYPE_FP8_E5M2) return launch_tokens_format<QT, PD_DTYPE_FP8_E5M2, D>(p, plan, stream);
    }
    return launch_tokens_format<QT, kTokenNative, D>(p, plan, stream);
}

}  // namespace pd

#endif  // PAGED_DECODE_TOKEN_LAUNCH_H
