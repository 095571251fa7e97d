// Host side of the attention of several tokens per sequence: argument checks,
// the launch plan, and the entry points. The kernels are in token_kernels.h.
#include <hip/hip_runtime.h>

#include <cmath>

#include "paged_decode.h"
#include "token_launch.h"

namespace pd {
namespace {

bool token_formats(int q_dtype, int kv_dtype) {
    if (q_dtype < PD_DTYPE_F32 || q_dtype > PD_DTYPE_BF16) return false;
    if (kv_dtype == q_dtype) return true;
    return q_dtype != PD_DTYPE_F32 && (kv_dtype == PD_DTYPE_FP8_E4M3 || kv_dtype == PD_DTYPE_FP8_E5M2);
}

bool token_shape(int batch, int tokens, int query_heads, int kv_heads, int head_dim, int page_size, int table_width) {
    if (batch < 1 || batch > 65535 || tokens < 1 || tokens > 65535) return false;
    if (query_heads < 1 || query_heads > 65535 || kv_heads < 1 || query_heads % kv_heads != 0) return false;
    if (head_dim != 64 && head_dim != 128) return false;
    if (page_size != 16 && page_size != 32) return false;
    return table_width >= 1 && table_width <= 65536;
}

int device_cus() {
    int device = 0, cus = 0;
    if (hipGetDevice(&device) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || cus <= 0)
        return 256;
    return cus;
}

size_t state_bytes(int head_dim) { return static_cast<size_t>(head_dim + 2) * sizeof(float); }

bool misaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

}  // namespace
}  // namespace pd

extern "C" {

size_t pd_decode_tokens_workspace(int q_dtype, int kv_dtype, int batch, int tokens, int query_heads, int kv_heads,
                                  int head_dim, int page_size, int table_width, int compute_units) {
    using namespace pd;
    if (!token_formats(q_dtype, kv_dtype) ||
        !token_shape(batch, tokens, query_heads, kv_heads, head_dim, page_size, table_width))
        return 0;
    const int cus = compute_units > 0 ? compute_units : device_cus();
    const int64_t reach = static_cast<int64_t>(table_width) * page_size;
    const int64_t states = most_token_states(q_dtype == PD_DTYPE_F32 ? 4 : 2, head_dim, batch, tokens, query_heads, kv_heads,
                                             reach, cus);
    return static_cast<size_t>(states) * state_bytes(head_dim);
}

int pd_decode_tokens(const void* q, int q_dtype, const void* k, const void* v, int kv_dtype, float k_scale,
                     float v_scale, const int32_t* table, const int32_t* lengths, const int32_t* counts, void* out,
                     void* workspace, size_t workspace_bytes, int batch, int tokens, int query_heads, int kv_heads,
                     int head_dim, int page_size, int table_width, int physical_pages, int causal, int hints,
                     const int32_t* length_bounds, void* stream) {
    using namespace pd;
    if (!q || !k || !v || !table || !lengths || !out || (!workspace && workspace_bytes > 0)) return PD_ERR_NULL_POINTER;
    if (!token_formats(q_dtype, kv_dtype)) return PD_ERR_DTYPE;
    if (!(k_scale > 0.0f && k_scale - k_scale == 0.0f && v_scale > 0.0f && v_scale - v_scale == 0.0f)) return PD_ERR_DTYPE;
    if (!token_shape(batch, tokens, query_heads, kv_heads, head_dim, page_size, table_width) || physical_pages < 1)
        return PD_ERR_SHAPE;
    if ((hints & ~(PD_HINT_UNSHARED_PAGES | PD_HINT_RAGGED_LENGTHS)) != 0) return PD_ERR_HINT;
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(out) || misaligned(workspace)) return PD_ERR_SHAPE;
    // Rows of one (sequence, KV head) and bytes of a cache row are 32-bit numbers.
    const int64_t rows = static_cast<int64_t>(tokens) * (query_heads / kv_heads);
    if (rows > (1 << 30)) return PD_ERR_SHAPE;
    const int64_t reach = static_cast<int64_t>(table_width) * page_size;
    int64_t bound = reach;
    if (length_bounds != nullptr) {
        bound = 0;
        for (int b = 0; b < batch; ++b) bound = std::max<int64_t>(bound, length_bounds[b]);
        bound = std::min(std::max<int64_t>(bound, 1), reach);
    }
    const int64_t max_states = static_cast<int64_t>(workspace_bytes / state_bytes(head_dim));
    TokenPlan plan = plan_tokens(q_dtype == PD_DTYPE_F32 ? 4 : 2, head_dim, batch, tokens, query_heads, kv_heads, bound,
                                       length_bounds, max_states, device_cus());
    if (token_workgroups(plan, kv_heads) * plan.waves * plan.groups * kWave > 0xFFFFFFFFLL) return PD_ERR_SHAPE;  // a launch's threads

    TokenParams p{};
    p.q = q;
    p.k = k;
    p.v = v;
    p.table = table;
    p.lengths = lengths;
    p.counts = counts;
    p.out = out;
    p.numerator = static_cast<float*>(workspace);
    p.stats = p.numerator + static_cast<size_t>(plan.states) * head_dim;
    p.batch = batch;
    p.tokens = tokens;
    p.query_heads = query_heads;
    p.kv_heads = kv_heads;
    p.group = query_heads / kv_heads;
    p.table_width = table_width;
    p.page_shift = page_size == 16 ? 4 : 5;
    p.physical_pages = physical_pages;
    p.causal = causal != 0;
    p.split = plan.split;
    p.items = plan.items;
    p.split_tokens = plan.split_tokens;
    p.tile_rows = plan.tile_rows;
    p.row_tiles = plan.row_tiles;
    p.head_waves = plan.head_waves;
    const int element = kv_dtype == PD_DTYPE_F32 ? 4 : kv_dtype == PD_DTYPE_F16 || kv_dtype == PD_DTYPE_BF16 ? 2 : 1;
    p.kv_row_bytes = static_cast<uint32_t>(kv_heads) * head_dim * element;
    p.scale_log2 = static_cast<float>(static_cast<double>(k_scale) / std::sqrt(static_cast<double>(head_dim)) * 1.4426950408889634);
    p.v_scale = v_scale;
    // K and V that the L2s hold stay cacheable (one sequence of 8192, 32 MB: 17.8 us, past the caches 18.4; 16 of 600, 38 MB: 17.9, 16.8).
    plan.once = (hints & PD_HINT_UNSHARED_PAGES) != 0 && 2 * batch * bound * p.kv_row_bytes > (32 << 20);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (q_dtype == PD_DTYPE_F32)
        return head_dim == 64 ? launch_tokens_f32_d64(p, plan, kv_dtype, s) : launch_tokens_f32_d128(p, plan, kv_dtype, s);
    if (q_dtype == PD_DTYPE_F16)
        return head_dim == 64 ? launch_tokens_f16_d64(p, plan, kv_dtype, s) : launch_tokens_f16_d128(p, plan, kv_dtype, s);
    return head_dim == 64 ? launch_tokens_bf16_d64(p, plan, kv_dtype, s) : launch_tokens_bf16_d128(p, plan, kv_dtype, s);
}

}  // extern "C"
