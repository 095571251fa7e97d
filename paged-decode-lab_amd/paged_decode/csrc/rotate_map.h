// Work and address map of the head norm / rotation kernels, shared by the
// device code in rotate.hip and the host: which token, head and dims a lane
// owns, and where it reads and writes them. Plain integer arithmetic (host and
// gfx950).
//
// A lane holds 16 dims of a head, as two chunks of eight that are rotated with
// each other: with halves paired (dims i and i + R/2 of the R rotated ones),
// chunk j of the first half and chunk j of the second; with neighbours paired
// (dims 2i and 2i + 1), sixteen dims in a row. Both need the angles of pairs
// 8 j to 8 j + 7, and nothing of another lane but the norm's sum of squares.
#ifndef PAGED_DECODE_ROTATE_MAP_H
#define PAGED_DECODE_ROTATE_MAP_H

#include "cache_map.h"

namespace pd {

constexpr int kRotateLaneDims = 16;  // dims of one lane: two chunks of eight
constexpr int kRotateChunk = 8;

// Token rows [batch, tokens, heads, head_dim] whose heads are contiguous and
// whose tokens and sequences lie `token_stride` and `batch_stride` elements
// apart (views of a fused projection).
struct TokenRows {
    const char* data;
    int64_t batch_stride, token_stride;
};

struct RotateParams {
    TokenRows q, k, v;       // data may be null: no such heads (v without a cache)
    char* q_out;             // [batch, tokens, query_heads, D]
    char* k_out;             // [batch, tokens, kv_heads, D] without a cache
    const int32_t* positions;  // [batch], or [batch, tokens] with per-token positions; null with an advance
    const int32_t* counts;   // live tokens per sequence, or null (all)
    const double* frequencies;  // radians per position of each pair, [rotary_dim / 2]
    const void* q_weight;    // norm weights, or null (no norm)
    const void* k_weight;
    AppendParams cache;      // table, lengths (advance), caches; k_new, v_new unused
    float eps, inv_dim, turn_scale, k_scale, v_scale;
    int batch, tokens;
    int q_heads, kv_heads;   // as launched: 0 for q or k left out
    int heads;               // q_heads + kv_heads (+ kv_heads with a cache)
    int head_groups;         // of a token: the heads that a wave holds at a time, a wave each
    int rotary_dim;          // 0: norm only
    int interleaved;
    int per_token_positions;
    int weight_f32;          // norm weights in FP32 (else the tokens' type)
    int q_weight_stride, k_weight_stride;  // elements between two heads' weights: 0 or D
    float largest;           // FP8 cache: its largest finite value
};

// Heads that one wave holds at a time.
PD_HD int rotate_heads_per_wave(int head_dim) { return kWave / (head_dim / kRotateLaneDims); }

// First dims of the two chunks of lane `j` of a head.
struct ChunkPair {
    int first, second;
};

PD_HD ChunkPair rotate_chunks(int rotary_dim, int interleaved, int j) {
    const int half_lanes = rotary_dim / kRotateLaneDims;
    if (!interleaved && j < half_lanes) return {j * kRotateChunk, j * kRotateChunk + rotary_dim / 2};
    return {j * kRotateLaneDims, j * kRotateLaneDims + kRotateChunk};
}

// Element offset of (sequence, token, head, dim) in token rows.
PD_HD int64_t token_row_offset(const TokenRows& r, int b, int token, int head, int head_dim) {
    return static_cast<int64_t>(b) * r.batch_stride + static_cast<int64_t>(token) * r.token_stride +
           static_cast<int64_t>(head) * head_dim;
}

}  // namespace pd

#endif  // PAGED_DECODE_ROTATE_MAP_H
