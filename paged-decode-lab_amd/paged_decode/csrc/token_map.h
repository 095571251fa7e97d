// Work map of the attention of several tokens per sequence, shared by the
// device code in token_kernels.h / tokens.hip and the host: which rows and
// cache tokens a workgroup takes, what a row sees, and where tiles lie in LDS.
// Plain integer arithmetic (host and gfx950).
//
// The query heads of one KV head and the tokens of one sequence are one list
// of rows: row = token * group + head of the group. A workgroup takes
// `tile_rows` of them and one split of the sequence's cache tokens.
#ifndef PAGED_DECODE_TOKEN_MAP_H
#define PAGED_DECODE_TOKEN_MAP_H

#include <stddef.h>

#include "partition_map.h"

namespace pd {

PD_HD int64_t lmax(int64_t a, int64_t b) { return a > b ? a : b; }

struct TokenParams {
    const void* q;
    const void* k;
    const void* v;
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* counts;   // or null: every token is live
    void* out;
    float* numerator;        // [rows of all tiles, splits, D], splits > 1 only
    float* stats;            // [rows of all tiles, splits, 2]
    int batch, tokens;
    int query_heads, kv_heads, group;
    int table_width, page_shift, physical_pages;
    int causal;
    int splits;              // of each sequence's cache tokens
    int split_tokens;        // tokens per split where `splits` of them reach the length
    int tile_rows, row_tiles;
    int head_waves;          // stream kernel: KV heads of a workgroup
    uint32_t kv_row_bytes;   // bytes from one cache token to the next: kv_heads * D * element
    float scale_log2;        // k_scale / sqrt(D) * log2(e)
    float v_scale;
};

// Live query tokens and cache tokens of sequence b.
PD_HD int token_count(const TokenParams& p, int b) {
    return p.counts ? imin(imax(p.counts[b], 0), p.tokens) : p.tokens;
}

PD_HD int token_context(const TokenParams& p, int b) {
    const int64_t reach = static_cast<int64_t>(p.table_width) << p.page_shift;
    return static_cast<int>(lmin(imax(p.lengths[b], 0), reach));
}

// Cache tokens that query token j of `count` sees.
PD_HD int token_sees(int causal, int context, int count, int j) {
    return causal ? imax(imin(context, context - count + j + 1), 0) : context;
}

// Tokens per split of a sequence: split_tokens, or more (a multiple of the
// unit) where the context outgrew what the host knew.
constexpr int kTokenSplitUnit = 64;

PD_HD int token_split(int splits, int split_tokens, int context) {
    const int even = (context + splits - 1) / splits;
    return imax(split_tokens, (even + kTokenSplitUnit - 1) / kTokenSplitUnit * kTokenSplitUnit);
}

// Workgroup `block` of the launch (one grid dimension). Tiles that see most come
// first, over all heads and splits, so that what remains at the end is short; a
// (sequence, KV head, split) keeps its place modulo their number, so that with a multiple of
// eight of them its tiles, which read the same K and V, run on one XCD.
struct TokenCoords {
    int b, kv_head, split, tile;
};

PD_HD TokenCoords token_coords(const TokenParams& p, uint32_t block) {
    const uint32_t units = static_cast<uint32_t>(p.batch * p.kv_heads * p.splits);
    const uint32_t rank = block / units;
    const uint32_t unit = block - rank * units;
    const uint32_t head = unit / p.splits;
    TokenCoords c;
    c.tile = p.row_tiles - 1 - static_cast<int>(rank);
    c.split = static_cast<int>(unit - head * p.splits);
    c.b = static_cast<int>(head / p.kv_heads);
    c.kv_head = static_cast<int>(head - static_cast<uint32_t>(c.b) * p.kv_heads);
    return c;
}

// Stream kernel: workgroups of one split's KV heads are neighbours, wave w has
// KV head w % head_waves of the workgroup's. Later splits, which short sequences
// have nothing in, come last.
PD_HD TokenCoords token_stream_coords(const TokenParams& p, uint32_t block, int wave) {
    const uint32_t head_groups = static_cast<uint32_t>(p.kv_heads / p.head_waves);
    const uint32_t unit = block / head_groups;
    const uint32_t part = unit / p.row_tiles;
    TokenCoords c;
    c.kv_head = static_cast<int>(block - unit * head_groups) * p.head_waves + wave % p.head_waves;
    c.tile = static_cast<int>(unit - part * p.row_tiles);
    c.split = static_cast<int>(part / p.batch);
    c.b = static_cast<int>(part - static_cast<uint32_t>(c.split) * p.batch);
    return c;
}

// State of row `row` (of the padded rows of all tiles) of (sequence, KV head) in split s.
PD_HD int64_t token_state(const TokenParams& p, int b, int kv_head, int row, int s) {
    const int64_t rows = static_cast<int64_t>(p.row_tiles) * p.tile_rows;
    return ((static_cast<int64_t>(b) * p.kv_heads + kv_head) * rows + row) * p.splits + s;
}

// Element offset of row `row` of (sequence, KV head) in q and out.
PD_HD int64_t token_q_row(const TokenParams& p, int b, int kv_head, int token, int head) {
    return (static_cast<int64_t>(b) * p.tokens + token) * p.query_heads + static_cast<int64_t>(kv_head) * p.group + head;
}

// 16-byte chunk position of chunk c of tile row r in LDS: chunks of a row are
// permuted so that neither the reads of one chunk of many rows (K) nor those
// of pairs of chunks of four rows (V, transposing) meet in a bank.
template <int kRowBytes>
PD_HD int token_chunk(int r, int c) {
    if (kRowBytes == 128) return r * 8 + (c ^ ((((r >> 1) & 3) << 1) | ((r >> 3) & 1)));      // 16-bit, D 64
    if (kRowBytes == 256) return r * 16 + (c ^ (((r & 7) << 1) | ((r >> 3) & 1)));            // 16-bit D 128, FP32 D 64
    return r * 32 + (c ^ (r & 15));                                                          // FP32, D 128
}

// The chunk of row r that lies at position `slot` of the row's chunks: the
// permutation is its own inverse.
template <int kRowBytes>
PD_HD int token_slot_chunk(int r, int slot) {
    return token_chunk<kRowBytes>(r, slot) - r * (kRowBytes / 16);
}

// ---------------------------------------------------------------------------
// Launch planning (host).

struct TokenPlan {
    bool stream;             // the kernel of few rows
    int tile_rows, row_tiles;
    int waves, head_waves;   // of a workgroup; stream kernel: KV heads among them
    int splits, split_tokens;
    int64_t workgroups;
    int64_t states;  // 0 with one split
};

constexpr int kStreamMaxRows = 32;     // rows that the stream kernel takes
constexpr int kStreamWaves = 8;        // waves of its workgroups (FP32 rows are twice as long: 4)
constexpr int kTokenMinSplit = 128;    // cache tokens per split, at least
constexpr int kTokenGroupsPerCu = 2;   // workgroups per CU that splits of the tile kernel aim at

// The workgroups that a launch with splits of `span` tokens has anything to do in.
inline int64_t live_splits(const int32_t* bounds, int batch, int64_t bound, int64_t span) {
    if (bounds == nullptr) return batch * ((bound + span - 1) / span);
    int64_t live = 0;
    for (int b = 0; b < batch; ++b) live += (lmin(imax(bounds[b], 0), bound) + span - 1) / span;
    return live;
}

// Splits that `unsplit` workgroups are cut into at most: 1 if they fill the device.
inline int64_t token_most_splits(int64_t unsplit, int64_t wanted) { return unsplit >= wanted ? 1 : 4 * wanted / unsplit; }

// q_bytes: of a q element. bound: cache tokens the host knows no sequence to
// exceed; bounds: and each of them (or null).
inline TokenPlan plan_tokens(int q_bytes, int head_dim, int batch, int tokens, int query_heads, int kv_heads, int64_t bound,
                             const int32_t* bounds, int64_t max_states, int compute_units) {
    TokenPlan t{};
    const int64_t rows = static_cast<int64_t>(tokens) * (query_heads / kv_heads);
    t.stream = rows <= kStreamMaxRows;
    if (t.stream) {
        t.tile_rows = rows <= 16 ? 16 : 32;
        t.waves = q_bytes == 4 && head_dim == 128 ? kStreamWaves / 2 : kStreamWaves;
        t.head_waves = kv_heads % 2 == 0 ? 2 : 1;
    } else {
        t.tile_rows = rows <= 64 || (q_bytes == 4 && head_dim == 128) ? 64 : 128;
        t.waves = 4;
        t.head_waves = 1;
    }
    t.row_tiles = static_cast<int>((rows + t.tile_rows - 1) / t.tile_rows);
    // Workgroups of one sequence's split, and how many the device should get.
    const int64_t each = static_cast<int64_t>(kv_heads / t.head_waves) * t.row_tiles;
    const int64_t wanted = static_cast<int64_t>(compute_units) * (t.stream ? 1 : kTokenGroupsPerCu);
    const int64_t states = static_cast<int64_t>(batch) * kv_heads * t.row_tiles * t.tile_rows;  // of one split
    // The shortest split with which the workgroups still fit the device at once; those that find nothing to do,
    // a short sequence's in later splits, count a quarter.
    const int64_t limit = lmin(token_most_splits(each * batch, wanted), max_states / states);
    int64_t span = bound;
    if (limit > 1) {
        const int64_t least = lmax(kTokenMinSplit, (bound + limit - 1) / limit);
        int64_t low = (least + kTokenSplitUnit - 1) / kTokenSplitUnit, high = (bound + kTokenSplitUnit - 1) / kTokenSplitUnit;
        while (low < high) {  // units of tokens; more of them, fewer workgroups
            const int64_t mid = (low + high) / 2;
            if (each * live_splits(bounds, batch, bound, mid * kTokenSplitUnit) <= wanted) high = mid;
            else low = mid + 1;
        }
        span = low * kTokenSplitUnit;
    }
    t.splits = static_cast<int>((bound + span - 1) / span);
    t.split_tokens = t.splits > 1 ? static_cast<int>(span) : kTokenSplitUnit;
    t.workgroups = each * batch * t.splits;
    t.states = t.splits > 1 ? states * t.splits : 0;
    return t;
}

// States with which no call of up to `tokens` tokens splits less than it would with
// more: a split has at least kTokenMinSplit tokens, and unsplit calls at least `wanted` workgroups.
inline int64_t most_token_states(int q_bytes, int head_dim, int batch, int tokens, int query_heads, int kv_heads, int64_t reach,
                                 int compute_units) {
    int64_t most = 0;
    for (int n = 1; n <= tokens; ++n) {
        const TokenPlan t = plan_tokens(q_bytes, head_dim, batch, n, query_heads, kv_heads, reach, nullptr, 0, compute_units);
        const int64_t wanted = static_cast<int64_t>(compute_units) * (t.stream ? 1 : kTokenGroupsPerCu);
        if (t.workgroups >= wanted) {
            if (t.stream) continue;
            break;  // and so for every larger n
        }
        const int64_t splits = lmin(token_most_splits(t.workgroups, wanted), (reach + kTokenMinSplit - 1) / kTokenMinSplit);
        const int64_t states = static_cast<int64_t>(batch) * kv_heads * t.row_tiles * t.tile_rows;
        if (splits > 1 && splits * states > most) most = splits * states;
    }
    return most;
}

}  // namespace pd

#endif  // PAGED_DECODE_TOKEN_MAP_H
