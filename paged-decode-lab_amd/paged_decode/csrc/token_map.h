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

#include <initializer_list>

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
    float* numerator;        // [items, kv_heads, rows of all tiles, D], where contexts are split
    float* stats;            // [items, kv_heads, rows of all tiles, 2]
    int batch, tokens;
    int query_heads, kv_heads, group;
    int table_width, page_shift, physical_pages;
    int causal;
    int split;               // how contexts are split: enum TokenSplit
    int items;               // (sequence, split) pairs of the launch
    int split_tokens;        // tokens per split, or more where the lengths outgrew what the host knew
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

// Contexts are whole (item = sequence), or cut into splits of split_tokens
// each. In a list, the sequences' splits follow one another, so that a short one
// takes no more items than it has tokens for; the device works out the list from the
// lengths, one lane a sequence (so up to kTokenListBatch of them), and takes longer splits where it
// would not fit the items. Larger batches have the same number of splits in every sequence.
enum TokenSplit { kTokenWhole = 0, kTokenList = 1, kTokenGrid = 2 };
constexpr int kTokenListBatch = 64;
constexpr int kTokenSplitUnit = 64;

PD_HD int token_ceil(int a, int b) { return (a + b - 1) / b; }

// Tokens per split of a sequence in a grid of `splits`: split_tokens, or more
// (a multiple of the unit) where the context outgrew what the host knew.
PD_HD int token_grid_span(int splits, int split_tokens, int context) {
    return imax(split_tokens, token_ceil(token_ceil(context, splits), kTokenSplitUnit) * kTokenSplitUnit);
}

// Workgroup `block` of the launch (one grid dimension). Tiles that see most come
// first, over all heads and items, so that what remains at the end is short; an
// (item, KV head) keeps its place modulo their number, so that with a multiple of
// eight of them its tiles, which read the same K and V, run on one XCD.
struct TokenCoords {
    int item, kv_head, tile;
};

PD_HD TokenCoords token_coords(const TokenParams& p, uint32_t block) {
    const uint32_t units = static_cast<uint32_t>(p.items * p.kv_heads);
    const uint32_t rank = block / units;
    const uint32_t unit = block - rank * units;
    TokenCoords c;
    c.tile = p.row_tiles - 1 - static_cast<int>(rank);
    c.item = static_cast<int>(unit / p.kv_heads);
    c.kv_head = static_cast<int>(unit - static_cast<uint32_t>(c.item) * p.kv_heads);
    return c;
}

// Stream kernel: wave w has KV head w % head_waves of the workgroup's. The
// workgroups of one item's KV heads follow one another on one XCD (eight of
// them, which take workgroups in turn), items in turn on the XCDs: heads in turn on them
// would have an XCD read the same few hundred bytes of every token's row, a part of its L2's channels.
// Items come in eights; those past the last one are empty.
constexpr int kXcds = 8;

PD_HD TokenCoords token_stream_coords(const TokenParams& p, uint32_t block, int wave) {
    const uint32_t head_groups = static_cast<uint32_t>(p.kv_heads / p.head_waves);
    const uint32_t slot = block / kXcds;
    const uint32_t unit = slot / head_groups;
    const uint32_t eight = unit / p.row_tiles;
    TokenCoords c;
    c.kv_head = static_cast<int>(slot - unit * head_groups) * p.head_waves + wave % p.head_waves;
    c.tile = static_cast<int>(unit - eight * p.row_tiles);
    c.item = static_cast<int>(eight * kXcds + block % kXcds);
    return c;
}

// State of row `row` (of the padded rows of all tiles) of (item, KV head).
PD_HD int64_t token_state(const TokenParams& p, int item, int kv_head, int row) {
    const int64_t rows = static_cast<int64_t>(p.row_tiles) * p.tile_rows;
    return (static_cast<int64_t>(item) * p.kv_heads + kv_head) * rows + row;
}

// Element offset of row `row` of (sequence, KV head) in q and out.
PD_HD int64_t token_q_row(const TokenParams& p, int b, int kv_head, int token, int head) {
    return (static_cast<int64_t>(b) * p.tokens + token) * p.query_heads + static_cast<int64_t>(kv_head) * p.group + head;
}

// 16-byte chunk position of chunk c of tile row r in LDS: chunks of a row are
// permuted so that neither the reads of one chunk of many rows (K) nor those
// of neighbouring rows that are transposed together (V: pairs of chunks of four rows;
// FP8 as stored: one chunk of four rows and of those 16 behind) meet in a bank. A read of 16 bytes a lane
// takes four rows from either end of 16 together with eight middle ones of the next chunk: the half of 16 rows that a row is in
// turns its pairs so that these differ (counted: no conflicts; without the turn a third of the LDS cycles, 239 -> 242 us of 2048 tokens).
// The permutation of a row is its own inverse, and that of 32 rows on (but for FP8 as stored: of 16) is the same.
template <int kRowBytes, bool kFp8>
PD_HD int token_slot_chunk(int r, int c) {
    if (kRowBytes == 64) return c ^ ((r >> 2) & 3) ^ ((r >> 4) & 1);                                     // FP8, D 64
    if (kRowBytes == 128 && kFp8) return c ^ ((((r >> 1) & 3) << 1) | (((r >> 3) ^ (r >> 4)) & 1));     // FP8, D 128
    const int half = (r >> 3) & 1;
    if (kRowBytes == 128) return c ^ ((((r >> 1) & 3) ^ (half << 1)) << 1) ^ half;                      // 16-bit, D 64
    if (kRowBytes == 256) return c ^ (((r & 7) ^ (half << 2)) << 1) ^ half;                             // 16-bit D 128, FP32 D 64
    return c ^ (r & 15);                                                                                // FP32, D 128
}

template <int kRowBytes, bool kFp8 = false>
PD_HD int token_chunk(int r, int c) {
    return r * (kRowBytes / 16) + token_slot_chunk<kRowBytes, kFp8>(r, c);
}

// ---------------------------------------------------------------------------
// Launch planning (host).

struct TokenPlan {
    bool stream;             // the kernel of few rows
    int tile_rows, row_tiles;
    int waves, head_waves;   // of a workgroup; stream kernel: KV heads among them
    int groups;              // tile kernel: see there
    bool products_first;     // tile kernel of 128 rows: see there
    bool once;               // stream kernel: see there; the caller's to set
    int split, items, split_tokens;
    int64_t workgroups;  // with whole contexts
    int64_t states;      // 0 with whole contexts
};

// Rows that the stream kernel takes: up to 16, and up to 32 where the tokens of all sequences and KV heads come to
// kStreamLoad per CU or q is FP32. Below, the tile kernel's splits have fewer states to merge (us, 32 heads on 8,
// stream / tile: FP16, 8 x 8 tokens on 4096 37 / 34, 16 x 8 on 1024 27.8 / 25.0, 2 x 5 on 1000 15.4 / 10.8; 16 x 8 on
// 4096 55.8 / 57.7, 40 x 8 on 1500 48.8 / 55.9; BF16, 12 x 8 on 8192 74.7 / 81.4; FP32, 16 x 5 on 2000 58 / 84).
constexpr int kStreamMaxRows = 32;
constexpr int kStreamLoad = 1600;
// Waves of its workgroups (FP32 rows of D 128 are twice as long: 4). With 4: FP32, 8 x 2 on 2048 34.6 us, with 8 31.5;
// E4M3, 16 x 8 on up to 8192 44.4, 45.5; others the same.
constexpr int kStreamWaves = 8;
// Cache tokens per split, at least: FP32 products take sixteen times as long (2 x 33 tokens on 1000: 13.2 us, with
// splits of 128 14.4), others pay more for the merge (BF16, 256 tokens on 256: 15.5 us, with splits of 64 16.4).
constexpr int token_min_split(int q_bytes) { return q_bytes == 4 ? 64 : 128; }
// Workgroups per CU that splits of the tile kernel aim at (FP16, 128 tokens on 16384: 65 us, with three 78).
constexpr int kTokenGroupsPerCu = 2;
// What splits cost, in cache tokens of a tile (of FP32 an eighth of as many): the merge's launch, and floats of states
// per token. Where two workgroups share a CU a token counts one and a half. By this rule, and against it (us, 32 heads
// on 8; FP16, 300 tokens on 600 whole 16.7, split 21.6; 256 on 256 whole 8.8, split 15.8; one on 200 whole 9.0, split
// 11.4; 16 x 2 on 600 split 16.8, whole 19.5; BF16, 512 on 4096 in four splits 53.4, in two 67.0; 1024 on 16384 split
// 291, whole 336).
constexpr int kTokenMergeCost = 280, kTokenStateCost = 128 * 120;

// Items of splits of `span` tokens.
inline int64_t token_items(int split, const int32_t* bounds, int batch, int64_t bound, int64_t span) {
    const int64_t most = (bound + span - 1) / span;
    if (split == kTokenGrid || bounds == nullptr) return batch * most;
    int64_t items = 0;
    for (int b = 0; b < batch; ++b) items += (lmin(imax(bounds[b], 0), bound) + span - 1) / span;
    return lmax(items, batch);
}

// Workgroups of a launch.
inline int64_t token_workgroups(const TokenPlan& t, int kv_heads) {
    if (!t.stream) return static_cast<int64_t>(t.items) * kv_heads * t.row_tiles;
    return static_cast<int64_t>((t.items + kXcds - 1) / kXcds * kXcds) * (kv_heads / t.head_waves) * t.row_tiles;
}

// Whether tiles of the tile kernel have 128 rows rather than 64: a tile of K and V in LDS then serves twice the rows, but
// there are half the workgroups. So where those of 128 rows fill the device (with D 64, whose products wait less on LDS,
// twice over), or do so in splits of 512 tokens of a context that is long next to the new tokens. Measured, 64 / 128 rows,
// 32 heads on 8: BF16, D 128, 1536 tokens on 8192 257 / 214 us, 512 on 4096 60 / 54, 1024 on 16384 339 / 291; 768 on 4096
// 77 / 85, 1024 on 1024 24 / 29; D 64, 512 on 4096 40 / 37, and 28 heads on 4, 5 sequences of 301 34 / 45.
inline bool wide_token_tiles(int q_bytes, int head_dim, int batch, int tokens, int64_t rows, int kv_heads, int64_t bound,
                             int64_t compute_units) {
    if (rows <= 64 || (q_bytes == 4 && head_dim == 128)) return false;  // (whose states of 128 rows the registers do not hold)
    const int64_t tiles = static_cast<int64_t>(batch) * kv_heads * ((rows + 127) / 128);
    if (head_dim == 128 ? tiles > compute_units : tiles >= kTokenGroupsPerCu * compute_units) return true;
    return bound >= 8 * static_cast<int64_t>(tokens) && tiles * (bound / 512) >= kTokenGroupsPerCu * compute_units;
}

// The launch without splits, and the workgroups that splits aim at.
inline TokenPlan plan_whole_tokens(int q_bytes, int head_dim, int batch, int tokens, int query_heads, int kv_heads,
                                   int64_t bound, int compute_units, int64_t& wanted) {
    TokenPlan t{};
    const int64_t rows = static_cast<int64_t>(tokens) * (query_heads / kv_heads);
    const int64_t load = static_cast<int64_t>(batch) * kv_heads * bound / compute_units;  // cache tokens per CU
    t.stream = rows <= 16 || (rows <= kStreamMaxRows && (q_bytes == 4 || load >= kStreamLoad));
    if (t.stream) {
        t.tile_rows = rows <= 16 ? 16 : 32;
        t.waves = q_bytes == 4 && head_dim == 128 ? kStreamWaves / 2 : kStreamWaves;
        // Two KV heads' rows lie side by side (us with two, one: 64 sequences of 2048 83, 91; E4M3, 16 x 8 on up to 8192 45.5, 49.4;
        // 4 x 4 on 4096 22.6, 21.0, one of 16384 19.5, 20.3).
        t.head_waves = kv_heads % 2 == 0 ? 2 : 1;
    } else {
        t.tile_rows = wide_token_tiles(q_bytes, head_dim, batch, tokens, rows, kv_heads, bound, compute_units) ? 128 : 64;
        t.waves = 4;
        t.head_waves = 1;
        t.products_first = t.tile_rows == 128 && bound >= 2 * static_cast<int64_t>(tokens);
    }
    t.row_tiles = static_cast<int>((rows + t.tile_rows - 1) / t.tile_rows);
    t.split = kTokenWhole;
    t.items = batch;
    t.split_tokens = 1 << 30;
    t.workgroups = static_cast<int64_t>(kv_heads / t.head_waves) * t.row_tiles * batch;
    t.groups = !t.stream && t.tile_rows == 64 && t.workgroups <= compute_units && 2 * t.workgroups > compute_units ? 2 : 1;
    wanted = static_cast<int64_t>(compute_units) * (t.stream ? 1 : kTokenGroupsPerCu);
    return t;
}

// q_bytes: of a q element. bound: cache tokens the host knows no sequence to
// exceed; bounds: and each of them (or null).
inline TokenPlan plan_tokens(int q_bytes, int head_dim, int batch, int tokens, int query_heads, int kv_heads, int64_t bound,
                             const int32_t* bounds, int64_t max_states, int compute_units) {
    int64_t wanted;
    TokenPlan t = plan_whole_tokens(q_bytes, head_dim, batch, tokens, query_heads, kv_heads, bound, compute_units, wanted);
    const int64_t each = t.workgroups / batch;  // workgroups of an item
    const int64_t states = static_cast<int64_t>(kv_heads) * t.row_tiles * t.tile_rows;  // and its states
    int64_t limit = lmin(wanted / each, max_states / states);  // items that fit the device at once
    if (t.stream && limit > kXcds) limit -= limit % kXcds;     // and each of its XCDs
    if (t.workgroups > compute_units || t.groups == 2 || limit <= batch) return t;
    const int split = batch <= kTokenListBatch ? kTokenList : kTokenGrid;
    // The shortest split with which the items fit; more tokens, fewer of them.
    int64_t low = token_min_split(q_bytes) / kTokenSplitUnit, high = (bound + kTokenSplitUnit - 1) / kTokenSplitUnit;
    while (low < high) {
        const int64_t mid = (low + high) / 2;
        if (token_items(split, bounds, batch, bound, mid * kTokenSplitUnit) <= limit) high = mid;
        else low = mid + 1;
    }
    // That, or of longer ones the cheapest, or none.
    int64_t best = bound, span = 0;
    for (int64_t x = low * kTokenSplitUnit; x < bound; x *= 2) {
        const int64_t items = token_items(split, bounds, batch, bound, x);
        const bool shared = !t.stream && items * each > compute_units;  // CUs by two workgroups, each then slower
        const int64_t fast = q_bytes == 4 ? 8 : 1;
        const int64_t cost = (shared ? x * 3 / 2 : x) + (kTokenMergeCost + items * states * head_dim / kTokenStateCost) / fast;
        if (cost < best) {
            best = cost;
            span = x;
        }
    }
    if (span == 0) return t;
    t.split = split;
    t.split_tokens = static_cast<int>(span);
    t.items = static_cast<int>(token_items(split, bounds, batch, bound, span));
    t.states = states * t.items;
    return t;
}

// States with which no call of up to `tokens` tokens splits less than it would with more, whatever its lengths: with
// the kernels of short and of long contexts.
inline int64_t most_token_states(int q_bytes, int head_dim, int batch, int tokens, int query_heads, int kv_heads, int64_t reach,
                                 int compute_units) {
    const int64_t splits = (reach + token_min_split(q_bytes) - 1) / token_min_split(q_bytes);
    int64_t most = 0;
    bool more = splits > 1;
    for (int n = 1; n <= tokens && more; ++n) {
        more = false;
        for (const int64_t bound : {int64_t{1}, reach}) {
            int64_t wanted;
            const TokenPlan t = plan_whole_tokens(q_bytes, head_dim, batch, n, query_heads, kv_heads, bound, compute_units, wanted);
            if (t.workgroups > compute_units && !t.stream) continue;  // and so for every larger n
            more = true;
            const int64_t items = lmin(wanted / (t.workgroups / batch), batch * splits);
            if (items > batch) most = lmax(most, items * kv_heads * t.row_tiles * t.tile_rows);
        }
    }
    return most;
}

}  // namespace pd

#endif  // PAGED_DECODE_TOKEN_MAP_H
