"""The work map of the attention of several tokens (token_map.h): the chunk permutations of tiles in LDS, that plans keep
to their workspace and cover every token, and that a launch's workgroups are every (item, KV head, tile) once."""
import subprocess

from gpu_util import no_child_processes_after_gpu_init
from test_address_audit import CSRC, compiler

SOURCE = r"""
#include <stdio.h>
#include <initializer_list>
#include <random>
#include <set>
#include <tuple>
#include <vector>
#include "token_map.h"
using namespace pd;
static long checks = 0, bad = 0;
static void check(bool ok) { ++checks; bad += !ok; }

template <int kRowBytes, bool kFp8>
void permutation() {
    const int period = kFp8 ? 32 : 16;  // of which the kernel adds multiples to a lane's address
    for (int r = 0; r < 64; ++r) {
        std::set<int> seen;
        for (int c = 0; c < kRowBytes / 16; ++c) {
            const int at = token_slot_chunk<kRowBytes, kFp8>(r, c);
            seen.insert(at);
            check(at >= 0 && at < kRowBytes / 16 && token_slot_chunk<kRowBytes, kFp8>(r, at) == c);
            check(token_slot_chunk<kRowBytes, kFp8>(r + period, c) == at);
        }
        check(seen.size() == kRowBytes / 16);
    }
    // One 16-byte chunk of 16 rows: every bank of 256 bytes alike often.
    if (kFp8) return;
    for (int c = 0; c < kRowBytes / 16; ++c) {
        int uses[16] = {};
        for (int r = 0; r < 16; ++r) ++uses[token_chunk<kRowBytes, kFp8>(r, c) % 16];
        for (int b = 0; b < 16; ++b) check(uses[b] == 1);
    }
}

int main() {
    permutation<64, true>();
    permutation<128, true>();
    permutation<128, false>();
    permutation<256, false>();
    permutation<512, false>();
    std::mt19937 rng(7);
    auto between = [&](int low, int high) { return std::uniform_int_distribution<int>(low, high)(rng); };
    int kinds[3] = {}, wide = 0, groups = 0, streams = 0;
    for (int round = 0; round < 20000; ++round) {
        const int q_bytes = between(0, 2) ? 2 : 4, dim = between(0, 1) ? 128 : 64, batch = between(0, 3) ? between(1, 20) : between(1, 200);
        const int kv = batch > kTokenListBatch ? between(1, 2) : between(1, 16), query = kv * between(1, 9), most = 1 << between(0, 12), tokens = between(1, most), cus = between(0, 4) ? 256 : between(1, 304);
        const int64_t reach = int64_t(16) << between(0, 12), bound = between(1, int(reach));
        std::vector<int32_t> bounds(batch);
        for (auto& b : bounds) b = between(-3, int(bound));
        bounds[between(0, batch - 1)] = int(bound);
        const int64_t room = most_token_states(q_bytes, dim, batch, tokens, query, kv, reach, cus);
        const int64_t states = between(0, 3) ? room : between(0, int(room));
        const bool known = between(0, 3) != 0;
        const TokenPlan t = plan_tokens(q_bytes, dim, batch, tokens, query, kv, bound, known ? bounds.data() : nullptr, states, cus);
        const int64_t rows = int64_t(tokens) * (query / kv);
        check(int64_t(t.row_tiles) * t.tile_rows >= rows && int64_t(t.row_tiles - 1) * t.tile_rows < rows);
        check((t.stream || rows > 16) && (!t.stream || rows <= kStreamMaxRows) && kv % t.head_waves == 0 && t.waves % t.head_waves == 0);
        check(q_bytes == 2 || dim == 64 || t.stream || t.tile_rows == 64);
        ++kinds[t.split], wide += t.tile_rows == 128, groups += t.groups == 2, streams += t.stream;
        TokenParams p{};
        p.batch = batch, p.tokens = tokens, p.query_heads = query, p.kv_heads = kv, p.items = t.items, p.row_tiles = t.row_tiles;
        p.tile_rows = t.tile_rows, p.head_waves = t.head_waves, p.split = t.split, p.split_tokens = t.split_tokens;
        if (t.split == kTokenWhole) {
            check(t.items == batch && t.states == 0 && t.split_tokens >= bound);
        } else {
            check(t.states == int64_t(t.items) * kv * t.row_tiles * t.tile_rows && t.states <= states);
            check(t.split_tokens % kTokenSplitUnit == 0 && t.split_tokens < bound && t.items >= batch);
            check(t.split == (batch <= kTokenListBatch ? kTokenList : kTokenGrid) && t.groups == 1);
            check(token_state(p, t.items - 1, kv - 1, t.row_tiles * t.tile_rows - 1) == t.states - 1);
            int64_t sum = 0;
            for (int b = 0; b < batch; ++b) sum += token_ceil(imax(known ? bounds[b] : int(bound), 0), t.split_tokens);
            check(sum <= t.items);
            if (t.split == kTokenGrid) {  // also where lengths outgrew the bounds
                const int splits = t.items / batch;
                check(t.items % batch == 0);
                for (int length : {0, 1, int(bound), int(reach)}) check(int64_t(splits) * token_grid_span(splits, t.split_tokens, length) >= length);
            }
        }
        const int64_t count = token_workgroups(t, kv);
        if (count > 4000) continue;
        std::set<std::tuple<int, int, int, int>> seen;
        for (int64_t block = 0; block < count; ++block)
            for (int wave = 0; wave < (t.stream ? t.waves : 1); ++wave) {
                const TokenCoords c = t.stream ? token_stream_coords(p, block, wave) : token_coords(p, block);
                check(c.kv_head >= 0 && c.kv_head < kv && c.tile >= 0 && c.tile < t.row_tiles && c.item >= 0);
                if (c.item < t.items) check(seen.emplace(c.item, c.kv_head, c.tile, t.stream ? wave / t.head_waves : 0).second);
            }
        check(int64_t(seen.size()) == int64_t(t.items) * kv * t.row_tiles * (t.stream ? t.waves / t.head_waves : 1));
    }
    for (int k : kinds) check(k > 100);
    check(wide > 100 && groups > 100 && streams > 100);
    printf("%ld checks, %ld bad\n", checks, bad);
    return bad != 0;
}
"""


def test_plans_cover_every_token_and_keep_to_their_workspace(tmp_path):
    no_child_processes_after_gpu_init()
    source, exe = tmp_path / "map.cpp", tmp_path / "map"
    source.write_text(SOURCE)
    subprocess.run([compiler("g++"), "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{CSRC}", str(source), "-o", str(exe)], check=True,
                   capture_output=True, text=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and ", 0 bad" in run.stdout, run.stdout
