"""Attention of several tokens per sequence on the GPU against 64-bit results (tests/rotary_oracle.py)."""
import ctypes
import math

import numpy as np
import pytest

from gpu_util import announce, require_gpu

require_gpu()

import torch  # noqa: E402

import rotary_oracle as oracle  # noqa: E402
from paged_decode import cabi  # noqa: E402
from paged_decode.layout import Layout  # noqa: E402
from paged_decode.rotary import Rotary, append_rotated, rotate_heads  # noqa: E402
from paged_decode.runtime import DecodePlan  # noqa: E402

pytestmark = pytest.mark.gpu

FORMATS = [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
           (torch.float16, torch.float8_e4m3fn), (torch.float16, torch.float8_e5m2),
           (torch.bfloat16, torch.float8_e4m3fn), (torch.bfloat16, torch.float8_e5m2)]


def problem(layout, q_type, kv_type, tokens, width, seed, spread=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    table = np.random.default_rng(seed).permutation(layout.physical_pages)[:layout.batch * width]
    table = table.reshape(layout.batch, width).astype(np.int32)
    shape = (layout.physical_pages, layout.page_size, layout.kv_heads, layout.head_dim)
    k, v = (torch.randn(shape, device="cuda", generator=gen).to(kv_type) for _ in range(2))
    q = (spread * torch.randn((layout.batch, tokens, layout.query_heads, layout.head_dim), device="cuda", generator=gen)).to(q_type)
    return table, q, k, v


def gathered(cache, pages, length, page_size):
    """[length, Hkv, D] of a sequence; None for the pages outside the cache."""
    wide = cache.view(torch.uint8) if cache.dtype.itemsize == 1 else cache
    ids = torch.from_numpy(np.clip(pages, 0, cache.shape[0] - 1)).long().cuda()
    rows = wide[ids].view(cache.dtype) if cache.dtype.itemsize == 1 else wide[ids]
    return rows.flatten(0, 1)[:length].float()


def check(layout, table, lengths, counts, q, k, v, out, causal, k_scale=1.0, v_scale=1.0):
    tokens = q.shape[1]
    for b in range(layout.batch):
        c = tokens if counts is None else min(max(int(counts[b]), 0), tokens)
        n = min(max(int(lengths[b]), 0), table.shape[1] * layout.page_size)
        live = -(-n // layout.page_size)
        bad = (table[b, :live] < 0) | (table[b, :live] >= layout.physical_pages)
        hidden = torch.from_numpy(np.repeat(bad, layout.page_size)[:n]).cuda()
        j = torch.arange(c, device="cuda")
        sees = (n - c + j + 1).clamp(0, n) if causal else torch.full_like(j, n)
        keys, values = (gathered(x, table[b, :live], n, layout.page_size) for x in (k, v))
        keys, values = (torch.where(hidden[:, None, None], 0.0, x) for x in (keys, values))
        expected, bound = oracle.attention(q[b, :c], keys, values, sees, k_scale, v_scale, hidden)
        oracle.assert_within(out[b, :c], expected, bound, q.dtype, f"sequence {b}")
        assert not out[b, c:].any()


def run(layout, table, lengths, q, k, v, *, counts=None, causal=True, k_scale=1.0, v_scale=1.0, width_tokens=None):
    plan = DecodePlan(layout, table, lengths, query_tokens=q.shape[1])
    out = torch.full_like(q, float("nan"))
    device_counts = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    got = plan.run_tokens(q, k, v, causal=causal, counts=device_counts, k_scale=k_scale, v_scale=v_scale, out=out)
    assert got is out
    own = plan.run_tokens(q, k, v, causal=causal, counts=device_counts, k_scale=k_scale, v_scale=v_scale)
    assert own.shape == q.shape and own.dtype == q.dtype and own.data_ptr() != out.data_ptr()
    assert torch.equal(own.view(torch.uint8), out.view(torch.uint8))  # the same call again, bit for bit
    check(layout, table, lengths, counts, q, k, v, out, causal, k_scale, v_scale)
    return plan


@pytest.mark.parametrize("q_type,kv_type", FORMATS, ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 64, 16), (7, 1, 128, 32), (6, 6, 128, 16)])
@pytest.mark.parametrize("causal", [True, False])
def test_ragged_lengths_and_counts(q_type, kv_type, heads, kv_heads, dim, page, causal):
    announce(f"tokens {q_type}/{kv_type} heads={heads}/{kv_heads} D={dim} page={page} causal={causal}")
    layout = Layout(6, heads, kv_heads, dim, page, 80)
    table, q, k, v = problem(layout, q_type, kv_type, 21, 13 if page == 16 else 7, seed=heads + dim)
    lengths = np.array([0, 1, 21, page * 6 + 1, 33, 64], dtype=np.int32)
    counts = [21, 1, 21, 5, 0, 30]
    scale = 1.0 if kv_type.itemsize > 1 else 0.7
    run(layout, table, lengths, q, k, v, counts=counts, causal=causal, k_scale=scale, v_scale=1.5 * scale)


@pytest.mark.parametrize("tokens", [1, 2, 4, 5, 8, 16, 17, 31, 64, 65, 130])
@pytest.mark.parametrize("context", [131, 700, 5000])
def test_token_counts_and_contexts(tokens, context):
    """Row tiles that end inside a token, contexts that are split over workgroups and are not."""
    announce(f"tokens n={tokens} L={context}")
    layout = Layout(2, 10, 2, 64, 16, 2 * 313)
    table, q, k, v = problem(layout, torch.float16, torch.float16, tokens, 313, seed=tokens)
    run(layout, table, np.array([context, max(context - 67, tokens)], dtype=np.int32), q, k, v)


@pytest.mark.parametrize("q_type,kv_type", FORMATS[:4], ids=str)
@pytest.mark.parametrize("dim", [64, 128])
def test_prompts(q_type, kv_type, dim):
    announce(f"prompt {q_type}/{kv_type} D={dim}")
    layout = Layout(2, 8, 2, dim, 32, 80)
    table, q, k, v = problem(layout, q_type, kv_type, 600, 40, seed=dim, spread=2.0)
    run(layout, table, np.array([600, 1203], dtype=np.int32), q, k, v)


@pytest.mark.parametrize("q_type,kv_type", FORMATS[:4], ids=str)
def test_large_scores_and_growing_maxima(q_type, kv_type):
    """Scores that grow along the context by far more than a rescaling step, and one far above the others."""
    announce(f"growing scores {q_type}/{kv_type}")
    layout = Layout(2, 4, 2, 64, 16, 40)
    table, q, k, v = problem(layout, q_type, kv_type, 9, 20, seed=2, spread=3.0)
    k = (k.float() * torch.linspace(0.1, 6.0, 40, device="cuda")[torch.from_numpy(np.argsort(table.ravel())).cuda()][:, None, None, None]).to(kv_type)
    run(layout, table, np.array([320, 250], dtype=np.int32), q, k, v)


@pytest.mark.parametrize("q_type,kv_type", [FORMATS[0], FORMATS[1], FORMATS[3]], ids=str)
def test_invalid_pages_are_skipped(q_type, kv_type):
    announce(f"invalid pages {q_type}/{kv_type}")
    layout = Layout(3, 4, 2, 64, 16, 60)
    table, q, k, v = problem(layout, q_type, kv_type, 12, 20, seed=3)
    lengths = np.array([300, 47, 16], dtype=np.int32)
    plan = DecodePlan(layout, table, lengths, query_tokens=12)
    table = table.copy()
    table[0, 3], table[0, 18], table[1, 2], table[2, 0] = -1, 60, 1 << 30, -7  # past the host's checks
    plan._table.copy_(torch.from_numpy(table))
    for causal in (True, False):
        out = plan.run_tokens(q, k, v, causal=causal)
        check(layout, table, lengths, None, q, k, v, out, causal)
    assert not out[2].any()


@pytest.mark.parametrize("q_type,kv_type", [FORMATS[0], FORMATS[1], FORMATS[2], FORMATS[4]], ids=str)
@pytest.mark.parametrize("tokens,context", [(3, 200), (40, 200), (6, 3000)])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_hidden_infinities_and_nan_reach_no_row(q_type, kv_type, tokens, context, value):
    """K and V of the last token, and of slots behind it, are not finite: rows that do not see them stay as they were."""
    announce(f"hidden {value} {q_type}/{kv_type} n={tokens} L={context}")
    layout = Layout(1, 4, 2, 64, 16, 190)
    table, q, k, v = problem(layout, q_type, kv_type, tokens, 190, seed=5)
    lengths = np.array([context], dtype=np.int32)
    clean = [x.clone() for x in (k, v)]
    for x in (k, v):
        page = x[int(table[0, (context - 1) // 16])]
        page[(context - 1) % 16, 1] = value
        for slot in range(context, -(-context // 16) * 16):
            page[slot % 16] = value
    plan = DecodePlan(layout, table, lengths, query_tokens=tokens)
    out = plan.run_tokens(q, k, v)[0]
    keys, values = (gathered(x, table[0, :-(-context // 16)], context, 16) for x in clean)
    sees = torch.arange(tokens, device="cuda") + context - tokens + 1
    full, bound = oracle.attention(q[0], keys, values, sees)
    oracle.assert_within(out[:-1], full[:-1], bound[:-1], q.dtype)
    oracle.assert_within(out[-1:, :2], full[-1:, :2], bound[-1:, :2], q.dtype)  # heads of the other KV head
    assert not torch.isfinite(out[-1, 2:]).any()


def test_captured_append_and_attention_replay():
    """A graph of rotated appends and of attention over what they wrote, replayed as contexts grow past the captured ones."""
    announce("captured append and attention")
    layout = Layout(3, 8, 2, 128, 16, 3 * 64)
    table = np.random.default_rng(7).permutation(192).reshape(3, 64).astype(np.int32)
    lengths = np.array([10, 0, 300], dtype=np.int32)
    tokens = 5
    plan = DecodePlan(layout, table, lengths, max_context=1024, query_tokens=tokens)
    gen = torch.Generator(device="cuda").manual_seed(1)
    f = torch.pow(torch.tensor(10000.0, dtype=torch.float64), -torch.arange(64, dtype=torch.float64) / 64)
    rotary = Rotary(f)
    k, v = (torch.randn((192, 16, 2, 128), device="cuda", generator=gen).half() for _ in range(2))
    qkv = torch.randn((3, tokens, 12, 128), device="cuda", generator=gen).half()
    counts = torch.full((3,), tokens, dtype=torch.int32, device="cuda")
    q, k_new, v_new = torch.split(qkv, (8, 2, 2), dim=2)
    q_rot, out = torch.empty((3, tokens, 8, 128), device="cuda", dtype=torch.float16), None
    plan.run_tokens(q_rot.zero_(), k, v)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            plan.append_rotated(k, v, k_new, v_new, rotary, q=q, counts=counts, out=q_rot)
            out = plan.run_tokens(q_rot, k, v, counts=counts)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    host_k, host_v = k.clone(), v.clone()
    now = lengths.copy()
    for step in range(40):
        qkv.copy_(torch.randn(qkv.shape, device="cuda", generator=gen).half())
        c = np.random.default_rng(step).integers(0, tokens + 1, size=3).astype(np.int32)
        counts.copy_(torch.from_numpy(c))
        graph.replay()
        torch.cuda.synchronize()
        positions = torch.from_numpy(now).cuda()
        q_now = append_rotated(layout, host_k, host_v, torch.from_numpy(table).cuda(), positions, k_new, v_new, rotary, q=q,
                               counts=counts)
        now = now + c
        np.testing.assert_array_equal(plan._lengths.cpu().numpy(), now)
        assert torch.equal(host_k, k) and torch.equal(host_v, v) and torch.equal(q_now, q_rot)
        if step % 8 == 0:
            check(layout, table, now, c, q_rot, k, v, out, True)
    check(layout, table, now, c, q_rot, k, v, out, True)


def test_one_token_agrees_with_the_decode_and_prompts_in_chunks_with_whole_ones():
    """The operators together: a prompt written and attended whole, in chunks, and token by token."""
    announce("prompt whole, in chunks and by tokens")
    layout = Layout(2, 8, 4, 64, 16, 40)
    table = np.random.default_rng(1).permutation(40).reshape(2, 20).astype(np.int32)
    gen = torch.Generator(device="cuda").manual_seed(2)
    f = torch.pow(torch.tensor(10000.0, dtype=torch.float64), -torch.arange(32, dtype=torch.float64) / 32)
    weights = [torch.rand(64, device="cuda", generator=gen).bfloat16() + 0.5 for _ in range(2)]
    rotary, n = Rotary(f, style="interleaved"), 130
    q, k_new, v_new = (torch.randn((2, n, h, 64), device="cuda", generator=gen).bfloat16() for h in (8, 4, 4))
    results = []
    for chunk in (n, 33, 1):
        plan = DecodePlan(layout, table, np.zeros(2, dtype=np.int32), max_context=320, query_tokens=chunk)
        k, v = (torch.zeros((40, 16, 4, 64), device="cuda", dtype=torch.bfloat16) for _ in range(2))
        parts = []
        for s in range(0, n, chunk):
            e = min(s + chunk, n)
            rotated = plan.append_rotated(k, v, k_new[:, s:e], v_new[:, s:e], rotary, q=q[:, s:e], q_weight=weights[0],
                                          k_weight=weights[1])
            parts.append(plan.run_tokens(rotated, k, v).clone())
            if chunk == 1:
                single = plan.run(rotated[:, 0].contiguous(), k, v)
                sees = torch.tensor([e], device="cuda")
                for b in range(2):
                    keys, values = (gathered(x, table[b, :-(-e // 16)], e, 16) for x in (k, v))
                    exact, bound = oracle.attention(rotated[b], keys, values, sees)
                    oracle.assert_within(single[b:b + 1].double(), exact, bound, torch.float32)
                    oracle.assert_within(parts[-1][b], exact, bound, torch.bfloat16)
        np.testing.assert_array_equal(plan._lengths.cpu().numpy(), [n, n])
        results.append((torch.cat(parts, 1), k, v))
    positions = torch.zeros(2, dtype=torch.int32, device="cuda")
    rotated, _ = rotate_heads(q, None, positions, rotary, q_weight=weights[0])
    for out, k, v in results:
        assert torch.equal(k, results[0][1]) and torch.equal(v, results[0][2])
        check(layout, table, np.array([n, n]), None, rotated, k, v, out, True)


def test_bounds_below_the_lengths_and_another_stream():
    """Lengths that grew on the device, seen through host bounds of before; a plan on a stream of its own."""
    announce("stale bounds, another stream")
    layout = Layout(2, 4, 2, 128, 32, 400)
    table, q, k, v = problem(layout, torch.bfloat16, torch.bfloat16, 4, 200, seed=9)
    plan = DecodePlan(layout, table, np.array([40, 6000], dtype=np.int32), max_context=6400, query_tokens=4)
    lengths = np.array([6399, 5000], dtype=np.int32)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        plan._lengths.copy_(torch.from_numpy(lengths))
        plan._bounds.copy_(torch.tensor([40, 700], dtype=torch.int32))
        out = plan.run_tokens(q, k, v)
    stream.synchronize()
    check(layout, table, lengths, None, q, k, v, out, True)


def test_refusals():
    announce("tokens refusals")
    layout = Layout(2, 4, 2, 64, 16, 8)
    table, q, k, v = problem(layout, torch.float16, torch.float16, 3, 4, seed=1)
    plan = DecodePlan(layout, table, np.array([9, 9]), query_tokens=3)
    with pytest.raises(ValueError):
        DecodePlan(layout, table, np.array([9, 9])).run_tokens(q, k, v)
    with pytest.raises(ValueError):
        plan.run_tokens(torch.cat((q, q), 1), k, v)                       # more than reserved
    with pytest.raises(ValueError):
        plan.run_tokens(q[:, 0], k, v)
    with pytest.raises(TypeError):
        plan.run_tokens(q.float(), k, v)
    with pytest.raises(ValueError):
        plan.run_tokens(q.transpose(1, 2).contiguous().transpose(1, 2), k, v)
    with pytest.raises(ValueError):
        plan.run_tokens(q.clone().requires_grad_(), k, v)
    with pytest.raises(ValueError):
        plan.run_tokens(q, k, v, k_scale=0.0)
    with pytest.raises(TypeError):
        plan.run_tokens(q, k, v, counts=torch.ones(2, device="cuda"))
    with pytest.raises(ValueError):
        plan.run_tokens(q, k, v, counts=torch.ones(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        plan.run_tokens(q, k, v, out=torch.empty_like(q, dtype=torch.float32))
    with pytest.raises(ValueError):
        plan.run_tokens(q, k, v, out=q)


@pytest.mark.parametrize("batch", [1, 3, 7])
def test_short_calls_repeat_bit_for_bit(batch):
    """Items are dealt to eight groups of workgroups; those without an item may not touch the last sequence's rows, whenever
    they run."""
    announce(f"repeated short calls of {batch} sequences")
    layout = Layout(batch, 8, 4, 64, 16, 4 * batch)
    table, q, k, v = problem(layout, torch.bfloat16, torch.bfloat16, 1, 4, seed=31)
    lengths = np.full(batch, 64, dtype=np.int32)
    plan = DecodePlan(layout, table, lengths, query_tokens=1)
    first = plan.run_tokens(q, k, v)
    check(layout, table, lengths, None, q, k, v, first, True)
    outs = torch.full((4000, *q.shape), float("nan"), device="cuda", dtype=q.dtype)
    for out in outs:
        plan.run_tokens(q, k, v, out=out)
    assert torch.equal(outs.view(torch.int16), first.view(torch.int16).expand(outs.shape))


# Which kernel a shape takes on 256 CUs: tiles of 64 rows by two groups of waves (129 to 256 of them), by one in splits, of 128 rows
# (more than 256 of them, or long contexts) with short and with long contexts, in splits, and the grid of splits of more than 64
# sequences by either kernel.
SHAPES = [(5, 8, 8, 64, 300, 420), (5, 8, 8, 128, 290, 500), (3, 4, 1, 64, 40, 1900), (17, 8, 8, 128, 160, 200), (17, 8, 8, 128, 160, 420),
          (17, 16, 16, 64, 150, 330), (2, 8, 8, 128, 160, 8200), (66, 2, 1, 128, 3, 1700), (70, 1, 1, 64, 40, 900)]


@pytest.mark.parametrize("q_type,kv_type", [FORMATS[0], FORMATS[2], FORMATS[3]], ids=str)
@pytest.mark.parametrize("batch,heads,kv_heads,dim,tokens,context", SHAPES)
def test_launches_of_every_kind(q_type, kv_type, batch, heads, kv_heads, dim, tokens, context):
    announce(f"launch of {batch} x {tokens} on {context}, {heads}/{kv_heads} heads of {dim}, {q_type}/{kv_type}")
    width = -(-context // 16)
    layout = Layout(batch, heads, kv_heads, dim, 16, batch * width)
    table, q, k, v = problem(layout, q_type, kv_type, tokens, width, seed=batch + dim)
    rng = np.random.default_rng(context)
    lengths = rng.integers(1, context + 1, size=batch).astype(np.int32)
    lengths[0], lengths[-1] = context, 0
    counts = rng.integers(0, tokens + 1, size=batch).astype(np.int32)
    counts[0] = tokens
    run(layout, table, lengths, q, k, v, counts=counts, causal=context % 200 != 0)


@pytest.mark.parametrize("batch,heads,kv_heads,dim,tokens,context", [SHAPES[0], SHAPES[1], SHAPES[4], SHAPES[6]])
def test_hidden_nan_in_tiles_of_every_kind(batch, heads, kv_heads, dim, tokens, context):
    """The last token's V is NaN: rows that do not see it are those of the clean cache, bit for bit or to rounding."""
    announce(f"hidden NaN, {batch} x {tokens} on {context}")
    width = -(-context // 16)
    layout = Layout(batch, heads, kv_heads, dim, 16, batch * width)
    table, q, k, v = problem(layout, torch.bfloat16, torch.bfloat16, tokens, width, seed=5)
    lengths = np.full(batch, context, dtype=np.int32)
    plan = DecodePlan(layout, table, lengths, query_tokens=tokens)
    clean = plan.run_tokens(q, k, v).clone()
    check(layout, table, lengths, None, q, k, v, clean, True)
    at = (context - 1) // 16
    for b in range(batch):
        v[int(table[b, at]), (context - 1) % 16] = math.nan
    out = plan.run_tokens(q, k, v)
    assert not torch.isfinite(out[:, -1]).any()
    v.nan_to_num_(0.0)
    for b in (0, batch - 1):
        keys, values = (gathered(x, table[b], context, 16) for x in (k, v))
        sees = torch.arange(tokens, device="cuda") + context - tokens + 1
        expected, bound = oracle.attention(q[b], keys, values, sees)
        oracle.assert_within(out[b, :-1], expected[:-1], bound[:-1], q.dtype, f"sequence {b}")


def test_two_graphs_of_one_plan_and_shared_pages():
    """Graphs that share the plan's workspace, replayed in turn with eager calls between them; sequences that share their pages."""
    announce("two graphs of a plan")
    layout = Layout(3, 8, 2, 128, 16, 260)
    table, _, k, v = problem(layout, torch.float16, torch.float16, 4, 80, seed=3)
    table[1, :60] = table[0, :60]
    lengths = np.array([1280, 1100, 961], dtype=np.int32)
    plan = DecodePlan(layout, table, lengths, query_tokens=40)
    gen = torch.Generator(device="cuda").manual_seed(8)
    q = [torch.randn((3, n, 8, 128), device="cuda", generator=gen).half() for n in (4, 40)]
    outs = [torch.empty_like(x) for x in q]
    graphs = []
    for x, out in zip(q, outs):
        plan.run_tokens(x, k, v, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.run_tokens(x, k, v, out=out)
        graphs.append(graph)
    for step in range(6):
        for x in q:
            x.copy_(torch.randn(x.shape, device="cuda", generator=gen))
        for graph in graphs if step % 2 else graphs[::-1]:
            graph.replay()
        eager = [plan.run_tokens(x, k, v, out=torch.empty_like(x)) for x in q]
        torch.cuda.synchronize()
        for x, out, own in zip(q, outs, eager):
            assert torch.equal(out, own)
            check(layout, table, lengths, None, x, k, v, out, True)


def test_caches_past_32_bits():
    """Pages that begin more than 2^32 bytes into a cache: written with rotation, and read by either kernel."""
    announce("caches past 32 bits")
    pages = (1 << 32) // (16 * 8 * 128 * 2) + 200
    layout = Layout(1, 8, 8, 128, 16, pages)
    table = (pages - 1 - np.arange(100, dtype=np.int32))[None].copy()
    table[0, 1::2] = np.arange(50)
    k, v = (torch.zeros((pages, 16, 8, 128), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    gen = torch.Generator(device="cuda").manual_seed(4)
    f = torch.pow(torch.tensor(10000.0, dtype=torch.float64), -torch.arange(64, dtype=torch.float64) / 64)
    rotary = Rotary(f)
    plan = DecodePlan(layout, table, np.zeros(1, dtype=np.int32), max_context=1600, query_tokens=1500)
    q, k_new, v_new = (torch.randn((1, 1500, 8, 128), device="cuda", generator=gen).bfloat16() for _ in range(3))
    rotated = plan.append_rotated(k, v, k_new, v_new, rotary, q=q)
    lengths = np.array([1500], dtype=np.int32)
    q_exact, k_exact = rotate_heads(q, k_new, torch.zeros(1, dtype=torch.int32, device="cuda"), rotary)
    assert torch.equal(rotated, q_exact)
    assert torch.equal(gathered(k, table[0, :94], 1500, 16), k_exact[0].float())
    assert torch.equal(gathered(v, table[0, :94], 1500, 16), v_new[0].float())
    check(layout, table, lengths, None, rotated, k, v, plan.run_tokens(rotated, k, v), True)
    last = rotated[:, -3:].contiguous()
    check(layout, table, lengths, None, last, k, v, plan.run_tokens(last, k, v), True)


@pytest.mark.parametrize("tokens", [2, 40])
@pytest.mark.parametrize("part", [0.0, 0.3, 1.0, 3.0])
def test_c_entry_with_less_and_more_workspace(tokens, part):
    announce(f"C entry, {tokens} tokens, {part} of the workspace")
    layout = Layout(2, 4, 2, 64, 16, 300)
    table, q, k, v = problem(layout, torch.float16, torch.float16, tokens, 150, seed=6)
    lengths = np.array([2400, 1999], dtype=np.int32)
    lib = cabi.load()
    size = lib.pd_decode_tokens_workspace(cabi.PD_DTYPE_F16, cabi.PD_DTYPE_F16, 2, tokens, 4, 2, 64, 16, 150, 0)
    assert size > 0
    size = int(size * part) // 16 * 16
    room = torch.full((size + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    ids, lens = torch.from_numpy(table).cuda(), torch.from_numpy(lengths).cuda()
    for hints in (0, cabi.PD_HINT_UNSHARED_PAGES, cabi.PD_HINT_RAGGED_LENGTHS):
        out = torch.full_like(q, float("nan"))
        status = lib.pd_decode_tokens(q.data_ptr(), cabi.PD_DTYPE_F16, k.data_ptr(), v.data_ptr(), cabi.PD_DTYPE_F16, 1.0, 1.0,
                                      ids.data_ptr(), lens.data_ptr(), None, out.data_ptr(), room.data_ptr() if size else None, size,
                                      2, tokens, 4, 2, 64, 16, 150, 300, 1, hints, None,
                                      ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert status == cabi.PD_OK
        check(layout, table, lengths, None, q, k, v, out, True)
    assert bool((room[size:] == 0xA5).all())

