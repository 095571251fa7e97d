"""Head norms with rotation and rotated appends on the GPU against 64-bit results (tests/rotary_oracle.py)."""
import numpy as np
import pytest

from gpu_util import announce, require_gpu

require_gpu()

import torch  # noqa: E402

import rotary_oracle as oracle  # noqa: E402
from paged_decode.layout import Layout  # noqa: E402
from paged_decode.rotary import Rotary, append_rotated, rotate_heads  # noqa: E402
from paged_decode.runtime import DecodePlan  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
FP8 = [torch.float8_e4m3fn, torch.float8_e5m2]


def frequencies(dims, base=10000.0):
    return torch.pow(torch.tensor(base, dtype=torch.float64), -torch.arange(0, dims, 2, dtype=torch.float64) / dims)


def rows(batch, tokens, heads, dim, dtype, fused, seed):
    """New queries, keys and values: each contiguous, or views of one fused tensor."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if fused:
        wide = torch.randn((batch, tokens, sum(heads), dim), device="cuda", generator=gen).to(dtype)
        return torch.split(wide, heads, dim=2)
    return tuple(torch.randn((batch, tokens, h, dim), device="cuda", generator=gen).to(dtype) for h in heads)


def weight(shape, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (1 + 0.3 * torch.randn(shape, device="cuda", generator=gen)).to(dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim,dims", [(64, 64), (64, 16), (128, 128), (128, 48)])
@pytest.mark.parametrize("style", ["half", "interleaved"])
@pytest.mark.parametrize("normed", [False, True])
def test_rotation_of_queries_and_keys(dtype, dim, dims, style, normed):
    announce(f"rotate {dtype} D={dim} R={dims} {style} normed={normed}")
    batch, tokens = 3, 5
    q, k, _ = rows(batch, tokens, (7, 3, 3), dim, dtype, fused=normed, seed=dim + dims)
    start = torch.tensor([0, 1000003, 77], dtype=torch.int32, device="cuda")
    rotary = Rotary(frequencies(dims), style=style)
    weights = (weight((dim,), dtype, 1), weight((3, dim), dtype, 2)) if normed else (None, None)
    got = rotate_heads(q, k, start, rotary, q_weight=weights[0], k_weight=weights[1], eps=1e-5)
    at = start.long()[:, None] + torch.arange(tokens, device="cuda")
    for x, w, y in zip((q, k), weights, got):
        expected, bound = oracle.rotated(x, at, frequencies(dims).cuda(), style, w, eps=1e-5)
        oracle.assert_within(y, expected, bound, dtype, f"{dtype} {style}")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_norms_alone_and_weights_in_single_precision(dtype):
    announce(f"norms alone {dtype}")
    q, _, _ = rows(2, 33, (5, 1, 1), 128, dtype, False, 9)
    w = weight((5, 128), torch.float32, 3)
    got, none = rotate_heads(q, None, torch.zeros(2, dtype=torch.int32, device="cuda"), None, q_weight=w, eps=0.0)
    assert none is None
    expected, bound = oracle.rotated(q, None, None, weight=w, eps=0.0)
    oracle.assert_within(got, expected, bound, dtype)


def test_positions_per_token_scale_and_single_token_rows():
    announce("positions per token")
    q, k, _ = rows(4, 1, (8, 2, 2), 64, torch.bfloat16, True, 4)
    rotary = Rotary(frequencies(64, 500000.0), scale=1.25)
    at = torch.tensor([[5], [1 << 20], [0], [-3]], dtype=torch.int32, device="cuda")
    whole = rotate_heads(q, k, at, rotary)
    single = rotate_heads(q[:, 0], k[:, 0], at[:, 0].contiguous(), rotary)
    for x, y, z in zip((q, k), whole, single):
        expected, bound = oracle.rotated(x, at, frequencies(64, 500000.0).cuda(), scale=1.25)
        oracle.assert_within(y, expected, bound, torch.bfloat16)
        assert torch.equal(y[:, 0], z)


@pytest.mark.parametrize("tokens", [1, 300, 5000])
def test_rows_from_few_to_many(tokens):
    """Odd head counts, so that a wave holds heads of q and k at once, at sizes that split tokens over waves and do not."""
    announce(f"rotate tokens={tokens}")
    q, k, _ = rows(1, tokens, (28, 4, 4), 128, torch.float16, True, tokens)
    rotary = Rotary(frequencies(128))
    got = rotate_heads(q, k, torch.tensor([11], dtype=torch.int32, device="cuda"), rotary)
    at = 11 + torch.arange(tokens, device="cuda")[None]
    for x, y in zip((q, k), got):
        expected, bound = oracle.rotated(x, at, frequencies(128).cuda())
        oracle.assert_within(y, expected, bound, torch.float16)


def test_rotation_in_place_and_of_nonfinite_values():
    announce("rotate in place, nonfinite")
    q, k, _ = rows(2, 3, (4, 4, 4), 64, torch.float32, False, 5)
    q[0, 1, 2, 5] = float("inf")
    k[1, 2, 0, 40] = float("nan")
    before = rotate_heads(q, k, torch.tensor([9, 10], dtype=torch.int32, device="cuda"), Rotary(frequencies(64)))
    after = rotate_heads(q, k, torch.tensor([9, 10], dtype=torch.int32, device="cuda"), Rotary(frequencies(64)), out=(q, k))
    assert after[0].data_ptr() == q.data_ptr() and after[1].data_ptr() == k.data_ptr()
    for x, y in zip(before, after):
        assert torch.equal(x.view(torch.int32), y.view(torch.int32))
    touched = ~torch.isfinite(before[0])  # the pair's two dims and nothing else
    assert touched.nonzero().tolist() == [[0, 1, 2, 5], [0, 1, 2, 37]]
    assert (~torch.isfinite(before[1])).nonzero().tolist() == [[1, 2, 0, 8], [1, 2, 0, 40]]


def expected_append(layout, cache, table, positions, counts, new, dtype, scale):
    """(cache values, bounds) in 64 bits: new is [(value, bound)] of [B, n, Hkv, D]; untouched cells keep theirs, bound 0."""
    cells, bounds = cache.double(), torch.zeros(cache.shape, dtype=torch.float64, device="cuda")
    value, bound = oracle.stored(*new, dtype, scale)
    width = table.shape[1]
    for b in range(layout.batch):
        for j in range(int(counts[b])):
            pos = int(positions[b]) + j
            if not 0 <= pos < width * layout.page_size:
                continue
            page = int(table[b, pos // layout.page_size])
            if 0 <= page < layout.physical_pages:
                cells[page, pos % layout.page_size] = value[b, j]
                bounds[page, pos % layout.page_size] = bound[b, j]
    return cells, bounds


def assert_cells(actual, cells, bounds):
    wrong = ~((actual.double() - cells).abs() <= bounds)
    assert not wrong.any(), f"{int(wrong.sum())} cells, first {wrong.nonzero()[0].tolist()}"


@pytest.mark.parametrize("dtype,cache_dtype", [(t, t) for t in TYPES] + [(t, f) for t in TYPES[1:] for f in FP8], ids=str)
@pytest.mark.parametrize("dim,page,tokens,fused,style", [(64, 16, 1, True, "half"), (128, 32, 19, False, "interleaved"),
                                                        (128, 16, 40, True, "half")])
def test_append_at_positions(dtype, cache_dtype, dim, page, tokens, fused, style):
    announce(f"append {dtype} -> {cache_dtype} D={dim} page={page} n={tokens}")
    layout = Layout(5, 6, 2, dim, page, 24)
    rng = np.random.default_rng(dim + tokens)
    table = rng.permutation(24)[:20].reshape(5, 4).astype(np.int32)
    table[1, 2], table[3, 0] = -1, 1 << 20             # not written
    positions = np.array([0, 2 * page - 1, 4 * page - 2, page - 1, -1], dtype=np.int32)
    counts = np.array([tokens, tokens, tokens, tokens + 7, 0 if tokens == 1 else tokens - 1], dtype=np.int32)
    live = np.minimum(counts, tokens)
    q, k_new, v_new = rows(5, tokens, (6, 2, 2), dim, dtype, fused, 8)
    scale = 1.0 if cache_dtype.itemsize > 1 else 0.02
    k_cache, v_cache = (torch.randn((24, page, 2, dim), device="cuda").to(dtype).to(cache_dtype) for _ in range(2))
    f = frequencies(dim)
    weights = weight((dim,), dtype, 5), weight((dim,), dtype, 6)
    at = torch.from_numpy(positions).cuda().long()[:, None] + torch.arange(tokens, device="cuda")
    k_exact = oracle.rotated(k_new, at, f.cuda(), style, weights[1])
    v_exact = v_new.double(), torch.zeros(v_new.shape, dtype=torch.float64, device="cuda")
    expected = [expected_append(layout, c, table, positions, live, e, cache_dtype, scale)
                for c, e in ((k_cache, k_exact), (v_cache, v_exact))]
    got = append_rotated(layout, k_cache, v_cache, torch.from_numpy(table).cuda(), torch.from_numpy(positions).cuda(), k_new,
                         v_new, Rotary(f, style=style), q=q, q_weight=weights[0], k_weight=weights[1], k_scale=scale,
                         v_scale=scale, counts=torch.from_numpy(counts).cuda())
    for cache, (cells, bounds) in zip((k_cache, v_cache), expected):
        assert_cells(cache, cells, bounds)
    q_exact, q_bound = oracle.rotated(q, at, f.cuda(), style, weights[0])
    dead = torch.arange(tokens, device="cuda") >= torch.from_numpy(live).cuda()[:, None]
    q_exact[dead], q_bound[dead] = 0, 0
    oracle.assert_within(got, q_exact, q_bound, dtype)
    assert not got[dead].any()


@pytest.mark.parametrize("cache_dtype", FP8, ids=str)
def test_quantised_append_rounds_as_a_cast_does(cache_dtype):
    """Every 16-bit value through the value path (no norm, no rotation): torch's own cast of x / scale, saturated."""
    announce(f"quantise {cache_dtype}")
    layout = Layout(1, 16, 16, 128, 32, 1)
    bits = torch.arange(1 << 16, dtype=torch.int32, device="cuda").to(torch.int16)
    v_new = bits.view(torch.float16).view(1, 32, 16, 128)
    k_cache, v_cache = (torch.zeros((1, 32, 16, 128), device="cuda").to(cache_dtype) for _ in range(2))
    append_rotated(layout, k_cache, v_cache, torch.zeros((1, 1), dtype=torch.int32, device="cuda"),
                   torch.zeros(1, dtype=torch.int32, device="cuda"), v_new, v_new, Rotary(frequencies(128)), v_scale=0.75)
    largest = torch.finfo(cache_dtype).max
    expected = (v_new.float() / 0.75).clamp(-largest, largest).to(cache_dtype)
    nan = torch.isnan(v_new)
    assert torch.equal(torch.isnan(v_cache.float()), nan.view(v_cache.shape))
    assert torch.equal(v_cache.view(torch.uint8)[~nan], expected.view(torch.uint8)[~nan])


def fits(table, length, count, page, pages, capacity):
    entries = table[length // page:-(-(length + count) // page)] if count else []
    return length + count <= min(capacity, len(table) * page) and all(0 <= e < pages for e in entries)


@pytest.mark.parametrize("tokens", [1, 3, 70])
def test_plan_append_is_all_or_nothing_and_advances(tokens):
    """One workgroup per sequence (few tokens) and a launch of its own for the lengths (many)."""
    announce(f"plan append n={tokens}")
    layout = Layout(6, 8, 2, 128, 16, 64)
    table = np.arange(60, dtype=np.int32).reshape(6, 10)
    table[2, 3:] = -1                                        # cannot grow past 48
    lengths = np.array([5, 100, 47, 160 - tokens, 0, 160], dtype=np.int32)
    counts = np.array([tokens, max(tokens - 2, 0), tokens, tokens, 0, 1], dtype=np.int32)
    lengths[2] = min(lengths[2], 48)
    plan = DecodePlan(layout, table, lengths, max_context=160)
    q, k_new, v_new = rows(6, tokens, (8, 2, 2), 128, torch.bfloat16, True, 3)
    k, v = (torch.randn((64, 16, 2, 128), device="cuda").bfloat16() for _ in range(2))
    f = frequencies(128)
    at = torch.from_numpy(lengths).cuda().long()[:, None] + torch.arange(tokens, device="cuda")
    taken = np.array([c if fits(table[b], int(lengths[b]), int(c), 16, 64, 160) else 0 for b, c in enumerate(counts)])
    expected = [expected_append(layout, c, table, lengths, taken, e, torch.bfloat16, 1.0) for c, e in
                ((k, oracle.rotated(k_new, at, f.cuda())), (v, (v_new.double(), torch.zeros_like(v_new, dtype=torch.float64))))]
    got = plan.append_rotated(k, v, k_new, v_new, Rotary(f), q=q, counts=torch.from_numpy(counts).cuda())
    for cache, (cells, bounds) in zip((k, v), expected):
        assert_cells(cache, cells, bounds)
    np.testing.assert_array_equal(plan._lengths.cpu().numpy(), lengths + taken)
    assert taken[5] == 0 and taken[0] == tokens
    q_exact, q_bound = oracle.rotated(q, at, f.cuda())
    dead = torch.arange(tokens, device="cuda") >= torch.from_numpy(counts).cuda()[:, None]
    q_exact[dead], q_bound[dead] = 0, 0
    oracle.assert_within(got, q_exact, q_bound, torch.bfloat16)


def test_refusals():
    announce("rotary refusals")
    q, k, v = rows(2, 4, (4, 2, 2), 64, torch.float16, False, 1)
    start = torch.zeros(2, dtype=torch.int32, device="cuda")
    rotary = Rotary(frequencies(64))
    layout = Layout(2, 4, 2, 64, 16, 4)
    kc, vc = (torch.zeros((4, 16, 2, 64), device="cuda", dtype=torch.float16) for _ in range(2))
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
    with pytest.raises(ValueError):
        rotate_heads(q, k, start, None)                                   # nothing to do
    with pytest.raises(TypeError):
        rotate_heads(q, k.bfloat16(), start, rotary)
    with pytest.raises(TypeError):
        rotate_heads(q, k, start.long(), rotary)
    with pytest.raises(ValueError):
        rotate_heads(q.transpose(1, 2), k, start, rotary)                 # heads not contiguous
    with pytest.raises(ValueError):
        rotate_heads(q.clone().requires_grad_(), k, start, rotary)
    with pytest.raises(ValueError):
        rotate_heads(q, k, start, Rotary(frequencies(128)))               # more dims than the head
    with pytest.raises(ValueError):
        rotate_heads(q, k, start, rotary, q_weight=torch.ones(32, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError):
        rotate_heads(q, k, start, rotary, out=(q.view(-1)[:k.numel()].view(k.shape).new_empty(q.shape), q.view(-1)[:k.numel()].view(k.shape)))
    with pytest.raises(TypeError):
        append_rotated(layout, kc.float(), vc.float(), table, start, k, v, rotary)
    with pytest.raises(ValueError):
        append_rotated(layout, kc, vc, table, start, k, v, rotary, k_scale=0.5)
    with pytest.raises(ValueError):
        append_rotated(layout, kc, vc, table, start, k, v[:, :3], rotary)
    with pytest.raises(ValueError):
        append_rotated(layout, kc, kc, table, start, k, v, rotary)
    with pytest.raises(TypeError):
        append_rotated(layout, kc, vc, table, start, k, v, rotary, counts=torch.ones(2, device="cuda"))
    plan = DecodePlan(layout, table.cpu().numpy(), np.array([3, 3]))
    with pytest.raises(ValueError):
        plan.append_rotated(kc, vc, k, v, rotary)                         # beyond the reserved context
    assert not kc.any() and not vc.any()
