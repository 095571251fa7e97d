"""Host-side checks of the rotation, the rotated append and the attention of several tokens, without a GPU: the C entries'
refusals come before any launch."""
import ctypes

import numpy as np
import pytest

from paged_decode import cabi
from paged_decode.layout import Layout
from paged_decode.runtime import DecodePlan

FAKE = 1 << 20  # an aligned address that is never dereferenced


@pytest.mark.parametrize("tokens", [0, -1, True, 1.0, 65536])
def test_plan_rejects_bad_query_tokens(tokens):
    with pytest.raises(ValueError):
        DecodePlan(Layout(1, 8, 2, 64, 16, 8), np.arange(8, dtype=np.int32)[None], np.array([127]), query_tokens=tokens)


def rotation(**over):
    values = dict(frequencies=FAKE, rotary_dim=64, style=0, scale=1.0, q_weight=FAKE, k_weight=FAKE,
                  weight_dtype=cabi.PD_DTYPE_F16, q_weight_per_head=0, k_weight_per_head=0, eps=1e-6)
    return cabi.Rotation(**{**values, **over})


def rotate(lib, rot=None, q=None, k=None, **over):
    a = dict(dtype=cabi.PD_DTYPE_F16, positions=FAKE, per=0, q_out=FAKE, k_out=FAKE, batch=2, tokens=3, hq=4, hkv=2, d=64)
    a.update(over)
    rot = rotation() if rot is None else rot
    q = cabi.TokenRows(FAKE, 768, 256) if q is None else q
    k = cabi.TokenRows(FAKE, 384, 128) if k is None else k
    return lib.pd_rotate_heads(ctypes.byref(rot), ctypes.byref(q), ctypes.byref(k), a["dtype"], a["positions"], a["per"],
                               a["q_out"], a["k_out"], a["batch"], a["tokens"], a["hq"], a["hkv"], a["d"], None)


@pytest.mark.parametrize("over,status", [
    (dict(dtype=cabi.PD_DTYPE_FP8_E4M3), cabi.PD_ERR_DTYPE), (dict(d=96), cabi.PD_ERR_SHAPE), (dict(batch=0), cabi.PD_ERR_SHAPE),
    (dict(tokens=0), cabi.PD_ERR_SHAPE), (dict(tokens=65536), cabi.PD_ERR_SHAPE), (dict(hq=0), cabi.PD_ERR_SHAPE),
    (dict(positions=None), cabi.PD_ERR_NULL_POINTER), (dict(q_out=None), cabi.PD_ERR_NULL_POINTER),
    (dict(k_out=None), cabi.PD_ERR_NULL_POINTER), (dict(q_out=FAKE + 8), cabi.PD_ERR_SHAPE),
    (dict(rot=rotation(rotary_dim=24)), cabi.PD_ERR_SHAPE), (dict(rot=rotation(rotary_dim=80)), cabi.PD_ERR_SHAPE),
    (dict(rot=rotation(rotary_dim=-16)), cabi.PD_ERR_SHAPE), (dict(rot=rotation(style=2)), cabi.PD_ERR_SHAPE),
    (dict(rot=rotation(frequencies=None)), cabi.PD_ERR_NULL_POINTER), (dict(rot=rotation(scale=float("nan"))), cabi.PD_ERR_SHAPE),
    (dict(rot=rotation(weight_dtype=cabi.PD_DTYPE_BF16)), cabi.PD_ERR_DTYPE),
    (dict(rot=rotation(eps=-1.0)), cabi.PD_ERR_SHAPE), (dict(rot=rotation(q_weight=FAKE + 2)), cabi.PD_ERR_SHAPE),
    (dict(q=cabi.TokenRows(None, 768, 256)), cabi.PD_ERR_NULL_POINTER), (dict(q=cabi.TokenRows(FAKE, 768, 260)), cabi.PD_ERR_SHAPE),
    (dict(batch=65535, tokens=2048), cabi.PD_ERR_SHAPE),  # more threads than a launch holds
    (dict(q=cabi.TokenRows(FAKE + 4, 768, 256)), cabi.PD_ERR_SHAPE), (dict(k=cabi.TokenRows(FAKE, -384, 128)), cabi.PD_ERR_SHAPE),
])
def test_rotation_refusals(over, status):
    assert rotate(cabi.load(), **over) == status


def append(lib, advance, rot=None, q=True, **over):
    a = dict(dtype=cabi.PD_DTYPE_F16, table=FAKE, at=FAKE, counts=None, q_out=FAKE, k=FAKE, v=FAKE, cache=cabi.PD_DTYPE_F16,
             ks=1.0, vs=1.0, batch=2, tokens=3, hq=4, hkv=2, d=64, page=16, width=4, pages=8, most=64)
    a.update(over)
    rot = rotation() if rot is None else rot
    rows = cabi.TokenRows(FAKE, 768, 256)
    args = [ctypes.byref(rot), ctypes.byref(rows) if q else None, ctypes.byref(rows), ctypes.byref(rows), a["dtype"], a["table"],
            a["at"], a["counts"], a["q_out"], a["k"], a["v"], a["cache"], a["ks"], a["vs"], a["batch"], a["tokens"], a["hq"],
            a["hkv"], a["d"], a["page"], a["width"], a["pages"]]
    if advance:
        return lib.pd_append_rotated_advance(*args, a["most"], None)
    return lib.pd_append_rotated(*args, None)


@pytest.mark.parametrize("advance", [False, True])
@pytest.mark.parametrize("over,status", [
    (dict(table=None), cabi.PD_ERR_NULL_POINTER), (dict(at=None), cabi.PD_ERR_NULL_POINTER),
    (dict(k=None), cabi.PD_ERR_NULL_POINTER), (dict(q_out=None), cabi.PD_ERR_NULL_POINTER),
    (dict(cache=cabi.PD_DTYPE_BF16), cabi.PD_ERR_DTYPE), (dict(dtype=cabi.PD_DTYPE_F32, cache=cabi.PD_DTYPE_FP8_E4M3), cabi.PD_ERR_DTYPE),
    (dict(ks=0.0), cabi.PD_ERR_DTYPE), (dict(vs=float("inf")), cabi.PD_ERR_DTYPE), (dict(ks=0.5), cabi.PD_ERR_DTYPE),
    (dict(page=8), cabi.PD_ERR_SHAPE), (dict(width=0), cabi.PD_ERR_SHAPE), (dict(pages=0), cabi.PD_ERR_SHAPE),
    (dict(tokens=0), cabi.PD_ERR_SHAPE), (dict(hkv=0), cabi.PD_ERR_SHAPE), (dict(d=80), cabi.PD_ERR_SHAPE),
    (dict(v=FAKE + 8), cabi.PD_ERR_SHAPE), (dict(rot=rotation(rotary_dim=128)), cabi.PD_ERR_SHAPE),
])
def test_append_refusals(advance, over, status):
    assert append(cabi.load(), advance, **over) == status


@pytest.mark.parametrize("most", [-1, (1 << 20) + 1])
def test_append_refuses_contexts_beyond_the_limit(most):
    assert append(cabi.load(), True, most=most) == cabi.PD_ERR_SHAPE


def tokens_call(lib, **over):
    a = dict(q=FAKE, qt=cabi.PD_DTYPE_F16, k=FAKE, v=FAKE, kt=cabi.PD_DTYPE_F16, ks=1.0, vs=1.0, table=FAKE, lengths=FAKE, counts=None,
             out=FAKE, ws=None, size=0, batch=2, tokens=3, hq=4, hkv=2, d=64, page=16, width=4, pages=8, causal=1, hints=0)
    a.update(over)
    return lib.pd_decode_tokens(*a.values(), None, None)


@pytest.mark.parametrize("over,status", [
    (dict(q=None), cabi.PD_ERR_NULL_POINTER), (dict(table=None), cabi.PD_ERR_NULL_POINTER), (dict(out=None), cabi.PD_ERR_NULL_POINTER),
    (dict(lengths=None), cabi.PD_ERR_NULL_POINTER), (dict(size=16), cabi.PD_ERR_NULL_POINTER), (dict(qt=cabi.PD_DTYPE_FP8_E4M3), cabi.PD_ERR_DTYPE),
    (dict(kt=cabi.PD_DTYPE_BF16), cabi.PD_ERR_DTYPE), (dict(qt=cabi.PD_DTYPE_F32, kt=cabi.PD_DTYPE_FP8_E5M2), cabi.PD_ERR_DTYPE),
    (dict(ks=-1.0), cabi.PD_ERR_DTYPE), (dict(vs=float("nan")), cabi.PD_ERR_DTYPE), (dict(batch=0), cabi.PD_ERR_SHAPE),
    (dict(tokens=0), cabi.PD_ERR_SHAPE), (dict(tokens=65536), cabi.PD_ERR_SHAPE), (dict(hq=5), cabi.PD_ERR_SHAPE), (dict(hkv=0), cabi.PD_ERR_SHAPE),
    (dict(d=32), cabi.PD_ERR_SHAPE), (dict(page=64), cabi.PD_ERR_SHAPE), (dict(width=65537), cabi.PD_ERR_SHAPE), (dict(pages=0), cabi.PD_ERR_SHAPE),
    (dict(q=FAKE + 2), cabi.PD_ERR_SHAPE), (dict(tokens=65535, hq=65535, hkv=1), cabi.PD_ERR_SHAPE),
    (dict(hints=4), cabi.PD_ERR_HINT),
    (dict(batch=65535, tokens=1, hq=2048, hkv=2048), cabi.PD_ERR_SHAPE), (dict(batch=65535, tokens=65535, hq=64, hkv=64), cabi.PD_ERR_SHAPE),
])
def test_token_attention_refusals(over, status):
    assert tokens_call(cabi.load(), **over) == status


def test_token_workspace_grows_with_the_tokens_and_is_bounded():
    lib = cabi.load()
    size = [lib.pd_decode_tokens_workspace(cabi.PD_DTYPE_F16, cabi.PD_DTYPE_F16, 4, n, 32, 8, 128, 16, 1024, 256) for n in (1, 4, 16, 512)]
    assert 0 < size[0] <= size[1] <= size[2] <= size[3] < 256 << 20
    assert lib.pd_decode_tokens_workspace(cabi.PD_DTYPE_F16, cabi.PD_DTYPE_F16, 4, 1, 32, 8, 128, 16, 4, 256) == 0  # too short to split
    assert lib.pd_decode_tokens_workspace(cabi.PD_DTYPE_F16, cabi.PD_DTYPE_F16, 4, 1, 32, 5, 128, 16, 4, 256) == 0
