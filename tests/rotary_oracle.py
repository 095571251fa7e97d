"""64-bit head norms, rotation and attention of several tokens, with bounds on what FP32 kernels may be off.

Everything is on torch float64 tensors (any device). ``u`` is the unit roundoff of FP32, 2^-24; a type's own is
``torch.finfo(t).eps / 2``.
"""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def half_subnormal(dtype):
    """Half the distance of the type's subnormal numbers: the rounding error next to zero."""
    info = torch.finfo(dtype)
    return info.tiny * info.eps / 2


def rotated(x, positions, frequencies, style="half", weight=None, eps=1e-6, scale=1.0):
    """(y, bound on the FP32 error before rounding) for heads x [B, n, H, D] at positions [B, n].

    The norm's sum of D squares, in any order, is off by at most D u relative, hence its root by D u / 2 (D <= 128: 64 u);
    the root, the quotient, and the products with the head and the weight add 4 u. A cosine or sine is off by at most 4 u
    absolute (FP32 argument of at most an eighth of a turn: 0.4 u; the function: under 2 u), its product and sum with the
    other one of the pair by 3 u: in all (64 + 4 + 4 + 3) u of |a| + |b|, and half of that where there is no norm.
    """
    x = x.double()
    terms = 7
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
        terms += 4 + x.shape[-1] / 2
    size = x.abs()
    if frequencies is not None:
        half = len(frequencies)
        angle = positions.double()[..., None, None] * frequencies.double()
        cos, sin = torch.cos(angle) * scale, torch.sin(angle) * scale
        if style == "half":
            first, second = slice(0, half), slice(half, 2 * half)
        else:
            first, second = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
        a, b = x[..., first], x[..., second]
        y = x.clone()
        y[..., first], y[..., second] = a * cos - b * sin, a * sin + b * cos
        size = size.clone()
        size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(scale)
        x = y
    return x, terms * U * size


def stored(y, bound, dtype, scale=1.0):
    """(value, bound) of y / scale rounded to ``dtype``, saturated where it is FP8."""
    y, bound = y / scale, bound / scale + 2 * U * (y / scale).abs()
    if dtype.itemsize == 1:
        y = y.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max)
    return y, bound * (1 + half_step(dtype)) + half_step(dtype) * y.abs() + half_subnormal(dtype)


def attention(q, k, v, sees, k_scale=1.0, v_scale=1.0, hidden=None):
    """(out, bound before rounding, for weights rounded to q's type) of one sequence.

    q [n, Hq, D], k, v [T, Hkv, D], sees [n] (how many leading tokens each row sees); hidden: tokens that no row sees.
    A score is a sum of D exact products in FP32: off by D u of sum |q k| (scaled), and its argument of 2^x, at most twice
    that size, by 4 u more of it; each weight then by that and 3 u relative, and by half a step of q's type where it is 16 bits.
    The sums over T tokens in any order add T u each, the quotient and scaling 4 u. A weight below the type's normal range
    is off by half a subnormal step, with the largest weight at least 1 (FP16: 2^6).
    """
    n, query_heads, dim = q.shape
    tokens, kv_heads = k.shape[:2]
    group = query_heads // kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    if tokens == 0:
        return out, bound
    own = half_step(q.dtype) if q.dtype != torch.float32 else 0.0
    below = half_subnormal(q.dtype) / (64 if q.dtype == torch.float16 else 1)
    blind = torch.arange(tokens, device=q.device)[None, :] >= sees[:, None]
    if hidden is not None:
        blind = blind | hidden[None, :]
    for h in range(query_heads):
        keys, values = k[:, h // group].double() * k_scale, v[:, h // group].double() * v_scale
        scores = q[:, h].double() @ keys.T / math.sqrt(dim)
        size = (q[:, h].double().abs() @ keys.abs().T / math.sqrt(dim)).masked_fill(blind, 0).amax(1, keepdim=True)
        weights = torch.softmax(scores.masked_fill(blind, -math.inf), 1)
        weights = torch.where(blind, 0.0, weights)
        values = torch.where(blind.all(0)[:, None], 0.0, values)
        out[:, h] = weights @ values
        spread = weights @ values.abs()
        each = 2 * ((dim + 8) * size + 3) * U + own + 2 * tokens * U + 4 * U
        bound[:, h] = spread * each + tokens * below * values.abs().amax() * (size < math.inf)
    return out, bound


def assert_within(actual, expected, bound, dtype, what=""):
    """|actual - expected| <= bound plus the rounding to dtype, elementwise; infinities and NaN where expected."""
    actual = actual.double()
    limit = bound * (1 + half_step(dtype)) + half_step(dtype) * expected.abs() + half_subnormal(dtype)
    wrong = ~((actual - expected).abs() <= limit)
    same = (actual == expected) | (torch.isnan(actual) & torch.isnan(expected))
    wrong &= ~same
    if wrong.any():
        at = tuple(int(i) for i in wrong.nonzero()[0])
        raise AssertionError(f"{what}: {int(wrong.sum())} of {wrong.numel()} off, first at {at}: {float(actual[at])} "
                             f"for {float(expected[at])}, limit {float(limit[at]):.3g}")
