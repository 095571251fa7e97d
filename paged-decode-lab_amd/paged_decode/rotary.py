"""Norms of queries and keys for each head with the position rotation, alone or on the way into the paged cache.

``rotate_heads`` norms and rotates new queries and keys; ``append_rotated``
does so while it writes the keys, and the values beside them, into the cache
(``DecodePlan.append_rotated`` at the plan's own lengths). The reference has
neither: its q and cache rows arrive as attention reads them
(docs/DESIGN.md:10-13).
"""
import math

import torch

from .layout import Layout
from .runtime import _FP8, check_scales, load_extension

_STYLES = {"half": 0, "interleaved": 1}
_TOKEN_TYPES = (torch.float32, torch.float16, torch.bfloat16)


class Rotary:
    """A position rotation: the frequencies of its pairs, kept on the device in 64 bits.

    ``frequencies`` (radians per position, one per pair) turn the first
    ``2 * len(frequencies)`` dims of a head; a multiple of 8 of them, at most
    ``head_dim / 2``. ``style`` says which dims form pair ``i``: ``"half"``
    those ``i`` and ``i + len(frequencies)``, ``"interleaved"`` those ``2 i``
    and ``2 i + 1``. ``scale`` multiplies cosine and sine (long-context
    schemes that also scale attention; 1.0 otherwise). Angles are products in
    64 bits, so far positions lose nothing.
    """

    def __init__(self, frequencies, *, style="half", scale=1.0, device=None):
        if style not in _STYLES:
            raise ValueError("style must be 'half' or 'interleaved'")
        if isinstance(scale, bool) or not isinstance(scale, (int, float)) or not math.isfinite(scale):
            raise ValueError("scale must be a finite number")
        frequencies = torch.as_tensor(frequencies).detach()
        if frequencies.dim() != 1 or frequencies.numel() not in range(8, 65, 8):
            raise ValueError("frequencies must be one-dimensional, 8 to 64 of them, a multiple of 8")
        if not torch.isfinite(frequencies).all():
            raise ValueError("frequencies must be finite")
        if device is None:
            device = frequencies.device if frequencies.is_cuda else "cuda"
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("Rotary requires a GPU (torch 'cuda') device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.style, self.scale = style, float(scale)
        self.dims = 2 * frequencies.numel()
        self._frequencies = frequencies.to(device=self.device, dtype=torch.float64, copy=True)
        self._style = _STYLES[style]


def rotate_heads(q, k, positions, rotary, *, q_weight=None, k_weight=None, eps=1e-6, out=None):
    """Norm and rotate the heads of new queries and keys in one launch; returns ``(q_out, k_out)``.

    ``q`` is ``[B, n, Hq, D]`` or ``[B, Hq, D]`` (one token), ``k`` likewise
    with its own heads, or None (``k_out`` is then None); float32, float16 or
    bfloat16. Heads are contiguous; tokens and sequences may lie apart by
    multiples of 16 bytes (views of a fused projection). ``positions`` is int32
    ``[B]`` (token ``j`` at ``positions[b] + j``) or ``[B, n]``. Weights are
    ``[D]`` or ``[H, D]``, of the inputs' type or float32; with one, the head
    is scaled by ``weight / sqrt(mean of squares + eps)`` first. ``rotary``
    None only norms. Everything is computed in 32 bits and rounded once.
    ``out`` gives the contiguous outputs ``(q_out, k_out)``; one may be its own
    contiguous input. Runs on the current stream.
    """
    rows_q, dim = _rows(q, "q")
    rows_k = None
    if k is not None:
        rows_k, k_dim = _rows(k, "k")
        if k_dim != dim or rows_k.shape[:2] != rows_q.shape[:2] or k.dim() != q.dim():
            raise ValueError("q and k must hold the same tokens and head_dim")
    _check_tokens(q, k)
    _check_rotation(rotary, dim, q, ((q_weight, rows_q), (k_weight, rows_k)), eps)
    batch, tokens = rows_q.shape[:2]
    if positions.device != q.device or positions.dtype != torch.int32 or not positions.is_contiguous():
        raise TypeError("positions must be a contiguous int32 tensor on the inputs' device")
    if tuple(positions.shape) not in ((batch,), (batch, tokens)):
        raise ValueError("positions must be [B] or [B, n]")
    per_token = positions.dim() == 2
    if out is None:
        q_out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
        k_out = None if k is None else torch.empty(k.shape, device=q.device, dtype=q.dtype)
    else:
        q_out, k_out = out
        for given, like in ((q_out, q), (k_out, k)):
            if (given is None) != (like is None):
                raise ValueError("out must give an output for each input")
            if given is not None:
                _check_out(given, like)
    load_extension().rotate_heads(rows_q, rows_k, positions, per_token, *_rotation(rotary, q_weight, k_weight, eps),
                                  q_out, k_out)
    return q_out, k_out


def append_rotated(layout: Layout, k_cache, v_cache, table, positions, k_new, v_new, rotary, *, q=None, q_weight=None,
                   k_weight=None, eps=1e-6, k_scale=1.0, v_scale=1.0, counts=None, out=None):
    """``append_kv`` with the new keys normed and rotated on the way, at their cache positions; returns the rotated ``q``.

    ``k_new``/``v_new`` are ``[B, n, Hkv, D]`` or ``[B, Hkv, D]`` and ``q``
    (optional) ``[B, n, Hq, D]`` or ``[B, Hq, D]``, strided and normed as in
    ``rotate_heads``. Token ``j`` of sequence ``b`` is rotated at, and written
    to, ``positions[b] + j``; ``counts`` (int32 ``[B]`` on the device) says how
    many of the ``n`` tokens a sequence brings: those behind write nothing and
    their rows of the returned q are zeros. Tokens outside the table's
    capacity or on page ids outside ``[0, physical_pages)`` are not written.
    The cache has the tokens' type, or FP8 under 16-bit tokens: it then holds
    ``k / k_scale`` and ``v / v_scale``, to nearest even, saturated at the
    largest finite value. ``out`` gives q's contiguous output (q itself, if
    contiguous). Runs on the current stream.
    """
    for t in (table, positions):
        if t.device != k_cache.device or t.dtype != torch.int32 or not t.is_contiguous():
            raise TypeError("table and positions must be contiguous int32 tensors on the cache device")
    if table.dim() != 2 or table.shape[0] != layout.batch or tuple(positions.shape) != (layout.batch,):
        raise ValueError("table must be [B, W] and positions [B]")
    return launch_append(layout, k_cache, v_cache, table, positions, k_new, v_new, rotary, q, q_weight, k_weight, eps,
                         k_scale, v_scale, counts, out, -1)


def launch_append(layout, k_cache, v_cache, table, positions, k_new, v_new, rotary, q, q_weight, k_weight, eps, k_scale,
                  v_scale, counts, out, max_context):
    """Checks and launch shared by ``append_rotated`` and ``DecodePlan.append_rotated`` (``max_context`` >= 0:
    ``positions`` are lengths, advanced by the call)."""
    rows_k, dim = _rows(k_new, "k_new")
    rows_v, _ = _rows(v_new, "v_new")
    expected = (layout.kv_heads, layout.head_dim)
    if k_new.shape != v_new.shape or rows_k.shape[0] != layout.batch or tuple(rows_k.shape[2:]) != expected:
        raise ValueError("new tokens must be [B, Hkv, D] or [B, tokens, Hkv, D] matching the layout")
    rows_q = None
    if q is not None:
        rows_q, _ = _rows(q, "q")
        if q.dim() != k_new.dim() or rows_q.shape[:2] != rows_k.shape[:2] or \
                tuple(rows_q.shape[2:]) != (layout.query_heads, layout.head_dim):
            raise ValueError("q must hold the new tokens' queries, [B, tokens, Hq, D] matching the layout")
    elif q_weight is not None or out is not None:
        raise ValueError("q_weight and out need q")
    cache_shape = (layout.physical_pages, layout.page_size, layout.kv_heads, layout.head_dim)
    if tuple(k_cache.shape) != cache_shape or tuple(v_cache.shape) != cache_shape:
        raise ValueError("cache shape does not match the layout")
    _check_tokens(k_new, v_new, q)
    fp8 = k_cache.dtype in _FP8
    if v_cache.dtype != k_cache.dtype or not (k_cache.dtype == k_new.dtype or (fp8 and k_new.dtype != torch.float32)):
        raise TypeError("the cache must have the new tokens' dtype, or float8_e4m3fn/float8_e5m2 under 16-bit tokens")
    for tensor in (k_cache, v_cache):
        if tensor.device != k_new.device or not tensor.is_contiguous():
            raise ValueError("cache tensors must be contiguous on the new tokens' device")
    check_scales(k_scale, v_scale)
    if not fp8 and (k_scale != 1.0 or v_scale != 1.0):
        raise ValueError("k_scale and v_scale apply to FP8 caches")
    _check_rotation(rotary, dim, k_new, ((q_weight, rows_q), (k_weight, rows_k)), eps)
    check_counts(counts, layout.batch, k_new.device)
    if q is not None:
        if out is None:
            out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
        else:
            _check_out(out, q)
    load_extension().append_rotated(rows_q, rows_k, rows_v, table, positions, counts,
                                    *_rotation(rotary, q_weight, k_weight, eps), out, k_cache, v_cache, float(k_scale),
                                    float(v_scale), max_context)
    return out


def check_counts(counts, batch, device):
    if counts is None:
        return
    if counts.device != device or counts.dtype != torch.int32 or not counts.is_contiguous():
        raise TypeError("counts must be a contiguous int32 tensor on the inputs' device")
    if tuple(counts.shape) != (batch,):
        raise ValueError("counts must be [B]")


def _rows(x, name):
    """(x as [B, n, H, D], D) with the strides the kernels take."""
    rows = x.unsqueeze(1) if x.dim() == 3 else x
    if rows.dim() != 4 or 0 in rows.shape:
        raise ValueError(f"{name} must be [B, H, D] or [B, tokens, H, D], none of them 0")
    if max(rows.shape[:3]) > 65535:
        raise ValueError(f"{name} exceeds 65535 sequences, tokens or heads")
    dim = rows.shape[3]
    if dim not in (64, 128):
        raise ValueError("head_dim must be 64 or 128")
    unit = 16 // x.element_size()
    if rows.stride(3) != 1 or (rows.shape[2] > 1 and rows.stride(2) != dim) or rows.data_ptr() % 16 or \
            (rows.shape[0] > 1 and rows.stride(0) % unit) or (rows.shape[1] > 1 and rows.stride(1) % unit):
        raise ValueError(f"{name} must have contiguous heads, and tokens and sequences apart by multiples of 16 bytes")
    return rows, dim


def _check_tokens(first, *others):
    for t in (first, *others):
        if t is None:
            continue
        if t.dtype not in _TOKEN_TYPES or t.dtype != first.dtype:
            raise TypeError("queries, keys and values must share float32, float16 or bfloat16")
        if not t.is_cuda or t.device != first.device:
            raise ValueError("inputs must be on one GPU")
        if t.requires_grad:
            raise ValueError("inference only: detach tensors requiring gradients")


def _check_rotation(rotary, dim, like, weights, eps):
    if rotary is None and all(w is None for w, _ in weights):
        raise ValueError("nothing to do: neither a rotation nor norm weights")
    if rotary is not None:
        if not isinstance(rotary, Rotary):
            raise TypeError("rotary must be a Rotary or None")
        if rotary.dims > dim:
            raise ValueError("the rotation turns more dims than a head has")
        if rotary.device != like.device:
            raise ValueError("the rotation lives on another device")
    if isinstance(eps, bool) or not isinstance(eps, (int, float)) or not 0 <= eps < math.inf:
        raise ValueError("eps must be finite and not negative")
    dtypes = {w.dtype for w, _ in weights if w is not None}
    if len(dtypes) > 1 or not dtypes <= {like.dtype, torch.float32}:
        raise TypeError("norm weights must share the inputs' dtype or float32")
    for w, rows in weights:
        if w is None:
            continue
        if rows is None or tuple(w.shape) not in ((dim,), (rows.shape[2], dim)):
            raise ValueError("norm weights must be [D] or [H, D], for heads that are given")
        if w.device != like.device or not w.is_contiguous() or w.data_ptr() % 16:
            raise ValueError("norm weights must be contiguous, 16-byte aligned, on the inputs' device")
        if w.requires_grad:
            raise ValueError("inference only: detach tensors requiring gradients")


def _check_out(out, like):
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError("out must have its input's shape, dtype and device")
    if not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out must be contiguous and 16-byte aligned")
    if out.requires_grad:
        raise ValueError("inference only: detach tensors requiring gradients")


def _rotation(rotary, q_weight, k_weight, eps):
    if rotary is None:
        return None, 0, 1.0, q_weight, k_weight, float(eps)
    return rotary._frequencies, rotary._style, rotary.scale, q_weight, k_weight, float(eps)
