"""Norms of queries and keys for each head with the position rotation, alone or on the way into the paged cache.

``rotate_heads`` norms and rotates new queries and keys; ``append_rotated``
does so while it writes the keys, and the values beside them, into the cache
(``DecodePlan.append_rotated`` at the plan's own lengths). The reference has
neither: it leaves what is written to the cache to its caller
(docs/DESIGN.md:11-13).
"""
import math

import torch

from .layout import Layout
from .runtime import dimensions, load_extension, rotation_arguments

_STYLES = {"half": 0, "interleaved": 1}


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
        self._arguments = (frequencies.to(device=self.device, dtype=torch.float64, copy=True), _STYLES[style], self.scale)


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
    q_out, k_out = (None, None) if out is None else out
    if out is not None and (q_out is None or (k_out is None) != (k is None)):
        raise ValueError("out must give an output for each input")
    return load_extension().rotate_heads(q, k, positions, *rotation_arguments(rotary), q_weight, k_weight, eps, q_out, k_out)


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
    return load_extension().append_rotated(dimensions(layout), k_cache, v_cache, table, positions, k_new, v_new, q,
                                           *rotation_arguments(rotary), q_weight, k_weight, eps, k_scale, v_scale, counts, out, -1)

