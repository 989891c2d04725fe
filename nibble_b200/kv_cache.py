"""Rotary positions, and a key/value cache held in 8 bits: tokens written, read back and attended over.

The reference leaves positions, cache and attention to HuggingFace (scripts/generate.py:260-365).  With 4-bit weights an FP16
cache soon is the larger part of what a decoded token reads; this one is half its size.

For every sequence and key/value head the tokens come in blocks of 32.  A block that is full is held as 8-bit codes with one FP32
scale for its keys and one for its values (``scale = max|x| / 127``, ``code = round_half_even(127 x / max|x|)``); the block that
is being filled is held as it came.  So what the cache holds depends on the tokens alone, not on how many came at a time, and
each number is rounded once.  A block with an infinity or NaN in it reads back as NaN.

Lengths, starts and counts are contiguous int64 tensors on the device, so that a captured CUDA graph serves every step; one that does not
fit the cache leaves that sequence alone (its outputs are zeros, but for queries that ``append`` turns, which are turned all the same) and is
reported by ``check()``.  None of these operators forms
gradients: an input that requires one, or carries a forward-mode tangent, is refused.  All of them run on the current stream of the tensors' device.
"""
from __future__ import annotations

import torch

from . import _native
from .cuda import _require_extension

_TYPES = {torch.float16: 0, torch.bfloat16: 1}


_ops = None


def _extension():
    global _ops
    if _ops is None:
        _require_extension()
        _ops = _native.load_torch_ops()
    return _ops


def apply_rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, scale: float = 1.0,
                 interleaved: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """FP16 or BF16 ``x`` ``[..., heads, head_dim]`` (two to four dimensions) with every head turned to its position.

    Pair ``j`` of a head at position ``p`` is turned by the angle ``p * inv_freq[j]``; pairs are ``(2j, 2j + 1)`` if
    ``interleaved``, else ``(j, j + rotary_dim / 2)``, with ``rotary_dim = 2 * inv_freq.numel()``; the head's numbers from
    ``rotary_dim`` on stay as they are.  Cosines and sines are multiplied by ``scale``.  Ways of stretching a context are a matter
    of ``inv_freq`` (FP32) and ``scale``.  Angles are formed in FP64, the rest in FP32, rounded once.  ``positions`` (int64, contiguous)
    has the shape of ``x`` without its last two dimensions.  ``out`` may be ``x`` itself, or a tensor of its shape, with any strides, that
    shares no memory with it; of one buffer, two parts of the same rows or parts whose extents are apart.  It counts as changed in place.
    """
    return _extension().rotary(x, positions, inv_freq, scale, interleaved, out)


class QuantizedKVCache:
    """The 8-bit cache of one attention layer: ``batch`` sequences of up to ``max_len`` tokens, ``kv_heads`` heads of
    ``head_dim`` (64 or 128) numbers, which come and are read back as ``dtype`` (FP16 or BF16).

    The cache does not count its tokens: every call says how many there are.  The length may be set back, as after refused
    drafts, as far as the beginning of the block before that of the furthest token that was written; the next ``append`` writes from there.
    """

    BLOCK = 32          # tokens that share a scale

    def __init__(self, batch: int, kv_heads: int, max_len: int, head_dim: int, dtype: torch.dtype = torch.float16,
                 device: torch.device | str | None = None):
        native = _extension()
        if dtype not in _TYPES:
            raise ValueError("a QuantizedKVCache holds torch.float16 or torch.bfloat16 numbers")
        if head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        size = native.kv8_bytes(batch, kv_heads, max_len, head_dim)
        if size == 0:
            raise ValueError("batch, kv_heads and max_len must be positive and within 2^31 blocks")
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise ValueError("a QuantizedKVCache lives on a CUDA device")
        self.batch, self.kv_heads, self.max_len, self.head_dim, self.dtype = batch, kv_heads, max_len, head_dim, dtype
        self.memory = torch.zeros((size,), dtype=torch.uint8, device=device)
        self.device = self.memory.device
        self._sizes = (batch, kv_heads, max_len, head_dim, _TYPES[dtype])

    def append(self, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, counts: torch.Tensor | None = None, *,
               q: torch.Tensor | None = None, inv_freq: torch.Tensor | None = None, rope_scale: float = 1.0,
               interleaved: bool = False) -> torch.Tensor | None:
        """Writes new tokens, ``k`` and ``v`` ``[batch, tokens, kv_heads, head_dim]`` in any order of the first three dimensions, at
        positions ``start[b], start[b] + 1, ...``; of sequence ``b`` the first ``counts[b]`` (default: all).

        With ``inv_freq`` the keys are turned to their positions on the way, and so are the queries ``q`` ``[batch, tokens, q_heads,
        head_dim]``, all ``tokens`` of them, which are returned: the same bits as ``apply_rotary`` in front, for a few tokens in one launch.
        """
        return _extension().kv8_append(self.memory, *self._sizes, k, v, start, counts, inv_freq, rope_scale, interleaved, q)

    def read(self, lengths: torch.Tensor, first: torch.Tensor | None = None,
             tokens: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """What the cache holds: keys and values ``[batch, tokens, kv_heads, head_dim]`` from position ``first[b]`` (default: 0)
        on (up to ``max_len``), of sequences of ``lengths[b]`` tokens; zeros behind the last.  ``tokens`` defaults to ``max_len``."""
        return _extension().kv8_read(self.memory, *self._sizes, lengths, first, self.max_len if tokens is None else tokens)

    def attention(self, q: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor | None = None,
                  softmax_scale: float | None = None) -> torch.Tensor:
        """Attention of the newest tokens over the cache, ``[batch, tokens, q_heads, head_dim]`` like ``q``.

        ``lengths[b]`` counts the newest tokens too; query ``i`` of ``counts[b]`` (default: all of ``tokens``) stands at position
        ``lengths[b] - counts[b] + i`` and sees the positions up to its own.  Query heads are a multiple of the cache's, consecutive
        ones sharing a head.  ``softmax_scale`` defaults to ``head_dim ** -0.5``.  Rows behind a sequence's last query, and
        rows that see nothing, are zeros.  Scores, sums and results are FP32, probabilities times their values' scale FP16 relative to the
        largest of them that a row sees.
        """
        return _extension().kv8_attention(self.memory, *self._sizes, q, lengths, counts,
                                          self.head_dim ** -0.5 if softmax_scale is None else softmax_scale)

    def check(self) -> None:
        """Raises if a call since the last check was given a length, start or count that does not fit, or gave up a bounded wait.
        Synchronises; clears what it reports."""
        word = self.memory[:4].view(torch.int32)
        status = int(word.item())
        if status:
            word.zero_()
            raise RuntimeError("attention over the 8-bit cache gave up waiting; its output is incomplete" if status & 2 else
                               "a length, start or count did not fit the 8-bit cache")
