"""-m gpu: rotary positions and the 8-bit cache where a call is out of the ordinary: works without a step, numbers far apart in size,
tokens taken back at a block's end, outputs beside their inputs, tangents."""
from __future__ import annotations

import pytest
import torch

import kv_oracle as oracle
from nibble_b200 import QuantizedKVCache, apply_rotary
from test_gpu_kv_cache import _draw, _held, _words

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [72, 200])
def test_infinities_of_the_newest_block_are_seen_beside_works_without_a_step(rows, dtype):
    """Many queries, as many units as make five rounds of the machine's CTAs, the three rounds in the middle without a query."""
    kv_heads, group, d = 8, 8, 64
    tokens, batch = rows // group, (5 * 148) // 8 + 1
    first, last = 148 // 8, 4 * 148 // 8
    lengths, counts = [40] * batch, [tokens if b <= first or b >= last else 0 for b in range(batch)]
    k, v = _draw((batch, 40, kv_heads, d), dtype, 1), _draw((batch, 40, kv_heads, d), dtype, 2)
    v[:, 33, :, 7] = float("inf")
    cache = QuantizedKVCache(batch, kv_heads, 64, d, dtype=dtype)
    cache.append(k, v, _words([0] * batch))
    q = _draw((batch, tokens, group * kv_heads, d), dtype, 3)
    for _ in range(3):
        got = cache.attention(q, _words(lengths), _words(counts))
        for b in range(batch):
            if counts[b] == 0:
                assert not got[b].any()
                continue
            sees = torch.arange(40 - tokens, 40, device="cuda") >= 33
            assert (got[b, sees, :, 7] == float("inf")).all(), b
            assert got[b, ~sees].isfinite().all() and got[b, :, :, :7].isfinite().all() and got[b, :, :, 8:].isfinite().all(), b
    cache.check()
