"""-m gpu: rotary positions and the 8-bit cache where a call is out of the ordinary: works without a step, numbers far apart in size,
tokens taken back at a block's end, outputs beside their inputs, tangents."""
from __future__ import annotations

import pytest
import torch

import kv_oracle as oracle
from nibble_b200 import QuantizedKVCache, apply_rotary
from test_gpu_kv_cache import _check_attention, _draw, _held, _words

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


@pytest.mark.parametrize("length", [20, 64, 90])
@pytest.mark.parametrize(("tokens", "q_heads", "head_dim"), [(1, 4, 128), (5, 8, 64), (20, 16, 128), (20, 16, 64)])
@pytest.mark.parametrize(("q_size", "k_size", "v_size"), [(120, -120, 117), (-122, 121, 0), (0, 0, -100), (118, -118, 1)])
def test_bf16_numbers_of_any_size(q_size, k_size, v_size, tokens, q_heads, head_dim, length):
    """Powers of two that all but use up the type's range, in few rows and many, in full blocks and in the one being filled."""
    dtype = torch.bfloat16
    k, v = (_draw((1, length, 1, head_dim), dtype, seed, 2.0 ** size) for seed, size in ((5, k_size), (6, v_size)))
    q = _draw((1, tokens, q_heads, head_dim), dtype, 7, 2.0 ** q_size)
    cache = QuantizedKVCache(1, 1, length + 3, head_dim, dtype=dtype)
    cache.append(k, v, _words([0]))
    _check_attention(cache, k, v, q, [length], None)
    cache.check()


@pytest.mark.parametrize(("tokens", "q_heads"), [(4, 8), (40, 8)])
def test_a_key_far_out_does_not_cost_others_their_bits(tokens, q_heads):
    """The block that is being filled, BF16, numbers of one key 10^12 times the others, which meet zeros in the queries."""
    length = 50
    k, v, q = (_draw((1, n, heads, 64), torch.bfloat16, seed) for n, heads, seed in ((length, 1, 8), (length, 1, 9), (tokens, q_heads, 10)))
    k[:, length - 3, :, :8] *= 1e12
    q[..., :8] = 0.0
    cache = QuantizedKVCache(1, 1, 64, 64, dtype=torch.bfloat16)
    cache.append(k, v, _words([0]))
    _check_attention(cache, k, v, q, [length], None)


def _equal_scores(dtype, tokens, q_heads, head_dim, length, q_size, k_size, seed):
    """A cache all of whose keys are the same, exactly so as codes and as they came, and queries of one number."""
    k = torch.full((1, length, 1, head_dim), 127.0 * 2.0 ** k_size, dtype=dtype, device="cuda")
    v = _draw((1, length, 1, head_dim), dtype, seed)
    cache = QuantizedKVCache(1, 1, length + 3, head_dim, dtype=dtype)
    cache.append(k, v, _words([0]))
    return cache, k, v, torch.full((1, tokens, q_heads, head_dim), q_size, dtype=dtype, device="cuda")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("length", [20, 64, 90, 700])
@pytest.mark.parametrize(("tokens", "q_heads", "head_dim"), [(1, 4, 128), (1, 8, 64), (5, 8, 64), (20, 16, 128), (20, 16, 64)])
def test_equal_scores_of_any_size_count_alike(tokens, q_heads, head_dim, length, sign, dtype):
    """Scores of 3 * 10^10 and more: what a row of them gives is the mean."""
    cache, k, v, q = _equal_scores(dtype, tokens, q_heads, head_dim, length, sign * 2.0 ** 14, 8, 11)
    _check_attention(cache, k, v, q, [length], None, 1.0)
    _check_attention(cache, k, v, q, [length], None, 0.7)
    cache.check()


@pytest.mark.parametrize(("tokens", "q_heads"), [(1, 8), (4, 8), (40, 8)])
@pytest.mark.parametrize("length", [50, 333])
def test_a_score_far_out(tokens, q_heads, length):
    """One key 10^12 times the others: it is all that a query sees, or nothing of it."""
    k, v = _draw((1, length, 1, 64), torch.bfloat16, 12), _draw((1, length, 1, 64), torch.bfloat16, 13)
    k[:, length - 3] *= 1e12
    cache = QuantizedKVCache(1, 1, length, 64, dtype=torch.bfloat16)
    cache.append(k, v, _words([0]))
    _check_attention(cache, k, v, _draw((1, tokens, q_heads, 64), torch.bfloat16, 14), [length], None)


@pytest.mark.parametrize("length", [20, 64, 90, 700])
@pytest.mark.parametrize(("tokens", "q_heads", "head_dim"), [(1, 4, 128), (1, 8, 64), (5, 8, 64), (20, 16, 128), (20, 16, 64)])
def test_scores_near_the_ends_of_fp32(tokens, q_heads, head_dim, length):
    """Scores of some -10^37, all equal: the mean, not a row that sees nothing."""
    for sign in (-1.0, 1.0):
        cache, k, v, q = _equal_scores(torch.bfloat16, tokens, q_heads, head_dim, length, sign * 2.0 ** 60, 49, 15)
        _check_attention(cache, k, v, q, [length], None, 1.0)
        cache.check()
