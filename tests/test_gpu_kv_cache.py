"""-m gpu: rotary positions, the 8-bit key/value cache written and read back, and attention over it, against their definitions in
64 bits (tests/kv_oracle.py)."""
from __future__ import annotations

import pytest
import torch

import kv_oracle as oracle
from nibble_b200 import QuantizedKVCache, apply_rotary

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def _words(values):
    return torch.tensor(values, dtype=torch.long, device="cuda")


def _draw(shape, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * spread).to(dtype).cuda()


def _same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0))


def _held(x, lengths):
    """What a cache of `lengths` gives back of [batch, tokens, heads, d], in the cache's type (code * scale is rounded to FP32 by the
    kernel first; the product of 7 and 24 bits has 31, so 64 bits hold it exactly and the two roundings are repeated here)."""
    return torch.stack([oracle.held(x[b], n).float().to(x.dtype) for b, n in enumerate(lengths)])


# ------------------------------------------------------------------ rotary positions

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("shape", "rotary_dim", "interleaved"), [
    ((1, 5, 64), 64, False), ((1, 36, 64), 64, True), ((9, 3, 128), 96, True), ((9, 3, 128), 96, False), ((17, 40, 128), 62, False),
    ((3, 2, 7, 80), 40, False), ((2, 33, 9, 256), 256, True), ((5, 1, 2), 2, False), ((4, 6, 66), 34, True), ((3, 64), 48, False),
    ((300, 72, 128), 128, False), ((130, 72, 128), 90, False), ((70, 9, 64), 36, False), ((33, 40, 128), 50, True), ((6, 5, 256), 254, False)])
def test_rotary_is_its_definition(shape, rotary_dim, interleaved, dtype):
    x = _draw(shape, dtype, sum(shape))
    g = torch.Generator().manual_seed(rotary_dim)
    positions = torch.randint(0, 1 << 20, shape[:-2], generator=g).cuda()
    inv_freq = (500000.0 ** (-torch.arange(0, rotary_dim, 2).double() / rotary_dim)).float().cuda()
    for scale in (1.0, 1.1386294):
        want = oracle.rotary(x, positions, inv_freq, scale, interleaved)
        got = apply_rotary(x, positions, inv_freq, scale=scale, interleaved=interleaved)
        assert got.dtype == dtype and got.shape == x.shape
        # FP32 factors (each off by a few 2^-24) and a sum of two products, then one rounding
        size = x.double().abs().amax(-1, keepdim=True) * scale * 2
        assert ((got.double() - want).abs() <= want.abs() * torch.finfo(dtype).eps / 2 + size * 2.0 ** -21 + 2.0 ** -25).all()
        assert torch.equal(got[..., rotary_dim:], x[..., rotary_dim:])
        same = x.clone()
        assert apply_rotary(same, positions, inv_freq, scale, interleaved, out=same) is same
        assert torch.equal(same, got)
        into = torch.full_like(x, 7.0)
        apply_rotary(x, positions, inv_freq, scale, interleaved, out=into)
        assert torch.equal(into, got)


def test_rotary_of_views_of_a_larger_row_and_odd_addresses():
    """Queries and keys as slices of a fused projection's output, turned in place; and rows that start at any address."""
    heads, d = 6, 64
    inv_freq = (10000.0 ** (-torch.arange(0, d, 2).double() / d)).float().cuda()
    positions = _words([[3, 4, 5], [700, 701, 702]])
    for offset in (0, 1, 8):
        row = _draw((2, 3, (heads + 4) * d + 16), torch.float16, offset)
        before = row.clone()
        view = row[:, :, offset:offset + heads * d].view(2, 3, heads, d)
        want = apply_rotary(view.contiguous(), positions, inv_freq)
        apply_rotary(view, positions, inv_freq, out=view)
        assert torch.equal(view, want)
        assert torch.equal(row[:, :, :offset], before[:, :, :offset])
        assert torch.equal(row[:, :, offset + heads * d:], before[:, :, offset + heads * d:])
    turned = _draw((2, heads, 3, d), torch.bfloat16, 5).transpose(1, 2)           # [batch, tokens, heads, d] by strides
    assert torch.equal(apply_rotary(turned, positions, inv_freq), apply_rotary(turned.contiguous(), positions, inv_freq))


def test_rotary_of_nothing_and_of_far_positions():
    inv_freq = torch.ones((32,), device="cuda")
    assert apply_rotary(torch.empty((0, 4, 64), dtype=torch.float16, device="cuda"), _words([]), inv_freq).shape == (0, 4, 64)
    x = torch.zeros((3, 1, 64), dtype=torch.float16, device="cuda")
    x[..., :32] = 1.0
    got = apply_rotary(x, _words([(1 << 40) + 1, 1 << 31, -5]), inv_freq)
    want = oracle.rotary(x.cpu(), torch.tensor([(1 << 40) + 1, 1 << 31, -5]), inv_freq.cpu(), 1.0, False)
    # the angle in turns: 2^40 / (2 pi) is 1.7e11, of which 64 bits keep 2^-15 of a turn's part in 10^9
    assert ((got.cpu().double() - want).abs() <= 2.0 ** -11 + 1e-3).all()


# ------------------------------------------------------------------ written and read back

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("head_dim", "kv_heads", "max_len", "pieces"), [
    (64, 2, 200, [1, 30, 1, 1, 64, 5, 90]), (128, 3, 129, [33, 31, 64, 1]), (128, 1, 96, [96]), (64, 1, 31, [7, 24]),
    (64, 4, 700, [5, 100, 27, 500, 1]), (128, 2, 1, [1])])
def test_what_is_held_does_not_depend_on_how_it_came(head_dim, kv_heads, max_len, pieces, dtype):
    k, v = _draw((2, max_len, kv_heads, head_dim), dtype, 1), _draw((2, max_len, kv_heads, head_dim), dtype, 2, 0.3)
    cache = QuantizedKVCache(2, kv_heads, max_len, head_dim, dtype=dtype)
    at = 0
    for piece in pieces:
        cache.append(k[:, at:at + piece], v[:, at:at + piece], _words([at, at]))
        at += piece
        got_k, got_v = cache.read(_words([at, at]))
        assert torch.equal(got_k, _held(k, [at, at])) and torch.equal(got_v, _held(v, [at, at])), at
    whole = QuantizedKVCache(2, kv_heads, max_len, head_dim, dtype=dtype)
    whole.append(k[:, :at], v[:, :at], _words([0, 0]))
    for a, b in zip(cache.read(_words([at, at])), whole.read(_words([at, at]))):
        assert torch.equal(a, b)
    for tensor, want in zip(cache.read(_words([at, at // 2]), first=_words([0, 0]), tokens=at), (k, v)):
        assert torch.equal(tensor[0], _held(want, [at, at])[0][:at])
    cache.check()


def test_token_by_token_over_several_blocks():
    k, v = _draw((1, 100, 2, 64), torch.float16, 3), _draw((1, 100, 2, 64), torch.float16, 4)
    cache = QuantizedKVCache(1, 2, 100, 64)
    for t in range(100):
        cache.append(k[:, t:t + 1], v[:, t:t + 1], _words([t]))
    got_k, got_v = cache.read(_words([100]))
    assert torch.equal(got_k, _held(k, [100])) and torch.equal(got_v, _held(v, [100]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_ragged_counts_leave_the_rest_alone(dtype):
    """Sequences of different lengths and counts, none among them; tokens behind a count and other sequences are not touched."""
    starts, counts = [0, 37, 64, 95, 10, 0], [70, 3, 0, 1, 54, 70]
    old = _draw((6, 100, 2, 128), dtype, 5)
    new = _draw((6, 70, 2, 128), dtype, 6)
    cache = QuantizedKVCache(6, 2, 165, 128, dtype=dtype)
    cache.append(old, old, _words([0] * 6), _words(starts))
    cache.append(new, new, _words(starts), _words(counts))
    ends = [s + c for s, c in zip(starts, counts)]
    want = torch.zeros((6, 165, 2, 128), dtype=dtype, device="cuda")
    for b in range(6):
        want[b, :starts[b]] = old[b, :starts[b]]
        want[b, starts[b]:ends[b]] = new[b, :counts[b]]
    for got in cache.read(_words(ends)):
        assert torch.equal(got, _held(want, ends))
    # ranges of it, beyond the last token too
    first = [0, 31, 64, 90, 33, 69]
    got, _ = cache.read(_words(ends), first=_words(first), tokens=40)
    for b in range(6):
        piece = torch.zeros((40, 2, 128), dtype=dtype, device="cuda")
        upto = min(ends[b], first[b] + 40)
        if upto > first[b]:
            piece[:upto - first[b]] = _held(want, ends)[b, first[b]:upto]
        assert torch.equal(got[b], piece), b
    cache.check()


def test_tokens_taken_back_are_written_again():
    """The length falls as far as the beginning of the block before the newest; what was there counts again."""
    k, v = _draw((1, 200, 1, 64), torch.float16, 7), _draw((1, 200, 1, 64), torch.float16, 8)
    other = _draw((1, 200, 1, 64), torch.float16, 9)
    for reached, back in ((100, 70), (100, 64), (96, 64), (97, 96), (65, 63), (33, 1), (130, 128)):
        cache = QuantizedKVCache(1, 1, 200, 64)
        cache.append(k[:, :reached], v[:, :reached], _words([0]))
        assert torch.equal(cache.read(_words([back]))[0], _held(k, [back]))
        for piece in (3, 60):
            cache.append(other[:, :piece], other[:, :piece], _words([back]))
            mixed = torch.cat((k[:, :back], other[:, :piece], k[:, back + piece:]), 1)
            assert torch.equal(cache.read(_words([back + piece]))[0], _held(mixed, [back + piece])), (reached, back, piece)
            if piece == 3 and (back + 3) // 32 != back // 32:
                break                                  # the block was closed: back again is not promised


def test_rows_at_any_stride_and_address():
    k = _draw((2, 3, 50, 64), torch.float16, 10)                       # [batch, heads, tokens, d]
    fused = _draw((2, 50, 3 * 64 * 2 + 5), torch.float16, 11)
    for offset in (0, 1, 3):
        by_stride, odd = k.transpose(1, 2), fused[:, :, offset:offset + 3 * 64].unflatten(-1, (3, 64))
        cache = QuantizedKVCache(2, 3, 64, 64)
        cache.append(by_stride, odd, _words([0, 0]))
        got_k, got_v = cache.read(_words([50, 50]))
        assert torch.equal(got_k, _held(torch.nn.functional.pad(by_stride.contiguous(), (0, 0, 0, 0, 0, 14)), [50, 50]))
        assert torch.equal(got_v, _held(torch.nn.functional.pad(odd.contiguous(), (0, 0, 0, 0, 0, 14)), [50, 50]))
    one = k[:, :, :1].transpose(1, 2).expand(2, 50, 3, 64)             # the same token again and again, stride zero
    cache = QuantizedKVCache(2, 3, 64, 64)
    cache.append(one, one, _words([0, 0]))
    assert torch.equal(cache.read(_words([50, 50]))[0][:, 40], one[:, 40])


@pytest.mark.parametrize("dtype", DTYPES)
def test_codes_at_ties_extremes_and_zero(dtype):
    big = torch.finfo(dtype).max
    g = torch.Generator().manual_seed(12)
    block = torch.zeros((5, 32, 1, 64))
    block[0] = torch.arange(32 * 64).view(32, 1, 64) % 255 - 127          # a scale of one: codes are the numbers
    block[1] = (torch.arange(32 * 64).view(32, 1, 64) % 509 - 254) / 2      # and ties
    block[1, 0, 0, 0] = 127.0
    block[2] = torch.randn((32, 1, 64), generator=g).to(dtype).float() * big / 8
    block[2, 3, 0, 5] = -big
    block[2] = block[2].clamp(-big, big)
    block[3] = torch.randn((32, 1, 64), generator=g) * torch.finfo(dtype).smallest_normal
    x = block.to(dtype).cuda()
    cache = QuantizedKVCache(5, 1, 32, 64, dtype=dtype)
    cache.append(x, x, _words([0] * 5))
    for got in cache.read(_words([32] * 5)):
        want = _held(x, [32] * 5)
        assert torch.equal(got[:3], want[:3]) and torch.equal(got[4], want[4])
        # (scales below the smallest normal FP32 are rounded there, in FP32 and BF16 both)
        assert ((got[3].double() - want[3].double()).abs() <= want[3].double().abs() * torch.finfo(dtype).eps + 1e-44).all()
        assert torch.equal(got[0].cpu().float(), block[0])


def test_numbers_that_are_not_finite_stay_with_their_block_and_head():
    x = _draw((1, 96, 2, 64), torch.float16, 13)
    for bad in (float("nan"), float("inf"), -float("inf")):
        k, v = x.clone(), x.clone()
        k[0, 40, 1, 3] = bad
        v[0, 70, 0, 9] = bad
        cache = QuantizedKVCache(1, 2, 96, 64)
        cache.append(k[:, :90], v[:, :90], _words([0]))
        got_k, got_v = cache.read(_words([90]))
        assert _same(got_k, _held(k, [90])) and _same(got_v, _held(v, [90]))     # (token 70 is held as it came)
        cache.append(k[:, 90:], v[:, 90:], _words([90]))
        assert _same(cache.read(_words([96]))[1], _held(v, [96]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("head_dim", "rotary_dim", "interleaved", "starts", "tokens"), [
    (64, 64, False, [0, 1500], 1), (128, 128, False, [31, 95], 70), (128, 48, True, [5, 0], 33), (64, 34, False, [100, 31], 2),
    (128, 128, True, [0, 0], 200)])
def test_turning_while_writing_is_turning_first(head_dim, rotary_dim, interleaved, starts, tokens, dtype):
    kv_heads, q_heads = 2, 10
    row = _draw((2, tokens, (q_heads + 2 * kv_heads) * head_dim), dtype, tokens)
    q, k, v = (part.unflatten(-1, (-1, head_dim)) for part in row.split([q_heads * head_dim] + [kv_heads * head_dim] * 2, -1))
    older = _draw((2, 1500, kv_heads, head_dim), dtype, 14)
    inv_freq = (10000.0 ** (-torch.arange(0, rotary_dim, 2).double() / rotary_dim)).float().cuda()
    start = _words(starts)
    places = start[:, None] + torch.arange(tokens, device="cuda")
    caches = [QuantizedKVCache(2, kv_heads, 1800, head_dim, dtype=dtype) for _ in range(2)]
    for cache in caches:
        cache.append(older, older, _words([0, 0]), start)
    turned = caches[0].append(k, v, start, q=q, inv_freq=inv_freq, rope_scale=1.25, interleaved=interleaved)
    assert torch.equal(turned, apply_rotary(q, places, inv_freq, scale=1.25, interleaved=interleaved))
    caches[1].append(apply_rotary(k, places, inv_freq, scale=1.25, interleaved=interleaved), v, start)
    assert torch.equal(caches[0].memory, caches[1].memory)
    assert caches[0].append(k, v, start, inv_freq=inv_freq) is None


def test_places_outside_the_cache_are_reported_and_nothing_is_written():
    x = _draw((3, 40, 1, 64), torch.float16, 15)
    cache = QuantizedKVCache(3, 1, 50, 64)
    cache.append(x, x, _words([0, 0, 0]))
    before = cache.memory.clone()
    for starts, counts in (([11, -1, 50], [40, 1, 1]), ([0, 0, 0], [-1, 41, 1 << 40]), ([1 << 62, 1 << 33, 51], [40, 40, 0])):
        cache.append(x, x, _words(starts), _words(counts))
        with pytest.raises(RuntimeError, match="did not fit"):
            cache.check()
        assert torch.equal(cache.memory, before)
    cache.check()
    for got in cache.read(_words([51, -3, 40])):
        assert not got[:2].any() and torch.equal(got[2, :40], _held(x, [40] * 3)[2])
    with pytest.raises(RuntimeError, match="did not fit"):
        cache.check()
    got, _ = cache.read(_words([40, 40, 40]), first=_words([-1, 45, 1 << 40]), tokens=3)
    assert not got.any()


# ------------------------------------------------------------------ attention

def _filled(batch, kv_heads, max_len, head_dim, dtype, lengths, seed=20):
    k = _draw((batch, max_len, kv_heads, head_dim), dtype, seed, 1.3)
    v = _draw((batch, max_len, kv_heads, head_dim), dtype, seed + 1, 0.7)
    k[:, :, :, 5] += 3.0                                              # a channel far out, as keys have them
    cache = QuantizedKVCache(batch, kv_heads, max_len, head_dim, dtype=dtype)
    cache.append(k, v, _words([0] * batch), _words(lengths))
    return cache, k, v


def _check_attention(cache, k, v, q, lengths, counts, scale=None):
    got = cache.attention(q, _words(lengths), None if counts is None else _words(counts), softmax_scale=scale)
    assert got.shape == q.shape and got.dtype == q.dtype and got.is_contiguous()
    counts = [q.shape[1]] * len(lengths) if counts is None else counts
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    for b, (length, count) in enumerate(zip(lengths, counts)):
        kb, vb = oracle.held(k[b], length)[:length], oracle.held(v[b], length)[:length]
        want, weight = oracle.attention(q[b], kb, vb, length, count, scale)
        top = float(vb.abs().max()) * length if length else 0.0
        bound = oracle.attention_bound(want, weight, q.dtype, top)
        off = (got[b].double() - want).abs()
        assert (off <= bound).all(), (b, length, count, float((off - bound).max()), float((off / bound.clamp_min(1e-30)).max()))
        assert not got[b, count:].any()
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("q_heads", "kv_heads", "head_dim"), [(8, 2, 64), (8, 1, 128), (3, 3, 128), (20, 1, 64), (36, 2, 128)])
def test_attention_of_one_token_at_every_kind_of_length(q_heads, kv_heads, head_dim, dtype):
    lengths = [1, 2, 31, 32, 33, 63, 64, 65, 100, 255, 256, 257, 300, 511, 0, 640]
    cache, k, v = _filled(len(lengths), kv_heads, 640, head_dim, dtype, lengths)
    q = _draw((len(lengths), 1, q_heads, head_dim), dtype, 22)
    _check_attention(cache, k, v, q, lengths, None)
    cache.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("tokens", "q_heads", "kv_heads", "head_dim"), [
    (2, 8, 2, 64), (5, 8, 1, 128), (4, 4, 4, 64), (9, 6, 1, 128), (33, 4, 2, 64), (70, 3, 1, 128)])
def test_attention_of_several_tokens(tokens, q_heads, kv_heads, head_dim, dtype):
    lengths = [tokens, tokens + 1, 97 + tokens, 200, 256, 301]
    counts = [tokens, 1, tokens // 2, tokens, 0, tokens]
    cache, k, v = _filled(len(lengths), kv_heads, 320, head_dim, dtype, lengths)
    q = _draw((len(lengths), tokens, q_heads, head_dim), dtype, 23)
    _check_attention(cache, k, v, q, lengths, counts)
    _check_attention(cache, k, v, q, lengths, None)
    cache.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("tokens", "q_heads", "kv_heads", "head_dim", "lengths"), [
    (128, 1, 1, 64, [128]), (256, 1, 1, 128, [256]), (100, 2, 1, 128, [1000]), (33, 8, 2, 64, [513, 33, 100]),
    (300, 8, 2, 128, [300, 777, 3011]), (257, 12, 4, 64, [257, 600]), (130, 3, 1, 64, [2000]), (700, 16, 4, 64, [700, 1000, 701, 900]),
    (40, 40, 8, 128, [40, 73, 4000])])
def test_attention_of_a_prompts_chunk(tokens, q_heads, kv_heads, head_dim, lengths, dtype):
    """Tiles and steps that end anywhere, units that are cut along the tokens and rounds of whole ones."""
    cache, k, v = _filled(len(lengths), kv_heads, max(lengths) + 5, head_dim, dtype, lengths)
    q = _draw((len(lengths), tokens, q_heads, head_dim), dtype, 46, 1.5)
    first = _check_attention(cache, k, v, q, lengths, None)
    assert torch.equal(cache.attention(q, _words(lengths)), first)
    counts = [max(0, tokens - 50 * b) for b in range(len(lengths))]
    _check_attention(cache, k, v, q, lengths, counts)
    _check_attention(cache, k, v, q, lengths, None, -0.05)
    cache.check()


@pytest.mark.parametrize("tokens", [1, 3, 40, 90])
def test_queries_without_a_position_and_short_caches(tokens):
    """More queries than tokens held: the ones in front of the first token see nothing."""
    lengths = [1, 0, 2, 35]
    for max_len in (35, 400):
        cache, k, v = _filled(4, 2, max_len, 64, torch.float16, lengths)
        q = _draw((4, tokens, 8, 64), torch.float16, 24)
        _check_attention(cache, k, v, q, lengths, None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("head_dim", "q_heads", "kv_heads", "tokens", "length"), [
    (128, 8, 1, 1, 20011), (64, 32, 4, 1, 9000), (128, 64, 8, 2, 4099), (64, 4, 4, 17, 5000)])
def test_attention_over_long_contexts(head_dim, q_heads, kv_heads, tokens, length, dtype):
    cache, k, v = _filled(1, kv_heads, length + 13, head_dim, dtype, [length])
    q = _draw((1, tokens, q_heads, head_dim), dtype, 25, 2.0)
    first = _check_attention(cache, k, v, q, [length], None)
    for _ in range(3):
        assert torch.equal(cache.attention(q, _words([length])), first)        # the same bits every time


def test_attention_with_scores_and_values_of_every_size():
    """A scale that makes one token win, or all count alike; blocks of values far apart in size, zeros among them."""
    length = 500
    k, v = _draw((1, 512, 1, 64), torch.float16, 26), _draw((1, 512, 1, 64), torch.float16, 27)
    sizes = torch.tensor([1e-3, 1.0, 0.0, 300.0, 1e-4, 30.0, 0.01, 1.0, 1e3, 1e-5, 5.0, 0.0, 2.0, 0.1, 100.0, 1.0])
    v = (v * sizes.half().cuda().repeat_interleave(32)[None, :, None, None]).contiguous()
    for order in (torch.arange(512), torch.arange(511, -1, -1)):
        vo = v[:, order.cuda()].contiguous()
        cache = QuantizedKVCache(1, 1, 512, 64)
        cache.append(k, vo, _words([0]), _words([length]))
        for spread, scale in ((1.0, None), (4.0, 1.0), (1.0, 0.0), (1.0, -0.125)):
            q = _draw((1, 1, 8, 64), torch.float16, 28, spread)
            _check_attention(cache, k, vo, q, [length], None, scale)


def test_what_is_masked_does_not_matter():
    """Infinities and NaN behind the last token, in tokens that a query does not see, and in stale tails."""
    bad = float("nan")
    for where in (bad, float("inf")):
        k, v = _draw((2, 100, 2, 64), torch.float16, 30), _draw((2, 100, 2, 64), torch.float16, 31)
        dirty_k, dirty_v = k.clone(), v.clone()
        for x in (dirty_k, dirty_v):
            x[0, 50:] = where                                          # a full block from 64 on, and half of one
            x[1, 99] = where                                           # in the tail
        cache = QuantizedKVCache(2, 2, 128, 64)
        cache.append(dirty_k, dirty_v, _words([0, 0]))
        q = _draw((2, 60, 8, 64), torch.float16, 32)
        got = cache.attention(q, _words([100, 100]))
        # queries stand at 40..99: those up to 49 of the first sequence see full blocks with a NaN in them (tokens 32..63 share a block)
        assert got[0].isnan().any(-1).all()
        clean = QuantizedKVCache(2, 2, 128, 64)
        clean.append(k, v, _words([0, 0]))
        want = clean.attention(q, _words([100, 100]))
        assert torch.equal(got[1, :59], want[1, :59]) and not got[1, 59].isfinite().any(-1).any()
        # the same cache, shorter: nothing of it is seen
        few = q[:, :32]
        assert torch.equal(cache.attention(few, _words([32, 99])), clean.attention(few, _words([32, 99])))
        # earlier queries of a sequence whose newest block alone is spoilt
        again = QuantizedKVCache(2, 2, 128, 64)
        again.append(k, v, _words([0, 0]), _words([64, 64]))
        again.append(dirty_k[:, 64:], dirty_v[:, 64:], _words([64, 64]), _words([32, 32]))
        got = again.attention(q, _words([96, 96]))
        held = clean.attention(q, _words([96, 96]))
        assert torch.equal(got[0, :28], held[0, :28]) and got[0, 28:].isnan().any(-1).all()
    # one infinity among the values: that dimension alone
    v[0, 99, 0, 7] = float("inf")
    cache = QuantizedKVCache(2, 2, 128, 64)
    cache.append(k, v, _words([0, 0]))
    got = cache.attention(q, _words([100, 100]))
    assert (got[0, 59, :4, 7] == float("inf")).all() and got[0, 59, :4, :7].isfinite().all() and got[0, :59].isfinite().all()
    q[0, 3, 2] = bad                                                    # a query that is NaN: its own row alone
    got = cache.attention(q, _words([100, 100]))
    assert got[0, 3, 2].isnan().all() and got[0, 3, 1].isfinite().all() and got[0, 4, 2].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("tokens", "q_heads", "kv_heads"), [(1, 8, 2), (5, 8, 2), (90, 8, 2), (300, 64, 1)])
def test_many_light_tokens_beside_a_heavy_one(tokens, q_heads, kv_heads, dtype):
    """Half of the result comes of thousands of small probabilities of small values: they keep their bits, whatever the block that is
    being filled is held as."""
    length = 8017
    k = torch.zeros((1, length, kv_heads, 64), dtype=dtype, device="cuda")
    k[:, 5] = 1.0
    v = (0.001 * (1.0 + 0.2 * _draw((1, length, kv_heads, 64), torch.float32, 52).clamp(-2, 2))).to(dtype)
    cache = QuantizedKVCache(1, kv_heads, length + 7, 64, dtype=dtype)
    cache.append(k, v, _words([0]))
    q = torch.full((1, tokens, q_heads, 64), 9.0 / 64, dtype=dtype, device="cuda")        # scores of nine, and of zero
    _check_attention(cache, k, v, q, [length], None, 1.0)
    cache.check()


@pytest.mark.parametrize("spread", [1.0, 3.0])
@pytest.mark.parametrize(("tokens", "q_heads", "kv_heads", "head_dim", "length"), [
    (1, 32, 4, 64, 500), (1, 8, 1, 128, 3001), (4, 8, 1, 128, 700), (5, 16, 2, 64, 999)])
def test_fp16_results_are_off_by_their_own_rounding(tokens, q_heads, kv_heads, head_dim, length, spread):
    """Few rows: what a probability's rounding leaves is not lost, so that the bound's parts for it fall away."""
    cache, k, v = _filled(1, kv_heads, length, head_dim, torch.float16, [length])
    q = _draw((1, tokens, q_heads, head_dim), torch.float16, 53, spread)
    got = cache.attention(q, _words([length]))[0].double()
    kh, vh = oracle.held(k[0], length), oracle.held(v[0], length)
    want, weight = oracle.attention(q[0], kh, vh, length, tokens, head_dim ** -0.5)
    bound = oracle.attention_bound(want, weight, torch.float16, float(vh.abs().max()) * length) - (weight + want.abs()) * 2.0 ** -11
    assert ((got - want).abs() <= bound).all()


def test_large_bf16_numbers():
    """Beyond FP16's range, in queries, keys and values, in full blocks and in the tail."""
    k, v = _draw((1, 80, 1, 128), torch.bfloat16, 33, 1e6), _draw((1, 80, 1, 128), torch.bfloat16, 34, 1e9)
    q = _draw((1, 1, 4, 128), torch.bfloat16, 35, 1e-5)
    cache = QuantizedKVCache(1, 1, 80, 128, dtype=torch.bfloat16)
    cache.append(k, v, _words([0]))
    _check_attention(cache, k, v, q, [80], None)
    q, k = _draw((1, 1, 4, 128), torch.bfloat16, 36, 1e8), k * 2.0 ** -52
    cache.append(k, v, _words([0]))
    _check_attention(cache, k, v, q, [80], None)


def test_lengths_outside_the_cache_give_zeros_and_are_reported():
    cache, k, v = _filled(4, 2, 300, 64, torch.float16, [300] * 4)
    q = _draw((4, 2, 8, 64), torch.float16, 37)
    got = cache.attention(q, _words([301, -1, 300, 1 << 40]))
    assert not got[0].any() and not got[1].any() and not got[3].any() and got[2].any()
    with pytest.raises(RuntimeError, match="did not fit"):
        cache.check()
    got = cache.attention(q, _words([300] * 4), _words([2, 3, -1, 1]))
    assert not got[1].any() and not got[2].any() and got[0].any() and not got[3, 1].any() and got[3, 0].any()
    with pytest.raises(RuntimeError, match="did not fit"):
        cache.check()


def test_queries_at_any_stride_and_address():
    lengths = [90, 33]
    cache, k, v = _filled(2, 2, 320, 64, torch.float16, lengths)
    fused = _draw((2, 3, 8 * 64 + 3), torch.float16, 38)
    for offset in (0, 1):
        q = fused[:, :, offset:offset + 512].unflatten(-1, (8, 64))
        assert torch.equal(cache.attention(q, _words(lengths)), cache.attention(q.contiguous(), _words(lengths)))
    q = _draw((2, 8, 3, 64), torch.float16, 39).transpose(1, 2)
    assert torch.equal(cache.attention(q, _words(lengths)), cache.attention(q.contiguous(), _words(lengths)))
    none = cache.attention(q[:, :0], _words(lengths))
    assert none.shape == (2, 0, 8, 64)
    cache.append(k[:, :0], v[:, :0], _words(lengths))


@pytest.mark.parametrize(("tokens", "kv_heads", "head_dim"), [(1, 4, 64), (20, 2, 128), (5, 3, 64)])
def test_more_sequences_than_the_machine_holds_at_once(tokens, kv_heads, head_dim):
    """Runs and units that cross sequences, and rounds of whole units in front of ones that are cut."""
    g = torch.Generator().manual_seed(tokens)
    lengths = torch.randint(0, 131, (170,), generator=g).tolist()
    counts = [min(length, int(torch.randint(0, tokens + 1, (1,), generator=g))) for length in lengths]
    cache, k, v = _filled(170, kv_heads, 130, head_dim, torch.float16, lengths)
    q = _draw((170, tokens, 8 * kv_heads, head_dim), torch.float16, 48)
    _check_attention(cache, k, v, q, lengths, counts)
    cache.check()


def test_offsets_that_pass_32_bits():
    """Eight heads of 2.2 million positions: codes of 2.25 GB each, of which the last two hundred positions are not zeros."""
    max_len, d, heads, some = 2_200_000, 128, 8, 203
    cache = QuantizedKVCache(1, heads, max_len, d)
    assert cache.memory.numel() > 1 << 32
    start = (max_len - some) // 32 * 32
    k, v = _draw((1, some, heads, d), torch.float16, 50), _draw((1, some, heads, d), torch.float16, 51, 100.0)
    cache.append(k, v, _words([start]))
    length = start + some
    for got, x in zip(cache.read(_words([length]), first=_words([start - 5]), tokens=some + 5), (k, v)):
        assert not got[:, :5].any() and torch.equal(got[:, 5:], _held(x, [some]))
    for count in (1, 70):
        # (scores of ten and more, so that the others do not vanish among two million of zero)
        q = 6.0 * k[:, some - count:some].repeat_interleave(2, 2)
        got = cache.attention(q, _words([length]), softmax_scale=0.02)
        kh, vh = oracle.held(k[0], some), oracle.held(v[0], some)
        for i in range(count):
            seen = some - count + i + 1
            score = torch.einsum("hd,thd->ht", q[0, i].double(), kh[:seen].repeat_interleave(2, 1)) * 0.02
            p = score.exp()
            p = p / (p.sum(-1, keepdim=True) + start)
            want = torch.einsum("ht,thd->hd", p, vh[:seen].repeat_interleave(2, 1))
            weight = torch.einsum("ht,thd->hd", p, vh[:seen].abs().repeat_interleave(2, 1))
            bound = oracle.attention_bound(want, weight, torch.float16, float(vh.abs().max()) * some)
            # (and FP32 sums of two million numbers: their own terms' roundings, at most a thousand to a run)
            assert ((got[0, i].double() - want).abs() <= bound + weight * 2.0 ** -14).all(), i
    cache.check()


# ------------------------------------------------------------------ as they are used together

@pytest.mark.parametrize("head_dim", [64, 128])
def test_programmatic_launches_change_nothing(head_dim, monkeypatch):
    """Each kernel started while the one in front ends: steps and chunks in a row, where every call reads what the last one wrote."""
    inv_freq = (10000.0 ** (-torch.arange(0, head_dim, 2).double() / head_dim)).float().cuda()
    chunks = [64, 1, 1, 40, 200, 1, 33, 1]
    rows = _draw((2, sum(chunks), 12, head_dim), torch.float16, 49)

    def run():
        cache = QuantizedKVCache(2, 2, 360, head_dim)
        lengths, outs, at = _words([0, 0]), [], 0
        for tokens in chunks:
            q, k, v = (part.clone() for part in rows[:, at:at + tokens].split([8, 2, 2], 2))
            apply_rotary(k, (lengths[:, None] + torch.arange(tokens, device="cuda")), inv_freq, out=k)
            q = cache.append(k, v, lengths, q=q, inv_freq=torch.zeros_like(inv_freq))
            lengths += tokens
            outs += [cache.attention(q, lengths), *cache.read(lengths)]
            at += tokens
        cache.check()
        return outs

    monkeypatch.delenv("W4A16_PDL", raising=False)
    want = run()
    monkeypatch.setenv("W4A16_PDL", "1")
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(), want))
    cache = QuantizedKVCache(2, 2, 360, head_dim)
    lengths = [_words([n, n]) for n in range(0, 351, 50)]
    parts = [part.contiguous() for part in rows[:, :350].split([8, 2, 2], 2)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):                       # seven chunks in a row, nothing between the launches
        outs = []
        for i in range(7):
            q, k, v = (part[:, 50 * i:50 * i + 50] for part in parts)
            outs.append(cache.attention(cache.append(k, v, lengths[i], q=q, inv_freq=inv_freq), lengths[i + 1]))
    graph.replay()
    first = [out.clone() for out in outs]
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(outs, first))
    monkeypatch.delenv("W4A16_PDL")
    plain = QuantizedKVCache(2, 2, 360, head_dim)
    for i in range(7):
        q, k, v = (part[:, 50 * i:50 * i + 50] for part in parts)
        assert torch.equal(plain.attention(plain.append(k, v, lengths[i], q=q, inv_freq=inv_freq), lengths[i + 1]), first[i])
    plain.check()
    cache.check()


def test_a_generation_in_a_captured_graph():
    """Steps of turning, writing and attending, captured once and replayed with the position in device memory, two such graphs by
    turns on one stream and the same calls made eagerly."""
    d, kv_heads, q_heads, steps, max_len = 64, 2, 8, 70, 400
    inv_freq = (10000.0 ** (-torch.arange(0, d, 2).double() / d)).float().cuda()
    prompt_k, prompt_v = (_draw((1, 250, kv_heads, d), torch.float16, s) for s in (40, 41))
    rows = _draw((steps, 1, 1, (q_heads + 2 * kv_heads) * d), torch.float16, 42)

    class Layer:
        def __init__(self):
            self.cache = QuantizedKVCache(1, kv_heads, max_len, d)
            self.cache.append(prompt_k, prompt_v, _words([0]))
            self.row, self.position = rows[0].clone(), _words([250])

        def step(self):
            q, k, v = (part.unflatten(-1, (-1, d)) for part in self.row.split([q_heads * d] + [kv_heads * d] * 2, -1))
            q = self.cache.append(k, v, self.position, q=q, inv_freq=inv_freq)
            self.position += 1
            return self.cache.attention(q, self.position)

    eager = Layer()
    want = []
    for t in range(steps):
        eager.row.copy_(rows[t])
        want.append(eager.step())
    layers, graphs, outs = [Layer(), Layer()], [], []
    for layer in layers:
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):                               # warm-up, taken back
            layer.step()
            layer.position -= 1
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer.step()
        graphs.append(graph)
        outs.append(out)
    for t in range(steps):
        for layer, graph, out in zip(layers, graphs, outs):
            layer.row.copy_(rows[t])
            graph.replay()
            assert torch.equal(out, want[t]), t
    assert all(torch.equal(layer.cache.memory, eager.cache.memory) for layer in layers)
    # and by the definition, at the end
    everything = torch.cat([rows[:, 0, 0]], 0)
    q, k, v = (part.unflatten(-1, (-1, d)) for part in everything.split([q_heads * d] + [kv_heads * d] * 2, -1))
    k = apply_rotary(k, torch.arange(250, 250 + steps, device="cuda"), inv_freq)
    q = apply_rotary(q, torch.arange(250, 250 + steps, device="cuda"), inv_freq)
    k, v = torch.cat((prompt_k[0], k)), torch.cat((prompt_v[0], v))
    length = 250 + steps
    kh, vh = oracle.held(k, length), oracle.held(v, length)
    exact, weight = oracle.attention(q[-1:], kh, vh, length, 1, d ** -0.5)
    assert ((want[-1][0].double() - exact).abs() <= oracle.attention_bound(exact, weight, torch.float16, float(vh.abs().max()) * length)).all()


def test_on_another_stream_than_the_first():
    cache, k, v = _filled(2, 2, 700, 128, torch.float16, [700, 433])
    q = _draw((2, 1, 16, 128), torch.float16, 43)
    want = cache.attention(q, _words([700, 433]))
    lengths = _words([700, 433])
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for stream in streams * 4:                                         # overlapping calls have workspaces of their own
        with torch.cuda.stream(stream):
            outs.append(cache.attention(q, lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs)


def test_refusals():
    cache = QuantizedKVCache(2, 2, 64, 64)
    k, q = _draw((2, 3, 2, 64), torch.float16, 44), _draw((2, 3, 8, 64), torch.float16, 45)
    at, inv_freq = _words([0, 0]), torch.ones((32,), device="cuda")
    bad = [
        lambda: cache.append(k.cpu(), k, at), lambda: cache.append(k.bfloat16(), k, at), lambda: cache.append(k[:1], k[:1], at),
        lambda: cache.append(k, k[:, :2], at), lambda: cache.append(k[..., ::2], k[..., ::2], at), lambda: cache.append(k, k, at.int()),
        lambda: cache.append(k, k, at[:1]), lambda: cache.append(k, k, at, at[:1]), lambda: cache.append(k, k, at, q=q),
        lambda: cache.append(k, k, at, inv_freq=torch.ones((33,), device="cuda")), lambda: cache.append(k, k, at.cpu()),
        lambda: cache.append(k, k, at, inv_freq=inv_freq.double()), lambda: cache.append(k.float(), k.float(), at),
        lambda: cache.append(k, k, at, q=q[:, :2], inv_freq=inv_freq), lambda: cache.append(k.requires_grad_(), k, at),
        lambda: cache.append(k.transpose(2, 3), k, at), lambda: cache.append(k[0], k[0], at),
        lambda: cache.read(at, tokens=-1), lambda: cache.read(at[:1]), lambda: cache.read(at, first=at.int()),
        lambda: cache.attention(q[:, :, :7], at), lambda: cache.attention(q[:1], at), lambda: cache.attention(q.bfloat16(), at),
        lambda: cache.attention(q[..., :32], at), lambda: cache.attention(q[:, :, :0], at), lambda: cache.attention(q, at.int()),
        lambda: cache.attention(q, at, counts=at.cpu()), lambda: cache.attention(q.clone().requires_grad_(), at),
        lambda: apply_rotary(q, at, inv_freq), lambda: apply_rotary(q, _words([[0] * 3] * 2), inv_freq.half()),
        lambda: apply_rotary(q, _words([[0] * 3] * 2), torch.ones((33,), device="cuda")),
        lambda: apply_rotary(q.float(), _words([[0] * 3] * 2), inv_freq), lambda: apply_rotary(q[..., :63], _words([[0] * 3] * 2), inv_freq[:8]),
        lambda: apply_rotary(q[:, :2], _words([[0] * 2] * 2), inv_freq, out=q[:, 1:]),
        lambda: apply_rotary(q[:1, :1].expand(2, 3, 8, 64), _words([[0] * 3] * 2), inv_freq, out=q[:1, :1].expand(2, 3, 8, 64)),
    ]
    for number, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {number} was not refused")
        k = k.detach()
    for arguments in ((0, 2, 64, 64), (2, 0, 64, 64), (2, 2, 0, 64), (2, 2, 64, 96), (1 << 20, 1 << 20, 64, 64)):
        with pytest.raises(ValueError):
            QuantizedKVCache(*arguments)
    with pytest.raises(ValueError):
        QuantizedKVCache(1, 1, 64, 64, dtype=torch.float32)
    with pytest.raises(ValueError):
        QuantizedKVCache(1, 1, 64, 64, device="cpu")
    torch.cuda.synchronize()
    cache.check()
    assert not cache.memory.any()
