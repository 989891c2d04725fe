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


def _block_tops(v, length):
    """The largest magnitude of each token's block (of its own, where the block is being filled): [length, heads]."""
    tops = v[:length].double().abs().amax(-1)
    full = length // 32 * 32
    tops[:full] = tops[:full].view(full // 32, 32, v.shape[1]).amax(1, keepdim=True).expand(-1, 32, -1).reshape(full, v.shape[1])
    return tops


def _check_seen(cache, k, v, q, length, scale):
    """Attention against its definition, within what the tokens that a query sees allow: a weight (probability times its values' scale)
    is held in FP16 times 2^9 (or 2^10) relative to the largest one seen, M / 127 at most with M the largest p x (largest of the token's
    block).  What is below FP16's normal numbers is off by half a step, 2^-25: times a code of 127 at most that is 2^-34 of M for each
    token; times a number of the block being filled, held up to 2^10, 2^-25 x 2^-9 x 2^10 / 127 < 2^-30 of it, 31 of them 2^-25; and such a number
    itself is off by 2^-34 of the block's largest, or (BF16, where those lie further apart it is taken as it is) by 2^-17 of its eight's
    largest at most, times its probability.  A sum of rounded
    weights is off by 2^-30 of itself for each of them at most (their scale is 2^-4 of the largest's or more).  The rest is
    kv_oracle.attention_bound's."""
    got = cache.attention(q, _words([length]), softmax_scale=scale)[0].double()
    tokens, q_heads, _ = q.shape[1:]
    group = q_heads // v.shape[2]
    kb, vb = oracle.held(k[0], length)[:length], oracle.held(v[0], length)[:length]
    want, weight = oracle.attention(q[0], kb, vb, length, tokens, scale)
    tops = _block_tops(v[0], length)
    hidden = torch.arange(length, device="cuda")[None, :] > (length - tokens + torch.arange(tokens, device="cuda"))[:, None]
    for head in range(v.shape[2]):
        rows = slice(head * group, (head + 1) * group)
        scores = torch.einsum("ihd,td->iht", q[0, :, rows].double(), kb[:, head]) * scale
        p = torch.softmax(scores.masked_fill(hidden[:, None, :], float("-inf")), -1)
        most = (p * tops[:, head]).amax(-1, keepdim=True)
        bound = oracle.attention_bound(want[:, rows], weight[:, rows], q.dtype, 0.0)
        bound = bound + most * (length * 2.0 ** -34 + 2.0 ** -25) + want[:, rows].abs() * length * 2.0 ** -30
        full = length // 32 * 32
        if full < length:
            tails = v[0, full:length, head].double().abs()
            if q.dtype == torch.float16:
                bound = bound + p[..., full:].sum(-1, keepdim=True) * float(tails.max()) * 2.0 ** -34
            else:
                bound = bound + (p[..., full:] @ tails.unflatten(-1, (-1, 8)).amax(-1).repeat_interleave(8, -1)) * 2.0 ** -17
        off = (got[:, rows] - want[:, rows]).abs()
        assert (off <= bound).all(), (head, float((off / bound).max()))
    cache.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("tokens", "q_heads", "kv_heads"), [(1, 8, 2), (5, 8, 2), (3, 32, 2), (90, 8, 2), (300, 64, 1)])
@pytest.mark.parametrize("where", ["unseen", "unseen in a full block", "unlikely", "unlikely and near"])
def test_values_far_out_do_not_cost_others_their_bits(where, tokens, q_heads, kv_heads, dtype):
    """Half of a row's result comes of thousands of small probabilities of small values, beside a value that is millions of times as large:
    behind the queries, or of a token that counts for nothing."""
    length = 8032 if where == "unseen in a full block" else 8017
    large = 60000.0 if dtype == torch.float16 else 1e6
    k = torch.zeros((1, length, kv_heads, 64), dtype=dtype, device="cuda")
    heavy = length - 5 if where == "unlikely and near" and tokens == 1 else 5
    k[:, heavy] = 1.0
    v = (0.01 * (1.0 + 0.2 * _draw((1, length, kv_heads, 64), torch.float32, 16).clamp(-2, 2))).to(dtype)
    if where.startswith("unseen"):
        v[:, length - 1, :, ::2] = large
    else:
        at = length - 9 if where == "unlikely and near" else 40
        k[:, at] = -60.0 / 9
        v[:, at, :, ::2] = large
    cache = QuantizedKVCache(1, kv_heads, length + 7, 64, dtype=dtype)
    cache.append(k, v, _words([0]))
    q = torch.full((1, tokens, q_heads, 64), 9.0 / 64, dtype=dtype, device="cuda")        # scores of nine, of zero, of -60
    _check_seen(cache, k, v, q, length, 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("tokens", "q_heads", "head_dim"), [(1, 8, 64), (6, 8, 128), (40, 8, 64), (400, 8, 128)])
def test_blocks_of_values_of_every_size(tokens, q_heads, head_dim, dtype):
    """Sizes that go up and down by thousands from block to block, some zero, with scores that do the same: the reference of the weights
    moves in either way, and pieces of a row meet with different ones."""
    length = 1500
    g = torch.Generator().manual_seed(17)
    low, high = (-16, 13) if dtype == torch.float16 else (-60, 90)
    sizes = 2.0 ** torch.randint(low, high, (47,), generator=g).double() * (torch.rand((47,), generator=g) > 0.1)
    sizes = sizes.cuda().repeat_interleave(32)[:length, None, None]
    k = _draw((1, length, 1, head_dim), dtype, 18)
    v = (_draw((1, length, 1, head_dim), torch.float32, 19).double() * sizes)[...].to(dtype)
    cache = QuantizedKVCache(1, 1, length + 9, head_dim, dtype=dtype)
    cache.append(k, v, _words([0]))
    for spread in (0.3, 2.0, 6.0):
        _check_seen(cache, k, v, _draw((1, tokens, q_heads, head_dim), dtype, 20, spread), length, head_dim ** -0.5)


@pytest.mark.parametrize("length", [20, 90, 3000])
@pytest.mark.parametrize(("tokens", "q_heads", "head_dim"), [(1, 8, 64), (6, 8, 128), (20, 16, 64), (300, 8, 128)])
def test_means_of_the_largest_values(tokens, q_heads, head_dim, length):
    """BF16 values as large as they come: their sums are beyond FP32, their means are not."""
    top = torch.finfo(torch.bfloat16).max
    k = _draw((1, length, 1, head_dim), torch.bfloat16, 21, 0.1)
    sign = torch.where(torch.arange(head_dim, device="cuda") % 3 == 0, -1.0, 1.0)
    v = (top * sign).to(torch.bfloat16).expand(1, length, 1, head_dim)
    cache = QuantizedKVCache(1, 1, length + 3, head_dim, dtype=torch.bfloat16)
    cache.append(k, v, _words([0]))
    got = cache.attention(_draw((1, tokens, q_heads, head_dim), torch.bfloat16, 22), _words([length]))
    first = max(0, tokens - length)
    # (a sum of rounded numbers over one of others: 2^-8 of the mean for all of them, which is a step of BF16 at most)
    assert got.isfinite().all() and not got[0, :first].any()
    assert ((got[0, first:].double() / (top * sign) - 1.0).abs() <= 2.0 ** -7).all()
    cache.check()


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize(("dtype", "head_dim"), [(torch.float16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("pieces", [[64], [20, 44], [20, 12, 32], [1] * 64, [96], [40, 56], [5, 91], [96 - 31, 31], [32], [31, 1], [128], [50, 78],
                                    [33], [70], [20, 57]])
def test_a_length_falls_to_the_block_before_the_last_tokens(pieces, dtype, head_dim, turned):
    """Whatever the last append ended on, and however the tokens came: read, attended over, and written on from there."""
    reached = sum(pieces)
    k, v, other = (_draw((2, 176, 2, head_dim), dtype, seed) for seed in (23, 24, 25))
    q = _draw((2, 1, 4, head_dim), dtype, 26)
    inv_freq = torch.zeros((head_dim // 2,), device="cuda") if turned else None           # (by no angle at all)

    def fill(cache):
        at = 0
        for piece in pieces:
            cache.append(k[:, at:at + piece], v[:, at:at + piece], _words([at, at]), inv_freq=inv_freq)
            at += piece
        return cache

    low = ((reached - 1) // 32 - 1) * 32
    for back in sorted({max(0, low), max(0, low) + 1, max(0, low) + 20, max(0, low) + 31, max(1, low + 32), reached}):
        if back > reached:
            continue
        cache = fill(QuantizedKVCache(2, 2, 176, head_dim, dtype=dtype))
        for got, x in zip(cache.read(_words([back, back])), (k, v)):
            assert torch.equal(got, _held(x, [back, back])), back
        fresh = QuantizedKVCache(2, 2, 176, head_dim, dtype=dtype)
        fresh.append(k[:, :back], v[:, :back], _words([0, 0]))
        assert torch.equal(cache.attention(q, _words([back, back])), fresh.attention(q, _words([back, back])))
        for piece in (7, 40):
            cache = fill(QuantizedKVCache(2, 2, 176, head_dim, dtype=dtype))
            cache.append(other[:, :piece], other[:, :piece], _words([back, back]), inv_freq=inv_freq)
            mixed = torch.cat((v[:, :back], other[:, :piece], v[:, back + piece:]), 1)
            assert torch.equal(cache.read(_words([back + piece] * 2))[1], _held(mixed, [back + piece] * 2)), (back, piece)
        cache.check()


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_tangents_are_refused():
    """Forward-mode differentiation and transformed tensors: no result that has lost them."""
    cache = QuantizedKVCache(1, 2, 64, 64)
    x, at, inv_freq = _draw((1, 3, 2, 64), torch.float16, 27), _words([0]), torch.ones((32,), device="cuda")
    places = _words([[0, 1, 2]])
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: apply_rotary(dual, places, inv_freq), lambda: apply_rotary(x, places, inv_freq, out=dual),
                     lambda: apply_rotary(x, places, torch.autograd.forward_ad.make_dual(inv_freq, inv_freq)),
                     lambda: cache.append(dual, x, at), lambda: cache.append(x, dual[:, :, :], at),
                     lambda: cache.append(x, x, at, q=dual, inv_freq=inv_freq), lambda: cache.attention(dual, at)):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
        with torch.autograd.forward_ad._set_fwd_grad_enabled(False):
            assert torch.equal(apply_rotary(dual, places, inv_freq), apply_rotary(x, places, inv_freq))
        assert torch.equal(cache.attention(torch.autograd.forward_ad.unpack_dual(dual).primal, at), torch.zeros_like(x))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: apply_rotary(t, places, inv_freq), (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: apply_rotary(t, places, inv_freq))(x[None])
    torch.cuda.synchronize()
    cache.check()
    assert not cache.memory.any()


def test_turning_in_place_counts_as_a_change():
    """A tensor saved for a backward pass, and the fused layers' memory of their last input."""
    from nibble_b200 import QuantizedLinear, fuse_parallel_linears

    x, places, inv_freq = _draw((3, 4, 64), torch.float16, 28), _words([5, 6, 7]), torch.ones((32,), device="cuda")
    weight = _draw((64, 64), torch.float16, 29).requires_grad_()
    out = x @ weight
    before = x._version
    with torch.no_grad():
        apply_rotary(x, places, inv_freq, out=x)
    assert x._version > before
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()
    into = torch.empty_like(x)
    kept = (x._version, into._version)
    apply_rotary(x, places, inv_freq, out=into)
    assert x._version == kept[0] and into._version > kept[1]
    with torch.inference_mode():
        plain = x.clone()
        assert torch.equal(apply_rotary(plain, places, inv_freq, out=plain), into)
        apply_rotary(x, places, inv_freq, out=into)

    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            for seed, name in enumerate(("q_proj", "k_proj", "v_proj")):
                linear = torch.nn.Linear(256, 128, bias=False)
                linear.weight.data = _draw((128, 256), torch.float32, 30 + seed, 0.02).cpu()
                setattr(self, name, QuantizedLinear.from_float(linear, group_size=128).cuda())

    block = Block()
    fuse_parallel_linears(block)
    rows = _draw((3, 256), torch.float16, 33)
    block.q_proj(rows)
    apply_rotary(rows.view(3, 4, 64), places, inv_freq, out=rows.view(3, 4, 64))
    got = block.k_proj(rows)
    block.q_proj(torch.zeros_like(rows))
    assert torch.equal(got, block.k_proj(rows.clone()))


def test_turned_into_another_place():
    """``out`` beside ``x``: memory of its own, rows with gaps, another part of the same rows; and what overlaps is refused."""
    d, inv_freq = 64, (10000.0 ** (-torch.arange(0, 64, 2).double() / 64)).float().cuda()
    places = _words([[4, 5, 6], [90, 91, 92]])
    row = _draw((2, 3, 20 * d), torch.float16, 34)
    q, k = row[..., :6 * d].unflatten(-1, (6, d)), row[..., 6 * d:12 * d].unflatten(-1, (6, d))
    want = apply_rotary(q.contiguous(), places, inv_freq)
    apart = torch.zeros((2, 3, 6, d), dtype=torch.float16, device="cuda")
    assert apply_rotary(q, places, inv_freq, out=apart) is apart and torch.equal(apart, want)
    slot = torch.zeros((2, 3, 9, d + 8), dtype=torch.float16, device="cuda")
    apply_rotary(q, places, inv_freq, out=slot[:, :, 2:8, :d])
    assert torch.equal(slot[:, :, 2:8, :d], want) and not slot[:, :, :2].any() and not slot[:, :, 8:].any() and not slot[..., d:].any()
    by_head = torch.zeros((2, 6, 3, d), dtype=torch.float16, device="cuda").transpose(1, 2)
    assert torch.equal(apply_rotary(q, places, inv_freq, out=by_head), want)
    kept = row.clone()
    apply_rotary(q, places, inv_freq, out=k)                                       # the same rows, the part behind
    assert torch.equal(k, want) and torch.equal(row[..., :6 * d], kept[..., :6 * d]) and torch.equal(row[..., 12 * d:], kept[..., 12 * d:])
    apply_rotary(q[:, :1], places[:, :1].contiguous(), inv_freq, out=q[:, 1:2])     # the next token's row
    assert torch.equal(q[:, 1:2], want[:, :1])
    one = row[0, 0].view(20, d)
    kept = one.clone()
    apply_rotary(one[0:16:2], _words(7), inv_freq, out=one[1:17:2])                # every other head into its neighbour
    assert torch.equal(one[0:16:2], kept[0:16:2]) and torch.equal(one[17:], kept[17:])
    assert torch.equal(one[1:17:2], apply_rotary(kept[0:16:2], _words(7), inv_freq))
    single = _draw((1, 2, 6 * d), torch.float16, 54)                               # dimensions with one entry, whose strides say nothing
    spaced = single.as_strided((1, 2, 3, d), (999, 6 * d, d, 1))
    want = apply_rotary(spaced.contiguous(), places[:1, :2].contiguous(), inv_freq)
    apply_rotary(spaced, places[:1, :2].contiguous(), inv_freq, out=single.as_strided((1, 2, 3, d), (7, 6 * d, d, 1), 3 * d))
    assert torch.equal(single[..., 3 * d:].unflatten(-1, (3, d)), want)
    apply_rotary(spaced, places[:1, :2].contiguous(), inv_freq, out=single.as_strided((1, 2, 3, d), (7, 6 * d, d, 1)))
    assert torch.equal(spaced, want)
    kept = row.clone()
    for into in (row[..., d:7 * d].unflatten(-1, (6, d)), row[..., 1:6 * d + 1].unflatten(-1, (6, d)), row[..., 5 * d:11 * d].unflatten(-1, (6, d)),
                 row[..., :12 * d].unflatten(-1, (6, 2 * d))[..., :d], row.view(-1).as_strided((2, 3, 6, d), (3 * 20 * d, 20 * d, d, 1), 8),
                 q.float(), q.bfloat16(), q[:, :, :5], q.cpu()):
        with pytest.raises(RuntimeError):
            apply_rotary(q, places, inv_freq, out=into)
    with pytest.raises(RuntimeError):
        apply_rotary(q[:, :2], places[:, :2].contiguous(), inv_freq, out=q[:, 1:])
    torch.cuda.synchronize()
    assert torch.equal(row, kept)


@pytest.mark.parametrize("length", [40, 64, 70])
def test_reading_from_a_place_beyond_the_cache(length):
    """Zeros, and reported, as for a length or start that does not fit; up to the cache's end there is nothing to report."""
    x = _draw((3, 70, 1, 64), torch.float16, 35)
    cache = QuantizedKVCache(3, 1, 70, 64)
    cache.append(x, x, _words([0, 0, 0]))
    lengths = _words([length] * 3)
    got, _ = cache.read(lengths, first=_words([70, length, 0]), tokens=40)
    assert not got[:2].any() and torch.equal(got[2], _held(x, [length] * 3)[2, :40])
    cache.check()
    for first in (71, 1 << 33, (1 << 63) - 1, (1 << 63) - 40, -1, -(1 << 63)):
        for part in cache.read(lengths, first=_words([first, 0, first]), tokens=40):
            assert not part[0].any() and not part[2].any() and torch.equal(part[1], _held(x, [length] * 3)[1, :40]), first
        with pytest.raises(RuntimeError, match="did not fit"):
            cache.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("tokens", "q_heads", "kv_heads", "head_dim", "length", "spread"), [
    (1, 64, 8, 64, 900, 1.0), (5, 32, 8, 128, 2000, 2.0), (64, 16, 4, 64, 1000, 1.0), (150, 16, 2, 128, 3000, 1.0), (150, 16, 2, 128, 700, 3.0),
    (600, 8, 1, 64, 600, 0.3)])
def test_errors_are_of_the_size_of_their_roundings(tokens, q_heads, kv_heads, head_dim, length, spread, dtype):
    """The root of the mean square of what results are off by, against that of the roundings they are made with: the result's own, evenly
    spread over a step (step^2 / 12), and a weight's to FP16, evenly spread over 2^-11 of it to either side at most (a third of that
    squared).  Few FP16 rows: the result's alone.  Where the sum is of the rounded weights (many FP16 rows) an error of p_t moves the result by
    p_t e_t (v_t - out), elsewhere by p_t e_t v_t.  1.03 for what is not in the sum: FP32's roundings, some 2^-18 of p, and the sample."""
    k, v = _draw((1, length, kv_heads, head_dim), dtype, 36), _draw((1, length, kv_heads, head_dim), dtype, 37)
    cache = QuantizedKVCache(1, kv_heads, length, head_dim, dtype=dtype)
    cache.append(k, v, _words([0]))
    q = _draw((1, tokens, q_heads, head_dim), dtype, 38, spread)
    got = cache.attention(q, _words([length]))[0].double()
    group, few = q_heads // kv_heads, tokens * q_heads // kv_heads <= 32
    kb, vb = oracle.held(k[0], length), oracle.held(v[0], length)
    hidden = torch.arange(length, device="cuda")[None, :] > (length - tokens + torch.arange(tokens, device="cuda"))[:, None]
    off = allowed = 0.0
    for head in range(kv_heads):
        rows = slice(head * group, (head + 1) * group)
        scores = torch.einsum("ihd,td->iht", q[0, :, rows].double(), kb[:, head]) * head_dim ** -0.5
        p = torch.softmax(scores.masked_fill(hidden[:, None, :], float("-inf")), -1)
        values = vb[:, head]
        out = p @ values
        off += float((got[:, rows] - out).square().sum())
        step = torch.finfo(dtype).eps * 2.0 ** out.abs().clamp_min(2.0 ** -14).log2().floor()
        allowed += float(step.square().sum()) / 12
        if few and dtype == torch.float16:
            continue
        moved = p.square() @ values.square()
        if dtype == torch.float16:
            moved = moved - 2 * out * (p.square() @ values) + out.square() * p.square().sum(-1, keepdim=True)
        allowed += float(moved.sum()) * 2.0 ** -22 / 3
    assert off ** 0.5 <= 1.03 * allowed ** 0.5, (off / allowed) ** 0.5


@pytest.mark.parametrize(("tokens", "q_heads", "kv_heads", "head_dim", "length"), [
    (1, 32, 4, 64, 500), (1, 8, 1, 128, 3001), (5, 16, 2, 64, 999), (90, 8, 2, 64, 1500), (200, 16, 2, 128, 700)])
@pytest.mark.parametrize("spread", [1.0, 3.0])
def test_bf16_sums_are_of_weights_that_are_not_rounded(tokens, q_heads, kv_heads, head_dim, length, spread):
    """So that of the bound on a kernel's error the part for a rounded sum, 2^-11 of the result, falls away."""
    k, v = _draw((1, length, kv_heads, head_dim), torch.bfloat16, 39), _draw((1, length, kv_heads, head_dim), torch.bfloat16, 40)
    cache = QuantizedKVCache(1, kv_heads, length, head_dim, dtype=torch.bfloat16)
    cache.append(k, v, _words([0]))
    q = _draw((1, tokens, q_heads, head_dim), torch.bfloat16, 41, spread)
    got = cache.attention(q, _words([length]))[0].double()
    kb, vb = oracle.held(k[0], length), oracle.held(v[0], length)
    want, weight = oracle.attention(q[0], kb, vb, length, tokens, head_dim ** -0.5)
    bound = oracle.attention_bound(want, weight, torch.bfloat16, float(vb.abs().max()) * length) - want.abs() * 2.0 ** -11
    assert ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("tokens", "q_heads", "kv_heads", "head_dim"), [(1, 8, 2, 64), (5, 8, 1, 128), (12, 8, 2, 64), (90, 8, 2, 64), (300, 16, 1, 128)])
def test_a_cache_far_larger_than_what_it_holds(tokens, q_heads, kv_heads, head_dim, dtype):
    """Runs and pieces are cut for the longest sequence that a cache takes; short and long ones in one of 50000 tokens, and in one that is
    full."""
    lengths = [tokens, 500, 33, 40, 1203]
    k, v = _draw((5, 1203, kv_heads, head_dim), dtype, 42), _draw((5, 1203, kv_heads, head_dim), dtype, 43)
    q = _draw((5, tokens, q_heads, head_dim), dtype, 44)
    for max_len in (1203, 50000):
        cache = QuantizedKVCache(5, kv_heads, max_len, head_dim, dtype=dtype)
        cache.append(k, v, _words([0] * 5), _words(lengths))
        first = _check_attention(cache, k, v, q, lengths, None)
        for _ in range(3):
            assert torch.equal(cache.attention(q, _words(lengths)), first)
        cache.check()


@pytest.mark.parametrize("length", [50, 90, 95, 33])
@pytest.mark.parametrize(("tokens", "q_heads", "kv_heads", "head_dim"), [(1, 8, 2, 64), (5, 8, 2, 128), (24, 32, 2, 64), (24, 32, 2, 128)])
@pytest.mark.parametrize("dims", [slice(None), slice(8, 24)])
@pytest.mark.parametrize(("k_size", "v_size"), [(1.0, 1e12), (1.0, 3e38), (1e30, 1.0), (1e20, 1e38), (1e-30, 1e-30), (1.0, 1e4)])
def test_tokens_far_out_in_the_block_being_filled(k_size, v_size, dims, tokens, q_heads, kv_heads, head_dim, length):
    """BF16, a token some or all of whose key or value is as large (or small) as the type has them, the last but two: in front of it nothing changes, and for
    those that see it it counts as the definition says."""
    k, v = (_draw((1, length, kv_heads, head_dim), torch.bfloat16, seed) for seed in (45, 46))
    top = torch.finfo(torch.bfloat16).max
    for x, size in ((k, k_size), (v, v_size)):
        x[:, length - 3, :, dims] = (x[:, length - 3, :, dims].float() * size).clamp(-top, top).to(torch.bfloat16)
    cache = QuantizedKVCache(1, kv_heads, length + 3, head_dim, dtype=torch.bfloat16)
    cache.append(k, v, _words([0]))
    _check_seen(cache, k, v, _draw((1, tokens, q_heads, head_dim), torch.bfloat16, 47), length, head_dim ** -0.5)


def test_what_later_tokens_are_does_not_matter_to_a_chunk():
    """The same result, to a rounding, for queries in front of them, BF16, whatever the keys and values behind are."""
    for head_dim, length in ((64, 60), (128, 91)):
        k, v = (_draw((1, length, 2, head_dim), torch.bfloat16, seed) for seed in (48, 49))
        q = _draw((1, 24, 32, head_dim), torch.bfloat16, 50)
        outs = []
        for size in (1.0, 0.0, 1e6, -1e30, 3e38):
            dirty_k, dirty_v = k.clone(), v.clone()
            for x in (dirty_k, dirty_v):
                x[:, length - 2:] = size
            cache = QuantizedKVCache(1, 2, length, head_dim, dtype=torch.bfloat16)
            cache.append(dirty_k, dirty_v, _words([0]))
            got = cache.attention(q, _words([length]))
            assert got[:, :22].isfinite().all()
            outs.append(got[:, :22])
        for out in outs[1:]:
            # (powers of two alone differ; exponents that they are added to are rounded in FP32, 2^-20 of a weight, and then to FP16)
            assert ((out.double() - outs[0].double()).abs() <= 2.0 ** -7 * outs[0].double().abs() + 2.0 ** -9).all()


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("scale", [0.125, -0.125, 0.0])
@pytest.mark.parametrize("large", [60000.0, 300.0, 1.0])
def test_small_values_beside_large_ones_in_the_block_being_filled(large, scale, strided):
    """FP16, values 2^14 apart and more, seen and not, by many queries, in whole units and in pieces of one, of either sign of the scale."""
    for length, tokens, q_heads in ((60, 24, 16), (4000 + 31, 24, 16), (1000 + 15, 150, 16)):
        k, v = _draw((1, length, 1, 64), torch.float16, 51), _draw((1, length, 1, 64), torch.float16, 52, 0.002)
        v[:, length - 9] *= large / 0.002 / 4
        v[:, length - 2, :, 8:16] *= large / 0.002 / 4
        cache = QuantizedKVCache(1, 1, length + 40, 64)
        cache.append(k, v, _words([0]))
        q = _draw((1, tokens, q_heads, 64 + strided), torch.float16, 53)[..., :64]
        _check_seen(cache, k, v, q, length, scale)
