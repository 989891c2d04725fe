"""The 8-bit cache's C entry points refuse what they cannot take before anything is launched, and lay a cache out as its
description says (no GPU needed)."""
from __future__ import annotations

import ctypes

import pytest

from nibble_b200 import _native

SOME = 256           # an address that is never used


def _cache(**changed):
    lib = _native.core()
    cache = _native.KV8Cache()
    need = lib.w4a16_kv8_cache_bytes(2, 4, 100, 128)
    assert lib.w4a16_kv8_cache_describe(SOME, need, 2, 4, 100, 128, 0, ctypes.byref(cache)) == 0
    for name, value in changed.items():
        setattr(cache, name, value)
    return cache


def test_layout_of_a_cache():
    lib = _native.core()
    for batch, heads, length, d in ((1, 1, 1, 64), (2, 4, 100, 128), (3, 8, 32, 64), (1, 2, 31, 128)):
        need = lib.w4a16_kv8_cache_bytes(batch, heads, length, d)
        cache = _native.KV8Cache()
        assert lib.w4a16_kv8_cache_describe(SOME, need, batch, heads, length, d, 1, ctypes.byref(cache)) == 0
        pairs, blocks = batch * heads, length // 32
        sizes = {"status": 4, "k_tail": pairs * 64 * d * 2, "v_tail": pairs * 64 * d * 2, "k_scales": pairs * blocks * 4,
                 "v_scales": pairs * blocks * 4, "k_codes": pairs * blocks * 32 * d, "v_codes": pairs * blocks * 32 * d}
        spans = sorted((getattr(cache, name), getattr(cache, name) + size) for name, size in sizes.items() if size > 0)
        assert spans[0][0] >= SOME and spans[-1][1] <= SOME + need
        assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:])) and all(begin % 256 == 0 for begin, _ in spans)
        assert (cache.batch, cache.kv_heads, cache.max_len, cache.head_dim, cache.type) == (batch, heads, length, d, 1)
    # 8 bits: little more than half of an FP16 cache
    assert lib.w4a16_kv8_cache_bytes(1, 8, 32768, 128) < 0.51 * (1 * 8 * 32768 * 128 * 2 * 2)
    for sizes in ((0, 1, 1, 64), (1, 0, 1, 64), (1, 1, 0, 64), (1, 1, 1, 96), (-1, 1, 1, 64), (1 << 32, 1, 1, 64), (1, 1, 1 << 31, 64),
                  (1 << 16, 1 << 15, 64, 64), (1 << 62, 1 << 62, 64, 64)):
        assert lib.w4a16_kv8_cache_bytes(*sizes) == 0
    cache, need = _native.KV8Cache(), lib.w4a16_kv8_cache_bytes(1, 1, 64, 64)
    describe = lib.w4a16_kv8_cache_describe
    assert describe(None, need, 1, 1, 64, 64, 0, ctypes.byref(cache)) == -1
    assert describe(SOME, need, 1, 1, 64, 64, 0, None) == -1
    assert describe(SOME, need - 1, 1, 1, 64, 64, 0, ctypes.byref(cache)) == -5
    assert describe(SOME + 16, need, 1, 1, 64, 64, 0, ctypes.byref(cache)) == -4
    assert describe(SOME, need, 1, 1, 64, 64, 2, ctypes.byref(cache)) == -6


def test_refusals_before_any_launch():
    lib = _native.core()
    before = lib.w4a16_launch_count()
    rows, odd = _native.Rows(SOME, 64, 64, 64), _native.Rows(SOME + 1, 64, 64, 64)
    spec = _native.RotarySpec(SOME, 64, 0, 1.0)
    ref = ctypes.byref
    cache = _cache()

    def append(cache=cache, k=rows, v=rows, tokens=1, start=SOME, rotary=None, q=None, q_out=None, q_heads=8):
        return lib.w4a16_kv8_append(ref(cache), ref(k), ref(v), tokens, start, None, None if rotary is None else ref(rotary),
                                    None if q is None else ref(q), None if q_out is None else ref(q_out), q_heads, 0, None)

    assert append(tokens=-1) == -2 and append(tokens=0) == 0
    assert append(k=_native.Rows()) == -1 and append(v=odd) == -4 and append(start=None) == -1
    assert append(cache=_cache(head_dim=80)) == -2 and append(cache=_cache(batch=0)) == -2 and append(cache=_cache(type=7)) == -6
    assert append(cache=_cache(k_codes=0)) == -1 and append(cache=_cache(v_tail=SOME + 8)) == -4
    assert append(q=rows, q_out=rows) == -6                                  # queries without rotary positions
    assert append(rotary=_native.RotarySpec(SOME, 63, 0, 1.0)) == -2 and append(rotary=_native.RotarySpec(SOME, 130, 0, 1.0)) == -2
    assert append(rotary=_native.RotarySpec(0, 64, 0, 1.0)) == -1 and append(rotary=spec, q=rows) == -1
    assert append(rotary=spec, q=rows, q_out=_native.Rows(SOME, 64, 128, 64)) == -6
    assert append(rotary=spec, q=rows, q_out=rows, q_heads=0) == -2

    def read(cache=cache, lengths=SOME, tokens=1, k_out=SOME, v_out=SOME):
        return lib.w4a16_kv8_read(ref(cache), lengths, None, tokens, k_out, v_out, 0, None)

    assert read(tokens=-1) == -2 and read(tokens=0) == 0 and read(lengths=None) == -1 and read(k_out=None) == -1
    assert read(v_out=SOME + 8) == -4 and read(cache=_cache(kv_heads=-1)) == -2

    def attention(cache=cache, q=rows, out=SOME, q_heads=8, tokens=1, lengths=SOME, workspace=SOME, size=1 << 40):
        return lib.w4a16_kv8_attention(ref(cache), ref(q), out, q_heads, tokens, lengths, None, 1.0, workspace, size, 0, None)

    assert attention(q_heads=6) == -2 and attention(q_heads=0) == -2 and attention(tokens=-1) == -2 and attention(tokens=0) == 0
    assert attention(tokens=1 << 40) == -2 and attention(q=odd) == -4 and attention(out=None) == -1 and attention(lengths=None) == -1
    assert attention(out=SOME + 8) == -4 and attention(workspace=SOME + 4) == -4 and attention(cache=_cache(status=0)) == -1

    def rotary(spec=spec, x=rows, out=rows, batch=1, tokens=1, heads=1, head_dim=64, positions=SOME, type_=0):
        return lib.w4a16_rotary(ref(spec), ref(x), ref(out), batch, tokens, heads, head_dim, positions, type_, 0, None)

    assert rotary(head_dim=63) == -2 and rotary(head_dim=258) == -2 and rotary(batch=-1) == -2 and rotary(head_dim=62) == -2
    assert rotary(positions=None) == -1 and rotary(type_=3) == -6 and rotary(x=odd) == -4
    assert rotary(out=_native.Rows(SOME, 64, 64, 128)) == -6 and rotary(tokens=0) == 0 and rotary(heads=0) == 0
    assert lib.w4a16_launch_count() == before


def test_workspace_query():
    lib = _native.core()
    need = lambda cache, heads, tokens: lib.w4a16_kv8_attention_workspace_bytes(ctypes.byref(cache), heads, tokens)  # noqa: E731
    assert need(_cache(max_len=31), 8, 1) == 0                  # no block can be full: nothing is shared
    long = _cache(max_len=32768)
    assert need(long, 64, 1) > 0 and need(long, 64, 8) >= need(long, 64, 1)
    assert need(long, 63, 1) == need(long, 64, 0) == need(long, 64, -1) == need(_cache(head_dim=1), 8, 1) == 0


def test_python_layer_without_a_gpu():
    import torch

    from nibble_b200 import QuantizedKVCache, apply_rotary

    with pytest.raises(ValueError):
        QuantizedKVCache(1, 1, 64, 64, device="cpu")
    with pytest.raises(ValueError):
        QuantizedKVCache(1, 1, 64, 80)
    with pytest.raises(RuntimeError):
        apply_rotary(torch.zeros((1, 1, 64), dtype=torch.float16), torch.zeros((1,), dtype=torch.long), torch.ones(32))
