"""-m gpu: the decode runner with its keys and values in 8 bits."""
from __future__ import annotations

import pytest
import torch

import kv_oracle

pytestmark = pytest.mark.gpu

transformers = pytest.importorskip("transformers")


def _model(seed, **overrides):
    from nibble_b200 import replace_linear_layers

    base = dict(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4,
                num_key_value_heads=2, max_position_embeddings=256, rms_norm_eps=1e-5, tie_word_embeddings=False)
    base.update(overrides)
    torch.manual_seed(seed)
    with torch.device("cuda"):
        model = transformers.AutoModelForCausalLM.from_config(transformers.LlamaConfig(**base), dtype=torch.float16)
    model.eval()
    replace_linear_layers(model, group_size=128)
    return model


def _tokens(model, count, seed):
    return torch.randint(0, model.config.vocab_size, (count,), generator=torch.Generator().manual_seed(seed)).cuda()


@torch.inference_mode()
def _logits(model, tokens):
    """What every step should give: the model's own layers, with the cache and the attention over it from their definitions.  A
    query sees the blocks that are full by then as codes and the rest as it came."""
    body, config = model.model, model.config
    heads, kv_heads = config.num_attention_heads, config.num_key_value_heads
    d = config.hidden_size // heads
    count = tokens.numel()
    places = torch.arange(count, device="cuda")
    inv_freq = body.rotary_emb.inv_freq.float()
    stream = body.embed_tokens(tokens)
    for block in body.layers:
        x, attn = block.input_layernorm(stream), block.self_attn
        q, k, v = attn.q_proj(x).view(count, heads, d), attn.k_proj(x).view(count, kv_heads, d), attn.v_proj(x).view(count, kv_heads, d)
        q, k = (kv_oracle.rotary(part, places, inv_freq, 1.0, False).half() for part in (q, k))
        rows = []
        for t in range(count):
            keys, values = kv_oracle.held(k[:t + 1].cpu(), t + 1).cuda(), kv_oracle.held(v[:t + 1].cpu(), t + 1).cuda()
            rows.append(kv_oracle.attention(q[t:t + 1], keys, values, t + 1, 1, d ** -0.5)[0])
        stream = stream + attn.o_proj(torch.cat(rows).half().view(count, -1))
        stream = stream + block.mlp(block.post_attention_layernorm(stream))
    return model.lm_head(body.norm(stream)).float()


@pytest.mark.parametrize(("fuse_inputs", "overrides"), [
    (True, {}), (False, {}), (True, dict(hidden_size=512, num_attention_heads=4, num_key_value_heads=1))])
def test_steps_follow_the_model(fuse_inputs, overrides):
    from nibble_b200.decode import LlamaDecodeRunner

    model = _model(0, **overrides)
    tokens = _tokens(model, 70, 2)
    want = _logits(model, tokens)
    runner = LlamaDecodeRunner(model, max_len=80, fuse_inputs=fuse_inputs, cache_bits=8)
    for t in range(tokens.numel()):
        runner.token.copy_(tokens[t:t + 1])
        runner.step()
        got = runner.logits[0].float()
        # (the bound of the 16-bit runner against the same forward: FP16 sums taken in another order, through three blocks)
        assert (got - want[t]).abs().max().item() < 2e-2 * want[t].abs().max().item(), t
        assert int(runner.position.item()) == t + 1 and int(runner.token.item()) == int(got.argmax().item())
    for cache in runner.caches:
        cache.check()
    assert runner.launches_per_step == (7 if fuse_inputs else 10) * 3 + (2 if fuse_inputs else 3)


@pytest.mark.parametrize(("count", "chunk"), [(70, 2048), (150, 64), (33, 32)])
def test_a_prompt_in_chunks_is_what_its_tokens_are_one_by_one(count, chunk):
    from nibble_b200.decode import LlamaDecodeRunner

    model = _model(5)
    prompt = _tokens(model, count, 6)
    runner = LlamaDecodeRunner(model, max_len=192, cache_bits=8)
    runner.prefill(prompt, batched=False)
    length = torch.tensor([count], device="cuda")
    stepped = [cache.read(length, tokens=count) for cache in runner.caches]
    runner.step()
    logits = runner.logits.float().clone()
    runner.PREFILL_CHUNK = chunk
    runner.prefill(prompt)
    assert int(runner.position.item()) == count
    for cache, (k, v) in zip(runner.caches, stepped):
        # FP16 sums in another order, as between the routes with a 16-bit cache, and a step of the codes where that tips one over
        step = 2 * torch.stack([k, v]).abs().max().item() / 127
        got = cache.read(length, tokens=count)
        torch.testing.assert_close(got[0], k, rtol=3e-2, atol=3e-2 + step)
        torch.testing.assert_close(got[1], v, rtol=3e-2, atol=3e-2 + step)
    runner.step()
    assert (runner.logits.float() - logits).abs().max().item() < 3e-2 * logits.abs().max().item()


def test_generate_is_repeatable_and_reports_a_full_cache():
    from nibble_b200.decode import LlamaDecodeRunner

    model = _model(1, num_hidden_layers=2)
    runner = LlamaDecodeRunner(model, max_len=75, cache_bits=8)
    for count in (4, 40):
        prompt = _tokens(model, count, count)
        first = runner.generate(prompt, 35)
        assert torch.equal(first, runner.generate(prompt, 35))
        # the graph was captured with another prompt in the caches: a new runner has seen nothing else
        assert torch.equal(first, LlamaDecodeRunner(model, max_len=75, cache_bits=8).generate(prompt, 35))
    with pytest.raises(ValueError):
        runner.generate(prompt, 36)
    runner.step()                                      # position 74, the last
    for cache in runner.caches:
        cache.check()
    runner.step()
    for cache in runner.caches:
        with pytest.raises(RuntimeError, match="did not fit"):
            cache.check()
    runner.step()
    runner.reset()
    assert torch.equal(first, runner.generate(prompt, 35))


def test_short_caches_and_refusals():
    from nibble_b200.decode import LlamaDecodeRunner

    model = _model(3, num_hidden_layers=2)
    prompt = _tokens(model, 3, 1)
    short = LlamaDecodeRunner(model, max_len=8, cache_bits=8).generate(prompt, 5)          # no block gets full: 16 bits throughout
    assert torch.equal(short[:1], LlamaDecodeRunner(model, max_len=8).generate(prompt, 1))
    with pytest.raises(ValueError):
        LlamaDecodeRunner(model, max_len=8, cache_bits=8, persistent=True)
    with pytest.raises(ValueError):
        LlamaDecodeRunner(model, max_len=8, cache_bits=4)
