"""-m gpu: what an 8-bit cache's status word says reaches whoever runs the steps."""
from __future__ import annotations

import pytest
import torch

from nibble_b200 import QuantizedKVCache
from test_gpu_decode_8bit import _model, _tokens

pytestmark = pytest.mark.gpu


def test_both_bits_of_the_word_are_reported():
    cache = QuantizedKVCache(1, 1, 64, 64)
    for word, what in ((1, "did not fit"), (2, "gave up"), (3, "gave up")):
        cache.memory[:4].view(torch.int32).fill_(word)
        with pytest.raises(RuntimeError, match=what):
            cache.check()
        cache.check()


@pytest.mark.parametrize(("word", "what"), [(1, "past the end"), (2, "gave up"), (3, "gave up")])
def test_a_prompt_in_chunks_reports_what_its_caches_do(word, what):
    """A word that one layer's attention left behind, as the kernel would: from ``prefill`` itself, not from a later ``generate``."""
    from nibble_b200.decode import LlamaDecodeRunner

    model = _model(7, num_hidden_layers=2)
    runner = LlamaDecodeRunner(model, max_len=96, cache_bits=8)
    prompt = _tokens(model, 40, 8)
    process = runner._prefill_8bit

    def with_a_word(ids):
        process(ids)
        runner.caches[1].memory[:4].view(torch.int32).fill_(word)

    runner._prefill_8bit = with_a_word
    with pytest.raises(RuntimeError, match=what):
        runner.prefill(prompt)
    runner._prefill_8bit = process
    runner.prefill(prompt)
    for cache in runner.caches:
        cache.check()
