"""-m gpu: what an 8-bit cache's status word says reaches whoever runs the steps."""
from __future__ import annotations

import pytest
import torch

from nibble_b200 import QuantizedKVCache

pytestmark = pytest.mark.gpu


def test_both_bits_of_the_word_are_reported():
    cache = QuantizedKVCache(1, 1, 64, 64)
    for word, what in ((1, "did not fit"), (2, "gave up"), (3, "gave up")):
        cache.memory[:4].view(torch.int32).fill_(word)
        with pytest.raises(RuntimeError, match=what):
            cache.check()
        cache.check()
