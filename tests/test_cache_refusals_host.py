"""More refusals of the cache operators and of the paths that call them: host only, no kernel is launched."""
import ctypes as C
import os
from types import SimpleNamespace

import pytest
import torch

from spacer_amd import _lib
from spacer_amd import kernels as K

BF = torch.bfloat16


def test_missing_lengths_and_rows_are_refused():
    """A cache without its lengths (or a writer without its rows) is a SpacerError like every other bad argument."""
    cache = SimpleNamespace(head_dim=64, kv_heads=2, n_seq=2, capacity=8, k=None, _ref=None, _shape=None)
    q = torch.zeros(2, 4 * 64, dtype=BF)
    kv = torch.zeros(2, 2 * 64, dtype=BF)
    lens = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: K.attn_cache(q, cache, None, None, None, 4, 1.0), lambda: K.attn_cache(q, None, None, cache, None, 4, 1.0),
                 lambda: K.attn_cache(q, cache, lens, cache, None, 4, 1.0), lambda: K.kv_write(cache, kv, kv, None), lambda: K.kv_append(cache, kv, kv, None),
                 lambda: K.decode_qkv_finish_cache(torch.zeros(2, 8 * 64), None, torch.zeros(2, 64), torch.zeros(2, 64), torch.zeros(2, 256, dtype=BF), cache, None, 4)):
        with pytest.raises(K.SpacerError, match="int32"):
            call()
