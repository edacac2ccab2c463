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


def test_adapter_passes_the_repetition_penalty_on():
    """generation_config.repetition_penalty as given, None or absent as 1; 0 reaches the rules, which refuse it."""
    from spacer_amd.hf_adapter import SpacerModel
    from spacer_amd.rollout import SamplingParams, _LogitRules
    seen = []
    model = object.__new__(SpacerModel)
    model.__dict__.update(seed=0, _calls=0, era_rule=False, device="cpu", cfg=SimpleNamespace(vocab=100), _pixels=lambda kw: (None, None),
                          roll=SimpleNamespace(generate=lambda prompts, n, sp: seen.append(sp) or torch.zeros(n, 2, dtype=torch.int64)))
    ids = torch.arange(4)[None]
    for given, want in (({}, 1.0), (dict(repetition_penalty=None), 1.0), (dict(repetition_penalty=1.3), 1.3), (dict(repetition_penalty=0.0), 0.0), (dict(repetition_penalty=0), 0.0)):
        out = model.generate(input_ids=ids, generation_config=SimpleNamespace(max_new_tokens=2, num_return_sequences=3, do_sample=True, top_k=5, **given))
        assert out.shape == (3, 6) and seen[-1].repetition_penalty == want, given
        if want == 0.0:
            assert _LogitRules.wanted(seen[-1])
            with pytest.raises(ValueError, match="repetition"):
                _LogitRules(seen[-1], [], [1], 100, 7, "cpu")
    assert not _LogitRules.wanted(SamplingParams())
