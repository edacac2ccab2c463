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


EINVAL = -1


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    return _lib.load()


def described(shape, strides, sstrides, fmt, delta, sdelta):
    """A cache whose v (v_scale) lies delta elements (sdelta floats) behind its k (k_scale); the memory is never touched."""
    size, base = 2 if fmt == _lib.SPACER_KV_BF16 else 1, 1 << 40
    return _lib.KvCache(format=fmt, n_seq=shape[0], kv_heads=shape[1], capacity=shape[2], head_dim=shape[3], k=base, v=base + delta * size,
                        k_scale=None if size == 2 else 2 * base, v_scale=None if size == 2 else 2 * base + 4 * sdelta,
                        stride_seq=strides[0], stride_head=strides[1], stride_pos=strides[2],
                        scale_stride_seq=sstrides[0], scale_stride_head=sstrides[1], scale_stride_pos=sstrides[2])


def refusal(lib, c):
    """What the writers say of a cache: the sources are refused last (before any launch), so an otherwise good call names them."""
    p, said = 0x10002, set()
    for rc in (lib.spacer_kv_write(C.byref(c), p, p, 1024, 4, p, None), lib.spacer_kv_append(C.byref(c), p, p, 1024, 1, p, 0, None)):
        assert rc == EINVAL
        said.add(lib.spacer_last_error().decode().split(": ", 1)[1])
    assert lib.spacer_decode_qkv_finish_cache(None, None, None, None, None, C.byref(c), None, 0, None, None, 0, 0.0, 4, None) == EINVAL
    last = lib.spacer_last_error().decode()
    assert len(said) == 1
    said = said.pop()
    assert ("share memory" in said) == ("share memory" in last), (said, last)
    return said


# (sequences, heads, positions, D) with strides in elements of two layouts, and of rows spread over wider memory
LAYOUTS = [((2, 3, 5, 64), (3 * 5 * 64, 5 * 64, 64)), ((2, 3, 5, 64), (5 * 3 * 64, 64, 3 * 64)), ((3, 2, 4, 128), (4096, 2048, 256)), ((1, 1, 7, 64), (0, 0, 192)), ((3, 1, 1, 128), (384, 0, 0)),
           ((1, 1, 1, 64), (0, 0, 0))]


@pytest.mark.parametrize("fmt", [_lib.SPACER_KV_BF16, _lib.SPACER_KV_INT8])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_rows_of_k_and_v_are_apart(lib, layout, fmt):
    """Against the sets of addresses: every distance between k and v up to beyond the cache's end, to either side."""
    shape, strides = layout
    n, h, cap, d = shape
    starts = {a * strides[0] + b * strides[1] + c * strides[2] for a in range(n) for b in range(h) for c in range(cap)}
    span, step = max(starts) + d, 16 // (2 if fmt == _lib.SPACER_KV_BF16 else 1)
    near = {x - y for x in starts for y in starts}
    for delta in range(-span - 32, span + 33):
        if delta % step or delta == 0:
            continue
        overlap = any(-d < delta - x < d for x in near)
        c = described(shape, strides, (1 << 20, 1 << 15, 1), fmt, delta, 1 << 30)
        assert refusal(lib, c) == ("rows of k and v share memory" if overlap else "source rows must start at multiples of 16 bytes"), delta


@pytest.mark.parametrize("layout", LAYOUTS)
def test_scales_of_k_and_v_are_apart(lib, layout):
    shape, strides = layout
    n, h, cap, _ = shape
    s = tuple(x // 64 for x in strides)
    starts = {a * s[0] + b * s[1] + c * s[2] for a in range(n) for b in range(h) for c in range(cap)}
    for delta in range(-max(starts) - 3, max(starts) + 4):
        if delta == 0:
            continue
        overlap = any((x + delta) in starts for x in starts)
        c = described(shape, strides, s, _lib.SPACER_KV_INT8, 1 << 35, delta)
        assert refusal(lib, c) == ("scales of k and v share memory" if overlap else "source rows must start at multiples of 16 bytes"), delta


def test_row_sums_to_clear_are_not_those_to_read(lib):
    """decode_qkv_finish_cache clears rowss_zero while it reads rowss."""
    p, rows = 0x10000, 300                               # (too many rows to clear: an otherwise good call ends there, before any launch)
    c = described((rows, 1, 1, 64), (64, 0, 0), (1, 0, 0), _lib.SPACER_KV_INT8, 1 << 30, 1 << 30)

    def finish(rowss, rowss_zero):
        assert lib.spacer_decode_qkv_finish_cache(p, None, p, p, p, C.byref(c), p, 0, rowss, rowss_zero, 64, 0.0, 4, None) == EINVAL
        return lib.spacer_last_error().decode()
    for other in (p, p + 4, p + 4 * (rows - 1), p - 4 * (rows - 1)):
        assert "overlaps" in finish(p, other)
    for other in (p + 4 * rows, p - 4 * rows):
        assert "at most 256" in finish(p, other)
    assert "at most 256" in finish(None, p)
