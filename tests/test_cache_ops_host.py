"""Refusals of the cache and logits operators, and the layout of spacer_kv_cache: host only, no kernel is launched."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from spacer_amd import _lib
from spacer_amd import kernels as K

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EINVAL, ENOMEM = -1, -3


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    return _lib.load()


def test_struct_layout(tmp_path):
    names = [f for f, _ in _lib.KvCache._fields_]
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "%s"\nint main(void) { printf("%%zu", sizeof(spacer_kv_cache));\n' % os.path.join(ROOT, "include", "spacer_hip.h")
    src += "".join(f'printf(" %zu", offsetof(spacer_kv_cache, {n}));\n' for n in names) + "return 0; }\n"
    (tmp_path / "p.c").write_text(src)
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-o", str(tmp_path / "p"), str(tmp_path / "p.c")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "p")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(_lib.KvCache)] + [getattr(_lib.KvCache, n).offset for n in names]


def cache(**kw):
    """A well-formed description of memory that is never touched."""
    f = dict(format=_lib.SPACER_KV_INT8, n_seq=2, capacity=64, kv_heads=2, head_dim=128, k=0x1000, v=0x2000, k_scale=0x3000, v_scale=0x4000,
             stride_seq=2 * 64 * 128, stride_head=64 * 128, stride_pos=128, scale_stride_seq=128, scale_stride_head=64, scale_stride_pos=1)
    f.update(kw)
    c = _lib.KvCache(**{k: v for k, v in f.items() if k != "struct_bytes"})
    if "struct_bytes" in kw:
        c.struct_bytes = kw["struct_bytes"]
    return c


BAD_CACHES = [dict(struct_bytes=8), dict(format=3), dict(format=-1), dict(head_dim=80), dict(head_dim=0), dict(n_seq=0), dict(capacity=-1), dict(kv_heads=0),
              dict(stride_pos=1 << 27), dict(scale_stride_pos=-1), dict(k=None), dict(v=0x2008), dict(stride_pos=136), dict(stride_head=8), dict(k_scale=None), dict(v_scale=None),
              dict(format=_lib.SPACER_KV_BF16, stride_pos=132)]


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_bad_caches_are_refused(lib, bad):
    c, good, p = cache(**bad), cache(), 0x10000
    assert lib.spacer_kv_write(C.byref(c), p, p, 256, 4, p, None) == EINVAL
    assert lib.spacer_kv_append(C.byref(c), p, p, 256, 1, p, 0, None) == EINVAL
    assert lib.spacer_kv_read(C.byref(c), None, p, p, 0, None) == EINVAL
    assert lib.spacer_decode_qkv_finish_cache(p, None, p, p, p, C.byref(c), p, 0, None, None, 0, 0.0, 4, None) == EINVAL
    assert lib.spacer_attn_cache(p, 512, C.byref(c), p, None, 1, None, None, 0, None, 0, p, 2, 1, 4, 1.0, p, 1 << 30, None) == EINVAL
    assert lib.spacer_attn_cache(p, 512, None, None, None, 1, C.byref(c), p, 0, None, 0, p, 2, 1, 4, 1.0, p, 1 << 30, None) == EINVAL
    assert lib.spacer_attn_cache_workspace_bytes(C.byref(good), C.byref(c), 1, 2, 1, 4) == -1
    assert lib.spacer_last_error()


def test_entries_refuse(lib):
    c, p = cache(), 0x10000
    r = C.byref(c)
    assert lib.spacer_kv_write(None, p, p, 256, 4, p, None) == EINVAL
    assert lib.spacer_kv_write(r, p, p, 256, 4, None, None) == EINVAL
    assert lib.spacer_kv_write(r, p, p, 256, -1, p, None) == EINVAL
    assert lib.spacer_kv_write(r, p + 2, p, 256, 4, p, None) == EINVAL
    assert lib.spacer_kv_write(r, p, p, 260, 4, p, None) == EINVAL
    assert lib.spacer_kv_append(r, p, p, 256, 1, None, 0, None) == EINVAL
    assert lib.spacer_kv_append(r, p, p, 256, 1 << 30, p, 0, None) == EINVAL
    assert lib.spacer_kv_read(r, None, p, None, 0, None) == EINVAL
    assert lib.spacer_kv_read(r, None, p + 4, p, 0, None) == EINVAL

    def attn(q=p, ld=512, prompt=r, plen=p, row0=None, rows=1, tail=r, tlen=p, o=p, B=2, N=1, Hq=4, ws=p, n=1 << 30, scale=1.0):
        return lib.spacer_attn_cache(q, ld, prompt, plen, row0, rows, tail, tlen, 0, None, 0, o, B, N, Hq, scale, ws, n, None)
    for kw in (dict(q=None), dict(q=p + 8), dict(ld=516), dict(prompt=None, tail=None), dict(plen=None), dict(tlen=None), dict(o=None), dict(B=3), dict(B=-1), dict(N=0), dict(N=65),
               dict(Hq=3), dict(Hq=0), dict(rows=0), dict(rows=2), dict(scale=0.0), dict(scale=-0.1), dict(scale=float("nan")), dict(scale=float("inf")), dict(prompt=C.byref(cache(head_dim=64))), dict(prompt=C.byref(cache(format=1))),
               dict(prompt=C.byref(cache(kv_heads=1)))):
        assert attn(**kw) == EINVAL, kw
    # (short contexts need no workspace)
    assert lib.spacer_attn_cache_workspace_bytes(r, r, 1, 2, 1, 4) == 0
    r = C.byref(cache(capacity=4096, stride_head=4096 * 128, stride_seq=2 * 4096 * 128, scale_stride_head=4096, scale_stride_seq=8192))
    need = lib.spacer_attn_cache_workspace_bytes(r, r, 1, 2, 1, 4)
    assert need > 0
    for kw in (dict(ws=None), dict(n=64), dict(ws=p + 4), dict(n=need - 1)):
        assert attn(prompt=r, tail=r, **kw) == ENOMEM, kw

    def logits(x=p, out=p, B=2, V=100, seen=p, counts=p, rep=1.0, f=0.0, pr=0.0, allowed=None, n=0, row=None):
        return lib.spacer_process_logits(x, 100, out, 100, B, V, seen, counts, rep, None, f, None, pr, None, None, 0, allowed, n, row, None)
    for kw in (dict(x=None), dict(out=None), dict(V=0), dict(B=-1), dict(B=70000), dict(rep=0.0), dict(rep=-1.0), dict(rep=float("nan")), dict(seen=None), dict(counts=None, f=0.1),
               dict(counts=None, pr=0.1), dict(allowed=p, n=3), dict(allowed=p, n=0, row=p)):
        assert logits(**kw) == EINVAL, kw
    assert logits(B=0) == 0
    assert lib.spacer_token_history_add(None, None, 2, 100, p, 4, 4, None, None) == EINVAL
    assert lib.spacer_token_history_add(p, None, 2, 0, p, 4, 4, None, None) == EINVAL
    assert lib.spacer_token_history_add(p, None, 2, 100, None, 4, 4, None, None) == EINVAL
    assert lib.spacer_token_history_add(p, None, 2, 100, p, 4, 0, None, None) == 0


def test_written_caches_own_their_rows(lib):
    """Rows or scales at one address: read, never written.  (With n = 0 a writer that refuses nothing returns before any launch.)"""
    token_major = dict(stride_seq=64 * 2 * 128, stride_head=128, stride_pos=2 * 128, scale_stride_seq=128, scale_stride_head=1, scale_stride_pos=2)
    one = dict(n_seq=1, stride_seq=0, scale_stride_seq=0)
    for good in (dict(), token_major, one, dict(format=_lib.SPACER_KV_BF16, k_scale=None, v_scale=None)):
        c = cache(**good)
        assert lib.spacer_kv_write(C.byref(c), 0x10000, 0x10000, 256, 0, 0x10000, None) == 0
        assert lib.spacer_kv_append(C.byref(c), 0x10000, 0x10000, 256, 0, 0x10000, 0, None) == 0
    for bad in (dict(stride_seq=0), dict(stride_head=0), dict(stride_pos=0), dict(stride_pos=112), dict(stride_head=63 * 128), dict(v=0x1000), dict(scale_stride_seq=0),
                dict(scale_stride_head=63), dict(scale_stride_pos=0), dict(v_scale=0x3000), dict(capacity=(1 << 30) + 1)):
        c, p = cache(**bad), 0x10000
        assert lib.spacer_kv_write(C.byref(c), p, p, 256, 0, p, None) == EINVAL, bad
        assert lib.spacer_kv_append(C.byref(c), p, p, 256, 0, p, 0, None) == EINVAL, bad
        assert lib.spacer_decode_qkv_finish_cache(p, None, p, p, p, C.byref(c), p, 0, None, None, 0, 0.0, 4, None) == EINVAL, bad


def test_logits_refuse_overlaps_and_sizes(lib):
    def logits(x, ld, out, ld_out, B, V=100):
        # (the history pointers are refused last: an otherwise good call ends at `counts` without `seen`, before any launch)
        rc = lib.spacer_process_logits(x, ld, out, ld_out, B, V, None, 0x9000, 1.0, None, 0.0, None, 0.0, None, None, 0, None, 0, None, None)
        assert rc == EINVAL
        return lib.spacer_last_error().decode()
    p = 0x100000
    for good in ((p, 100, p, 100, 4), (p, 104, p, 200, 1), (p, 200, p + 400, 200, 4), (p + 400, 200, p, 200, 4), (p, 0, p + 400, 100, 4), (p, 100, p + 1600, 128, 4)):
        assert "counts without seen" in logits(*good), good
    for bad in ((p, 100, p + 4, 100, 4), (p, 100, p, 104, 4), (p, 200, p + 400, 208, 4), (p, 200, p + 396, 200, 4), (p, 200, p + 404, 200, 4), (p, 0, p, 0, 4), (p, 100, p + 4000, 99, 4),
                (p + 4, 100, p, 100, 1)):
        assert "overlap" in logits(*bad), bad
    assert "vocab" in logits(p, 1 << 31, p, 1 << 31, 1, V=(1 << 30) + 1)
    assert lib.spacer_token_history_add(p, None, 1, (1 << 30) + 1, p, 4, 4, None, None) == EINVAL
    assert lib.spacer_token_history_add(p, None, 1, 100, p, 1 << 30, (1 << 30) + 1, None, None) == EINVAL


def test_python_layer_refuses():
    z = torch.zeros(1, 2, 16, 128, dtype=torch.int8)
    s = torch.zeros(1, 2, 16)
    with pytest.raises(K.SpacerError, match="GPU"):
        K.KVCache(z, z, s, s)
    with pytest.raises(K.SpacerError, match="alike"):
        K.KVCache(z, z[:, :1], s, s)
    with pytest.raises(K.SpacerError, match="dtype"):
        K.KVCache(z.half(), z.half(), s, s)
    with pytest.raises(K.SpacerError, match="dtype"):
        K.KVCache.empty(1, 2, 3, 128, "fp4", device="cpu")
    with pytest.raises(K.SpacerError, match="fp32"):
        K.process_logits(torch.zeros(2, 10, dtype=torch.float16))
    with pytest.raises(K.SpacerError, match="history"):
        K.process_logits(torch.zeros(2, 10), repetition=1.1)
    with pytest.raises(K.SpacerError, match="allowed_row"):
        K.process_logits(torch.zeros(2, 10), allowed_row=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(K.SpacerError, match="bias"):
        K.process_logits(torch.zeros(2, 10), bias=torch.zeros(9))
    with pytest.raises(K.SpacerError, match="ids"):
        K.token_history_add_(torch.zeros(2, 1, dtype=torch.int32), None, torch.zeros(2, 4, dtype=torch.int32))
    with pytest.raises(K.SpacerError, match="cache"):
        K.attn_cache(torch.zeros(2, 128, dtype=torch.bfloat16), None, None, None, None, 1, 1.0)


def test_logit_rules_refuse_and_pack():
    """SamplingParams' rules: what leaves nothing to draw or is no number is refused before any kernel; the allowed ids as bits."""
    from spacer_amd.rollout import SamplingParams, _LogitRules
    inf, nan = float("inf"), float("nan")

    def rules(**kw):
        sp = SamplingParams(**kw)
        assert _LogitRules.wanted(sp)
        return _LogitRules(sp, [], [1], 100, 7, "cpu")
    for kw in (dict(logit_bias={100: 1.0}), dict(logit_bias={-1: 1.0}), dict(logit_bias={3: nan}), dict(logit_bias={3: inf}), dict(allowed_token_ids=[]), dict(allowed_token_ids=[100]),
               dict(allowed_token_ids=[5, -1]), dict(allowed_token_ids=[3], logit_bias={3: -inf}), dict(allowed_token_ids=[7], suppress_eos=True), dict(allowed_token_ids=[7], synthetic_lengths=(2, 4)), dict(repetition_penalty=0.0),
               dict(repetition_penalty=-1.0), dict(repetition_penalty=nan), dict(repetition_penalty=inf), dict(frequency_penalty=nan), dict(presence_penalty=-inf)):
        with pytest.raises(ValueError):
            rules(**kw)
    assert not _LogitRules.wanted(SamplingParams())
    r = rules(allowed_token_ids=[0, 31, 32, 99, 99], logit_bias={2: -inf, 99: 0.5})
    assert r.allowed.tolist() == [[(1 << 31 | 1) - 2 ** 32, 1, 0, 8]] and r.seen is None
    assert r.bias[2] == -inf and r.bias[99] == 0.5 and int((r.bias != 0).sum()) == 2
