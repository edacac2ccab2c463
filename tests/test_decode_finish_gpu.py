"""decode_qkv_finish, decode_qkv_finish_normed and decode_qkv_finish_cache without a bias, and the cache form at widths, formats and lengths of its own."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from spacer_amd import kernels as K        # noqa: E402
from test_cache_ops_gpu import BF, E4M3, I8, make_cache, rnd, same  # noqa: E402


def tables(B, D, low, dev):
    """Rotary tables whose first cosine ends in the bits `low`: read as a bf16 number these are an infinity, a NaN, or a finite one."""
    ang = rnd((B, D // 2), 3).float()
    cos, sin = torch.cat([ang.cos()] * 2, 1), torch.cat([ang.sin()] * 2, 1)
    bits = cos.view(torch.int32)
    bits[0, 0] = (bits[0, 0] & ~0xFFFF) | low
    return cos.to(dev), sin.to(dev)


LOW = [0x7F80, 0x7FC0, 0xFF80, 0xFFFF, 0x3F80]


@pytest.mark.parametrize("low", LOW)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("norm", [False, True])
def test_finish_without_a_bias(dev, low, D, norm):
    """No bias is a bias of zeros, whatever the rotary table holds."""
    B, Hq, Hkv, cap = 3, 4, 2, 5
    acc0 = rnd((B, (Hq + 2 * Hkv) * D), 1).float().to(dev)
    cos, sin = tables(B, D, low, dev)
    pos = torch.tensor([2], dtype=torch.int32, device=dev)
    rowss = (rnd((B,), 4).abs() * 300 + 50).float().to(dev)
    out = []
    for bias in (None, torch.zeros((Hq + 2 * Hkv) * D, dtype=BF, device=dev)):
        q, tk, tv = torch.zeros(B, Hq * D, device=dev, dtype=BF), *(torch.zeros(B, cap, Hkv, D, device=dev, dtype=BF) for _ in range(2))
        if norm:
            K.decode_qkv_finish_normed(acc0.clone(), bias, cos, sin, q, tk, tv, pos, rowss, torch.ones(B, device=dev), 256, 1e-6, Hq, Hkv, D)
        else:
            K.decode_qkv_finish(acc0.clone(), bias, cos, sin, q, tk, tv, pos, Hq, Hkv, D)
        out.append((q, tk, tv))
    for a, b in zip(*out):
        assert bool(a.isfinite().all()) and torch.equal(a, b)


@pytest.mark.parametrize("low", LOW)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF, E4M3, I8])
@pytest.mark.parametrize("norm", [False, True])
def test_finish_cache_without_a_bias(dev, low, D, dtype, norm):
    """... and every sequence's row goes to that sequence's own length; lengths outside the cache are dropped."""
    B, Hq, Hkv, cap = 5, 4, 2, 7
    acc0 = rnd((B, (Hq + 2 * Hkv) * D), 1).float().to(dev)
    cos, sin = tables(B, D, low, dev)
    lens = torch.tensor([0, 6, 3, 7, -1], dtype=torch.int32, device=dev)
    kw = dict(rowss=(rnd((B,), 4).abs() * 300 + 50).float().to(dev), norm_cols=256, eps=1e-6) if norm else {}
    out = []
    for bias in (None, torch.zeros((Hq + 2 * Hkv) * D, dtype=BF, device=dev)):
        cache, q = make_cache(B, cap, Hkv, D, dtype, dev), torch.zeros(B, Hq * D, device=dev, dtype=BF)
        K.decode_qkv_finish_cache(acc0.clone(), bias, cos, sin, q, cache, lens, Hq, **kw)
        out.append((q, *K.kv_read(cache, dtype=torch.float32)))
    for a, b in zip(*out):
        assert bool(a.isfinite().all()) and torch.equal(a, b)
    # the rows lie where the lengths say: those of kv_append from a bf16 cache that took them at position 0
    plain = make_cache(B, 1, Hkv, D, BF, dev)
    K.decode_qkv_finish_cache(acc0.clone(), None, cos, sin, torch.zeros(B, Hq * D, device=dev, dtype=BF), plain, torch.zeros(1, dtype=torch.int32, device=dev), Hq, **kw)
    want = make_cache(B, cap, Hkv, D, dtype, dev)
    K.kv_append(want, *(x[:, 0].reshape(B, -1).contiguous() for x in K.kv_read(plain)), lens)
    for a, b in zip(out[0][1:], K.kv_read(want, dtype=torch.float32)):
        assert same(a, b)
    assert float(out[0][1][3:].abs().max()) == 0.0
