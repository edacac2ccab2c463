"""Key/value caches in bf16 / e4m3 / int8, the decode attention that reads them, and the logits operators, against plain 64-bit restatements.

Codes, scales, bit maps and counts are compared exactly.  Attention: with A = sum_j w_j |v_j| of an output (w the softmax weights) an error is at most
  2^-8 |o|            the output's own rounding to bf16
  2^-8 M + 2^-13 A    every weight is rounded to bf16 by a factor 1 + d_j, |d_j| <= 2^-8, and the sum counts the rounded ones: the quotient is off by
                      sum_j w_j d_j (v_j - o) / (1 + sum_j w_j d_j), with M = sum_j w_j |v_j - o| <= 2 A at most 2^-8 M (1 + 2^-7); int8 sums are off by
                      another 2^-17 (a reciprocal in two bf16 numbers): 2^-15 M + 2^-17 |o| <= 2^-13 A in all beside 2^-8 M
  2 E A               E bounds the scores' error in 32 bits: (D + 4) 2^-24 max_j sum_d |q_d k_jd| scale (products and sums), + 2^-21 for exp2 and its argument
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from spacer_amd import kernels as K        # noqa: E402

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E4M3, I8 = torch.float8_e4m3fn, torch.int8


def rnd(shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g, dtype=F64) * scale


def rows_like(shape, seed):
    """bf16 rows of very different sizes with a few large channels, on the CPU."""
    x = rnd(shape, seed) * torch.exp(2.0 * rnd((*shape[:-1], 1), seed + 1)) * (0.3 + 3.0 * (torch.arange(shape[-1]) % 17 == 3))
    return x.to(BF)


def codes_ref(x, dtype):
    """(codes as numbers, scales) of bf16 rows, on the CPU in 64 bits."""
    x = x.double()
    amax = x.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    amax = torch.where(bad, 1.0, amax)
    if dtype == E4M3:
        s = torch.full_like(amax, 2.0 ** -126)
        for e in range(-125, 121):
            s = torch.where(amax / s > 448, 2.0 ** e, s)
        q = (x / s).float().to(E4M3).double()        # x / s is exact; the cast rounds to nearest even
    else:
        s = (amax / 127).float().double()
        q = torch.where(s > 0, torch.round(x / torch.where(s > 0, s, 1.0)), 0.0).clamp(-127, 127)
    q = torch.where(bad, 0.0, q)
    return q, torch.where(bad, math.nan, s).squeeze(-1)


def make_cache(n, cap, hkv, d, dtype, dev, layout="head"):
    if layout == "head":
        return K.KVCache.empty(n, cap, hkv, d, dtype, dev)
    kv = [torch.zeros(n, cap, hkv + 1, d, device=dev, dtype=torch.uint8 if dtype != BF else BF)[:, :, :hkv].transpose(1, 2) for _ in range(2)]
    if dtype == BF:
        return K.KVCache(*kv)
    sc = [torch.zeros(n, cap, hkv, device=dev).transpose(1, 2) for _ in range(2)]
    return K.KVCache(kv[0].view(dtype), kv[1].view(dtype), *sc)


def same(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


# ------------------------------------------------------------------------------------------------------------- writing and reading
@pytest.mark.parametrize("dtype", [BF, E4M3, I8])
@pytest.mark.parametrize("n,cap,hkv,d,layout", [(1, 1, 1, 128, "head"), (3, 37, 2, 128, "head"), (2, 70, 4, 64, "token"), (5, 19, 3, 128, "token"), (1, 600, 8, 64, "head")])
def test_kv_write_and_read(dev, dtype, n, cap, hkv, d, layout):
    T = 2 * cap + 3
    k, v = rows_like((T, hkv, d), 1), rows_like((T, hkv, d), 5)
    k[0, 0] = 0.0
    if T > 6:
        k[1, 0, 3], v[2, 0, 0] = math.nan, math.inf
        v[3, 0] *= 1e-38
        k[4, 0] = torch.arange(d) % 9 - 4.5             # ties of the int8 quotient: amax 4.5
        k[4, 0, 0] = 127.0
        k[5, 0], v[5, 0, :] = 1.0, -(2.0 ** -133)       # the smallest bf16 number
    packed = torch.zeros(T, 8 + 2 * hkv * d, dtype=BF, device=dev)           # columns of wider rows
    packed[:, 8:8 + hkv * d], packed[:, 8 + hkv * d:] = k.reshape(T, -1), v.reshape(T, -1)
    cache = make_cache(n, cap, hkv, d, dtype, dev, layout)
    g = torch.Generator().manual_seed(3)
    rows = torch.randint(-2, T + 2, (n * cap,), generator=g, dtype=torch.int32)     # repeated, missing and out-of-range rows
    before = [x.clone() for x in K.kv_read(cache, dtype=F32)]
    K.kv_write(cache, packed[:, 8:8 + hkv * d], packed[:, 8 + hkv * d:], rows.to(dev))
    got = K.kv_read(cache, dtype=F32)
    ok = ((rows >= 0) & (rows < T)).view(n, cap)
    at = rows.clamp(0, T - 1).long()
    for x, codes, scale, out, old in ((k, cache.k, cache.k_scale, got[0], before[0]), (v, cache.v, cache.v_scale, got[1], before[1])):
        assert same(out[~ok.to(dev)], old[~ok.to(dev)])
        want = x[at].view(n, cap, hkv, d)
        if dtype == BF:
            assert same(out[ok.to(dev)], want[ok])
            continue
        q, s = codes_ref(want, dtype)
        assert same(codes.transpose(1, 2)[ok.to(dev)].float(), q[ok])
        assert same(scale.transpose(1, 2)[ok.to(dev)], s[ok])
        assert same(out[ok.to(dev)], (q[ok].float() * s[ok].float()[..., None]))
        out16 = K.kv_read(cache, dtype=BF)[0 if codes is cache.k else 1]
        assert same(out16, out.to(BF))
    lens = torch.tensor([(7 * i) % (cap + 2) for i in range(n)], dtype=torch.int32)
    cut = K.kv_read(cache, lens.to(dev), dtype=F32)
    keep = torch.arange(cap) < lens[:, None]
    assert same(cut[0], torch.where(keep[..., None, None], got[0].cpu(), torch.zeros(())))


@pytest.mark.parametrize("dtype", [E4M3, I8])
@pytest.mark.parametrize("exponent", [-133, -126, -100, -97, -96, -30, 0, 90, 127])
def test_kv_write_every_quotient(dev, dtype, exponent):
    """Every bf16 number of the 9 binades below a row's maximum, for every significand of that maximum: codes and scales are exact."""
    top = torch.arange(128, 256, dtype=F64) * 2.0 ** (exponent - 7)
    rows = []
    for shift in range(9):
        for part in (0, 1):
            sig = torch.arange(128 + 64 * part, 192 + 64 * part, dtype=F64)
            x = torch.stack([sig, -sig], 1).view(-1) * 2.0 ** (exponent - 7 - shift)
            row = x[None].expand(128, -1).clone()
            row[row.abs() > top[:, None]] = 0.0
            row[:, 5] = top * (-1) ** shift
            rows.append(row)
    x = torch.cat(rows).to(BF)                            # (numbers below 2^-133 round to 0 or to it)
    n = x.shape[0]
    cache = make_cache(1, n, 1, 128, dtype, dev)
    K.kv_write(cache, x.to(dev), x.flip(1).to(dev), torch.arange(n, dtype=torch.int32, device=dev))
    for codes, scale, want in ((cache.k, cache.k_scale, x), (cache.v, cache.v_scale, x.flip(1))):
        q, s = codes_ref(want, dtype)
        assert same(scale[0, 0], s) and same(codes[0, 0].float(), q)


@pytest.mark.parametrize("dtype", [BF, E4M3, I8])
@pytest.mark.parametrize("N,shared", [(1, False), (1, True), (5, False)])
def test_kv_append(dev, dtype, N, shared):
    n, cap, hkv, d = 4, 12, 3, 128
    cache = make_cache(n, cap, hkv, d, dtype, dev)
    k, v = rows_like((n * N, hkv, d), 11), rows_like((n * N, hkv, d), 13)
    lens = torch.tensor([9] if shared else [0, 9, -2, 40], dtype=torch.int32)
    K.kv_append(cache, k.reshape(n * N, -1).to(dev), v.reshape(n * N, -1).to(dev), lens.to(dev))
    want = [torch.zeros(n, cap, hkv, d) for _ in range(2)]
    for s in range(n):
        for i in range(N):
            p = int(lens[0 if shared else s]) + i
            if 0 <= p < cap:
                for w, x in zip(want, (k, v)):
                    if dtype == BF:
                        w[s, p] = x[s * N + i].float()
                    else:
                        q, sc = codes_ref(x[s * N + i], dtype)
                        w[s, p] = q.float() * sc.float()[..., None]
    for got, w in zip(K.kv_read(cache, dtype=F32), want):
        assert same(got, w)


def test_decode_qkv_finish_cache(dev):
    """The decode step's writer: q as decode_qkv_finish (one bf16 step of room: the two are compiled with different contraction), and in every format the codes
    that kv_append makes of the bf16 rows."""
    B, Hq, Hkv, D, cap = 5, 4, 2, 128, 9
    acc0 = rnd((B, (Hq + 2 * Hkv) * D), 1).float().to(dev)
    bias = rnd(((Hq + 2 * Hkv) * D,), 2).to(BF).to(dev)
    ang = rnd((B, D // 2), 3).float()
    cos, sin = torch.cat([ang.cos()] * 2, 1).to(dev), torch.cat([ang.sin()] * 2, 1).to(dev)
    pos = torch.tensor([4], dtype=torch.int32, device=dev)
    rowss = (rnd((B,), 4).abs() * 300 + 50).float().to(dev)
    for norm in (False, True):
        kw = dict(rowss=rowss, rowss_zero=torch.ones(B, device=dev), norm_cols=256, eps=1e-6) if norm else {}
        q0, tk, tv = torch.zeros(B, Hq * D, device=dev, dtype=BF), *(torch.zeros(B, cap, Hkv, D, device=dev, dtype=BF) for _ in range(2))
        acc = acc0.clone()
        if norm:
            K.decode_qkv_finish_normed(acc, bias, cos, sin, q0, tk, tv, pos, rowss, torch.ones(B, device=dev), 256, 1e-6, Hq, Hkv, D)
        else:
            K.decode_qkv_finish(acc, bias, cos, sin, q0, tk, tv, pos, Hq, Hkv, D)
        plain = make_cache(B, cap, Hkv, D, BF, dev)
        for dtype in (BF, E4M3, I8):
            cache, q, acc = make_cache(B, cap, Hkv, D, dtype, dev), torch.zeros_like(q0), acc0.clone()
            K.decode_qkv_finish_cache(acc, bias, cos, sin, q, plain if dtype == BF else cache, pos, Hq, **kw)
            assert float(acc.abs().max()) == 0
            if norm:
                assert float(kw["rowss_zero"].abs().max()) == 0
                kw["rowss_zero"].fill_(1.0)
            assert float(((q.float() - q0.float()).abs() - 2.0 ** -7 * q0.float().abs()).max()) <= 1e-6
            if dtype == BF:
                for a, b in zip(K.kv_read(plain), (tk, tv)):
                    assert float(((a.float() - b.float()).abs() - 2.0 ** -7 * b.float().abs()).max()) <= 1e-6
                continue
            want = make_cache(B, cap, Hkv, D, dtype, dev)
            k, v = K.kv_read(plain)
            K.kv_append(want, k[:, 4].reshape(B, -1).contiguous(), v[:, 4].reshape(B, -1).contiguous(), pos)
            for a, b in zip(K.kv_read(cache, dtype=F32), K.kv_read(want, dtype=F32)):
                assert same(a, b)


# ------------------------------------------------------------------------------------------------------------- attention
def filled(n, cap, hkv, d, dtype, dev, seed, layout="head"):
    """A cache of random rows written by kv_write, and its values [n, hkv, cap, d] in 64 bits on the CPU."""
    cache = make_cache(n, cap, hkv, d, dtype, dev, layout)
    k, v = (rnd((n * cap, hkv * d), seed + i).to(BF).to(dev) for i in range(2))
    K.kv_write(cache, k, v, torch.arange(n * cap, dtype=torch.int32, device=dev))
    return cache, [x.double().cpu().transpose(1, 2) for x in K.kv_read(cache, dtype=F32)]


def attn_ref(q, prompt, plen, owner, tail, tlen, masks, hq, scale, nodes):
    """(output, tolerance) [B * nodes, hq * d] in 64 bits; prompt / tail: (k, v) values or None; owner[b]: prompt of sequence b or None; masks[b][i]: ints."""
    B = q.shape[0] // nodes
    hkv, d = (prompt or tail)[0].shape[1], (prompt or tail)[0].shape[3]
    rep = hq // hkv
    q = q.double().cpu().view(B, nodes, hq, d)
    out, tol = torch.zeros(B, nodes, hq, d, dtype=F64), torch.zeros(B, nodes, hq, d, dtype=F64)
    for b in range(B):
        for i in range(nodes):
            ks, vs = [], []
            if prompt is not None and owner[b] is not None:
                n = min(max(plen[owner[b]], 0), prompt[0].shape[2])
                ks.append(prompt[0][owner[b], :, :n]); vs.append(prompt[1][owner[b], :, :n])
            if tail is not None:
                cap = tail[0].shape[2]
                n = min(max(tlen[b], 0), cap)
                pick = list(range(n)) + [n + j for j in range(nodes) if masks[b][i] >> j & 1 and n + j < cap]
                ks.append(tail[0][b][:, pick]); vs.append(tail[1][b][:, pick])
            k, v = torch.cat(ks, 1).repeat_interleave(rep, 0), torch.cat(vs, 1).repeat_interleave(rep, 0)
            if k.shape[1] == 0:
                continue
            x = torch.einsum("hd,hld->hl", q[b, i], k) * scale
            w = torch.softmax(x, -1)
            o, a = torch.einsum("hl,hld->hd", w, v), torch.einsum("hl,hld->hd", w, v.abs())
            e = (d + 4) * 2.0 ** -24 * torch.einsum("hd,hld->hl", q[b, i].abs(), k.abs()).amax(-1) * scale + 2.0 ** -21
            spread = torch.einsum("hl,hld->hd", w, (v - o[:, None]).abs())
            out[b, i], tol[b, i] = o, 2.0 ** -8 * (o.abs() + spread) + 2.0 ** -13 * a + 2 * e[:, None] * a
    return out.view(B * nodes, hq * d), tol.view(B * nodes, hq * d)


def chain(nodes):
    return [(2 << i) - 1 for i in range(nodes)]


def random_tree(nodes, seed):
    g = torch.Generator().manual_seed(seed)
    m = []
    for i in range(nodes):
        m.append((m[int(torch.randint(0, i, (1,), generator=g))] if i and torch.rand(1, generator=g) < 0.8 else 0) | (1 << i))
    return m


def as_int64(masks, dev):
    return torch.tensor([[x - 2 ** 64 if x >= 2 ** 63 else x for x in row] for row in masks], dtype=torch.int64, device=dev)


def close(got, want, tol, what=""):
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol.clamp_min(1e-30))[bad].max()):.3g} tolerances"


SHAPES = [
    # prompts, rows, plens, tail cap, tail lengths, nodes, hq, hkv, d
    (1, 1, [1], 1, [0], 1, 1, 1, 128),
    (1, 2, [203], 64, [17, 17], 1, 12, 2, 128),
    (2, 3, [33, 0], 40, [0, 5, 31, 32, 33, 39], 1, 14, 2, 128),
    (3, 8, [1030, 64, 511], 70, [3 * i for i in range(24)], 1, 28, 4, 128),
    (2, 2, [96, 31], 50, [0, 1, 2, 40], 1, 24, 1, 64),
    (1, 4, [70], 90, [0, 9, 60, 77], 13, 16, 2, 128),
    (2, 1, [129, 3], 200, [0, 136], 64, 8, 8, 64),
    (1, 2, [40], 100, [31, 98], 5, 2, 1, 64),          # the second sequence's nodes leave the cache at its end
    (1, 3, [2500], 20, [4, 5, 6], 2, 6, 2, 128),
    # contexts past the one-launch form, by the columns that share the prompt's and the sequence's keys: 16, 32, 64 and more
    (1, 2, [700], 33, [5, 32], 1, 6, 2, 128), (1, 2, [800], 33, [5, 32], 1, 6, 2, 64),
    (1, 1, [600], 40, [3], 7, 12, 3, 128), (1, 1, [900], 40, [33], 7, 12, 3, 64),
    (2, 1, [600, 555], 100, [0, 36], 64, 16, 2, 128), (2, 1, [33, 640], 100, [31, 36], 33, 6, 2, 64),
    (2, 4, [520, 1], 1100, [1099, 1000, 64, 63, 0, 500, 999, 31], 1, 28, 4, 64),
]


@pytest.mark.parametrize("dtype", [BF, E4M3, I8])
@pytest.mark.parametrize("shape", SHAPES)
def test_attn_cache(dev, dtype, shape):
    nP, rows, plens, tcap, tlens, nodes, hq, hkv, d = shape
    B = nP * rows
    layout = "token" if B % 2 else "head"
    prompt, pval = filled(nP, max(plens), hkv, d, dtype, dev, 21, layout)
    tail, tval = filled(B, tcap, hkv, d, dtype, dev, 31, layout)
    wide = (rnd((B * nodes, hq * d + 8), 41) * 1.5).to(BF).to(dev)
    q = wide[:, :hq * d]
    trees = [random_tree(nodes, 100 + b) for b in range(B)]
    owner = [b // rows for b in range(B)]
    pl, tl = torch.tensor(plens, dtype=torch.int32, device=dev), torch.tensor(tlens, dtype=torch.int32, device=dev)
    for tree, masks in ((None, [chain(nodes)] * B), (as_int64(trees, dev), trees), (as_int64(trees, dev)[0].contiguous(), [trees[0]] * B)):
        got = K.attn_cache(q, prompt, pl, tail, tl, hq, d ** -0.5, rows_per_prompt=rows, nodes=nodes, tree=tree)
        close(got, *attn_ref(q, pval, plens, owner, tval, tlens, masks, hq, d ** -0.5, nodes), what=f"{shape} {dtype}")


# every form of the launch (one or two of them, 16 or 32 columns per workgroup for the prompt's and for the sequence's keys) in every format and width
FORMS = [
    (4, 4, [100, 1, 0, 77], 40, 5, 64, 16), (1, 3, [1900], 40, 1, 8, 2), (2, 16, [1900, 33], 40, 1, 28, 2), (2, 2, [1, 1900], 40, 21, 8, 2),
    (2, 32, [250, 1900], 40, 1, 28, 2), (4, 2, [0, 1900, 65, 320], 70, 64, 16, 2),
]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [BF, E4M3, I8])
@pytest.mark.parametrize("form", FORMS)
def test_attn_cache_forms(dev, dtype, form, d):
    nP, rows, plens, tcap, nodes, hq, hkv = form
    B = nP * rows
    prompt, pval = filled(nP, max(plens), hkv, d, dtype, dev, 61)
    tail, tval = filled(B, tcap, hkv, d, dtype, dev, 71, "token")
    tlens = [(13 * b) % (tcap + 1) for b in range(B)]
    q = (rnd((B * nodes, hq * d), 81) * 1.5).to(BF).to(dev)
    trees = [random_tree(nodes, 200 + b) for b in range(B)]
    got = K.attn_cache(q, prompt, torch.tensor(plens, dtype=torch.int32, device=dev), tail, torch.tensor(tlens, dtype=torch.int32, device=dev), hq, d ** -0.5,
                       rows_per_prompt=rows, nodes=nodes, tree=as_int64(trees, dev))
    close(got, *attn_ref(q, pval, plens, [b // rows for b in range(B)], tval, tlens, trees, hq, d ** -0.5, nodes), what=f"{form} {dtype} {d}")


@pytest.mark.parametrize("d", [64, 128])
def test_attn_cache_nan_codes(dev, d):
    """e4m3 NaN codes (a caller's own: the writers make none) in a drafted node's value row reach the nodes that see it, and no other."""
    hq, hkv, nodes, B = 4, 2, 5, 2
    tail, tval = filled(B, 60, hkv, d, E4M3, dev, 2)
    tlen = [27, 40]
    for b in range(B):
        tail.v.view(torch.uint8)[b, :, tlen[b] + 2, d // 2] = 0x7F if b else 0xFF
        tail.k.view(torch.uint8)[b, :, tlen[b] + 2, 3] = 0x7F
    q = rnd((B * nodes, hq * d), 3).to(BF).to(dev)
    masks = [[1, 3, 5, 9, 17], [1, 2, 4, 14, 24]]        # nodes 2 (both) and 3 (second sequence) see node 2
    got = K.attn_cache(q, None, None, tail, torch.tensor(tlen, dtype=torch.int32, device=dev), hq, 0.1, nodes=nodes, tree=as_int64(masks, dev))
    sees = torch.tensor([[m >> 2 & 1 for m in row] for row in masks]).bool().view(-1)
    want, tol = attn_ref(q, None, None, None, tval, tlen, [[m & ~4 for m in row] for row in masks], hq, 0.1, nodes)
    close(got[~sees.to(dev)], want[~sees], tol[~sees])
    assert bool(got[sees.to(dev)].isnan().all())


@pytest.mark.parametrize("dtype", [BF, I8])
def test_attn_cache_parts(dev, dtype):
    """Only a prompt, only a tail, ragged prompt owners with sequences that none owns, one length for all, lengths outside the cache."""
    hq, hkv, d, B = 7, 1, 128, 6
    prompt, pval = filled(3, 45, hkv, d, dtype, dev, 1)
    tail, tval = filled(B, 33, hkv, d, dtype, dev, 2)
    q = rnd((B, hq * d), 3).to(BF).to(dev)
    pl = torch.tensor([45, 900, -3], dtype=torch.int32, device=dev)
    one = torch.tensor([11], dtype=torch.int32, device=dev)
    masks = [[1]] * B
    s = d ** -0.5
    close(K.attn_cache(q, prompt, pl, None, None, hq, s, rows_per_prompt=2), *attn_ref(q, pval, [45, 900, -3], [b // 2 for b in range(B)], None, None, masks, hq, s, 1))
    close(K.attn_cache(q, None, None, tail, one, hq, s), *attn_ref(q, None, None, None, tval, [11] * B, masks, hq, s, 1))
    row0 = torch.tensor([0, 3, 3, 5], dtype=torch.int32, device=dev)
    out = torch.full((B, hq * d), 7.0, device=dev, dtype=BF)
    K.attn_cache(q, prompt, pl, tail, one, hq, s, rows_per_prompt=3, row0=row0, out=out)
    close(out, *attn_ref(q, pval, [45, 900, -3], [0, 0, 0, 2, 2, None], tval, [11] * B, masks, hq, s, 1))
    far = torch.tensor([0, 33, 40, -5, 32, 31], dtype=torch.int32, device=dev)
    close(K.attn_cache(q, None, None, tail, far, hq, s), *attn_ref(q, None, None, None, tval, far.tolist(), masks, hq, s, 1))


@pytest.mark.parametrize("longest", [45, 1900])          # one launch, and two
def test_attn_cache_uneven_owners(dev, longest):
    """row0 alone: any number of sequences per prompt, none, and sequences of no prompt in front and behind."""
    hq, hkv, d, B = 7, 1, 128, 9
    prompt, pval = filled(4, longest, hkv, d, E4M3, dev, 1)
    tail, tval = filled(B, 33, hkv, d, E4M3, dev, 2)
    q = rnd((B, hq * d), 3).to(BF).to(dev)
    plen, tlen, masks = [longest, 7, 33, longest - 1], list(range(B)), [[1]] * B
    row0 = torch.tensor([1, 6, 6, 7, 8], dtype=torch.int32, device=dev)
    got = K.attn_cache(q, prompt, torch.tensor(plen, dtype=torch.int32, device=dev), tail, torch.tensor(tlen, dtype=torch.int32, device=dev), hq, d ** -0.5, row0=row0)
    close(got, *attn_ref(q, pval, plen, [None, 0, 0, 0, 0, 0, 2, 3, None], tval, tlen, masks, hq, d ** -0.5, 1))


@pytest.mark.parametrize("dtype", [BF, I8])
def test_expanded_cache(dev, dtype):
    """One sequence's rows seen as several: read like copies, refused by the writers."""
    hq, hkv, d, B = 4, 2, 64, 3
    one, val = filled(1, 40, hkv, d, dtype, dev, 1)
    shared = K.KVCache(*(None if x is None else x.expand(B, *x.shape[1:]) for x in (one.k, one.v, one.k_scale, one.v_scale)))
    k, _ = K.kv_read(shared, dtype=F32)
    assert torch.equal(k.double().cpu().transpose(1, 2), val[0].expand(B, -1, -1, -1))
    q = rnd((B, hq * d), 3).to(BF).to(dev)
    n = [3, 39, 20]
    got = K.attn_cache(q, None, None, shared, torch.tensor(n, dtype=torch.int32, device=dev), hq, 0.1)
    close(got, *attn_ref(q, None, None, None, [x.expand(B, -1, -1, -1) for x in val], n, [[1]] * B, hq, 0.1, 1))
    rows = torch.zeros(B, hkv * d, device=dev, dtype=BF)
    with pytest.raises(K.SpacerError, match="share memory"):
        K.kv_append(shared, rows, rows, torch.tensor(n, dtype=torch.int32, device=dev))
    with pytest.raises(K.SpacerError, match="share memory"):
        K.kv_write(shared, rows, rows, torch.zeros(B * 40, device=dev, dtype=torch.int32))


@pytest.mark.parametrize("dtype", [BF, E4M3, I8])
def test_attn_cache_rows_that_see_nothing(dev, dtype):
    hq, hkv, d, nodes = 4, 2, 128, 3
    tail, tval = filled(2, 8, hkv, d, dtype, dev, 2)
    q = rnd((2 * nodes, hq * d), 3).to(BF).to(dev)
    masks = [[0, 1, 0], [0, 0, 7]]
    got = K.attn_cache(q, None, None, tail, torch.tensor([0, 0], dtype=torch.int32, device=dev), hq, 0.1, nodes=nodes, tree=as_int64(masks, dev))
    want, tol = attn_ref(q, None, None, None, tval, [0, 0], masks, hq, 0.1, nodes)
    close(got, want, tol)
    for row in (0, 2, 3, 4):
        assert float(got[row].float().abs().max()) == 0.0


@pytest.mark.parametrize("dtype", [BF, E4M3, I8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("every", [2, 3, 70])            # of so many rows one is ordinary (70: the first of them), the others zero or of 2^-100
def test_attn_cache_rows_of_zeros(dev, dtype, d, every):
    """Rows of zeros and rows far below the others carry weight and add nothing."""
    hq, hkv, B, cap, nodes = 8, 2, 2, 69, 3
    tail = make_cache(B, cap, hkv, d, dtype, dev)
    size = torch.tensor([1.0 if i % every == 0 else 0.0 if i % 2 else 2.0 ** -100 for i in range(B * cap)], dtype=F64)
    k, v = rnd((B * cap, hkv * d), 5).to(BF), (rnd((B * cap, hkv * d), 6) * size[:, None]).to(BF)
    K.kv_write(tail, k.to(dev), v.to(dev), torch.arange(B * cap, dtype=torch.int32, device=dev))
    val = [x.double().cpu().transpose(1, 2) for x in K.kv_read(tail, dtype=F32)]
    q = rnd((B * nodes, hq * d), 7).to(BF).to(dev)
    tlen, masks = [66, 35], [chain(nodes)] * B
    got = K.attn_cache(q, None, None, tail, torch.tensor(tlen, dtype=torch.int32, device=dev), hq, d ** -0.5, nodes=nodes)
    close(got, *attn_ref(q, None, None, None, val, tlen, masks, hq, d ** -0.5, nodes))


@pytest.mark.parametrize("dtype", [BF, E4M3, I8])
@pytest.mark.parametrize("which", ["k", "v", "kv"])
def test_attn_cache_hidden_nonfinite(dev, dtype, which):
    """NaN and infinite rows behind the lengths reach nobody; a node's reach exactly the nodes that see it."""
    hq, hkv, d, nodes, B = 4, 2, 128, 5, 2
    tail, tval = filled(B, 60, hkv, d, dtype, dev, 2)
    tlen = [27, 40]
    bad_k, bad_v = rnd((B * 60, hkv * d), 8), rnd((B * 60, hkv * d), 9)
    if "k" in which:
        bad_k[:, 5] = math.nan
    if "v" in which:
        bad_v[:, 7], bad_v[:, 9] = math.nan, math.inf
    rows = torch.full((B, 60), -1, dtype=torch.int32)
    for b in range(B):
        rows[b, tlen[b] + nodes:] = 0
        rows[b, tlen[b] + 2] = 1                         # node 2 is poisoned
    K.kv_write(tail, bad_k.to(BF).to(dev), bad_v.to(BF).to(dev), rows.view(-1).to(dev))
    q = rnd((B * nodes, hq * d), 3).to(BF).to(dev)
    masks = [[1, 3, 5, 9, 17], [1, 2, 4, 14, 24]]        # nodes 2 (both) and 3 (second sequence) see node 2
    got = K.attn_cache(q, None, None, tail, torch.tensor(tlen, dtype=torch.int32, device=dev), hq, 0.1, nodes=nodes, tree=as_int64(masks, dev))
    clean = [x.clone() for x in tval]
    sees = torch.tensor([[m >> 2 & 1 for m in row] for row in masks]).bool().view(-1)
    want, tol = attn_ref(q, None, None, None, clean, tlen, [[m & ~4 for m in row] for row in masks], hq, 0.1, nodes)
    close(got[~sees.to(dev)], want[~sees], tol[~sees])
    poisoned = got[sees.to(dev)].view(-1, hq, d)[:, :hq // hkv].isnan()                  # the poisoned columns belong to kv head 0
    assert bool(poisoned.any(-1).all()) and (which == "v" or bool(poisoned.all()))       # (a NaN score spoils the whole row, a NaN value at least its own channel)


def test_attn_cache_far_offsets_and_spikes(dev):
    """Positions behind 2^31 bytes of one sequence's cache, and keys whose scores jump late."""
    hq, hkv, d, cap = 2, 1, 128, 300
    big = torch.zeros(cap, 8 * 1024 * 1024, device=dev, dtype=torch.uint8)               # a position every 8 MiB
    kv = [big[:, o:o + d].view(1, 1, cap, d).view(I8) for o in (0, 4096)]
    sc = [torch.ones(1, 1, cap, device=dev) for _ in range(2)]
    cache = K.KVCache(kv[0], kv[1], *sc)
    k, v = rnd((cap, d), 1).to(BF), rnd((cap, d), 2).to(BF)
    q = rnd((1, hq * d), 3).to(BF)
    k[290], k[120] = (q[0, :d].float() * 9).to(BF), (q[0, :d].float() * 4).to(BF)
    K.kv_write(cache, k.to(dev), v.to(dev), torch.arange(cap, dtype=torch.int32, device=dev))
    val = [x.double().cpu().transpose(1, 2) for x in K.kv_read(cache, dtype=F32)]
    n = torch.tensor([cap - 1], dtype=torch.int32, device=dev)
    got = K.attn_cache(q.to(dev), None, None, cache, n, hq, d ** -0.5)
    close(got, *attn_ref(q, None, None, None, val, [cap - 1], [[1]], hq, d ** -0.5, 1))


@pytest.mark.parametrize("longest", [150, 1900])         # one launch, and two with a workspace
def test_cache_step_in_graphs(dev, longest):
    """append -> attention captured twice (two graphs, own caches), replayed with lengths and inputs that change on the device, with eager work between the
    replays and on a side stream: every replay equals the eager result bit for bit."""
    hq, hkv, d, B, cap = 14, 2, 128, 6, 90
    prompt, _ = filled(2, longest, hkv, d, E4M3, dev, 1)
    pl = torch.tensor([longest, 77], dtype=torch.int32, device=dev)
    runs = []
    for i in range(2):
        tail, _ = filled(B, cap, hkv, d, E4M3, dev, 50 + i)
        st = dict(tail=tail, n=torch.zeros(B, dtype=torch.int32, device=dev), q=torch.zeros(B, hq * d, device=dev, dtype=BF),
                  k=torch.zeros(B, hkv * d, device=dev, dtype=BF), v=torch.zeros(B, hkv * d, device=dev, dtype=BF), out=torch.zeros(B, hq * d, device=dev, dtype=BF))

        def step(st=st):
            K.kv_append(st["tail"], st["k"], st["v"], st["n"])
            K.attn_cache(st["q"], prompt, pl, st["tail"], st["n"], hq, d ** -0.5, rows_per_prompt=3, out=st["out"])
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        runs.append((st, graph, step))
    side = torch.cuda.Stream()
    for it in range(4):
        for i, (st, graph, step) in enumerate(runs):
            st["n"].copy_(torch.tensor([(7 * it + 11 * b + i) % (cap - 1) for b in range(B)], dtype=torch.int32))
            for j, name in enumerate("qkv"):
                st[name].copy_(rnd(tuple(st[name].shape), 1000 * it + 10 * i + j).to(BF))
        for st, graph, _ in runs:
            graph.replay()
        got = [st["out"].clone() for st, _, _ in runs]
        torch.cuda.synchronize()
        for (st, _, step), g in zip(runs, got):
            st["out"].zero_()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            assert torch.equal(st["out"], g)


# ------------------------------------------------------------------------------------------------------------- logits
def unpack(words, vocab):
    at = torch.arange(vocab)
    return ((words.cpu().long()[..., at // 32] >> (at % 32)) & 1).bool()


def pack(bits):
    n = bits.shape[-1]
    wide = torch.zeros(*bits.shape[:-1], (n + 31) // 32 * 32, dtype=torch.int64)
    wide[..., :n] = bits
    w = (wide.view(*bits.shape[:-1], -1, 32) << torch.arange(32)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()


def logits_ref(x, seen, counts, rep, freq, pres, bias, mask):
    x = x.double().clone()
    x = torch.where(seen, torch.where(x > 0, x / rep[:, None], x * rep[:, None]), x)
    x = x - freq[:, None] * counts - pres[:, None] * (counts > 0)
    if bias is not None:
        x = x + bias.double()
    return x.float().masked_fill(~mask, -math.inf)


@pytest.mark.parametrize("vocab", [1, 31, 33, 1000, 1022, 4096 + 7, 151936])
@pytest.mark.parametrize("B", [1, 5])
def test_process_logits(dev, vocab, B):
    g = torch.Generator().manual_seed(vocab + B)
    n = 40
    prompt = torch.randint(-3, vocab + 3, (B, n), generator=g)
    comp = torch.randint(0, vocab, (B, n), generator=g)
    comp[:, ::3] = comp[:, :1]                            # a token that repeats
    lens = torch.randint(0, n + 1, (B,), generator=g).int()
    seen, counts = K.token_history(B, vocab, dev)
    K.token_history_add_(seen, None, prompt.to(dev), vocab=vocab)
    K.token_history_add_(seen, counts, comp.to(dev), lens.to(dev))
    want_c, want_s = torch.zeros(B, vocab, dtype=torch.int32), torch.zeros(B, vocab, dtype=torch.bool)
    for b in range(B):
        for t in prompt[b].tolist():
            if 0 <= t < vocab:
                want_s[b, t] = True
        for t in comp[b, :int(lens[b])].tolist():
            want_s[b, t] = True
            want_c[b, t] += 1
    assert torch.equal(counts.cpu(), want_c) and torch.equal(unpack(seen, vocab), want_s)

    x = (4 * torch.randn(B, vocab, generator=g)).float()
    x[0, 0], x[0, vocab // 2], x[-1, vocab - 1] = math.inf, -math.inf, math.nan
    rep, freq, pres = 0.5 + torch.rand(B, generator=g), torch.rand(B, generator=g), torch.rand(B, generator=g)
    table = torch.rand(3, vocab, generator=g) < 0.6
    table[1] = False                                      # a state that allows nothing
    pick = torch.randint(-1, 4, (B,), generator=g).int()
    mask = torch.stack([table[int(p)] if 0 <= p < 3 else torch.ones(vocab, dtype=torch.bool) for p in pick])
    every = torch.ones(B, vocab, dtype=torch.bool)
    rows = torch.randn(B, vocab, generator=g)
    z = torch.zeros(B, dtype=F64)
    o = torch.ones(B, dtype=F64)
    cases = [
        (dict(), logits_ref(x, want_s, want_c, o, z, z, None, every)),
        (dict(repetition=1.3), logits_ref(x, want_s, want_c, o * float(torch.tensor(1.3)), z, z, None, every)),
        (dict(repetition=rep.to(dev), counts=counts, frequency=freq.to(dev), presence=pres.to(dev)), logits_ref(x, want_s, want_c, rep.double(), freq.double(), pres.double(), None, every)),
        (dict(bias=rows[0].to(dev)), logits_ref(x, want_s, want_c, o, z, z, rows[0], every)),
        (dict(allowed=pack(table).to(dev), allowed_row=pick.to(dev)), logits_ref(x, want_s, want_c, o, z, z, None, mask)),
        (dict(repetition=rep.to(dev), counts=counts, frequency=0.25, presence=-0.5, bias=rows.to(dev), allowed=pack(mask).to(dev)),
         logits_ref(x, want_s, want_c, rep.double(), z + 0.25, z - 0.5, rows, mask)),
        (dict(allowed=pack(table[:1]).to(dev)), logits_ref(x, want_s, want_c, o, z, z, None, table[:1].expand(B, -1))),
    ]
    for kw, want in cases:
        for pad in (0, 5):                                # rows at multiples of 16 bytes where the vocabulary allows it, and not
            wide = torch.full((B, (vocab + 3) // 4 * 4 + pad), 99.0, device=dev)
            view = wide[:, :vocab]
            view.copy_(x)
            out = torch.full_like(wide, 55.0)
            got = K.process_logits(view, seen=seen, out=out[:, :vocab], **kw)
            # one rounding of a 64-bit value on both sides (fma or not differs below 2^-52): at most the neighbouring fp32 number where that value is next to a tie
            ok = (got.cpu() == want) | (got.cpu().isnan() & want.isnan()) | ((got.cpu().double() - want.double()).abs() <= 2.0 ** -23 * want.double().abs())
            assert ok.all(), (kw.keys(), pad)
            assert same(view, x) and bool((out[:, vocab:] == 55.0).all()) and bool((wide[:, vocab:] == 99.0).all())
            inp = K.process_logits(view, seen=seen, **kw)
            assert inp is view and same(view, got) and bool((wide[:, vocab:] == 99.0).all())


@pytest.mark.parametrize("B,n,vocab", [(1, 1, 1), (2, 300, 70), (3, 40000, 1000), (130, 1030, 33), (1, 100001, 152064), (1, 100001, 600000)])
@pytest.mark.parametrize("kind", ["any", "one", "two"])
def test_token_history(dev, B, n, vocab, kind):
    """Runs of one id, ids that alternate, ids outside the vocabulary, rows of every length, a second call on top; rows that share the ids."""
    g = torch.Generator().manual_seed(n + vocab)
    ids = torch.randint(-2, vocab + 2, (B, n), generator=g)
    if kind != "any":
        ids[:, n // 8:] = torch.tensor([vocab // 2, vocab // 2 if kind == "one" else vocab - 1]).repeat(n)[:n - n // 8]
    lens = torch.tensor([n, 0, n + 7, n // 2, -1]).repeat(B)[:B].int()
    seen, counts = K.token_history(B, vocab, dev)
    K.token_history_add_(seen, counts, ids.to(dev), lens.to(dev))
    want = torch.stack([torch.bincount(r[:max(int(m), 0)].clamp(-1, vocab) + 1, minlength=vocab + 2)[1:-1] for r, m in zip(ids, lens)])
    assert torch.equal(counts.cpu().long(), want) and torch.equal(unpack(seen, vocab), want > 0)
    marked = seen.clone()
    K.token_history_add_(marked, None, ids[0].to(dev).expand(B, -1), vocab=vocab)
    first = torch.bincount(ids[0].clamp(-1, vocab) + 1, minlength=vocab + 2)[1:-1]
    assert torch.equal(unpack(marked, vocab), (want + first) > 0) and torch.equal(counts.cpu().long(), want)
    K.token_history_add_(seen, counts, ids.to(dev))
    want = want + torch.stack([torch.bincount(r.clamp(-1, vocab) + 1, minlength=vocab + 2)[1:-1] for r in ids])
    assert torch.equal(counts.cpu().long(), want) and torch.equal(unpack(seen, vocab), want > 0)


def test_sampler_draws_what_the_mask_allows(dev):
    """history -> logits -> sampler, as a decode step runs them: greedy picks the best allowed token that the penalties leave."""
    B, vocab = 4, 2048
    x = rnd((B, vocab), 5).float().to(dev)
    seen, counts = K.token_history(B, vocab, dev)
    step = torch.zeros(1, dtype=torch.int32, device=dev)
    allowed = torch.zeros(1, vocab, dtype=torch.bool)
    allowed[0, 100:200] = True
    drawn = []
    for i in range(5):
        logits = K.process_logits(x, seen=seen, counts=counts, presence=1000.0, allowed=pack(allowed).to(dev), out=torch.empty_like(x))
        ids = K.sample_top_p(logits, step, top_k=1, top_p=1.0, seed=1)
        K.token_history_add_(seen, counts, ids[:, None])
        drawn.append(ids.cpu())
    order = torch.argsort(x.cpu()[:, 100:200], dim=1, descending=True)[:, :5] + 100
    assert torch.equal(torch.stack(drawn, 1), order)


@pytest.mark.parametrize("n", [1, 2, 49, 50, 700, 5000])
@pytest.mark.parametrize("wide", [False, True])
def test_sampler_with_few_allowed_tokens(dev, n, wide):
    """A mask that leaves fewer tokens than top_k of a large vocabulary: the draw is the one from these tokens alone (same order, same numbers, same uniform)."""
    B, vocab = 8, 151936
    x = rnd((B, vocab), 15).float().to(dev)
    ids = torch.randperm(vocab, generator=torch.Generator().manual_seed(n))[:n].sort().values
    allowed = torch.zeros(1, vocab, dtype=torch.bool)
    allowed[0, ids] = True
    logits = K.process_logits(x, allowed=pack(allowed).to(dev), out=torch.empty_like(x))
    alone = x[:, ids.to(dev)].contiguous()
    ws = K.sample_workspace(B, vocab, dev) if wide else None
    for step in range(4):
        at = torch.tensor([step], dtype=torch.int32, device=dev)
        for top_k, top_p in ((1, 1.0), (50, 0.9), (50, 1.0)):
            got = K.sample_top_p(logits, at, top_k=top_k, top_p=top_p, seed=3, workspace=ws)
            want = K.sample_top_p(alone, at, top_k=min(top_k, n), top_p=top_p, seed=3)
            assert torch.equal(ids.to(dev)[want], got), (step, top_k, top_p)


def test_sampler_where_nothing_is_allowed(dev):
    """All of a row forbidden: some token of the vocabulary, beside rows that are not disturbed."""
    B, vocab = 4, 151936
    x = rnd((B, vocab), 15).float().to(dev)
    allowed = torch.ones(B, vocab, dtype=torch.bool)
    allowed[1] = False
    logits = K.process_logits(x, allowed=pack(allowed).to(dev), out=torch.empty_like(x))
    at = torch.zeros(1, dtype=torch.int32, device=dev)
    for ws in (None, K.sample_workspace(B, vocab, dev)):
        got, want = K.sample_top_p(logits, at, seed=3, workspace=ws), K.sample_top_p(x, at, seed=3)
        assert torch.equal(got[[0, 2, 3]], want[[0, 2, 3]]) and 0 <= int(got[1]) < vocab
