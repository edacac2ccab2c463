"""attn_cache where numbers stop being finite and where callers leave the ordinary layouts, in the one-launch form (short capacities) and in the two-launch
one, whose key ranges meet in a second kernel.  Both have to give the definition's answer: the launch is chosen by capacities, not by the data.
Reference and tolerances: test_cache_ops_gpu.attn_ref."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from spacer_amd import kernels as K        # noqa: E402
from test_cache_ops_gpu import BF, E4M3, F32, I8, attn_ref, close, filled, make_cache, rnd  # noqa: E402

FORMATS = [BF, E4M3, I8]
LONGEST = [45, 1900]                       # prompt capacities: one launch, two launches


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def forms(prompt, tail, rows, B, hq, longest):
    """The capacities take the form that the case is about."""
    assert (K.attn_cache_workspace_bytes(prompt, tail, rows, B, 1, hq) > 0) == (longest == LONGEST[1])


def poison(cache, which, seq, head, positions):
    """The rows of one kv head become what the writers make of a row with a NaN: scale NaN and codes 0, in bf16 the row itself with a NaN in it."""
    for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        if (x is cache.k) == (which == "k"):
            if s is None:
                x[seq, head, positions, 5] = math.nan
            else:
                s[seq, head, positions] = math.nan
                x.view(torch.uint8)[seq, head, positions] = 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("longest", LONGEST)
def test_nan_query(dev, dtype, d, longest):
    """A query head with a NaN gives NaN, wherever its keys lie; the others what they gave."""
    hq, hkv, B = 12, 2, 4
    prompt, pval = filled(2, longest, hkv, d, dtype, dev, 1)
    tail, tval = filled(B, 40, hkv, d, dtype, dev, 2)
    forms(prompt, tail, 2, B, hq, longest)
    q = rnd((B, hq, d), 3).to(BF)
    bad = torch.zeros(B, hq, dtype=torch.bool)
    for b, h in ((0, 0), (1, 11), (3, 5)):
        q[b, h, 7 + h] = math.nan
        bad[b, h] = True
    plen, tlen = [longest, longest // 2], [0, 3, 39, 17]
    got = K.attn_cache(q.view(B, -1).to(dev), prompt, i32(plen, dev), tail, i32(tlen, dev), hq, d ** -0.5, rows_per_prompt=2).view(B, hq, d)
    want, tol = attn_ref(torch.where(bad[..., None], 0.0, q).view(B, -1), pval, plen, [0, 0, 1, 1], tval, tlen, [[1]] * B, hq, d ** -0.5, 1)
    assert bool(got[bad.to(dev)].isnan().all())
    close(got[~bad.to(dev)], want.view(B, hq, d)[~bad], tol.view(B, hq, d)[~bad])


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("longest", LONGEST)
@pytest.mark.parametrize("part", ["prompt", "own", "one of the prompt"])
def test_nan_rows_of_a_whole_range(dev, dtype, which, longest, part):
    """NaN rows reach every column that sees them, also where they are all that a range of keys holds (a rollout's first own token, a whole prompt)."""
    hq, hkv, d, B = 8, 2, 128, 4
    prompt, pval = filled(2, longest, hkv, d, dtype, dev, 1)
    tail, tval = filled(B, 40, hkv, d, dtype, dev, 2)
    forms(prompt, tail, 2, B, hq, longest)
    plen, tlen = [longest, longest - 5], [0, 0, 3, 39]
    bad = torch.zeros(B, hq, dtype=torch.bool)
    if part == "own":
        poison(tail, which, 1, 0, slice(0, 1))
        bad[1, :4] = True
    else:
        poison(prompt, which, 1, 1, slice(0, longest) if part == "prompt" else slice(longest // 2, longest // 2 + 1))
        bad[2:, 4:] = True
    q = rnd((B, hq * d), 3).to(BF)
    got = K.attn_cache(q.to(dev), prompt, i32(plen, dev), tail, i32(tlen, dev), hq, d ** -0.5, rows_per_prompt=2).view(B, hq, d)
    want, tol = attn_ref(q, pval, plen, [0, 0, 1, 1], tval, tlen, [[1]] * B, hq, d ** -0.5, 1)      # (values read before the rows were spoiled)
    close(got[~bad.to(dev)], want.view(B, hq, d)[~bad], tol.view(B, hq, d)[~bad])
    hit = got[bad.to(dev)].isnan()
    if which == "v" and dtype == BF:                      # a NaN number of a value row is one channel's
        assert bool(hit[:, 5].all()) and not bool(hit[:, :5].any()) and not bool(hit[:, 6:].any())
    else:
        assert bool(hit.all())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("longest", LONGEST)
@pytest.mark.parametrize("first", [0, 64])
def test_scores_of_minus_infinity(dev, d, longest, first):
    """Keys whose score is -infinity weigh nothing, also where a wave meets nothing else in its first tiles."""
    hq, hkv, B, n = 8, 2, 4, 32 if longest == LONGEST[0] else 640
    prompt, pval = filled(2, longest, hkv, d, BF, dev, 1)
    tail, tval = filled(B, 40, hkv, d, BF, dev, 2)
    forms(prompt, tail, 2, B, hq, longest)
    first = min(first, longest - n)
    q = rnd((B, hq, d), 3).to(BF)
    q[..., 9] = q[..., 9].abs() + 0.5
    prompt.k[:, :, first:first + n, 9] = -math.inf
    plen, tlen = [longest, longest], [0, 3, 39, 17]
    keep = [i for i in range(longest) if not first <= i < first + n]
    want = attn_ref(q.view(B, -1), [x[:, :, keep] for x in pval], [len(keep)] * 2, [0, 0, 1, 1], tval, tlen, [[1]] * B, hq, d ** -0.5, 1)
    close(K.attn_cache(q.view(B, -1).to(dev), prompt, i32(plen, dev), tail, i32(tlen, dev), hq, d ** -0.5, rows_per_prompt=2), *want)


@pytest.mark.parametrize("dtype", FORMATS)
@pytest.mark.parametrize("longest", LONGEST)
@pytest.mark.parametrize("rows", [1, 2, 5])
def test_prompts_of_more_sequences_than_rows_per_prompt(dev, dtype, longest, rows):
    """With row0 the number of sequences per prompt is row0's: rows_per_prompt only says what to launch for."""
    hq, hkv, d, B, nodes = 14, 2, 128, 14, 2
    prompt, pval = filled(4, longest, hkv, d, dtype, dev, 1)
    tail, tval = filled(B, 40, hkv, d, dtype, dev, 2)
    forms(prompt, tail, rows, B, hq, longest)
    row0 = [1, 6, 6, 13, 14]
    owner = [None] + [0] * 5 + [2] * 7 + [3]
    plen, tlen = [longest, 7, 33, longest - 1], [2 * b for b in range(B)]
    q = rnd((B * nodes, hq * d), 3).to(BF).to(dev)
    n = K.attn_cache_workspace_bytes(prompt, tail, rows, B, nodes, hq)
    ws = torch.full((n,), 0x7F, dtype=torch.uint8, device=dev)              # what nobody wrote is huge
    got = K.attn_cache(q, prompt, i32(plen, dev), tail, i32(tlen, dev), hq, d ** -0.5, rows_per_prompt=rows, row0=i32(row0, dev), nodes=nodes, workspace=ws)
    close(got, *attn_ref(q, pval, plen, owner, tval, tlen, [[1, 3]] * B, hq, d ** -0.5, nodes))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("scale", [3.0, -2.0, 2.0 ** -130, 0.3])
@pytest.mark.parametrize("longest", LONGEST)
def test_e4m3_scales_that_are_no_powers_of_two(dev, d, which, scale, longest):
    """attn_cache takes e4m3 scales by their exponents: any other number in a row that is seen gives NaN and nobody else is touched; 0 is the scale of a row of zeros."""
    hq, hkv, B = 8, 2, 4
    prompt, pval = filled(2, longest, hkv, d, E4M3, dev, 1)
    tail, tval = filled(B, 40, hkv, d, E4M3, dev, 2)
    s = dict(k=(prompt.k_scale, tail.k_scale), v=(prompt.v_scale, tail.v_scale))[which]
    s[0][1, 1, 33] = scale                                # a key of the second prompt, kv head 1
    s[1][0, 0, 5] = scale                                 # the newest key of the first sequence, kv head 0
    s[1][1, :, 6:] = scale                                # behind the newest key of the second: nobody's
    for x, t in ((tail.k, tail.k_scale), (tail.v, tail.v_scale)):
        x.view(torch.uint8)[2, 0, 1] = 0
        t[2, 0, 1] = 0.0
    tval = [x.clone() for x in tval]
    for x in tval:
        x[2, 0, 1] = 0.0
    bad = torch.zeros(B, hq, dtype=torch.bool)
    bad[2:, 4:] = True
    bad[0, :4] = True
    q = rnd((B, hq * d), 3).to(BF)
    plen, tlen = [longest, longest], [5, 5, 3, 39]
    got = K.attn_cache(q.to(dev), prompt, i32(plen, dev), tail, i32(tlen, dev), hq, d ** -0.5, rows_per_prompt=2).view(B, hq, d)
    want, tol = attn_ref(q, pval, plen, [0, 0, 1, 1], tval, tlen, [[1]] * B, hq, d ** -0.5, 1)
    close(got[~bad.to(dev)], want.view(B, hq, d)[~bad], tol.view(B, hq, d)[~bad])
    assert bool(got[bad.to(dev)].isnan().all())
    if which == "k" and scale > 1:                        # a hidden node's own
        nodes = 3
        q = rnd((B * nodes, hq * d), 4).to(BF)
        s[1][:, :, 20] = scale
        masks = [[1, 1, 5]] * B
        tree = torch.tensor(masks[0], dtype=torch.int64, device=dev)
        got = K.attn_cache(q.to(dev), None, None, tail, i32([19] * B, dev), hq, d ** -0.5, nodes=nodes, tree=tree).view(B * nodes, hq, d)
        want, tol = attn_ref(q, None, None, None, tval, [19] * B, masks, hq, d ** -0.5, nodes)
        fine = torch.ones(B, nodes, hq, dtype=torch.bool)
        fine[0, :, :4] = False                            # (position 5 of the first sequence)
        fine[1] = False                                   # (positions from 6 on of the second)
        fine = fine.view(B * nodes, hq)
        close(got[fine.to(dev)], want.view(B * nodes, hq, d)[fine], tol.view(B * nodes, hq, d)[fine])
