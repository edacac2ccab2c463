"""NaN logits at the sampler: they count as forbidden, whatever their sign, and a row of nothing else still gives a token of the vocabulary."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from spacer_amd import kernels as K        # noqa: E402

F32 = torch.float32


def signed_nan(negative):
    """A NaN with the sign bit as asked for (arithmetic on the host makes either)."""
    return torch.tensor([0xFFC00000 - 2 ** 32 if negative else 0x7FC00000], dtype=torch.int32).view(F32)


def logits(B, vocab, seed=15):
    return torch.randn(B, vocab, generator=torch.Generator().manual_seed(seed)) * 2


def workspaces(B, vocab, dev):
    return [None, K.sample_workspace(B, vocab, dev)]


@pytest.mark.parametrize("vocab", [1, 7, 50, 1024, 1025, 151936])
@pytest.mark.parametrize("negative", [False, True])
def test_rows_of_nan(dev, vocab, negative):
    B = 4
    x = logits(B, vocab).to(dev)
    x[1], x[3] = signed_nan(negative).to(dev), signed_nan(negative).to(dev)
    x[3, ::2] = -math.inf                                 # ... beside forbidden ones
    at = torch.zeros(1, dtype=torch.int32, device=dev)
    clean = torch.where(x.isnan(), -math.inf, x)
    for top_k in {1, min(50, vocab)}:
        for ws in workspaces(B, vocab, dev):
            got = K.sample_top_p(x, at, top_k=top_k, seed=3, workspace=ws).cpu()
            assert bool(((got >= 0) & (got < vocab)).all())
            assert torch.equal(got[[0, 2]], K.sample_top_p(clean, at, top_k=top_k, seed=3, workspace=ws).cpu()[[0, 2]])
            mat, ids = torch.full((B, 2), -1, dtype=torch.int64, device=dev), torch.empty(B, dtype=torch.int64, device=dev)
            K.sample_top_p_step(x, at, 1, mat, top_k=top_k, seed=3, suppress_eos=vocab > 1, eos_id=0, out_ids=ids, workspace=ws)
            assert torch.equal(mat[:, 1], ids) and bool(((ids >= 0) & (ids < vocab)).all()) and bool((mat[:, 0] == -1).all())


@pytest.mark.parametrize("vocab", [60, 1024, 4097, 151936])
@pytest.mark.parametrize("share", [1, 3, 40])             # NaN: one logit, every third, all but every fortieth
@pytest.mark.parametrize("negative", [False, True])
def test_nan_among_logits(dev, vocab, share, negative):
    """The draw and its log-probability are those of the same row with -infinity in the NaN's places, bit for bit."""
    B = 8
    x = logits(B, vocab).to(dev)
    where = torch.zeros(B, vocab, dtype=torch.bool)
    if share == 1:
        where[torch.arange(B), torch.randint(0, vocab, (B,), generator=torch.Generator().manual_seed(1))] = True
    elif share == 3:
        where[:, ::3] = True
    else:
        where[:] = True
        where[:, 5::40] = False
    clean = x.masked_fill(where.to(dev), -math.inf)
    x = torch.where(where.to(dev), signed_nan(negative).to(dev), x)
    for step in range(3):
        at = torch.tensor([step], dtype=torch.int32, device=dev)
        for top_k, top_p in ((1, 1.0), (50, 0.9), (50, 1.0)):
            for ws in workspaces(B, vocab, dev):
                out = []
                for row in (x, clean):
                    logp = torch.zeros(B, device=dev)
                    out.append((K.sample_top_p(row, at, top_k=top_k, top_p=top_p, seed=3, out_logp=logp, workspace=ws), logp))
                assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
                assert not bool(where[torch.arange(B), out[0][0].cpu()].any())


@pytest.mark.parametrize("wide", [False, True])
def test_edge_of_the_draw_with_log_probabilities(dev, wide):
    """Rows whose draw no candidate's interval takes (sums that are no numbers: an infinite logit, nothing allowed) beside ordinary ones, with the pass for the
    log-probability behind them: the infinite logit is drawn, ordinary rows are not disturbed."""
    B, vocab = 64, 151936
    x = logits(B, vocab).to(dev)
    clean = x.clone()
    x[::4, 777] = math.inf
    x[1::4] = -math.inf
    at = torch.zeros(1, dtype=torch.int32, device=dev)
    ws = K.sample_workspace(B, vocab, dev) if wide else None
    want_p = torch.zeros(B, device=dev)
    want = K.sample_top_p(clean, at, seed=3, out_logp=want_p, workspace=ws)
    for _ in range(4):
        logp = torch.zeros(B, device=dev)
        got = K.sample_top_p(x, at, seed=3, out_logp=logp, workspace=ws)
        for r in (2, 3):
            assert torch.equal(got[r::4], want[r::4]) and torch.equal(logp[r::4], want_p[r::4])
        assert bool((got[::4] == 777).all()) and bool(logp[::4].isnan().all()) and bool(logp[1::4].isnan().all())
        assert bool(((got >= 0) & (got < vocab)).all())
