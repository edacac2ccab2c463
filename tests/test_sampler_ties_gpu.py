"""Ties of the top_k-th logit beyond the sampler's candidate list (1024): those of the lowest indices are kept, whatever the order of a launch's waves."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from spacer_amd import kernels as K        # noqa: E402

CAP = 1024


@pytest.mark.parametrize("vocab", [1025, 4099, 152064])
@pytest.mark.parametrize("above", [0, 1, 30])
@pytest.mark.parametrize("kind", ["some", "all", "forbidden"])
def test_ties_beyond_the_list(dev, vocab, above, kind):
    """The draw is the one from the logits above and the lowest-numbered ties alone (same order, same numbers, same uniform), in every one of several launches of both
    forms.  "some": the ties lie among smaller logits; "all": every other logit is a tie; "forbidden": the others are -infinity."""
    B = 12
    g = torch.Generator().manual_seed(vocab + above)
    x = torch.randn(B, vocab, generator=g)
    if kind != "some":
        x[:] = 3.0 if kind == "all" else -math.inf
    alone, ids = torch.full((B, CAP), -math.inf), torch.zeros(B, CAP, dtype=torch.int64)
    for b in range(B):
        order = torch.randperm(vocab, generator=g)
        top, ties = order[:above], order[above:] if kind == "all" else order[above:above + min(2000, vocab - above)]
        x[b, ties] = 3.0 if kind == "all" else 11.0
        x[b, top] = 11.5 + torch.rand(above, generator=g)
        keep = torch.cat([top, ties.sort().values[:CAP - above]]).sort().values
        ids[b, :keep.numel()] = keep
        alone[b, :keep.numel()] = x[b, keep]
    x, alone, ids = x.to(dev), alone.to(dev), ids.to(dev)
    for step in range(2):
        at = torch.tensor([step], dtype=torch.int32, device=dev)
        for top_k, top_p, temperature in ((above + 1, 1.0, 1.0), (50, 0.9, 0.7), (CAP, 1.0, 1.0)):
            want = ids.gather(1, K.sample_top_p(alone, at, top_k=top_k, top_p=top_p, temperature=temperature, seed=3)[:, None])[:, 0]
            for ws in (None, K.sample_workspace(B, vocab, dev)) * 3:
                assert torch.equal(K.sample_top_p(x, at, top_k=top_k, top_p=top_p, temperature=temperature, seed=3, workspace=ws), want), (step, top_k)


def test_nothing_allowed_gives_the_first_token(dev):
    """All ties of -infinity: the lowest index, every time."""
    B, vocab = 9, 151936
    x = torch.full((B, vocab), -math.inf, device=dev)
    at = torch.zeros(1, dtype=torch.int32, device=dev)
    for ws in (None, K.sample_workspace(B, vocab, dev)) * 3:
        assert bool((K.sample_top_p(x, at, seed=3, workspace=ws) == 0).all())
