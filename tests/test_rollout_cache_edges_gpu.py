"""8-bit rollouts: what the caches may hold where nothing has been written, and every cache call of a decode loop against the definition."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from spacer_amd import kernels as K                    # noqa: E402
from spacer_amd import rollout as R                    # noqa: E402
from spacer_amd.qwen2vl.config import TINY             # noqa: E402
from spacer_amd.rollout import SamplingParams          # noqa: E402
from test_rollout_cache_gpu import engine, tiny        # noqa: E402, F401


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("Kn", [3, [4, 2]])
def test_unwritten_slots_may_hold_anything(tiny, dev, monkeypatch, fmt, Kn):           # noqa: F811
    """Prompts of two lengths: caches that start as NaN codes and NaN scales give the tokens that cleared ones give, and the prompts' are not cleared."""
    monkeypatch.setattr(K.PLAN, "skinny_blocks", 1)
    sp = SamplingParams(max_new_tokens=9, top_k=20, top_p=0.95, seed=4, suppress_eos=True, kv_cache=fmt)
    plain, cleared = R._LayerCaches.__init__, []

    def filled(with_nan):
        def init(self, *args, clear=True):
            plain(self, *args, clear=clear)
            cleared.append(clear)
            for x in self.codes:
                x.view(torch.uint8).fill_(0x7F if with_nan else 0)
            for x in self.scales:
                x.fill_(float("nan") if with_nan else 0.0)
        return init
    out = []
    for with_nan in (False, True):
        monkeypatch.setattr(R._LayerCaches, "__init__", filled(with_nan))
        out.append(engine(tiny).generate(tiny["prompts"], Kn, sp))
    assert torch.equal(*out) and cleared == [False, True] * 2
