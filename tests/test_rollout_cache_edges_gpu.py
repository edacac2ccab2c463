"""8-bit rollouts: what the caches may hold where nothing has been written, and every cache call of a decode loop against the definition."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from spacer_amd import kernels as K                    # noqa: E402
from spacer_amd import rollout as R                    # noqa: E402
from spacer_amd.qwen2vl.config import TINY             # noqa: E402
from spacer_amd.rollout import SamplingParams          # noqa: E402
from test_cache_ops_gpu import F32, attn_ref, close     # noqa: E402
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


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("Kn", [1, 3, [4, 2]])
def test_decode_loop_against_the_definition(tiny, dev, monkeypatch, fmt, Kn):          # noqa: F811
    """A decode loop, call by call.  Attention of every step and layer is the definition over the values that the caches hold, with owners, prompt lengths and
    positions counted here (bounds: test_cache_ops_gpu).  What the first layer's own cache holds (it depends on the tokens alone) is the bf16 loop's row of
    the same token at the same position, rounded once: e4m3 within 2^-4 |x| (codes below the normal ones 2^-10 scale, scale < max|x| / 224), int8 within
    max|x| / 254, of a bf16 number that may be one step of 2^-7 |x| away (the two writers are compiled with different contraction), with 2^-17 max|x| for
    the rotary's cancellation."""
    monkeypatch.setattr(K.PLAN, "skinny_blocks", 1)
    C, L = 9, TINY.layers
    counts = [Kn, Kn] if isinstance(Kn, int) else Kn
    B, plens = sum(counts), [p.ids.numel() for p in tiny["prompts"]]
    owner = [p for p, k in enumerate(counts) for _ in range(k)]
    sp = dict(max_new_tokens=C, top_k=20, top_p=0.95, seed=5, suppress_eos=True)
    attn, calls, tails = K.attn_cache, [], {}

    def values(cache):
        return [x.double().cpu().transpose(1, 2) for x in K.kv_read(cache, dtype=F32)]

    def checked(q, prompt, plen, tail, tlen, hq, scale, **kw):
        out = attn(q, prompt, plen, tail, tlen, hq, scale, **kw)
        step, layer = divmod(len(calls), L)
        close(out, *attn_ref(q, values(prompt), plens, owner, values(tail), [step] * B, [[1]] * B, hq, scale, 1), what=f"token {step + 1}, layer {layer}")
        calls.append(layer)
        if layer == 0:
            tails["narrow"] = tail
        return out
    with monkeypatch.context() as m:
        m.setattr(K, "attn_cache", checked)
        tokens = engine(tiny).generate(tiny["prompts"], Kn, SamplingParams(**sp, kv_cache=fmt), use_graph=False)
    assert len(calls) == (C - 1) * L
    # the same tokens through bf16 caches
    draw, finish = K.sample_top_p_step, (K.decode_qkv_finish, K.decode_qkv_finish_normed)
    drawn = []

    def forced(*args, **kw):
        draw(*args, **kw)
        kw["out_ids"].copy_(tokens[:, len(drawn)])
        drawn.append(0)
        return kw["out_ids"]

    def recorded(f):
        def call(acc, bias, cos, sin, q, tk, tv, *rest):
            f(acc, bias, cos, sin, q, tk, tv, *rest)
            tails.setdefault("wide", (tk, tv))
        return call
    with monkeypatch.context() as m:
        m.setattr(K, "sample_top_p_step", forced)
        for f in finish:
            m.setattr(K, f.__name__, recorded(f))
        engine(tiny).generate(tiny["prompts"], Kn, SamplingParams(**sp), use_graph=False)
    assert len(drawn) == C
    for got, want in zip(K.kv_read(tails["narrow"], dtype=F32), tails["wide"]):
        got, want = got[:, :C - 1].double().cpu(), want[:, :C - 1].double().cpu()
        top = want.abs().amax(-1, keepdim=True)
        assert float(top.min()) > 0
        x = want.abs() * (1 + 2.0 ** -7)
        step = torch.maximum(2.0 ** -4 * x, 2.0 ** -10 * top / 224) if fmt == "e4m3" else top * (1 + 2.0 ** -7) / 254
        close(got, want, step + 2.0 ** -7 * want.abs() + 2.0 ** -17 * top)
