"""Rollouts over 8-bit key/value caches and with logits rules: the cache and logits operators as RolloutEngine uses them, and a drafted tree verified in
one pass against the same tokens decoded one by one."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from golden_util import load_tiny                      # noqa: E402
from oracle import qwen2vl_fp32 as O                   # noqa: E402
from spacer_amd import kernels as K                    # noqa: E402
from spacer_amd.qwen2vl.config import TINY             # noqa: E402
from spacer_amd.qwen2vl.engine import Qwen2VLEngine    # noqa: E402
from spacer_amd.qwen2vl.weights import FlatParams, export_state_dict, load_state_dict  # noqa: E402
from spacer_amd.rollout import PromptInput, RolloutEngine, SamplingParams  # noqa: E402
from test_cache_ops_gpu import as_int64, attn_ref, filled, rnd  # noqa: E402

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def tiny(dev):
    g = load_tiny()
    params = FlatParams.empty(TINY, dev)
    load_state_dict(params, g["w"])
    wb = {k: v.float().cpu() for k, v in export_state_dict(params).items()}
    wb["visual.patch_embed.proj.weight"] = wb["visual.patch_embed.proj.weight"].reshape(TINY.vit_dim, -1)
    pix, grid = K.patchify(g["frames"].to(dev), kpad=TINY.patch_kpad)
    rows, _ = O.patchify_frames(g["frames"], g["cfg"])
    prompts = [PromptInput(g["prompt"].to(dev), pix, [tuple(grid)]), PromptInput(g["prompt"][-9:].to(dev), None, None)]
    return dict(g=g, params=params, wb=wb, prompts=prompts, rows=rows.to(BF).float(), grid=tuple(grid))


def engine(tiny):
    return RolloutEngine(Qwen2VLEngine(TINY, tiny["params"]))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("Kn", [1, 3, 12, [4, 2]])
def test_rollout_on_8bit_caches(tiny, dev, monkeypatch, fmt, Kn):
    """eager == graph bit for bit; greedy tokens are the oracle's arg-max within the bf16 path's budget (3e-2 for numbers rounded by 2^-8) times the
    coarser rounding of K and V: e4m3 2^-4 = 16 * 2^-8; int8 half a step is max / 254, at 4 standard deviations 4 * 2^-8 of an ordinary number."""
    monkeypatch.setattr(K.PLAN, "skinny_blocks", 1)
    roll = engine(tiny)
    sp = SamplingParams(max_new_tokens=9, top_k=1, top_p=1.0, suppress_eos=True, kv_cache=fmt)
    a = roll.generate(tiny["prompts"], Kn, sp, use_graph=False)
    st = {}
    b = roll.generate(tiny["prompts"], Kn, sp, use_graph=True, stats=st)
    assert st["graph"] and torch.equal(a, b)
    counts = [Kn, Kn] if isinstance(Kn, int) else Kn
    assert a.shape == (sum(counts), 9)
    assert all(torch.equal(a[0], a[i]) for i in range(counts[0])) and all(torch.equal(a[counts[0]], a[counts[0] + i]) for i in range(counts[1]))
    g, budget = tiny["g"], 3e-2 * (1 + (16 if fmt == "e4m3" else 4))
    for row, (pids, rows, grids) in ((0, (g["prompt"], tiny["rows"], [tiny["grid"]])), (counts[0], (g["prompt"][-9:], None, None))):
        comp = a[row].cpu()
        lg = O.full_logits(tiny["wb"], g["cfg"], torch.cat([pids, comp]), rows, grids)
        for t in range(9):
            x = lg[pids.numel() - 1 + t].clone()
            x[TINY.eos_token_id] = float("-inf")
            assert float(x.max() - x[comp[t]]) < budget, (row, t)
    # the first token never reads the cache: the same as with a bf16 cache
    c = roll.generate(tiny["prompts"], Kn, SamplingParams(max_new_tokens=9, top_k=1, top_p=1.0, suppress_eos=True), use_graph=False)
    assert torch.equal(a[:, 0], c[:, 0])


def test_8bit_prefill_beside_a_kept_tape(tiny, dev):
    """The prompt caches of a taped pass and of an untaped one are the e4m3 image of what the bf16 prefill writes."""
    roll = engine(tiny)
    from spacer_amd.rollout import _LayerCaches
    prompts = [tiny["prompts"][0], PromptInput(tiny["prompts"][0].ids, tiny["prompts"][0].pix, tiny["prompts"][0].grids)]
    P = prompts[0].ids.numel()
    pk, pv, _, plen, _ = roll._prefill(prompts, False)
    caches = _LayerCaches(TINY.layers, 2, P, TINY.kv_heads, TINY.head_dim, "e4m3", dev)
    roll._prefill(prompts[:1], False, keep_tape=True, out=(caches, None, 0))
    roll._prefill(prompts[1:], False, out=(caches, None, 1))
    for i in range(TINY.layers):
        want = K.KVCache.empty(2, P, TINY.kv_heads, TINY.head_dim, "e4m3", dev)
        K.kv_write(want, pk[i].reshape(2 * P, -1), pv[i].reshape(2 * P, -1), torch.arange(2 * P, dtype=torch.int32, device=dev))
        for a, b in zip(K.kv_read(caches.layers[i]), K.kv_read(want)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_rollout_rules(tiny, dev, monkeypatch, fmt):
    """Penalties, bias and allowed ids hold for every drawn token, the first included, and in the replayed graph as in the eager loop."""
    monkeypatch.setattr(K.PLAN, "skinny_blocks", 1)
    roll = engine(tiny)
    allowed = list(range(100, 140)) + [1023]
    base = dict(max_new_tokens=12, top_k=50, top_p=0.95, seed=11, suppress_eos=True, kv_cache=fmt)
    for sp in (SamplingParams(**base, allowed_token_ids=allowed, logit_bias={101: float("-inf"), 1023: 3.0}, presence_penalty=1000.0),
               SamplingParams(**base, repetition_penalty=1.3, frequency_penalty=0.5)):
        a = roll.generate(tiny["prompts"], 4, sp, use_graph=False)
        assert torch.equal(a, roll.generate(tiny["prompts"], 4, sp, use_graph=True))
        if sp.allowed_token_ids:
            for row in a.tolist():
                assert len(set(row)) == len(row) and set(row) <= set(allowed) - {101}        # no token twice, all of them allowed
    # an overwhelming repetition penalty keeps greedy decoding off every token of the prompt and of the completion with a positive logit
    sp = SamplingParams(max_new_tokens=12, top_k=1, top_p=1.0, suppress_eos=True, kv_cache=fmt, repetition_penalty=1e6)
    out = roll.generate(tiny["prompts"][1:], 2, sp)
    seen = set(tiny["prompts"][1].ids.tolist())
    for t in out[0].tolist():
        assert t not in seen
        seen.add(t)
    for bad in (dict(repetition_penalty=0.0), dict(allowed_token_ids=[]), dict(allowed_token_ids=[TINY.vocab]), dict(logit_bias={-1: 1.0}), dict(kv_cache="fp4"),
                dict(logit_bias={3: float("nan")}), dict(allowed_token_ids=[TINY.eos_token_id])):
        with pytest.raises(ValueError):
            roll.generate(tiny["prompts"][1:], 2, SamplingParams(**{**base, **bad}))


@pytest.mark.parametrize("dtype", ["bf16", "e4m3", "int8"])
def test_drafted_tree_equals_one_by_one(dev, dtype):
    """A tree of drafted tokens in one call, against its longest branch appended and attended token by token: both within their bounds of the definition."""
    hq, hkv, d, B, P, cap, n0 = 12, 2, 128, 4, 75, 60, 21
    fmt = K.KV_DTYPES[dtype]
    prompt, pval = filled(2, P, hkv, d, fmt, dev, 5)
    masks, branch = [1, 3, 5, 7 + 4, 21, 53], [0, 2, 4, 5]                   # node 5 hangs on 4, 4 on 2, 2 on 0
    nodes = len(masks)
    q, k, v = (rnd((B, nodes, h * d), s).to(BF).to(dev) for h, s in ((hq, 1), (hkv, 2), (hkv, 3)))
    pl, n = torch.tensor([P, 40], dtype=torch.int32, device=dev), torch.full((B,), n0, dtype=torch.int32, device=dev)
    one, _ = filled(B, cap, hkv, d, fmt, dev, 9)
    two, _ = filled(B, cap, hkv, d, fmt, dev, 9)
    K.kv_append(one, k.view(B * nodes, -1), v.view(B * nodes, -1), n)
    got = K.attn_cache(q.view(B * nodes, -1), prompt, pl, one, n, hq, d ** -0.5, rows_per_prompt=2, nodes=nodes, tree=as_int64([masks], dev)[0].contiguous())
    tval = [x.double().cpu().transpose(1, 2) for x in K.kv_read(one, dtype=F32)]
    want, tol = attn_ref(q.view(B * nodes, -1), pval, [P, 40], [0, 0, 1, 1], tval, [n0] * B, [masks] * B, hq, d ** -0.5, nodes)
    assert bool(((got.double().cpu() - want).abs() <= tol).all())
    for i, node in enumerate(branch):
        at = n + i
        K.kv_append(two, k[:, node].contiguous(), v[:, node].contiguous(), at)
        step = K.attn_cache(q[:, node].contiguous(), prompt, pl, two, at, hq, d ** -0.5, rows_per_prompt=2)
        w, t = want.view(B, nodes, -1)[:, node], tol.view(B, nodes, -1)[:, node]
        assert bool(((step.double().cpu() - w).abs() <= t).all()), node
