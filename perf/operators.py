"""The rollout's cache and logits operators, as cases that can be timed and compared.

Three operators of token generation, each with its plain form (elementary torch operations in 32 bits, or 64 where 32 lose what matters)
beside the call that a program makes of ``spacer_amd.kernels``:

* ``kv``      a key/value cache in 8 bits, quantised as it is written (a prompt's rows, or the newest tokens of every rollout) and read back;
* ``attn``    attention of one new token, or of a tree of drafted tokens, over [the prompt's cache shared by its rollouts | the rollout's own];
* ``logits``  penalties for repeated tokens, a bias and a grammar's mask on the logits that the sampler draws from.

Formulas.  A cache row is one token's D numbers x of one kv head, amax = max |x|:
  e4m3  scale s = the smallest power of two with amax / s <= 448 (never below 2^-126), code = x / s rounded to the nearest e4m3 number
  int8  scale s = amax / 127 in 32 bits, code = x / s rounded to the nearest whole number, ties to even; an all-zero row has s = 0 and codes 0
  the value that a code stands for is code * s.
Attention of query row i (a rollout's node) and query head h over the visible keys j of kv head h // (Hq / Hkv):
  o = sum_j softmax_j(scale q . k_j) v_j; visible are the prompt's keys, the rollout's earlier tokens, and the nodes whose bit is set in
  the node's mask (no mask: the nodes up to and including itself).  A row that sees no key gives zeros.
Logits of a row with the tokens seen so far (prompt and generated) and their counts (generated):
  x = x > 0 ? x / r : x r  on seen tokens;  x -= f count + p [count > 0];  x += bias;  x = -inf where the grammar forbids the token.
"""
import math

import torch

own = False


# --------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # --- cache: a short text prompt's rows (launch latency is what counts); the keys and values are columns of packed q|k|v rows
        dict(name="kv_write_short", op="kv", fmt="e4m3", seqs=1, cap=157, hq=12, hkv=2, dim=128, short=0, nodes=0),
        # ... eight video prompts of one training step, ragged lengths
        dict(name="kv_write_group", op="kv", fmt="int8", seqs=8, cap=1391, hq=28, hkv=4, dim=128, short=83, nodes=0),
        # ... four of the longest prompts that the trainer's defaults allow
        dict(name="kv_write_long", op="kv", fmt="e4m3", seqs=4, cap=16384, hq=28, hkv=4, dim=128, short=1201, nodes=0),
        # ... the newest token of each of 64 rollouts appended to its own cache
        dict(name="kv_append_step", op="kv", fmt="int8", seqs=64, cap=96, hq=28, hkv=4, dim=128, short=1, nodes=1),
        # --- attention: two rollouts of a short prompt (latency)
        dict(name="attn_decode_small", op="attn", fmt="int8", prompts=1, rows=2, plen=203, pshort=0, tcap=64, tlen=17, tstep=0, nodes=1, tree="chain",
             hq=12, hkv=2, dim=128),
        # ... the decode step of a training step's rollouts: 8 video prompts x 8 rollouts
        dict(name="attn_decode_group", op="attn", fmt="e4m3", prompts=8, rows=8, plen=1391, pshort=83, tcap=512, tlen=300, tstep=0, nodes=1, tree="chain",
             hq=28, hkv=4, dim=128),
        # ... long prompts, every rollout at a length of its own
        dict(name="attn_decode_long", op="attn", fmt="int8", prompts=8, rows=8, plen=16384, pshort=1201, tcap=1024, tlen=700, tstep=5, nodes=1, tree="chain",
             hq=28, hkv=4, dim=128),
        # ... a tree of drafted tokens for single sequences, cache in 16 bits
        dict(name="attn_tree_bf16", op="attn", fmt="bf16", prompts=8, rows=1, plen=2311, pshort=97, tcap=640, tlen=211, tstep=31, nodes=13, tree="tree",
             hq=16, hkv=2, dim=128),
        # ... trees of 32 drafted tokens for 32 rollouts, and a narrower head
        dict(name="attn_tree_group", op="attn", fmt="e4m3", prompts=4, rows=8, plen=5498, pshort=411, tcap=1024, tlen=333, tstep=17, nodes=32, tree="tree",
             hq=16, hkv=4, dim=64),
        # --- logits: the eight rollouts of one prompt, one penalty, history kept up to date
        dict(name="logits_repeat", op="logits", batch=8, vocab=151936, ids=911, rebuild=False, frequency=False, bias="none", masks=0),
        # ... 64 rollouts, all penalties, a bias for every row's vocabulary and a grammar with 5 states
        dict(name="logits_full", op="logits", batch=64, vocab=152064, ids=1903, rebuild=False, frequency=True, bias="row", masks=5),
        # ... 128 rows whose history is built from the prompts' and completions' ids first
        dict(name="logits_rebuild", op="logits", batch=128, vocab=152064, ids=2051, rebuild=True, frequency=True, bias="all", masks=1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["kv", "attn", "attn", "logits"])
    hq, hkv = rng.choice([(28, 4), (12, 2), (16, 2), (2, 1), (16, 4), (8, 8), (24, 1)])
    if op == "kv":
        fmt, dim, nodes = rng.choice(["e4m3", "int8"]), rng.choice([128, 128, 64]), rng.choice([0, 0, 1, 7])
        seqs = _log_int(rng, 1, 96)
        cap = _log_int(rng, max(nodes, 1), max(nodes, 1, min(16384, 130000 // (seqs * hkv))))
        return dict(op=op, fmt=fmt, seqs=seqs, cap=cap, hq=hq, hkv=hkv, dim=dim, short=rng.randrange(0, max(1, cap // seqs) + 1), nodes=nodes)
    if op == "attn":
        nodes = rng.choice([1, 1, 1, 2, 5, 16, 33, 64])
        prompts, rows = _log_int(rng, 1, 8), rng.choice([1, 2, 3, 8])
        plen = _log_int(rng, 1, min(16384, 220000 // (nodes * rows)))
        tcap = nodes + _log_int(rng, 1, 1024)
        tlen = rng.randrange(0, tcap - nodes + 1)
        return dict(op=op, fmt=rng.choice(["bf16", "e4m3", "int8"]), prompts=prompts, rows=rows, plen=plen, pshort=rng.randrange(0, max(1, plen // prompts) + 1),
                    tcap=tcap, tlen=tlen, tstep=rng.randrange(0, max(1, tlen // (prompts * rows)) + 1), nodes=nodes, tree=rng.choice(["chain", "tree", "tree"]),
                    hq=hq, hkv=hkv, dim=rng.choice([128, 128, 64]))
    batch = _log_int(rng, 1, 128)
    return dict(op=op, batch=batch, vocab=rng.choice([1024, _log_int(rng, 33, 152064), 151936, 152064]), ids=_log_int(rng, 1, 2051), rebuild=rng.random() < 0.3,
                frequency=rng.random() < 0.6, bias=rng.choice(["none", "all", "row"]), masks=rng.choice([0, 1, 5]))


# -------------------------------------------------------------------------------------------------------------- inputs
def _lengths(n, most, short):
    """Sequence i has `short` tokens less than the one before it, and none less than 0."""
    return [max(0, most - i * short) for i in range(n)]


def _cache_lengths(c):
    return _lengths(c["seqs"], c["cap"] - max(c["nodes"], 0), c["short"])


def _tail_lengths(c):
    return _lengths(c["prompts"] * c["rows"], c["tlen"], c["tstep"])


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _keys_values(g, *shape):
    """Keys with a few large channels, values with a token's own size: what a decoder's projections give."""
    x = torch.randn(*shape, generator=g, device="cuda")
    return (x * (0.4 + 2.0 * torch.rand(shape[-1], generator=g, device="cuda") ** 6) * torch.exp(0.5 * torch.randn(*shape[:-1], 1, generator=g, device="cuda"))).bfloat16()


def _codes(x, fmt):
    """(codes, scales) of bf16 rows x[..., D]; fmt bf16: the rows and no scales."""
    if fmt == "bf16":
        return x, None
    amax = x.float().abs().amax(-1, keepdim=True)
    if fmt == "e4m3":
        m, e = torch.frexp(amax)
        s = ((e - torch.where(m <= 0.875, 9, 8)).clamp_min(-126) + 127 << 23).int().view(torch.float32)      # a power of two, made of its exponent's bits
        return (x.float() / s).to(torch.float8_e4m3fn), s.squeeze(-1)
    s = (amax.double() / 127).float()
    q = torch.where(s > 0, x.double() / torch.where(s > 0, s, 1.0).double(), 0.0).round()
    return q.to(torch.int8), s.squeeze(-1)


def _values(codes, scales):
    return codes.float() if scales is None else codes.float() * scales[..., None]


def _bits(masks):
    """bool [..., n] -> int32 [..., ceil(n / 32)], bit n % 32 of word n // 32."""
    n = masks.shape[-1]
    wide = torch.zeros(*masks.shape[:-1], (n + 31) // 32 * 32, dtype=torch.int64, device=masks.device)
    wide[..., :n] = masks
    words = (wide.view(*masks.shape[:-1], -1, 32) << torch.arange(32, device=masks.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    if case["op"] == "kv":
        n, cap, hkv, d, nodes = case["seqs"], case["cap"], case["hkv"], case["dim"], case["nodes"]
        lens = _cache_lengths(case)
        tokens = n * nodes if nodes else sum(lens)
        qkv = _keys_values(g, max(tokens, 1), case["hq"] + 2 * hkv, d).view(max(tokens, 1), -1)
        a = case["hq"] * d
        s["k"], s["v"] = qkv[:tokens, a:a + hkv * d], qkv[:tokens, a + hkv * d:]
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        if not nodes:        # source row of every (sequence, position) slot; -1 behind a sequence's end
            at = torch.arange(cap, device="cuda").expand(n, cap)
            first = torch.tensor([sum(lens[:i]) for i in range(n)], device="cuda")
            s["rows"] = torch.where(at < s["lengths"][:, None], at + first[:, None], -1).int().view(-1).contiguous()
        old_k, old_v = _keys_values(g, n, hkv, cap, d), _keys_values(g, n, hkv, cap, d)
        s["old"] = (*_codes(old_k, case["fmt"]), *_codes(old_v, case["fmt"]))
        if own:
            from spacer_amd import kernels as K
            s["cache"] = K.KVCache(s["old"][0].clone(), s["old"][2].clone(), s["old"][1].clone(), s["old"][3].clone())
    elif case["op"] == "attn":
        n_p, rows, nodes, hq, hkv, d = case["prompts"], case["rows"], case["nodes"], case["hq"], case["hkv"], case["dim"]
        b = n_p * rows
        s["q"] = _keys_values(g, b * nodes, hq, d).view(b * nodes, hq * d)
        pk, pv = _keys_values(g, n_p, hkv, case["plen"], d), _keys_values(g, n_p, hkv, case["plen"], d)
        tk, tv = _keys_values(g, b, hkv, case["tcap"], d), _keys_values(g, b, hkv, case["tcap"], d)
        s["prompt"] = (*_codes(pk, case["fmt"]), *_codes(pv, case["fmt"]))
        s["tail"] = (*_codes(tk, case["fmt"]), *_codes(tv, case["fmt"]))
        s["prompt_len"] = torch.tensor(_lengths(n_p, case["plen"], case["pshort"]), dtype=torch.int32, device="cuda")
        s["tail_len"] = torch.tensor(_tail_lengths(case), dtype=torch.int32, device="cuda")
        s["tree"] = None
        if case["tree"] == "tree":       # every node hangs on one of the nodes before it: its mask is its parent's and its own bit
            parent = (torch.rand(b, nodes, generator=g, device="cuda") * torch.arange(nodes, device="cuda")).long().cpu().tolist()
            masks = []
            for row in parent:
                m = []
                for i, p in enumerate(row):
                    m.append((m[p] if i else 0) | (1 << i))
                masks.append([v - 2 ** 64 if v >= 2 ** 63 else v for v in m])
            s["tree"] = torch.tensor(masks, dtype=torch.int64, device="cuda")
        if own:
            from spacer_amd import kernels as K
            s["prompt_cache"], s["tail_cache"] = (K.KVCache(c[0], c[2], c[1], c[3]) for c in (s["prompt"], s["tail"]))
    else:
        b, vocab, n = case["batch"], case["vocab"], case["ids"]
        s["logits"] = 4.0 * torch.randn(b, vocab, generator=g, device="cuda")
        u = torch.rand(b, 2 * n, generator=g, device="cuda")
        ids = (vocab * u ** 3).long().clamp_(max=vocab - 1)          # some tokens come often, most not at all
        s["prompt_ids"], s["out_ids"] = ids[:, :n].contiguous(), ids[:, n:].contiguous()
        s["out_len"] = torch.tensor(_lengths(b, n, n // b // 2), dtype=torch.int32, device="cuda")
        live = torch.arange(n, device="cuda") < s["out_len"][:, None]
        s["counts"] = torch.zeros(b, vocab, dtype=torch.int32, device="cuda").scatter_add_(1, s["out_ids"], live.int())
        prompt = torch.zeros(b, vocab, dtype=torch.int32, device="cuda").scatter_add_(1, s["prompt_ids"], torch.ones_like(s["prompt_ids"], dtype=torch.int32))
        s["seen"] = _bits((prompt + s["counts"]) > 0)
        s["repetition"] = 1.05
        s["frequency"] = 0.1 + 0.2 * torch.rand(b, generator=g, device="cuda") if case["frequency"] else None
        s["presence"] = 0.3 if case["frequency"] else None
        s["bias"] = {"none": None, "all": torch.randn(vocab, generator=g, device="cuda")}.get(case["bias"], torch.randn(b, vocab, generator=g, device="cuda"))
        s["allowed"] = s["allowed_row"] = None
        if case["masks"]:
            s["allowed"] = _bits(torch.rand(case["masks"], vocab, generator=g, device="cuda") < torch.linspace(0.9, 0.02, case["masks"], device="cuda")[:, None])
            s["allowed_row"] = torch.randint(-1, case["masks"], (b,), generator=g, device="cuda").int()
    return s


# ----------------------------------------------------------------------------------------------------------- one pass
def run(state):
    return {"kv": _run_kv, "attn": _run_attn, "logits": _run_logits}[state["op"]](state)


def _out_type(s):
    return torch.float32 if s["fmt"] == "int8" else torch.bfloat16


def _run_kv(s):
    """Writes the new rows and returns the values of the whole cache, [sequences, positions, kv heads, D] each for keys and values."""
    if own:
        from spacer_amd import kernels as K
        if s["nodes"]:
            K.kv_append(s["cache"], s["k"], s["v"], s["lengths"])
        else:
            K.kv_write(s["cache"], s["k"], s["v"], s["rows"])
        return K.kv_read(s["cache"], dtype=_out_type(s))
    n, cap, hkv, d = s["seqs"], s["cap"], s["hkv"], s["dim"]
    if s["nodes"]:
        at = torch.arange(cap, device="cuda") - s["lengths"][:, None].long()
        fresh = (at >= 0) & (at < s["nodes"])
        rows = torch.arange(n, device="cuda")[:, None] * s["nodes"] + at.clamp(0, s["nodes"] - 1)
    else:
        rows = s["rows"].view(n, cap).long()
        fresh = rows >= 0
    return tuple(_plain_update(x, rows, fresh, old, scale, s) for x, old, scale in ((s["k"], s["old"][0], s["old"][1]), (s["v"], s["old"][2], s["old"][3])))


def _plain_update(x, rows, fresh, old, scale, s):
    was = _values(old, scale).transpose(1, 2)
    if x.shape[0] == 0:
        return was.to(_out_type(s)).contiguous()
    new = _values(*_codes(x.reshape(-1, s["hkv"], s["dim"]), s["fmt"]))[rows.clamp(min=0)]
    return torch.where(fresh[..., None, None], new, was).to(_out_type(s)).contiguous()


def _run_attn(s):
    scale = s["dim"] ** -0.5
    if own:
        from spacer_amd import kernels as K
        return K.attn_cache(s["q"], s["prompt_cache"], s["prompt_len"], s["tail_cache"], s["tail_len"], s["hq"], scale, rows_per_prompt=s["rows"],
                            nodes=s["nodes"], tree=s["tree"])
    n_p, rows, nodes, hq, hkv, d = s["prompts"], s["rows"], s["nodes"], s["hq"], s["hkv"], s["dim"]
    b, rep = n_p * rows, hq // hkv
    pk, pv, tk, tv = (_values(*c) for c in (s["prompt"][:2], s["prompt"][2:], s["tail"][:2], s["tail"][2:]))
    q = s["q"].float().view(n_p, rows, nodes, hkv, rep, d).permute(0, 3, 1, 2, 4, 5).contiguous() * scale     # [prompt, kv head, row, node, head, D]
    a = torch.matmul(q.view(n_p, hkv, -1, d), pk.transpose(2, 3).contiguous())
    a = a.masked_fill((torch.arange(pk.shape[2], device="cuda") >= s["prompt_len"][:, None])[:, None, None], -math.inf).view(n_p, hkv, rows, nodes * rep, -1)
    t = torch.matmul(q.transpose(1, 2).reshape(b, hkv, nodes * rep, d), tk.transpose(2, 3).contiguous())
    at = torch.arange(tk.shape[2], device="cuda") - s["tail_len"][:, None].long()                                # [row, position]: index of the node, or below 0
    inside = at.clamp(0, nodes - 1)[:, None, :].expand(b, nodes, -1)
    if s["tree"] is None:
        hit = inside <= torch.arange(nodes, device="cuda")[:, None]
    else:
        hit = ((s["tree"][:, :, None] >> inside) & 1).bool()
    see = (at < 0)[:, None, :] | (hit & (at < nodes)[:, None, :])
    t = t.view(b, hkv, nodes, rep, -1).masked_fill(~see[:, None, :, None], -math.inf).view(n_p, rows, hkv, nodes * rep, -1).transpose(1, 2)
    m = torch.maximum(a.amax(-1, keepdim=True), t.amax(-1, keepdim=True))
    m = torch.where(m.isinf(), 0.0, m)
    a, t = torch.exp(a - m), torch.exp(t - m)
    total = a.sum(-1, keepdim=True) + t.sum(-1, keepdim=True)
    o = torch.matmul(a.view(n_p, hkv, -1, a.shape[-1]), pv).view(n_p, hkv, rows, nodes * rep, d)
    o = o + torch.matmul(t.transpose(1, 2).reshape(b, hkv, nodes * rep, -1), tv).view(n_p, rows, hkv, nodes * rep, d).transpose(1, 2)
    o = torch.where(total > 0, o / total, 0.0).view(n_p, hkv, rows, nodes, rep, d).permute(0, 2, 3, 1, 4, 5)
    return o.reshape(b * nodes, hq * d).to(torch.bfloat16)


def _unpack(words, vocab):
    at = torch.arange(vocab, device=words.device)
    return ((words[..., at // 32] >> (at % 32)) & 1).bool()


def _run_logits(s):
    b, vocab = s["logits"].shape
    if own:
        from spacer_amd import kernels as K
        seen, counts = s["seen"], s["counts"]
        if s["rebuild"]:
            seen, counts = K.token_history(b, vocab, s["logits"].device)
            K.token_history_add_(seen, None, s["prompt_ids"])
            K.token_history_add_(seen, counts, s["out_ids"], s["out_len"])
        return K.process_logits(s["logits"], seen=seen, counts=counts if s["frequency"] is not None else None, repetition=s["repetition"],
                                frequency=s["frequency"], presence=s["presence"], bias=s["bias"], allowed=s["allowed"], allowed_row=s["allowed_row"],
                                out=torch.empty_like(s["logits"]))
    if s["rebuild"]:
        live = torch.arange(s["ids"], device="cuda") < s["out_len"][:, None]
        counts = torch.zeros(b, vocab, dtype=torch.int32, device="cuda").scatter_add_(1, s["out_ids"], live.int())
        seen = (counts > 0).scatter_(1, s["prompt_ids"], True)
    else:
        counts, seen = s["counts"], _unpack(s["seen"], vocab)
    x = s["logits"].double()
    x = torch.where(seen, torch.where(x > 0, x / s["repetition"], x * s["repetition"]), x)
    if s["frequency"] is not None:
        x = x - s["frequency"].double()[:, None] * counts - s["presence"] * (counts > 0)
    if s["bias"] is not None:
        x = x + s["bias"].double()
    x = x.float()
    if s["allowed"] is not None:
        mask = _unpack(s["allowed"], vocab)[s["allowed_row"].clamp(min=0).long()] | (s["allowed_row"] < 0)[:, None]
        x = x.masked_fill(~mask, -math.inf)
    return x


# --------------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "kv":
        lens = _cache_lengths(case)
        fresh = case["seqs"] * case["nodes"] if case["nodes"] else sum(lens)
        row = case["hkv"] * case["dim"]
        every = case["seqs"] * case["cap"]
        out = 4 if case["fmt"] == "int8" else 2
        write = fresh * (2 * 2 * row + 2 * (row + 4 * case["hkv"])) + (0 if case["nodes"] else 4 * every)
        return dict(bytes=write + every * (2 * (row + 4 * case["hkv"]) + 2 * out * row), flops=4 * fresh * row + 2 * every * row)
    if case["op"] == "attn":
        size = 2 * case["dim"] if case["fmt"] == "bf16" else case["dim"] + 4
        keys, tails = _lengths(case["prompts"], case["plen"], case["pshort"]), [t + case["nodes"] for t in _tail_lengths(case)]
        cols = case["nodes"] * case["hq"]
        rows = case["prompts"] * case["rows"]
        return dict(bytes=2 * case["hkv"] * size * (sum(keys) + sum(tails)) + 2 * 2 * rows * cols * case["dim"],
                    flops=4 * case["dim"] * cols * (case["rows"] * sum(keys) + sum(tails)))
    b, v, n = case["batch"], case["vocab"], case["ids"]
    total = b * v * 8 + b * ((v + 31) // 32) * 4
    total += (b if case["bias"] == "row" else 1 if case["bias"] == "all" else 0) * v * 4
    total += case["masks"] * ((v + 31) // 32) * 4
    total += 2 * b * n * 8 if case["rebuild"] else 0
    total += b * min(n, v) * 4 if case["frequency"] else 0
    return dict(bytes=total, flops=4 * b * v)


# -------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The definition in 64 bits, written apart from the plain form: sums as sums, one sequence or row at a time."""
    s = prepare(case, seed)
    return {"kv": _exact_kv, "attn": _exact_attn, "logits": _exact_logits}[case["op"]](s)


def _power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_row_values(x, fmt):
    x = x.double()
    top = x.abs().max(-1, keepdim=True).values
    if fmt == "int8":
        scale = (top / 127).float().double()
        n = torch.floor(x / scale.clamp_min(1e-300))
        part = x / scale.clamp_min(1e-300) - n
        up = (part > 0.5) | ((part == 0.5) & (n % 2 == 1))
        return torch.where(scale > 0, (n + up) * scale, 0.0)
    scale = _power(torch.ceil(torch.log2((top / 448).clamp_min(2.0 ** -126))))
    scale = torch.where(top / (scale / 2) <= 448, torch.clamp(scale / 2, min=2.0 ** -126), scale)       # (where the logarithm rounded up)
    scale = torch.where(top / scale > 448, scale * 2, scale)
    y = x / scale
    step = _power(torch.frexp(y.abs().clamp_min(2.0 ** -6)).exponent - 4)       # 3 bits behind the leading one, subnormal below 2^-6
    return torch.round(y / step) * step * scale


def _exact_kv(s):
    out = []
    lens = s["lengths"].tolist()
    for x, old, scale in ((s["k"], s["old"][0], s["old"][1]), (s["v"], s["old"][2], s["old"][3])):
        full = (old.double() * scale.double()[..., None]).transpose(1, 2).contiguous()
        first = 0
        for i, n in enumerate(lens):
            a, b = (n, n + s["nodes"]) if s["nodes"] else (0, n)
            full[i, a:b] = _exact_row_values(x[first:first + b - a].reshape(b - a, s["hkv"], s["dim"]), s["fmt"]) if b > a else full[i, a:b]
            first += b - a
        out.append(full)
    return tuple(out)


def _exact_attn(s):
    plen, tlen, rep, nodes = s["prompt_len"].tolist(), s["tail_len"].tolist(), s["hq"] // s["hkv"], s["nodes"]
    wide = lambda c, k: c[k].double() if c[k + 1] is None else c[k].double() * c[k + 1].double()[..., None]  # noqa: E731
    out = torch.zeros(s["prompts"] * s["rows"], nodes, s["hkv"], rep, s["dim"], dtype=torch.float64, device="cuda")
    q = s["q"].double().view(-1, nodes, s["hkv"], rep, s["dim"])
    tk, tv = wide(s["tail"], 0), wide(s["tail"], 2)
    for p in range(s["prompts"]):
        one = [None if c is None else c[p] for c in s["prompt"]]
        pk, pv = wide(one, 0)[:, :plen[p]], wide(one, 2)[:, :plen[p]]
        for b in range(p * s["rows"], (p + 1) * s["rows"]):
            n = tlen[b] + nodes
            k, v = torch.cat([pk, tk[b, :, :n]], 1), torch.cat([pv, tv[b, :, :n]], 1)
            see = torch.ones(nodes, k.shape[1], dtype=torch.bool, device="cuda")
            if s["tree"] is None:
                see[:, -nodes:] = torch.tril(see[:, -nodes:])
            else:
                words = [w % 2 ** 64 for w in s["tree"][b].tolist()]
                see[:, -nodes:] = torch.tensor([[bool(w >> j & 1) for j in range(nodes)] for w in words], device="cuda")
            x = torch.matmul(q[b].permute(1, 0, 2, 3).reshape(s["hkv"], nodes * rep, -1), k.transpose(1, 2).contiguous()) * s["dim"] ** -0.5
            x = x.view(s["hkv"], nodes, rep, -1).masked_fill(~see[None, :, None], -math.inf)
            w = torch.softmax(x, -1).view(s["hkv"], nodes * rep, -1)
            out[b] = torch.matmul(w, v).view(s["hkv"], nodes, rep, -1).permute(1, 0, 2, 3)
    return out.view(-1, s["hq"] * s["dim"])


def _exact_logits(s):
    out = []
    bias = s["bias"] if s["bias"] is None or s["bias"].dim() == 2 else s["bias"].expand(s["batch"], -1)
    for b in range(s["batch"]):
        x, vocab = s["logits"][b].double(), s["vocab"]
        count = torch.bincount(s["out_ids"][b, :int(s["out_len"][b])], minlength=vocab)
        seen = (count + torch.bincount(s["prompt_ids"][b], minlength=vocab)) > 0
        x[seen] = torch.where(x[seen] > 0, x[seen] / s["repetition"], x[seen] * s["repetition"])
        if s["frequency"] is not None:
            x -= float(s["frequency"][b]) * count + s["presence"] * (count > 0)
        if bias is not None:
            x += bias[b].double()
        if s["allowed"] is not None and int(s["allowed_row"][b]) >= 0:
            words = s["allowed"][int(s["allowed_row"][b])]
            forbidden = ((words[:, None] >> torch.arange(32, device="cuda")) & 1).view(-1)[:vocab] == 0
            x[forbidden] = -math.inf
        out.append(x)
    return torch.stack(out)
