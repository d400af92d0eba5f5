"""The measured work of the operators behind several replies to one prompt: the log probabilities of drawn tokens, the
copies of cache pages and state slots that a fork makes, and decode attention whose rows share a prefix.

A case names its operator in ``op``:

* ``logprobs``: ``rows`` rows of ``vocab`` logits (``dtype``; a row starts every ``vocab + gap`` elements), a given token
  per row, the ``top`` best alternatives, entropy and rank.  ``masked``: a third of the vocabulary is at minus infinity,
  as a grammar leaves it;
* ``copy``: ``copies`` pages of ``arrays`` arrays ``[pages, heads, page, dim]``, ``fan`` of them from the same source, whole or
  (``slots``) their first so many slots; ``heads`` = 0: state slots, rows of ``dim`` elements;
* ``attention``: ``rows`` single query rows in ``groups`` groups and ``alone`` rows of their own; the rows of group g share
  their first ``prefix`` / (g + 1) positions (whole pages) and have ``own_lo`` to ``own_hi`` positions of their own.

Sizes are those of ``bench.py`` (Qwen1.5-MoE-A2.7B: 24 layers, 16 heads of 128; Qwen2-57B-A14B: 28 layers, 28 heads of 128 on
4; 151,936 tokens) and generic ones.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ cases
def _logprobs(rows, vocab, top, dtype="float32", gap=0, masked=False):
    return dict(op="logprobs", rows=rows, vocab=vocab, top=top, dtype=dtype, gap=gap, masked=masked)


def _copy(arrays, copies, fan, heads, page, dim, slots, dtype="bfloat16"):
    return dict(op="copy", arrays=arrays, copies=copies, fan=fan, heads=heads, page=page, dim=dim, slots=slots, dtype=dtype)


def _attention(rows, groups, alone, prefix, own_lo, own_hi, q_heads, kv_heads, dim, page=16, dtype="bfloat16", sink=False,
               softcap=0.0):
    return dict(op="attention", rows=rows, groups=groups, alone=alone, prefix=prefix, own_lo=own_lo, own_hi=own_hi,
                q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, sink=sink, softcap=softcap)


def listed():
    return [
        # one reply that asks for its tokens' log probabilities and five alternatives each: a step's smallest call
        dict(_logprobs(1, 151936, 5), name="logprobs_one_row"),
        # a decode step of 64 replies with twenty alternatives
        dict(_logprobs(64, 151936, 20), name="logprobs_64_rows_top20"),
        # a prompt's tokens scored (perplexity, ranking of given replies)
        dict(_logprobs(2048, 151936, 0), name="logprobs_prompt_2048"),
        # bfloat16 logits of a smaller vocabulary, rows that start off any boundary, a grammar's mask: ties everywhere
        dict(_logprobs(509, 32003, 8, "bfloat16", 7, True), name="logprobs_bf16_masked"),
        # one prompt forked into eight replies: the page that is part full, in all layers' keys and values
        dict(_copy(48, 7, 7, 16, 16, 128, 11), name="copy_fork_one_into_8"),
        # 64 prompts forked into four replies each, 57B sizes
        dict(_copy(56, 192, 3, 4, 16, 128, 5), name="copy_fork_64_into_4"),
        # four sequences of 2,048 tokens copied whole
        dict(_copy(48, 512, 1, 16, 16, 128, 16), name="copy_whole_sequences"),
        # recurrent states (24 layers, 16 heads of 128 x 128 float32) of one request handed to eight
        dict(_copy(1, 8, 8, 0, 1, 24 * 16 * 128 * 128, 1, "float32"), name="copy_states_into_8"),
        # four replies to a short prompt, just begun
        dict(_attention(4, 1, 0, 496, 1, 40, 16, 16, 128), name="attention_4_replies"),
        # 64 replies behind a long common prompt, grouped-query heads
        dict(_attention(64, 1, 0, 8192, 16, 512, 28, 4, 128), name="attention_64_rows_8192"),
        # three prompts of different lengths and rows of their own, a sink, heads between the kernels' sizes
        dict(_attention(45, 3, 5, 2000, 1, 300, 24, 4, 96, sink=True), name="attention_3_prompts_sink"),
        # 128 samples of one very long context: as many products as bytes
        dict(_attention(128, 1, 0, 16384, 1, 128, 28, 4, 128), name="attention_128_rows_16384"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "copy", "attention"])
    if op == "logprobs":
        vocab = _log_int(rng, 1000, 160000)
        rows = _log_int(rng, 1, min(2048, max(1, 2048 * 151936 // vocab)))
        top = rng.choice([0, 1, 2, 5, 8, 20, 32])
        if top and rows * vocab > 64 << 20:
            rows = (64 << 20) // vocab
        return _logprobs(rows, vocab, top, rng.choice(["float32", "float32", "bfloat16"]), rng.choice([0, 0, 1, 5, 8]),
                         rng.random() < 0.25)
    if op == "copy":
        page = rng.choice([16, 16, 32, 64])
        heads = rng.choice([0, 1, 2, 4, 8, 16])
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        size = 2 if dtype == "bfloat16" else 4
        if heads == 0:
            arrays, page, dim, slots = 1, 1, _log_int(rng, 1 << 12, 1 << 23), 1
        else:
            arrays, dim = 2 * rng.randint(2, 28), rng.choice([64, 80, 96, 128, 256])
            slots = rng.randint(1, page)
        most = max(1, (1600 << 20) // (arrays * max(heads, 1) * page * dim * size))
        copies = _log_int(rng, 1, min(512, most))
        return _copy(arrays, copies, rng.choice([1, 3, 7, 15]), heads, page, dim, slots, dtype)
    q_heads, kv_heads, dim = rng.choice([(16, 16, 128), (28, 4, 128), (24, 4, 96), (16, 4, 64), (8, 2, 128), (16, 1, 256),
                                         (20, 4, 80)])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    rows = _log_int(rng, 2, 128 if dtype == "bfloat16" else 32)
    groups = rng.randint(1, max(1, min(4, rows // 2)))
    alone = rng.randint(0, rows - 2 * groups) // 4
    most = min(16384, (1 << 30) // (rows * kv_heads * dim))
    if dtype == "float32":
        most = min(most, 4096)
    prefix = _log_int(rng, 32, most)
    own_hi = _log_int(rng, 2, max(2, min(600, most // 2)))
    return _attention(rows, groups, alone, prefix, rng.randint(1, own_hi), own_hi, q_heads, kv_heads, dim,
                      rng.choice([16, 16, 32]), dtype, rng.random() < 0.25, rng.choice([0.0, 0.0, 0.0, 30.0]))


# ------------------------------------------------------------------------------------------------ inputs
def _spread(lo, hi, n, i):
    """The i-th of n lengths from lo to hi, evenly spread over the logarithm."""
    return lo if n <= 1 else int(round(lo * (hi / lo) ** (i / (n - 1))))


def _layout(case):
    """The rows of an attention case: per group (its rows, its prefix) and every row's number of positions."""
    rows, groups, alone, page = case["rows"], case["groups"], case["alone"], case["page"]
    order = [(i * 7919 + 3) % rows if math.gcd(7919, rows) == 1 else i for i in range(rows)]
    shared = order[alone:]
    members = [sorted(shared[g::groups]) for g in range(groups)]
    prefix = [max(page, case["prefix"] // (g + 1) // page * page) for g in range(groups)]
    lengths = [_spread(case["own_lo"], case["own_hi"], rows, i) for i in range(rows)]
    for g in range(groups):
        for r in members[g]:
            lengths[r] += prefix[g]
    return list(zip(members, prefix)), lengths


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    dev = "cuda"
    if case["op"] == "logprobs":
        R, V = case["rows"], case["vocab"]
        wide = torch.randn((R, V + case["gap"]), generator=g, device=dev, dtype=torch.float32).mul_(2.5)
        # a head's logits have a few tokens far above the rest, some rows far enough to be all but certain
        lift = torch.rand((R, 1), generator=g, device=dev).mul_(14.0)
        favoured = torch.randint(0, V, (R, 6), generator=g, device=dev)
        wide.scatter_add_(1, favoured, lift * torch.rand((R, 6), generator=g, device=dev))
        tokens = torch.where(torch.rand(R, generator=g, device=dev) < 0.7, favoured[:, 0],
                             torch.randint(0, V, (R,), generator=g, device=dev))
        if case["masked"]:
            gone = (torch.arange(V + case["gap"], device=dev)[None, :] + torch.arange(R, device=dev)[:, None]) % 3 == 0
            tokens = torch.where(gone.gather(1, tokens[:, None])[:, 0], (tokens + 1) % (V - V % 3), tokens)
            tokens = torch.where(gone.gather(1, tokens[:, None])[:, 0], (tokens + 1) % (V - V % 3), tokens)
            wide.masked_fill_(gone, -math.inf)
        wide = wide.to(dtype)
        state = {"logits": wide[:, :V], "tokens": tokens.to(torch.int32), "top": case["top"],
                 "logprob": torch.empty(R, device=dev), "entropy": torch.empty(R, device=dev),
                 "rank": torch.empty(R, dtype=torch.int32, device=dev), "top_ids": None, "top_logprobs": None}
        if case["top"]:
            state["top_ids"] = torch.empty((R, case["top"]), dtype=torch.int32, device=dev)
            state["top_logprobs"] = torch.empty((R, case["top"]), device=dev)
        return dict(state, op="logprobs")
    if case["op"] == "copy":
        n, heads = case["copies"], case["heads"]
        sources = (n + case["fan"] - 1) // case["fan"]
        places = sources + n + 3
        shape = (places, heads, case["page"], case["dim"]) if heads else (places, case["dim"])
        pool = torch.randn((case["arrays"],) + shape, generator=g, device=dev, dtype=dtype)
        where = torch.randperm(places, generator=g, device=dev).to(torch.int32)
        src = where[:sources].repeat_interleave(case["fan"])[:n].contiguous()
        dst = where[sources:sources + n].contiguous()
        slots = torch.full((n,), case["slots"], dtype=torch.int32, device=dev) if case["slots"] < case["page"] else None
        state = {"op": "copy", "pool": pool, "src": src, "dst": dst, "slots": slots}
        if own:
            from nano_vllm_cpp_b200.csrc import ops
            state["arrays"] = ops.PageArrays(list(pool))           # a cache's arrays, for its whole life
        return state
    groups, lengths = _layout(case)
    R, Hq, Hkv, D, page = case["rows"], case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    width = max((n + page - 1) // page for n in lengths)
    table = torch.full((R, width), -1, dtype=torch.int32)
    used = 0
    first = [0] * R
    for members, prefix in groups:
        n = prefix // page
        for r in members:
            table[r, :n] = torch.arange(used, used + n, dtype=torch.int32)
            first[r] = n
        used += n
    for r in range(R):
        n = (lengths[r] + page - 1) // page
        table[r, first[r]:n] = torch.arange(used, used + n - first[r], dtype=torch.int32)
        used += n - first[r]
    shuffled = torch.randperm(used, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.where(table >= 0, shuffled[table.clamp(min=0).long()], table)
    k = torch.randn((used, Hkv, page, D), generator=g, device=dev, dtype=dtype)
    v = torch.randn((used, Hkv, page, D), generator=g, device=dev, dtype=dtype)
    qkv = torch.randn((R, (Hq + 2 * Hkv) * D), generator=g, device=dev, dtype=dtype).mul_(1.5)
    state = {"op": "attention", "qkv": qkv, "k": k, "v": v, "table": table.to(dev), "page": page, "Hq": Hq, "Hkv": Hkv, "D": D,
             "positions": torch.tensor([n - 1 for n in lengths], dtype=torch.int32, device=dev),
             "row_entry": torch.arange(R, dtype=torch.int32, device=dev), "longest": max(lengths),
             "scale": 1.0 / math.sqrt(D), "sink": 0.5 if case["sink"] else None, "softcap": case["softcap"],
             "out": torch.empty((R, Hq * D), dtype=dtype, device=dev)}
    if own:
        from nano_vllm_cpp_b200.csrc import ops
        state["shared"] = ops.SharedPrefix(groups, R, dev)         # a step's, for all of its layers
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "logprobs":
        return _plain_logprobs(state)
    if state["op"] == "copy":
        pool, src, dst = state["pool"], state["src"].long(), state["dst"].long()
        new = pool[:, src]
        if state["slots"] is not None:
            live = torch.arange(pool.shape[3], device=pool.device)[None, :] < state["slots"][:, None]
            new = torch.where(live[None, :, None, :, None], new, pool[:, dst])
        pool[:, dst] = new
        return pool
    return _plain_attention(state)


def _run_own(state):
    from nano_vllm_cpp_b200.csrc import ops
    if state["op"] == "logprobs":
        ops.token_logprobs(state["logits"], state["tokens"], state["logprob"], entropy=state["entropy"], rank=state["rank"],
                           top_ids=state["top_ids"], top_logprobs=state["top_logprobs"])
        out = {n: state[n] for n in ("logprob", "entropy", "rank")}
        if state["top"]:
            out.update(top_ids=state["top_ids"], top_logprobs=state["top_logprobs"])
        return out
    if state["op"] == "copy":
        ops.copy_pages(state["arrays"], state["src"], state["dst"], slots=state["slots"])
        return state["pool"]
    ops.attention_decode_shared(state["qkv"], state["k"], state["v"], state["table"], state["row_entry"], state["positions"],
                                state["scale"], state["out"], state["Hq"], state["Hkv"], state["D"], state["longest"],
                                state["shared"], sink_score=state["sink"], softcap=state["softcap"])
    return state["out"]


def _plain_logprobs(state):
    x, tokens, top = state["logits"].float(), state["tokens"].long(), state["top"]
    R, V = x.shape
    m = x.amax(dim=1, keepdim=True)
    d = x - m
    e = d.exp()
    # the sum without its largest terms, so that a row that is all but certain keeps its small numbers
    most = d == 0
    n1 = most.sum(dim=1, dtype=torch.float32)
    log_z = n1.log() + torch.log1p(torch.where(most, torch.zeros_like(e), e).sum(dim=1) / n1)
    mean = torch.where(e > 0, e * d, torch.zeros_like(e)).sum(dim=1) / log_z.exp()
    at = x.gather(1, tokens[:, None])
    ahead = (x > at) | ((x == at) & (torch.arange(V, device=x.device)[None, :] < tokens[:, None]))
    out = {"logprob": (at - m)[:, 0] - log_z, "entropy": log_z - mean, "rank": ahead.sum(dim=1, dtype=torch.int32)}
    if top:
        best, ids = x.sort(dim=1, descending=True, stable=True)
        out.update(top_ids=ids[:, :top].to(torch.int32).contiguous(), top_logprobs=best[:, :top] - m - log_z[:, None])
    return out


def _gathered(cache, state, dtype):
    """Every row's keys (or values), [rows, kv heads, positions, D]: zeros where the table ends."""
    table = state["table"].long()
    R, width = table.shape
    rows = cache[table.clamp(min=0)].to(dtype)                     # [rows, pages, kv heads, page, D]
    return rows.permute(0, 2, 1, 3, 4).reshape(R, state["Hkv"], width * state["page"], state["D"])


def _plain_attention(state):
    R, Hq, Hkv, D = state["qkv"].shape[0], state["Hq"], state["Hkv"], state["D"]
    q = state["qkv"][:, :Hq * D].float().reshape(R, Hkv, Hq // Hkv, D)
    k = _gathered(state["k"], state, torch.float32)
    s = (q @ k.transpose(2, 3)) * state["scale"]
    del k
    if state["softcap"] > 0:
        s = state["softcap"] * torch.tanh(s / state["softcap"])
    seen = torch.arange(s.shape[3], device=s.device)[None, :] <= state["positions"][:, None]
    s = torch.where(seen[:, None, None, :], s, torch.full_like(s, -math.inf))
    m = s.amax(dim=3, keepdim=True)
    e = (s - m).exp()
    z = e.sum(dim=3, keepdim=True)
    if state["sink"] is not None:
        z = z + (state["sink"] - m).exp()
    o = (e / z) @ _gathered(state["v"], state, torch.float32)
    return o.reshape(R, Hq * D).to(state["qkv"].dtype)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (16 + 8 * case["top"]), "flops": 4 * n}
    if case["op"] == "copy":
        sources = (case["copies"] + case["fan"] - 1) // case["fan"]
        each = case["arrays"] * max(case["heads"], 1) * case["slots"] * case["dim"] * size
        return {"bytes": each * (sources + case["copies"]), "flops": 0}
    groups, lengths = _layout(case)
    positions = sum(lengths) - sum(prefix * (len(members) - 1) for members, prefix in groups)
    kv = 2 * positions * case["kv_heads"] * case["dim"] * size
    return {"bytes": kv + 2 * case["rows"] * case["q_heads"] * case["dim"] * size,
            "flops": 4 * sum(lengths) * case["q_heads"] * case["dim"]}


# ------------------------------------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "copy":
        return None                                                # nothing is computed
    if case["op"] == "logprobs":
        R, top = case["rows"], case["top"]
        got = {"logprob": torch.empty(R, dtype=torch.float64, device="cuda"), "entropy": torch.empty(R, dtype=torch.float64, device="cuda"),
               "rank": None}
        if top:
            got.update(top_ids=None, top_logprobs=torch.empty((R, top), dtype=torch.float64, device="cuda"))
        for a in range(0, R, 128):
            x = state["logits"][a:a + 128].double()
            lp = torch.log_softmax(x, dim=1)
            # log_softmax leaves 1e-16 of a certain token's distance from one: from the others' sum instead
            b = x.argmax(dim=1, keepdim=True)
            others = torch.exp(lp.scatter(1, b, -math.inf)).sum(dim=1, keepdim=True)
            lp = lp.scatter(1, b, torch.log1p(-others))
            got["logprob"][a:a + 128] = lp.gather(1, state["tokens"][a:a + 128].long()[:, None])[:, 0]
            got["entropy"][a:a + 128] = torch.special.entr(lp.exp()).sum(dim=1)
            if top:
                got["top_logprobs"][a:a + 128] = lp.topk(top, dim=1).values
        return got
    R, Hq, Hkv, D, page = state["qkv"].shape[0], state["Hq"], state["Hkv"], state["D"], state["page"]
    out = torch.empty((R, Hq, D), dtype=torch.float64, device="cuda")
    ends = (state["positions"] + 1).tolist()
    for r in range(R):
        pages = state["table"][r, :(ends[r] + page - 1) // page].long()
        keys = state["k"][pages].double().transpose(0, 1).reshape(Hkv, -1, D)[:, :ends[r]]
        values = state["v"][pages].double().transpose(0, 1).reshape(Hkv, -1, D)[:, :ends[r]]
        q = state["qkv"][r, :Hq * D].double().view(Hkv, Hq // Hkv, D)
        s = torch.einsum("hgd,hnd->hgn", q, keys) * state["scale"]
        if state["softcap"] > 0:
            s = torch.tanh(s / state["softcap"]) * state["softcap"]
        if state["sink"] is not None:
            s = torch.cat([s, torch.full_like(s[:, :, :1], state["sink"])], dim=2)
        p = torch.softmax(s, dim=2)[:, :, :ends[r]]
        out[r] = torch.einsum("hgn,hnd->hgd", p, values).reshape(Hq, D)
    return out.view(R, Hq * D)
