"""The operators of several replies to one prompt against plain forms in float64: token log probabilities, copies of cache
pages and state slots, decode attention over shared prefixes; and the three one after the other, captured and replayed."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF, NAN = math.inf, math.nan


def ops():
    from nano_vllm_cpp_b200.csrc import ops as o
    return o


def rnd(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV).to(dtype)


# ------------------------------------------------------------------------------------------------ log probabilities
def order(x):
    """Ids by (logit descending, id ascending), NaN last."""
    x = torch.where(torch.isnan(x), torch.full_like(x, -INF), x.double())       # (a stable sort keeps the ids' order)
    return x.sort(dim=1, descending=True, stable=True).indices


def call_logprobs(x, tokens, K, **kw):
    R = x.shape[0]
    got = dict(logprob=torch.full((R,), 7.0, device=DEV), entropy=torch.full((R,), 7.0, device=DEV),
               rank=torch.full((R,), 7, dtype=torch.int32, device=DEV), ids=torch.full((R, K), 7, dtype=torch.int32, device=DEV),
               top=torch.full((R, K), 7.0, device=DEV))
    ops().token_logprobs(x, tokens, got["logprob"], entropy=got["entropy"], rank=got["rank"], top_ids=got["ids"] if K else None,
                         top_logprobs=got["top"] if K else None, **kw)
    return got


def check_logprobs(x, tokens, K):
    got = call_logprobs(x, tokens, K)
    R, V = x.shape
    lp = torch.log_softmax(x.double(), dim=1)
    best = lp.argmax(dim=1, keepdim=True)
    lp = lp.scatter(1, best, torch.log1p(-torch.exp(lp.scatter(1, best, -INF)).sum(dim=1, keepdim=True)))
    H = torch.special.entr(lp.exp()).sum(dim=1)
    ids = order(x)
    rank = (ids == tokens[:, None].long()).int().argmax(dim=1)
    # sums of at most V / 256 + 64 float32 terms in a row, each with an exponential of two units: relative to Z, hence
    # absolute in log Z; a difference from the maximum and one from log Z add half a unit of theirs each
    tol = (V / 256 + 80) * 2.0 ** -24
    want = lp.gather(1, tokens[:, None].long())[:, 0]
    assert torch.all((got["logprob"] == want) | ((got["logprob"].double() - want).abs() <= tol + 2.0 ** -22 * want.abs()))    # (a masked token's is -inf)
    # the entropy's terms are at most 1 / e each and are summed in the same chains beside log Z
    assert torch.all((got["entropy"].double() - H).abs() <= tol * (1 + 2 * H) + 2.0 ** -22 * H)
    assert torch.equal(got["rank"].long(), rank)
    if K:
        assert torch.equal(got["ids"].long(), ids[:, :K])
        top = lp.gather(1, ids[:, :K])
        seen = torch.isfinite(top)
        assert torch.equal(torch.isfinite(got["top"]), seen)
        assert torch.all((got["top"].double() - top)[seen].abs() <= (tol + 2.0 ** -22 * top.abs())[seen])


@pytest.mark.parametrize("R,V,K", [(1, 1, 1), (1, 2, 2), (3, 33, 32), (2, 1000, 5), (5, 4096, 0), (7, 4097, 8), (1, 50257, 20), (1, 151936, 32),
                                   (2, 151936, 5), (9, 32003, 1), (40, 8191, 3), (150, 2049, 20), (600, 1027, 2), (1300, 515, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_log_probabilities(R, V, K, dtype):
    x = (rnd(R, V, seed=V + R) * 3).to(dtype)                                 # (bfloat16: ties at every rank)
    tokens = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(R)).to(torch.int32).to(DEV)
    check_logprobs(x, tokens, K)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset,gap", [(0, 1), (1, 0), (3, 5), (8, 16), (5, 3)])
def test_log_probabilities_of_rows_off_any_boundary(offset, gap, dtype):
    R, V = 6, 9001
    flat = (rnd(offset + R * (V + gap), seed=3) * 2).to(dtype)
    x = flat[offset:].view(R, V + gap)[:, :V]
    check_logprobs(x, torch.tensor([0, 1, V - 1, V - 2, 17, 4096], dtype=torch.int32, device=DEV), 20)


@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "one class", "zeros of both signs", "spikes", "mask"])
@pytest.mark.parametrize("V,K", [(9000, 32), (70001, 20)])
def test_log_probabilities_of_ordered_rows(kind, V, K):
    i = torch.arange(V, device=DEV, dtype=torch.float32)
    x = {"mask": torch.where(i % (V // 7) == 3, i * 1e-4, -INF), "equal": torch.zeros_like(i) + 0.25, "rising": i * 1e-3, "falling": -i * 1e-3, "one class": torch.where(i % 1024 == 5, 5 - i * 1e-4, -i * 1e-4),
         "zeros of both signs": torch.where(i % 3 == 0, -0.0, 0.0), "spikes": torch.where(i % 997 == 0, 9.0, 0.0)}[kind]
    check_logprobs(torch.stack([x, x.flip(0)]), torch.tensor([V // 2, V - 1], dtype=torch.int32, device=DEV), K)


def test_log_probabilities_of_an_all_but_certain_token_keep_their_bits():
    V = 5000
    x = rnd(2, V, seed=1)
    x[0, 77] = 30.0
    x[1, 4999] = 60.0
    got = call_logprobs(x, torch.tensor([77, 4999], dtype=torch.int32, device=DEV), 1)
    others = x.double().clone()
    others[0, 77] = others[1, 4999] = -INF
    want = -torch.log1p((others - torch.tensor([[30.0], [60.0]], device=DEV)).exp().sum(dim=1))
    assert torch.all((got["logprob"].double() / want - 1).abs() <= (V / 256 + 80) * 2.0 ** -24 + 60 * 2.0 ** -24)    # (e^-60: an argument's half unit)
    assert torch.equal(got["top"][:, 0], got["logprob"])
    # the others' mass s = sum e^d (7.7e-10 in the first row: 5,000 of e^-30, times e^(1/2)), each some thirty nats away
    d = others - torch.tensor([[30.0], [60.0]], device=DEV)
    H = torch.log1p(d.exp().sum(dim=1)) - torch.where(d > -INF, d.exp() * d, torch.zeros_like(d)).sum(dim=1) / (1 + d.exp().sum(dim=1))
    assert torch.all((got["entropy"].double() / H - 1).abs() <= (V / 256 + 80) * 2.0 ** -23 + 60 * 2.0 ** -24)


def test_log_probabilities_of_masked_and_improper_rows():
    V = 6000
    x = rnd(7, V, seed=2) * 2
    tokens = torch.tensor([3, 3, 5, 5, 5, 5, 4000], dtype=torch.int32, device=DEV)
    x[0, ::2] = -INF                              # a mask
    x[1, torch.arange(V, device=DEV) != 3] = -INF # one token left
    x[2] = -INF                                   # nothing left
    x[3, 100] = NAN
    x[4, 200] = INF
    x[5, 300], x[5, 301] = INF, NAN
    x[6] = torch.finfo(torch.float32).min         # a mask of the type's lowest value, everywhere: uniform
    got = call_logprobs(x, tokens, 8)
    want = torch.log_softmax(x[0].double(), 0)
    assert abs(float(got["logprob"][0]) - float(want[3])) < 1e-5
    assert float(got["logprob"][1]) == 0.0 and float(got["entropy"][1]) == 0.0 and got["ids"][1].tolist() == [3, 0, 1, 2, 4, 5, 6, 7]
    assert got["top"][1].tolist() == [0.0] + [-INF] * 7
    for r in (2, 3, 4, 5):
        assert math.isnan(float(got["logprob"][r])) and math.isnan(float(got["entropy"][r])) and bool(torch.isnan(got["top"][r]).all())
    assert torch.equal(got["ids"].long(), order(x)[:, :8])
    assert int(got["rank"][2]) == 5 and got["ids"][4, 0] == 200 and got["ids"][5, 0] == 300
    assert abs(float(got["logprob"][6]) + math.log(V)) < 1e-5 and abs(float(got["entropy"][6]) - math.log(V)) < 1e-5
    assert int(got["rank"][6]) == 4000


def test_log_probabilities_of_tokens_outside_the_vocabulary():
    o = ops()
    err = o.ErrorFlag(DEV)
    got = call_logprobs(rnd(3, 700, seed=4), torch.tensor([5, 700, -1], dtype=torch.int32, device=DEV), 2, err=err)
    assert torch.isnan(got["logprob"]).tolist() == [False, True, True] and got["rank"][1:].tolist() == [-1, -1]
    assert bool(torch.isfinite(got["entropy"]).all())
    with pytest.raises(o.KernelError):
        err.check("logprobs")


def test_log_probabilities_of_rows_far_apart():
    """Rows that begin beyond 2^32 bytes, and beyond 2^31 elements."""
    gap = (1 << 31) + 8
    pool = torch.empty(2 * gap + 5000, dtype=torch.bfloat16, device=DEV)                   # 8.6 GB
    x = pool.as_strided((3, 5000), (gap, 1))
    x.copy_(rnd(3, 5000, seed=12))
    check_logprobs(x, i32([0, 4999, 77]), 6)


def test_log_probabilities_give_the_same_bits_twice():
    x = rnd(300, 20011, seed=5) * 3
    tokens = torch.arange(300, dtype=torch.int32, device=DEV)
    a, b = call_logprobs(x, tokens, 10), call_logprobs(x, tokens, 10)
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_log_probabilities_leave_what_is_not_asked_for():
    o = ops()
    x, tokens = rnd(4, 3001, seed=6), torch.tensor([1, 2, 3, 4], dtype=torch.int32, device=DEV)
    full = call_logprobs(x, tokens, 3)
    H, lp = torch.empty(4, device=DEV), torch.empty(4, device=DEV)
    o.token_logprobs(x, None, None, entropy=H)
    o.token_logprobs(x, tokens, lp)
    assert torch.equal(H, full["entropy"]) and torch.equal(lp, full["logprob"])
    ids, top = torch.empty((4, 3), dtype=torch.int32, device=DEV), torch.empty((4, 3), device=DEV)
    o.token_logprobs(x, None, None, top_ids=ids, top_logprobs=top)
    assert torch.equal(ids, full["ids"]) and torch.equal(top, full["top"])
    o.token_logprobs(x[:0], tokens[:0], lp[:0])                                # no rows


def test_log_probabilities_refuse():
    o = ops()
    x, t, y = rnd(4, 100), torch.zeros(4, dtype=torch.int32, device=DEV), torch.empty(4, device=DEV)
    ids, top = torch.empty((4, 3), dtype=torch.int32, device=DEV), torch.empty((4, 3), device=DEV)
    for a, kw in [((x.half(), t, y), {}), ((x, t.long(), y), {}), ((x, t[:3], y), {}), ((x, t, y.double()), {}), ((x.t(), t, y), {}),
                  ((x, None, y), {}), ((x[0], t, y), {}), ((x, t, y), dict(top_ids=ids)), ((x, t, y), dict(top_ids=ids, top_logprobs=top[:, :2])),
                  ((x, t, y), dict(top_ids=ids.repeat(1, 11), top_logprobs=top.repeat(1, 11))), ((x[:, :2], t, y), dict(top_ids=ids, top_logprobs=top)),
                  ((x[:1].expand(4, 100), t, y), {})]:
        with pytest.raises(o.KernelError):
            o.token_logprobs(*a, **kw)


# ------------------------------------------------------------------------------------------------ copies
def copied(a, src, dst, slots):
    """The plain form, on a copy."""
    b = a.clone()
    for i, (s, d) in enumerate(zip(src, dst)):
        n = a.shape[2] if a.dim() == 4 and slots is None else (slots[i] if a.dim() == 4 else None)
        if a.dim() == 4:
            b[d, :, :n] = a[s, :, :n]
        else:
            b[d] = a[s]
    return b


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("shapes", [[(9, 2, 16, 64)] * 4, [(9, 4, 32, 128), (9, 4, 32, 64), (9, 1, 32, 40)], [(9, 3, 16, 5), (9, 1, 16, 1), (9, 2, 16, 6)],
                                    [(9, 16, 16, 256)] * 70])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("slots", [None, [1, 16, 0, 7]])
def test_page_copies(shapes, dtype, slots):
    o = ops()
    pool = [rnd(*s, seed=i, dtype=dtype) for i, s in enumerate(shapes)]
    src, dst = [3, 3, 8, 0], [1, 7, 2, 5]
    want = [copied(a, src, dst, slots) for a in pool]
    o.copy_pages(o.PageArrays(pool), i32(src), i32(dst), slots=None if slots is None else i32(slots))
    assert all(torch.equal(a, b) for a, b in zip(pool, want))


@pytest.mark.parametrize("elements", [1, 7, 130, 4096, 1 << 20])
@pytest.mark.parametrize("offset", [0, 1, 2])
def test_state_copies(elements, offset):
    o = ops()
    flat = rnd(offset + 11 * elements, seed=elements)
    pool = flat[offset:].view(11, elements)
    src, dst = [0, 0, 0, 4, 9], [1, 10, 3, 8, 2]
    want = copied(pool, src, dst, None)
    o.copy_pages(o.PageArrays([pool]), i32(src), i32(dst))
    assert torch.equal(pool, want)


def test_many_page_copies_and_none():
    o = ops()
    pool = [rnd(70001, 1, 16, 8, seed=1, dtype=torch.bfloat16)]
    before = pool[0].clone()
    plan = o.PageArrays(pool)
    o.copy_pages(plan, i32([]), i32([]))
    assert torch.equal(pool[0], before)
    src, dst = torch.zeros(70000, dtype=torch.int32, device=DEV), torch.arange(1, 70001, dtype=torch.int32, device=DEV)
    o.copy_pages(plan, src, dst, slots=torch.full_like(src, 9))
    assert torch.equal(pool[0][1:, :, :9], before[:1, :, :9].expand(70000, 1, 9, 8)) and torch.equal(pool[0][:, :, 9:], before[:, :, 9:])


def test_page_copies_far_into_a_cache():
    """Pages whose bytes lie beyond 2^32."""
    o = ops()
    pool = torch.zeros((40000, 4, 16, 1024), dtype=torch.bfloat16, device=DEV)             # 5.2 GB
    pool[39999] = 3.0
    pool[39990, :, 4:] = 2.0
    o.copy_pages(o.PageArrays([pool]), i32([39999, 39990]), i32([0, 39998]), slots=i32([16, 5]))
    assert bool((pool[0] == 3).all()) and bool((pool[39998, :, 4] == 2).all()) and float(pool[39998, :, 5:].abs().max()) == 0


def test_page_copies_outside_the_arrays_are_not_made():
    o = ops()
    pool = [rnd(5, 2, 16, 8, seed=1)]
    want, err = copied(pool[0], [2], [3], None), o.ErrorFlag(DEV)
    o.copy_pages(o.PageArrays(pool), i32([2, 0, -1, 1, 5]), i32([3, 5, 0, -2, 0]), err=err)
    assert torch.equal(pool[0], want)
    with pytest.raises(o.KernelError):
        err.check("copies")


def test_page_copies_refuse():
    o = ops()
    a = rnd(5, 2, 16, 8)
    for bad in ([a, rnd(6, 2, 16, 8)], [a, rnd(5, 2, 32, 8)], [a.transpose(1, 2)], [rnd(5, 2, 8)]):
        with pytest.raises(o.KernelError):
            o.PageArrays(bad)
    plan = o.PageArrays([a])
    for args in ((i32([0]), i32([1, 2])), (i32([0]).long(), i32([1])), (i32([0]), i32([1]), i32([1, 2]))):
        with pytest.raises(o.KernelError):
            o.copy_pages(plan, *args)


# ------------------------------------------------------------------------------------------------ attention
@pytest.fixture(autouse=True, params=[True, False], ids=["shared", "as pays"])
def sharing(request, monkeypatch):
    """The tests' prefixes are short: they are shared whether or not that pays, and once more as it does."""
    if "attention" not in request.node.name and "together" not in request.node.name:
        if not request.param:
            pytest.skip("no attention here")
    elif request.param:
        monkeypatch.setattr(ops(), "attention_sharing_pays", lambda rows, members, groups, *a: groups > 0)


class Case:
    """Rows with tables, keys and values; ``groups``: (rows, shared positions), ``lengths``: positions of every row.  The pages that
    hold shared positions only are one page for the group; a page that a prefix ends in is each row's own, with the same content
    below the end."""

    def __init__(self, Hq, Hkv, D, lengths, groups, page=16, dtype=torch.bfloat16, seed=0, extra=0):
        self.Hq, self.Hkv, self.D, self.page, self.groups, self.lengths = Hq, Hkv, D, page, groups, lengths
        R = len(lengths)
        width = max((n + page - 1) // page for n in lengths) + 2
        for own, n in groups:
            width = max(width, (n + page - 1) // page)
        table = torch.full((R, width), -1, dtype=torch.int64)
        used, lead_of = 0, {}
        for own, n in groups:
            for r in own:
                lead_of[r] = (own[0], n)
            whole = (n + page - 1) // page                # (the leading row holds the whole prefix, whatever its position)
            table[own[0], :whole] = torch.arange(used, used + whole)
            used += whole
            for r in own[1:]:
                table[r, :n // page] = table[own[0], :n // page]
        for r, n in enumerate(lengths):
            for p in range((n + page - 1) // page):
                if table[r, p] < 0:
                    table[r, p] = used
                    used += 1
        perm = torch.randperm(used + extra, generator=torch.Generator().manual_seed(seed))
        self.k, self.v = (rnd(used + extra, Hkv, page, D, seed=seed + s, dtype=dtype) for s in (1, 2))
        self.table = torch.where(table >= 0, perm[table.clamp(min=0)], table).to(torch.int32).to(DEV)
        for r, (lead, n) in lead_of.items():              # the part of a prefix in its last, own page
            if r != lead and n % page and n // page < (lengths[r] + page - 1) // page:
                a, b = int(self.table[lead, n // page]), int(self.table[r, n // page])
                self.k[b, :, :n % page], self.v[b, :, :n % page] = self.k[a, :, :n % page], self.v[a, :, :n % page]
        self.q = rnd(R, (Hq + 2 * Hkv) * D, seed=seed + 3, dtype=dtype) * 1.5
        self.positions = i32([n - 1 for n in lengths])
        self.entry = torch.arange(R, dtype=torch.int32, device=DEV)
        self.scale = 1.0 / math.sqrt(D)

    def run(self, rows=None, groups=None, out=None, shared=None, stale=0.0, **kw):
        o = ops()
        groups = self.groups if groups is None else groups
        R = len(self.lengths) if rows is None else rows.numel()
        shared = o.SharedPrefix(groups, R, DEV) if shared is None else shared
        out = torch.full((len(self.lengths), self.Hq * self.D), stale, dtype=self.k.dtype, device=DEV) if out is None else out
        o.attention_decode_shared(self.q, self.k, self.v, self.table, self.entry, self.positions, self.scale, out, self.Hq, self.Hkv,
                                  self.D, max(self.lengths), shared, rows=rows, **kw)
        return out

    def want(self, sink=None, softcap=0.0, gate=None):
        """Every row by itself in float64, and what bounds the error: sum p |v|, and the largest sum |q k| of a score."""
        R, G = len(self.lengths), self.Hq // self.Hkv
        out = torch.empty(R, self.Hq, self.D, dtype=torch.float64, device=DEV)
        weight, score = torch.empty_like(out), torch.empty(R, self.Hq, 1, dtype=torch.float64, device=DEV)
        for r, n in enumerate(self.lengths):
            pages = self.table[r, :(n + self.page - 1) // self.page].long()
            k, v = (c[pages].double().transpose(0, 1).reshape(self.Hkv, -1, self.D)[:, :n] for c in (self.k, self.v))
            q = self.q[r, :self.Hq * self.D].double().view(self.Hkv, G, self.D)
            s = q @ k.transpose(1, 2) * self.scale
            score[r] = (q.abs() @ k.abs().transpose(1, 2)).amax(2).view(self.Hq, 1) * self.scale
            if softcap > 0:
                s = softcap * torch.tanh(s / softcap)
            if sink is not None:
                s = torch.cat([s, torch.full_like(s[:, :, :1], sink)], 2)
            p = torch.softmax(s, 2)[:, :, :n]
            g = 1.0 if gate is None else torch.sigmoid(gate[r].double()).view(self.Hkv, G, 1)
            out[r] = (p @ v * g).view(self.Hq, self.D)
            weight[r] = (p @ v.abs() * g).view(self.Hq, self.D)
        return out.view(R, -1), weight.view(R, -1), score.expand_as(out).reshape(R, -1)

    def tolerance(self, want, weight, score, softcap=0.0):
        """A score is a sum of D products (relative 2^-24 each, of sum |q k|), a weight its exponential, and a cap adds some units of
        its own size; the output is a sum of such weights.  bfloat16: a weight rounded once and the result rounded once, half a
        unit (2^-8) each."""
        n = max(self.lengths)
        s = (self.D + 8) * 2.0 ** -24 * score + 16 * 2.0 ** -24 * softcap
        tol = (2 * s + (n / 64 + 96) * 2.0 ** -24) * weight
        return tol + (2.0 ** -8 * (weight + want.abs()) if self.k.dtype == torch.bfloat16 else 2.0 ** -24 * want.abs())

    def check(self, sink=None, softcap=0.0, gate=None, **kw):
        got = self.run(sink_score=sink, softcap=softcap, gate=gate, stale=NAN, **kw)
        want, weight, score = self.want(sink, softcap, gate)
        off = (got.double() - want).abs()
        assert bool(torch.isfinite(got).all())
        assert bool((off <= self.tolerance(want, weight, score, softcap)).all()), float((off / self.tolerance(want, weight, score, softcap)).max())


HEADS = [(16, 16, 128, 16), (28, 4, 128, 16), (24, 4, 96, 16), (8, 2, 64, 32), (16, 1, 256, 16), (20, 4, 80, 64), (6, 2, 40, 16), (4, 4, 32, 16),
         (4, 2, 128, 48), (3, 1, 16, 16), (40, 2, 64, 16)]
# rows in no order, rows of their own, a group of one, a row inside its prefix, rows that end with it, odd prefixes
GROUPS = [([([3, 0, 5], 300), ([1, 4], 37), ([6], 64), ([8, 7], 130)], [301, 44, 17, 333, 37, 300, 90, 100, 131, 1]),
          ([(list(range(10)), 160)], [161, 175, 176, 177, 240, 160, 300, 200, 190, 162]),
          ([([0, 1], 0)], [5, 33, 1, 500]), ([], [5, 33, 1, 500])]


@pytest.mark.parametrize("Hq,Hkv,D,page", HEADS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("which", range(len(GROUPS)))
def test_attention_over_shared_prefixes(Hq, Hkv, D, page, dtype, which):
    groups, lengths = GROUPS[which]
    Case(Hq, Hkv, D, lengths, groups, page, dtype, seed=which).check()


@pytest.mark.parametrize("Hq,Hkv,D,page", [(16, 16, 128, 16), (28, 4, 128, 16), (24, 4, 96, 32), (16, 1, 256, 16), (6, 2, 40, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sink,softcap,gated", [(0.7, 0.0, False), (None, 5.0, False), (-3.0, 20.0, True), (None, 0.0, True)])
def test_attention_over_shared_prefixes_with_sink_cap_and_gate(Hq, Hkv, D, page, dtype, sink, softcap, gated):
    groups, lengths = GROUPS[0]
    gate = rnd(len(lengths), Hq + 3, seed=9)[:, 2:2 + Hq] if gated else None
    c = Case(Hq, Hkv, D, lengths, groups, page, dtype, seed=4)
    c.check(sink, softcap, gate)
    c.check(sink, softcap, gate, float_weights=True)


@pytest.mark.parametrize("rows,prefix,Hq,Hkv", [(70, 1000, 4, 4), (33, 513, 28, 4), (19, 2047, 14, 2), (2, 20000, 4, 2), (130, 64, 2, 1), (300, 16, 2, 2)])
def test_attention_over_long_prefixes_and_many_rows(rows, prefix, Hq, Hkv):
    """Tiles that end inside a row's heads, keys that end inside a block, more pages than a block keeps places of."""
    lengths = [prefix + 1 + (r * 37) % 90 for r in range(rows)]
    Case(Hq, Hkv, 128, lengths, [(list(range(rows)), prefix)], seed=rows).check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_of_some_rows_leaves_the_others(dtype):
    groups, lengths = GROUPS[0]
    c = Case(8, 2, 64, lengths, groups, 16, dtype)
    rows = i32([7, 3, 9, 0, 5])                   # batch rows; groups name places among them
    got = c.run(rows=rows, groups=[([1, 3, 4], 300)], stale=3.0)
    want, weight, score = c.want()
    at = rows.long()
    assert bool(((got.double() - want).abs() <= c.tolerance(want, weight, score))[at].all())
    rest = [r for r in range(len(lengths)) if r not in at.tolist()]
    assert bool((got[rest] == 3.0).all())


def test_attention_over_a_prefix_is_the_same_bits_twice_and_near_the_kernel_without_groups():
    o = ops()
    c = Case(28, 4, 128, [700 + 13 * r for r in range(12)], [(list(range(12)), 656)], seed=8)
    a, b = c.run(), c.run()
    assert torch.equal(a, b)
    plain = torch.empty_like(a)
    o.attention_decode(c.q, c.k, c.v, c.table, c.entry, c.positions, c.scale, 0, plain, 28, 4, 128, max(c.lengths))
    want, weight, score = c.want()
    tol = c.tolerance(want, weight, score)
    assert bool(((a.double() - want).abs() <= tol).all()) and bool(((plain.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.bfloat16, 40), (torch.float32, 128)])
def test_attention_with_infinities_and_nan_where_no_row_looks(dtype, D):
    """Slots behind a row's position, and pages that no row holds, may hold anything."""
    groups, lengths = [([0, 1, 2], 40)], [41, 55, 47]
    c = Case(4, 2, D, lengths, groups, 16, dtype, extra=3)
    want, weight, score = c.want()
    used = torch.zeros(c.k.shape[0], c.page, dtype=torch.bool, device=DEV)
    for r, n in enumerate(lengths):
        for j in range(n):
            used[int(c.table[r, j // 16]), j % 16] = True
    bad = torch.tensor([NAN, INF, -INF], device=DEV).to(dtype)
    for x in (c.k, c.v):
        x.copy_(torch.where(used[:, None, :, None], x, bad[torch.arange(16, device=DEV) % 3][None, None, :, None]))
    got = c.run(stale=NAN)
    assert bool(((got.double() - want).abs() <= c.tolerance(want, weight, score)).all())


@pytest.mark.parametrize("D,page", [(64, 16), (80, 32), (96, 64), (128, 32), (256, 16)])
@pytest.mark.parametrize("sink", [None, 0.5])
def test_attention_with_infinities_and_nan_behind_the_rows_ends(D, page, sink):
    """The same for the other head and page sizes, with a row that ends where its prefix does and one without a prefix."""
    lengths = [page * 2, page * 4 + 9, page * 3 + 1, 5, page * 2 + page // 2]
    c = Case(6, 2, D, lengths, [([0, 1, 2, 4], page * 2)], page, extra=2)
    want, weight, score = c.want(sink)
    used = torch.zeros(c.k.shape[0], page, dtype=torch.bool, device=DEV)
    for r, n in enumerate(lengths):
        for j in range(n):
            used[int(c.table[r, j // page]), j % page] = True
    bad = torch.tensor([NAN, INF, -INF], device=DEV).to(c.k.dtype)
    for x in (c.k, c.v):
        x.copy_(torch.where(used[:, None, :, None], x, bad[torch.arange(page, device=DEV) % 3][None, None, :, None]))
    got = c.run(stale=NAN, sink_score=sink)
    assert bool(((got.double() - want).abs() <= c.tolerance(want, weight, score)).all())


def test_attention_of_queries_off_any_boundary():
    c = Case(8, 2, 64, *GROUPS[0][::-1])
    q = torch.empty(c.q.numel() + 4, dtype=c.q.dtype, device=DEV)[4:].view_as(c.q)
    c.q = q.copy_(c.q)
    assert c.q.data_ptr() % 16 == 8
    c.check()


def test_attention_of_many_rows_with_long_keys_of_their_own():
    """More keys in a split than a warp keeps places of."""
    lengths = [2100 + r % 40 for r in range(520)]
    Case(4, 2, 64, lengths, [([0, 1], 16)]).check()


def test_attention_on_two_streams_at_once():
    c, d = (Case(16, 16, 128, [500 + r for r in range(8)], [(list(range(8)), 480)], seed=s) for s in (1, 2))
    alone = c.run(), d.run()
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(5):
        for s, x in zip(streams, (c, d)):
            with torch.cuda.stream(s):
                got.append((x is d, x.run()))
    torch.cuda.synchronize()
    assert all(torch.equal(out, alone[which]) for which, out in got)


def test_attention_by_arrays_with_room_for_more_rows_and_groups():
    """One object whose arrays are replaced by those of other groups, as steps of a captured shape replace them."""
    o = ops()
    groups, lengths = GROUPS[0]
    c = Case(8, 2, 64, lengths, groups)
    facts = o.SharedPrefix.facts(groups, 10)
    pack = lambda g: i32(o.SharedPrefix.pack(g, 10, 7)[0])
    shared = o.SharedPrefix(groups[:1], 10, DEV, facts=facts, room=(10, 7), buf=pack(groups[:1]))
    want, weight, score = c.want()
    for g in (groups[:1], groups, groups[1:3]):
        shared.bind(pack(g))
        shared.reach = 300
        got = c.run(shared=shared, stale=NAN)
        assert bool(((got.double() - want).abs() <= c.tolerance(want, weight, score)).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_far_into_a_cache(dtype):
    """Pages whose bytes lie beyond 2^32."""
    c = Case(8, 2, 128, [70, 81, 66, 90], [([0, 1, 2], 64)], 16, dtype)
    n = (1 << 32) // (2 * 16 * 128 * c.k.element_size()) + 50
    far = torch.arange(c.k.shape[0], device=DEV) * 3 + n - 3 * c.k.shape[0]
    k, v = (torch.zeros((n, 2, 16, 128), dtype=dtype, device=DEV) for _ in range(2))
    k[far], v[far] = c.k, c.v
    c.k, c.v, c.table = k, v, torch.where(c.table >= 0, far[c.table.clamp(min=0).long()].to(torch.int32), c.table)
    c.check()


def test_attention_reports_a_missing_page():
    o = ops()
    for dtype, D in ((torch.bfloat16, 128), (torch.float32, 64)):
        c = Case(4, 2, D, [200, 210], [([0, 1], 192)], 16, dtype)
        c.table[0, 3] = -1
        err = o.ErrorFlag(DEV)
        c.run(err=err)
        with pytest.raises(o.KernelError):
            err.check("shared")


def test_attention_refuses():
    o = ops()
    c = Case(4, 2, 64, [40, 50], [([0, 1], 32)])
    two, three = o.SharedPrefix(c.groups, 2, DEV), o.SharedPrefix(c.groups, 3, DEV)
    out = torch.empty(2, 256, dtype=torch.bfloat16, device=DEV)

    def call(q=c.q, k=c.k, v=c.v, scale=0.1, out=out, Hq=4, Hkv=2, D=64, shared=two, **kw):
        o.attention_decode_shared(q, k, v, c.table, c.entry, c.positions, scale, out, Hq, Hkv, D, 50, shared, **kw)

    call()
    for kw in (dict(q=c.q.float()), dict(k=c.k.float()), dict(out=out.float()), dict(out=out[:, :128].contiguous()), dict(Hq=3), dict(D=32),
               dict(shared=three), dict(scale=0.0), dict(scale=-1.0), dict(softcap=-1.0), dict(q=c.q[:, :128].contiguous()),
               dict(shared=o.SharedPrefix([([0, 1], 16 * c.table.shape[1] + 16)], 2, DEV)), dict(v=c.v[:-1]), dict(k=c.k.transpose(1, 2)), dict(Hkv=1), dict(gate=torch.zeros(2, 3, device=DEV))):
        with pytest.raises(o.KernelError):
            call(**kw)


def test_attention_of_no_rows():
    o = ops()
    c = Case(4, 2, 64, [40, 50], [([0, 1], 32)])
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    got = c.run(rows=none, groups=[], stale=2.0)
    assert bool((got == 2.0).all()) and o.SharedPrefix([], 0, DEV).buf.numel() == 1


def test_attention_captured_twice_and_replayed_side_by_side():
    """Two captures of the operator, each with a scratch of its own, replayed on two streams at once with new queries."""
    cases = [Case(16, 4, 64, [300 + 7 * r for r in range(6)], [(list(range(6)), 288)], seed=s) for s in (1, 2)]
    plans, outs, graphs = [], [], []
    for c in cases:
        plans.append(ops().SharedPrefix(c.groups, 6, DEV))
        outs.append(c.run(shared=plans[-1]))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.run(shared=plans[-1], out=outs[-1])
        graphs.append(g)
    for k in range(3):
        for i, c in enumerate(cases):
            c.q.copy_(rnd(*c.q.shape, seed=100 + 2 * k + i, dtype=torch.bfloat16))
        torch.cuda.synchronize()
        streams = torch.cuda.Stream(), torch.cuda.Stream()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(4):
                    g.replay()
        torch.cuda.synchronize()
        for c, out in zip(cases, outs):
            want, weight, score = c.want()
            assert bool(((out.double() - want).abs() <= c.tolerance(want, weight, score)).all())


# ------------------------------------------------------------------------------------------------ the three together
@pytest.mark.parametrize("captured", [False, True])
def test_fork_decode_and_rank_together(captured):
    """A request of 90 positions forked into five: its part-full page copied for each, a key and value written behind the fork,
    attention over the shared pages, and the log probabilities of given tokens under logits made from it; eager, and as a
    replayed graph whose inputs change."""
    o = ops()
    Hq, Hkv, D, page, n, replies, V = 8, 2, 64, 16, 90, 5, 3001
    full = n // page
    k, v = rnd(40, Hkv, page, D, seed=1, dtype=torch.bfloat16), rnd(40, Hkv, page, D, seed=2, dtype=torch.bfloat16)
    table = torch.full((replies, 8), -1, dtype=torch.int32)
    table[:, :full] = torch.arange(full, dtype=torch.int32) + 3
    table[:, full] = torch.tensor([20, 21, 22, 23, 24])
    table = table.to(DEV)
    plan, shared = o.PageArrays([k, v]), o.SharedPrefix([(list(range(replies)), full * page)], replies, DEV)
    src, dst, slots = i32([20] * 4), i32([21, 22, 23, 24]), i32([n - full * page] * 4)
    q = rnd(replies, (Hq + 2 * Hkv) * D, seed=3, dtype=torch.bfloat16)
    newest = rnd(2, replies, Hkv, D, seed=4, dtype=torch.bfloat16)
    head = rnd(Hq * D, V, seed=5) * 0.05
    tokens = i32([1, 2, 3, 4, 5])
    positions, entry = i32([n] * replies), torch.arange(replies, dtype=torch.int32, device=DEV)
    out = torch.empty(replies, Hq * D, dtype=torch.bfloat16, device=DEV)
    lp, ids, top = torch.empty(replies, device=DEV), torch.empty((replies, 4), dtype=torch.int32, device=DEV), torch.empty((replies, 4), device=DEV)
    logits = torch.empty(replies, V, device=DEV)

    def step():
        o.copy_pages(plan, src, dst, slots=slots)
        pages = table[:, full].long()
        k[pages, :, n % page], v[pages, :, n % page] = newest[0], newest[1]
        o.attention_decode_shared(q, k, v, table, entry, positions, D ** -0.5, out, Hq, Hkv, D, n + 1, shared)
        torch.mm(out.float(), head, out=logits)
        o.token_logprobs(logits, tokens, lp, top_ids=ids, top_logprobs=top)

    def check():
        for r in range(replies):
            kk, vv = (torch.cat([c[3:3 + full].transpose(0, 1).reshape(Hkv, -1, D), c[20, :, :n % page], newest[i, r][:, None]], 1).double()
                      for i, c in enumerate((k, v)))
            p = torch.softmax(q[r, :Hq * D].double().view(Hkv, -1, D) @ kk.transpose(1, 2) * D ** -0.5, 2)
            want = (p @ vv).reshape(-1)
            assert bool(((out[r].double() - want).abs() <= 2.0 ** -8 * ((p @ vv.abs()).reshape(-1) + want.abs()) + 1e-5).all())
        want = torch.log_softmax(logits.double(), 1)
        assert float((lp.double() - want.gather(1, tokens[:, None].long())[:, 0]).abs().max()) <= 100 * 2.0 ** -24 * 10
        assert torch.equal(ids.long(), order(logits)[:, :4])

    step()
    check()
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for seed in (11, 12):
            q.copy_(rnd(*q.shape, seed=seed, dtype=torch.bfloat16))
            newest.copy_(rnd(*newest.shape, seed=seed + 50, dtype=torch.bfloat16))
            k[20].copy_(rnd(Hkv, page, D, seed=seed + 90, dtype=torch.bfloat16))
            tokens.copy_(i32([seed, 0, V - 1, 7, 8]))
            graph.replay()
            torch.cuda.synchronize()
            check()
