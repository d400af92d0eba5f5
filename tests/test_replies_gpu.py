"""Several replies to one prompt through the engine: forked caches go on as if each request had run by itself, replies are those of
requests of their own, log probabilities are those of the logits, and rows that share a prefix keep their results."""
import math

import pytest
import torch

import helpers
import plain_bizodra
import plain_sevelorn
import test_bizodra_gpu
import test_sevelorn_gpu
from helpers import prompt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    out = {c: helpers.model_folder(c, tmp_path_factory) for c in ("A", "C", "D")}
    biz, sev = test_bizodra_gpu, test_sevelorn_gpu
    cfg = biz.CONFIGS["P"]                              # recurrent states beside pages, a convolution's kept inputs
    out["P"] = plain_bizodra.write_folder(cfg, plain_bizodra.random_weights(cfg, 3), str(tmp_path_factory.mktemp("P")))
    cfg = sev.CONFIGS["R"]                              # states, a convolution before every mixer, keys of an earlier call
    out["R"] = plain_sevelorn.write_folder(cfg, plain_sevelorn.make_weights(cfg, 7), str(tmp_path_factory.mktemp("R")))
    return out


VOCAB = {"P": 210, "R": 344}


def ids_for(case, n, salt=0):
    if case in VOCAB:
        g = torch.Generator().manual_seed(31 * n + salt)
        return [int(t) for t in torch.randint(0, VOCAB[case], (n,), generator=g)]
    return prompt(case, n, salt=salt)


def engine(mdir, **kw):
    from nano_vllm_cpp_b200 import LLMEngine
    kw.setdefault("dtype", "float32")
    kw.setdefault("max_num_seqs", 12)
    return LLMEngine(mdir, kw.pop("max_model_len", 256), kw.pop("num_kv_blocks", 160), log_stats=False, **kw)


def make_runner(mdir, dtype, max_tokens=2048, max_requests=12, **kw):
    from nano_vllm_cpp_b200.engine.runner import ModelRunner
    return ModelRunner(mdir, dtype=dtype, max_tokens=max_tokens, max_requests=max_requests, max_model_len=512, **kw)


def entry(rid, tokens, want=None):
    from nano_vllm_cpp_b200.engine.batch import StepEntry
    return StepEntry(rid, tokens, list(range(len(tokens))) if want is None else want)


@pytest.fixture
def always_shared(monkeypatch):
    """The models here are small: their prefixes are shared whether or not that pays."""
    from nano_vllm_cpp_b200.csrc import ops
    monkeypatch.setattr(ops, "attention_sharing_pays", lambda rows, members, groups, *a: groups > 0)


# ------------------------------------------------------------------------------------------------ forks
@pytest.mark.parametrize("case", ["A", "C", "P", "R"])
@pytest.mark.parametrize("n", [1, 16, 43, 64])
def test_forked_requests_go_on_by_themselves(case, n, folders):
    """float32, where a row's sums do not depend on its batch: the parent and two forks go on with tokens of their own, one
    fork of a fork later, and give the bits of requests that ran the same tokens from the start."""
    r = make_runner(folders[case], "float32")
    base, tails = ids_for(case, n), [ids_for(case, 21, salt=s) for s in (1, 2, 3, 4)]
    r.step([entry("a", base)])
    r.fork("a", ["b", "c"])
    r.manager.check()
    got = {x: [] for x in "abcd"}
    for k in range(9):
        logits = r.step([entry(x, [tails[i][k]]) for i, x in enumerate("abc")])
        for i, x in enumerate("abc"):
            got[x].append(logits[i].clone())
    r.fork("b", ["d"])
    for k in range(9, 21):
        row = dict(zip("abcd", r.step([entry(x, [tails[i][k]]) for i, x in enumerate("abcd")])))
        for x in "abcd":
            got[x].append(row[x].clone())
    r.manager.check()
    for x in "abcd":
        r.close(x)
    r.manager.check()
    for i, x in enumerate("abcd"):
        own = tails[i] if x != "d" else tails[1][:9] + tails[3][9:]
        r.step([entry("alone", base, [])])
        want = torch.cat([r.step([entry("alone", [t])]).clone() for t in own])      # (a captured step keeps one tensor)
        r.close("alone")
        have = torch.stack(got[x])
        assert torch.equal(have, want[-len(have):]), (x, float((have - want[-len(have):]).abs().max()))


def test_a_fork_of_all_or_none(folders):
    from nano_vllm_cpp_b200.cache import NoFreeSlot
    r = make_runner(folders["A"], "float32", max_requests=3)
    r.step([entry("a", ids_for("A", 20))])
    free = r.manager.pools[0].num_free()
    with pytest.raises(NoFreeSlot):
        r.fork("a", ["b", "c", "d"])
    assert r.manager.pools[0].num_free() == free and r.manager.free_slots() == 2 and not r.manager.has("b")
    r.fork("a", ["b", "c"])
    r.manager.check()


# ------------------------------------------------------------------------------------------------ replies
@pytest.mark.parametrize("case", ["A", "C", "D", "P"])
@pytest.mark.parametrize("sampling", [dict(temperature=0.0), dict(temperature=0.9, seed=11),
                                      dict(temperature=0.8, seed=5, top_p=0.8, repetition_penalty=1.3)])
def test_replies_are_those_of_requests_of_their_own(case, sampling, folders):
    from nano_vllm_cpp_b200 import SamplingParams
    prompts = [ids_for(case, n, salt=7) for n in (5, 37, 64)]
    eng = engine(folders[case], prefill_chunk=24)
    outs = eng.generate(prompts, SamplingParams(n=3, max_tokens=14, ignore_eos=True, **sampling))
    eng.runner.manager.check()
    assert eng.runner.manager.free_slots() == 12 and len(outs) == 3
    for p, o in zip(prompts, outs):
        assert len(o["replies"]) == 3 and o["replies"][0]["token_ids"] == o["token_ids"]
        for i, reply in enumerate(o["replies"]):
            own = dict(sampling, **({"seed": sampling["seed"] + i} if "seed" in sampling else {}))
            alone = eng.generate([p], SamplingParams(max_tokens=14, ignore_eos=True, **own))
            assert reply["token_ids"] == alone[0]["token_ids"], (len(p), i)


@pytest.mark.parametrize("room", [dict(num_kv_blocks=9), dict(max_num_seqs=2)])
def test_replies_without_room_for_forks_run_their_prompt_again(room, folders):
    from nano_vllm_cpp_b200 import SamplingParams
    p = ids_for("A", 37, salt=3)
    sp = dict(temperature=0.9, seed=4, max_tokens=12, ignore_eos=True)
    small = engine(folders["A"], max_model_len=64, enable_prefix_caching=False, **room)
    out = small.generate([p, p], SamplingParams(n=4, **sp))
    small.runner.manager.check()
    roomy = engine(folders["A"])
    for o in out:
        assert [x["token_ids"] for x in o["replies"]] == [roomy.generate([p], SamplingParams(**dict(sp, seed=4 + i)))[0]["token_ids"] for i in range(4)]


def test_replies_of_one_token_and_of_stop_tokens(folders):
    from nano_vllm_cpp_b200 import SamplingParams
    p = ids_for("A", 20, salt=5)
    eng = engine(folders["A"])
    first = [eng.generate([p], SamplingParams(temperature=1.0, seed=s, max_tokens=1))[0]["token_ids"] for s in (3, 4, 5)]
    out = eng.generate([p], SamplingParams(temperature=1.0, seed=3, max_tokens=1, n=3))
    assert [x["token_ids"] for x in out[0]["replies"]] == first
    assert eng.runner.manager.free_slots() == 12
    stop = engine(folders["A"], eos=first[1][0])
    out = stop.generate([p], SamplingParams(temperature=1.0, seed=3, max_tokens=6, n=3))[0]["replies"]
    assert out[1]["token_ids"] == first[1] and len(out[0]["token_ids"]) >= 1
    stop.runner.manager.check()
    assert stop.runner.manager.free_slots() == 12


def test_replies_beside_other_requests(folders):
    """Requests with and without further replies, log probabilities and the nucleus rule, in one run, and some added later."""
    from nano_vllm_cpp_b200 import SamplingParams
    sps = [SamplingParams(temperature=0.0, max_tokens=10, ignore_eos=True), SamplingParams(temperature=0.7, seed=2, max_tokens=7, n=2, ignore_eos=True),
           SamplingParams(temperature=0.7, seed=9, top_p=0.7, max_tokens=9, logprobs=2, ignore_eos=True),
           SamplingParams(temperature=0.0, max_tokens=5, n=3, logprobs=1, ignore_eos=True)]
    prompts = [ids_for("C", n, salt=n) for n in (30, 12, 50, 33)]
    eng = engine(folders["C"], max_num_batched_tokens=48)
    outs = eng.generate(prompts, sps)
    assert [("replies" in o, "logprobs" in o) for o in outs] == [(False, False), (True, False), (False, True), (True, True)]
    for p, sp, o in zip(prompts, sps, outs):
        for i, reply in enumerate(o.get("replies", [o])):
            alone = engine(folders["C"]).generate([p], SamplingParams(temperature=sp.temperature, seed=None if sp.seed is None else sp.seed + i,
                                                                     top_p=sp.top_p, max_tokens=sp.max_tokens, ignore_eos=True))
            assert reply["token_ids"] == alone[0]["token_ids"]
            if sp.logprobs is not None:
                assert [s.token for s in reply["logprobs"]] == reply["token_ids"] and {len(s.top) for s in reply["logprobs"]} == {sp.logprobs}


# ------------------------------------------------------------------------------------------------ log probabilities
def check_scores(scores, tokens, logits, top):
    """Against float64 over the engine's own logits: some hundred terms of a sum, each rounded a few times."""
    lp = torch.log_softmax(logits.double(), dim=1).cpu()
    order = logits.double().cpu().sort(dim=1, descending=True, stable=True).indices
    assert len(scores) == len(tokens) == len(lp)
    for s, t, row, ids in zip(scores, tokens, lp, order):
        assert s.token == t and abs(s.logprob - float(row[t])) <= 1e-5
        assert s.rank == int((ids == t).nonzero()) and abs(s.entropy - float(torch.special.entr(row.exp()).sum())) <= 1e-5
        assert [i for i, _ in s.top] == ids[:top].tolist() and all(abs(p - float(row[i])) <= 1e-5 for i, p in s.top)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("run_ahead", [True, False])
def test_log_probabilities_of_a_reply(dtype, run_ahead, folders):
    from nano_vllm_cpp_b200 import SamplingParams
    p = ids_for("D", 19, salt=2)
    eng = engine(folders["D"], dtype=dtype, run_ahead=run_ahead)
    out = eng.generate([p, p[:7]], SamplingParams(temperature=0.8, seed=3, max_tokens=12, logprobs=5, ignore_eos=True))
    plain = eng.generate([p], SamplingParams(temperature=0.8, seed=3, max_tokens=12, ignore_eos=True))
    assert "logprobs" not in plain[0] and (dtype == "bfloat16" or plain[0]["token_ids"] == out[0]["token_ids"])
    for ids, o in zip((p, p[:7]), out):
        logits = eng.runner.step([entry("x", ids, [len(ids) - 1])])
        rows = [logits.clone()]
        for t in o["token_ids"][:-1]:
            rows.append(eng.runner.step([entry("x", [t])]).clone())
        eng.runner.close("x")
        if dtype == "float32":
            check_scores(o["logprobs"], o["token_ids"], torch.cat(rows), 5)
        else:                                            # (another batch's logits: their roundings move the numbers)
            lp = torch.log_softmax(torch.cat(rows).double(), 1).cpu()
            assert all(abs(s.logprob - float(row[s.token])) <= 0.1 for s, row in zip(o["logprobs"], lp))


@pytest.mark.parametrize("n", [1, 2, 33, 100])
def test_scores_of_given_tokens(n, folders):
    eng = engine(folders["C"], max_num_batched_tokens=40)
    ids = ids_for("C", n, salt=6)
    scores = eng.score([ids, ids[:1]], top=4)
    assert scores[1] == []
    eng.runner.manager.check()
    assert eng.runner.manager.free_slots() == 12
    logits = eng.runner.step([entry("x", ids)])
    eng.runner.close("x")
    check_scores(scores[0], ids[1:], logits[:-1], 4)
    for bad in (dict(prompts=[[]]), dict(prompts=[[1] * 300]), dict(prompts=[ids], top=33), dict(prompts=[ids], top=-1)):
        with pytest.raises(ValueError):
            eng.score(**bad)
    with pytest.raises(Exception):
        eng.score([[0, 10 ** 6]])
    assert eng.runner.manager.free_slots() == 12


# ------------------------------------------------------------------------------------------------ shared prefixes
@pytest.mark.parametrize("graphs", [False, True])
def test_steps_whose_rows_share_prefixes(graphs, folders, always_shared):
    """bfloat16: two families of forks and a lone request decode beside one another, as launched steps and as replayed ones, while
    members leave; every row's logits are those of the run that shares nothing, within the tolerance of the dtype."""
    runners = [make_runner(folders["D"], "bfloat16", shared_prefix=s, cuda_graphs=graphs) for s in (True, False)]
    shared = []
    inner = runners[0]._shared_rows
    runners[0]._shared_rows = lambda entries: shared.append(inner(entries)) or shared[-1]
    a, b = ids_for("D", 150, salt=1), ids_for("D", 70, salt=2)
    for r in runners:
        r.step([entry("a0", a, []), entry("b0", b, []), entry("c0", ids_for("D", 40, salt=3), [])])
        r.fork("a0", ["a1", "a2", "a3"])
        r.fork("b0", ["b1"])
    live = ["b0", "a2", "c0", "a0", "a3", "b1", "a1"]
    tokens = {x: ids_for("D", 24, salt=10 + i) for i, x in enumerate(live)}
    for k in range(24):
        if k == 12:
            for r in runners:
                r.close("a0")                            # the leading request of its family in the step's order goes on without it
            live.remove("a0")
        got, want = (r.step([entry(x, [tokens[x][k]]) for x in live]).double().cpu() for r in runners)
        assert float((got - want).abs().max()) <= 2e-2 + 3e-2 * float(want.abs().max())
    assert shared[1] == ([([0, 5], 64), ([1, 3, 4, 6], 144)], 7) and shared[-1] == ([([0, 4], 64), ([1, 3, 5], 144)], 6)
    assert bool(runners[0]._graphs) == graphs
    # a step of portions beside single rows
    mixed = [entry("new", ids_for("D", 20, salt=50))] + [entry(x, [tokens[x][0]]) for x in live]
    got, want = (r.step(mixed).double().cpu() for r in runners)
    assert float((got - want).abs().max()) <= 2e-2 + 3e-2 * float(want.abs().max())
    assert shared[-1] == ([([0, 4], 64), ([1, 3, 5], 144)], 6)


@pytest.mark.parametrize("limit", [32, 1, 0])
def test_captured_steps_whose_families_change_size(limit, folders, always_shared, monkeypatch):
    """Ten replies and a lone request, then nine and two: one captured shape.  Shapes beyond the limit run as if nothing was shared.
    The results are those of a run that launches the same operators (another operator's rounding may turn a router's near tie)."""
    from nano_vllm_cpp_b200.engine import runner
    monkeypatch.setattr(runner, "MAX_SHARED_GRAPHS", limit)
    runners = [make_runner(folders["D"], "bfloat16", shared_prefix=s, cuda_graphs=g) for s, g in ((True, True), (limit > 0, False))]
    for r in runners:
        r.step([entry("a0", ids_for("D", 70, salt=1), []), entry("c0", ids_for("D", 40, salt=3), [])])
        r.fork("a0", [f"a{i}" for i in range(1, 10)])
    live = ["c0"] + [f"a{i}" for i in range(10)]
    for k in range(9):
        if k == 3:
            for r in runners:
                r.close("a4")
                r.step([entry("c1", ids_for("D", 33, salt=7), [])])
            live[live.index("a4")] = "c1"
        if k == 6:
            for r in runners:
                r.close("c1")
                r.fork("c0", ["c2"])
            live[live.index("c1")] = "c2"                # (two groups: another shape)
        step = [entry(x, [ids_for("D", 9, salt=20 + i)[k]]) for i, x in enumerate(live)]
        got, want = (r.step(step).double().cpu() for r in runners)
        assert float((got - want).abs().max()) <= 2e-2 + 3e-2 * float(want.abs().max())
    captured = [g[-1] is not None for g in runners[0]._graphs.values()]
    assert captured == {32: [True, True], 1: [True, False], 0: [False]}[limit]


@pytest.mark.parametrize("case", ["C", "R"])
def test_models_with_windows_and_states_share_what_they_can(case, folders, always_shared):
    """Layers with a window keep to themselves; layers that read another's keys share as it does."""
    runners = [make_runner(folders[case], "bfloat16", shared_prefix=s, cuda_graphs=False) for s in (True, False)]
    ids = ids_for(case, 100, salt=4)
    outs = []
    for r in runners:
        r.step([entry("a", ids, [])])
        r.fork("a", ["b", "c"])
        outs.append(torch.cat([r.step([entry(x, [ids_for(case, 8, salt=i)[k]]) for i, x in enumerate("abc")]).double().cpu() for k in range(8)]))
    scale = float(outs[1].abs().max())
    assert float((outs[0] - outs[1]).abs().max()) <= 2e-2 + 4e-2 * scale


def test_replies_with_shared_prefixes_follow_the_plain_model(folders, always_shared):
    from nano_vllm_cpp_b200 import SamplingParams
    p = ids_for("D", 90, salt=8)
    eng = engine(folders["D"], dtype="bfloat16", shared_prefix=True)
    used = []
    inner = eng.runner._shared_rows
    eng.runner._shared_rows = lambda e: used.append(inner(e)) or used[-1]
    out = eng.generate([p, p[:50] + [1, 2, 3]], SamplingParams(n=4, temperature=0.0, max_tokens=16, ignore_eos=True, logprobs=0))
    assert any(u is not None and len(u[0]) >= 1 for u in used) and eng.runner._graphs
    for ids, o in zip((p, p[:50] + [1, 2, 3]), out):
        for reply in o["replies"]:
            assert helpers.assert_greedy_follows_plain(folders["D"], ids, reply["token_ids"], "bfloat16", "shared") >= 3
            assert all(math.isfinite(s.logprob) and s.top == [] for s in reply["logprobs"])


def test_a_float32_run_shares_nothing(folders):
    assert make_runner(folders["D"], "float32", shared_prefix=True)._whole_group is None


def test_the_command_line_prints_replies_and_scores(folders, capsys):
    from nano_vllm_cpp_b200 import cli
    args = [folders["A"], "--tokens", "1,2,3", "--max-tokens", "4", "--dtype", "float32", "--max-model-len", "64", "--num-kv-blocks", "16",
            "--max-num-seqs", "4", "--temperature", "0", "--ignore-eos"]
    assert cli.main(args + ["--n", "2", "--logprobs", "3", "--shared-prefix"]) == 0
    lines = capsys.readouterr().out.splitlines()
    assert sum(line.startswith("token_ids: ") for line in lines) == 2 and sum("entropy" in line for line in lines) == 8
    assert cli.main(args + ["--score", "--logprobs", "1"]) == 0
    lines = capsys.readouterr().out.splitlines()
    assert len(lines) == 3 and lines[-1].startswith("sum: -")
