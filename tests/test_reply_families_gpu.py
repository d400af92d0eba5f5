"""Families of replies behind one system prompt, and replies whose forks and first tokens come beside other requests' steps."""
import pytest
import torch

from test_replies_gpu import always_shared, engine, entry, folders, ids_for, make_runner      # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graphs", [False, True])
def test_families_behind_one_system_prompt_share_their_prompts(graphs, folders, always_shared):
    """bfloat16: three families behind 48 common tokens and one request that parts from them early; every row's logits are those of the
    run that shares nothing, within the tolerance of the dtype."""
    runners = [make_runner(folders["D"], "bfloat16", shared_prefix=s, cuda_graphs=graphs) for s in (True, False)]
    shared = []
    inner = runners[0]._shared_rows
    runners[0]._shared_rows = lambda entries: shared.append(inner(entries)) or shared[-1]
    for r in runners:
        r.step([entry("system", ids_for("D", 48, salt=1), [])])
        for f, n in enumerate((100, 64, 33)):
            r.fork("system", [f"{f}0"])
            r.step([entry(f"{f}0", ids_for("D", n, salt=2 + f), [])])
            r.fork(f"{f}0", [f"{f}{k}" for k in range(1, 3)])
        r.fork("system", ["early"])
    live = ["10", "00", "21", "early", "11", "01", "20", "02", "12", "22"]
    for k in range(12):
        step = [entry(x, [ids_for("D", 12, salt=20 + i)[k]]) for i, x in enumerate(live)]
        got, want = (r.step(step).double().cpu() for r in runners)
        assert float((got - want).abs().max()) <= 2e-2 + 3e-2 * float(want.abs().max())
    assert shared[-1] == ([([0, 4, 8], 112), ([1, 5, 7], 144), ([2, 6, 9], 80)], 10)
    assert bool(runners[0]._graphs) == graphs


@pytest.fixture
def copies(monkeypatch):
    """How many copies each launch made."""
    from nano_vllm_cpp_b200.csrc import ops
    made, inner = [], ops.copy_pages
    monkeypatch.setattr(ops, "copy_pages", lambda arrays, src, dst, **kw: made.append(src.numel()) or inner(arrays, src, dst, **kw))
    return made


@pytest.mark.parametrize("case,launches", [("A", [9]), ("P", [9, 9])])
def test_the_forks_of_a_step_are_copied_together(case, launches, folders, copies):
    """Three prompts that one step completes, four replies each: one launch per cache group and state buffer."""
    from nano_vllm_cpp_b200 import SamplingParams
    prompts = [ids_for(case, n, salt=7) for n in (5, 37, 50)]
    eng = engine(folders[case])
    outs = eng.generate(prompts, SamplingParams(n=4, temperature=0.9, seed=11, max_tokens=6, ignore_eos=True))
    assert copies == launches[:1] * len(eng.runner.cache.windows) + launches[1:] * len(eng.runner.cache.state_buffers)
    for p, o in zip(prompts, outs):
        for i, reply in enumerate(o["replies"]):
            alone = eng.generate([p], SamplingParams(temperature=0.9, seed=11 + i, max_tokens=6, ignore_eos=True))
            assert reply["token_ids"] == alone[0]["token_ids"], (len(p), i)
    eng.runner.manager.check()


def test_prompts_of_whole_pages_copy_nothing(folders, copies):
    from nano_vllm_cpp_b200 import SamplingParams
    eng = engine(folders["A"])
    eng.generate([ids_for("A", 32), ids_for("A", 64)], SamplingParams(n=3, temperature=0.5, seed=1, max_tokens=3, ignore_eos=True))
    assert copies == []


def test_forks_for_which_there_is_room(folders, copies):
    """A family is opened as far as slots go; nothing stays open where the copies fail."""
    r = make_runner(folders["A"], "float32", max_requests=5)
    r.step([entry("a", ids_for("A", 20)), entry("b", ids_for("A", 30))])
    r.fork_replies([("a", ["a1", "a2"]), ("b", ["b1", "b2", "b3"])])
    assert copies == [3] and [r.manager.has(x) for x in ("a1", "a2", "b1", "b2", "b3")] == [True, True, True, False, False]
    r.manager.check()
    for x in ("a1", "a2", "b1"):
        r.close(x)
    free = r.manager.pools[0].num_free()

    def refuse(*a):
        raise RuntimeError("no copies")

    r.cache.copy_forks = refuse
    with pytest.raises(RuntimeError, match="no copies"):
        r.fork_replies([("a", ["a1"]), ("b", ["b1"])])
    assert r.manager.free_slots() == 3 and r.manager.pools[0].num_free() == free
    r.manager.check()


@pytest.mark.parametrize("late", [dict(top_p=0.7, temperature=0.9, seed=3), dict(n=2, temperature=0.9, seed=3)])
def test_told_tokens_are_those_of_the_results(late, folders):
    """A request ends by its stop token while the step behind is under way, and a request that wants the plain order comes just then:
    what the steps report as new tokens is what the sequences hold."""
    from nano_vllm_cpp_b200 import SamplingParams
    p = ids_for("A", 20, salt=5)
    stop = engine(folders["A"]).generate([p], SamplingParams(temperature=1.0, seed=3, max_tokens=8, ignore_eos=True))[0]["token_ids"]
    at = next(i for i in range(3, 8) if stop[i] not in stop[:i])
    eng = engine(folders["A"], eos=stop[at])
    for after in range(1, at + 3):
        told, done = {}, {}
        first = eng.add_request(p, SamplingParams(temperature=1.0, seed=3, max_tokens=20))
        eng.add_request(ids_for("A", 30, salt=6), SamplingParams(temperature=0.0, max_tokens=20, ignore_eos=True))
        steps = 0
        while not eng.is_finished():
            out = eng.step()
            steps += 1
            for seq_id, token in out.new_tokens:
                told.setdefault(seq_id, []).append(token)
            done.update(out.finished)
            if steps == after:
                eng.add_request(ids_for("A", 9, salt=7), SamplingParams(max_tokens=6, ignore_eos=True, **late))
        assert done[first] == stop[:at + 1] and told == done, after


def test_steps_run_ahead_while_prompts_with_replies_wait(folders):
    """Two requests hold all slots while three prompts with further replies wait: only the steps that complete such a prompt are followed
    in the plain order.  Every reply is that of a request of its own, and the tokens told step by step are the results'."""
    from nano_vllm_cpp_b200 import SamplingParams
    eng = engine(folders["C"], max_num_seqs=2, max_num_batched_tokens=64)
    counted = dict(ahead=0)
    inner = eng._stand_ins

    def stand_ins(cur):
        assert not cur.replies
        counted["ahead"] += 1
        inner(cur)

    eng._stand_ins = stand_ins
    long = [eng.add_request(ids_for("C", n, salt=2), SamplingParams(temperature=0.0, max_tokens=30, ignore_eos=True)) for n in (20, 31)]
    sps = [SamplingParams(temperature=0.8, seed=4 + 10 * k, n=2 + k % 2, max_tokens=8, ignore_eos=True, logprobs=k % 2 or None) for k in range(3)]
    prompts = [ids_for("C", n, salt=3) for n in (70, 33, 12)]
    first = [eng.add_request(p, sp) for p, sp in zip(prompts, sps)]
    told, done = {}, {}
    for step in range(29):
        out = eng.step()
        done.update(out.finished)
        for seq_id, token in out.new_tokens:
            told.setdefault(seq_id, []).append(token)
    assert counted["ahead"] >= 28
    while not eng.is_finished():
        out = eng.step()
        done.update(out.finished)
        for seq_id, token in out.new_tokens:
            told.setdefault(seq_id, []).append(token)
    assert counted["ahead"] > 28 and told == done and len(done) == 2 + 2 + 3 + 2
    eng.runner.manager.check()
    alone = engine(folders["C"])
    for p, sp, q in zip(prompts, sps, first):
        for i in range(sp.n):
            own = SamplingParams(temperature=0.8, seed=sp.seed + i, max_tokens=8, ignore_eos=True)
            assert done[q + i] == alone.generate([p], own)[0]["token_ids"]
    assert done[long[0]] == alone.generate([ids_for("C", 20, salt=2)], SamplingParams(temperature=0.0, max_tokens=30, ignore_eos=True))[0]["token_ids"]
