"""Forks in the cache manager and the scheduler, common prefixes of requests, and what sampling parameters refuse; no GPU."""
import random

import pytest

from nano_vllm_cpp_b200.cache import CacheManager, NoFreePages, NoFreeSlot
from nano_vllm_cpp_b200.config import SamplingParams
from nano_vllm_cpp_b200.engine.scheduler import Scheduler
from nano_vllm_cpp_b200.engine.sequence import Sequence, SequenceStatus


def run(m, rid, n):
    """n more tokens of a request."""
    at = m.get(rid).num_tokens
    m.extend(rid, at, at + n)
    m.commit(rid, at + n)


@pytest.mark.parametrize("n", [1, 15, 16, 17, 48, 50])
def test_a_fork_shares_full_pages_and_copies_the_part_full_one(n):
    m = CacheManager([0], 20, 16, 4)
    m.open(5)
    run(m, 5, n)
    before = m.get(5).tables[0]
    f = m.fork(5, 9)
    a, b = m.get(5), m.get(9)
    assert b.num_tokens == n and a.tables[0] == before and (f.slot_from, f.slot_to) == (a.slot, b.slot) and a.slot != b.slot
    assert b.tables[0][:n // 16] == before[:n // 16]
    if n % 16:
        assert f.pages == [(0, before[-1], b.tables[0][-1], n % 16)] and b.tables[0][-1] != before[-1]
    else:
        assert f.pages == [] and b.tables[0] == before
    m.check()
    run(m, 5, 20)
    run(m, 9, 40)                               # each goes on by itself
    m.check()
    assert m.get(5).tables[0][:n // 16] == m.get(9).tables[0][:n // 16] and not set(m.get(5).tables[0][n // 16:]) & set(m.get(9).tables[0][n // 16:])
    m.close(5)
    m.check()
    m.close(9)
    m.check()
    assert m.pools[0].num_free() == 20


def test_forks_of_windows_chunks_and_kept_positions():
    m = CacheManager([0, 32, (32, 4), ("chunk", 64)], 40, 16, 6)
    m.open("a")
    for k in (70, 30, 1, 27):
        run(m, "a", k)
    n = 128
    f = m.fork("a", "b")
    assert f.pages == [] and m.get("b").tables == m.get("a").tables        # (a multiple of the page)
    m.check()
    for k in range(40):
        run(m, "a", 1)
        run(m, "b", 1)
        m.check()
    f = m.fork("b", ("c", 1))
    assert len(f.pages) == 4 and {p[3] for p in f.pages} == {(n + 40) % 16} and {p[0] for p in f.pages} == {0, 1, 2, 3}
    for rid in ("a", ("c", 1), "b"):
        run(m, rid, 100)
        m.check()
    for rid in ("b", "a", ("c", 1)):
        m.close(rid)
        m.check()


def test_a_fork_that_finds_no_room_changes_nothing():
    m = CacheManager([0], 4, 16, 2)
    m.open(1)
    run(m, 1, 60)
    with pytest.raises(NoFreePages):
        m.fork(1, 2)
    m.check()
    assert not m.has(2) and m.free_slots() == 1
    m.close(1)
    m.open(1)
    run(m, 1, 20)
    m.fork(1, 2)
    with pytest.raises(NoFreeSlot):
        m.fork(1, "x")
    assert not m.has("x")
    with pytest.raises(KeyError):
        m.fork("nobody", "y")
    with pytest.raises(RuntimeError):
        m.fork(1, 2)
    m.check()


def test_a_request_without_pages_forks_its_slot():
    m = CacheManager([], [], 16, 3, has_state=True)
    m.open(1)
    f = m.fork(1, 2)
    assert f.pages == [] and f.slot_from != f.slot_to
    m.check()


def test_forks_and_hashed_pages():
    m = CacheManager([0], 30, 16, 8, prefix_caching=True)
    tokens = list(range(100))
    m.open(1)
    m.extend(1, 0, 40)
    m.commit(1, 40, tokens[:40])
    m.fork(1, 2)
    for rid, more in ((1, tokens[40:64]), (2, [7] * 24)):
        m.extend(rid, 40, 64)
        m.commit(rid, 64, tokens[:40] + more)
    m.check()
    assert [p for p, _ in m.match_prefix(tokens[:64] + [0])] == m.get(1).tables[0]
    assert [p for p, _ in m.match_prefix(tokens[:40] + [7] * 24 + [0])] == m.get(2).tables[0]
    m.close(2)
    m.close(1)
    m.check()


def common(tables, fulls):
    """The plain rule: requests with one first page; as many pages as all of them have in common."""
    out, seen = [], {}
    for i, (t, full) in enumerate(zip(tables, fulls)):
        if full:
            seen.setdefault(t[0], []).append(i)
    for members in seen.values():
        if len(members) > 1:
            n = min(fulls[i] for i in members)
            k = 0
            while k < n and len({tables[i][k] for i in members}) == 1:
                k += 1
            out.append((members, k))
    return sorted(out)


def test_common_prefixes_of_forks_against_the_plain_rule():
    rnd = random.Random(3)
    for _ in range(60):
        m = CacheManager([0], 400, 16, 40)
        live = []
        for k in range(rnd.randint(1, 14)):
            if live and rnd.random() < 0.7:
                m.fork(rnd.choice(live), k)
            else:
                m.open(k)
            live.append(k)
            for rid in live:
                if rnd.random() < 0.5:
                    run(m, rid, rnd.randint(1, 40))
        rnd.shuffle(live)
        want = common([m.get(r).tables[0] for r in live], [m.get(r).num_tokens // 16 for r in live])
        got = m.shared_prefixes(live, 0)
        assert sorted(got) == [(members, n * 16) for members, n in want]
        assert [g[0][0] for g in got] == sorted(g[0][0] for g in got) and m.shared_prefixes([], 0) == []


def test_replies_join_the_running_queue_or_wait():
    m = CacheManager([0], 8, 16, 3)
    s = Scheduler(m, max_num_seqs=3, max_num_batched_tokens=256, max_model_len=128)
    parent = Sequence(list(range(20)), SamplingParams(n=3, max_tokens=5, ignore_eos=True))
    assert [q.seq_id for q in parent.replies] == [parent.seq_id + 1, parent.seq_id + 2] and not parent.forked and parent.replies[0].forked
    s.add(parent)
    step = s.schedule()
    assert [(x.start, x.count, x.samples) for x in step] == [(0, 20, True)]
    m.commit(parent.seq_id, 20)
    m.fork(parent.seq_id, parent.replies[0].seq_id)                    # the second reply found no room, say
    assert s.postprocess(step, {parent.seq_id: 100}) == []
    for q, t in zip(parent.replies, (101, 102)):
        q.token_ids.append(t)
        s.add_reply(q)
    assert [q.status for q in [parent] + parent.replies] == [SequenceStatus.RUNNING, SequenceStatus.RUNNING, SequenceStatus.WAITING]
    step = s.schedule()
    assert [(x.seq.seq_id - parent.seq_id, x.start, x.count) for x in step] == [(0, 20, 1), (1, 20, 1), (2, 0, 21)]
    done = s.postprocess(step, {x.seq.seq_id: 7 for x in step})
    n = 1
    while not s.is_finished():
        step = s.schedule()
        done += s.postprocess(step, {x.seq.seq_id: 7 for x in step})
        n += 1
    assert n == 4 and sorted(q.seq_id - parent.seq_id for q in done) == [0, 1, 2]
    assert [q.completion_token_ids for q in [parent] + parent.replies] == [[t, 7, 7, 7, 7] for t in (100, 101, 102)]
    m.check()
    assert m.pools[0].num_free() == 8 and m.free_slots() == 3


def test_replies_draw_from_streams_of_their_own():
    a = Sequence([1], SamplingParams(n=3, seed=40))
    assert [q.seed for q in [a] + a.replies] == [40, 41, 42]
    b = Sequence([1], SamplingParams(n=4), base_seed=2)
    assert len({q.seed for q in [b] + b.replies}) == 4
    assert Sequence([1], SamplingParams(seed=9)).seed == 9 and Sequence([1], SamplingParams()).replies == []


@pytest.mark.parametrize("kw", [dict(n=0), dict(n=-1), dict(logprobs=-1), dict(logprobs=33)])
def test_sampling_parameters_refuse(kw):
    with pytest.raises(ValueError):
        SamplingParams(**kw).validate()


def test_sampling_parameters_take():
    for kw in (dict(n=5), dict(logprobs=0), dict(logprobs=32), dict(logprobs=None)):
        SamplingParams(**kw).validate()


def test_requests_that_are_not_open_share_nothing():
    """Names that the manager does not know, beside the request that was named first."""
    m = CacheManager([0], 20, 16, 4)
    m.open("first")
    run(m, "first", 40)
    assert m.shared_prefixes(["first", "nobody", 7, ("nor", 1)], 0) == []
    m.fork("first", "second")
    assert m.shared_prefixes(["nobody", "second", 7, "first"], 0) == [([1, 3], 32)]
    m.close("first")
    assert m.shared_prefixes(["first", "second", "nobody"], 0) == []


def least_read(tables, fulls):
    """What sets save at most, in pages: every way to put the requests into sets is tried."""
    def common(members):
        n = min(fulls[i] for i in members)
        k = 0
        while k < n and len({tables[i][k] for i in members}) == 1:
            k += 1
        return k

    def ways(rest):
        if not rest:
            return 0
        first, others = rest[0], rest[1:]
        most = ways(others)
        for mask in range(1, 1 << len(others)):
            members = [first] + [x for b, x in enumerate(others) if mask >> b & 1]
            n = common(members)
            if n:
                most = max(most, (len(members) - 1) * n + ways([x for b, x in enumerate(others) if not mask >> b & 1]))
        return most
    return ways(list(range(len(tables)))), common


@pytest.mark.parametrize("seed", range(40))
def test_best_sets_of_forks_against_every_way_to_make_them(seed):
    rnd = random.Random(seed)
    m = CacheManager([0], 400, 16, 40)
    live = []
    for k in range(rnd.randint(2, 7)):
        if live and rnd.random() < 0.85:
            m.fork(rnd.choice(live), k)
        else:
            m.open(k)
        live.append(k)
        for rid in live:
            if rnd.random() < 0.5:
                run(m, rid, rnd.randint(1, 60))
    rnd.shuffle(live)
    tables, fulls = [m.get(r).tables[0] for r in live], [m.get(r).num_tokens // 16 for r in live]
    most, pages_of = least_read(tables, fulls)
    got = m.shared_prefixes(live, 0, best=True)
    assert sum((len(members) - 1) * n for members, n in got) == most * 16
    members = [i for own, _ in got for i in own]
    assert len(members) == len(set(members)) and all(len(own) > 1 and own == sorted(own) and 0 < n == 16 * pages_of(own) for own, n in got)
    assert [own[0] for own, _ in got] == sorted(own[0] for own, _ in got)


def test_families_behind_one_system_prompt_are_sets_of_their_own():
    """Eight prompts of 2,064 tokens that begin with the same 64, eight replies each: by first pages one set of 64 with 64 positions."""
    m = CacheManager([0], 4000, 16, 80)
    m.open("system")
    run(m, "system", 64)
    rids = []
    for f in range(8):
        m.fork("system", (f, 0))
        run(m, (f, 0), 2000)
        for r in range(1, 8):
            m.fork((f, 0), (f, r))
        rids += [(f, r) for r in range(8)]
    random.Random(1).shuffle(rids)
    for rid in rids:
        run(m, rid, 30)
    assert m.shared_prefixes(rids, 0) == [(list(range(64)), 64)]
    got = m.shared_prefixes(rids, 0, best=True)
    assert sorted(n for _, n in got) == [2064] * 8 and all(len({rids[i][0] for i in own}) == 1 and len(own) == 8 for own, _ in got)
    # requests that part from them early, and a lone one behind the system prompt
    m.fork("system", "early")
    run(m, "early", 20)
    m.fork((3, 0), "late")
    more = rids + ["early", "late"]
    got = m.shared_prefixes(more, 0, best=True)
    assert sorted((len(own), n) for own, n in got) == [(8, 2064)] * 7 + [(9, 2064)] and 64 not in [i for own, _ in got for i in own]
    # two that have more in common with one another than with their family, which is better off whole
    run(m, "late", 40)
    m.fork("late", "later")
    got = m.shared_prefixes(rids + ["late", "later"], 0, best=True)
    assert sorted((len(own), n) for own, n in got) == [(8, 2064)] * 7 + [(10, 2064)]


def test_best_sets_of_many_requests_that_part_one_after_the_other():
    m = CacheManager([0], 4000, 16, 300)
    m.open(0)
    for k in range(1, 300):
        run(m, k - 1, 16)
        m.fork(k - 1, k)
    got = m.shared_prefixes(list(range(300)), 0, best=True)
    # request k holds k + 1 pages (the last k): those from a on, with a + 1 pages in common, save (299 - a) (a + 1), more below
    assert sum((len(own) - 1) * n for own, n in got) >= 16 * 150 * 150 and m.shared_prefixes([], 0, best=True) == []
