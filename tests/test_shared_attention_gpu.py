"""Decode attention over shared prefixes where rows, groups and launches must keep apart: queries that are no numbers beside
healthy ones, groups of different lengths."""
import math

import pytest
import torch

from test_reply_operators_gpu import Case, i32, ops, rnd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF, NAN = math.inf, math.nan


@pytest.fixture(autouse=True)
def always_shared(monkeypatch):
    """The tests' prefixes are short: they are shared whether or not that pays."""
    monkeypatch.setattr(ops(), "attention_sharing_pays", lambda rows, members, groups, *a: groups > 0)


# ------------------------------------------------------------------------------------------------ rows keep to themselves
@pytest.mark.parametrize("Hq,Hkv,D", [(28, 4, 128), (24, 4, 96), (8, 2, 64), (16, 1, 256)])
@pytest.mark.parametrize("float_weights", [False, True])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_a_query_that_is_no_number_stays_in_its_row(Hq, Hkv, D, float_weights, bad):
    """A long and a short group: most splits have no keys of the short one, whose rows fill a tile with a bad one among them."""
    lengths = [2050 + r for r in range(12)] + [70 + 3 * r for r in range(16)]
    c = Case(Hq, Hkv, D, lengths, [(list(range(12)), 2048), (list(range(12, 28)), 64)])
    want, weight, score = c.want()
    tol = c.tolerance(want, weight, score)
    healthy = torch.tensor([r for r in range(28) if r != 17], device=DEV)
    clean = c.run(float_weights=float_weights)
    c.q[17] = bad
    for _ in range(50):
        got = c.run(float_weights=float_weights, stale=3.0)
        assert torch.equal(got[healthy], clean[healthy]) and bool(torch.isnan(got[17]).all())
    assert bool(((clean.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("Hq,Hkv,D,page", [(8, 2, 64, 16), (28, 4, 128, 32), (6, 2, 112, 16), (4, 2, 40, 16)])
@pytest.mark.parametrize("captured", [False, True])
def test_arrays_without_groups_behind_the_kernel_that_writes_the_queries(Hq, Hkv, D, page, captured):
    """A call with room for groups, bound to arrays that have none (a step whose last family has ended), waits for the kernel in
    front, which is still at work on the queries when the call's kernels may begin."""
    o = ops()
    lengths = [5, 33, 170, 64]
    c = Case(Hq, Hkv, D, lengths, [([0, 1], page), ([2, 3], page)], page)
    shared = o.SharedPrefix(c.groups, 4, DEV, room=(4, 2))
    shared.bind(i32(o.SharedPrefix.pack([], 4, 2)[0]))
    x, w = rnd(4, 16384, seed=7, dtype=torch.bfloat16), rnd(c.q.shape[1], 16384, seed=8, dtype=torch.bfloat16) / 128
    out = torch.empty(4, Hq * D, dtype=torch.bfloat16, device=DEV)

    def step():
        c.q.fill_(NAN)
        o.gemm_plain(x, w, c.q)
        c.run(shared=shared, out=out)

    step()
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        step = graph.replay
    for k in range(20):
        x.copy_(rnd(4, 16384, seed=20 + k, dtype=torch.bfloat16))
        out.fill_(NAN)
        step()
        torch.cuda.synchronize()
        want, weight, score = c.want()
        assert bool(((out.double() - want).abs() <= c.tolerance(want, weight, score)).all())


@pytest.mark.parametrize("Hq,Hkv,D", [(28, 4, 128), (8, 2, 64), (6, 2, 112), (6, 2, 40), (16, 1, 256)])
@pytest.mark.parametrize("captured", [False, True])
def test_layers_one_after_the_other_in_the_same_buffers(Hq, Hkv, D, captured):
    """As a step's layers call it: the product in front writes the queries into one buffer, over those of the layer before, and the
    calls' scratch is the same memory; no layer takes the queries, parts or sums of another."""
    o = ops()
    lengths = [700 + 13 * r for r in range(8)] + [40, 3]
    c = Case(Hq, Hkv, D, lengths, [(list(range(8)), 656)])
    shared, layers, q = o.SharedPrefix(c.groups, 10, DEV), 12, c.q
    xs = [rnd(10, 2048, seed=s, dtype=torch.bfloat16) for s in range(layers)]
    w = rnd(q.shape[1], 2048, seed=99, dtype=torch.bfloat16) / 45
    outs = [torch.empty(10, Hq * D, dtype=torch.bfloat16, device=DEV) for _ in range(layers)]

    def step():
        for x, out in zip(xs, outs):
            o.gemm_plain(x, w, q)
            c.run(shared=shared, out=out)

    step()
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        step = graph.replay
    for _ in range(5):
        for out in outs:
            out.fill_(NAN)
        step()
    torch.cuda.synchronize()
    for x, out in zip(xs, outs):
        c.q = torch.empty_like(q)
        o.gemm_plain(x, w, c.q)
        want, weight, score = c.want()
        assert bool(((out.double() - want).abs() <= c.tolerance(want, weight, score)).all())


# ------------------------------------------------------------------------------------------------ pages that are not there
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.bfloat16, 112), (torch.float32, 64)])
def test_the_c_entry_without_an_error_flag_passes_a_missing_page_by(dtype, D):
    """Nobody is told, and nothing else happens: rows that do not read the page have their results."""
    o = ops()
    c = Case(4, 2, D, [200, 210, 90], [([0, 1], 192)], 16, dtype)
    c.table[0, 3] = -1
    shared, out = o.SharedPrefix(c.groups, 3, DEV), torch.empty(3, 4 * D, dtype=dtype, device=DEV)
    scratch = torch.empty(3 * 4 * 2 * (D + 2), dtype=torch.float32, device=DEV)
    first, group, members, cu, lens, leads = shared.places
    dt = o.dt(c.q)
    assert o.lib().nv_attention_decode_shared(c.q.data_ptr(), dt, c.q.shape[1], c.k.data_ptr(), c.v.data_ptr(), dt, c.table.data_ptr(),
                                              c.table.shape[1], c.entry.data_ptr(), c.positions.data_ptr(), None, 3, first, group, members, 2,
                                              cu, lens, leads, 1, c.scale, out.data_ptr(), dt, 4, 2, D, 16, c.k.shape[0], 1, 1,
                                              scratch.data_ptr(), None, 0, 0.0, 0, 0.0, None, 0, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    c.table[0, 3] = 0
    want, weight, score = c.want()
    assert bool(((out.double() - want).abs() <= c.tolerance(want, weight, score))[2].all())


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.bfloat16, 112), (torch.float32, 64)])
def test_bound_arrays_that_reach_beyond_the_block_tables(dtype, D):
    """Refused where ``bind`` says how far they reach; else reported, and the rows, which end inside the tables, have their results."""
    o = ops()
    c = Case(4, 2, D, [160, 150, 33, 130], [([0, 1, 2], 160)], 16, dtype)
    c.table = c.table[:, :10].contiguous()
    shared = o.SharedPrefix(c.groups, 4, DEV)
    far = i32(o.SharedPrefix.pack([([0, 1, 2], 100000)], 4)[0])
    shared.bind(far, reach=100000)
    with pytest.raises(o.KernelError):
        c.run(shared=shared)
    want, weight, score = c.want()
    for bound in (True, False):
        shared.bind(far if bound else i32(o.SharedPrefix.pack(c.groups, 4)[0]))
        shared.buf.copy_(far)                                               # (a replaced content, as steps of one shape replace it)
        err = o.ErrorFlag(DEV)
        got = c.run(shared=shared, err=err)
        assert bool(((got.double() - want).abs() <= c.tolerance(want, weight, score)).all())
        with pytest.raises(o.KernelError):
            err.check("shared")


# ------------------------------------------------------------------------------------------------ precision
@pytest.mark.parametrize("Hq,Hkv,D", [(28, 4, 128), (24, 4, 96), (8, 2, 64), (16, 1, 256), (6, 2, 112)])
@pytest.mark.parametrize("grouped", [True, False])
def test_a_cap_beside_a_sink_costs_no_bits(Hq, Hkv, D, grouped):
    """A cap far above the scores: its function is the identity there, and an error in units of the cap would be one of 2 % in a weight
    or more.  Weights keep all their bits beside a sink; tanhf is off by two units of its result at most, the scale and the cap by
    half a unit each, within the eight units of a score that the tolerance holds beside the products' own."""
    lengths = [301, 44, 17, 333, 37, 300, 90, 100, 131, 1]
    c = Case(Hq, Hkv, D, lengths, [([3, 0, 5], 300), ([8, 7], 96)] if grouped else [], seed=6)
    got = c.run(sink_score=0.5, softcap=1e5, stale=NAN)
    want, weight, score = c.want(sink=0.5, softcap=1e5)
    assert bool(((got.double() - want).abs() <= c.tolerance(want, weight, score)).all())


@pytest.mark.parametrize("Hq,Hkv,D", [(28, 4, 128), (8, 2, 64), (16, 1, 256)])
@pytest.mark.parametrize("softcap", [0.5, 2.0, 8.0])
def test_caps_among_the_scores(Hq, Hkv, D, softcap):
    """Scores on both sides of half the cap and far beyond it: the cap's function is a series below and an exponential above."""
    lengths = [301, 44, 17, 333, 37, 300, 90, 100, 131, 1]
    c = Case(Hq, Hkv, D, lengths, [([3, 0, 5], 300), ([8, 7], 96)], seed=11)
    got = c.run(sink_score=-0.5, softcap=softcap, stale=NAN)
    want, weight, score = c.want(sink=-0.5, softcap=softcap)
    assert bool(((got.double() - want).abs() <= c.tolerance(want, weight, score)).all())
