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
