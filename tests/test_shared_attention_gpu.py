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
