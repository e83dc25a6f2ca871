"""The oracle of filtered sampling and acceptance against its definition, by
hand and by counting (CPU)."""

import math

import numpy as np
import pytest

from oracle.filtered import Row, accept


def test_order_and_ties():
    r = Row([1.0, 3.0, 2.0, 3.0, -np.inf], temperature=1.0, top_k=3)
    assert r.kept()[0].tolist() == [1, 3, 2]
    assert Row([1.0, 3.0, 3.0], top_k=1).kept()[0].tolist() == [1]
    assert [Row([0.0] * 4).sample(u) for u in (0.0, 0.2499, 0.25, 0.5, 0.9999)] == [0, 0, 1, 2, 3]


def test_top_p_takes_the_fewest_that_reach_it():
    x = np.log([0.5, 0.3, 0.15, 0.05])
    assert [Row(x, top_p=p).n for p in (0.0, 0.49, 0.51, 0.79, 0.81, 0.94, 0.96, 1.0)] == [1, 1, 2, 2, 3, 3, 4, 4]
    assert Row([0.0] * 10, top_p=0.5).n == 5
    # of what top-k left: 0.5 of 0.8 is 0.625
    assert Row(x, top_k=2, top_p=0.62).n == 1 and Row(x, top_k=2, top_p=0.63).n == 2


def test_min_p_and_rows_of_one_token():
    x = np.log([0.5, 0.3, 0.15, 0.05])
    assert [Row(x, min_p=m).n for m in (0.0, 0.09, 0.11, 0.29, 0.31, 0.61, 1.0, 2.0)] == [4, 4, 3, 3, 2, 1, 1, 1]
    assert Row([np.nan, 1.0]).sample(0.9) == 0 and Row([-np.inf] * 3).sample(0.9) == 0
    assert Row([1.0, 2.0, 2.0], temperature=0.0).sample(0.99) == 1
    assert Row([np.inf, 0.0, np.inf]).kept()[1].tolist() == [1.0, 1.0, 0.0]


def test_admits_agrees_with_sample():
    x = np.random.default_rng(3).normal(size=200) * 2
    for u in (0.0, 0.3, 0.77, 0.999):
        r = Row(x, 0.8, 50, 0.9, 0.01)
        assert r.admits(r.n, r.sample(u), u, 1e-12) is None
        assert r.admits(r.n + 1, r.sample(u), u, 1e-12) and r.admits(r.n, int(r.order[-1]), u, 1e-12)


@pytest.mark.parametrize("setting", [dict(), dict(top_k=3), dict(top_p=0.8), dict(min_p=0.2), dict(top_k=4, top_p=0.9)])
def test_accepted_tokens_follow_the_filtered_target(setting):
    """Over a fine grid of uniform numbers the first token's frequencies are
    the filtered target's: drafts drawn from the filtered draft row."""
    rng = np.random.default_rng(11)
    target, draft = rng.normal(size=(2, 6)) * 1.5, rng.normal(size=(1, 6)) * 1.5
    want, q = Row(target[0], 0.7, **setting).probabilities(), Row(draft[0], 0.7, **setting).probabilities()
    got = np.zeros(6)
    grid = (np.arange(200) + 0.5) / 200
    for d in np.flatnonzero(q):
        for u in grid:
            hits = [accept(target, draft, [int(d)], [u, v], 0.7, **setting)[0] for v in grid[::8]]
            got += q[d] * np.bincount(hits, minlength=6) / len(hits) / len(grid)
    # each of the two grids resolves a probability to half its step, for each of up to 6 drafts
    assert np.abs(got - want).max() <= 6 * (0.5 / 200 + 0.5 / 25)
    assert math.isclose(got.sum(), 1.0, rel_tol=1e-12)


def test_row_samples_where_there_are_no_draft_rows():
    x = np.log([[0.6, 0.4], [0.1, 0.9], [0.5, 0.5]])
    assert accept(x, None, [0, 1], [0.5, 0.5, 0.7]) == [0, 1, 1]
    assert accept(x, None, [1, 1], [0.5, 0.5, 0.7]) == [0]
    assert accept(x, x[:2], [0, 0], [0.99, 0.99, 0.2], temperature=0.0) == [0, 1]
    assert accept(x, x[:2], [7, 0], [0.0, 0.0, 0.2]) == [0]  # no token: refused; no residual, the target itself
