"""Calls of the operators for several continuations of a request that their documentation allows and the tests beside them do
not make. Tolerances, derived before the first run, stand at each test."""

import numpy as np
import pytest

from test_gpu_decode import kda_make
from test_gpu_move import run as move_run
from test_gpu_tree import check_rows, run_tree, tree64, wild

pytestmark = pytest.mark.gpu


# ---- the recurrence over trees --------------------------------------------------------------------------------------


@pytest.mark.parametrize("most", [1, 5, 16, 20, 24, 32, 40, 63])
@pytest.mark.parametrize("requests", [2, 67])
def test_more_nodes_than_stated_are_skipped_whatever_the_batch(cuda, most, requests):
    """Trees of max_nodes nodes and of one and several more, in a batch that runs at once and in a larger one: the latter are
    skipped with status 1 and their rows left."""
    rng = np.random.default_rng(most)
    H = 5
    for over in (1, min(64, most + 16) - most):
        sizes = [most] * requests
        sizes[1] = most + over
        ends = np.cumsum([0] + sizes)
        trees = [wild(rng, n) for n in sizes]
        d = kda_make(rng, int(ends[-1]), H, 3)
        seqs = [(int(ends[r]), int(ends[r + 1]), r % 3, 1) for r in range(requests)]
        out, status = run_tree(cuda, d, H, seqs, sum(trees, []), max_nodes=most)
        assert status == 1
        assert (out[ends[1]:ends[2]] == -77.0).all()
        pick = [0, 2, requests - 1] if requests > 2 else [0]
        want = tree64(d, [seqs[r] for r in pick], [trees[r] for r in pick], H)
        for r in pick:
            check_rows(out[ends[r]:ends[r + 1]], want[ends[r]:ends[r + 1]], H)


# ---- moves ----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("n", [2, 40])
def test_an_entry_past_the_view_does_not_take_a_destination(cuda, n):
    """An entry that moves nothing because its source is past the rows is not the first of its destination."""
    src = np.full((1, 1, n), -1, np.int32)
    dst = np.full((1, 1, n), -1, np.int32)
    src[0, 0, [0, n - 1]], dst[0, 0, [0, n - 1]] = [9, 1], [3, 3]
    got, want, status, between = move_run(cuda, [(8, 64), (12, 4096)], [0, 0], src, dst, pitch=16)
    assert status == 1 and between
    assert all((g == w).all() for g, w in zip(got, want))
