"""Calls of the operators for several continuations of a request that their documentation allows and the tests beside
them do not make. Tolerances, derived before the first run, stand at each test."""

import gc

import numpy as np
import pytest
import torch

from test_gpu_beam import run as beam_run
from test_gpu_decode import D, kda_make
from test_gpu_move import run as move_run
from test_gpu_tree import check_rows, run_tree, tree64, wild
from test_gpu_verify_stage import cfg

pytestmark = pytest.mark.gpu


# ---- the recurrence over trees --------------------------------------------------------------------------------------


@pytest.mark.parametrize("most", [1, 5, 16, 20, 24, 32, 40, 63])
@pytest.mark.parametrize("requests", [2, 67])
def test_more_nodes_than_stated_are_skipped_whatever_the_batch(cuda, most, requests):
    """Trees of max_nodes nodes and of one and several more, in a batch that runs at once and in a larger one: the
    latter are skipped with status 1 and their rows left."""
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


@pytest.mark.parametrize("size", [3.0, 100.0])
def test_states_far_larger_than_the_outputs(cuda, size):
    """A node's value takes the place of what the state has for its key, and its query is that key: the output is the
    value's, a small difference of products of the state. The state and the vectors enter their product as two bf16
    parts (2^-9, and 2^-9 of that is what they leave), high x high, high x low and low x high: a product s x is off
    by 3 x 2^-18 |s x| at most, and the tensor core's sums by another 2^-18 of the magnitudes: 2^-16. The two
    products (with k and with q, the first's share weighted by k . q) make it twice that of the magnitudes' sum,
    beside the bf16 store's 2^-8 and the tests' 1e-3 of the row's largest for the rest."""
    rng = np.random.default_rng(int(size))
    H, n = 2, 6
    P = H * D
    d = kda_make(rng, n, H, 1)
    d["rst"] = (rng.standard_normal((1, H, D, D)) * size).astype(np.float32)
    d["x"][:, :P] = d["x"][:, P:2 * P]                       # queries as keys, through the same conv
    d["w"][:P] = d["w"][P:2 * P]
    d["cst"][:, :, :P] = d["cst"][:, :, P:2 * P]
    d["g"][:] = -30.0                                        # decays of 1
    d["beta"][:] = 30.0                                      # the state's value for the key is replaced
    to_bf16 = lambda v: torch.from_numpy(np.ascontiguousarray(v)).to(torch.bfloat16).float().numpy()
    d = {k: to_bf16(v) if k in ("g", "beta", "x") else v for k, v in d.items()}
    tree, seqs = [-1] * n, [(0, n, 0, 1)]
    want = tree64(d, seqs, [tree], H).reshape(n, H, D)
    out, status = run_tree(cuda, d, H, seqs, tree)
    assert status == 0
    out = out.reshape(n, H, D)
    # the keys' magnitudes times the state's: at most the 2-norm of the state's row (the key's is 1)
    mass = np.linalg.norm(d["rst"][0].astype(np.float64), axis=2) * D ** -0.5
    bar = 2.0 ** -8 * np.abs(want) + 1e-3 * np.abs(want).max(axis=2, keepdims=True) + 2 * 2.0 ** -16 * mass
    assert (np.abs(out - want) <= bar).all(), (np.abs(out - want) / bar).max()


# ---- beam selection -------------------------------------------------------------------------------------------------


def lse_errors(cuda, x, bf16=False):
    """Rows x as requests of one beam whose score makes the best candidate's about 0, where float32 is fine: the
    kernel's log sums less the true ones, and the largest logits."""
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.bfloat16 if bf16 else torch.float32)
    x = t.double().numpy()
    top = x.max(axis=1)
    lse = top + np.log(np.exp(x - top[:, None]).sum(axis=1))
    given = (lse - top).astype(np.float32)
    s, p, v = beam_run(cuda, t, given[:, None], 1, bf16=bf16)
    assert (v[:, 0] == x.argmax(axis=1)).all()
    return (given.astype(np.float64) + top - lse) - s[:, 0], given, s[:, 0]


@pytest.mark.parametrize("V", [700, 5003, 32768, 151552])
@pytest.mark.parametrize("bf16", [False, True])
def test_log_sums_of_peaked_rows(cuda, V, bf16):
    """One logit 20 to 40 above the rest, wherever it lies. Its term is the reference's own, 1; the others are at most
    151,552 e^-16 = 2 % of it, each right to 2^-18: 1e-7, and 2^-24 of the score's own magnitude (below 2 %). No
    score is above its beam's."""
    rng = np.random.default_rng(V)
    rows = 48
    x = rng.uniform(-2, 2, (rows, V)).astype(np.float32)
    at = rng.integers(0, V, rows)
    at[:4] = [0, V - 1, V // 2, min(V - 1, 33)]
    x[np.arange(rows), at] = (2 + rng.uniform(20, 40, rows)).astype(np.float32)
    err, given, score = lse_errors(cuda, x, bf16)
    assert np.abs(err).max() <= 1.2e-7, np.abs(err).max()
    scores = -rng.random((6, 8)).astype(np.float32)
    t = torch.from_numpy(x)
    s, p, v = beam_run(cuda, t, scores, 8, bf16=bf16)
    for g in range(6):
        assert (s[g] <= scores[g][p[g]]).all()


@pytest.mark.parametrize("bf16", [False, True])
def test_log_sums_of_other_rows(cuda, bf16):
    """Where the mass of a row lies within 16 of its largest logit a term's exponent is off by half a step of the
    difference (below 16: 2^-21), half a step of its product with log2 e (below 23.1: 2^-20 ln 2), and log2 e's own
    1.4e-8 of it: 1.4e-6; the exponential by 2^-22, a thread's sums of at most 16 terms by 15 x 2^-24, the warps'
    and parts' weights by 2^-22 each: 3.1e-6 in all, below 2^-18 = 3.8e-6, if every rounding of the row falls to
    one side. In the last two rows nearly all of the mass lies equally deep below the one largest logit, where the
    roundings do fall alike."""
    rng = np.random.default_rng(9)
    V = 151552
    rows = [rng.standard_normal(V), rng.standard_normal(V) * 3, rng.uniform(-8, 0, V), np.linspace(-8, 8, V),
            np.linspace(8, -8, V), np.linspace(0, 0.05, V), np.full(V, 2.7), rng.integers(-3, 3, V) * 1.1,
            np.repeat(rng.standard_normal(V // 32) * 2, 32)]
    for depth in (5.3, 11.9):
        row = np.full(V, -depth)
        row[rng.integers(0, V)] = 0.0
        rows.append(row + 0.77)
    err, _, _ = lse_errors(cuda, np.stack(rows), bf16)
    assert np.abs(err).max() <= 2.0 ** -18, err


@pytest.mark.parametrize("scale", [1e-17, 1e-25, 1e-38])
def test_a_beams_logits_that_its_scores_do_not_tell_apart(cuda, scale):
    """Logits so small that score + logit - log sum is one number in 64 bits for all: the candidates are those of the
    largest logits, in their order, equal ones by the lower token; of two beams the lower one's."""
    rng = np.random.default_rng(3)
    V, k = 6001, 12
    x = (rng.integers(-4, 5, (2, V)) * scale).astype(np.float32)
    x[0, rng.permutation(V)[:9]] = (rng.permutation(9) + 5) * np.float32(scale)
    for rows, B in ((x, 2), (x[:1], 1)):
        s, p, v = beam_run(cuda, rows, np.full((1, B), -1.0, np.float32), k)
        want = np.lexsort((np.arange(V), -x[0].astype(np.float64)))[:k]
        assert (p == 0).all() and (v[0] == want).all(), (v[0], want)
        assert np.abs(s - (-1.0 - np.log(V))).max() <= 2.0 ** -18 + 2.0 ** -20


def test_finished_beams_among_equal_scores(cuda):
    """Rows of one candidate each, whose score is their beam's own: finished and live beams of one score in the order of
    the beams."""
    V = 4096
    x = np.full((5, V), -np.inf, np.float32)
    x[[0, 1, 2, 3, 4], [7, 4000, 0, 31, 5]] = [3.0, -2.0, 0.0, 1e4, 2.5]
    s, p, v = beam_run(cuda, x, np.full((1, 5), -1.25, np.float32), 6, finished=np.array([[1, 0, 1, 0, 0]], np.uint8), pad=9)
    assert p[0].tolist() == [0, 1, 2, 3, 4, -1] and v[0].tolist() == [9, 4000, 9, 31, 5, -1]
    assert (s[0, :5] == -1.25).all() and s[0, 5] == -np.inf


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


# ---- a stage's trees ------------------------------------------------------------------------------------------------

SMALL = dict(hidden=512, inter=256, experts=16, top_k=4, num_blocks=20, seed=6, routing="softmax")
RES = {"a": ([67, 68], [2, 3, 4, 5, 6, 7]), "b": ([69, 70], [8, 9, 10, 11, 12, 13])}
AT = {"a": 130, "b": 30}


def started(cuda, rng, **over):
    from ssengine_b200.messages import Chunk, Plan
    from ssengine_b200.stage import StageModel

    st = StageModel(cfg(**{**SMALL, **over}), 0, cuda)
    st.forward(Plan(0, [Chunk(r, 0, AT[r], *RES[r], True, rng.integers(0, 1000, AT[r]).tolist()) for r in "ab"]))
    return st


def step(k, names, trees, tokens, at=AT):
    from ssengine_b200.messages import Chunk, Plan

    return Plan(k, [Chunk(r, at[r], len(t), *RES[r], True, tok) for r, t, tok in zip(names, trees, tokens)])


def test_trees_given_up_leave_no_rows(cuda):
    """An acceptance of nothing, and a verify that fails on its way, leave no memory behind."""
    st = started(cuda, np.random.default_rng(1))
    trees, tokens = [[-1, 0, 0, 2], [-1, -1, 1]], [[1, 2, 3, 4], [5, 6, 7]]

    def held():
        gc.collect()
        torch.cuda.synchronize()
        return torch.cuda.memory_allocated(cuda)

    st.verify(step(1, "ab", trees, tokens), trees)
    st.accept([[0, 2], [1]])
    before = held()
    at = {"a": 132, "b": 31}
    st.verify(step(2, "ab", trees, tokens, at), trees)
    st.accept([[], []])
    assert held() == before

    def failing(layer, *_):
        if layer is st.layers[-1]:
            raise RuntimeError("a check")

    st.layer_hook = failing
    with pytest.raises(RuntimeError):
        st.verify(step(3, "ab", trees, tokens, at), trees)
    st.layer_hook = None
    assert st.trees is None and held() == before
    with pytest.raises(ValueError):
        st.accept([[0], [0]])


def test_several_trees_in_flight(cuda):
    """Two microbatches verified before either is accepted, accepted in the other order: what each alone leaves."""
    rng = [np.random.default_rng(2) for _ in range(2)]
    st, ref = (started(cuda, r) for r in rng)
    trees = {"a": [-1, 0, 0, 2, 1], "b": [-1, 0, -1, 1]}
    tokens = {"a": [9, 8, 7, 6, 5], "b": [4, 3, 2, 1]}
    paths = {"a": [0, 2, 3], "b": [0, 1, 3]}                  # b's is a path of a's tree too, as far as it goes
    got, open_ = {}, {}
    for k, r in enumerate("ab"):
        st.verify(step(1 + k, r, [trees[r]], [tokens[r]]), [trees[r]])
        got[r], open_[r] = st.last_logits.clone(), st.trees
    for r in "ab":
        st.accept([paths[r]], trees=open_[r])
    for r in "ab":
        with pytest.raises(ValueError):                       # a step is accepted once
            st.accept([paths[r]], trees=open_[r])
    for k, r in enumerate("ab"):
        ref.verify(step(1 + k, r, [trees[r]], [tokens[r]]), [trees[r]])
        assert torch.equal(got[r], ref.last_logits)
        ref.accept([paths[r]])
    torch.cuda.synchronize()
    same = lambda x, y: torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))
    for a, b, dsa in zip(st.kda_states, ref.kda_states, st.is_dsa):
        if dsa:
            assert same(a[1], b[1]) and same(a[2], b[2])
        else:
            blocks = RES["a"][1] + RES["b"][1]
            assert all(same(u[blocks], v[blocks]) for u, v in zip(a, b))
    at = {r: AT[r] + len(paths[r]) for r in "ab"}
    more = step(5, "ab", [[-1], [-1]], [[11], [12]], at)
    assert torch.equal(st.decode(more), ref.decode(more)) and torch.equal(st.last_logits, ref.last_logits)
    assert int(st.status.item()) == 0 and int(ref.status.item()) == 0


def test_a_node_past_the_selection_is_as_the_dense_decode(cuda):
    """Behind a context that the indexer would choose from, `verify` takes the whole context only where it is told to;
    a chain is then the dense decode of the same tokens, row by row (the attention is one operator's arithmetic,
    the recurrence's closed form differs: the stage's chained bound, 6e-2)."""
    from ssengine_b200.messages import Chunk, Plan
    from ssengine_b200.stage import StageModel

    rng = np.random.default_rng(4)
    n, tree = 2049, [-1, 0, 1]
    res = (list(range(67, 67 + 17)), [3, 4, 5, 6, 7, 8])
    prompt, draft = rng.integers(0, 1000, n).tolist(), rng.integers(0, 1000, 3).tolist()
    st, ref = (StageModel(cfg(**{**SMALL, "mb_tokens": 2176}), 0, cuda) for _ in range(2))
    for s in (st, ref):
        s.forward(Plan(0, [Chunk("a", 0, n, *res, True, prompt)]))
    plan = Plan(1, [Chunk("a", n, 3, *res, True, draft)])
    with pytest.raises(ValueError, match="selected"):
        st.verify(plan, [tree])
    assert st.trees is None
    short = Plan(1, [Chunk("a", n, 2, *res, True, draft[:2])])
    st.verify(short, [[-1, 0]])                               # 2,051 tokens: the selection is all of them
    st.verify(plan, [tree], attention="dense")
    logits = st.last_logits.clone()
    for i in range(3):
        ref.decode(Plan(2 + i, [Chunk("a", n + i, 1, *res, True, draft[i:i + 1])]), attention="dense")
        got, want = logits[i].double(), ref.last_logits[0].double()
        assert float((got - want).norm() / want.norm()) < 6e-2, i
    with pytest.raises(ValueError):
        st.verify(plan, [tree], attention="sparse")


def test_a_stages_first_trees_use_what_its_build_reserved(cuda, monkeypatch):
    """The first verify and accept ask for no workspace, map no memory and load no kernel that the build did not run."""
    from ssengine_b200 import kvpages, lib

    ran = []
    real = lib.load()

    class Recorded:
        def __getattr__(self, name):
            f = getattr(real, name)
            if not name.startswith("ssb_"):
                return f
            return lambda *a: (ran.append(name), f(*a))[1]

    monkeypatch.setattr(lib, "load", lambda path=None: Recorded())
    st = started(cuda, np.random.default_rng(3))
    built = set(ran)
    assert {"ssb_kda_decode_tree", "ssb_kda_advance", "ssb_mla_decode_tree", "ssb_move_rows"} <= built

    def none(*_):
        raise AssertionError("a step asked for a workspace")

    monkeypatch.setattr(lib, "stream_scratch", none)
    torch.cuda.synchronize()
    mapped = torch.cuda.memory_reserved(cuda)
    trees = [[-1, 0, 0, 2], [-1, -1, 1]]
    st.verify(step(1, "ab", trees, [[1, 2, 3, 4], [5, 6, 7]]), trees)
    st.accept([[0, 2], [1]])
    torch.cuda.synchronize()
    assert set(ran) == built and torch.cuda.memory_reserved(cuda) == mapped
    assert int(st.status.item()) == 0 and st.trees is None
