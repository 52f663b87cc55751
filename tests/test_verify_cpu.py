"""`stage.Trees` on the host: the checks of a plan's trees and of the accepted paths, and the tables made of them."""

from types import SimpleNamespace

import pytest
import torch


def trees_of(parents, starts=(5, 130), device="cpu", dsa=True):
    from ssengine_b200.messages import Chunk
    from ssengine_b200.stage import Trees

    chunks = [Chunk(f"r{i}", s, len(p), [70 + 10 * i, 71 + 10 * i], [10 * i + g for g in range(1, 7)], True, [0] * len(p))
              for i, (s, p) in enumerate(zip(starts, parents))]
    batch = SimpleNamespace(order=list(range(len(chunks))), last_rows=None,
                            dsa=dict(positions=None, page_table=torch.zeros(2, 2, dtype=torch.int32)) if dsa else None)
    return Trees(chunks, parents, batch, torch.device(device)), batch


def test_rows_of_the_trees():
    t, batch = trees_of([[-1, 0, 0, 2], [-1, -1, 1]])
    assert t.parents.tolist() == [-1, 0, 0, 2, -1, -1, 1] and t.reqs.tolist() == [0, 0, 0, 0, 1, 1, 1]
    assert t.context.tolist() == [5] * 4 + [130] * 3 and t.ancestors.tolist() == [1, 3, 5, 13, 1, 2, 6]
    assert batch.dsa["positions"].tolist() == [5, 6, 6, 7, 130, 130, 131] and batch.last_rows.tolist() == list(range(7))
    assert t.most == 4 and t.parents.dtype == torch.int32 and t.ancestors.dtype == torch.int64


def test_accepted_tables():
    t, _ = trees_of([[-1, 0, 0, 2], [-1, -1, 1]], starts=(126, 0))
    a = t.accepted([[0, 2, 3], [1]])
    assert a["rows"].tolist() == [0, 2, 3, 5] and a["rows64"].tolist() == [0, 2, 3, 5] and a["most"] == 3
    assert a["kpool"].tolist() == [[0, 3, 126, 6], [3, 1, 0, 16]]
    for g in range(5):
        assert a["seqs"][g].tolist() == [[0, 3, 1 + g, 1], [3, 4, 11 + g, 0]]
    assert a["src"].tolist() == [[70 * 128 + 126, 71 * 128 + 0, 71 * 128 + 1], [80 * 128 + 1, -1, -1]]
    assert a["dst"].tolist() == [[70 * 128 + 126, 70 * 128 + 127, 71 * 128], [80 * 128, -1, -1]]
    assert t.accepted([[], []]) is None
    assert t.accepted([(), (0,)])["rows"].tolist() == [4]


@pytest.mark.parametrize("paths", [
    [[0]], [[0], [0], []], [[1], []], [[0, 3], []], [[0, 2, 2], []], [[4], []], [[-1], []], [[0], [0, 2]],
])
def test_what_is_no_path_is_refused(paths):
    t, _ = trees_of([[-1, 0, 0, 2], [-1, -1, 1]])
    with pytest.raises(ValueError):
        t.accepted(paths)


@pytest.mark.parametrize("parents", [[[-1, 1], [-1]], [[0], [-1]], [[-1], list(range(-1, 64))]])
def test_what_is_no_tree_is_refused(parents):
    with pytest.raises(ValueError):
        trees_of(parents)


def test_a_tree_of_another_length_and_nothing_to_accept_are_refused():
    from ssengine_b200.messages import Chunk
    from ssengine_b200.stage import StageModel, Trees

    batch = SimpleNamespace(order=[0], last_rows=None, dsa=None)
    with pytest.raises(ValueError):
        Trees([Chunk("a", 0, 3, [1], [0] * 6, True, None)], [[-1, 0]], batch, torch.device("cpu"))
    with pytest.raises(ValueError):
        Trees([Chunk("a", 0, 1, [1], [0] * 6, True, None)], [[-1], [-1]], batch, torch.device("cpu"))
    st = object.__new__(StageModel)
    st.trees, st.kda = None, False
    with pytest.raises(ValueError):
        st.accept([[0]])
    with pytest.raises(ValueError):
        st.verify(None, [])


def test_a_step_that_fails_leaves_nothing_to_accept(monkeypatch):
    from ssengine_b200.messages import Chunk, Plan
    from ssengine_b200.stage import StageModel

    st = object.__new__(StageModel)
    st.trees, st.kda, st.device = None, True, torch.device("cpu")
    monkeypatch.setattr(st, "prepare", lambda plan: SimpleNamespace(order=[0], last_rows=None, dsa=None), raising=False)
    monkeypatch.setattr(st, "run", lambda *a, **kw: "rows", raising=False)
    plan = Plan(0, [Chunk("a", 3, 2, [1], [0] * 6, True, [4, 5])])
    assert st.verify(plan, [[-1, 0]]) == "rows" and st.trees.trees == [[-1, 0]]

    def failing(*a, **kw):
        raise RuntimeError("out of memory")

    monkeypatch.setattr(st, "run", failing, raising=False)
    with pytest.raises(RuntimeError):
        st.verify(plan, [[-1, -1]])
    with pytest.raises(ValueError):
        st.accept([[0]])
    st.trees = "left over"
    with pytest.raises(ValueError):
        st.verify(plan, [[-1, 1]])
    assert st.trees is None


def test_what_the_layers_keep_ends_with_its_trees(monkeypatch):
    """An acceptance of nothing and a verify that fails on its way leave none of the layers' rows alive."""
    import gc
    import weakref

    from ssengine_b200.messages import Chunk, Plan
    from ssengine_b200.stage import StageModel

    st = object.__new__(StageModel)
    st.trees, st.kda, st.device, rows = None, True, torch.device("cpu"), []
    monkeypatch.setattr(st, "prepare", lambda plan: SimpleNamespace(order=[0], last_rows=None, dsa=None), raising=False)

    def run(batch, hidden, edge, tree, fails=False):
        tree.steps.append(torch.zeros(3))
        rows.append(weakref.ref(tree.steps[0]))
        if fails:
            raise RuntimeError("a check")

    plan = Plan(0, [Chunk("a", 3, 2, [1], [0] * 6, True, [4, 5])])
    monkeypatch.setattr(st, "run", run, raising=False)
    st.verify(plan, [[-1, 0]])
    assert rows[0]() is not None
    st.accept([[]])
    gc.collect()
    assert rows[0]() is None
    monkeypatch.setattr(st, "run", lambda *a, **kw: run(*a, **kw, fails=True), raising=False)
    with pytest.raises(RuntimeError):
        st.verify(plan, [[-1, 0]])
    gc.collect()
    assert rows[1]() is None and st.trees is None


def test_each_step_in_flight_is_accepted_by_name_and_once(monkeypatch):
    from ssengine_b200.messages import Chunk, Plan
    from ssengine_b200.stage import StageModel

    st = object.__new__(StageModel)
    st.trees, st.kda, st.device = None, True, torch.device("cpu")
    st.status, st.kda_states, st.is_dsa, st.kda_group, took = None, [("conv", "rec")], [False], [0], []
    attn = SimpleNamespace(accept=lambda kept, rows, seqs, *_: took.append((kept, rows.tolist(), seqs[0].tolist())))
    st.layers = [SimpleNamespace(attn=attn)]
    monkeypatch.setattr(st, "prepare", lambda plan: SimpleNamespace(order=[0], last_rows=None, dsa=None), raising=False)
    monkeypatch.setattr(st, "run", lambda b, h, e, tree: tree.steps.append(tree.chunks[0].req_id), raising=False)
    held = {}
    for i, r in enumerate("abc"):
        st.verify(Plan(i, [Chunk(r, 3 + i, 3, [1], [20 * i + g for g in range(6)], True, [4, 5, 6])]), [[-1, 0, 0]])
        held[r] = st.trees
    with pytest.raises(ValueError):
        st.accept([[0, 1]])                                # three are open, and none is named
    st.accept([[0, 1]], trees=held["a"])
    assert st.trees is held["c"]
    with pytest.raises(ValueError):
        st.accept([[0]], trees=held["a"])
    with pytest.raises(ValueError):
        st.accept([[1]], trees=held["b"])                  # no path: the step stays open
    other = object.__new__(StageModel)
    other.trees, other.kda = None, True
    with pytest.raises(ValueError):
        other.accept([[0]], trees=held["b"])
    with pytest.raises(ValueError):
        st.accept([[0], []], trees=trees_of([[-1, 0], [-1]])[0])          # no stage has verified these
    st.accept([[0]], trees=held["b"])
    st.accept([[0, 2]])
    assert took == [("a", [0, 1], [0, 2, 0, 1]), ("b", [0], [0, 1, 20, 1]), ("c", [0, 2], [0, 2, 40, 1])]
    assert st.trees is None
    with pytest.raises(ValueError):
        st.accept([[0, 2]], trees=held["c"])


@pytest.mark.parametrize("kind", ["hybrid", "kda"])
def test_nodes_past_the_selection_are_refused_unless_dense(monkeypatch, kind):
    from ssengine_b200.layers import DsaAttention
    from ssengine_b200.messages import Chunk, Plan
    from ssengine_b200.stage import SELECTED_TOKENS, StageModel

    assert SELECTED_TOKENS == 4 * DsaAttention.TOPK + 3
    st = object.__new__(StageModel)
    st.trees, st.kda, st.device, st.cfg = None, True, torch.device("cpu"), SimpleNamespace(layer_kind=kind)
    batch = lambda plan: SimpleNamespace(order=[0, 1], last_rows=None, dsa=None)
    monkeypatch.setattr(st, "prepare", batch, raising=False)
    monkeypatch.setattr(st, "run", lambda *a, **kw: "rows", raising=False)
    trees = [[-1, -1], [-1, 0, 0, 1]]                       # the second is three nodes deep
    at = lambda start: Plan(0, [Chunk(r, n, len(t), [1], [0] * 6, True, [0] * len(t))
                                for r, n, t in zip("ab", (5, start), trees)])
    assert st.verify(at(2048), trees) == "rows"             # 2,051 tokens
    if kind == "hybrid":
        with pytest.raises(ValueError, match="2052"):
            st.verify(at(2049), trees)
        assert st.trees is None
    else:
        assert st.verify(at(2049), trees) == "rows"         # no attention that selects
    assert st.verify(at(2049), trees, attention="dense") == "rows" and st.trees.reach == 2052
    with pytest.raises(ValueError):
        st.verify(at(5), trees, attention="none")


def test_a_second_verify_of_a_request_ends_the_first(monkeypatch):
    """Its nodes took the cache rows of the first one's."""
    from ssengine_b200.messages import Chunk, Plan
    from ssengine_b200.stage import StageModel

    st = object.__new__(StageModel)
    st.trees, st.kda, st.device = None, True, torch.device("cpu")
    st.layers = st.is_dsa = st.kda_states = st.kda_group = []
    batch = lambda plan: SimpleNamespace(order=list(range(len(plan.chunks))), last_rows=None, dsa=None)
    monkeypatch.setattr(st, "prepare", batch, raising=False)
    monkeypatch.setattr(st, "run", lambda *a, **kw: None, raising=False)

    def verify(names):
        st.verify(Plan(0, [Chunk(r, 3, 2, [1], [0] * 6, True, [4, 5]) for r in names]), [[-1, 0]] * len(names))
        return st.trees

    ab, c, b = verify("ab"), verify("c"), verify("b")
    with pytest.raises(ValueError):
        st.accept([[0], [0]], trees=ab)
    st.accept([[0]], trees=c)
    with pytest.raises(ValueError):                          # a step that is refused takes no rows
        st.verify(Plan(0, [Chunk("b", 3, 2, [1], [0] * 6, True, [4, 5])]), [[-1, 5]])
    st.accept([[0]], trees=b)
