"""`StageModel.verify` and `accept` on the GPU: trees of drafted tokens through a whole stage.

The logits of every node against those of its path decoded token by token as a request of its own (`StageModel.decode`, dense
attention), and the requests' next steps after a path was accepted against that request's. The two chains differ by the
recurrence's closed form (16-bit operands) and by the attention's splits, which the 4-bit projections turn into code flips:
held to 6e-2 relative, the bound of two chained runs of this model's four layers (test_gpu_model.py); another path, state or
page moves logits by their own scale. What a stage split changes nothing about is equal bit for bit."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

CHAINED = 6e-2


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def cfg(**over):
    from ssengine_b200.stage import StageConfig

    return StageConfig(**{**dict(layer_split=(4,), hidden=256, inter=128, experts=8, top_k=2, vocab=1000, mb_tokens=256,
                                 num_blocks=80, seed=5, layer_kind="hybrid", kda_heads=2, q_lora=256, mla_nope=64,
                                 routing="sigmoid"), **over})


def path(parents, i):
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out[::-1]


def wild_tree(n, seed):
    rng = np.random.default_rng(seed)
    return [-1] + [int(rng.integers(max(-1, i - 4), i)) for i in range(1, n)]


TREES = [[-1, 0, 0, 2, 1, -1, 5, 3], [-1, -1, 0, 1, 3]]
PROMPTS = [126, 61]


@pytest.mark.parametrize("kind", ["hybrid", "kda"])
def test_every_node_is_its_path_decoded(cuda, kind):
    from ssengine_b200.messages import Chunk, Plan
    from ssengine_b200.stage import StageModel

    c = cfg(layer_kind=kind)
    rng = np.random.default_rng(70)
    prompts = [rng.integers(0, c.vocab, n).tolist() for n in PROMPTS]
    drafts = [rng.integers(0, c.vocab, len(t)).tolist() for t in TREES]
    st, ref = StageModel(c, 0, cuda), StageModel(c, 0, cuda)
    res = [([67 + 2 * r, 68 + 2 * r], [2 + 6 * r + g for g in range(6)]) for r in range(2)]
    st.forward(Plan(0, [Chunk(f"r{r}", 0, n, *res[r], True, prompts[r]) for r, n in enumerate(PROMPTS)]))
    states = [[t.clone() for t in s] for s in st.kda_states]
    toks = st.verify(Plan(1, [Chunk(f"r{r}", PROMPTS[r], len(t), *res[r], True, drafts[r])
                              for r, t in enumerate(TREES)]), TREES)
    torch.cuda.synchronize()
    logits = st.last_logits.clone()
    assert toks.shape == (13,) and (toks == logits.argmax(dim=1)).all() and int(st.status.item()) == 0
    same = lambda a, b: torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
    blocks = [b for _, bl in res for b in bl]
    for dsa, before, after in zip(st.is_dsa, states, st.kda_states):     # pool keys, tail ring; KDA states untouched
        if dsa:
            assert same(after[1], before[1]) and same(after[2], before[2])
        else:
            assert all(same(x[blocks], y[blocks]) for x, y in zip(after, before))

    # every leaf's path as a request of its own: prefilled alike (both prompts in one plan), then token by token
    leaves = [(r, i) for r, t in enumerate(TREES) for i in range(len(t)) if i not in t]
    first = np.cumsum([0] + [len(t) for t in TREES])
    final = {}
    for k, (r, leaf) in enumerate(leaves):
        rows = [([67 + 4 * k + 2 * j, 68 + 4 * k + 2 * j], [2 + 6 * j + g for g in range(6)]) for j in range(2)]
        ref.forward(Plan(100 * k, [Chunk(f"{k}.{j}", 0, n, *rows[j], True, prompts[j]) for j, n in enumerate(PROMPTS)]))
        for d, node in enumerate(path(TREES[r], leaf)):
            ref.decode(Plan(100 * k + d + 1, [Chunk(f"{k}.{r}", PROMPTS[r] + d, 1, *rows[r], True, [drafts[r][node]])]),
                       attention="dense")
            err = rel(logits[first[r] + node], ref.last_logits[0])
            assert err < CHAINED, (r, node, err)

    # accept a path of each (of the second one node), go on: two plain steps
    paths = [[0, 2, 3], [1]]
    st.accept(paths)
    rows = [([67 + 2 * j, 68 + 2 * j], [2 + 6 * j + g for g in range(6)]) for j in range(2)]
    ref.forward(Plan(900, [Chunk(f"z{j}", 0, n, *rows[j], True, prompts[j]) for j, n in enumerate(PROMPTS)]))
    ref.decode(Plan(901, [Chunk(f"z{j}", PROMPTS[j], len(p), *rows[j], True, [drafts[j][i] for i in p])
                          for j, p in enumerate(paths)]), attention="dense")
    more = rng.integers(0, c.vocab, (3, 2))
    at = [n + len(p) for n, p in zip(PROMPTS, paths)]
    for d in range(2):
        plan = Plan(910 + d, [Chunk(f"z{j}", at[j] + d, 1, *rows[j], True, [int(more[d, j])]) for j in range(2)])
        st.decode(plan)
        got = st.last_logits.clone()
        ref.decode(plan)
        for j in range(2):
            assert rel(got[j], ref.last_logits[j]) < CHAINED, (d, j)
    for dsa, a, b in zip(st.is_dsa, st.kda_states, ref.kda_states):
        if dsa:
            pages = rows[0][0]
            keys = lambda t: t.view(-1, 32, 128)[pages[0], :at[0] // 4].float()
            assert rel(keys(a[1]), keys(b[1])) < CHAINED
            f8 = lambda t: t.view(torch.float8_e4m3fn).view(-1, 128, 576)[pages].float()[0]
            assert rel(f8(a[0])[:at[0]], f8(b[0])[:at[0]]) < CHAINED
        else:
            blk = [rows[0][1][g] for g in range(5)]
            assert rel(a[1][blk], b[1][blk]) < CHAINED or not a[1][blk].any()
    assert int(st.status.item()) == 0


def test_two_stages_verify_as_one(cuda):
    """Across a stage edge the step and the acceptance equal the unsplit stage's, bit for bit; a second verify of other
    trees in the place of accept; an empty path."""
    from ssengine_b200.messages import Chunk, Plan
    from ssengine_b200.stage import StageModel

    base = dict(hidden=512, inter=256, experts=16, top_k=4, num_blocks=14, seed=6, routing="softmax")
    whole = StageModel(cfg(**base), 0, cuda)
    s0, s1 = (StageModel(cfg(layer_split=(2, 2), **base), i, cuda) for i in range(2))
    rng = np.random.default_rng(71)
    ta, tb = rng.integers(0, 1000, 300).tolist(), rng.integers(0, 1000, 100).tolist()
    a, b = ([67, 68], [2, 3, 4, 5, 6, 7]), ([69], [8, 9, 10, 11, 12, 13])
    first = Plan(0, [Chunk("a", 0, 130, *a, True, ta[:130]), Chunk("b", 0, 30, *b, True, tb[:30])])
    whole.forward(first)
    s1.forward(first, s0.forward(first))
    na, nb = 130, 30
    for k in range(3):
        for again in range(2 if k == 1 else 1):
            trees = [[-1] + [int(rng.integers(-1, i)) for i in range(1, 5 + k)], [-1, 0, -1]]
            step = Plan(1 + k, [Chunk("a", na, 5 + k, *a, True, ta[150:155 + k]), Chunk("b", nb, 3, *b, True, tb[50:53])])
            t_whole = whole.verify(step, trees)
            t_split = s1.verify(step, trees, s0.verify(step, trees))
            torch.cuda.synchronize()
            assert torch.equal(t_whole, t_split) and torch.equal(whole.last_logits, s1.last_logits)
            assert torch.isfinite(whole.last_logits).all()
        paths = [path(trees[0], int(rng.integers(0, 5 + k))), [0, 1] if k != 2 else []]
        for st in (whole, s0, s1):
            st.accept(paths)
        na, nb = na + len(paths[0]), nb + len(paths[1])
        step = Plan(10 + k, [Chunk("a", na, 1, *a, True, ta[200:201]), Chunk("b", nb, 1, *b, True, tb[60:61])])
        w = whole.decode(step)
        assert torch.equal(w, s1.decode(step, s0.decode(step))) and torch.equal(whole.last_logits, s1.last_logits)
        na, nb = na + 1, nb + 1
    for st in (whole, s0, s1):
        assert int(st.status[0]) == 0


@pytest.mark.parametrize("fp8", [False, True])
def test_an_accepted_path_leaves_the_pages_of_its_decode(cuda, fp8):
    """A stage that begins with its attention layer, given the rows of the layers before it: the path's latent rows, pool keys
    and tail are those of the same rows decoded one after another, bit for bit."""
    from ssengine_b200.messages import Chunk, Plan
    from ssengine_b200.stage import StageModel

    base = dict(layer_split=(3, 1), hidden=512, inter=256, experts=16, top_k=4, num_blocks=14, seed=8, indexer_fp8=fp8)
    st, ref = (StageModel(cfg(**base), 1, cuda) for _ in range(2))
    gen = torch.Generator(cuda).manual_seed(3)
    rows = lambda n: torch.randn(n, st.hidden_width, generator=gen, device=cuda).to(torch.bfloat16)
    a, b = ([67, 68], [2, 3, 4, 5, 6, 7]), ([69, 70], [8, 9, 10, 11, 12, 13])
    at = [121, 6]
    first, x = Plan(0, [Chunk("a", 0, at[0], *a, True, None), Chunk("b", 0, at[1], *b, True, None)]), rows(sum(at))
    for s in (st, ref):
        s.forward(first, x)
    for k, (trees, paths) in enumerate([([wild_tree(20, 1), [-1, -1, 1]], [None, [1, 2]]),
                                        ([[-1], wild_tree(64, 2)], [[0], None]),
                                        ([wild_tree(5, 3), [-1, -1]], [[], [1]])]):
        paths = [path(t, len(t) - 1) if p is None else p for t, p in zip(trees, paths)]
        x = rows(sum(map(len, trees)))
        st.verify(Plan(1 + k, [Chunk(n, s, len(t), *r, True, None) for n, s, t, r in zip("ab", at, trees, (a, b))]), trees, x)
        st.accept(paths)
        off = len(trees[0])
        taken = torch.cat([x[paths[0]], x[[off + i for i in paths[1]]]])
        ref.decode(Plan(1 + k, [Chunk(n, s, len(p), *r, True, None) for n, s, p, r in zip("ab", at, paths, (a, b)) if p]), taken,
                   attention="dense")
        at = [s + len(p) for s, p in zip(at, paths)]
        torch.cuda.synchronize()
        same = lambda u, v: torch.equal(u.contiguous().view(torch.uint8), v.contiguous().view(torch.uint8))
        (lat, pool, tail), (lat_r, pool_r, tail_r) = st.kda_states[0], ref.kda_states[0]
        assert same(pool, pool_r) and same(tail, tail_r)
        for n, r in zip(at, (a, b)):
            pages = lambda t: t.view(torch.uint8).view(-1, 128, 576)[r[0]].view(-1, 576)[:n]
            assert torch.equal(pages(lat), pages(lat_r))
    assert int(st.status.item()) == 0
