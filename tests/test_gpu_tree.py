"""GPU parity of the operators for trees of drafted tokens: `mla.decode_tree` (`ssb_mla_decode_tree`),
`KdaLayer.decode_tree` (`ssb_kda_decode_tree`) and `KdaLayer.advance` (`ssb_kda_advance`), against float64 restatements.

Tolerances, derived before the first run:
- attention: those of `mla.decode` (test_gpu_decode.py), whose arithmetic the tree form shares: 5e-3 relative L2 of a head's
  row, 2e-3 absolute for the log-sum-exp;
- recurrence outputs: the bf16 store rounds each value by at most 2^-9 of it, the bar 2^-8; beside it 1e-3 of the row's
  largest: the state and the nodes' vectors may enter their product with 16 significant bits (2^-17 each), the magnitudes
  of 128 products total about sqrt(128) times their sum's, 11.3 x 2^-16 = 1.7e-4, through the substitution down the tree
  (weights of at most 1, shrinking with the decays) about three times that;
- advanced states: fp32 throughout, a few 2^-22 a token: 1e-5 relative L2; conv rows exact."""

import numpy as np
import pytest
import torch

from test_gpu_decode import BMM1, D, Cache, attention64, check, kda_make, queries, recurrence64
from oracle import kda as ok

pytestmark = pytest.mark.gpu

CHAIN = lambda n: list(range(-1, n - 1))
STAR = lambda n: [-1] * n
BINARY = lambda n: [(i - 1) // 2 if i else -1 for i in range(n)]


def wild(rng, n):
    return [int(rng.integers(max(-1, i - 6), i)) for i in range(n)]


def path(parents, i):
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out[::-1]


# ---- attention ------------------------------------------------------------------------------------------------------


def call_tree(cuda, q, cache, lens, masks, reqs=None, bmm1=BMM1, bmm2=1.0, lse=True, **kw):
    from ssengine_b200 import mla

    dev = lambda a: None if a is None else torch.as_tensor(np.ascontiguousarray(a)).to(cuda)
    T, H = q.shape[:2]
    out = torch.full((T, H, 512), float("nan"), dtype=torch.bfloat16, device=cuda)
    ls = torch.full((T, H), float("nan"), device=cuda) if lse else None
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    mla.decode_tree(q.to(cuda), dev(cache.bytes), dev(cache.table), dev(np.asarray(lens, np.int32)),
                    dev(np.asarray(masks, np.int64)), bmm1, out, bmm2=bmm2, reqs=dev(reqs), lse=ls, status=status, **kw)
    torch.cuda.synchronize()
    return out.double().cpu().numpy(), None if ls is None else ls.double().cpu().numpy(), int(status.item())


def tree_rows(trees, lens):
    """Rows of every request's nodes: (context lengths, masks, requests, visible positions)."""
    from ssengine_b200 import mla

    rows = ([], [], [], [])
    for r, (tree, n) in enumerate(zip(trees, lens)):
        masks, _ = mla.tree_masks(tree)
        for i in range(len(tree)):
            rows[0].append(n)
            rows[1].append(int(masks[i]))
            rows[2].append(r)
            rows[3].append(np.concatenate([np.arange(n), n + np.array(path(tree, i))]).astype(np.int64))
    return rows


@pytest.mark.parametrize("heads", [1, 16, 64, 65])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_trees_behind_contexts_of_every_kind(cuda, heads, kind):
    """Contexts around the units of 64 tokens and the pages of 128, none at all, trees from one node to 64; NaN behind."""
    rng = np.random.default_rng(heads)
    lens = [1, 0, 63, 64, 65, 127, 128, 1000, 100, 33]
    trees = [CHAIN(1), STAR(5), CHAIN(2), BINARY(7), wild(rng, 63), wild(rng, 64), CHAIN(64), wild(rng, 12), STAR(64), [-1]]
    cache = Cache(rng, [n + len(t) for n, t in zip(lens, trees)], pad_width=1)
    seq, masks, reqs, seen = tree_rows(trees, lens)
    q, q64 = queries(rng, len(seq), heads, kind)
    out, lse, status = call_tree(cuda, q, cache, seq, masks, np.array(reqs, np.int32), bmm2=0.5)
    assert status == 0
    for t, r in enumerate(reqs):
        check(out[t], lse[t], *attention64(q64[t], cache.kv[r][seen[t]], BMM1, 0.5))


def test_any_set_of_bits(cuda):
    """Masks that are no path: none, the last node alone, every second, negative words; empty rows; a row that sees nothing
    of a whole unit in the middle."""
    rng = np.random.default_rng(3)
    lens = [0, 0, 0, 500, 500, 64, 10, -5, 1]
    masks = [0, 1 << 62, -(1 << 63), 0, 0x5555555555555555, -1, 1 << 60, 7, 2]
    cache = Cache(rng, [max(n, 0) + 64 for n in lens])
    q, q64 = queries(rng, len(lens), 64, "bf16")
    out, lse, status = call_tree(cuda, q, cache, lens, masks)
    assert status == 0
    for t, (n, m) in enumerate(zip(lens, masks)):
        seen = [] if n < 0 else list(range(n)) + [n + j for j in range(64) if (m >> j) & 1]
        check(out[t], lse[t], *attention64(q64[t], cache.kv[t][np.array(seen, np.int64)], BMM1, 1.0))


def test_unseen_nodes_may_hold_nan(cuda):
    """Every drafted token that a row does not see is NaN for it: siblings' rows never meet its products."""
    rng = np.random.default_rng(4)
    cache = Cache(rng, [300 + 40])
    tree = wild(rng, 40)
    q, q64 = queries(rng, 1, 64, "bf16")
    for i in (0, 7, 39):
        p = path(tree, i)
        mine = cache.bytes.copy()
        away = [j for j in range(40) if j not in p]
        mine[cache.slots(0, 300 + np.array(away))] = 0x7F
        view = type("C", (), dict(bytes=mine, table=cache.table))
        out, lse, _ = call_tree(cuda, q, view, [300], [sum(1 << j for j in p)])
        check(out[0], lse[0], *attention64(q64[0], cache.kv[0][np.r_[0:300, 300 + np.array(p)]], BMM1, 1.0))


@pytest.mark.parametrize("heads", [1, 3, 16, 21, 32, 33, 64])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_a_nan_node_reaches_its_descendants_alone(cuda, heads, kind):
    """Nodes of one call, two of them with NaN in their cache rows: their descendants' outputs are NaN, no other node's."""
    rng = np.random.default_rng(heads)
    for n in (5, 64, 100, 250):
        tree = wild(rng, 30)
        cache = Cache(rng, [n + 30])
        bad = [4, 17]
        cache.bytes[cache.slots(0, n + np.array(bad)), [100, 511]] = 0x7F
        cache.bytes[cache.slots(0, n + np.array(bad)), [7, 300]] = 0xFF
        seq, masks, reqs, seen = tree_rows([tree], [n])
        q, q64 = queries(rng, 30, heads, kind)
        out, lse, status = call_tree(cuda, q, cache, seq, masks, np.array(reqs, np.int32))
        assert status == 0
        for i in range(30):
            if set(path(tree, i)) & set(bad):
                assert np.isnan(out[i]).all() and np.isnan(lse[i]).all(), (n, i)
            else:
                check(out[i], lse[i], *attention64(q64[i], cache.kv[0][seen[i]], BMM1, 1.0))


@pytest.mark.parametrize("heads", [1, 2, 7, 16, 22, 32])
def test_rows_that_share_a_tile(cuda, heads):
    """Few heads: neighbouring rows of a request share a tile. Rows of one request with several context lengths, requests
    that take turns, rows without a node or without any token among them, empty and bad requests; with and without lse."""
    rng = np.random.default_rng(50 + heads)
    lens = [300, 0, 129, 5]
    cache = Cache(rng, [n + 64 for n in lens])
    rows = []
    for r in (0, 0, 0, 1, 1, 2, 2, 2, 2, 2, 0, 3, 3, 9, 9, 2, 2, 1, 0):
        for _ in range(int(rng.integers(1, 9))):
            n = lens[r] if r < 4 else 10
            n = n if rng.random() < 0.8 else max(n - int(rng.integers(0, 3)), 0)
            w = 0 if rng.random() < 0.15 else int(rng.integers(0, 2 ** 63)) * 2 + 1
            rows.append((r, n, w - 2 ** 64 if w >= 2 ** 63 else w))
    reqs, seq, masks = (np.array([x[i] for x in rows]) for i in range(3))
    q, q64 = queries(rng, len(rows), heads, "bf16")
    for lse in (True, False):
        out, ls, status = call_tree(cuda, q, cache, seq, masks, reqs.astype(np.int32), lse=lse)
        assert status == 1
        for t, (r, n, w) in enumerate(rows):
            pos = [] if r > 3 else list(range(n)) + [n + j for j in range(64) if (w >> j) & 1]
            kv = cache.kv[min(r, 3)][np.array(pos, np.int64)]
            check(out[t], ls[t] if lse else None, *attention64(q64[t], kv, BMM1, 1.0))


def test_shared_tiles_over_a_long_context(cuda):
    """Shared tiles cut into parts and joined, rows in ranges of several requests, a caller's workspace full of ones."""
    from ssengine_b200 import mla

    rng = np.random.default_rng(60)
    lens = [9001, 700, 20000]
    trees = [wild(rng, 20), wild(rng, 33), wild(rng, 9)]
    cache = Cache(rng, [n + len(t) for n, t in zip(lens, trees)])
    seq, masks, reqs, seen = tree_rows(trees, lens)
    for heads in (16, 30):
        q, q64 = queries(rng, len(seq), heads, "e4m3")
        ws = torch.full((mla.decode_workspace_bytes(len(seq), heads),), 0xFF, dtype=torch.uint8, device=cuda)
        out, lse, status = call_tree(cuda, q, cache, seq, masks, np.array(reqs, np.int32), workspace=ws)
        assert status == 0
        for t in range(0, len(seq), 3):
            check(out[t], lse[t], *attention64(q64[t], cache.kv[reqs[t]][seen[t]], BMM1, 1.0))


def test_chain_equals_decode(cuda):
    """A chain's nodes are the draft rows of `mla.decode`, bit for bit: the same units of the same tokens."""
    from ssengine_b200 import mla

    rng = np.random.default_rng(5)
    cache = Cache(rng, [777])
    q, _ = queries(rng, 5, 64, "bf16")
    out, _, _ = call_tree(cuda, q, cache, [772] * 5, [(2 << i) - 1 for i in range(5)], np.zeros(5, np.int32))
    want = torch.empty(5, 64, 512, dtype=torch.bfloat16, device=cuda)
    mla.decode(q.to(cuda), torch.from_numpy(cache.bytes).to(cuda), torch.from_numpy(cache.table).to(cuda),
               torch.tensor([773, 774, 775, 776, 777], dtype=torch.int32, device=cuda), BMM1, want,
               reqs=torch.zeros(5, dtype=torch.int32, device=cuda))
    torch.cuda.synchronize()
    assert (out == want.double().cpu().numpy()).all()


def test_long_context_is_split(cuda):
    rng = np.random.default_rng(6)
    cache = Cache(rng, [40001 + 3])
    q, q64 = queries(rng, 3, 64, "bf16")
    out, lse, status = call_tree(cuda, q, cache, [40001] * 3, [1, 3, 5], np.zeros(3, np.int32))
    assert status == 0
    for t, p in enumerate(([0], [0, 1], [0, 2])):
        check(out[t], lse[t], *attention64(q64[t], cache.kv[0][np.r_[0:40001, 40001 + np.array(p)]], BMM1, 1.0))


@pytest.mark.parametrize("heads", [2, 16, 64])
def test_thousands_of_rows(cuda, heads):
    """More rows than the plan keeps close by (4,096), and one that fills that place to the last row."""
    rng = np.random.default_rng(heads)
    lens = [int(n) for n in rng.integers(0, 150, 72)]
    trees = [wild(rng, 57) for _ in lens]
    lens[3] = -1                                         # a request whose rows hold nothing
    cache = Cache(rng, [max(n, 0) + 57 for n in lens])
    seq, masks, reqs, seen = tree_rows(trees, lens)
    q, q64 = queries(rng, len(seq), heads, "bf16")
    for T in (4096, 4104):
        out, lse, status = call_tree(cuda, q[:T], cache, seq[:T], masks[:T], np.array(reqs[:T], np.int32))
        assert status == 0 and np.isfinite(out).all()
        for t in [0, 3 * 57, 4 * 57 - 1, 4095, T - 1] + [int(t) for t in rng.integers(0, T, 40)]:
            some = seen[t] if lens[reqs[t]] >= 0 else np.zeros(0, np.int64)
            check(out[t], lse[t], *attention64(q64[t], cache.kv[reqs[t]][some], BMM1, 1.0))


def test_missing_pages_and_bad_requests(cuda):
    """A missing page in the tree or past the table leaves its tokens out; a bad request gives zeros and status 1."""
    rng = np.random.default_rng(7)
    cache = Cache(rng, [256 + 20, 128 + 30, 384])          # the last one fills its pages
    cache.table[0, 2] = -1                                  # nodes 0 .. 19 of request 0 lie there
    q, q64 = queries(rng, 4, 64, "e4m3")
    out, lse, status = call_tree(cuda, q, cache, [256, 150, 300, 2 ** 31 - 1], [3, 1, 255, 1], np.array([0, 1, 7, 2], np.int32))
    assert status == 1
    check(out[0], lse[0], *attention64(q64[0], cache.kv[0][:256], BMM1, 1.0))
    check(out[1], lse[1], *attention64(q64[1], cache.kv[1][:151], BMM1, 1.0))
    check(out[2], lse[2], *attention64(q64[2], cache.kv[2][:0], BMM1, 1.0))
    check(out[3], lse[3], *attention64(q64[3], cache.kv[2], BMM1, 1.0))      # the table ends before the length


def test_captured_tree_call_follows_masks_and_lengths(cuda):
    from ssengine_b200 import mla

    rng = np.random.default_rng(8)
    cache = Cache(rng, [464, 364])
    kv, tb = torch.from_numpy(cache.bytes).to(cuda), torch.from_numpy(cache.table).to(cuda)
    q, q64 = queries(rng, 2, 64, "bf16")
    q = q.to(cuda)
    seq = torch.tensor([100, 300], dtype=torch.int32, device=cuda)
    anc = torch.tensor([1, 1], dtype=torch.int64, device=cuda)
    out = torch.empty(2, 64, 512, dtype=torch.bfloat16, device=cuda)
    mla.decode_tree(q, kv, tb, seq, anc, BMM1, out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        mla.decode_tree(q, kv, tb, seq, anc, BMM1, out)
    for lens, words in (([64, 300], [5, 1 << 40]), ([400, 0], [-1, 0]), ([1, 129], [9, 3])):
        seq.copy_(torch.tensor(lens, dtype=torch.int32))
        anc.copy_(torch.tensor(words))
        g.replay()
        torch.cuda.synchronize()
        got = out.double().cpu().numpy()
        for t in range(2):
            seen = list(range(lens[t])) + [lens[t] + j for j in range(64) if (words[t] >> j) & 1]
            check(got[t], None, *attention64(q64[t], cache.kv[t][np.array(seen, np.int64)], BMM1, 1.0))


# ---- recurrence -----------------------------------------------------------------------------------------------------


def tree64(d, seqs, trees, H, lower_bound=-5.0):
    """Every node from its parent's state in float64: outputs [T, P] (NaN where no sequence has the row)."""
    P = H * D
    x, w = np.asarray(d["x"], np.float64)[:, :3 * P], np.asarray(d["w"], np.float64)
    gate = np.exp(ok.gate(d["g"], d["a_log"], d["dtb"], lower_bound, H, D)).reshape(-1, H, D)
    b = 1.0 / (1.0 + np.exp(-np.asarray(d["beta"], np.float64)))
    out = np.full((x.shape[0], P), np.nan)
    for (s, e, blk, init), parents in zip(seqs, trees):
        state = {-1: np.array(d["rst"][blk], np.float64) if init else np.zeros((H, D, D))}
        hist = {-1: np.array(d["cst"][blk], np.float64) if init else np.zeros((3, 3 * P))}
        for i, p in enumerate(parents):
            t = s + i
            hist[i] = np.concatenate([hist[p], x[t:t + 1]])[-4:]
            full = np.concatenate([np.zeros((4 - len(hist[i]), 3 * P)), hist[i]])
            y = (full.T * w).sum(1)
            y = (y / (1.0 + np.exp(-y))).reshape(3, H, D)
            q = y[0] / np.sqrt((y[0] ** 2).sum(1, keepdims=True) + 1e-6)
            k = y[1] / np.sqrt((y[1] ** 2).sum(1, keepdims=True) + 1e-6)
            S = state[p] * gate[t][:, None, :]
            u = b[t][:H, None] * (y[2] - np.einsum("hvk,hk->hv", S, k))
            state[i] = S + u[:, :, None] * k[:, None, :]
            out[t] = (np.einsum("hvk,hk->hv", state[i], q) * D ** -0.5).reshape(P)
    return out


def kda_layer(d, cuda):
    from ssengine_b200.kda import KdaLayer

    f = lambda a, t: torch.from_numpy(np.ascontiguousarray(a)).to(cuda, t)
    L = KdaLayer(f(d["w"], torch.bfloat16), f(d["a_log"], torch.float32), f(d["dtb"], torch.float32))
    dev = dict(x=f(d["x"], torch.bfloat16), g=f(d["g"], torch.bfloat16), beta=f(d["beta"], torch.bfloat16),
               cst=f(d["cst"], torch.bfloat16), rst=f(d["rst"], torch.float32))
    return L, dev


def run_tree(cuda, d, H, seqs, parents, max_nodes=64, stream=None):
    L, dev = kda_layer(d, cuda)
    T = dev["x"].shape[0]
    out = torch.full((T, H * D), -77.0, dtype=torch.bfloat16, device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    st = torch.tensor(seqs, dtype=torch.int32, device=cuda).reshape(-1, 4)
    par = torch.tensor(parents, dtype=torch.int32, device=cuda)
    torch.cuda.synchronize()
    before = dev["cst"].clone(), dev["rst"].clone()
    L.decode_tree(dev["x"], dev["g"], dev["beta"], out, st, par, dev["cst"], dev["rst"], max_nodes=max_nodes, stream=stream,
                  status=status)
    torch.cuda.synchronize()
    assert torch.equal(dev["cst"].view(torch.int16), before[0].view(torch.int16))      # left as they are
    assert torch.equal(dev["rst"].view(torch.int32), before[1].view(torch.int32))
    return out.double().cpu().numpy(), int(status.item())


def check_rows(out, want, H):
    """Heads' rows of nodes within the bar; rows of no sequence untouched."""
    for t in range(out.shape[0]):
        if np.isnan(want[t]).all():
            assert (out[t] == -77.0).all(), t
            continue
        o, w = out[t].reshape(H, D), want[t].reshape(H, D)
        bar = 2.0 ** -8 * np.abs(w) + 1e-3 * np.abs(w).max(axis=1, keepdims=True)
        assert (np.abs(o - w) <= bar).all(), (t, np.abs(o - w).max(), np.abs(w).max())


@pytest.mark.parametrize("H", [1, 2, 5])
@pytest.mark.parametrize("nodes", [1, 2, 3, 8, 15, 16, 17, 24, 31, 32, 33, 48, 63, 64])
def test_trees_of_every_size(cuda, H, nodes):
    rng = np.random.default_rng(100 * H + nodes)
    trees = [wild(rng, nodes), CHAIN(nodes), STAR(nodes), BINARY(nodes)][:4 if H < 5 else 1]
    T = nodes * len(trees)
    seqs = [(nodes * r, nodes * (r + 1), r, int(r != 3)) for r in range(len(trees))]
    d = kda_make(rng, T, H, len(trees))
    out, status = run_tree(cuda, d, H, seqs, sum(trees, []), max_nodes=nodes)
    assert status == 0
    check_rows(out, tree64(d, seqs, trees, H), H)


def test_ragged_trees_share_blocks_and_leave_rows(cuda):
    """Sequences of any length in any order, rows between them left alone, two trees on one block, a fresh request whose
    block holds NaN, a sequence without rows."""
    rng = np.random.default_rng(11)
    H = 2
    trees = [wild(rng, 20), wild(rng, 5), CHAIN(37), [], STAR(3), BINARY(64)]
    at, seqs = 2, []
    for r, t in enumerate(trees):
        seqs.append((at, at + len(t), [1, 1, 3, 2, 4, 0][r], int(r != 4)))
        at += len(t) + (r % 2)
    parents = np.full(at + 3, 99)                           # rows of no sequence: never looked at
    for (s, e, _, _), t in zip(seqs, trees):
        parents[s:e] = t
    d = kda_make(rng, at + 3, H, 6)
    d["rst"][4] = np.nan
    d["cst"][4] = np.nan
    order = [3, 0, 5, 1, 4, 2]
    out, status = run_tree(cuda, d, H, [seqs[i] for i in order], parents.tolist())
    assert status == 0
    check_rows(out, tree64(d, seqs, trees, H), H)


def test_what_is_no_tree_is_skipped(cuda):
    rng = np.random.default_rng(12)
    H, good = 2, wild(rng, 6)
    d = kda_make(rng, 64, H, 3)
    cases = [((8, 12, 0, 1), [-1, 1, 0, 0]), ((8, 12, 0, 1), [-1, -2, 0, 0]), ((8, 12, 0, 1), [0, 0, 0, 0]),
             ((8, 12, -1, 1), [-1, 0, 1, 2]), ((-1, 3, 0, 1), [-1] * 4), ((60, 65, 0, 1), [-1] * 4), ((12, 8, 0, 1), [-1] * 4),
             ((8, 25, 0, 1), [-1] * 17)]
    for seq, par in cases:
        parents = [-1] * 64
        parents[:6] = good
        parents[8:8 + len(par)] = par
        out, status = run_tree(cuda, d, H, [(0, 6, 1, 1), seq], parents, max_nodes=16)
        assert status == 1, seq
        check_rows(out, tree64(d, [(0, 6, 1, 1)], [good], H), H)


def test_extreme_gates(cuda):
    """Decays near 0 (their products down a path underflow) and at 1, betas at 0 and 1, huge and tiny conv inputs."""
    rng = np.random.default_rng(13)
    H, n = 2, 40
    trees = [CHAIN(n), wild(rng, n)]
    d = kda_make(rng, 2 * n, H, 2)
    d["g"] = d["g"] * 40.0
    d["beta"] = d["beta"] * 30.0
    d["x"][::7] *= 30.0
    d["x"][3::7] *= 1e-3
    seqs = [(0, n, 0, 1), (n, 2 * n, 1, 1)]
    d = {k: (torch.from_numpy(np.ascontiguousarray(v)).to(torch.bfloat16).float().numpy() if k in ("g", "beta", "x") else v)
         for k, v in d.items()}
    out, status = run_tree(cuda, d, H, seqs, sum(trees, []))
    assert status == 0
    check_rows(out, tree64(d, seqs, trees, H), H)


def test_batches_of_trees(cuda):
    """More requests and heads than run at once, trees of 1 to 32 nodes, one node's value NaN."""
    rng = np.random.default_rng(21)
    H, R = 5, 67
    trees = [wild(rng, int(n)) for n in rng.integers(1, 33, R)]
    trees[5], trees[6], trees[7] = CHAIN(32), STAR(31), BINARY(32)
    ends = np.cumsum([0] + [len(t) for t in trees])
    d = kda_make(rng, int(ends[-1]), H, R)
    d["x"][ends[7] + 2, 2 * H * D + 3 * D + 11] = np.nan
    seqs = [(int(ends[r]), int(ends[r + 1]), R - 1 - r, int(r % 5 != 2)) for r in range(R)]
    want = tree64(d, seqs, trees, H)
    out, status = run_tree(cuda, d, H, seqs, sum(trees, []), max_nodes=32)
    assert status == 0
    gone = np.isnan(want)
    assert gone.any() and (gone.sum(axis=0) > 0).sum() == 1 and (np.isnan(out) == gone).all()
    check_rows(np.where(gone, 0, out), np.where(gone, 0, want), H)


@pytest.mark.parametrize("n", [12, 30, 50])
@pytest.mark.parametrize("where", ["v", "k", "q", "gate", "beta"])
def test_what_is_not_finite_reaches_its_descendants_alone(cuda, n, where):
    """One node's input NaN or infinite: what the recurrence makes NaN is (of a value one channel, of a key, a gate or a beta
    the head, of a query the node and those whose conv has it), every other output is as if it were not there."""
    rng = np.random.default_rng(n)
    H, P = 2, 2 * D
    trees = [wild(rng, n), STAR(n)]
    d = kda_make(rng, 2 * n, H, 2)
    d = {k: (torch.from_numpy(np.ascontiguousarray(v)).to(torch.bfloat16).float().numpy() if k in ("g", "beta", "x") else v)
         for k, v in d.items()}
    seqs = [(0, n, 0, 1), (n, 2 * n, 1, 1)]
    for bad in (np.nan, np.inf):
        if bad == np.inf and where in ("gate", "beta"):
            continue                                      # finite there: a decay of e^-5 or 1, a beta of 0 or 1
        e = {k: np.array(v) for k, v in d.items()}
        for row in (n // 3, n + 4):
            if where == "beta":
                e["beta"][row, 1] = bad
            elif where == "gate":
                e["g"][row, D + 17] = bad
            else:
                e["x"][row, {"q": 0, "k": 1, "v": 2}[where] * P + D + 17] = bad
        with np.errstate(all="ignore"):
            want = tree64(e, seqs, trees, H).reshape(-1, H, D)
        out, status = run_tree(cuda, e, H, seqs, sum(trees, []))
        out = out.reshape(-1, H, D)
        gone = ~np.isfinite(want)
        assert status == 0 and gone.any() and not gone[:, 0].any() and (~np.isfinite(out) == gone).all()
        bar = 2.0 ** -8 * np.abs(want) + 1e-3 * np.where(gone, 0, np.abs(want)).max(axis=2, keepdims=True)
        assert (np.abs(out - want) <= bar)[~gone].all()


def test_strided_rows_streams_and_repeats(cuda):
    """Rows cut from wider ones, another stream, the same bits every time and for every max_nodes' form."""
    rng = np.random.default_rng(14)
    H, n = 3, 13
    tree = wild(rng, n)
    d = kda_make(rng, n, H, 2)
    L, dev = kda_layer(d, cuda)
    wide = torch.zeros(n, 3 * H * D + 400, dtype=torch.bfloat16, device=cuda)
    wide[:, 10:10 + dev["x"].shape[1]] = dev["x"]
    gw = torch.zeros(n, H * D + 6, dtype=torch.bfloat16, device=cuda)
    gw[:, 2:2 + H * D] = dev["g"]
    beta = wide[:, 3 * H * D + 100:3 * H * D + 100 + H]
    beta.copy_(dev["beta"])
    ow = torch.full((n, H * D + 9), -77.0, dtype=torch.bfloat16, device=cuda)
    out = ow[:, 5:5 + H * D]
    seqs = torch.tensor([[0, n, 1, 1]], dtype=torch.int32, device=cuda)
    par = torch.tensor(tree, dtype=torch.int32, device=cuda)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for most, stream in ((64, None), (13, side), (32, None), (13, None)):
        out.fill_(0)
        torch.cuda.synchronize()
        L.decode_tree(wide[:, 10:], gw[:, 2:], beta, out, seqs, par, dev["cst"], dev["rst"], max_nodes=most, stream=stream)
        torch.cuda.synchronize()
        got.append(out.clone())
    assert torch.equal(got[1], got[3])
    for o in got:
        check_rows(o.double().cpu().numpy(), tree64(d, [(0, n, 1, 1)], [tree], H), H)
    assert (ow[:, :5] == -77.0).all() and (ow[:, 5 + H * D:] == -77.0).all()


# ---- advance --------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("H", [1, 2, 5])
def test_advance_is_the_recurrence_of_the_rows(cuda, H):
    """Runs of 0 to 9 listed rows, fresh requests, the same row twice; rows and blocks of no sequence left alone."""
    rng = np.random.default_rng(20 + H)
    T, lens = 60, [1, 4, 0, 9, 2, 5]
    d = kda_make(rng, T, H, len(lens) + 2)
    rows = rng.integers(0, T, sum(lens) + 3)
    rows[6] = rows[7]
    seqs, at = [], 1
    for r, n in enumerate(lens):
        seqs.append((at, at + n, [5, 0, 3, 1, 7, 4][r], int(r != 3)))
        at += n
    picked = {**d, "x": d["x"][rows], "g": d["g"][rows], "beta": d["beta"][rows]}
    _, cst, rst = recurrence64(picked, seqs, H)
    L, dev = kda_layer(d, cuda)
    before = dev["cst"].clone(), dev["rst"].clone()
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    L.advance(dev["x"], dev["g"], dev["beta"], torch.tensor(rows, dtype=torch.int32, device=cuda),
              torch.tensor(seqs, dtype=torch.int32, device=cuda), dev["cst"], dev["rst"], status=status)
    torch.cuda.synchronize()
    assert int(status.item()) == 0
    touched = {b for s, e, b, _ in seqs if e > s}
    for b in range(len(lens) + 2):
        got = dev["rst"][b].double().cpu().numpy()
        if b not in touched:
            assert torch.equal(dev["rst"][b], before[1][b]) and torch.equal(dev["cst"][b], before[0][b])
            continue
        assert np.linalg.norm(got - rst[b]) <= 1e-5 * np.linalg.norm(rst[b]), b
        assert (dev["cst"][b].double().cpu().numpy() == cst[b]).all(), b


def test_advance_skips_what_it_cannot_take(cuda):
    rng = np.random.default_rng(30)
    H, T = 2, 10
    for seq, rows in (((2, 4, 0, 1), [1, 2, 3, 10]), ((2, 4, 0, 1), [1, 2, -1, 3]), ((2, 5, 0, 1), [1, 2, 3, 4]),
                      ((-1, 2, 0, 1), [1, 2, 3, 4]), ((3, 2, 0, 1), [1, 2, 3, 4]), ((2, 4, -1, 1), [1, 2, 3, 4])):
        d = kda_make(rng, T, H, 2)
        L, dev = kda_layer(d, cuda)
        want = recurrence64({**d, "x": d["x"][[1, 2]], "g": d["g"][[1, 2]], "beta": d["beta"][[1, 2]]}, [(0, 2, 1, 1)], H)
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        L.advance(dev["x"], dev["g"], dev["beta"], torch.tensor(rows, dtype=torch.int32, device=cuda),
                  torch.tensor([(0, 2, 1, 1), seq], dtype=torch.int32, device=cuda), dev["cst"], dev["rst"], status=status)
        torch.cuda.synchronize()
        assert int(status.item()) == 1, seq
        assert (dev["rst"][0].cpu().numpy() == d["rst"][0]).all()
        got = dev["rst"][1].double().cpu().numpy()
        assert np.linalg.norm(got - want[2][1]) <= 1e-5 * np.linalg.norm(want[2][1])


def test_captured_tree_step_and_advance(cuda):
    """One graph of a tree's check and the advance by its path, replayed with other trees, paths and inputs."""
    rng = np.random.default_rng(31)
    H, n = 2, 12
    d = kda_make(rng, n, H, 2)
    L, dev = kda_layer(d, cuda)
    par = torch.tensor(CHAIN(n), dtype=torch.int32, device=cuda)
    seqs = torch.tensor([(0, n, 1, 1)], dtype=torch.int32, device=cuda)
    rows = torch.zeros(4, dtype=torch.int32, device=cuda)
    moves = torch.tensor([(0, 0, 1, 1)], dtype=torch.int32, device=cuda)
    out = torch.empty(n, H * D, dtype=torch.bfloat16, device=cuda)

    def step():
        L.decode_tree(dev["x"], dev["g"], dev["beta"], out, seqs, par, dev["cst"], dev["rst"], max_nodes=16)
        L.advance(dev["x"], dev["g"], dev["beta"], rows, moves, dev["cst"], dev["rst"])

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    host = dict(d)
    for k in range(3):
        tree = wild(rng, n)
        take = path(tree, int(rng.integers(0, n)))[:4]
        x = kda_make(rng, n, H, 2)["x"]
        par.copy_(torch.tensor(tree, dtype=torch.int32))
        rows[:len(take)].copy_(torch.tensor(take, dtype=torch.int32))
        moves.copy_(torch.tensor([(0, len(take), 1, 1)], dtype=torch.int32))
        dev["x"].copy_(torch.from_numpy(x).to(torch.bfloat16))
        host["x"], host["cst"], host["rst"] = x, dev["cst"].float().cpu().numpy(), dev["rst"].cpu().numpy()
        g.replay()
        torch.cuda.synchronize()
        check_rows(out.double().cpu().numpy(), tree64(host, [(0, n, 1, 1)], [tree], H), H)
        picked = {**host, **{c: np.asarray(host[c])[take] for c in ("x", "g", "beta")}}
        _, cst, rst = recurrence64(picked, [(0, len(take), 1, 1)], H)
        assert np.linalg.norm(dev["rst"][1].double().cpu().numpy() - rst[1]) <= 1e-5 * np.linalg.norm(rst[1])
        assert (dev["cst"][1].double().cpu().numpy() == cst[1]).all()
