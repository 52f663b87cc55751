"""Rows of cache views moved by lists on the GPU (`kvpages.RowMover`, `ssb_move_rows`; `StageKv.move_states`, `move_pages`,
`move_tokens`) against copies on the host, byte for byte."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def moved(views, lists, src, dst):
    """The rule, view by view: of a group's entries (both ids given, not equal, within the rows) the first per destination."""
    out = [v.copy() for v in views]
    for v, o, l in zip(views, out, lists):
        for g in range(src.shape[1]):
            seen = set()
            for s, d in zip(src[l, g].tolist(), dst[l, g].tolist()):
                if s < 0 or d < 0 or s >= len(v) or d >= len(v):
                    continue
                if d in seen:
                    continue
                seen.add(d)
                o[d] = v[s]
    return out


def run(cuda, shapes, lists, src, dst, pitch=None, seed=0, stream=None):
    """Views of `shapes` (rows, bytes), rows `pitch` bytes longer apart; -> (got, wanted, status, the bytes between rows kept)."""
    from ssengine_b200.kvpages import RowMover

    rng = np.random.default_rng(seed)
    wide = [torch.from_numpy(rng.integers(0, 256, (r, n + (pitch or 0)), dtype=np.uint8)).to(cuda) for r, n in shapes]
    host = [w.cpu().numpy() for w in wide]
    views = [w[:, :n] for w, (_, n) in zip(wide, shapes)]
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(cuda)
    torch.cuda.synchronize()
    RowMover(views, lists)(t(src), t(dst), stream=stream, status=status)
    torch.cuda.synchronize()
    want = moved([h[:, :n] for h, (_, n) in zip(host, shapes)], lists, src, dst)
    between = all((w[:, n:].cpu().numpy() == h[:, n:]).all() for w, h, (_, n) in zip(wide, host, shapes))
    return [v.cpu().numpy() for v in views], want, int(status.item()), between


@pytest.mark.parametrize("n", [1, 2, 3, 4, 7, 16, 17, 33, 64])
@pytest.mark.parametrize("nbytes", [16, 576, 4096, 32768 + 48])
def test_permutations_in_place(cuda, n, nbytes):
    """Every group of a random map of its own rows (cycles, one source for several, rows kept), two views, ragged slices."""
    rng = np.random.default_rng(n * 7 + nbytes)
    G = 3
    ids = rng.permutation(G * n + 5)[:G * n].reshape(1, G, n).astype(np.int32)
    src = np.stack([row[rng.integers(0, n, n)] for row in ids[0]])[None]
    src[0, 0] = np.roll(ids[0, 0], 1)                      # one cycle through all
    got, want, status, between = run(cuda, [(G * n + 5, nbytes), (G * n + 9, 3 * nbytes)], [0, 0], src, ids, pitch=32)
    assert status == 0 and between
    assert all((g == w).all() for g, w in zip(got, want))


def test_lists_of_their_own_and_entries_left_out(cuda):
    rng = np.random.default_rng(1)
    src = np.full((3, 2, 5), -1, np.int32)
    dst = np.full((3, 2, 5), -1, np.int32)
    src[0, 0], dst[0, 0] = [1, 2, 3, -1, 4], [0, 1, 2, 9, -1]     # a shift; ids missing on either side
    src[0, 1], dst[0, 1] = [7, 7, 7, 8, 5], [7, 5, 6, 6, 8]       # one source for two, one kept, one destination twice
    src[1, 0], dst[1, 0] = [0, 1, 0, 1, 0], [1, 0, 2, 3, 4]
    src[2, 1], dst[2, 1] = [3, 3, 3, 3, 3], [0, 0, 0, 0, 0]
    shapes = [(10, 640), (6, 16), (4, 70000 // 16 * 16), (10, 576)]
    got, want, status, between = run(cuda, shapes, [0, 1, 2, 0], src, dst, pitch=16)
    assert status == 0 and between
    assert all((g == w).all() for g, w in zip(got, want))


def test_ids_past_a_view_move_nothing_there(cuda):
    src = np.array([[[0, 1, 9], [4, 3, 2 ** 31 - 1]]], np.int32)
    dst = np.array([[[5, 2 ** 31 - 1, 6], [3, 6, 7]]], np.int32)
    got, want, status, between = run(cuda, [(8, 64), (6, 64)], [0, 0], src, dst)
    assert status == 1
    assert all((g == w).all() for g, w in zip(got, want))


def test_nothing_to_do_and_a_single_row(cuda):
    for src, dst, rows in ((np.zeros((1, 0, 3)), np.zeros((1, 0, 3)), 4), (np.zeros((1, 3, 0)), np.zeros((1, 3, 0)), 4),
                           (np.array([[[0]]]), np.array([[[0]]]), 1)):
        got, want, status, _ = run(cuda, [(rows, 48)], [0], src.astype(np.int32), dst.astype(np.int32))
        assert status == 0 and (got[0] == want[0]).all()


def test_rows_past_two_to_the_31_bytes(cuda):
    """Row addresses past 2^32 bytes: 1,100 rows 4,939,776 bytes apart, 1 MiB of them moved."""
    from ssengine_b200.kvpages import RowMover

    big = torch.zeros(1100, 8576 * 576, dtype=torch.uint8, device=cuda)
    part = big[:, :1 << 20]
    rng = np.random.default_rng(3)
    rows = {i: rng.integers(0, 256, 1 << 20, dtype=np.uint8) for i in (1099, 3, 600)}
    for i, b in rows.items():
        part[i] = torch.from_numpy(b).to(cuda)
    t = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)
    RowMover([part])(t([[1099, 3, 600]]), t([[3, 1098, 1099]]))
    torch.cuda.synchronize()
    for d, s in ((3, 1099), (1098, 3), (1099, 600), (600, 600)):
        assert (part[d].cpu().numpy() == rows[s]).all()
    assert not big[1098, 1 << 20:].any()


def test_another_stream_and_a_captured_call(cuda):
    from ssengine_b200.kvpages import RowMover

    rng = np.random.default_rng(5)
    src = np.array([[[1, 2, 0]]], np.int32)
    dst = np.array([[[0, 1, 2]]], np.int32)
    got, want, _, _ = run(cuda, [(4, 4096)], [0], src, dst, stream=torch.cuda.Stream())
    assert (got[0] == want[0]).all()
    view = torch.from_numpy(rng.integers(0, 256, (6, 1600), dtype=np.uint8)).to(cuda)
    s, d = torch.from_numpy(src).to(cuda), torch.from_numpy(dst).to(cuda)
    mover = RowMover([view])
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        mover(s, d)
    for a, b in (([1, 2, 0], [0, 1, 2]), ([5, 5, -1], [0, 4, 1]), ([0, 3, 4], [3, 0, 5])):
        s.copy_(torch.tensor([[a]], dtype=torch.int32))
        d.copy_(torch.tensor([[b]], dtype=torch.int32))
        host = view.cpu().numpy()
        g.replay()
        torch.cuda.synchronize()
        assert (view.cpu().numpy() == moved([host], [0], np.array([[a]]), np.array([[b]]))[0]).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_stage_moves_touch_their_views_only(cuda, fp8):
    """States, pages and tokens of a stage's caches (three KDA layers of two heads and a DSA layer, then five more KDA
    layers): each view moved by its list, every other byte kept."""
    from ssengine_b200.kvpages import StageKv

    layers = list(range(9))
    kv = StageKv(layers, lambda i: i % 4 == 3, 20, 2, cuda, pool_fp8=fp8)
    rng = np.random.default_rng(9)
    tensors = kv.pages + kv.pool + kv.tail
    fill = lambda t: t.view(torch.uint8).copy_(torch.from_numpy(
        rng.integers(0, 256, tuple(t.view(torch.uint8).shape), dtype=np.uint8)))
    for t in tensors:
        fill(t)
    host = lambda: [t.view(torch.uint8).cpu().numpy().copy() for t in tensors]
    t = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)
    n_dsa = len(kv.dsa_layers)

    before = host()
    # a block belongs to one state group: layers of different groups share a tensor
    src = [[[1 + 3 * g, 2 + 3 * g]] for g in range(6)]
    dst = [[[3 + 3 * g, 1 + 3 * g]] for g in range(6)]
    kv.move_states(t(src), t(dst))
    torch.cuda.synchronize()
    want = [b.copy() for b in before]
    state = kv.rec_off + 2 * 128 * 128 * 4
    for i in kv.kda_layers:
        g, j = kv.group[i], kv.slot[i]
        for s, d in zip(src[g][0], dst[g][0]):
            want[j][d, :state] = before[j][s, :state]
    for j in range(n_dsa):
        for s, d in zip(src[5][0], dst[5][0]):
            want[len(kv.pages) + n_dsa + j][d] = before[len(kv.pages) + n_dsa + j][s]
    assert all((a == b).all() for a, b in zip(host(), want))

    before = host()
    src, dst = [70, 3, 500], [3, 140, 70]
    kv.move_pages(t([src]), t([dst]))
    torch.cuda.synchronize()
    want = [b.copy() for b in before]
    rows = 33 if fp8 else 32
    for s, d in zip(src, dst):
        for j in range(n_dsa):
            a, b = want[j].reshape(20 * 67, -1), before[j].reshape(20 * 67, -1)
            a[d] = b[s]
            p = len(kv.pages) + j
            want[p][d * rows:(d + 1) * rows] = before[p][s * rows:(s + 1) * rows]
    assert all((a == b).all() for a, b in zip(host(), want))

    before = host()
    src, dst = [9000, 9003, 9010], [9000, 9001, 9002]
    kv.move_tokens(t([src]), t([dst]))
    torch.cuda.synchronize()
    want = [b.copy() for b in before]
    for s, d in zip(src, dst):
        for j in range(n_dsa):
            want[j].reshape(-1, 576)[d] = before[j].reshape(-1, 576)[s]
    assert all((a == b).all() for a, b in zip(host(), want))
