"""A beam search's selection on the GPU (`beam.select`, `ssb_beam_select`) against the definition in float64.

Tolerances, derived before the first run: a candidate's score is a float32 rounding (2^-24 of it) of a float64 sum whose log
sum of exponentials is off by at most the exponentials' own error, 2^-22 relative, and a thread's fp32 sum of at most 592
terms (151,552 over 256 threads), 592 x 2^-24 = 3.5e-5 at worst and about its square root, 1.5e-6, as the roundings fall:
the bar 4e-5 absolute. Tokens and parents are equal wherever neighbouring candidates lie further apart than twice that;
where they do not (they may then change places), the sets have to agree up to such neighbours. Equal candidates (the same
logits in the same or in identical beams) are in exact order."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = 4e-5


def select64(x, scores, k, finished=None, pad=0):
    """(scores, parents, tokens) of the k best of each request, -inf / -1 / -1 where there are fewer."""
    G, B = scores.shape
    V = x.shape[1]
    out = np.full((G, k), -np.inf), np.full((G, k), -1, np.int64), np.full((G, k), -1, np.int64)
    for g in range(G):
        c = []
        for b in range(B):
            s = float(scores[g, b])
            if not np.isfinite(s):
                continue
            if finished is not None and finished[g, b]:
                c.append((-s, b, pad))
                continue
            row = x[g * B + b].astype(np.float64)
            with np.errstate(all="ignore"):
                m = np.nanmax(row) if not np.isnan(row).all() else np.nan
                lse = m + np.log(np.exp(row - m).sum()) if np.isfinite(m) else m
            if not np.isfinite(lse):
                continue
            best = np.lexsort((np.arange(V), -row))[:k]
            c += [(-(s + (row[v] - lse)), b, int(v)) for v in best if row[v] > -np.inf]
        for i, (s, b, v) in enumerate(sorted(c)[:k]):
            out[0][g, i], out[1][g, i], out[2][g, i] = -s, b, v
    return out


def run(cuda, x, scores, k, finished=None, pad=0, bf16=False, **kw):
    from ssengine_b200 import beam

    t = x if torch.is_tensor(x) else torch.from_numpy(np.ascontiguousarray(x, np.float32))
    t = t.to(cuda, torch.bfloat16 if bf16 else torch.float32) if not t.is_cuda else t
    f = None if finished is None else torch.from_numpy(np.ascontiguousarray(finished)).to(cuda)
    s, p, v = beam.select(t, torch.from_numpy(np.ascontiguousarray(scores, np.float32)).to(cuda), k, finished=f, pad=pad, **kw)
    torch.cuda.synchronize()
    return s.double().cpu().numpy(), p.long().cpu().numpy(), v.cpu().numpy()


def check(got, want, exact=False):
    assert ((got[0] == -np.inf) == (want[0] == -np.inf)).all()
    live = want[0] > -np.inf
    assert (np.abs(got[0][live] - want[0][live]) <= TOL + 2.0 ** -23 * np.abs(want[0][live])).all()
    assert (got[1][~live] == -1).all() and (got[2][~live] == -1).all()
    for g in range(len(want[0])):
        n = int(live[g].sum())
        a = list(zip(got[1][g, :n].tolist(), got[2][g, :n].tolist()))
        b = list(zip(want[1][g, :n].tolist(), want[2][g, :n].tolist()))
        if a == b:
            continue
        assert not exact, (g, a, b)
        assert len(set(a)) == n
        for i in range(n):                                   # changed places lie within the bar of one another
            if a[i] != b[i] and a[i] in b:
                assert abs(want[0][g, i] - want[0][g, b.index(a[i])]) <= 2 * TOL, (g, i)
            elif a[i] != b[i]:
                assert abs(want[0][g, i] - want[0][g, n - 1]) <= 2 * TOL, (g, i)


@pytest.mark.parametrize("V", [1, 2, 31, 32, 33, 255, 1000, 2047, 4097, 32001, 151552])
@pytest.mark.parametrize("bf16", [False, True])
def test_vocabularies(cuda, V, bf16):
    rng = np.random.default_rng(V)
    G, B = 3, 4
    x = torch.from_numpy(rng.standard_normal((G * B, V)).astype(np.float32) * 3)
    x = x.to(torch.bfloat16) if bf16 else x
    scores = -rng.random((G, B)).astype(np.float32) * 5
    for k in (1, 4, 11):
        check(run(cuda, x, scores, k, bf16=bf16), select64(x.float().numpy(), scores, k))


@pytest.mark.parametrize("G,B,k", [(1, 1, 1), (1, 1, 64), (1, 64, 64), (200, 2, 3), (7, 16, 32), (2, 5, 7), (40, 8, 16)])
def test_requests_beams_and_counts(cuda, G, B, k):
    rng = np.random.default_rng(G * 100 + B)
    V = 5003
    x = rng.standard_normal((G * B, V)).astype(np.float32) * 4
    scores = -rng.random((G, B)).astype(np.float32)
    finished = rng.random((G, B)) < 0.3
    check(run(cuda, x, scores, k), select64(x, scores, k))
    check(run(cuda, x, scores, k, finished=finished, pad=5002), select64(x, scores, k, finished, 5002))
    check(run(cuda, x, scores, k, finished=np.ones((G, B), np.uint8), pad=0), select64(x, scores, k, np.ones((G, B)), 0))


def test_equal_candidates_go_to_the_lower_place(cuda):
    """Constant rows, few distinct logits, identical beams with identical scores, -0 and 0: exact order."""
    rng = np.random.default_rng(2)
    G, B, V, k = 4, 3, 6001, 13
    rows = [np.zeros((G * B, V)), rng.integers(0, 3, (G * B, V)).astype(float), np.tile(rng.standard_normal(V) * 2, (G * B, 1)),
            np.where(rng.random((G * B, V)) < 0.5, -0.0, 0.0)]
    for x in rows:
        x = x.astype(np.float32)
        scores = np.full((G, B), -1.5, np.float32)
        same = np.tile(x[:1], (G * B, 1))                    # every beam the same: equal candidates in every beam
        check(run(cuda, same, scores, k), select64(same, scores, k), exact=True)
        check(run(cuda, x, scores - np.arange(B, dtype=np.float32) * 0.5, k),
              select64(x, scores - np.arange(B, dtype=np.float32) * 0.5, k))


def test_orders_that_fill_the_lists(cuda):
    """Ascending rows (every logit beats all before it), descending ones, one huge value at the end."""
    V, k = 40009, 64
    up = np.linspace(-8, 8, V).astype(np.float32)
    end = np.full(V, -3.0, np.float32)
    end[-1] = 30.0
    x = np.stack([up, up[::-1], np.concatenate([up[::2], up[1::2]]), end])
    scores = np.array([[0.0, -0.25, -0.5, -40.0]], np.float32)
    check(run(cuda, x, scores, k), select64(x, scores, k))
    for b in range(4):
        check(run(cuda, x[b:b + 1], scores[:, :1], k), select64(x[b:b + 1], scores[:, :1], k), exact=b != 3)


def test_what_is_no_candidate(cuda):
    """Masked logits, rows with none left, NaN and infinite logits, scores of -inf, +inf and NaN; fewer candidates than k."""
    rng = np.random.default_rng(4)
    G, B, V, k = 3, 6, 3001, 8
    x = rng.standard_normal((G * B, V)).astype(np.float32)
    scores = -rng.random((G, B)).astype(np.float32)
    x[0] = -np.inf
    x[1, 5] = np.nan
    x[2, 77] = np.inf
    x[3, 1000:] = -np.inf
    scores[0, 4], scores[0, 5] = -np.inf, np.nan
    x[B:2 * B] = -np.inf                                     # request 1: five candidates in all
    x[B + 2, 2999], x[B + 2, 3], x[B + 5, 0], x[B + 5, 3000], x[B + 5, 1500] = 1.0, 1.0, -2.0, 5.0, 0.0
    scores[1, 0] = np.inf
    x[2 * B:] = -np.inf                                      # request 2: none
    got, want = run(cuda, x, scores, k), select64(x, scores, k)
    check(got, want)
    assert (want[0][1] > -np.inf).sum() == 5 and not (want[0][2] > -np.inf).any()
    big = rng.standard_normal((4, V)).astype(np.float32) * 1e30
    s = np.zeros((1, 4), np.float32)
    got, want = run(cuda, big, s, k), select64(big, s, k)
    assert (got[1] == want[1]).all() and (got[2] == want[2]).all()
    assert np.allclose(got[0], want[0], rtol=1e-6, atol=TOL)


def test_rows_apart_odd_addresses_streams_and_workspaces(cuda):
    """Rows cut out of wider ones at every offset from a 16-byte boundary, another stream, a caller's workspace full of ones,
    the caller's outputs; the same bits every time."""
    from ssengine_b200 import beam

    rng = np.random.default_rng(6)
    V, k = 9001, 5
    scores = -rng.random((2, 3)).astype(np.float32)
    sc = torch.from_numpy(scores).to(cuda)
    side = torch.cuda.Stream()
    for bf16 in (False, True):
        wide = torch.from_numpy(rng.standard_normal((6, V + 29)).astype(np.float32) * 3)
        wide = wide.to(torch.bfloat16) if bf16 else wide
        for off in range(9):
            x = wide.to(cuda)[:, off:off + V]
            want = select64(wide[:, off:off + V].float().numpy(), scores, k)
            ws = torch.full((beam.workspace_bytes(2, 3, V, k),), 0xFF, dtype=torch.uint8, device=cuda)
            out = (torch.empty(2, k, device=cuda), torch.empty(2, k, dtype=torch.int32, device=cuda),
                   torch.empty(2, k, dtype=torch.int64, device=cuda))
            torch.cuda.synchronize()
            beam.select(x, sc, k, out=out, workspace=ws, stream=side if off % 2 else None)
            torch.cuda.synchronize()
            check((out[0].double().cpu().numpy(), out[1].long().cpu().numpy(), out[2].cpu().numpy()), want)
            again = beam.select(x, sc, k)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_captured_selection_follows_its_inputs(cuda):
    from ssengine_b200 import beam

    rng = np.random.default_rng(7)
    G, B, V, k = 2, 4, 20011, 4
    x, sc = torch.empty(G * B, V, device=cuda), torch.empty(G, B, device=cuda)
    fin = torch.zeros(G, B, dtype=torch.bool, device=cuda)
    x.zero_(), sc.zero_()
    beam.select(x, sc, k, finished=fin)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = beam.select(x, sc, k, finished=fin)
    for i in range(3):
        hx, hs = rng.standard_normal((G * B, V)).astype(np.float32) * 3, -rng.random((G, B)).astype(np.float32)
        hf = rng.random((G, B)) < 0.3
        x.copy_(torch.from_numpy(hx))
        sc.copy_(torch.from_numpy(hs))
        fin.copy_(torch.from_numpy(hf))
        g.replay()
        torch.cuda.synchronize()
        check((out[0].double().cpu().numpy(), out[1].long().cpu().numpy(), out[2].cpu().numpy()), select64(hx, hs, k, hf, 0))


def test_scores_in_place(cuda):
    """A search's loop keeps its scores in one tensor: the new ones take the place of those read."""
    from ssengine_b200 import beam

    rng = np.random.default_rng(31)
    G, B, V = 150, 8, 4100
    scores = -rng.random((G, B)).astype(np.float32) * 6
    finished = rng.random((G, B)) < 0.2
    x = [rng.standard_normal((G * B, V)).astype(np.float32) * 3 for _ in range(3)]
    kept = torch.from_numpy(scores).to(cuda)
    f = torch.from_numpy(finished).to(cuda)
    out = (kept, torch.empty(G, B, dtype=torch.int32, device=cuda), torch.empty(G, B, dtype=torch.int64, device=cuda))
    for step in x:
        before = kept.cpu().numpy()
        got = beam.select(torch.from_numpy(step).to(cuda), kept, B, finished=f, out=out)
        torch.cuda.synchronize()
        assert got[0] is kept
        check(tuple(t.cpu().numpy() for t in got), select64(step, before, B, finished))


def test_no_requests(cuda):
    from ssengine_b200 import beam

    s, p, v = beam.select(torch.empty(0, 100, device=cuda), torch.empty(0, 4, device=cuda), 4)
    assert s.shape == (0, 4) and p.shape == (0, 4) and v.shape == (0, 4)


def test_rows_past_two_to_the_31_values(cuda):
    """The last rows of a batch of more than 2^31 logits."""
    G, B, V, k = 57, 256 // 4, 600_011, 4
    x = torch.zeros(G * B, V, dtype=torch.bfloat16, device=cuda)
    rng = np.random.default_rng(8)
    hot = {}
    for g in range(G):
        for i, v in enumerate(rng.permutation(V)[:k]):
            b = int(rng.integers(0, B))
            x[g * B + b, int(v)] = 60.0 - i
            hot.setdefault(g, []).append((b, int(v)))
    from ssengine_b200 import beam

    s, p, t = beam.select(x, torch.zeros(G, B, device=cuda), k)
    torch.cuda.synchronize()
    for g in range(G):
        got = set(zip(p[g].tolist(), t[g].tolist()))
        assert got <= set(hot[g]) | {(b, 0) for b in range(B)} and (p[g, 0].item(), t[g, 0].item()) in hot[g]
