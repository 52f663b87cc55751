"""GPU parity of the decode-step operators: `mla.decode` / `mla.decode_selected` (`ssb_mla_decode`) and
`KdaLayer.decode` (`ssb_kda_decode`), against float64 restatements.

Tolerances, derived before the first run:
- attention rows (one head's 512 values): the bf16 output rounds each value by at most 2^-9 of it (2^-9 / sqrt(3) of
  the norm = 1.1e-3), and the softmax weights may enter the second product with 8 significant bits (at most 2^-8 of each
  weight; for weights and values without a common direction 2^-8 / sqrt(3) = 2.3e-3 of the norm): together 2.6e-3, the
  bar at twice that, 5e-3 relative L2; log-sum-exp: 576 fp32 additions of terms whose magnitudes sum to about 30 after
  the scale: at most 576 x 2^-24 x 30 = 1e-3, the bar 2e-3 absolute (scaled with the scores where they are larger);
- recurrence: everything fp32 up to the bf16 output: per output at most 2^-8 of it (one bf16 step) plus 1e-4 of the
  row's largest (cancelling fp32 sums of 128 terms); states per token a few 2^-22: 1e-5 relative L2; conv rows exact."""

import numpy as np
import pytest
import torch

from oracle import kda as ok
from oracle import mla as omla
from oracle.mhc import bf16

pytestmark = pytest.mark.gpu

D = 128
TOL = 5e-3
TOL_LSE = 2e-3
BMM1 = 256 ** -0.5
NAN8 = 0x7F


def attention64(q, kv, bmm1, bmm2):
    """q [H, 576], kv [n, 576] float64 -> (out [H, 512], lse [H])."""
    if kv.shape[0] == 0:
        return np.zeros((q.shape[0], 512)), np.full(q.shape[0], -np.inf)
    s = (q @ kv.T) * bmm1
    m = s.max(axis=1, keepdims=True)
    p = np.exp(s - m)
    z = p.sum(axis=1, keepdims=True)
    return bmm2 * (p / z) @ kv[:, :512], (m + np.log(z))[:, 0]


class Cache:
    """Requests of given lengths over shuffled pages; every byte outside the visible tokens is an e4m3 NaN."""

    def __init__(self, rng, lens, pad_width=0, scale=1.0):
        self.lens = lens
        pages = [-(-n // 128) for n in lens]
        total = sum(pages) + 3
        perm = rng.permutation(total).astype(np.int32)
        self.table = np.full((len(lens), max(pages + [1]) + pad_width), -1, np.int32)
        self.bytes = np.full((total * 128, 576), NAN8, np.uint8)
        self.kv = []
        at = 0
        for r, n in enumerate(lens):
            self.table[r, :pages[r]] = perm[at:at + pages[r]]
            at += pages[r]
            rows = omla.quantize(rng.standard_normal((n, 576)).astype(np.float32) * scale, 1.0)
            if n:
                self.bytes[self.slots(r, np.arange(n))] = rows
            self.kv.append(omla.e4m3_decode(rows))

    def slots(self, r, pos):
        return self.table[r, pos // 128].astype(np.int64) * 128 + pos % 128


def queries(rng, T, H, kind, scale=1.5):
    q = rng.standard_normal((T, H, 576)).astype(np.float32) * scale
    if kind == "e4m3":
        b = omla.quantize(q, 1.0)
        return torch.from_numpy(b), omla.e4m3_decode(b)
    t = torch.from_numpy(q).to(torch.bfloat16)
    return t, t.double().numpy()


def call(cuda, q, cache, seq_lens=None, indices=None, reqs=None, lse=True, table=None, bmm1=BMM1, bmm2=1.0, **kw):
    from ssengine_b200 import mla

    dev = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    q = q.to(cuda) if not q.is_cuda else q
    T, H = q.shape[:2]
    out = torch.full((T, H, 512), float("nan"), dtype=torch.bfloat16, device=cuda)
    ls = torch.full((T, H), float("nan"), device=cuda) if lse else None
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    kv, tb = dev(cache.bytes), dev(cache.table if table is None else table)
    common = dict(bmm2=bmm2, reqs=dev(reqs), lse=ls, status=status, **kw)
    if indices is None:
        mla.decode(q, kv, tb, dev(seq_lens), bmm1, out, **common)
    else:
        mla.decode_selected(q, kv, dev(indices), tb, bmm1, out, seq_lens=dev(seq_lens), **common)
    torch.cuda.synchronize()
    return out.double().cpu().numpy(), None if ls is None else ls.double().cpu().numpy(), int(status.item())


def check(out, lse, want_out, want_lse, tol_lse=TOL_LSE):
    for h in range(out.shape[0]):
        n = np.linalg.norm(want_out[h])
        if n == 0:
            assert not out[h].any()
            assert lse is None or lse[h] == -np.inf
            continue
        err = np.linalg.norm(out[h] - want_out[h]) / n
        assert err < TOL, (h, err)
        if lse is not None:
            assert abs(lse[h] - want_lse[h]) < tol_lse, (h, lse[h], want_lse[h])


LENS = [1, 0, 127, 128, 129, 31, 1000, 2, 257, 640]


@pytest.mark.parametrize("heads", [1, 16, 63, 64, 65, 128])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_dense_rows(cuda, heads, kind):
    """Lengths around the unit of 128, an empty row, one token; every head count class; NaN past each length."""
    rng = np.random.default_rng(heads)
    cache = Cache(rng, LENS, pad_width=2)
    q, q64 = queries(rng, len(LENS), heads, kind)
    out, lse, status = call(cuda, q, cache, seq_lens=np.array(LENS, np.int32), bmm2=0.5)
    assert status == 0
    for t in range(len(LENS)):
        check(out[t], lse[t], *attention64(q64[t], cache.kv[t], BMM1, 0.5))


@pytest.mark.parametrize("n", [1, 2, 33, 128, 300, 9000, 70001])
def test_one_row_is_split_and_joined(cuda, n):
    rng = np.random.default_rng(n)
    cache = Cache(rng, [n])
    q, q64 = queries(rng, 1, 64, "bf16")
    out, lse, status = call(cuda, q, cache, seq_lens=np.array([n], np.int32))
    assert status == 0
    check(out[0], lse[0], *attention64(q64[0], cache.kv[0], BMM1, 1.0))


def test_many_rows_share_ranges(cuda):
    """More rows than SMs, most of them shorter than a range: whole rows inside a range, cut rows at its ends."""
    rng = np.random.default_rng(7)
    lens = [int(x) for x in rng.integers(0, 700, 333)]
    lens[5], lens[200] = 3000, 0
    cache = Cache(rng, lens)
    q, q64 = queries(rng, len(lens), 8, "bf16")
    out, lse, status = call(cuda, q, cache, seq_lens=np.array(lens, np.int32))
    assert status == 0
    for t in range(len(lens)):
        check(out[t], lse[t], *attention64(q64[t], cache.kv[t], BMM1, 1.0))


def test_draft_rows_and_request_map(cuda):
    """Rows mapped to requests out of order, several per request with causal lengths; lengths past the table and
    requests outside it."""
    rng = np.random.default_rng(3)
    lens = [700, 45, 260]
    cache = Cache(rng, lens)
    rows = [(2, 257), (2, 258), (2, 259), (2, 260), (0, 699), (0, 700), (1, 1), (1, 44), (0, 0), (2, -5), (7, 10),
            (-1, 10)]
    reqs, seq = np.array([r for r, _ in rows], np.int32), np.array([n for _, n in rows], np.int32)
    q, q64 = queries(rng, len(rows), 64, "bf16")
    out, lse, status = call(cuda, q, cache, seq_lens=seq, reqs=reqs)
    assert status == 1                                    # two rows name a request outside the table
    for t, (r, n) in enumerate(rows):
        kv = cache.kv[r][:max(n, 0)] if 0 <= r < 3 else np.zeros((0, 576))
        check(out[t], lse[t], *attention64(q64[t], kv, BMM1, 1.0))


def test_missing_pages_and_long_lengths(cuda):
    """Tokens on a negative page, past the table's width or past the cache are left out."""
    rng = np.random.default_rng(5)
    cache = Cache(rng, [1000, 500])
    table = cache.table.copy()
    table[0, 2] = -1
    table[0, 4] = cache.bytes.shape[0] // 128 + 9         # outside the cache
    q, q64 = queries(rng, 2, 64, "bf16")
    # row 0 claims more tokens than its table holds pages for; its last page is whole for the claim's sake
    last = table[0, 7]
    cache.bytes[last * 128:(last + 1) * 128] = omla.quantize(rng.standard_normal((128, 576)).astype(np.float32), 1.0)
    out, lse, status = call(cuda, q, cache, seq_lens=np.array([5000, 0], np.int32), table=table)
    assert status == 0
    pos = np.array([p for p in range(1024) if p // 128 not in (2, 4)])
    kv = omla.e4m3_decode(cache.bytes[table[0, pos // 128].astype(np.int64) * 128 + pos % 128])
    check(out[0], lse[0], *attention64(q64[0], kv, BMM1, 1.0))
    check(out[1], lse[1], *attention64(q64[1], np.zeros((0, 576)), BMM1, 1.0))


def selection(rng, length, pools=512):
    idx = np.full(4 * pools + 3, -1, np.int32)
    whole = length // 4
    n = min(pools, whole)
    ids = np.sort(rng.choice(whole, n, replace=False)) if n else np.zeros(0, int)
    idx[:4 * n] = (ids[:, None] * 4 + np.arange(4)).ravel()
    idx[4 * pools:4 * pools + length - 4 * whole] = np.arange(4 * whole, length)
    return idx


@pytest.mark.parametrize("kind,heads", [("bf16", 64), ("e4m3", 64), ("bf16", 5), ("e4m3", 128)])
def test_selected_rows(cuda, kind, heads):
    """The indexer's expanded layout: short rows leave most columns empty, long ones fill 2,051; an empty row; rows
    whose selection reaches past the visible length."""
    rng = np.random.default_rng(heads + 1)
    lens = [1, 3, 4, 77, 2050, 9001, 600, 0]
    cache = Cache(rng, lens)
    idx = np.stack([selection(rng, n) for n in lens])
    seq = np.array(lens, np.int32)
    seq[5], seq[6] = 4000, 599                            # some selected tokens are no longer visible
    q, q64 = queries(rng, len(lens), heads, kind)
    out, lse, status = call(cuda, q, cache, seq_lens=seq, indices=idx)
    assert status == 0
    for t in range(len(lens)):
        pos = idx[t][(idx[t] >= 0) & (idx[t] < seq[t])]
        check(out[t], lse[t], *attention64(q64[t], cache.kv[t][pos], BMM1, 1.0))


def test_selected_without_lengths_duplicates_and_width(cuda):
    """No seq_lens; positions listed twice count twice; a column count that is no multiple of anything and a row pitch
    wider than it; rows of one page table row."""
    rng = np.random.default_rng(9)
    cache = Cache(rng, [900, 300])
    T, n = 5, 333
    idx = np.full((T, n + 20), 5, np.int32)               # columns past n_idx are not read
    for t in range(T):
        r = t % 2
        idx[t, :n] = rng.integers(0, cache.lens[r], n)
        idx[t, rng.permutation(n)[:40 * t]] = -1
    idx[4, :n] = -1
    q, q64 = queries(rng, T, 64, "bf16")
    out, lse, status = call(cuda, q, cache, indices=idx, reqs=np.array([0, 1, 0, 1, 0], np.int32), n_idx=n)
    assert status == 0
    for t in range(T):
        pos = idx[t, :n][idx[t, :n] >= 0]
        check(out[t], lse[t], *attention64(q64[t], cache.kv[t % 2][pos], BMM1, 1.0))


def test_dense_equals_selected(cuda):
    """All positions listed, in another order, = dense, within the tolerance."""
    rng = np.random.default_rng(21)
    lens = [1500, 2303]
    cache = Cache(rng, lens)
    q, q64 = queries(rng, 2, 64, "e4m3")
    idx = np.full((2, 2304), -1, np.int32)
    for t, n in enumerate(lens):
        idx[t, rng.permutation(2304)[:n]] = np.arange(n)
    a, _, _ = call(cuda, q, cache, seq_lens=np.array(lens, np.int32))
    b, _, _ = call(cuda, q, cache, indices=idx)
    for t in range(2):
        for h in range(64):
            assert np.linalg.norm(a[t, h] - b[t, h]) < TOL * np.linalg.norm(a[t, h])


@pytest.mark.parametrize("gain", [1e-3, 30.0, 3000.0])
def test_extreme_scores(cuda, gain):
    """Scores from almost equal to thousands apart (one token takes everything), of either sign, in every order."""
    rng = np.random.default_rng(int(gain * 10))
    lens = [1300, 128, 400]
    cache = Cache(rng, lens)
    q, q64 = queries(rng, 3, 64, "bf16", scale=1.0)
    out, lse, _ = call(cuda, q, cache, seq_lens=np.array(lens, np.int32), bmm1=BMM1 * gain)
    for t in range(3):
        # an error of a few 2^-24 of |q||k| in a score is a relative error of a weight times the gain: near-ties of the
        # two largest weights move with it
        tol = TOL + 4 * gain * BMM1 * 24 * 24 * 2.0 ** -22
        want, wl = attention64(q64[t], cache.kv[t], BMM1 * gain, 1.0)
        for h in range(64):
            assert np.linalg.norm(out[t, h] - want[h]) < tol * np.linalg.norm(want[h]), (t, h)
        assert np.abs(lse[t] - wl).max() < TOL_LSE * max(1.0, gain)


def test_a_sink_token_and_a_long_flat_tail(cuda):
    """One token whose weight is 2^17 times each of 60,000 others: together they hold a third of the mass, so weights
    far below the largest must not be lost."""
    rng = np.random.default_rng(2)
    n = 60000
    cache = Cache(rng, [n])
    kv = cache.kv[0].copy()
    kv[:, 512:] = 0.0
    kv[1:, 512:] = 0.0
    kv[0, 512:] = 1.0
    q = np.zeros((1, 64, 576), np.float32)
    q[0, :, 512:] = 17 * np.log(2.0) / BMM1 / 64
    kv[:, 0:512] += 1.0                                   # a common direction: a lost tail would show
    b = omla.quantize(kv.astype(np.float32), 1.0)
    cache.bytes[cache.slots(0, np.arange(n))] = b
    t = torch.from_numpy(q).to(torch.bfloat16)
    for pos in (0, 31234, n - 1):                         # the sink first, in the middle, last
        order = np.arange(n)
        order[[0, pos]] = order[[pos, 0]]
        cache.bytes[cache.slots(0, np.arange(n))] = b[order]
        out, lse, _ = call(cuda, t, cache, seq_lens=np.array([n], np.int32))
        check(out[0], lse[0], *attention64(t[0].double().numpy(), omla.e4m3_decode(b), BMM1, 1.0))


def test_a_jump_of_hundreds_in_the_running_maximum(cuda):
    """Scores that rise by hundreds (base 2) from one part of a row to the next, and fall again: the accumulated sums
    have to follow whichever part holds the maximum."""
    rng = np.random.default_rng(4)
    n = 128 * 300
    cache = Cache(rng, [n])
    kv = omla.e4m3_decode(omla.quantize(rng.standard_normal((n, 576)).astype(np.float32), 1.0))
    step = (np.arange(n) // 1000).astype(np.float64)
    level = np.where(step < 20, step, 40 - step) * 1.0    # up to 20 and down again
    kv[:, 512:] = 0.0
    kv[:, 512] = omla.e4m3_decode(omla.quantize(level.astype(np.float32), 1.0))
    cache.bytes[cache.slots(0, np.arange(n))] = omla.quantize(kv.astype(np.float32), 1.0)
    q = np.zeros((1, 64, 576), np.float32)
    q[0, :, 512] = 400.0                                  # 25 a level (36 in base 2), up to 500
    t = torch.from_numpy(q).to(torch.bfloat16)
    for sign in (1.0, -1.0):
        out, lse, _ = call(cuda, t * sign, cache, seq_lens=np.array([n], np.int32))
        check(out[0], lse[0], *attention64((t * sign)[0].double().numpy(), kv, BMM1, 1.0), tol_lse=0.05)


def test_infinite_and_nan_scores(cuda):
    """A visible NaN latent or a NaN query makes its own row NaN, and no other row or head."""
    rng = np.random.default_rng(6)
    cache = Cache(rng, [300, 300, 300])
    q, q64 = queries(rng, 3, 64, "bf16")
    q[1, 7, 3] = float("nan")
    cache.bytes[cache.slots(2, np.array([200]))[0], 30] = NAN8
    out, lse, _ = call(cuda, q, cache, seq_lens=np.array([300, 300, 250], np.int32))
    check(out[0], lse[0], *attention64(q64[0], cache.kv[0], BMM1, 1.0))
    keep = [h for h in range(64) if h != 7]
    want, wl = attention64(q64[1], cache.kv[1], BMM1, 1.0)
    check(out[1][keep], lse[1][keep], want[keep], wl[keep])
    assert np.isnan(out[1, 7]).all()
    assert np.isnan(out[2]).any(axis=1).all()


def test_strided_queries_offsets_streams_and_repeats(cuda):
    """Query rows cut from wider rows, another stream, a caller's workspace full of NaN, the same bits every time."""
    from ssengine_b200 import mla

    rng = np.random.default_rng(8)
    lens = [5000, 130, 2222]
    cache = Cache(rng, lens)
    wide = torch.from_numpy(rng.standard_normal((3, 20, 600)).astype(np.float32)).to(torch.bfloat16).to(cuda)
    q = wide[:, 2:18, 8:584]
    seq = torch.tensor(lens, dtype=torch.int32, device=cuda)
    kv, tb = torch.from_numpy(cache.bytes).to(cuda), torch.from_numpy(cache.table).to(cuda)
    ws = torch.full((mla.decode_workspace_bytes(3, 16),), 0xFF, dtype=torch.uint8, device=cuda)
    outs = []
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(3):
        out = torch.empty(3, 16, 512, dtype=torch.bfloat16, device=cuda)
        torch.cuda.synchronize()
        mla.decode(q, kv, tb, seq, BMM1, out, workspace=ws if i else None, stream=side if i == 2 else None)
        torch.cuda.synchronize()
        outs.append(out.view(torch.int16).cpu().numpy())
    assert (outs[0] == outs[1]).all() and (outs[0] == outs[2]).all()
    got = torch.from_numpy(outs[0]).view(torch.bfloat16).double().numpy()
    for t in range(3):
        check(got[t], None, *attention64(q[t].double().cpu().numpy(), cache.kv[t], BMM1, 1.0))


def test_captured_call_follows_the_lengths(cuda):
    """A graph captured once, replayed as the rows grow by a token a step."""
    from ssengine_b200 import mla

    rng = np.random.default_rng(12)
    cache = Cache(rng, [400, 900])
    kv, tb = torch.from_numpy(cache.bytes).to(cuda), torch.from_numpy(cache.table).to(cuda)
    q, q64 = queries(rng, 2, 64, "bf16")
    q = q.to(cuda)
    seq = torch.tensor([120, 700], dtype=torch.int32, device=cuda)
    out = torch.empty(2, 64, 512, dtype=torch.bfloat16, device=cuda)
    ws = torch.empty(mla.decode_workspace_bytes(2, 64), dtype=torch.uint8, device=cuda)
    mla.decode(q, kv, tb, seq, BMM1, out, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        mla.decode(q, kv, tb, seq, BMM1, out, workspace=ws)
    for lens in ([127, 800], [128, 0], [129, 900], [400, 5]):
        seq.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        got = out.double().cpu().numpy()
        for t in range(2):
            check(got[t], None, *attention64(q64[t], cache.kv[t][:lens[t]], BMM1, 1.0))


def test_pages_past_two_to_the_31_bytes(cuda):
    rng = np.random.default_rng(13)
    rows = 31000 * 128                                    # 2.3 GB of cache
    kv = torch.zeros(rows, 576, dtype=torch.uint8, device=cuda)
    part = omla.quantize(rng.standard_normal((300, 576)).astype(np.float32), 1.0)
    pages = np.array([[30999, 0, 30500]], np.int32)
    slots = pages[0, np.arange(300) // 128].astype(np.int64) * 128 + np.arange(300) % 128
    kv[torch.from_numpy(slots).to(cuda)] = torch.from_numpy(part).to(cuda)
    from ssengine_b200 import mla

    q, q64 = queries(rng, 1, 64, "bf16")
    out = torch.empty(1, 64, 512, dtype=torch.bfloat16, device=cuda)
    mla.decode(q.to(cuda), kv, torch.from_numpy(pages).to(cuda), torch.tensor([300], dtype=torch.int32, device=cuda),
               BMM1, out)
    torch.cuda.synchronize()
    check(out[0].double().cpu().numpy(), None, *attention64(q64[0], omla.e4m3_decode(part), BMM1, 1.0))


# ---- KDA ------------------------------------------------------------------------------------------------------------


def kda_make(rng, T, H, blocks, extra=24):
    P = H * D
    return dict(x=bf16(rng.standard_normal((T, 3 * P + extra))), w=bf16(rng.uniform(-0.6, 0.6, (3 * P, 4))),
                g=bf16(rng.standard_normal((T, P))), beta=bf16(rng.standard_normal((T, H))),
                a_log=rng.uniform(-1, 1, H).astype(np.float32), dtb=(rng.standard_normal(P) * 0.5).astype(np.float32),
                cst=bf16(rng.standard_normal((blocks, 3, 3 * P))),
                rst=(rng.standard_normal((blocks, H, D, D)) * 0.1).astype(np.float32))


def recurrence64(d, seqs, H, lower_bound=-5.0):
    """Token by token in float64 with no rounding between the inputs and the output."""
    P = H * D
    x, w = np.asarray(d["x"], np.float64)[:, :3 * P], np.asarray(d["w"], np.float64)
    cst, rst = np.array(d["cst"], np.float64), np.array(d["rst"], np.float64)
    gate = np.exp(ok.gate(d["g"], d["a_log"], d["dtb"], lower_bound, H, D))
    b = 1.0 / (1.0 + np.exp(-np.asarray(d["beta"], np.float64)))
    out = np.full((x.shape[0], P), np.nan)
    for s, e, blk, init in seqs:
        if e == s:
            continue
        hist = cst[blk] if init else np.zeros_like(cst[blk])
        S = rst[blk].copy() if init else np.zeros_like(rst[blk])
        for t in range(s, e):
            hist = np.concatenate([hist, x[t:t + 1]])
            y = ok.silu((w.T * hist[-4:]).sum(axis=0)).reshape(3, H, D)
            q, k = ok.l2norm(y[0]), ok.l2norm(y[1])
            S = S * gate[t][:, None, :]
            u = b[t][:, None] * (y[2] - np.einsum("hvk,hk->hv", S, k))
            S = S + u[:, :, None] * k[:, None, :]
            out[t] = (D ** -0.5 * np.einsum("hvk,hk->hv", S, q)).ravel()
        cst[blk], rst[blk] = hist[-3:], S
    return out, cst, rst


def kda_dev(cuda, d):
    from ssengine_b200.kda import KdaLayer

    bf = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(torch.bfloat16).to(cuda)
    f32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(cuda)
    return (KdaLayer(bf(d["w"]), f32(d["a_log"]), f32(d["dtb"]), -5.0),
            dict(x=bf(d["x"]), g=bf(d["g"]), beta=bf(d["beta"]), cst=bf(d["cst"]), rst=f32(d["rst"])))


def kda_check(out, cst, rst, want, seqs, tol_state=1e-5):
    wo, wc, wr = want
    for s, e, blk, _ in seqs:
        for t in range(s, e):
            bound = 2.0 ** -8 * np.abs(wo[t]) + 1e-4 * np.abs(wo[t]).max()
            assert (np.abs(out[t] - wo[t]) <= bound).all(), (t, float((np.abs(out[t] - wo[t]) / bound).max()))
    assert (cst == wc).all()
    for blk in range(rst.shape[0]):
        assert np.linalg.norm(rst[blk] - wr[blk]) <= tol_state * np.linalg.norm(wr[blk]), blk


def kda_run(cuda, d, seqs, H, **kw):
    from ssengine_b200.kda import seq_table

    L, dev = kda_dev(cuda, d)
    out = torch.full((d["x"].shape[0], H * D), 77.0, dtype=torch.bfloat16, device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    L.decode(dev["x"], dev["g"], dev["beta"], out, seq_table(seqs, cuda), dev["cst"], dev["rst"], status=status, **kw)
    torch.cuda.synchronize()
    return (out.double().cpu().numpy(), dev["cst"].double().cpu().numpy(), dev["rst"].double().cpu().numpy(),
            int(status.item()))


@pytest.mark.parametrize("H", [1, 2, 7])
@pytest.mark.parametrize("seqs", [
    [(0, 1, 3, 1)],
    [(0, 1, 0, 0)],
    [(0, 1, 4, 1), (1, 2, 1, 1), (2, 3, 5, 0), (3, 4, 2, 1)],
    [(0, 2, 4, 1), (2, 3, 1, 0), (3, 3, 0, 1), (5, 13, 5, 1), (13, 17, 2, 0)],     # rows 3, 4 outside, an empty run
])
def test_kda_runs(cuda, H, seqs):
    """Single tokens and runs, fresh and continued, an empty run (its block kept), rows outside every run untouched, a
    fresh run over a block of NaN."""
    rng = np.random.default_rng(H)
    T = max(e for _, e, _, _ in seqs)
    d = kda_make(rng, T, H, 7)
    for _, _, blk, init in seqs:
        if not init:
            d["cst"][blk], d["rst"][blk] = np.nan, np.nan
    want = recurrence64(d, seqs, H)
    out, cst, rst, status = kda_run(cuda, d, seqs, H)
    assert status == 0
    inside = np.zeros(T, bool)
    for s, e, _, _ in seqs:
        inside[s:e] = True
    assert (out[~inside] == 77.0).all()
    kda_check(out, cst, rst, want, seqs)


def test_kda_many_requests_and_heads(cuda):
    """A decode batch: more (request, head) pairs than fit the GPU at once; the state pool's other blocks untouched."""
    rng = np.random.default_rng(31)
    R, H = 70, 16
    d = kda_make(rng, R, H, R + 3)
    blocks = rng.permutation(R + 3)[:R]
    seqs = [(r, r + 1, int(blocks[r]), 1) for r in range(R)]
    out, cst, rst, status = kda_run(cuda, d, seqs, H)
    assert status == 0
    kda_check(out, cst, rst, recurrence64(d, seqs, H), seqs)


def test_kda_decode_continues_a_prefill(cuda):
    """100 tokens by the chunked form, then 3 single steps, against one float64 recurrence over 103 (the chunked form's
    2e-2: its operands are bf16); and the two forms against each other on the same rows."""
    from ssengine_b200.kda import seq_table

    rng = np.random.default_rng(17)
    H, n = 2, 103
    d = kda_make(rng, n, H, 3)
    want = recurrence64(d, [(0, n, 1, 0)], H)
    L, dev = kda_dev(cuda, d)
    out = torch.zeros(n, H * D, dtype=torch.bfloat16, device=cuda)
    L.prefill(dev["x"][:100], dev["g"][:100], dev["beta"][:100], out[:100], seq_table([(0, 100, 1, 0)], cuda),
              dev["cst"], dev["rst"])
    for t in range(100, n):
        L.decode(dev["x"], dev["g"], dev["beta"], out, seq_table([(t, t + 1, 1, 1)], cuda), dev["cst"], dev["rst"])
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    assert np.linalg.norm(got[100:] - want[0][100:]) < 2e-2 * np.linalg.norm(want[0][100:])
    assert (dev["cst"].double().cpu().numpy()[1] == want[1][1]).all()
    r = dev["rst"].double().cpu().numpy()[1]
    assert np.linalg.norm(r - want[2][1]) < 2e-2 * np.linalg.norm(want[2][1])
    # the recurrent form over the same 100 rows
    L2, dev2 = kda_dev(cuda, d)
    out2 = torch.zeros(n, H * D, dtype=torch.bfloat16, device=cuda)
    L2.decode(dev2["x"], dev2["g"], dev2["beta"], out2, seq_table([(0, n, 1, 0)], cuda), dev2["cst"], dev2["rst"])
    torch.cuda.synchronize()
    kda_check(out2.double().cpu().numpy(), dev2["cst"].double().cpu().numpy()[1:2], dev2["rst"].double().cpu().numpy()[1:2],
              (want[0], want[1][1:2], want[2][1:2]), [(0, n, 0, 0)], tol_state=1e-4)


def test_kda_strides_streams_and_state_views(cuda):
    """Column views of one projection, a padded state pool (block strides as when states share latent blocks), another
    stream, extreme gates and inputs (decay to 0 and no decay, SiLU at +-80)."""
    from ssengine_b200.kda import seq_table

    rng = np.random.default_rng(19)
    H, T = 3, 4
    P = H * D
    d = kda_make(rng, T, H, 6)
    d["g"] = bf16(rng.choice([-60.0, 60.0, 0.5], size=(T, P)))
    d["x"][0] *= 80.0
    d["x"] = bf16(d["x"])
    seqs = [(0, 1, 2, 1), (1, 2, 0, 1), (2, 4, 5, 1)]
    want = recurrence64(d, seqs, H)
    L, dev = kda_dev(cuda, d)
    proj = torch.zeros(T, 3 * P + 2 + H + 5, dtype=torch.bfloat16, device=cuda)      # an even, otherwise odd pitch
    proj = torch.nn.functional.pad(proj, (0, proj.shape[1] % 2))
    proj[:, :3 * P] = dev["x"][:, :3 * P]
    proj[:, 3 * P + 1:3 * P + 1 + H] = dev["beta"]
    beta = proj[:, 3 * P + 1:3 * P + 1 + H]
    rec = torch.zeros(6, H * D * D + 64, device=cuda)[:, :H * D * D].view(6, H, D, D)
    rec.copy_(dev["rst"])
    cst = torch.zeros(6, 9 * P + 10, dtype=torch.bfloat16, device=cuda)[:, :9 * P].view(6, 3, 3 * P)
    cst.copy_(dev["cst"])
    out = torch.zeros(T, P + 6, dtype=torch.bfloat16, device=cuda)
    table = seq_table(seqs, cuda)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    L.decode(proj, dev["g"], beta, out, table, cst, rec, stream=side)
    torch.cuda.synchronize()
    assert not out[:, P:].any()
    kda_check(out[:, :P].double().cpu().numpy(), cst.double().cpu().numpy(), rec.double().cpu().numpy(), want, seqs)


def test_kda_refuses_runs_outside_the_rows(cuda):
    rng = np.random.default_rng(23)
    d = kda_make(rng, 3, 2, 4)
    seqs = [(0, 1, 1, 1), (2, 9, 2, 1), (1, 2, -1, 1)]
    out, cst, rst, status = kda_run(cuda, d, seqs, 2)
    assert status == 1
    want = recurrence64(d, seqs[:1], 2)
    assert (out[1:] == 77.0).all()
    kda_check(out, cst, rst, want, seqs[:1])
