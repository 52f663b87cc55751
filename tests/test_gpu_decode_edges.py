"""Calls of the decode-step operators at the edges of what they take, against float64 restatements with the bars of
tests/test_gpu_decode.py."""

import numpy as np
import pytest
import torch

from oracle import mla as omla
from test_gpu_decode import BMM1, TOL, Cache, attention64, call, check, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths", [True, False])
@pytest.mark.parametrize("form", ["n_idx", "empty", "slice"])
def test_a_selection_without_columns(cuda, form, lengths):
    """No column listed is no token seen: zeros and lse -inf, however the empty selection is written."""
    from ssengine_b200 import mla

    rng = np.random.default_rng(61)
    lens = [300, 1, 90]
    cache = Cache(rng, lens)
    q, _ = queries(rng, 3, 8, "bf16")
    full = torch.zeros(3, 40, dtype=torch.int32, device=cuda)
    idx, n = {"n_idx": (full, 0), "empty": (torch.empty(3, 0, dtype=torch.int32, device=cuda), None),
              "slice": (full[:, :0], None)}[form]
    out = torch.full((3, 8, 512), float("nan"), dtype=torch.bfloat16, device=cuda)
    lse = torch.zeros(3, 8, device=cuda)
    seq = torch.tensor(lens, dtype=torch.int32, device=cuda) if lengths else None
    mla.decode_selected(q.to(cuda), torch.from_numpy(cache.bytes).to(cuda), idx,
                        torch.from_numpy(cache.table).to(cuda), BMM1, out, n_idx=n, seq_lens=seq, lse=lse)
    torch.cuda.synchronize()
    assert not out.any() and bool((lse == float("-inf")).all())


def test_query_values_far_below_their_heads_largest(cuda):
    """One value of 2^7 a head that meets keys of 0, all others 2^-8 .. 2^-7 (2^-15 of it): the scores are theirs alone.
    The two parts of such a value are off by at most 2^-14 (2^-21 of the largest), 2^-14 / sqrt(3) on average; over 575
    keys of variance 1 that is 24 x 3.5e-5 a score. bmm1 makes the scores' spread 1, so that a score is off by
    24 x 3.5e-5 / (24 x 0.0059) = 0.6 %; the bar is twice that beside the usual one."""
    rng = np.random.default_rng(67)
    n, H = 900, 64
    cache = Cache(rng, [n])
    kv = omla.e4m3_decode(omla.quantize(rng.standard_normal((n, 576)).astype(np.float32), 1.0))
    kv[:, 0] = 0.0
    cache.bytes[cache.slots(0, np.arange(n))] = omla.quantize(kv.astype(np.float32), 1.0)
    q = rng.uniform(2.0 ** -8, 2.0 ** -7, (1, H, 576)) * rng.choice([-1.0, 1.0], (1, H, 576))
    q[:, :, 0] = 128.0
    q = torch.from_numpy(q.astype(np.float32)).to(torch.bfloat16)
    q64 = q.double().numpy()
    spread = 24.0 * np.sqrt((q64[0, :, 1:] ** 2).mean())
    out, _, _ = call(cuda, q, cache, seq_lens=np.array([n], np.int32), bmm1=1.0 / spread)
    want, _ = attention64(q64[0], kv, 1.0 / spread, 1.0)
    tol = TOL + 2 * 24.0 * 2.0 ** -14 / np.sqrt(3.0) / spread
    for h in range(H):
        err = np.linalg.norm(out[0, h] - want[h]) / np.linalg.norm(want[h])
        assert err < tol, (h, err, tol)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_one_row_or_one_head_with_any_stride(cuda, kind):
    """A single row has no row stride and a single head no head stride: whatever the tensor states there is not used."""
    rng = np.random.default_rng(71)
    cache = Cache(rng, [333, 100])
    q, q64 = queries(rng, 2, 3, kind)
    q = q.to(cuda)
    for rows, heads in (([0], [0, 1, 2]), ([0, 1], [1]), ([1], [2])):
        part = q[rows][:, heads].contiguous()
        st = list(part.stride())
        if len(rows) == 1:
            st[0] = 7
        if len(heads) == 1:
            st[1] = 1
        lens = [cache.lens[r] for r in rows]
        out, lse, status = call(cuda, part.as_strided(part.shape, st), cache, seq_lens=np.array(lens, np.int32),
                                reqs=np.array(rows, np.int32))
        assert status == 0
        for i, r in enumerate(rows):
            check(out[i], lse[i], *attention64(q64[r][heads], cache.kv[r], BMM1, 1.0))


def test_one_selected_row_with_any_pitch(cuda):
    rng = np.random.default_rng(72)
    cache = Cache(rng, [500])
    q, q64 = queries(rng, 1, 64, "bf16")
    idx = np.sort(rng.choice(500, 100, replace=False)).astype(np.int32)
    from ssengine_b200 import mla

    out = torch.empty(1, 64, 512, dtype=torch.bfloat16, device=cuda)
    mla.decode_selected(q.to(cuda), torch.from_numpy(cache.bytes).to(cuda),
                        torch.from_numpy(idx).to(cuda).as_strided((1, 100), (1, 1)),
                        torch.from_numpy(cache.table).to(cuda), BMM1, out)
    torch.cuda.synchronize()
    check(out[0].double().cpu().numpy(), None, *attention64(q64[0], cache.kv[0][idx], BMM1, 1.0))


def test_kda_one_row_with_any_stride(cuda):
    """A single row of projections, gates, betas and outputs has no pitch."""
    from ssengine_b200.kda import seq_table
    from test_gpu_decode import kda_check, kda_dev, kda_make, recurrence64

    rng = np.random.default_rng(73)
    H = 2
    d = kda_make(rng, 1, H, 3)
    want = recurrence64(d, [(0, 1, 2, 1)], H)
    L, dev = kda_dev(cuda, d)
    one = lambda t: t.as_strided(t.shape, (1, 1))
    out = torch.zeros(1, H * 128, dtype=torch.bfloat16, device=cuda)
    L.decode(one(dev["x"]), one(dev["g"]), one(dev["beta"]), one(out), seq_table([(0, 1, 2, 1)], cuda), dev["cst"],
             dev["rst"])
    torch.cuda.synchronize()
    kda_check(out.double().cpu().numpy(), dev["cst"].double().cpu().numpy(), dev["rst"].double().cpu().numpy(), want,
              [(0, 1, 2, 1)])


def test_no_rows(cuda):
    """A step without rows (empty tensors have no address) writes nothing and is no error."""
    from ssengine_b200 import mla
    from ssengine_b200.kda import KdaLayer

    cache = torch.zeros(256, 576, dtype=torch.uint8, device=cuda)
    i32 = dict(dtype=torch.int32, device=cuda)
    bf = dict(dtype=torch.bfloat16, device=cuda)
    for R in (0, 2):
        table = torch.zeros(R, 2, **i32)
        q, out = torch.empty(0, 64, 576, **bf), torch.empty(0, 64, 512, **bf)
        assert mla.decode(q, cache, table, torch.empty(0, **i32), BMM1, out) is out
        assert mla.decode_selected(q, cache, torch.empty(0, 2051, **i32), table, BMM1, out) is out
    H = 2
    P = H * 128
    L = KdaLayer(torch.zeros(3 * P, 4, **bf), torch.zeros(H, device=cuda), torch.zeros(P, device=cuda))
    conv, rec = torch.ones(3, 3, 3 * P, **bf), torch.ones(3, H, 128, 128, device=cuda)
    for seqs in (torch.empty(0, 4, **i32), torch.tensor([[0, 0, 1, 1]], **i32)):
        status = torch.zeros(1, **i32)
        out = torch.empty(0, P, **bf)
        assert L.decode(torch.empty(0, 3 * P, **bf), torch.empty(0, P, **bf), torch.empty(0, H, **bf), out, seqs, conv,
                        rec, status=status) is out
        torch.cuda.synchronize()
        assert int(status[0]) == 0 and bool((conv == 1).all()) and bool((rec == 1).all())


def test_lengths_around_a_unit_of_64_tokens(cuda):
    rng = np.random.default_rng(79)
    lens = [63, 64, 65, 191, 192, 193, 0, 255, 256, 320, 321]
    cache = Cache(rng, lens)
    for kind in ("bf16", "e4m3"):
        q, q64 = queries(rng, len(lens), 64, kind)
        out, lse, status = call(cuda, q, cache, seq_lens=np.array(lens, np.int32))
        assert status == 0
        for t in range(len(lens)):
            check(out[t], lse[t], *attention64(q64[t], cache.kv[t], BMM1, 1.0))


def test_graphs_outlive_larger_calls_on_their_stream(cuda):
    """Graphs of growing sizes captured on one stream with the default workspace, larger calls on that stream after them,
    and the memory that these gave back in other hands: every graph still gives its own results, and touches nothing."""
    from ssengine_b200 import mla

    rng = np.random.default_rng(83)
    lens = [int(n) for n in rng.integers(1, 900, 80)]
    cache = Cache(rng, lens)
    kv, tb = torch.from_numpy(cache.bytes).to(cuda), torch.from_numpy(cache.table).to(cuda)
    q, q64 = queries(rng, 80, 80, "bf16")
    q, seq = q.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)
    side = torch.cuda.Stream()
    graphs = []
    for T, H in ((1, 64), (4, 64), (40, 64), (20, 80)):
        out = torch.empty(T, H, 512, dtype=torch.bfloat16, device=cuda)
        args = (q[:T, :H], kv, tb, seq[:T], BMM1, out)
        with torch.cuda.stream(side):
            mla.decode(*args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            mla.decode(*args)
        graphs.append((graph, out, T, H))
    big = torch.empty(80, 80, 512, dtype=torch.bfloat16, device=cuda)
    with torch.cuda.stream(side):
        mla.decode(q, kv, tb, seq, BMM1, big)
    torch.cuda.synchronize()
    others = [torch.full((1 << 20,), 3.0, device=cuda) for _ in range(64)]
    for graph, out, T, H in graphs:
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.double().cpu().numpy()
        for t in range(T):
            check(got[t], None, *attention64(q64[t, :H], cache.kv[t], BMM1, 1.0))
    assert all(bool((o == 3.0).all()) for o in others)


@pytest.mark.parametrize("what", ["a_log", "dt_bias", "status", "conv_state", "seqs"])
def test_kda_refuses_host_tensors(cuda, what):
    """A tensor left on the host is refused before the launch."""
    from test_gpu_decode import kda_dev, kda_make

    rng = np.random.default_rng(89)
    H = 2
    L, dev = kda_dev(cuda, kda_make(rng, 1, H, 2))
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    a = dict(a_log=L.a_log, dt_bias=L.dt_bias, status=status, conv_state=dev["cst"],
             seqs=torch.tensor([[0, 1, 1, 1]], dtype=torch.int32, device=cuda))
    a[what] = a[what].cpu()
    L.a_log, L.dt_bias = a["a_log"], a["dt_bias"]
    out = torch.full((1, H * 128), 7.0, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError):
        L.decode(dev["x"], dev["g"], dev["beta"], out, a["seqs"], a["conv_state"], dev["rst"], status=a["status"])
    torch.cuda.synchronize()
    assert bool((out == 7.0).all())


def test_attention_refuses_a_host_status(cuda):
    from ssengine_b200 import mla

    i32 = dict(dtype=torch.int32, device=cuda)
    out = torch.full((1, 4, 512), 7.0, dtype=torch.bfloat16, device=cuda)
    for status in (torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.uint8, device=cuda),
                   torch.zeros(0, **i32)):
        with pytest.raises(ValueError):
            mla.decode(torch.zeros(1, 4, 576, dtype=torch.bfloat16, device=cuda),
                       torch.zeros(256, 576, dtype=torch.uint8, device=cuda), torch.zeros(1, 2, **i32),
                       torch.ones(1, **i32), BMM1, out, status=status)
    torch.cuda.synchronize()
    assert bool((out == 7.0).all())


@pytest.mark.parametrize("attention", ["selected", "dense"])
def test_a_stages_step_uses_what_its_build_reserved(cuda, monkeypatch, attention):
    """Neither the first step nor one of a full microbatch's rows asks for a workspace of its own, and none maps memory."""
    from ssengine_b200 import lib
    from ssengine_b200.messages import Chunk, Plan
    from ssengine_b200.stage import StageConfig, StageModel

    rows = 128
    st = StageModel(StageConfig(layer_split=(4,), hidden=512, inter=256, experts=16, top_k=4, vocab=1000, num_blocks=14,
                                mb_tokens=rows, seed=6, layer_kind="hybrid", kda_heads=2, q_lora=256, mla_nope=64), 0,
                    cuda)
    a, b = ([67, 68], [2, 3, 4, 5, 6, 7]), ([69], [8, 9, 10, 11, 12, 13])
    rng = np.random.default_rng(3)
    tok = lambda n: rng.integers(0, 1000, n).tolist()
    st.forward(Plan(0, [Chunk("a", 0, 100, *a, True, tok(100)), Chunk("b", 0, 20, *b, True, tok(20))]))

    def none(*_):
        raise AssertionError("a step asked for a workspace")

    monkeypatch.setattr(lib, "stream_scratch", none)
    torch.cuda.synchronize()
    mapped = torch.cuda.memory_reserved(cuda)
    st.decode(Plan(1, [Chunk("a", 100, 1, *a, True, tok(1)), Chunk("b", 20, 1, *b, True, tok(1))]), attention=attention)
    st.decode(Plan(2, [Chunk("a", 101, rows - 50, *a, True, tok(rows - 50)), Chunk("b", 21, 50, *b, True, tok(50))]),
              attention=attention)
    torch.cuda.synchronize()
    assert int(st.status[0]) == 0 and torch.cuda.memory_reserved(cuda) == mapped
    assert torch.isfinite(st.last_logits).all()
