"""`StageModel.decode` on the GPU: the decode-step operators together, as a stage runs them.

The stage (the tiny hybrid model: three KDA layers, then a DSA layer) prefills five requests, then takes steps of new
tokens - one a request, drafts of several, a request whose first token this is - through `KdaLayer.decode` and
`mla.decode_selected` / `mla.decode`. Judged teacher-forced: the oracle starts every step from the device's own states
and every layer from the device layer's own inputs. A KDA layer's residual is held within 3e-2 of the oracle's layer and
the logits within 2e-2 of the oracle's head, the bars of the prefill path. The oracle's DSA layer carries the prefill
kernel's rounding of the softmax weights (3 bits), which the decode forms do not have, and its 4-bit projections turn
that difference into one of some percent of the layer's rows; so that layer is judged in its parts: the attention within
5e-3 of each row of the formula in 64 bits over the block's own query and cache (the operator's own errors: weights in 8
bits, 2^-9, and the bf16 output, 2^-9), the output projection within 1e-3 of the oracle's and the boundary's residual
within 3e-2 of the oracle's, each on the device's own input. The contexts stay below 2,048 tokens, where the selection
is the whole context and both attention forms have one formula.

The attention block alone, over contexts above 2,048 tokens (the selection leaves tokens out): the block's attention
against the formula in 64 bits over its own query, cache and selection, within the same 5e-3 of each row."""

import numpy as np
import pytest
import torch

from model_params import row_chunks, stage_params, stage_states
from oracle import dsa as od
from oracle import kda as ok
from oracle import mhc as omhc
from oracle import model as omodel

pytestmark = pytest.mark.gpu


def rel(a, b):
    return float(np.linalg.norm(np.asarray(a, np.float64) - b) / max(np.linalg.norm(b), 1e-30))


def attention_formula(q8, keys, scale):
    """softmax(scale q8 keys^T) keys[:, :512] in 64 bits; q8 [H, 576] and keys [n, 576] as e4m3 bytes."""
    deq = lambda t: t.view(torch.float8_e4m3fn).float().double()
    k = deq(keys)
    return torch.softmax(deq(q8) @ k.t() * scale, dim=1) @ k[:, :512]


def row_rel(got, want):
    return float((got.double() - want).norm() / want.norm())


LENGTHS = {"p0": 306, "p1": 212, "p2": 110, "p3": 9, "p4": 2}              # each request's tokens over the run
PREFILL = [("p0", 0, 300), ("p1", 0, 200), ("p2", 0, 100), ("p3", 0, 5)]
STEPS = [[("p0", 300, 1), ("p1", 200, 1), ("p2", 100, 1), ("p3", 5, 1)],
         [("p0", 301, 4), ("p1", 201, 8), ("p2", 101, 2), ("p3", 6, 3), ("p4", 0, 1)],
         [("p4", 1, 1), ("p1", 209, 1)]]


@pytest.mark.parametrize("attention", ["selected", "dense"])
def test_decode_steps_match_the_oracle(cuda, attention):
    from ssengine_b200 import weights
    from ssengine_b200.messages import Chunk, Plan
    from ssengine_b200.stage import StageConfig, StageModel

    cfg = StageConfig(layer_split=(4,), hidden=256, inter=128, experts=8, top_k=2, vocab=4096, mb_tokens=1024,
                      num_blocks=40, seed=0, layer_kind="hybrid", kda_heads=2, q_lora=256, mla_nope=64,
                      mla_v_dim=256, routing="sigmoid", weight_init="normal", init_std=0.02)
    st = StageModel(cfg, 0, cuda)
    caught = []
    n = lambda t: t.float().cpu().numpy()
    st.layer_hook = lambda layer, res, x_prev, post, comb: caught.append(tuple(n(t) for t in (res, x_prev, post, comb)))
    blk = st.layers[3].attn
    forward = blk.forward
    blk.forward = lambda *a, **kw: outs.append(forward(*a, keep=True, **kw)) or outs[-1]     # its parts and output kept
    outs = []
    params = stage_params(st)
    gs_x, gs_h = weights.GS_X, weights.GS_H
    rng = np.random.default_rng(15)
    prompts = {r: rng.integers(0, cfg.vocab, n) for r, n in LENGTHS.items()}
    res_of = {r: (list(range(67 * (1 + j), 67 * (1 + j) + 4)), [10 + 6 * j + g for g in range(6)])
              for j, r in enumerate(LENGTHS)}

    def plan_of(k, mb):
        return Plan(k, [Chunk(r, start, n, *res_of[r], True, prompts[r][start:start + n].tolist())
                        for r, start, n in mb])

    st.forward(plan_of(0, PREFILL))
    for k, mb in enumerate(STEPS):
        plan = plan_of(k + 1, mb)
        before = stage_states(st)
        caught.clear()
        outs.clear()
        batch = st.prepare(plan)
        tokens = st.run(batch, None, decode=attention)
        torch.cuda.synchronize()
        assert int(st.status.item()) == 0
        assert len(caught) == 4 and tokens.shape == (len(mb),)
        rows, order = row_chunks(plan)
        tok = np.concatenate([np.asarray(c["token_ids"], np.int64) for c in rows])
        inp = (np.repeat(params["embed"][tok][:, None, :], 4, axis=1), None, None, None)
        for li, (L, stt) in enumerate(zip(params["layers"][:3], before)):
            res, _, _, _ = omodel.layer_forward(L, stt, rows, *inp, gs_x, gs_h)
            g = caught[li]
            assert rel(g[0], res) < 3e-2, (k, li, rel(g[0], res))
            inp = g
        kv, table = st.kv.latent(3), batch.dsa["page_table"].long()
        row = 0
        for r, c in enumerate(rows):
            for i in range(c["n"]):
                pos = torch.arange(c["start"] + i + 1, device=cuda)
                want = attention_formula(blk.parts["q8"][row], kv[table[r][pos // 128] * 128 + pos % 128], blk.scale)
                assert row_rel(blk.parts["o_lat"][row], want) < 5e-3, (k, row)
                row += 1
        assert row == outs[0].shape[0]
        L = params["layers"][3]
        x_a = od.bf16(ok.nvfp4_linear(n(blk.parts["o_in"]), *L["attn"]["o_proj"], gs_x))
        assert rel(n(outs[0]), x_a) < 1e-3, (k, rel(n(outs[0]), x_a))
        x_prev, res, post, comb = inp[1], inp[0], inp[2], inp[3]
        res, post, comb, _ = omhc.post_pre(x_prev, res, post, comb, *L["bound_a"])
        res = omhc.post_pre(n(outs[0]), res, post, comb, *L["bound_b"])[0]
        assert rel(caught[3][0], res) < 3e-2, (k, rel(caught[3][0], res))
        res, x_prev, post, comb = caught[-1]
        o_logits, _ = omodel.head(params, rows, omhc.post(x_prev, res, post, comb))
        in_rows = {c: j for j, c in enumerate(order)}
        got = st.last_logits.cpu().numpy()
        want = o_logits[[in_rows[i] for i in range(len(mb))]]
        assert rel(got, want) < 2e-2, (k, rel(got, want))


def test_two_stages_equal_one(cuda):
    """The step across a stage edge (two stages) equals the unsplit stage's, bit for bit."""
    from ssengine_b200.messages import Chunk, Plan
    from ssengine_b200.stage import StageConfig, StageModel

    base = dict(hidden=512, inter=256, experts=16, top_k=4, vocab=1000, num_blocks=14, mb_tokens=256, seed=6,
                layer_kind="hybrid", kda_heads=2, q_lora=256, mla_nope=64)
    whole = StageModel(StageConfig(layer_split=(4,), **base), 0, cuda)
    s0 = StageModel(StageConfig(layer_split=(2, 2), **base), 0, cuda)
    s1 = StageModel(StageConfig(layer_split=(2, 2), **base), 1, cuda)
    rng = np.random.default_rng(10)
    ta, tb = rng.integers(0, 1000, 150).tolist(), rng.integers(0, 1000, 40).tolist()
    a, b = ([67, 68], [2, 3, 4, 5, 6, 7]), ([69], [8, 9, 10, 11, 12, 13])
    first = Plan(0, [Chunk("a", 0, 130, *a, True, ta[:130]), Chunk("b", 0, 30, *b, True, tb[:30])])
    whole.forward(first)
    s1.forward(first, s0.forward(first))
    for k in range(3):
        step = Plan(1 + k, [Chunk("a", 130 + k, 1, *a, True, ta[130 + k:131 + k]),
                            Chunk("b", 30 + 3 * k, 3, *b, True, tb[30 + 3 * k:33 + 3 * k])])
        t_whole = whole.decode(step)
        t_split = s1.decode(step, s0.decode(step))
        torch.cuda.synchronize()
        assert int(whole.status[0]) == 0 and int(s0.status[0]) == 0 and int(s1.status[0]) == 0
        assert torch.equal(t_whole, t_split)
        assert torch.equal(whole.last_logits, s1.last_logits)
        assert torch.isfinite(whole.last_logits).all()


@pytest.mark.parametrize("indexer_fp8", [False, True])
@pytest.mark.parametrize("form", ["selected", "dense"])
def test_attention_block_over_long_contexts(cuda, form, indexer_fp8):
    from ssengine_b200 import indexer
    from ssengine_b200.layers import DsaAttention

    H = 512
    blk = DsaAttention(41, H, cuda, q_lora=256, nope=64, v_dim=256, indexer_fp8=indexer_fp8)
    reqs = [(4999, 1), (2600, 3), (0, 1)]                # (start position, new rows)
    T = sum(n for _, n in reqs)
    lens = [s + n for s, n in reqs]
    width = -(-max(lens) // 128)
    g = torch.Generator(device=cuda)
    g.manual_seed(3)
    perm = torch.randperm(3 * width, generator=g, device=cuda).to(torch.int32)
    table = perm.view(3, width).contiguous()
    qsl = np.cumsum([0] + [n for _, n in reqs]).astype(np.int32)
    positions = np.concatenate([np.arange(s, s + n) for s, n in reqs]).astype(np.int64)
    row_req = np.repeat(np.arange(3), [n for _, n in reqs]).astype(np.int32)
    tab = table.cpu().numpy()
    slots = np.array([tab[r][p // 128] * 128 + p % 128 for r, p in zip(row_req, positions)], np.int64)
    kv_cache = torch.randn(3 * width * 128, 576, generator=g, device=cuda).to(torch.float8_e4m3fn).view(torch.uint8)
    if indexer_fp8:
        codes = torch.randn(3 * width, 32, 128, generator=g, device=cuda).to(torch.float8_e4m3fn).view(torch.uint8)
        scales = torch.ones(3 * width, 1, 32, device=cuda).view(torch.uint8).view(3 * width, 1, 128)
        pool = torch.cat([codes, scales], dim=1).view(-1, 128).contiguous()
    else:
        pool = torch.randn(3 * width * 32, 128, generator=g, device=cuda).to(torch.bfloat16)
    ring = torch.randn(4, 2, 4, 128, generator=g, device=cuda).to(torch.bfloat16)
    y = torch.randn(T, H, generator=g, device=cuda).to(torch.bfloat16)
    kreq = np.array([(qsl[r], n, s, r + 1) for r, (s, n) in enumerate(reqs)], np.int32)
    groups = indexer.work_groups(qsl[:-1], [n for _, n in reqs], [s for s, _ in reqs])
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    d = lambda a, dt: torch.from_numpy(np.ascontiguousarray(a)).to(dt).to(cuda)
    args = (y, d(positions, torch.int64), d(slots, torch.int64), d(qsl, torch.int32), table, d(kreq, torch.int32), 3,
            d(groups, torch.int32))
    pool2, ring2, cache2 = pool.clone(), ring.clone(), kv_cache.clone()
    blk.forward(*args, cache2, pool2, ring2, status, keep=True)              # the prefill form's writes
    tok_prefill = blk.parts["tok"][:, :2051].clone()
    out = blk.forward(*args, kv_cache, pool, ring, status, keep=True,
                      decode=(form, d(row_req, torch.int32), d(positions + 1, torch.int32)))
    torch.cuda.synchronize()
    assert int(status[0]) == 0 and torch.isfinite(out.float()).all()
    assert torch.equal(kv_cache, cache2) and torch.equal(pool, pool2) and torch.equal(ring, ring2)
    if form == "selected":
        assert torch.equal(blk.parts["tok"][:, :2051], tok_prefill)
    for t in range(T):
        if form == "selected":
            pos = tok_prefill[t]
            pos = pos[pos >= 0].long()
            assert pos.numel() == min(positions[t] + 1, 4 * min(512, (positions[t] + 1) // 4) + (positions[t] + 1) % 4)
        else:
            pos = torch.arange(positions[t] + 1, device=cuda)
        want = attention_formula(blk.parts["q8"][t], kv_cache[table[row_req[t]].long()[pos // 128] * 128 + pos % 128],
                                 blk.scale)
        assert row_rel(blk.parts["o_lat"][t], want) < 5e-3, (t, row_rel(blk.parts["o_lat"][t], want))


def test_captured_step(cuda):
    """A captured step of the attention block replays on changed inputs: nothing in it needs the host."""
    from ssengine_b200 import kda, mla

    T, H = 4, 64
    g = torch.Generator(device=cuda)
    g.manual_seed(5)
    cache = torch.randn(T * 4 * 128, 576, generator=g, device=cuda).to(torch.float8_e4m3fn).view(torch.uint8)
    table = torch.arange(T * 4, device=cuda, dtype=torch.int32).view(T, 4)
    q = torch.randn(T, H, 576, generator=g, device=cuda).to(torch.bfloat16)
    lens = torch.tensor([300, 1, 0, 512], dtype=torch.int32, device=cuda)
    out = torch.empty(T, H, 512, dtype=torch.bfloat16, device=cuda)
    P = 2 * 128
    layer = kda.KdaLayer((torch.randn(3 * P, 4, generator=g, device=cuda) * 0.3).to(torch.bfloat16),
                         torch.rand(2, generator=g, device=cuda), torch.randn(P, generator=g, device=cuda))
    seqs = kda.seq_table([(t, t + 1, t, 1) for t in range(T)], cuda)
    proj = torch.randn(T, 3 * P, generator=g, device=cuda).to(torch.bfloat16)
    gate, beta = proj[:, :P].contiguous(), proj[:, :2].contiguous()
    conv = torch.zeros(T, 3, 3 * P, dtype=torch.bfloat16, device=cuda)
    rec = torch.zeros(T, 2, 128, 128, device=cuda)
    o2 = torch.empty(T, P, dtype=torch.bfloat16, device=cuda)

    def step():
        mla.decode(q, cache, table, lens, 0.06, out)
        layer.decode(proj, gate, beta, o2, seqs, conv, rec)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for lengths in ([300, 1, 0, 512], [17, 512, 129, 128]):
        lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        q.copy_(torch.randn(T, H, 576, generator=g, device=cuda))
        conv0, rec0 = conv.clone(), rec.clone()
        graph.replay()
        got, got2, conv1, rec1 = out.clone(), o2.clone(), conv.clone(), rec.clone()
        conv.copy_(conv0), rec.copy_(rec0)
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, out) and torch.equal(got2, o2)
        assert torch.equal(conv1, conv) and torch.equal(rec1, rec)
