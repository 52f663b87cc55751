"""The operators for several continuations of a request together, as they are used, on a stage's own caches.

- Speculation: two requests' trees of drafts checked step after step (`mla.decode_tree`, `KdaLayer.decode_tree`), a path of
  each accepted, its tokens brought to the front (`StageKv.move_tokens`) and the states advanced along it
  (`KdaLayer.advance`); every step's outputs against the formulas in 64 bits over the accepted history. The bars are those
  of the operators alone (test_gpu_tree.py): the states' own error, 1e-5 a token, does not show in them.
- Beams: a search on the tiny hybrid stage: one prefill, the request forked (`StageKv.move_states`, `move_pages`), steps of
  `StageModel.decode` and `beam.select` with the beams' states and pages following their parents; then every surviving
  hypothesis replayed as a request of its own. The replay's log probability of a hypothesis is within 5e-2 of the search's
  score: logits of unit scale within 2e-2 of one another (the stage's bar for two runs whose 4-bit requantizations may
  differ), over the five tokens' log sums. Another beam's state or page would move a token's logit by the logits' own
  scale."""

import numpy as np
import pytest
import torch

from test_gpu_decode import BMM1, D, attention64, check, kda_make, recurrence64
from test_gpu_tree import check_rows, kda_layer, path, tree64, wild
from oracle import mla as omla

pytestmark = pytest.mark.gpu


def test_speculation_steps(cuda):
    from ssengine_b200 import kvpages, mla

    rng = np.random.default_rng(40)
    H, R = 2, 2
    kv = kvpages.StageKv([2, 3], lambda i: i == 3, 6, H, cuda)          # one KDA layer, one DSA layer
    latent, conv, rec = kv.latent(3), kv.conv_state(2), kv.rec_state(2)
    latent.fill_(0x7F)                                                  # NaN wherever nothing was written
    pages = [[70, 68, 90], [69, 71, 72]]                                # of block 1; states in blocks 3 and 4
    table = torch.tensor(pages, dtype=torch.int32, device=cuda)
    slot = lambda r, p: pages[r][p // 128] * 128 + p % 128
    blocks = [3, 4]
    base = kda_make(rng, 1, H, R)
    L, _ = kda_layer(base, cuda)
    for r in range(R):
        conv[blocks[r]] = torch.from_numpy(base["cst"][r]).to(cuda, torch.bfloat16)
        rec[blocks[r]] = torch.from_numpy(base["rst"][r]).to(cuda)
    cst, rst = np.array(base["cst"], np.float64), np.array(base["rst"], np.float64)
    lens = [120, 61]
    keys = []
    for r in range(R):
        b = omla.quantize(rng.standard_normal((lens[r], 576)).astype(np.float32), 1.0)
        latent[torch.tensor([slot(r, p) for p in range(lens[r])], device=cuda)] = torch.from_numpy(b).to(cuda)
        keys.append(omla.e4m3_decode(b))
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)

    for step in range(6):
        trees = [wild(rng, int(rng.integers(1, 20))) for _ in range(R)]
        sizes = [len(t) for t in trees]
        T, first = sum(sizes), [0, sizes[0]]
        new = omla.quantize(rng.standard_normal((T, 576)).astype(np.float32), 1.0)
        where = [slot(r, lens[r] + i) for r in range(R) for i in range(sizes[r])]
        latent[torch.tensor(where, device=cuda)] = torch.from_numpy(new).to(cuda)
        q = torch.from_numpy(rng.standard_normal((T, 16, 576)).astype(np.float32)).to(torch.bfloat16)
        masks = torch.cat([mla.tree_masks(t)[0] for t in trees]).to(cuda)
        out = torch.empty(T, 16, 512, dtype=torch.bfloat16, device=cuda)
        reqs = [r for r in range(R) for _ in range(sizes[r])]
        mla.decode_tree(q.to(cuda), latent, table, i32([lens[r] for r in reqs]), masks, BMM1, out, reqs=i32(reqs),
                        status=status)
        d = kda_make(rng, T, H, R)
        d.update(w=base["w"], a_log=base["a_log"], dtb=base["dtb"], cst=cst, rst=rst)
        _, dev = kda_layer(d, cuda)
        o = torch.empty(T, H * D, dtype=torch.bfloat16, device=cuda)
        seqs = [(first[r], first[r] + sizes[r], r, 1) for r in range(R)]
        L.decode_tree(dev["x"], dev["g"], dev["beta"], o, i32([(s, e, blocks[r], i) for s, e, r, i in seqs]),
                      i32(sum(trees, [])), conv, rec, max_nodes=max(sizes), status=status)
        torch.cuda.synchronize()
        got = out.double().cpu().numpy()
        dec = omla.e4m3_decode(new)
        for r in range(R):
            for i in range(sizes[r]):
                t = first[r] + i
                seen = np.concatenate([keys[r], dec[[first[r] + j for j in path(trees[r], i)]]])
                check(got[t], None, *attention64(q[t].double().numpy(), seen, BMM1, 1.0))
        check_rows(o.double().cpu().numpy(), tree64(d, seqs, trees, H), H)

        takes = [path(trees[r], int(rng.integers(0, sizes[r])))[:5] for r in range(R)]
        width = max(len(a) for a in takes)
        src = [[slot(r, lens[r] + j) for j in takes[r]] + [-1] * (width - len(takes[r])) for r in range(R)]
        dst = [[slot(r, lens[r] + i) for i in range(len(takes[r]))] + [-1] * (width - len(takes[r])) for r in range(R)]
        kv.move_tokens(i32(src), i32(dst), status=status)
        rows = [first[r] + j for r in range(R) for j in takes[r]]
        ends = np.cumsum([0] + [len(a) for a in takes])
        L.advance(dev["x"], dev["g"], dev["beta"], i32(rows), i32([(int(ends[r]), int(ends[r + 1]), blocks[r], 1)
                                                                   for r in range(R)]), conv, rec, status=status)
        picked = {**d, **{c: np.asarray(d[c])[rows] for c in ("x", "g", "beta")}}
        _, cst, rst = recurrence64(picked, [(int(ends[r]), int(ends[r + 1]), r, 1) for r in range(R)], H)
        for r in range(R):
            keys[r] = np.concatenate([keys[r], dec[[first[r] + j for j in takes[r]]]])
            lens[r] += len(takes[r])
            back = latent[torch.tensor([slot(r, p) for p in range(lens[r])], device=cuda)].cpu().numpy()
            assert (omla.e4m3_decode(back) == keys[r]).all()
        torch.cuda.synchronize()
        assert int(status.item()) == 0
        for r in range(R):
            g = rec[blocks[r]].double().cpu().numpy()
            assert np.linalg.norm(g - rst[r]) <= 1e-4 * np.linalg.norm(rst[r])
            assert (conv[blocks[r]].double().cpu().numpy() == cst[r]).all()
    assert lens[0] > 128                                                # a tree lay across a page's end


def test_beam_search_on_a_stage(cuda):
    from ssengine_b200 import beam
    from ssengine_b200.messages import Chunk, Plan
    from ssengine_b200.stage import StageConfig, StageModel

    cfg = StageConfig(layer_split=(4,), hidden=256, inter=128, experts=8, top_k=2, vocab=1000, mb_tokens=256, num_blocks=40,
                      seed=3, layer_kind="hybrid", kda_heads=2, q_lora=256, mla_nope=64, routing="sigmoid")
    B, steps, n = 3, 5, 254
    rng = np.random.default_rng(41)
    prompt = rng.integers(0, cfg.vocab, n).tolist()
    st = StageModel(cfg, 0, cuda)
    # page 67 full and shared; the second one, and the next, of every beam its own; all in block 1
    own = [[68 + 2 * b, 69 + 2 * b] for b in range(B)]
    blocks = [[2 + 6 * b + g for g in range(6)] for b in range(B)]
    chunk = lambda b, start, toks: Chunk(f"beam{b}", start, len(toks), [67] + own[b], blocks[b], True, toks)
    st.forward(Plan(0, [chunk(0, 0, prompt)]))
    first = st.last_logits.clone()
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)
    dst_s = i32(blocks).t().contiguous().view(6, 1, B)                   # [state group, request, beam]
    dst_p = i32(own).t().contiguous()                                    # a group a page place
    # the fork: beam 0's states and open page to the others
    st.kv.move_states(dst_s[:, :, :1].expand(-1, -1, B).contiguous(), dst_s)
    st.kv.move_pages(dst_p[:, :1].expand(-1, B).contiguous(), dst_p)
    scores = torch.tensor([[0.0]], device=cuda)
    scores, parents, tokens = beam.select(first, scores, B)
    hyps = [[int(t)] for t in tokens[0]]
    for step in range(steps - 1):
        st.decode(Plan(1 + step, [chunk(b, n + step, [hyps[b][-1]]) for b in range(B)]))
        scores, parents, tokens = beam.select(st.last_logits, scores, B)
        pick = parents[0].long()
        st.kv.move_states(dst_s[:, :, pick].contiguous(), dst_s, status=st.status)
        st.kv.move_pages(dst_p[:, pick].contiguous(), dst_p, status=st.status)
        hyps = [hyps[p] + [t] for p, t in zip(parents[0].tolist(), tokens[0].tolist())]
    torch.cuda.synchronize()
    assert int(st.status.item()) == 0
    assert len({tuple(h) for h in hyps}) == B
    want = scores[0].tolist()
    assert want == sorted(want, reverse=True)

    fresh = StageModel(cfg, 0, cuda)
    pages = [[67 + 4 * b, 68 + 4 * b, 69 + 4 * b] for b in range(B)]
    chunk = lambda b, start, toks: Chunk(f"h{b}", start, len(toks), pages[b], blocks[b], True, toks)
    for b in range(B):
        fresh.forward(Plan(b, [chunk(b, 0, prompt)]))
        logits = [fresh.last_logits[0].double()]
        for i in range(steps - 1):
            fresh.decode(Plan(10 + i, [chunk(b, n + i, [hyps[b][i]])]))
            logits.append(fresh.last_logits[0].double())
        got = sum(float(torch.log_softmax(l, 0)[t]) for l, t in zip(logits, hyps[b]))
        assert abs(got - want[b]) < 5e-2, (b, got, want[b])
