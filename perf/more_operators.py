"""The operators of several continuations of one request, as they are measured: a tree of drafted tokens checked at once
(attention over the paged e4m3 latent cache, the KDA recurrence along every branch, the states advanced by the accepted
path), cache rows moved by lists (beams' states reordered, pages forked, accepted tokens compacted), and a beam search's
selection.

Every case is one call of one operator. `run` makes that call through the package's entry points where `own` is set;
otherwise it computes the operator from its formula with elementary torch operations in 32 bits (64 where candidates of
different beams are compared), rounded once.

  tree attention   node i of a request sees positions 0 .. L - 1 and L + j for every node j on its path (i included):
                   s_j = bmm1 q_h . kv_j (576 values), out_h = bmm2 sum_j softmax(s)_j kv_j[:512]
  tree recurrence  y = SiLU(conv4(x)) with the taps on the node's path, then on the request's conv rows; S_i <- from the
                   parent's state: S diag(exp(gate)); u = sigmoid(beta) (v - S k); S + u k^T; out_i = 128^-1/2 S q; the
                   request's state block stays as it is
  advance          the same steps along a list of accepted rows, the block's conv rows and state moved on
  move             row dst[i] <- what row src[i] held before the call, for every list and every view that goes by it
  beams            score[b] + x[b, v] - log sum_v exp x[b, v], the k largest of a request's beams x vocabulary in order,
                   ties to the lowest b V + v; a finished beam has one candidate, the pad token at its own score
"""

import math
import random

import torch

own = False

LAT, ROPE, PAGE = 512, 64, 128
DQ = LAT + ROPE
D = 128                                   # KDA head dim
MAX_CONTEXT = 131072
BMM1 = 256 ** -0.5                        # the model's softmax scale: query heads of 192 + 64 values
LOWER_BOUND = -5.0                        # the KDA gate's lower bound
BLOCK_BYTES = 8576 * DQ                   # a cache block: 8,576 latent rows or one KDA layer's state
POOL_PAGE = 32 * 128 * 2                  # the pool keys of a page


def listed():
    return [
        # one request, a tree of 24 drafts over a short context of odd length: the latency of a check
        dict(name="tree_1x24", op="tree", rows=1, nodes=24, heads=64, dist="same", tokens=4001, q="bf16"),
        # a batch of the prompt stream's lengths with trees of 16 to 32 drafts: the largest
        dict(name="tree_8x32", op="tree", rows=8, nodes=32, heads=64, dist="lognormal", tokens=8192, q="bf16"),
        # a quarter of the heads (tensor-parallel ranks), the FP8 query that the stage packs
        dict(name="tree_20x12_16heads_q8", op="tree", rows=20, nodes=12, heads=16, dist="lognormal", tokens=4096,
             q="e4m3"),
        # one request's tree, the 32-head layer: latency
        dict(name="kda_tree_1x24", op="kda_tree", rows=1, nodes=24, heads=32),
        # an ordinary batch of the 64-head layer
        dict(name="kda_tree_16x32", op="kda_tree", rows=16, nodes=32, heads=64),
        # many requests with trees up to the largest the operator takes
        dict(name="kda_tree_48x64", op="kda_tree", rows=48, nodes=64, heads=64),
        # the accepted path of one request
        dict(name="advance_1", op="advance", rows=1, most=5, heads=32),
        # the accepted paths of a batch, 1 to 6 tokens each
        dict(name="advance_64", op="advance", rows=64, most=6, heads=64),
        # accepted tokens moved to the front of their trees in three layers' latent rows
        dict(name="compact_64", op="compact", rows=64, nodes=32, most=6, layers=3),
        # beams reordered in place: three KDA layers' states, their current page in three DSA layers
        dict(name="reorder_8x4", op="reorder", rows=8, beams=4, layers=3),
        # one request's four beams over the model's vocabulary
        dict(name="beams_1x4", op="beams", rows=1, beams=4, k=4, vocab=151552, x="fp32", finished=False),
        # a batch of beam searches, some beams finished
        dict(name="beams_64x8", op="beams", rows=64, beams=8, k=8, vocab=151552, x="fp32", finished=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "kda_tree", "kda_tree", "advance", "compact", "reorder", "beams", "beams"])
    if op == "tree":
        heads = rng.choice([64, 64, 32, 16, rng.randint(1, 64)])
        rows, nodes = _log_int(rng, 1, 32), _log_int(rng, 1, 64)
        # the products stay below the largest listed case's
        most = max(64, min(MAX_CONTEXT, 1000000 // (rows * nodes)))
        return dict(op=op, rows=rows, nodes=nodes, heads=heads, dist=rng.choice(["same", "lognormal"]),
                    tokens=_log_int(rng, 16, most), q=rng.choice(["bf16", "bf16", "e4m3"]))
    if op == "kda_tree":
        return dict(op=op, rows=_log_int(rng, 1, 40), nodes=_log_int(rng, 1, 64), heads=rng.choice([16, 32, 64, 64]))
    if op == "advance":
        return dict(op=op, rows=_log_int(rng, 1, 64), most=rng.randint(1, 6), heads=rng.choice([16, 32, 64, 64]))
    if op == "compact":
        nodes = rng.randint(4, 64)
        return dict(op=op, rows=_log_int(rng, 1, 64), nodes=nodes, most=rng.randint(1, min(nodes, 12)),
                    layers=rng.randint(1, 3))
    if op == "reorder":
        return dict(op=op, rows=_log_int(rng, 1, 8), beams=rng.randint(2, 4), layers=rng.randint(1, 3))
    beams, k = rng.randint(1, 8), rng.randint(1, 16)
    return dict(op=op, rows=_log_int(rng, 1, 64), beams=beams, k=k, vocab=_log_int(rng, 1000, 151552),
                x=rng.choice(["fp32", "fp32", "bf16"]), finished=rng.random() < 0.5)


# ------------------------------------------------------------------ the cases' plans (the work goes by the case alone)
def _lengths(case):
    if case["dist"] == "same":
        return [case["tokens"]] * case["rows"]
    rng = random.Random(case["tokens"] * 1009 + case["rows"])
    return [max(1, min(MAX_CONTEXT, int(case["tokens"] * math.exp(rng.gauss(0.0, 0.8))))) for _ in range(case["rows"])]


def _trees(case):
    """Each request's tree as its nodes' parents (-1: the context's last token), parents before children."""
    rng = random.Random(case["rows"] * 131 + case["nodes"])
    out = []
    for _ in range(case["rows"]):
        n = case["nodes"] if case["rows"] == 1 else rng.randint((case["nodes"] + 1) // 2, case["nodes"])
        parents = [-1]
        for i in range(1, n):
            parents.append(-1 if rng.random() < 0.12 else rng.randint(max(0, i - 8), i - 1))
        out.append(parents)
    return out


def _paths(parents):
    """Each node's path from the root's child to itself."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [i])
    return out


def _mask(path):
    m = sum(1 << j for j in path)
    return m - (1 << 64) if m >> 63 else m                    # as the int64 word's bits


def _run_lengths(case):
    rng = random.Random(case["rows"] * 7919 + case["most"])
    return [case["most"] if case["rows"] == 1 else rng.randint(1, case["most"]) for _ in range(case["rows"])]


def _accepted(case):
    """Ascending accepted nodes of each request."""
    rng = random.Random(case["rows"] * 31 + case["nodes"])
    return [sorted(rng.sample(range(case["nodes"]), n)) for n in _run_lengths(case)]


def _beam_parents(case):
    rng = random.Random(case["rows"] * 17 + case["beams"])
    return [[min(rng.randrange(case["beams"]), rng.randrange(case["beams"])) for _ in range(case["beams"])]
            for _ in range(case["rows"])]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _e4m3(x):
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


# ------------------------------------------------------------------ inputs
def _tree_inputs(case, seed):
    g = _generator(seed)
    dev = dict(device="cuda")
    lens, trees = _lengths(case), _trees(case)
    pages = [-(-(n + len(t)) // PAGE) for n, t in zip(lens, trees)]
    total = sum(pages) + 3
    order = torch.randperm(total, generator=g, **dev).to(torch.int32)
    table = torch.full((len(lens), max(pages)), -1, dtype=torch.int32, **dev)
    at = 0
    for r, n in enumerate(pages):
        table[r, :n] = order[at:at + n]
        at += n
    cache = torch.empty(total * PAGE, DQ, dtype=torch.uint8, **dev)
    step = 1 << 18
    for i in range(0, cache.shape[0], step):
        n = min(step, cache.shape[0] - i)
        cache[i:i + n] = _e4m3(torch.randn(n, DQ, generator=g, **dev))
    T = sum(len(t) for t in trees)
    q = torch.randn(T, case["heads"], DQ, generator=g, **dev) * 1.5
    q = q.to(torch.bfloat16) if case["q"] == "bf16" else _e4m3(q)
    masks = torch.tensor([_mask(p) for t in trees for p in _paths(t)], dtype=torch.int64, **dev)
    return dict(q=q, cache=cache, table=table, lens=lens, trees=trees, masks=masks,
                reqs=_i32([r for r, t in enumerate(trees) for _ in t]),
                seq_lens=_i32([lens[r] for r, t in enumerate(trees) for _ in t]))


def _kda_inputs(case, seed):
    g = _generator(seed)
    dev = dict(device="cuda")
    H, P = case["heads"], case["heads"] * D
    tree = case["op"] == "kda_tree"
    runs = [len(t) for t in _trees(case)] if tree else _run_lengths(case)
    # an advance takes its rows out of a larger step's
    R, n = len(runs), sum(runs)
    T = n if tree else 4 * n
    blocks = torch.randperm(R + 2, generator=g, **dev)[:R].tolist()
    seqs, at = [], 0
    for r, m in enumerate(runs):
        seqs.append((at, at + m, blocks[r], 0 if r % 7 == 5 else 1))
        at += m
    ld = -(-(3 * P + 256 + H) // 256) * 256                   # the fused input projection's row
    s = dict(H=H, P=P, T=T, seqs=seqs,
             proj=torch.randn(T, ld, generator=g, **dev).to(torch.bfloat16),
             gate=torch.randn(T, P, generator=g, **dev).to(torch.bfloat16),
             conv=torch.randn(R + 2, 3, 3 * P, generator=g, **dev).to(torch.bfloat16),
             rec=torch.randn(R + 2, H, D, D, generator=g, **dev) * 0.1,
             w=((torch.rand(3 * P, 4, generator=g, **dev) - 0.5) * 1.2).to(torch.bfloat16),
             a_log=torch.rand(H, generator=g, **dev) * 2 - 1, dt_bias=torch.randn(P, generator=g, **dev) * 0.5)
    s["beta"] = s["proj"][:, 3 * P + 256:3 * P + 256 + H]
    if tree:
        s["trees"] = _trees(case)
        s["out"] = torch.empty(T, P, dtype=torch.bfloat16, **dev)
    else:
        rng = random.Random(case["rows"])
        s["row_list"] = sorted(rng.sample(range(T), n))
    return s


def _bytes(g, *shape):
    return torch.randint(0, 256, shape, dtype=torch.uint8, device="cuda", generator=g)


def _move_inputs(case, seed):
    g = _generator(seed)
    if case["op"] == "compact":
        R, n = case["rows"], case["nodes"]
        slots = 128 * (R + 1)
        first = [int(v) for v in (torch.randint(0, 128 - n + 1, (R,), generator=g, device="cuda") + 128 *
                                  torch.randperm(R + 1, generator=g, device="cuda")[:R]).tolist()]
        acc = _accepted(case)
        width = max(len(a) for a in acc)
        src = [[f + j for j in a] + [-1] * (width - len(a)) for f, a in zip(first, acc)]
        dst = [[f + i for i in range(len(a))] + [-1] * (width - len(a)) for f, a in zip(first, acc)]
        return dict(views=[_bytes(g, slots, DQ) for _ in range(case["layers"])], lists=[0] * case["layers"],
                    src=[src], dst=[dst])
    R, B = case["rows"], case["beams"]
    states = _state_bytes(64)
    n = R * B + 2
    views = [_bytes(g, n, BLOCK_BYTES)[:, :states] for _ in range(case["layers"])]
    views += [_bytes(g, n + 5, PAGE * DQ) for _ in range(case["layers"])]
    views += [_bytes(g, n + 5, POOL_PAGE) for _ in range(case["layers"])]
    blocks = torch.randperm(n, generator=g, device="cuda")[:R * B].view(R, B).tolist()
    pages = torch.randperm(n + 5, generator=g, device="cuda")[:R * B].view(R, B).tolist()
    parents = _beam_parents(case)
    pick = lambda ids: [[row[p] for p in par] for row, par in zip(ids, parents)]
    return dict(views=views, lists=[0] * case["layers"] + [1] * (2 * case["layers"]), src=[pick(blocks), pick(pages)],
                dst=[blocks, pages])


def _state_bytes(heads):
    return 3 * 3 * heads * D * 2 + heads * D * D * 4          # conv rows, then the recurrent state (256-byte multiples)


def _beam_inputs(case, seed):
    g = _generator(seed)
    G, B, V = case["rows"], case["beams"], case["vocab"]
    x = torch.randn(G * B, V, generator=g, device="cuda") * 3.0
    scores = -torch.rand(G, B, generator=g, device="cuda") * 8.0
    finished = None
    if case["finished"]:
        finished = torch.rand(G, B, generator=g, device="cuda") < 0.2
        finished[:, 0] = False                                # a search whose beams are all finished has ended
    return dict(x=x.to(torch.bfloat16) if case["x"] == "bf16" else x, scores=scores, finished=finished, k=case["k"],
                pad=V // 2)


def _inputs(case, seed):
    s = {"tree": _tree_inputs, "kda_tree": _kda_inputs, "advance": _kda_inputs, "compact": _move_inputs,
         "reorder": _move_inputs, "beams": _beam_inputs}[case["op"]](case, seed)
    s["op"] = case["op"]
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    dev = dict(device="cuda")
    op = s["op"]
    if op == "tree":
        s["out"] = torch.empty(s["q"].shape[0], s["q"].shape[1], LAT, dtype=torch.bfloat16, **dev)
    elif op in ("kda_tree", "advance"):
        s["seq_table"] = _i32(s["seqs"])
        if op == "kda_tree":
            s["parents"] = _i32([p for t in s["trees"] for p in t])
        else:
            s["rows"] = _i32(s["row_list"])
    elif op in ("compact", "reorder"):
        s["src_table"], s["dst_table"] = _i32(s["src"]), _i32(s["dst"])
    s["status"] = torch.zeros(1, dtype=torch.int32, **dev)
    if own:
        import __graft_entry__

        __graft_entry__.import_package()
        from ssengine_b200 import beam, kda, kvpages, lib, mla

        lib.load()
        if op == "tree":
            s["mla"] = mla
            n = mla.decode_workspace_bytes(s["q"].shape[0], s["q"].shape[1])
            s["workspace"] = torch.empty(n, dtype=torch.uint8, **dev)
        elif op in ("kda_tree", "advance"):
            s["layer"] = kda.KdaLayer(s["w"], s["a_log"], s["dt_bias"], LOWER_BOUND)
        elif op in ("compact", "reorder"):
            s["mover"] = kvpages.RowMover(s["views"], s["lists"])
        else:
            s["beam"] = beam
            n = beam.workspace_bytes(*s["scores"].shape, s["x"].shape[1], s["k"])
            s["workspace"] = torch.empty(n, dtype=torch.uint8, **dev)
            shape = (s["scores"].shape[0], s["k"])
            s["picked"] = tuple(torch.empty(shape, dtype=t, **dev) for t in (torch.float32, torch.int32, torch.int64))
    return s


def run(s):
    if own:
        return _run_own(s)
    return {"tree": _plain_tree, "kda_tree": _plain_kda_tree, "advance": _plain_advance, "compact": _plain_move,
            "reorder": _plain_move, "beams": _plain_beams}[s["op"]](s)


def _run_own(s):
    op = s["op"]
    if op == "tree":
        return s["mla"].decode_tree(s["q"], s["cache"], s["table"], s["seq_lens"], s["masks"], BMM1, s["out"],
                                    reqs=s["reqs"], workspace=s["workspace"], status=s["status"])
    if op == "kda_tree":
        return s["layer"].decode_tree(s["proj"], s["gate"], s["beta"], s["out"], s["seq_table"], s["parents"],
                                      s["conv"], s["rec"], max_nodes=max(len(t) for t in s["trees"]),
                                      status=s["status"])
    if op == "advance":
        s["layer"].advance(s["proj"], s["gate"], s["beta"], s["rows"], s["seq_table"], s["conv"], s["rec"],
                           status=s["status"])
        return dict(conv_state=s["conv"], rec_state=s["rec"])
    if op == "beams":
        scores, parents, tokens = s["beam"].select(s["x"], s["scores"], s["k"], finished=s["finished"], pad=s["pad"],
                                                   out=s["picked"], workspace=s["workspace"])
        return dict(scores=scores, parents=parents, tokens=tokens)
    s["mover"](s["src_table"], s["dst_table"], status=s["status"])
    return s["views"]


# ------------------------------------------------------------------ the plain forms
def _plain_tree(s):
    out = s["out"]
    q = s["q"].float() if s["q"].dtype == torch.bfloat16 else s["q"].view(torch.float8_e4m3fn).float()
    bit = torch.arange(64, device="cuda")
    t = 0
    for r, (length, tree) in enumerate(zip(s["lens"], s["trees"])):
        n, H = len(tree), q.shape[1]
        pos = torch.arange(length + n, device="cuda")
        kv = s["cache"][s["table"][r].long()[pos // PAGE] * PAGE + pos % PAGE].view(torch.float8_e4m3fn).float()
        keep = torch.ones(n, length + n, dtype=torch.bool, device="cuda")
        keep[:, length:] = ((s["masks"][t:t + n, None] >> bit[None, :n]) & 1) != 0
        for i in range(0, n, 8):                              # the scores of 8 nodes at a time
            a = torch.matmul(q[t + i:t + min(i + 8, n)], kv.T) * BMM1
            a = a.masked_fill_(~keep[i:i + 8, None, :], float("-inf"))
            p = torch.exp(a - a.amax(dim=2, keepdim=True))
            o = torch.matmul(p, kv[:, :LAT]) / p.sum(dim=2, keepdim=True)
            out[t + i:t + min(i + 8, n)] = o.to(torch.bfloat16)
        t += n
    return out


def _conv_kda(s, taps, rows, heads):
    """The step's q, k (normalised), v, decay and beta for the heads of a slice. taps fp32 [n, 4, 3P]."""
    y = (taps * s["w"].float().t()[None]).sum(dim=1)
    y = y / (1.0 + torch.exp(-y))
    q, k, v = y.view(-1, 3, s["H"], D)[:, :, heads].unbind(1)
    q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + 1e-6)
    k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    z = s["gate"][rows].float().view(-1, s["H"], D)[:, heads] + s["dt_bias"].view(1, s["H"], D)[:, heads]
    a = torch.exp(LOWER_BOUND / (1.0 + torch.exp(-torch.exp(s["a_log"])[None, heads, None] * z)))
    b = 1.0 / (1.0 + torch.exp(-s["beta"][rows].float()[:, heads]))
    return q, k, v, a, b


def _delta_step(S, k, v, a, b):
    S = S * a[:, :, None, :]
    u = b[:, :, None] * (v - (S * k[:, :, None, :]).sum(-1))
    return S + u[:, :, :, None] * k[:, :, None, :]


def _plain_kda_tree(s):
    H, P, seqs, trees = s["H"], s["P"], s["seqs"], s["trees"]
    blk = torch.tensor([b for _, _, b, _ in seqs], device="cuda")
    init = torch.tensor([float(i) for _, _, _, i in seqs], device="cuda")
    # the conv's rows: every request's three kept ones, then the step's; a node's taps by their place
    held = (s["conv"][blk].float() * init[:, None, None]).view(-1, 3 * P)
    rows = torch.cat([held, s["proj"][:, :3 * P].float()])
    base, taps = len(seqs) * 3, []
    for r, (first, _, _, _) in enumerate(seqs):
        for i, path in enumerate(_paths(trees[r])):
            chain = [3 * r, 3 * r + 1, 3 * r + 2] + [base + first + j for j in path]
            taps.append(chain[-4:])
    taps = torch.tensor(taps, device="cuda")
    out = torch.empty(s["T"], P, device="cuda")
    most = max(len(t) for t in trees)
    every = torch.arange(s["T"], device="cuda")
    for h in range(0, H, 8):
        heads = slice(h, min(h + 8, H))
        q, k, v, a, b = _conv_kda(s, rows[taps], every, heads)
        S = torch.empty(len(seqs), most + 1, q.shape[1], D, D, device="cuda")
        S[:, 0] = s["rec"][blk][:, heads] * init[:, None, None, None]
        for j in range(most):
            act = [r for r in range(len(seqs)) if j < len(trees[r])]
            t = torch.tensor([seqs[r][0] + j for r in act], device="cuda")
            up = torch.tensor([trees[r][j] + 1 for r in act], device="cuda")
            act = torch.tensor(act, device="cuda")
            new = _delta_step(S[act, up], k[t], v[t], a[t], b[t])
            S[act, j + 1] = new
            o = (new * q[t][:, :, None, :]).sum(-1) * D ** -0.5
            out.view(s["T"], H, D)[t, heads] = o
    s["out"].copy_(out.to(torch.bfloat16))
    return s["out"]


def _plain_advance(s):
    P, H, seqs = s["P"], s["H"], s["seqs"]
    blk = torch.tensor([b for _, _, b, _ in seqs], device="cuda")
    init = torch.tensor([float(i) for _, _, _, i in seqs], device="cuda")
    win = s["conv"][blk].float() * init[:, None, None]
    S = s["rec"][blk] * init[:, None, None, None]
    for j in range(max(e - b for b, e, _, _ in seqs)):
        act = [r for r, (b, e, _, _) in enumerate(seqs) if b + j < e]
        rows = torch.tensor([s["row_list"][seqs[r][0] + j] for r in act], device="cuda")
        act = torch.tensor(act, device="cuda")
        full = torch.cat([win[act], s["proj"][rows, :3 * P].float()[:, None, :]], dim=1)
        _, k, v, a, b = _conv_kda(s, full, rows, slice(0, H))
        S[act], win[act] = _delta_step(S[act], k, v, a, b), full[:, 1:]
    s["rec"][blk] = S
    s["conv"][blk] = win.to(torch.bfloat16)
    return dict(conv_state=s["conv"], rec_state=s["rec"])


def _plain_move(s):
    for view, l in zip(s["views"], s["lists"]):
        src, dst = s["src_table"][l].flatten().long(), s["dst_table"][l].flatten().long()
        ok = (src >= 0) & (dst >= 0)
        src, dst = src[ok], dst[ok]
        view[dst] = view[src].clone()
    return s["views"]


def _plain_beams(s):
    x, k = s["x"].double(), s["k"]
    G, B = s["scores"].shape
    V = x.shape[1]
    m = x.amax(dim=1, keepdim=True)
    lse = torch.log(torch.exp(x - m).sum(dim=1, keepdim=True)) + m
    cand = (s["scores"].double().view(-1, 1) + (x - lse)).view(G, B, V)
    if s["finished"] is not None:
        cand = torch.where(s["finished"][:, :, None], torch.full_like(cand, float("-inf")), cand)
        cand[:, :, s["pad"]] = torch.where(s["finished"], s["scores"].double(), cand[:, :, s["pad"]])
    cand = cand.view(G, B * V)
    place = torch.arange(B * V, device="cuda")
    scores, ids = [], []
    for _ in range(k):                                        # the largest left, the lowest place of equal ones
        best = cand.amax(dim=1, keepdim=True)
        at = torch.where(cand == best, place[None], torch.full_like(place[None], B * V)).amin(dim=1, keepdim=True)
        scores.append(best)
        ids.append(at)
        cand.scatter_(1, at, float("-inf"))
    ids = torch.cat(ids, dim=1)
    return dict(scores=torch.cat(scores, dim=1).float(), parents=(ids // V).to(torch.int32), tokens=ids % V)


# ------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    return {"tree": _exact_tree, "kda_tree": _exact_kda_tree, "advance": _exact_advance, "beams": _exact_beams,
            "compact": lambda s: None, "reorder": lambda s: None}[case["op"]](s)     # moved bytes: nothing is computed


def _exact_tree(s):
    """Node by node over its own list of cache rows."""
    e4m3 = torch.arange(256, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()
    q = s["q"].double() if s["q"].dtype == torch.bfloat16 else e4m3[s["q"].int()]
    out = torch.zeros(q.shape[0], q.shape[1], LAT, dtype=torch.float64, device="cuda")
    t = 0
    for r, tree in enumerate(s["trees"]):
        table = s["table"][r].long()
        length = s["lens"][r]
        for path in _paths(tree):
            pos = torch.cat([torch.arange(length, device="cuda"), length + torch.tensor(path, device="cuda")])
            kv = e4m3[s["cache"][table[pos // PAGE] * PAGE + pos % PAGE].int()]
            out[t] = torch.softmax((q[t] @ kv.T) * BMM1, dim=1) @ kv[:, :LAT]
            t += 1
    return out


def _exact_step(s, S, hist, row):
    """One token in float64 from the state [H, value, key] and the conv rows before it: (new state, output [P])."""
    H = s["H"]
    y = torch.nn.functional.silu(torch.einsum("ct,tc->c", s["w"].double(), hist[-4:])).view(3, H, D)
    q = y[0] * torch.rsqrt(y[0].square().sum(1, keepdim=True) + 1e-6)
    k = y[1] * torch.rsqrt(y[1].square().sum(1, keepdim=True) + 1e-6)
    z = s["a_log"].double().exp()[:, None] * (s["gate"][row].double() + s["dt_bias"].double()).view(H, D)
    S = S * torch.exp(LOWER_BOUND * torch.sigmoid(z))[:, None, :]
    u = torch.sigmoid(s["beta"][row].double())[:, None] * (y[2] - torch.einsum("hvk,hk->hv", S, k))
    S = S + torch.einsum("hv,hk->hvk", u, k)
    return S, (torch.einsum("hvk,hk->hv", S, q) / math.sqrt(D)).flatten()


def _start(s, block, init):
    conv, rec = s["conv"][block].double(), s["rec"][block].double()
    return (conv, rec) if init else (torch.zeros_like(conv), torch.zeros_like(rec))


def _exact_kda_tree(s):
    """Every node from its parent's state, request by request."""
    P = s["P"]
    out = torch.zeros(s["T"], P, dtype=torch.float64, device="cuda")
    for r, (first, _, block, init) in enumerate(s["seqs"]):
        conv, rec = _start(s, block, init)
        states, hists = {-1: rec}, {-1: conv}
        for i, parent in enumerate(s["trees"][r]):
            hists[i] = torch.cat([hists[parent], s["proj"][first + i:first + i + 1, :3 * P].double()])[-4:]
            states[i], out[first + i] = _exact_step(s, states[parent], hists[i], first + i)
    return out


def _exact_advance(s):
    conv, rec = s["conv"].double(), s["rec"].double()
    for first, end, block, init in s["seqs"]:
        hist, S = _start(s, block, init)
        for row in s["row_list"][first:end]:
            hist = torch.cat([hist, s["proj"][row:row + 1, :3 * s["P"]].double()])
            S, _ = _exact_step(s, S, hist, row)
        conv[block], rec[block] = hist[-3:], S
    return dict(conv_state=conv, rec_state=rec)


def _exact_beams(s):
    """Request by request; a beam's candidates are its k largest logits, the lowest tokens of equal ones."""
    G, B = s["scores"].shape
    k = s["k"]
    scores = torch.zeros(G, k, dtype=torch.float64, device="cuda")
    parents = torch.zeros(G, k, dtype=torch.int32, device="cuda")
    tokens = torch.zeros(G, k, dtype=torch.int64, device="cuda")
    for g in range(G):
        found = []
        for b in range(B):
            score = float(s["scores"][g, b])
            if s["finished"] is not None and bool(s["finished"][g, b]):
                found.append((-score, b, s["pad"]))
                continue
            x = s["x"][g * B + b].double()
            kth = torch.topk(x, min(k, x.numel())).values[-1]
            some = torch.nonzero(x >= kth).flatten()
            lse = torch.logsumexp(x, 0)
            found += [(-(score + v), b, t) for v, t in zip((x[some] - lse).tolist(), some.tolist())]
        found = sorted(found)[:k]
        scores[g] = torch.tensor([-f[0] for f in found], dtype=torch.float64, device="cuda")
        parents[g] = torch.tensor([f[1] for f in found], dtype=torch.int32, device="cuda")
        tokens[g] = torch.tensor([f[2] for f in found], device="cuda")
    return dict(scores=scores, parents=parents, tokens=tokens)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "tree":
        lens, trees = _lengths(case), _trees(case)
        H, T = case["heads"], sum(len(t) for t in trees)
        io = T * (H * (DQ * (2 if case["q"] == "bf16" else 1) + LAT * 2) + 16)
        seen = sum(len(t) * n + sum(len(p) for p in _paths(t)) for n, t in zip(lens, trees))
        # the nodes of a request read the same pages
        return dict(bytes=io + sum(n + len(t) for n, t in zip(lens, trees)) * DQ, flops=seen * H * 2 * (DQ + LAT))
    if op in ("kda_tree", "advance"):
        H, P = case["heads"], case["heads"] * D
        tree = op == "kda_tree"
        runs = [len(t) for t in _trees(case)] if tree else _run_lengths(case)
        R, T = len(runs), sum(runs)
        state = R * (H * D * D * 4 + 3 * 3 * P * 2) * (1 if tree else 2)
        rows = T * (3 * P * 2 + P * 2 + H * 2 + 4 + (P * 2 if tree else 0))
        # per node S k and S q of the request's state, and a dot and an update a pair on its path; an advance decays,
        # multiplies and updates
        pairs = sum(len(p) for t in _trees(case) for p in _paths(t)) if tree else 0
        return dict(bytes=state + rows + 3 * P * 4 * 2 + P * 4 + H * 4,
                    flops=H * (T * D * D * 4 + pairs * D * 8) if tree else T * H * D * D * 5)
    if op == "compact":
        moved = sum(sum(a != i for i, a in enumerate(acc)) for acc in _accepted(case))
        return dict(bytes=2 * moved * DQ * case["layers"] + 8 * sum(_run_lengths(case)), flops=0)
    if op == "reorder":
        par = _beam_parents(case)
        new = sum(p != b for row in par for b, p in enumerate(row))
        read = sum(len({p for b, p in enumerate(row) if p != b}) for row in par)
        return dict(bytes=(new + read) * case["layers"] * (_state_bytes(64) + PAGE * DQ + POOL_PAGE), flops=0)
    G, B, V = case["rows"], case["beams"], case["vocab"]
    return dict(bytes=G * B * (V * (4 if case["x"] == "fp32" else 2) + 4) + G * case["k"] * 16, flops=G * B * V * 4)
