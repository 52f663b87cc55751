"""The decode-step operators as they are measured: attention of new tokens over the paged e4m3 latent cache (all of a
row's tokens, or the tokens that the indexer selected), and the recurrent form of the KDA layer.

Every case is one call of one operator. `run` makes that call through the package's entry points where `own` is set;
otherwise it computes the operator from its formula with elementary torch operations in 32 bits, rounded once.

  attention   s_j = bmm1 q_h . kv_j (576 values), out_h = bmm2 sum_j softmax(s)_j kv_j[:512]; position p of a request
              lies in cache row page_table[request, p / 128] * 128 + p % 128
  recurrence  y = SiLU(conv4(x)); q, k L2-normalised per head; S <- S diag(exp(gate)); u = sigmoid(beta) (v - S k);
              S <- S + u k^T; out = 128^-1/2 S q, token after token, conv rows and S kept in the request's state block
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


def listed():
    return [
        # one request, a short context of odd length: the latency of a step
        dict(name="mla_1x1000", op="mla", rows=1, drafts=1, heads=64, dist="same", tokens=1000, q="bf16"),
        # one request at the longest context the stages reserve for
        dict(name="mla_1x131072", op="mla", rows=1, drafts=1, heads=64, dist="same", tokens=131072, q="bf16"),
        # a batch of the prompt stream's lengths (lognormal, median 8,192): ragged, unequal work per row
        dict(name="mla_32_ragged", op="mla", rows=32, drafts=1, heads=64, dist="lognormal", tokens=8192, q="bf16"),
        # a full decode batch at long contexts: the largest
        dict(name="mla_64x32768", op="mla", rows=64, drafts=1, heads=64, dist="same", tokens=32768, q="bf16"),
        # a quarter of the heads (tensor-parallel ranks), the FP8 query that the prefill attention takes
        dict(name="mla_48_16heads_q8", op="mla", rows=48, drafts=1, heads=16, dist="lognormal", tokens=4096, q="e4m3"),
        # four draft tokens a request checked at once, each with its own causal length over the same pages
        dict(name="mla_8x4_drafts", op="mla", rows=8, drafts=4, heads=64, dist="lognormal", tokens=16384, q="bf16"),
        # the indexer's 512 pools of 4 tokens and the 3 tail columns, one request
        dict(name="selected_1", op="selected", rows=1, heads=64, dist="same", tokens=50001, q="bf16"),
        # the same for a decode batch; rows shorter than the selection width leave columns empty
        dict(name="selected_96", op="selected", rows=96, heads=64, dist="lognormal", tokens=8192, q="e4m3"),
        # one token of one request, the 32-head layer: latency
        dict(name="kda_1x32", op="kda", rows=1, most=1, heads=32),
        # an ordinary decode batch of the 64-head layer, an odd number of requests
        dict(name="kda_61x64", op="kda", rows=61, most=1, heads=64),
        # runs of 1 to 8 tokens a request (drafts, short continuations), some requests fresh
        dict(name="kda_24x64_runs", op="kda", rows=24, most=8, heads=64),
        # the largest batch: 1 GB of recurrent state read and written
        dict(name="kda_256x64", op="kda", rows=256, most=1, heads=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["mla", "mla", "selected", "kda"])
    if op == "kda":
        most = rng.choice([1, 1, 1, rng.randint(2, 8)])
        return dict(op=op, rows=_log_int(rng, 1, 256 // most), most=most, heads=rng.choice([16, 32, 64, 64]))
    heads = rng.choice([64, 64, 64, 32, 16, rng.randint(1, 64)])
    q = rng.choice(["bf16", "bf16", "e4m3"])
    if op == "selected":
        return dict(op=op, rows=_log_int(rng, 1, 128), heads=heads, dist="lognormal",
                    tokens=_log_int(rng, 500, 16384), q=q)
    drafts = rng.choice([1, 1, 1, rng.randint(2, 4)])
    rows = _log_int(rng, 1, 64 // drafts)
    # the sum of the tokens stays below the largest listed case's
    most = min(MAX_CONTEXT, 1000000 // (rows * drafts))
    return dict(op=op, rows=rows, drafts=drafts, heads=heads, dist=rng.choice(["same", "lognormal"]),
                tokens=_log_int(rng, min(64, most), most), q=q)


def _lengths(case):
    """Cache tokens of each request (from the case alone, so that its work does not change with the seed)."""
    if case["dist"] == "same":
        return [case["tokens"]] * case["rows"]
    rng = random.Random(case["tokens"] * 1009 + case["rows"])
    return [max(1, min(MAX_CONTEXT, int(case["tokens"] * math.exp(rng.gauss(0.0, 0.8))))) for _ in range(case["rows"])]


def _row_lengths(case):
    """Tokens that each query row sees: the drafts of a request are its last tokens, one position apart."""
    n = case.get("drafts", 1)
    return [max(0, ln - (n - 1 - i)) for ln in _lengths(case) for i in range(n)]


def _run_lengths(case):
    rng = random.Random(case["rows"] * 7919 + case["most"])
    return [rng.randint(1, case["most"]) for _ in range(case["rows"])]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _e4m3(x):
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def _attention_inputs(case, seed):
    g = _generator(seed)
    dev = dict(device="cuda")
    lens = _lengths(case)
    pages = [-(-n // PAGE) for n in lens]
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
    n = case.get("drafts", 1)
    rows = _row_lengths(case)
    reqs = torch.arange(len(lens), dtype=torch.int32, **dev).repeat_interleave(n)
    q = torch.randn(len(rows), case["heads"], DQ, generator=g, **dev) * 1.5
    q = q.to(torch.bfloat16) if case["q"] == "bf16" else _e4m3(q)
    s = dict(q=q, cache=cache, table=table, reqs=reqs, rows=rows, seq_lens=torch.tensor(rows, dtype=torch.int32, **dev))
    if case["op"] == "selected":
        s["indices"] = torch.stack([_selection(ln, g) for ln in lens])
    return s


def _selection(length, g, pools=512):
    """The indexer's expanded selection of a row at position length - 1: up to 512 of the complete pools of 4 tokens,
    ascending, then the tokens of the incomplete pool; -1 where there is none."""
    out = torch.full((4 * pools + 3,), -1, dtype=torch.int32, device="cuda")
    whole = length // 4
    n = min(pools, whole)
    if n:
        ids = torch.randperm(whole, generator=g, device="cuda")[:n].sort().values
        out[:4 * n] = (ids[:, None] * 4 + torch.arange(4, device="cuda")).flatten().to(torch.int32)
    tail = torch.arange(4 * whole, length, device="cuda", dtype=torch.int32)
    out[4 * pools:4 * pools + tail.numel()] = tail
    return out


def _kda_inputs(case, seed):
    g = _generator(seed)
    dev = dict(device="cuda")
    H, P = case["heads"], case["heads"] * D
    lens = _run_lengths(case)
    R, T = len(lens), sum(lens)
    blocks = torch.randperm(R + 2, generator=g, **dev)[:R].tolist()
    seqs, at = [], 0
    for r, n in enumerate(lens):
        fresh = case["most"] > 1 and r % 5 == 4
        seqs.append((at, at + n, blocks[r], 0 if fresh else 1))
        at += n
    ld = -(-(3 * P + 256 + H) // 256) * 256                   # the fused input projection's row
    proj = torch.randn(T, ld, generator=g, **dev).to(torch.bfloat16)
    gate = torch.randn(T, P, generator=g, **dev).to(torch.bfloat16)
    conv = torch.randn(R + 2, 3, 3 * P, generator=g, **dev).to(torch.bfloat16)
    rec = torch.randn(R + 2, H, D, D, generator=g, **dev) * 0.1
    w = ((torch.rand(3 * P, 4, generator=g, **dev) - 0.5) * 1.2).to(torch.bfloat16)
    a_log = torch.rand(H, generator=g, **dev) * 2 - 1
    dt_bias = torch.randn(P, generator=g, **dev) * 0.5
    return dict(H=H, P=P, T=T, seqs=seqs, proj=proj, beta=proj[:, 3 * P + 256:3 * P + 256 + H], gate=gate, conv=conv,
                rec=rec, w=w, a_log=a_log, dt_bias=dt_bias, out=torch.empty(T, P, dtype=torch.bfloat16, **dev))


def _inputs(case, seed):
    return _kda_inputs(case, seed) if case["op"] == "kda" else _attention_inputs(case, seed)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["op"] = case["op"]
    if case["op"] == "kda":
        s["seq_table"] = torch.tensor(s["seqs"], dtype=torch.int32, device="cuda")
    else:
        s["out"] = torch.empty(s["q"].shape[0], s["q"].shape[1], LAT, dtype=torch.bfloat16, device="cuda")
    if own:
        import __graft_entry__

        __graft_entry__.import_package()
        from ssengine_b200 import kda, lib, mla

        s["mla"] = mla
        if case["op"] == "kda":
            s["layer"] = kda.KdaLayer(s["w"], s["a_log"], s["dt_bias"], LOWER_BOUND)
        else:
            n = mla.decode_workspace_bytes(s["q"].shape[0], s["q"].shape[1])
            s["workspace"] = torch.empty(n, dtype=torch.uint8, device="cuda")
        s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        lib.load()
    return s


def run(s):
    if own:
        return _run_own(s)
    return {"kda": _plain_kda, "mla": _plain_attention, "selected": _plain_selected}[s["op"]](s)


def _run_own(s):
    if s["op"] == "kda":
        s["layer"].decode(s["proj"], s["gate"], s["beta"], s["out"], s["seq_table"], s["conv"], s["rec"],
                          status=s["status"])
        return dict(out=s["out"], conv_state=s["conv"], rec_state=s["rec"])
    if s["op"] == "mla":
        return s["mla"].decode(s["q"], s["cache"], s["table"], s["seq_lens"], BMM1, s["out"], reqs=s["reqs"],
                               workspace=s["workspace"], status=s["status"])
    return s["mla"].decode_selected(s["q"], s["cache"], s["indices"], s["table"], BMM1, s["out"], reqs=s["reqs"],
                                    seq_lens=s["seq_lens"], workspace=s["workspace"], status=s["status"])


def _query32(q):
    return q.float() if q.dtype == torch.bfloat16 else q.view(torch.float8_e4m3fn).float()


def _plain_rows(q, cache, slots, keep):
    """q fp32 [n, H, 576], slots int64 [n, m] (any row where not kept), keep bool [n, m] -> fp32 [n, H, 512]."""
    kv = cache[slots].view(torch.float8_e4m3fn).float()
    kv = kv.masked_fill_(~keep[:, :, None], 0.0)
    s = torch.bmm(q, kv.transpose(1, 2)) * BMM1
    s = s.masked_fill_(~keep[:, None, :], float("-inf"))
    m = s.amax(dim=2, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    z = p.sum(dim=2, keepdim=True)
    o = torch.bmm(p, kv[:, :, :LAT])
    return torch.where(z > 0, o / z, torch.zeros_like(o))


def _groups(rows, budget=1 << 20):
    """Runs of rows whose padded tokens fit a bounded buffer."""
    i = 0
    while i < len(rows):
        j, most = i, 0
        while j < len(rows) and max(most, rows[j]) * (j + 1 - i) <= budget:
            most = max(most, rows[j])
            j += 1
        yield i, j, most
        i = j


def _plain_attention(s):
    q, out = _query32(s["q"]), s["out"]
    for i, j, most in _groups(s["rows"]):
        pos = torch.arange(most, device="cuda")
        pages = s["table"][s["reqs"][i:j].long()][:, pos // PAGE]
        keep = (pos[None, :] < s["seq_lens"][i:j, None]) & (pages >= 0)
        slots = torch.where(keep, pages * PAGE + (pos % PAGE)[None, :], torch.zeros_like(pages)).long()
        out[i:j] = _plain_rows(q[i:j], s["cache"], slots, keep).to(torch.bfloat16)
    return out


def _plain_selected(s):
    q, out, idx = _query32(s["q"]), s["out"], s["indices"].long()
    keep = (idx >= 0) & (idx < s["seq_lens"][:, None])
    idx = torch.where(keep, idx, torch.zeros_like(idx))
    pages = torch.gather(s["table"][s["reqs"].long()].long(), 1, idx // PAGE)
    keep = keep & (pages >= 0)
    slots = torch.where(keep, pages * PAGE + idx % PAGE, torch.zeros_like(idx))
    step = 64
    for i in range(0, q.shape[0], step):
        out[i:i + step] = _plain_rows(q[i:i + step], s["cache"], slots[i:i + step], keep[i:i + step]).to(torch.bfloat16)
    return out


def _plain_kda(s):
    H, P = s["H"], s["P"]
    seqs, w = s["seqs"], s["w"].float()
    blk = torch.tensor([b for _, _, b, _ in seqs], device="cuda")
    init = torch.tensor([bool(i) for _, _, _, i in seqs], device="cuda")
    win = s["conv"][blk].float() * init[:, None, None]
    S = s["rec"][blk] * init[:, None, None, None]                                 # [R, H, value, key]
    decay_rate = torch.exp(s["a_log"])[None, :, None]
    for j in range(max(e - b for b, e, _, _ in seqs)):
        act = [r for r, (b, e, _, _) in enumerate(seqs) if b + j < e]
        every = len(act) == len(seqs)
        rows = torch.tensor([seqs[r][0] + j for r in act], device="cuda")
        act = torch.tensor(act, device="cuda")
        x = s["proj"][rows, :3 * P].float()
        full = torch.cat([win if every else win[act], x[:, None, :]], dim=1)       # [n, 4, 3P]
        y = (full * w.t()[None]).sum(dim=1)
        y = y / (1.0 + torch.exp(-y))
        q, k, v = y.view(-1, 3, H, D).unbind(1)
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + 1e-6)
        k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)
        z = decay_rate * (s["gate"][rows].float().view(-1, H, D) + s["dt_bias"].view(1, H, D))
        a = torch.exp(LOWER_BOUND / (1.0 + torch.exp(-z)))
        b = 1.0 / (1.0 + torch.exp(-s["beta"][rows].float()))
        Sa = (S if every else S[act]) * a[:, :, None, :]
        u = b[:, :, None] * (v - (Sa * k[:, :, None, :]).sum(-1))
        Sa = Sa + u[:, :, :, None] * k[:, :, None, :]
        o = (Sa * q[:, :, None, :]).sum(-1) * D ** -0.5
        s["out"][rows] = o.reshape(-1, P).to(torch.bfloat16)
        if every:
            S, win = Sa, full[:, 1:]
        else:
            S[act], win[act] = Sa, full[:, 1:]
    s["rec"][blk] = S
    s["conv"][blk] = win.to(torch.bfloat16)
    return dict(out=s["out"], conv_state=s["conv"], rec_state=s["rec"])


def exact(case, seed):
    s = _inputs(case, seed)
    return _exact_kda(s) if case["op"] == "kda" else _exact_attention(s)


def _exact_attention(s):
    """Row by row in float64 over the row's own list of cache rows."""
    e4m3 = torch.arange(256, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()
    q = s["q"].double() if s["q"].dtype == torch.bfloat16 else e4m3[s["q"].int()]
    out = torch.zeros(q.shape[0], q.shape[1], LAT, dtype=torch.float64, device="cuda")
    for t, length in enumerate(s["rows"]):
        pos = torch.arange(length, device="cuda")
        if "indices" in s:
            pos = s["indices"][t].long()
            pos = pos[(pos >= 0) & (pos < length)]
        if pos.numel() == 0:
            continue
        kv = e4m3[s["cache"][s["table"][int(s["reqs"][t])].long()[pos // PAGE] * PAGE + pos % PAGE].int()]
        out[t] = torch.softmax((q[t] @ kv.T) * BMM1, dim=1) @ kv[:, :LAT]
    return out


def _exact_kda(s):
    """Sequence by sequence and token by token in float64; the state as [value, key] matrices."""
    H, P = s["H"], s["P"]
    conv, rec = s["conv"].double(), s["rec"].double()
    out = torch.zeros(s["T"], P, dtype=torch.float64, device="cuda")
    taps = s["w"].double()
    for first, end, b, init in s["seqs"]:
        hist = conv[b] if init else torch.zeros_like(conv[b])
        S = rec[b] if init else torch.zeros_like(rec[b])
        for t in range(first, end):
            hist = torch.cat([hist, s["proj"][t:t + 1, :3 * P].double()])
            y = torch.nn.functional.silu(torch.einsum("ct,tc->c", taps, hist[-4:])).view(3, H, D)
            q = y[0] * torch.rsqrt(y[0].square().sum(1, keepdim=True) + 1e-6)
            k = y[1] * torch.rsqrt(y[1].square().sum(1, keepdim=True) + 1e-6)
            z = s["a_log"].double().exp()[:, None] * (s["gate"][t].double() + s["dt_bias"].double()).view(H, D)
            S = S * torch.exp(LOWER_BOUND * torch.sigmoid(z))[:, None, :]
            u = torch.sigmoid(s["beta"][t].double())[:, None] * (y[2] - torch.einsum("hvk,hk->hv", S, k))
            S = S + torch.einsum("hv,hk->hvk", u, k)
            out[t] = (torch.einsum("hvk,hk->hv", S, q) / math.sqrt(D)).flatten()
        conv[b] = hist[-3:]
        rec[b] = S
    return dict(out=out, conv_state=conv, rec_state=rec)


def work(case):
    if case["op"] == "kda":
        H, P = case["heads"], case["heads"] * D
        lens = _run_lengths(case)
        R, T = len(lens), sum(lens)
        # state blocks and conv rows in and out once; each token's q | k | v, gate, beta and output; the weights
        state = 2 * R * (H * D * D * 4 + 3 * 3 * P * 2)
        rows = T * (3 * P * 2 + P * 2 + H * 2 + P * 2)
        return dict(bytes=state + rows + 3 * P * 4 * 2 + P * 4 + H * 4, flops=T * H * D * D * 7)
    rows = _row_lengths(case)
    H = case["heads"]
    qb = 2 if case["q"] == "bf16" else 1
    io = len(rows) * H * (DQ * qb + LAT * 2)
    if case["op"] == "selected":
        used = [min(512, n // 4) * 4 + n % 4 for n in rows]
        return dict(bytes=io + sum(used) * DQ + len(rows) * 2051 * 4, flops=sum(used) * H * 2 * (DQ + LAT))
    # the drafts of a request read the same pages
    return dict(bytes=io + sum(_lengths(case)) * DQ, flops=sum(rows) * H * 2 * (DQ + LAT))
