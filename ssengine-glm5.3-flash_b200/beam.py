"""A beam search's selection through the C ABI (`ssb_beam_select`): what follows the lm_head of a step whose rows are
the beams of its requests, beside the greedy argmax (`ssb_argmax_rows`). The beams' pages and states then follow
their parents with `kvpages.StageKv.move_states` / `move_pages`. No fallback: without the CUDA library these calls
raise."""

from __future__ import annotations

import functools

import torch

from . import lib

MAX_BEAMS, MAX_K = 64, 64


@functools.cache
def workspace_bytes(requests: int, beams: int, vocab: int, k: int) -> int:
    """Device bytes of the workspace of one `select` call (`ssb_beam_workspace_bytes`)."""
    so = lib.load()
    # what an int32 argument would cut off is refused here
    fits = 1 <= beams <= MAX_BEAMS and 1 <= k <= MAX_K
    n = so.ssb_beam_workspace_bytes(requests, beams, vocab, k) if fits else -1
    if n < 0:
        raise ValueError(f"bad beam workspace query: {requests} requests x {beams} beams (1..{MAX_BEAMS}), vocabulary "
                         f"{vocab}, k={k} (1..{MAX_K})")
    return int(n)


def select(logits: torch.Tensor, scores: torch.Tensor, k: int, finished: torch.Tensor | None = None, pad: int = 0,
           out: tuple | None = None, workspace: torch.Tensor | None = None, stream=None) -> tuple:
    """The k best continuations of each request's beams: of the candidates (b, v) with score scores[g, b] + logits[g *
    B + b, v] - log sum exp of that row the k best in order, equal ones by the lower b * V + v (a beam's own by
    their logits). logits fp32 or bf16 [G * B, V] with unit column stride, scores fp32 [G, B] (the beams' log
    probabilities so far; B 1..64; -inf: a beam that is not there), k 1..64 -> (scores fp32 [G, k], parents int32
    [G, k]: the beam continued, tokens int64 [G, k]), new tensors or the three of `out` (with k == B the first may
    be `scores` itself). A beam with finished[g, b] (bool or uint8 [G, B]) has one candidate: token `pad` at its
    own score, its logits not read. A logit of -inf is no candidate; nor is any of a beam whose score or log sum is
    infinite or NaN. Places without a candidate get -inf, -1, -1. `workspace`: uint8, `workspace_bytes(G, B, V, k)`
    (default: one kept per stream, or in a capture one of the graph's own)."""
    so = lib.load()
    if scores.dtype is not torch.float32 or scores.dim() != 2 or not scores.is_contiguous():
        raise ValueError(f"scores: contiguous float32 [requests, beams], got {scores.dtype} {tuple(scores.shape)}")
    G, B = scores.shape
    bf16 = logits.dtype is torch.bfloat16
    if not (bf16 or logits.dtype is torch.float32) or logits.dim() != 2 or logits.shape[0] != G * B or \
            (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError(f"logits: float32 or bf16 [{G * B}, vocabulary] with unit column stride, got {logits.dtype} "
                         f"{tuple(logits.shape)} strides {logits.stride()}")
    V = logits.shape[1]
    if finished is not None and (finished.dtype not in (torch.bool, torch.uint8) or finished.shape != (G, B) or
                                 not finished.is_contiguous()):
        raise ValueError(f"finished: contiguous bool or uint8 {(G, B)}, got {finished.dtype} {tuple(finished.shape)}")
    if not 0 <= pad < max(V, 1):
        raise ValueError(f"pad token {pad} outside the vocabulary of {V}")
    need = workspace_bytes(G, B, V, k)
    if out is None:
        dev = dict(device=logits.device)
        out = (torch.empty(G, k, dtype=torch.float32, **dev), torch.empty(G, k, dtype=torch.int32, **dev),
               torch.empty(G, k, dtype=torch.int64, **dev))
    else:
        if len(out) != 3:
            raise ValueError(f"out: three tensors, got {len(out)}")
        for t, dtype in zip(out, (torch.float32, torch.int32, torch.int64)):
            if t.dtype is not dtype or t.shape != (G, k) or not t.is_contiguous():
                raise ValueError(f"out: contiguous {dtype} {(G, k)}, got {t.dtype} {tuple(t.shape)}")
    if workspace is not None and (workspace.dtype != torch.uint8 or not workspace.is_contiguous() or
                                  workspace.numel() < need):
        raise ValueError(f"workspace: contiguous uint8 of {need} bytes or more")
    lib.check_device((logits, scores, finished, *out, workspace), None, stream)
    if workspace is None:
        workspace = lib.stream_scratch(logits.device, need, stream)
    rc = so.ssb_beam_select(logits.data_ptr(), int(bf16), logits.stride(0), G, B, V, scores.data_ptr(),
                            None if finished is None else finished.data_ptr(), pad, k, out[0].data_ptr(),
                            out[1].data_ptr(), out[2].data_ptr(), workspace.data_ptr(), workspace.numel(),
                            lib.stream_ptr(stream))
    lib.check("ssb_beam_select", rc)
    return out
