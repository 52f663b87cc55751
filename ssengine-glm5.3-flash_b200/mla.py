"""Sparse MLA prefill, the attention of new tokens, the FP8 latent-cache append and the FP8 query pack of one DSA layer
through the C ABI (`ssb_sparse_mla`, `ssb_mla_decode`, `ssb_mla_decode_tree`, `ssb_mla_cache_append`, `ssb_mla_q_pack`).

Mirrors the reference's calls: the TRTLLM sparse MLA with FP8 query and cache (`trtllm_batch_decode_with_kv_cache_mla`
with the indexer's top-k token lists and bmm1 = scale * q_scale * k_scale, bmm2 = k_scale; split at 32,768 rows:
ssengine/model/pp_patch.py:643-672; ssengine/kernels.py config 25), the fork's FP8 MLA cache write
(`concat_and_cache_mla`, config 23) and the query's `scaled_fp8_quant`. The latent cache is e4m3 rows of 576 bytes
(latent 512 + rope 64). No fallback: without the CUDA library these calls raise.
"""

from __future__ import annotations

import functools

import torch

from . import lib

HEADS, DQ, DV = 64, 576, 512


def sparse_mla(q8: torch.Tensor, kv_cache: torch.Tensor, indices: torch.Tensor, qsl: torch.Tensor,
               page_table: torch.Tensor, bmm1: float, out: torch.Tensor, bmm2: float = 1.0, n_idx: int | None = None,
               stream=None, status: torch.Tensor | None = None) -> torch.Tensor:
    """q8 e4m3 bytes uint8 [T, 64, 576], kv_cache e4m3 bytes uint8 [slots, 576], indices int32 [T, >= n_idx], qsl int32
    [R + 1], page_table int32 [R, width] -> out bf16 [T, 64, 512]."""
    so = lib.load()
    assert q8.dtype == torch.uint8 and q8.is_contiguous() and q8.shape[1:] == (HEADS, DQ)
    assert kv_cache.dtype == torch.uint8 and kv_cache.is_contiguous() and kv_cache.shape[1] == DQ
    assert indices.dtype == torch.int32 and indices.stride(1) == 1
    assert out.dtype == torch.bfloat16 and out.is_contiguous()
    n = indices.shape[1] if n_idx is None else n_idx
    rc = so.ssb_sparse_mla(q8.data_ptr(), q8.shape[0], kv_cache.data_ptr(), indices.data_ptr(), indices.stride(0), n,
                           qsl.data_ptr(), qsl.shape[0] - 1, page_table.data_ptr(), page_table.shape[1], bmm1, bmm2,
                           out.data_ptr(), None if status is None else status.data_ptr(), lib.stream_ptr(stream))
    lib.check("ssb_sparse_mla", rc)
    return out


@functools.cache
def decode_workspace_bytes(T: int, heads: int) -> int:
    """Device bytes of the workspace of one `decode` / `decode_selected` call (`ssb_mla_decode_workspace_bytes`)."""
    n = lib.load().ssb_mla_decode_workspace_bytes(T, heads)
    if n < 0:
        raise ValueError(f"bad MLA decode workspace query: T={T}, heads={heads} (1..128)")
    return int(n)


def decode(q: torch.Tensor, kv_cache: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, bmm1: float,
           out: torch.Tensor, bmm2: float = 1.0, reqs: torch.Tensor | None = None, lse: torch.Tensor | None = None,
           workspace: torch.Tensor | None = None, stream=None, status: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new tokens over all of their request's cache: row t sees positions 0 .. seq_lens[t] - 1 of the
    pages in row reqs[t] (default t) of page_table int32 [R, width]. q [T, H, 576], H = 1..128, bf16 or e4m3 bytes
    (uint8) with unit stride in the last dimension and 16-byte row and head strides; kv_cache e4m3 bytes uint8
    [slots, 576]; seq_lens, reqs int32 [T]; -> out bf16 [T, H, 512] and, when given, lse fp32 [T, H]. A row without a
    token gets zeros (lse -inf). bmm1 = softmax scale * q_scale * k_scale, bmm2 = k_scale, as `sparse_mla`. Split over
    the tokens and joined in `workspace` (uint8, `decode_workspace_bytes(T, H)`; default: one kept per stream, or in a
    capture one of the graph's own); the lengths are read on the device. `status` (int32 [1] on the device) receives 1
    for a reqs entry outside the table, 4 if a bounded wait gave up (the call's outputs are then undefined)."""
    return _decode(q, kv_cache, None, page_table, seq_lens, bmm1, out, bmm2, None, reqs, lse, workspace, stream, status)


def decode_selected(q: torch.Tensor, kv_cache: torch.Tensor, indices: torch.Tensor, page_table: torch.Tensor,
                    bmm1: float, out: torch.Tensor, bmm2: float = 1.0, n_idx: int | None = None,
                    seq_lens: torch.Tensor | None = None, reqs: torch.Tensor | None = None,
                    lse: torch.Tensor | None = None, workspace: torch.Tensor | None = None, stream=None,
                    status: torch.Tensor | None = None) -> torch.Tensor:
    """`decode` over the positions listed in the first n_idx columns of indices int32 [T, >= n_idx] (the indexer's
    expanded selection; -1 = none), those at or past seq_lens[t] left out when seq_lens is given (it also tells how
    much work a short row holds, which balances the split). No column (n_idx 0 or indices [T, 0]): no token, as for
    any row that has none."""
    if indices.dtype != torch.int32 or indices.dim() != 2 or indices.stride(1) != 1 or indices.shape[0] < q.shape[0]:
        raise ValueError(f"indices: int32 [{q.shape[0]}, n] with unit column stride, got {indices.dtype} "
                         f"{tuple(indices.shape)}")
    n = indices.shape[1] if n_idx is None else n_idx
    if not 0 <= n <= indices.shape[1]:
        raise ValueError(f"n_idx {n} of {indices.shape[1]} columns")
    return _decode(q, kv_cache, indices, page_table, seq_lens, bmm1, out, bmm2, n, reqs, lse, workspace, stream, status)


def decode_tree(q: torch.Tensor, kv_cache: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                ancestors: torch.Tensor, bmm1: float, out: torch.Tensor, bmm2: float = 1.0,
                reqs: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                workspace: torch.Tensor | None = None, stream=None, status: torch.Tensor | None = None) -> torch.Tensor:
    """`decode` for the nodes of trees of drafted tokens, a request's nodes in its cache behind its context (at most 64):
    row t sees positions 0 .. seq_lens[t] - 1 and seq_lens[t] + j for every bit j of ancestors[t] (int64 [T]: the nodes on
    the row's path, itself among them, as `tree_masks` makes them; any set is taken). A row without either gets zeros."""
    if ancestors.dtype is not torch.int64 or ancestors.shape != q.shape[:1] or not ancestors.is_contiguous():
        raise ValueError(f"ancestors: contiguous int64 [{q.shape[0]}], got {ancestors.dtype} {tuple(ancestors.shape)}")
    if seq_lens is None:
        raise ValueError("seq_lens: int32 [T], the context before each row's tree")
    return _decode(q, kv_cache, None, page_table, seq_lens, bmm1, out, bmm2, None, reqs, lse, workspace, stream, status,
                   ancestors)


def tree_masks(parents) -> tuple[torch.Tensor, torch.Tensor]:
    """One tree's parents (a parent before its children, -1 for a root; at most 64 nodes) -> (ancestors int64 [n]: bit j set
    where node j is on the node's path, itself among them; depths int64 [n]: nodes above it, so that a node's position is
    the context's length + its depth), on the host. ValueError if it is no such tree."""
    masks, depths = [], []
    for i, p in enumerate(parents):
        p = int(p)
        if not -1 <= p < i or i > 63:
            raise ValueError(f"node {i} with parent {p}: parents come first, at most 64 nodes")
        masks.append((masks[p] if p >= 0 else 0) | 1 << i)
        depths.append(depths[p] + 1 if p >= 0 else 0)
    signed = [m - (1 << 64) if m >> 63 else m for m in masks]
    return torch.tensor(signed, dtype=torch.int64), torch.tensor(depths, dtype=torch.int64)


def _decode(q, kv_cache, indices, page_table, seq_lens, bmm1, out, bmm2, n_idx, reqs, lse, workspace, stream, status,
            ancestors=None):
    so = lib.load()
    e4m3 = q.dtype is torch.uint8
    if not (e4m3 or q.dtype is torch.bfloat16) or q.dim() != 3 or q.shape[2] != DQ or q.stride(2) != 1:
        raise ValueError(f"q: bf16 or e4m3 bytes [T, heads, {DQ}] with unit stride in the last dimension, got {q.dtype} "
                         f"{tuple(q.shape)} strides {q.stride()}")
    T, H, _ = q.shape
    if kv_cache.dtype != torch.uint8 or kv_cache.dim() != 2 or kv_cache.shape[1] != DQ or not kv_cache.is_contiguous():
        raise ValueError(f"kv_cache: contiguous uint8 [slots, {DQ}], got {kv_cache.dtype} {tuple(kv_cache.shape)}")
    if out.dtype != torch.bfloat16 or out.shape != (T, H, DV) or not out.is_contiguous():
        raise ValueError(f"out: contiguous bf16 {(T, H, DV)}, got {out.dtype} {tuple(out.shape)}")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or not page_table.is_contiguous():
        raise ValueError(f"page_table: contiguous int32 [R, width], got {page_table.dtype} {tuple(page_table.shape)}")
    if seq_lens is not None and (seq_lens.dtype is not torch.int32 or seq_lens.shape != (T,) or
                                 not seq_lens.is_contiguous()):
        raise ValueError(f"seq_lens: contiguous int32 {(T,)}, got {seq_lens.dtype} {tuple(seq_lens.shape)}")
    if reqs is not None and (reqs.dtype is not torch.int32 or reqs.shape != (T,) or not reqs.is_contiguous()):
        raise ValueError(f"reqs: contiguous int32 {(T,)}, got {reqs.dtype} {tuple(reqs.shape)}")
    if lse is not None and (lse.dtype is not torch.float32 or lse.shape != (T, H) or not lse.is_contiguous()):
        raise ValueError(f"lse: contiguous float32 {(T, H)}, got {lse.dtype} {tuple(lse.shape)}")
    rows, width = page_table.shape
    if reqs is None and rows < T:
        raise ValueError(f"page_table has {rows} rows for {T} query rows and no reqs")
    need = decode_workspace_bytes(T, H)
    if workspace is not None and (workspace.dtype != torch.uint8 or not workspace.is_contiguous() or
                                  workspace.numel() < need):
        raise ValueError(f"workspace: contiguous uint8 of {need} bytes or more")
    lib.check_device((q, kv_cache, page_table, out, seq_lens, indices, reqs, lse, workspace, ancestors), status,
                     stream)
    if workspace is None:
        workspace = lib.stream_scratch(q.device, need, stream)
    ptr = lambda t: None if t is None else t.data_ptr()
    ldq, head_stride, _ = q.stride()
    # a selection without columns has no address of its own (NULL means every visible token): any other one, never read
    listed = None if indices is None else indices.data_ptr() or page_table.data_ptr()
    if ancestors is not None:
        rc = so.ssb_mla_decode_tree(q.data_ptr(), int(e4m3), ldq, head_stride, T, H, kv_cache.data_ptr(),
                                    kv_cache.shape[0], page_table.data_ptr(), rows, width, ptr(reqs), ptr(seq_lens),
                                    ptr(ancestors), bmm1, bmm2, out.data_ptr(), ptr(lse), workspace.data_ptr(),
                                    workspace.numel(), ptr(status), lib.stream_ptr(stream))
        lib.check("ssb_mla_decode_tree", rc)
        return out
    rc = so.ssb_mla_decode(q.data_ptr(), int(e4m3), ldq, head_stride, T, H, kv_cache.data_ptr(),
                           kv_cache.shape[0], page_table.data_ptr(), rows, width, ptr(reqs), ptr(seq_lens),
                           listed, 0 if indices is None else indices.stride(0), n_idx or 0, bmm1, bmm2,
                           out.data_ptr(), ptr(lse), workspace.data_ptr(), workspace.numel(), ptr(status),
                           lib.stream_ptr(stream))
    lib.check("ssb_mla_decode", rc)
    return out


def cache_append(src: torch.Tensor, slots: torch.Tensor, kv_cache: torch.Tensor, k_scale: float = 1.0,
                 stream=None) -> None:
    """Rows of src bf16 [T, 576] into kv_cache uint8 [slots, 576] as e4m3(x / k_scale) at slots int64 [T] (< 0:
    skipped)."""
    so = lib.load()
    assert src.dtype == torch.bfloat16 and src.stride(1) == 1 and slots.dtype == torch.int64
    assert kv_cache.dtype == torch.uint8 and kv_cache.shape[1] == DQ
    rc = so.ssb_mla_cache_append(src.data_ptr(), src.stride(0), slots.data_ptr(), src.shape[0], kv_cache.data_ptr(),
                                 k_scale, lib.stream_ptr(stream))
    lib.check("ssb_mla_cache_append", rc)


def q_pack(lat: torch.Tensor, rows_pad: int, rope: torch.Tensor, rope_stride: int, T: int, q8: torch.Tensor,
           q_scale: float = 1.0, stream=None) -> torch.Tensor:
    """lat bf16 [64 * rows_pad, 512] (head-major absorbed queries), rope: bf16 rows whose head h slice starts at column
    h * rope_stride (64 values) -> q8 uint8 [T, 64, 576] = e4m3([lat | rope] / q_scale)."""
    so = lib.load()
    assert lat.dtype == torch.bfloat16 and lat.is_contiguous() and lat.shape == (HEADS * rows_pad, DV)
    assert rope.dtype == torch.bfloat16 and rope.stride(1) == 1
    assert q8.dtype == torch.uint8 and q8.is_contiguous() and q8.shape == (T, HEADS, DQ)
    rc = so.ssb_mla_q_pack(lat.data_ptr(), rows_pad, rope.data_ptr(), rope.stride(0), rope_stride, T, q8.data_ptr(),
                           q_scale, lib.stream_ptr(stream))
    lib.check("ssb_mla_q_pack", rc)
    return q8
