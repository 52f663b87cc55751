"""KDA prefill of one layer through the C ABI: the host side of `ssb_kda_prefill` / `ssb_kda_conv`.

Mirrors the reference's interface for this path: `kda_prefill_forward(self, qkv_proj_states, g1, beta,
core_attn_out)` (ssengine/model/pp_patch.py:215-244) with the layer's conv weight, `A_log`, `dt_bias` and lower bound
(`route_kda`, :247-256), the per-microbatch sequence table (first row, end row, state block, has initial state) of
`KdaPrefillMeta` (:189-197), and the layer's state pages (conv state [blocks, 3, 3P] bf16, recurrent state [blocks, H,
128, 128] fp32; pp_patch.py:223). `conv_qkv` mirrors `kda_conv.conv_qkv` (ssengine/model/kda_conv.py:146-164).
There is no fallback: without the CUDA library these calls raise.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import lib

HEAD_DIM = 128

def workspace_bytes(heads: int, T: int, R: int) -> int:
    """Device bytes of the chunk workspace of one prefill call (`ssb_kda_workspace_bytes`)."""
    n = lib.load().ssb_kda_workspace_bytes(heads, T, R)
    if n < 0:
        raise ValueError(f"bad KDA workspace query: heads={heads}, T={T}, R={R}")
    return int(n)




def seq_table(seqs, device) -> torch.Tensor:
    """[(first row, end row, state block, has initial state)] -> int32 [R, 4] on `device` (the reference's
    `KdaPrefillMeta.seqs`, kda_conv.tables' per-sequence rows)."""
    rows = [(int(s), int(e), int(b), int(bool(i))) for s, e, b, i in seqs]
    t = torch.tensor(rows, dtype=torch.int32).reshape(-1, 4)
    return t.to(device)


def _row_pitch(name: str, t: torch.Tensor, rows: int, cols: int) -> int:
    """The row pitch of a bf16 matrix of at least rows x cols with unit column stride; ValueError otherwise."""
    if t.dtype is torch.bfloat16 and t.dim() == 2:
        (n, m), (pitch, unit) = t.shape, t.stride()
        if n >= rows and m >= cols and unit == 1:
            return pitch
    raise ValueError(f"{name}: bf16 [{rows}, >= {cols}] with unit column stride, got {t.dtype} {tuple(t.shape)} strides "
                     f"{t.stride()}")


@dataclass
class KdaLayer:
    """One KDA layer's parameters on the device."""
    conv_weight: torch.Tensor     # bf16 [3 * H * 128, 4]
    a_log: torch.Tensor           # fp32 [H]
    dt_bias: torch.Tensor         # fp32 [H * 128]
    lower_bound: float = -5.0

    @property
    def heads(self) -> int:
        return self.a_log.numel()

    def c_struct(self, conv_state: torch.Tensor, rec_state: torch.Tensor) -> lib.KdaLayerC:
        w, a_log, dt_bias = self.conv_weight, self.a_log, self.dt_bias
        H = a_log.numel()
        C = 3 * H * HEAD_DIM
        assert w.dtype is torch.bfloat16 and w.shape == (C, 4) and w.is_contiguous() and a_log.dtype is torch.float32
        assert dt_bias.dtype is torch.float32 and dt_bias.numel() == H * HEAD_DIM
        assert a_log.is_contiguous() and dt_bias.is_contiguous()
        cs, rs = conv_state.stride(), rec_state.stride()
        (_, taps, cols), (_, heads, dv, dk) = conv_state.shape, rec_state.shape
        assert conv_state.dtype is torch.bfloat16 and taps == 3 and cols == C and cs[1:] == (C, 1)
        assert rec_state.dtype is torch.float32 and heads == H and dv == HEAD_DIM and dk == HEAD_DIM
        assert rs[1:] == (HEAD_DIM * HEAD_DIM, HEAD_DIM, 1) or (H == 1 and rs[2:] == (HEAD_DIM, 1))
        return lib.KdaLayerC(H, HEAD_DIM, w.data_ptr(), a_log.data_ptr(), dt_bias.data_ptr(), self.lower_bound,
                             HEAD_DIM ** -0.5, conv_state.data_ptr(), cs[0], rec_state.data_ptr(), rs[0])

    def prefill(self, qkv: torch.Tensor, g: torch.Tensor, beta: torch.Tensor, out: torch.Tensor, seqs: torch.Tensor,
                conv_state: torch.Tensor, rec_state: torch.Tensor, stream=None, status: torch.Tensor | None = None,
                workspace: torch.Tensor | None = None) -> None:
        """qkv bf16 [T, >= 3P] (q | k | v first), g bf16 [T, >= P] raw gate, beta bf16 [T, >= H] raw; writes out bf16
        [T, >= P] for the rows of `seqs` (int32 [R, 4] on the device) and updates both state pages in place. `status`
        (int32 [1] on the device) receives 4 if a bounded copy wait gave up. `workspace`: uint8 device tensor of at
        least `workspace_bytes(heads, T, R)` (default: the device's shared scratch)."""
        so = lib.load()
        T = qkv.shape[0]
        for t in (qkv, g, beta, out):
            assert t.dtype == torch.bfloat16 and t.stride(1) == 1 and t.shape[0] >= T
        assert seqs.dtype == torch.int32 and seqs.is_contiguous()
        need = workspace_bytes(self.heads, T, seqs.shape[0])
        if workspace is None:
            workspace = lib.scratch(qkv.device, need)
        assert workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.numel() >= need
        L = self.c_struct(conv_state, rec_state)
        rc = so.ssb_kda_prefill_ws(ctypes.byref(L), qkv.data_ptr(), qkv.stride(0), g.data_ptr(), g.stride(0),
                                   beta.data_ptr(), beta.stride(0), T, seqs.data_ptr(), seqs.shape[0], out.data_ptr(),
                                   out.stride(0), workspace.data_ptr(), workspace.numel(),
                                   None if status is None else status.data_ptr(), lib.stream_ptr(stream))
        lib.check("ssb_kda_prefill_ws", rc)

    def decode(self, qkv: torch.Tensor, g: torch.Tensor, beta: torch.Tensor, out: torch.Tensor, seqs: torch.Tensor,
               conv_state: torch.Tensor, rec_state: torch.Tensor, stream=None,
               status: torch.Tensor | None = None) -> torch.Tensor:
        """The recurrent form for new tokens: the arguments of `prefill`, the same state blocks, any number of rows a
        sequence (one in a decode step), token after token in one launch without a workspace. Rows outside every
        sequence are not written. `status` (int32 [1] on the device) receives 1 if a sequence reaches outside the rows
        or names a negative block (it is skipped). Returns `out`."""
        so = lib.load()
        H, T = self.a_log.numel(), qkv.shape[0]
        P = H * HEAD_DIM
        ldx, ldg = _row_pitch("qkv", qkv, T, 3 * P), _row_pitch("g", g, T, P)
        ldb, ldo = _row_pitch("beta", beta, T, H), _row_pitch("out", out, T, P)
        if seqs.dtype is not torch.int32 or seqs.dim() != 2 or seqs.shape[1] != 4 or not seqs.is_contiguous():
            raise ValueError(f"seqs: contiguous int32 [R, 4], got {seqs.dtype} {tuple(seqs.shape)}")
        lib.check_device((qkv, g, beta, out, seqs, conv_state, rec_state, self.conv_weight, self.a_log, self.dt_bias),
                         status, stream)
        L = self.c_struct(conv_state, rec_state)
        rc = so.ssb_kda_decode(ctypes.byref(L), qkv.data_ptr(), ldx, g.data_ptr(), ldg, beta.data_ptr(), ldb, T,
                               seqs.data_ptr(), seqs.shape[0], out.data_ptr(), ldo,
                               None if status is None else status.data_ptr(), lib.stream_ptr(stream))
        lib.check("ssb_kda_decode", rc)
        return out

    def conv_qkv(self, qkv: torch.Tensor, seqs: torch.Tensor, conv_state: torch.Tensor, rec_state: torch.Tensor,
                 stream=None):
        """The short conv alone -> q, k, v bf16 [T, P] each; the conv state blocks of `seqs` updated."""
        so = lib.load()
        T, P = qkv.shape[0], self.heads * HEAD_DIM
        out = torch.empty(3, T, P, dtype=torch.bfloat16, device=qkv.device)
        L = self.c_struct(conv_state, rec_state)
        rc = so.ssb_kda_conv(ctypes.byref(L), qkv.data_ptr(), qkv.stride(0), T, seqs.data_ptr(), seqs.shape[0],
                             out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), lib.stream_ptr(stream))
        lib.check("ssb_kda_conv", rc)
        return out[0], out[1], out[2]
