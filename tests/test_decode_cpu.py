"""Refusals of the decode-step operators that need no GPU: the Python entry points' checks of types, shapes and strides
and the C entry points' own (called with addresses that are never read: every refusal comes before a launch)."""

import ctypes

import pytest
import torch

BMM1 = 256 ** -0.5


def attention_args(T=2, H=4, **over):
    a = dict(q=torch.zeros(T, H, 576, dtype=torch.bfloat16), kv_cache=torch.zeros(256, 576, dtype=torch.uint8),
             page_table=torch.zeros(T, 2, dtype=torch.int32), seq_lens=torch.ones(T, dtype=torch.int32), bmm1=BMM1,
             out=torch.zeros(T, H, 512, dtype=torch.bfloat16))
    a.update(over)
    return a


@pytest.mark.parametrize("over", [
    dict(q=torch.zeros(2, 4, 576)),
    dict(q=torch.zeros(2, 4, 512, dtype=torch.bfloat16)),
    dict(q=torch.zeros(2, 4 * 576, dtype=torch.bfloat16)),
    dict(q=torch.zeros(2, 576, 4, dtype=torch.bfloat16).transpose(1, 2)),
    dict(kv_cache=torch.zeros(256, 576, dtype=torch.bfloat16)),
    dict(kv_cache=torch.zeros(256, 640, dtype=torch.uint8)[:, :576]),
    dict(out=torch.zeros(2, 4, 576, dtype=torch.bfloat16)),
    dict(out=torch.zeros(2, 4, 512)),
    dict(page_table=torch.zeros(2, 2, dtype=torch.int64)),
    dict(page_table=torch.zeros(1, 2, dtype=torch.int32)),
    dict(seq_lens=torch.ones(3, dtype=torch.int32)),
    dict(seq_lens=torch.ones(2, dtype=torch.int64)),
    dict(reqs=torch.zeros(1, dtype=torch.int32)),
    dict(lse=torch.zeros(2, 4, dtype=torch.bfloat16)),
    dict(workspace=torch.zeros(64, dtype=torch.uint8)),
    dict(workspace=torch.zeros(1 << 10)),
])
def test_attention_refuses(over):
    from ssengine_b200 import mla

    with pytest.raises(ValueError):
        mla.decode(**attention_args(**over))


@pytest.mark.parametrize("over", [
    dict(indices=torch.zeros(2, 8, dtype=torch.int64)),
    dict(indices=torch.zeros(1, 8, dtype=torch.int32)),
    dict(indices=torch.zeros(8, 2, dtype=torch.int32).t()),
    dict(indices=torch.zeros(2, 8, dtype=torch.int32), n_idx=9),
    dict(indices=torch.zeros(2, 8, dtype=torch.int32), n_idx=-1),
])
def test_selected_attention_refuses(over):
    from ssengine_b200 import mla

    with pytest.raises(ValueError):
        mla.decode_selected(**attention_args(**over))


def test_heads_and_workspace_sizes():
    from ssengine_b200 import mla

    assert mla.decode_workspace_bytes(1, 64) < mla.decode_workspace_bytes(1, 128)
    assert mla.decode_workspace_bytes(1, 1) == mla.decode_workspace_bytes(1, 64)
    assert mla.decode_workspace_bytes(0, 64) <= mla.decode_workspace_bytes(4096, 64)
    for T, H in ((1, 0), (1, 129), (-1, 64)):
        with pytest.raises(ValueError):
            mla.decode_workspace_bytes(T, H)
    with pytest.raises(ValueError):
        mla.decode(**attention_args(H=129))


def c_attention(so, **over):
    a = dict(q=1 << 12, e4m3=0, ldq=4 * 576, hs=576, T=2, H=4, kv=1 << 12, rows=256, table=1 << 12, R=2, width=2,
             reqs=None, seq=1 << 12, idx=None, ldi=0, n=0, out=1 << 12, ws=1 << 12, wsb=1 << 40)
    a.update(over)
    return so.ssb_mla_decode(a["q"], a["e4m3"], a["ldq"], a["hs"], a["T"], a["H"], a["kv"], a["rows"], a["table"],
                             a["R"], a["width"], a["reqs"], a["seq"], a["idx"], a["ldi"], a["n"], 0.1, 1.0, a["out"],
                             None, a["ws"], a["wsb"], None, None)


@pytest.mark.parametrize("over,rc", [
    (dict(q=None), 1), (dict(q=(1 << 12) + 8), 1), (dict(ldq=4 * 576 + 4), 1), (dict(hs=570), 1), (dict(e4m3=2), 1),
    (dict(e4m3=1, hs=584), 1), (dict(T=-1), 1), (dict(H=0), 1), (dict(H=129), 1), (dict(kv=None), 1),
    (dict(kv=(1 << 12) + 4), 1), (dict(rows=-1), 1), (dict(table=None), 1), (dict(R=0), 1), (dict(R=1), 1),
    (dict(width=0), 1), (dict(seq=None), 1), (dict(idx=1 << 12, ldi=4, n=5), 1), (dict(idx=1 << 12, ldi=4, n=-1), 1),
    (dict(out=None), 1), (dict(out=(1 << 12) + 8), 1), (dict(ws=None), 1), (dict(ws=(1 << 12) + 16), 1),
    (dict(wsb=1024), 3),
])
def test_c_attention_refuses(over, rc):
    from ssengine_b200 import lib

    assert c_attention(lib.load(), **over) == rc


def test_c_attention_of_no_rows():
    from ssengine_b200 import lib

    assert c_attention(lib.load(), T=0) == 0


def kda_args(H=2, T=3, **over):
    P = H * 128
    bf = dict(dtype=torch.bfloat16)
    a = dict(qkv=torch.zeros(T, 3 * P, **bf), g=torch.zeros(T, P, **bf), beta=torch.zeros(T, H, **bf),
             out=torch.zeros(T, P, **bf), seqs=torch.zeros(1, 4, dtype=torch.int32),
             conv_state=torch.zeros(2, 3, 3 * P, **bf), rec_state=torch.zeros(2, H, 128, 128))
    a.update(over)
    return a


@pytest.mark.parametrize("over", [
    dict(qkv=torch.zeros(3, 768)),
    dict(qkv=torch.zeros(3, 760, dtype=torch.bfloat16)),
    dict(qkv=torch.zeros(768, 3, dtype=torch.bfloat16).t()),
    dict(g=torch.zeros(2, 256, dtype=torch.bfloat16)),
    dict(beta=torch.zeros(3, 1, dtype=torch.bfloat16)),
    dict(out=torch.zeros(3, 128, dtype=torch.bfloat16)),
    dict(out=torch.zeros(3, 256)),
    dict(seqs=torch.zeros(1, 4, dtype=torch.int64)),
    dict(seqs=torch.zeros(4, dtype=torch.int32)),
    dict(seqs=torch.zeros(1, 3, dtype=torch.int32)),
])
def test_kda_refuses(over):
    from ssengine_b200.kda import KdaLayer

    L = KdaLayer(torch.zeros(768, 4, dtype=torch.bfloat16), torch.zeros(2), torch.zeros(256))
    with pytest.raises(ValueError):
        L.decode(**kda_args(**over))


@pytest.mark.parametrize("over,rc", [
    (dict(x=None), 1), (dict(x=(1 << 12) + 2), 1), (dict(ldx=769), 1), (dict(ldx=766), 1), (dict(g=None), 1),
    (dict(ldg=254), 1), (dict(ldg=257), 1), (dict(beta=None), 1), (dict(ldb=1), 1), (dict(T=-1), 1),
    (dict(seqs=None), 1), (dict(seqs=(1 << 12) + 8), 1), (dict(R=-1), 1), (dict(out=None), 1), (dict(ldo=255), 1),
    (dict(rec=None), 1), (dict(rec=(1 << 12) + 8), 1), (dict(rs=2 * 128 * 128 + 2), 1), (dict(rs=128 * 128), 1),
    (dict(conv=None), 1), (dict(cs=9 * 256 - 2), 1), (dict(cs=9 * 256 + 1), 1), (dict(w=None), 1), (dict(dim=64), 1),
    (dict(R=0), 0),
])
def test_c_kda_refuses(over, rc):
    from ssengine_b200 import lib

    a = dict(x=1 << 12, ldx=768, g=1 << 12, ldg=256, beta=1 << 12, ldb=2, T=3, seqs=1 << 12, R=1, out=1 << 12, ldo=256,
             rec=1 << 12, rs=2 * 128 * 128, conv=1 << 12, cs=9 * 256, w=1 << 12, dim=128)
    a.update(over)
    L = lib.KdaLayerC(2, a["dim"], a["w"], 1 << 12, 1 << 12, -5.0, 128 ** -0.5, a["conv"], a["cs"], a["rec"], a["rs"])
    assert lib.load().ssb_kda_decode(ctypes.byref(L), a["x"], a["ldx"], a["g"], a["ldg"], a["beta"], a["ldb"], a["T"],
                                     a["seqs"], a["R"], a["out"], a["ldo"], None, None) == rc


def test_stage_and_block_refuse_unknown_forms():
    from ssengine_b200.layers import DsaAttention
    from ssengine_b200.stage import StageModel

    with pytest.raises(ValueError):
        object.__new__(StageModel).run(None, None, decode="sparse")
    with pytest.raises(ValueError):
        DsaAttention.forward(object.__new__(DsaAttention), *[None] * 12, decode=("sparse", None, None))
