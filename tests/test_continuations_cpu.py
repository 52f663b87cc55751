"""Refusals of the operators for several continuations of a request that need no GPU: the Python entry points' checks and
the C entry points' own (called with addresses that are never read: every refusal comes before a launch); tree masks."""

import ctypes

import pytest
import torch

from test_decode_cpu import BMM1, attention_args, kda_args

BF = dict(dtype=torch.bfloat16)
I32 = dict(dtype=torch.int32)


def test_tree_masks():
    from ssengine_b200 import mla

    masks, depths = mla.tree_masks([-1, 0, 0, 1, -1, 3])
    assert masks.tolist() == [1, 3, 5, 11, 16, 43] and depths.tolist() == [0, 1, 1, 2, 0, 3]
    masks, depths = mla.tree_masks(range(-1, 63))
    assert masks[63].item() == -1 and masks[62].item() == 2 ** 63 - 1 and depths[63].item() == 63
    assert mla.tree_masks([])[0].shape == (0,)
    for bad in ([0], [-1, 1], [-1, -2], list(range(-1, 64))):
        with pytest.raises(ValueError):
            mla.tree_masks(bad)


@pytest.mark.parametrize("over", [
    dict(ancestors=torch.ones(2, **I32)),
    dict(ancestors=torch.ones(3, dtype=torch.int64)),
    dict(ancestors=torch.ones(4, dtype=torch.int64)[::2]),
    dict(seq_lens=None),
    dict(seq_lens=torch.ones(2, dtype=torch.int64)),
    dict(page_table=torch.zeros(1, 2, **I32)),
    dict(out=torch.zeros(2, 4, 512)),
])
def test_tree_attention_refuses(over):
    from ssengine_b200 import mla

    with pytest.raises(ValueError):
        mla.decode_tree(**attention_args(**{"ancestors": torch.ones(2, dtype=torch.int64), **over}))


@pytest.mark.parametrize("over,rc", [
    (dict(anc=None), 1), (dict(anc=(1 << 12) + 4), 1), (dict(seq=None), 1), (dict(q=None), 1), (dict(H=129), 1),
    (dict(R=1), 1), (dict(width=0), 1), (dict(e4m3=2), 1), (dict(wsb=1024), 3), (dict(T=0, anc=None), 0),
])
def test_c_tree_attention_refuses(over, rc):
    from ssengine_b200 import lib

    a = dict(q=1 << 12, e4m3=0, ldq=4 * 576, hs=576, T=2, H=4, kv=1 << 12, rows=256, table=1 << 12, R=2, width=2,
             seq=1 << 12, anc=1 << 12, out=1 << 12, ws=1 << 12, wsb=1 << 40)
    a.update(over)
    assert lib.load().ssb_mla_decode_tree(a["q"], a["e4m3"], a["ldq"], a["hs"], a["T"], a["H"], a["kv"], a["rows"],
                                          a["table"], a["R"], a["width"], None, a["seq"], a["anc"], 0.1, 1.0, a["out"],
                                          None, a["ws"], a["wsb"], None, None) == rc


def layer():
    from ssengine_b200.kda import KdaLayer

    return KdaLayer(torch.zeros(768, 4, **BF), torch.zeros(2), torch.zeros(256))


@pytest.mark.parametrize("over", [
    dict(parents=torch.zeros(3, dtype=torch.int64)),
    dict(parents=torch.zeros(2, **I32)),
    dict(parents=torch.zeros(6, **I32)[::2]),
    dict(max_nodes=0),
    dict(max_nodes=65),
    dict(qkv=torch.zeros(3, 768)),
    dict(out=torch.zeros(3, 256)),
    dict(seqs=torch.zeros(1, 3, **I32)),
])
def test_tree_recurrence_refuses(over):
    with pytest.raises(ValueError):
        layer().decode_tree(**kda_args(**{"parents": torch.zeros(3, **I32), **over}))


@pytest.mark.parametrize("over", [
    dict(rows=torch.zeros(3, dtype=torch.int64)),
    dict(rows=torch.zeros(3, 1, **I32)),
    dict(rows=torch.zeros(6, **I32)[::2]),
    dict(g=torch.zeros(2, 256, **BF)),
    dict(beta=torch.zeros(3, 1, **BF)),
    dict(seqs=torch.zeros(1, 4, dtype=torch.int64)),
])
def test_advance_refuses(over):
    a = kda_args(**{"rows": torch.zeros(3, **I32), **over})
    a.pop("out")
    with pytest.raises(ValueError):
        layer().advance(**a)


def c_layer(a):
    from ssengine_b200 import lib

    return ctypes.byref(lib.KdaLayerC(2, a["dim"], a["w"], 1 << 12, 1 << 12, -5.0, 128 ** -0.5, a["conv"], a["cs"], a["rec"],
                                      a["rs"]))


C_KDA = dict(x=1 << 12, ldx=768, g=1 << 12, ldg=256, beta=1 << 12, ldb=2, T=3, seqs=1 << 12, R=1, out=1 << 12, ldo=256,
             rec=1 << 12, rs=2 * 128 * 128, conv=1 << 12, cs=9 * 256, w=1 << 12, dim=128, parents=1 << 12, nodes=64,
             rows=1 << 12, n=3)


@pytest.mark.parametrize("over,rc", [
    (dict(parents=None), 1), (dict(parents=(1 << 12) + 2), 1), (dict(nodes=0), 1), (dict(nodes=65), 1), (dict(out=None), 1),
    (dict(ldo=255), 1), (dict(x=None), 1), (dict(ldx=769), 1), (dict(rec=None), 1), (dict(seqs=None), 1), (dict(dim=64), 1),
    (dict(T=-1), 1), (dict(R=0), 0), (dict(T=0, R=0, x=None, g=None, beta=None, out=None, parents=None, seqs=None), 0),
])
def test_c_tree_recurrence_refuses(over, rc):
    from ssengine_b200 import lib

    a = {**C_KDA, **over}
    assert lib.load().ssb_kda_decode_tree(c_layer(a), a["x"], a["ldx"], a["g"], a["ldg"], a["beta"], a["ldb"], a["T"],
                                          a["parents"], a["seqs"], a["R"], a["nodes"], a["out"], a["ldo"], None,
                                          None) == rc


@pytest.mark.parametrize("over,rc", [
    (dict(rows=None), 1), (dict(rows=(1 << 12) + 2), 1), (dict(n=-1), 1), (dict(x=None), 1), (dict(ldg=257), 1),
    (dict(rec=(1 << 12) + 8), 1), (dict(cs=9 * 256 + 1), 1), (dict(seqs=None), 1), (dict(R=0), 0),
])
def test_c_advance_refuses(over, rc):
    from ssengine_b200 import lib

    a = {**C_KDA, **over}
    assert lib.load().ssb_kda_advance(c_layer(a), a["x"], a["ldx"], a["g"], a["ldg"], a["beta"], a["ldb"], a["T"],
                                      a["rows"], a["n"], a["seqs"], a["R"], None, None) == rc


@pytest.mark.parametrize("views,lists", [
    ([], None),
    ([torch.zeros(4, 32, dtype=torch.uint8)], [0, 0]),
    ([torch.zeros(4, 32, dtype=torch.uint8)], [-1]),
    ([torch.zeros(4, 24, dtype=torch.uint8)], None),
    ([torch.zeros(4, 40, dtype=torch.uint8)[:, :32]], None),                       # rows 40 bytes apart
    ([torch.zeros(32, 4).t()], None),
    ([torch.zeros(4, 64, dtype=torch.uint8).as_strided((4, 32), (16, 1))], None),  # rows over one another
    ([torch.zeros(0, 32, dtype=torch.uint8)], None),
    ([torch.zeros(4, 0, dtype=torch.uint8)], None),
    ([torch.zeros(64, dtype=torch.uint8)[8:40].view(1, 32)], None),
    ([torch.zeros(4, 32, dtype=torch.uint8)] * 81, None),
])
def test_mover_refuses_views(views, lists):
    from ssengine_b200.kvpages import RowMover

    with pytest.raises(ValueError):
        RowMover(views, lists)


@pytest.mark.parametrize("src,dst", [
    (torch.zeros(1, 2, 3, dtype=torch.int64), torch.zeros(1, 2, 3, dtype=torch.int64)),
    (torch.zeros(1, 2, 3, **I32), torch.zeros(1, 2, 4, **I32)),
    (torch.zeros(2, 3, **I32), torch.zeros(2, 3, **I32)),                          # two lists
    (torch.zeros(1, 2, 3, **I32), torch.zeros(1, 2, 3, **I32)),
    (torch.zeros(2, 2, 65, **I32), torch.zeros(2, 2, 65, **I32)),
    (torch.zeros(2, 3, 2, **I32).transpose(1, 2), torch.zeros(2, 2, 3, **I32)),
])
def test_mover_refuses_lists(src, dst):
    from ssengine_b200.kvpages import RowMover

    v = torch.zeros(4, 32, dtype=torch.uint8)
    with pytest.raises(ValueError):
        RowMover([v, v], [0, 1])(src, dst)


def test_stage_moves_refuse_shapes():
    from ssengine_b200.kvpages import StageKv

    kv = StageKv([2, 3], lambda i: i == 3, 2, 2, "cpu")
    with pytest.raises(ValueError):
        kv.move_states(torch.zeros(5, 1, 1, **I32), torch.zeros(5, 1, 1, **I32))
    for f in (kv.move_pages, kv.move_tokens):
        with pytest.raises(ValueError):
            f(torch.zeros(1, 1, 1, **I32), torch.zeros(1, 1, 1, **I32))


@pytest.mark.parametrize("over,rc", [
    (dict(n_views=-1), 1), (dict(n_views=81), 1), (dict(views=None), 1), (dict(src=None), 1), (dict(dst=None), 1),
    (dict(src=(1 << 12) + 2), 1), (dict(lists=-1), 1), (dict(groups=-1), 1), (dict(n=-1), 1), (dict(n=65), 1),
    (dict(base=None), 1), (dict(base=(1 << 12) + 8), 1), (dict(stride=40), 1), (dict(stride=16), 1), (dict(nbytes=40), 1),
    (dict(nbytes=0), 1), (dict(rows=-1), 1), (dict(list=1), 1), (dict(list=-1), 1), (dict(nbytes=1 << 45, stride=1 << 45), 1),
    (dict(groups=1 << 31), 1), (dict(n_views=0), 0), (dict(groups=0), 0), (dict(n=0), 0),
])
def test_c_move_refuses(over, rc):
    from ssengine_b200 import lib

    a = dict(n_views=1, views=True, src=1 << 12, dst=1 << 12, lists=1, groups=1, n=2, base=1 << 12, stride=32, nbytes=32,
             rows=4, list=0)
    a.update(over)
    v = (lib.MoveViewC * 1)(lib.MoveViewC(a["base"], a["stride"], a["nbytes"], a["rows"], a["list"]))
    assert lib.load().ssb_move_rows(v if a["views"] else None, a["n_views"], a["src"], a["dst"], a["lists"], a["groups"],
                                    a["n"], None, None) == rc


def beam_args(**over):
    a = dict(logits=torch.zeros(6, 50), scores=torch.zeros(2, 3), k=4)
    a.update(over)
    return a


@pytest.mark.parametrize("over", [
    dict(logits=torch.zeros(6, 50, dtype=torch.float16)),
    dict(logits=torch.zeros(5, 50)),
    dict(logits=torch.zeros(50, 6).t()),
    dict(logits=torch.zeros(2, 3, 50)),
    dict(scores=torch.zeros(6)),
    dict(scores=torch.zeros(2, 3, dtype=torch.float64)),
    dict(scores=torch.zeros(3, 2).t()),
    dict(k=0),
    dict(k=65),
    dict(finished=torch.zeros(2, 3)),
    dict(finished=torch.zeros(3, 2, dtype=torch.bool)),
    dict(pad=50),
    dict(pad=-1),
    dict(out=(torch.zeros(2, 4), torch.zeros(2, 4, **I32), torch.zeros(2, 4, **I32))),
    dict(out=(torch.zeros(2, 3), torch.zeros(2, 4, **I32), torch.zeros(2, 4, dtype=torch.int64))),
    dict(workspace=torch.zeros(8, dtype=torch.uint8)),
    dict(workspace=torch.zeros(1 << 16)),
    dict(logits=torch.zeros(2 * 65, 50), scores=torch.zeros(2, 65)),
    dict(logits=torch.zeros(6, 0)),
])
def test_beam_refuses(over):
    from ssengine_b200 import beam

    with pytest.raises(ValueError):
        beam.select(**beam_args(**over))


@pytest.mark.parametrize("over,rc", [
    (dict(x=None), 1), (dict(x=(1 << 12) + 2), 1), (dict(bf16=2), 1), (dict(ld=49), 1), (dict(G=-1), 1), (dict(B=0), 1),
    (dict(B=65), 1), (dict(V=0), 1), (dict(scores=None), 1), (dict(pad=50), 1), (dict(pad=-1), 1), (dict(k=0), 1),
    (dict(k=65), 1), (dict(os=None), 1), (dict(op=None), 1), (dict(ot=None), 1), (dict(ot=(1 << 12) + 4), 1),
    (dict(ws=None), 1), (dict(ws=(1 << 12) + 16), 1), (dict(wsb=64), 3), (dict(G=0, x=None), 0),
])
def test_c_beam_refuses(over, rc):
    from ssengine_b200 import lib

    a = dict(x=1 << 12, bf16=0, ld=50, G=2, B=3, V=50, scores=1 << 12, fin=None, pad=0, k=4, os=1 << 12, op=1 << 12,
             ot=1 << 12, ws=1 << 12, wsb=1 << 30)
    a.update(over)
    assert lib.load().ssb_beam_select(a["x"], a["bf16"], a["ld"], a["G"], a["B"], a["V"], a["scores"], a["fin"], a["pad"],
                                      a["k"], a["os"], a["op"], a["ot"], a["ws"], a["wsb"], None) == rc


def test_beam_workspace_sizes():
    from ssengine_b200 import beam, lib

    assert beam.workspace_bytes(1, 4, 151552, 4) > 0
    assert beam.workspace_bytes(64, 8, 151552, 8) < 1 << 22
    so = lib.load()
    for bad in ((-1, 4, 100, 4), (1, 0, 100, 4), (1, 4, 0, 4), (1, 4, 1 << 31, 4), (1, 4, 100, 65)):
        assert so.ssb_beam_workspace_bytes(*bad) == -1


def test_beam_rows_are_cut_into_what_runs_at_once():
    """A part's keys and its sum (16 bytes) for each CTA: no more than 3 on each of 148 SMs unless the rows alone are more."""
    from ssengine_b200 import beam

    for G, B, k in ((1, 4, 4), (2, 4, 4), (4, 8, 8), (16, 4, 4), (16, 8, 8), (37, 4, 1), (64, 8, 8), (148, 4, 16)):
        most = max(148 * 3, G * B)
        assert beam.workspace_bytes(G, B, 151552, k) <= most * (8 * k + 16) + 512, (G, B, k)


@pytest.mark.parametrize("over", [
    dict(k=(1 << 32) + 4), dict(k=-(1 << 32) + 4), dict(out=(torch.zeros(2, 4), torch.zeros(2, 4, **I32))),
])
def test_beam_refuses_what_its_arguments_cannot_hold(over):
    """A k that 32 bits cut to a fair one, outputs that are not three."""
    from ssengine_b200 import beam

    with pytest.raises(ValueError):
        beam.select(**beam_args(**over))
    if "k" in over:
        with pytest.raises(ValueError):
            beam.workspace_bytes(2, 3, 50, over["k"])
