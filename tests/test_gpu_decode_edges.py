"""Calls of the decode-step operators at the edges of what they take, against float64 restatements with the bars of
tests/test_gpu_decode.py."""

import numpy as np
import pytest
import torch

from test_gpu_decode import BMM1, Cache, queries

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
