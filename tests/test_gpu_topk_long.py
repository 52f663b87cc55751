"""The canonical top-k over long rows whose threshold value many columns hold, several rows a block, again and again: the
block's shared counters are read by every warp before they are used anew. Exact, against the oracle."""

import numpy as np
import pytest
import torch

from oracle import topk as otopk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width,k", [(9000, 512), (32768, 512), (20000, 2048)])
def test_long_rows_with_ties_at_the_threshold(cuda, width, k):
    from ssengine_b200 import lib

    so = lib.load()
    rng = np.random.default_rng(width + k)
    distinct = 24
    lg = rng.standard_normal((distinct, width)).astype(np.float32)
    for r in range(distinct):                              # ties: a few, more than the tie buffer, more than the list
        ties = (0, 2, 40, 700, 3000, 6000)[r % 6]
        if ties:
            at = rng.permutation(width)[:ties + k - min(ties, k) // 2 - 1]
            lg[r, at[:ties]] = 5.0
            lg[r, at[ties:]] = 6.0 + rng.random(at.size - ties)
    lg[5] = 0.25                                           # every column alike
    ks = rng.integers(0, 9, distinct).astype(np.int32)
    ke = (width - rng.integers(0, 9, distinct)).astype(np.int32)
    want = otopk.canonical_topk(lg, ks, ke, k)
    times = 200                                            # 4,800 rows: several a block
    order = np.concatenate([rng.permutation(distinct) for _ in range(times)])
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    pick = dev(order)
    logits, a, b = dev(lg)[pick].contiguous(), dev(ks)[pick].contiguous(), dev(ke)[pick].contiguous()
    expect = dev(want)[pick]
    for _ in range(5):
        out = torch.full((order.size, k), -7, dtype=torch.int32, device=cuda)
        lib.check("ssb_topk_canonical", so.ssb_topk_canonical(logits.data_ptr(), order.size, width, a.data_ptr(),
                                                              b.data_ptr(), k, out.data_ptr(), width, lib.stream_ptr()))
        torch.cuda.synchronize()
        assert torch.equal(out, expect)
