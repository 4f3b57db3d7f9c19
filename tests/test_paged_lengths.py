"""Attention over the paged 4-bit cache with lengths that the block tables cannot hold."""
import numpy as np
import pytest

import paged_oracle as P
from test_paged import attend, check, cuda, on_torch, one_case  # noqa: F401  (a fixture)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [-4, 2 ** 31 - 1, 305])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_attention_leaves_a_sequence_out_whose_length_does_not_fit(on_torch, dtype, bad, which):
    """Its rows stay as they were, the other sequences' are right, and the next synchronising call tells."""
    L, dev = on_torch
    q, cu, lens, table, pages = one_case(np.random.default_rng(40), dtype, lens=(70, 300, 150), new=(2, 3, 1))
    assert table.shape[1] * 16 == 304
    want, size = P.attention(q.float().cpu().numpy(), cu, lens, table, pages, 16, 0.1)
    wrong = lens.copy()
    wrong[which] = bad
    out, ws = attend(L, dev, q, cuda(cu), cuda(wrong), cuda(table), cuda(pages), 16, 0.1)
    with pytest.raises(L.LuminalB200Error) as e:
        dev.sync()
    assert e.value.code == -1
    own = np.arange(cu[which], cu[which + 1])
    rest = np.setdiff1d(np.arange(cu[-1]), own)
    assert (out[own] == 7).all()
    check(out[rest], want[rest], size[rest], dtype)
    good, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(pages), 16, 0.1, ws=ws)
    dev.sync()
    check(good, want, size, dtype)
