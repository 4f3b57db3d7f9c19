"""Attention over the paged 4-bit cache where the ranges of values differ by orders of magnitude: between groups of 32 features, between the keys that rows of one tile see, down to the smallest halves."""
import numpy as np
import pytest

import paged_oracle as P
from test_paged import attend, check, cuda, on_torch, one_case  # noqa: F401  (a fixture)


def value_meta(pages, D):
    """[page, kv head, block, scale / minimum, group, places] of the values' halves."""
    return pages[..., 16 * D:].view(np.float16).reshape(*pages.shape[:3], 2, 2, D // 32, 16)[..., 1, :, :, :]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,G,new,lens", [(128, 4, (2, 1), (70, 600)), (128, 8, (5, 2), (70, 600)), (128, 4, (2, 1), (9000, 300)), (64, 8, (5, 2), (70, 600)), (256, 4, (2, 1), (70, 600)),
                                          (160, 1, (1, 1), (33, 700))])
@pytest.mark.parametrize("what", ["one group large", "one group large, the others small", "every group another size", "one group of the smallest halves", "a large key that some rows do not see",
                                  "a large key that takes no part", "one group constant, one large", "all of the smallest halves"])
def test_ranges_that_differ(on_torch, dtype, D, G, new, lens, what):
    import torch
    L, dev = on_torch
    rng = np.random.default_rng(31)
    scale, last = D ** -0.5, D // 32 - 1
    q, cu, lens, table, pages = one_case(rng, dtype, D=D, G=G, lens=lens, new=new)
    meta = value_meta(pages, D)
    places = P.places(D)[4]                                                 # of (token % 16, group) among 2 D halves; values' scales are the second quarter
    def of_key(b, pos):
        block = pages[table[b, pos // 16], :, 0, 16 * D:].view(np.float16)
        return block, places[pos % 16]
    if what == "one group large":
        meta[:, :, :, 0, last] = meta[:, :, :, 0, last].astype(np.float32) * 40000
    elif what == "one group large, the others small":
        meta[:] = meta.astype(np.float32) * 1e-3
        meta[:, :, :, 0, 1] = meta[:, :, :, 0, 1].astype(np.float32) * 4e7
    elif what == "every group another size":
        for g, f in enumerate([1e-4, 1.0, 300.0, 15000.0][:last + 1]):
            meta[:, :, :, :, g] = np.clip(meta[:, :, :, :, g].astype(np.float32) * f, -60000, 60000)
    elif what == "one group of the smallest halves":
        meta[:, :, :, 0, last] = rng.integers(1, 4, meta[:, :, :, 0, last].shape) * 2.0 ** -24
        meta[:, :, :, 1, last] = 0
    elif what == "a large key that some rows do not see":
        for b in range(2):
            block, p = of_key(b, int(lens[b]) - 1)
            block[:, p] = np.float16(40000)
    elif what == "a large key that takes no part":
        meta[:] = meta.astype(np.float32) * 1e-2
        for b in range(2):
            block, p = of_key(b, 5)
            block[:, p] = np.float16(30000)
            k = P.places(D)[3][5]
            block[:, k] = 0                                              # a key of -12 everywhere: its score is about 100 below the others
            block[:, k + D // 2] = np.float16(-12)
        q = q.abs()
    elif what == "one group constant, one large":
        meta[:, :, :, 0, 0] = 0
        meta[:, :, :, 0, 1] = meta[:, :, :, 0, 1].astype(np.float32) * 40000
    elif what == "all of the smallest halves":
        meta[:, :, :, 0] = rng.integers(1, 4, meta[:, :, :, 0].shape) * 2.0 ** -24
        meta[:, :, :, 1] = 0
    want, size = P.attention(q.float().cpu().numpy(), cu, lens, table, pages, 16, scale)
    out, ws = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(pages), 16, scale)
    dev.sync()
    if dtype == "bf16" and "smallest" in what:
        # a result below bf16's normal numbers has none to lose; the limit's own terms are relative
        assert np.abs(want).max() > 2.0 ** -126
    check(out, want, size, dtype)
    again, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(pages), 16, scale, ws=ws)
    dev.sync()
    assert torch.equal(out, again)
