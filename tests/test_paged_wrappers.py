"""What the Python wrappers of the paged 4-bit cache make of arrays of other shapes, and which calls they and the library refuse."""
import numpy as np
import pytest

import paged_oracle as P
from test_paged import attend, check, cuda, on_torch, one_case  # noqa: F401  (a fixture)


class Flat:
    """A cache as the wrappers see one: shape, element size."""

    def __init__(self, *shape, size=1):
        self.shape, self.size = shape, size

    def element_size(self): return self.size


def test_kv_heads_of_a_cache(lib_built):
    from importlib import import_module
    heads = import_module("luminal_jl_b200.paged")._kv_heads
    each = lib_built.kv4_page_bytes(64, 5, 96)
    assert heads(Flat(7, 5, 4, 20 * 96), 64, 96) == 5
    assert heads(Flat(7, each), 64, 96) == 5 and heads(Flat(7, each // 4, size=4), 64, 96) == 5 and heads(Flat(1, each // 2, size=2), 64, 96) == 5
    for bad in (Flat(7, each - 20), Flat(7, 16), Flat(7)):
        with pytest.raises(ValueError):
            heads(bad, 64, 96)
    with pytest.raises(lib_built.LuminalB200Error):
        heads(Flat(7, each), 8, 96)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_over_pages_in_one_piece(on_torch, dtype):
    """A cache whose only axis besides its pages is their bytes, and one of words."""
    import torch
    L, dev = on_torch
    q, cu, lens, table, pages = one_case(np.random.default_rng(50), dtype, heads=3, page=32)
    want, size = P.attention(q.float().cpu().numpy(), cu, lens, table, pages, 32, 0.1)
    d = cuda(pages)
    for cache in (d, d.flatten(1), d.flatten(1).view(torch.int32)):
        out, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cache, 32, 0.1)
        dev.sync()
        check(out, want, size, dtype)
