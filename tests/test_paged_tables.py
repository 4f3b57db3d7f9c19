"""Block tables and free lists with entries that name no page of the cache."""
import numpy as np
import pytest

import paged_oracle as P
from test_paged import cuda, on_torch  # noqa: F401  (a fixture)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 600])
@pytest.mark.parametrize("entry", [-1, 4000, 2 ** 31 - 1])
def test_reserve_tells_of_pages_that_are_not_in_the_cache(on_torch, n, entry):
    """From the free list, or the last page that a sequence holds: their tokens get no slot, all others the oracle's, and the next synchronising call tells."""
    import torch
    L, dev = on_torch
    page, n_pages = 16, 2000
    lens, add = np.full(n, 20, np.int32), np.full(n, 14, np.int32)                     # 12 of the 14 on the second page, 2 on a new one
    table = np.full((n, 4), -1, np.int32)
    table[:, :2] = np.arange(2 * n).reshape(n, 2)
    free = np.arange(n_pages - 1, -1, -1).astype(np.int32)
    top = n_pages - 2 * n                                                              # the list's top: page 2 n, then upwards
    for place in ("table", "list"):
        d_table, d_free = table.copy(), free.copy()
        if place == "table":
            d_table[1, 1] = entry
        else:
            d_free[top - 2] = entry                                                    # the second page to be taken: sequence 1's
        status, lens2, table2, top2, cu2, slots2 = P.reserve(lens, add, table, free, top, page, n * 14)
        table2[1, 1 if place == "table" else 2] = entry                                # what the list says is in the table, for attention to meet
        slots2[slice(14, 26) if place == "table" else slice(26, 28)] = -1
        args = cuda(lens), cuda(add), cuda(d_table), cuda(d_free), cuda(np.array([top], np.int32))
        cu, slots, st = (torch.full((k,), 77, dtype=torch.int32, device="cuda") for k in (n + 1, n * 14, 1))
        L.kv_reserve(dev, *args, page_size=page, lens_out=args[0], n_free_out=args[4], cu_rows=cu, slots=slots, status=st)
        with pytest.raises(L.LuminalB200Error) as e:
            dev.sync()
        assert e.value.code == -1
        dev.sync()
        assert status == 0 and st.item() == 0 and args[4].item() == top2
        for got, w in ((args[0], lens2), (args[2], table2), (cu, cu2), (slots, slots2)):
            assert np.array_equal(got.cpu().numpy(), w)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 600])
@pytest.mark.parametrize("entry", [-1, 2000, 2 ** 31 - 1])
def test_shrink_gives_nothing_back_where_a_table_names_no_page(on_torch, n, entry):
    L, dev = on_torch
    page, n_pages = 16, 2000
    lens = np.full(n, 40, np.int32)
    table = np.full((n, 4), -1, np.int32)
    table[:, :3] = np.arange(3 * n).reshape(n, 3)
    free = np.full(n_pages, -7, np.int32)
    top = n_pages - 3 * n
    free[:top] = np.arange(3 * n, n_pages)
    good, drop = table.copy(), np.full(n, 30, np.int32)
    for b, place in ((0, 1), (n - 1, 2)):
        table = good.copy()
        table[b, place] = entry
        d_lens, d_free, d_top = cuda(lens), cuda(free), cuda(np.array([top], np.int32))
        L.kv_shrink(dev, d_lens, cuda(drop), cuda(table), d_free, d_top, page_size=page, lens_out=d_lens, n_free_out=d_top)
        with pytest.raises(L.LuminalB200Error) as e:
            dev.sync()
        assert e.value.code == -1
        dev.sync()
        assert np.array_equal(d_lens.cpu().numpy(), lens) and d_top.item() == top and np.array_equal(d_free.cpu().numpy(), free)
    # an entry that stays in the table is not looked at
    table = good.copy()
    table[1, 0], table[1, 3] = entry, entry
    d_lens, d_free, d_top = cuda(lens), cuda(free), cuda(np.array([top], np.int32))
    want = P.shrink(lens, drop, table, free, top, page)
    L.kv_shrink(dev, d_lens, cuda(drop), cuda(table), d_free, d_top, page_size=page, lens_out=d_lens, n_free_out=d_top)
    dev.sync()
    assert np.array_equal(d_lens.cpu().numpy(), want[0]) and np.array_equal(d_free.cpu().numpy(), want[1]) and d_top.item() == want[2]
