"""The refusals of the paged 4-bit cache's operators, each by the check that is meant: with a context that stays alive through the call, so none is refused for its handle."""
from importlib import import_module

import numpy as np
import pytest

import test_paged as T
from test_paged import on_torch  # noqa: F401  (a fixture)


class Context(T.FakeContext):
    alive = []

    def __init__(self):
        super().__init__()
        Context.alive.append(self)


def cases(test, *names):
    """The parameters of a test of test_paged.py."""
    marks = [m for m in test.pytestmark if m.name == "parametrize"]
    return pytest.mark.parametrize(",".join(names), [m.args[1] for m in marks if m.args[0] == names[0]][0])


def refused(L, name, *args):
    """The message with which the library refuses a call."""
    with pytest.raises(L.LuminalB200Error) as e:
        import_module("luminal_jl_b200._lib").call(name, Context().handle, *args)
    assert e.value.code == -1 and "context" not in str(e.value)
    return str(e.value)


@cases(T.test_attention_refuses, "change")
def test_attention(lib_built, change):
    assert "kv4_attention" in refused(lib_built, "lmb200_kv4_attention", *T._args(**change))


@pytest.mark.parametrize("name", ["append", "read"])
@cases(T.test_store_refuses, "change")
def test_store(lib_built, name, change):
    a = dict(dtype=1, k=256, v=512, ks=256, vs=256, rows=3, heads=4, D=64, slots=256, pages=256, n_pages=9, page=16)
    a.update(change)
    if a["heads"] > 4:
        a.update(ks=a["heads"] * a["D"], vs=a["heads"] * a["D"])
    assert "kv4" in refused(lib_built, "lmb200_kv4_" + name, *a.values())


@cases(T.test_reserve_and_shrink_refuse, "change")
def test_reserve_and_shrink(lib_built, change):
    a = dict(n_seq=2, page=16, max_pages=4, n_pages=9, rows=3, lens=256, add=256, table=256, free=256, n_free=256, lens_out=256, n_free_out=256, cu=256, slots=256, status=256)
    a.update(change)
    assert "kv_reserve" in refused(lib_built, "lmb200_kv_reserve", *a.values())
    if not set(change) & {"rows", "cu", "slots", "status"}:
        assert "kv_shrink" in refused(lib_built, "lmb200_kv_shrink", *[v for k, v in a.items() if k not in ("rows", "cu", "slots", "status")])


@cases(T.test_verify_refuses, "change")
def test_verify(lib_built, change):
    a = dict(dtype=0, target=256, ts=100, draft=256, ds=100, vocab=100, rows=5, n_seq=2, cu=256, tokens=256, T=256, au=256, su=256, out=512, n_out=256, drop=256, ws=256, ws_bytes=1 << 30)
    a.update(change)
    assert "verify_drafts" in refused(lib_built, "lmb200_verify_drafts", *a.values())


def test_wrappers(lib_built, monkeypatch):
    """The calls of test_paged.py's wrapper tests: refused by what a wrapper or the library says of their arrays."""
    monkeypatch.setattr(T, "FakeContext", Context)
    paged = import_module("luminal_jl_b200.paged")
    lib = import_module("luminal_jl_b200._lib")
    said, check = [], lib.check

    def listen(status):
        try:
            check(status)
        except lib_built.LuminalB200Error as e:
            said.append(str(e))
            raise
    monkeypatch.setattr(paged._lib, "check", listen)
    T.test_wrappers_refuse_arrays_that_do_not_fit(lib_built)
    T.test_wrappers_refuse_arrays_of_another_gpu(lib_built)
    assert not [s for s in said if "context" in s or "CUDA" in s], said


@pytest.mark.parametrize("change", [dict(rows=(1 << 30) - 1, group=2), dict(rows=(1 << 30) - 7, group=2), dict(rows=2147483645 // 5, group=5, q_stride=1280, out_stride=1280)])
def test_attention_rows_whose_tiles_leave_32_bits(lib_built, change):
    """Rows times query heads fit 32 bits, rounded up to tiles of 8 or 16 they do not."""
    assert change["rows"] * change["group"] < 2 ** 31
    assert "rows for each of" in refused(lib_built, "lmb200_kv4_attention", *T._args(heads=1, max_pages=1, **change))


# rows of 512 elements of 2 bytes
@pytest.mark.parametrize("change", [dict(out_stride=1024), dict(out_stride=520), dict(out=4096 + 16), dict(out=4096 - 1008), dict(out=4096 + 1024), dict(out=4096 + 1040, q_stride=1000, out_stride=1000),
                                    dict(out=4096 + 2 * 1024, out_stride=1024), dict(rows=1, out=4096 + 512)])
def test_attention_out_over_q_in_part(lib_built, change):
    assert "lies over q" in refused(lib_built, "lmb200_kv4_attention", *T._args(**{**dict(q=4096, out=4096, rows=3), **change}))


@pytest.mark.parametrize("change", [dict(v=4096), dict(v=4096 + 256), dict(v=4096 + 768), dict(vs=512), dict(rows=1, v=4096 + 16), dict(v=4096 + 496, ks=500 + 4, vs=500 + 4)])
def test_read_into_the_same_memory(lib_built, change):
    a = dict(dtype=1, k=4096, v=4096, ks=256, vs=256, rows=3, heads=4, D=64, slots=256, pages=256, n_pages=9, page=16)
    a.update(change)
    assert "share memory" in refused(lib_built, "lmb200_kv4_read", *a.values())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_side_by_side_in_one_array(on_torch, dtype):
    """q and out, keys and values as columns of the rows of one array, and one behind the other: the bits of arrays of their own."""
    import torch
    L, dev = on_torch
    q, cu, lens, table, pages = T.one_case(np.random.default_rng(60), dtype, lens=(70, 300), new=(2, 4))
    args = T.cuda(cu), T.cuda(lens), T.cuda(table), T.cuda(pages)
    want, ws = T.attend(L, dev, q, *args, 16, 0.1)
    n = q[0].numel()
    for first, second in ((0, n), (n, 0), (8, n + 16)):
        both = torch.zeros(len(q), 2 * n + 64, dtype=q.dtype, device="cuda")
        a, b = (both[:, i:i + n].unflatten(1, q.shape[1:]) for i in (first, second))
        a.copy_(q)
        T.attend(L, dev, a, *args, 16, 0.1, ws=ws, out=b)
        dev.sync()
        assert torch.equal(b, want) and torch.equal(a, q)
    both = torch.cat([q, torch.zeros_like(q)])
    T.attend(L, dev, both[:len(q)], *args, 16, 0.1, ws=ws, out=both[len(q):])
    slots = T.cuda(np.r_[0:20].astype(np.int32))
    k, v = (torch.zeros(20, 2, 128, dtype=q.dtype, device="cuda") for _ in range(2))
    L.kv4_read(dev, k, v, slots, args[3], page_size=16)
    kv = torch.zeros(20, 4, 128, dtype=q.dtype, device="cuda")
    L.kv4_read(dev, kv[:, 2:], kv[:, :2], slots, args[3], page_size=16)
    dev.sync()
    assert torch.equal(both[len(q):], want) and torch.equal(kv[:, 2:], k) and torch.equal(kv[:, :2], v)
