"""The refusals of the paged 4-bit cache's operators, each by the check that is meant: with a context that stays alive through the call, so none is refused for its handle."""
import ctypes as C
from importlib import import_module

import numpy as np
import pytest

import test_paged as T


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
