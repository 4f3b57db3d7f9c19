"""The paged 4-bit cache, its block tables and the verification of drafts against a 64-bit NumPy oracle: every kind of size and
mask where they can go wrong, refusals, and a serving loop of all of them together.

Tolerances.  Tables, slots, tokens, levels, scales and minima are equal.  kv4_read gives float32(m + n s), rounded once, and bf16 of that.  Attention: let A = sum p (|m| + s n) and
X = 1 + the largest sum |scale q| (|m| + s n) of a row (the oracle's `size` is A X).  Scores are float32 sums of at most 2 D exact products and a 22-bit split of q: off by at most
2^-18 X, which changes a weight by as much; weights are split to 22 bits (float32) or rounded twice to 11 bits (bf16: 2 x 2^-11), and sums of n terms in float32 add 2^-18.  So float32:
4 x 2^-18 A X; bf16: 2^-10 A + the same, and 2^-8 |out| for the result's own rounding (2^-24 for float32 is inside the first term)."""
import ctypes as C

import numpy as np
import pytest

import paged_oracle as P


# ---------------------------------------------------------------------------------------------------------------------
# without a GPU
# ---------------------------------------------------------------------------------------------------------------------
def test_page_bytes(lib_built):
    L = lib_built
    assert L.kv4_page_bytes(64, 8, 128) == 8 * 4 * 20 * 128
    assert L.kv4_page_bytes(16, 1, 32) == 640
    for page, heads, dim in ((0, 8, 128), (48, 8, 128), (512, 8, 128), (64, 0, 128), (64, 8, 0), (64, 8, 80), (64, 8, 288), (-16, 8, 64)):
        with pytest.raises(L.LuminalB200Error):
            L.kv4_page_bytes(page, heads, dim)
    with pytest.raises(L.LuminalB200Error):
        L.verify_drafts_workspace(-1)


@pytest.mark.parametrize("D", [32, 96, 256])
def test_a_block_has_a_place_for_everything(D):
    kb, vb, shift, km, vm = P.places(D)
    seen = np.zeros((20 * D, 2), int)
    for b in (kb, vb):
        np.add.at(seen, (b.ravel(), shift.ravel() // 4), 1)
    for m in (km, km + D // 2, vm, vm + D // 2):
        for half in (0, 1):
            np.add.at(seen, (16 * D + 2 * m.ravel() + half, 0), 1)
            np.add.at(seen, (16 * D + 2 * m.ravel() + half, 1), 1)
    assert (seen == 1).all()


def test_oracle_quantises_to_the_nearest_level():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 64)).astype(np.float32)
    n, s, m = P.quantise(x)
    y = P.values(n, s, m)
    # the nearest of 16 levels: half a step, and what rounding s and m to 11 bits moves the top and bottom levels by
    step = s.astype(np.float64).repeat(32, -1)
    assert (np.abs(y - x) <= step / 2 + 2.0 ** -11 * (np.abs(m).astype(np.float64).repeat(32, -1) + 15 * step)).all()
    c = np.full((1, 32), 0.3, np.float32)
    n, s, m = P.quantise(c)
    assert (s == 0).all() and (n == 0).all() and (P.values(n, s, m) == np.float16(0.3)).all()


class FakeContext:
    """Memory that a call takes for a context: enough for calls that are refused before they touch the device."""

    def __init__(self):
        self.mem = (C.c_uint32 * 4096)()
        self.mem[0] = 0x4C4D4231
        self.handle = C.c_uint64(C.addressof(self.mem))


def _args(**change):
    a = dict(dtype=1, q=256, q_stride=512, out=256, out_stride=512, rows=3, n_seq=2, cu=256, lens=256, table=256, max_pages=4, pages=256, n_pages=9, page=16, heads=2, group=2,
             D=128, scale=0.1, window=0, ws=256, ws_bytes=1 << 40)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change", [dict(dtype=2), dict(q=0), dict(out=0), dict(cu=0), dict(lens=0), dict(table=0), dict(pages=0), dict(ws=0), dict(q_stride=511), dict(out_stride=500),
                                    dict(q_stride=516), dict(q=258), dict(out=264 + 4), dict(rows=-1), dict(n_seq=0), dict(n_seq=8193), dict(max_pages=0),
                                    dict(max_pages=1 << 28), dict(n_pages=0), dict(n_pages=1 << 28), dict(page=24), dict(heads=0), dict(group=0), dict(group=1 << 20), dict(D=64 + 16),
                                    dict(D=512), dict(window=-1), dict(ws_bytes=0), dict(ws=260), dict(max_pages=(1 << 26) + 1), dict(rows=(1 << 30) + 1),
                                    dict(rows=1 << 29, group=4, q_stride=1024, out_stride=1024)])
def test_attention_refuses(lib_built, change):
    from importlib import import_module
    _lib = import_module("luminal_jl_b200._lib")
    ctx = FakeContext()
    with pytest.raises(lib_built.LuminalB200Error) as e:
        _lib.call("lmb200_kv4_attention", ctx.handle, *_args(**change))
    assert e.value.code == -1


@pytest.mark.parametrize("name", ["lmb200_kv4_append", "lmb200_kv4_read"])
@pytest.mark.parametrize("change", [dict(dtype=2), dict(k=0), dict(v=0), dict(ks=255), dict(vs=260), dict(k=258), dict(rows=-1), dict(heads=0), dict(heads=70000), dict(D=48), dict(D=0),
                                    dict(slots=0), dict(pages=0), dict(pages=8), dict(n_pages=0), dict(page=8), dict(rows=(1 << 31) - 1, heads=60000)])
def test_store_refuses(lib_built, name, change):
    from importlib import import_module
    _lib = import_module("luminal_jl_b200._lib")
    a = dict(dtype=1, k=256, v=256, ks=256, vs=256, rows=3, heads=4, D=64, slots=256, pages=256, n_pages=9, page=16)
    a.update(change)
    if a["heads"] > 4:
        a.update(ks=a["heads"] * a["D"], vs=a["heads"] * a["D"])
    with pytest.raises(lib_built.LuminalB200Error) as e:
        _lib.call(name, FakeContext().handle, *a.values())
    assert e.value.code == -1


@pytest.mark.parametrize("change", [dict(n_seq=0), dict(n_seq=8193), dict(page=20), dict(max_pages=0), dict(n_pages=0), dict(n_pages=1 << 28), dict(rows=-1), dict(lens=0), dict(add=0),
                                    dict(table=0), dict(free=0), dict(n_free=0), dict(lens_out=0), dict(n_free_out=0), dict(cu=0), dict(slots=0), dict(status=0), dict(max_pages=(1 << 26) + 1),
                                    dict(rows=(1 << 30) + 1)])
def test_reserve_and_shrink_refuse(lib_built, change):
    from importlib import import_module
    _lib = import_module("luminal_jl_b200._lib")
    a = dict(n_seq=2, page=16, max_pages=4, n_pages=9, rows=3, lens=256, add=256, table=256, free=256, n_free=256, lens_out=256, n_free_out=256, cu=256, slots=256, status=256)
    a.update(change)
    with pytest.raises(lib_built.LuminalB200Error):
        _lib.call("lmb200_kv_reserve", FakeContext().handle, *a.values())
    if set(change) & {"rows", "cu", "slots", "status"}:
        return
    for k in ("rows", "cu", "slots", "status"):
        del a[k]
    with pytest.raises(lib_built.LuminalB200Error):
        _lib.call("lmb200_kv_shrink", FakeContext().handle, *a.values())


@pytest.mark.parametrize("change", [dict(dtype=2), dict(target=0), dict(target=258), dict(draft=257), dict(ts=99), dict(ds=99), dict(vocab=0), dict(rows=-1), dict(rows=70000), dict(n_seq=0),
                                    dict(cu=0), dict(tokens=0), dict(au=0), dict(su=0), dict(out=0), dict(n_out=0), dict(drop=0), dict(ws=0), dict(ws=264), dict(ws_bytes=100), dict(out=256)])
def test_verify_refuses(lib_built, change):
    from importlib import import_module
    _lib = import_module("luminal_jl_b200._lib")
    a = dict(dtype=0, target=256, ts=100, draft=256, ds=100, vocab=100, rows=5, n_seq=2, cu=256, tokens=256, T=256, au=256, su=256, out=512, n_out=256, drop=256, ws=256, ws_bytes=1 << 30)
    a.update(change)
    with pytest.raises(lib_built.LuminalB200Error) as e:
        _lib.call("lmb200_verify_drafts", FakeContext().handle, *a.values())
    assert e.value.code == -1


def test_wrappers_refuse_arrays_that_do_not_fit(lib_built):
    import torch
    L = lib_built

    class Dev:
        handle, ordinal = FakeContext().handle, 0

    class Gpu:
        """Looks like a tensor on the GPU."""

        def __init__(self, *shape, dtype=torch.int32, contiguous=True):
            self.shape, self.dtype, self.is_cuda, self._c = shape, dtype, True, contiguous

        def data_ptr(self): return 256
        def get_device(self): return 0
        def is_contiguous(self): return self._c
        def element_size(self): return torch.empty(0, dtype=self.dtype).element_size()

        def stride(self, i=None):
            s = [1]
            for d in reversed(self.shape[1:]):
                s.insert(0, s[0] * d)
            return tuple(s) if i is None else s[i]

    i32, f32, bf16 = torch.int32, torch.float32, torch.bfloat16
    pages = Gpu(4, 2, 1, 20 * 64, dtype=torch.uint8)
    k, slots = Gpu(3, 2, 64, dtype=bf16), Gpu(3)
    bad = [
        lambda: L.kv4_append(Dev, k, Gpu(3, 2, 64, dtype=f32), slots, pages, page_size=16),
        lambda: L.kv4_append(Dev, k, Gpu(3, 2, 32, dtype=bf16), slots, pages, page_size=16),
        lambda: L.kv4_append(Dev, Gpu(3, 2, 64, dtype=torch.float16), k, slots, pages, page_size=16),
        lambda: L.kv4_append(Dev, k, k, Gpu(2), pages, page_size=16),
        lambda: L.kv4_append(Dev, k, k, Gpu(3, dtype=torch.int64), pages, page_size=16),
        lambda: L.kv4_append(Dev, k, k, slots, Gpu(4, 2, 1, 20 * 64 - 4, dtype=torch.uint8), page_size=16),
        lambda: L.kv4_append(Dev, k, k, slots, pages, page_size=32),
        lambda: L.kv4_append(Dev, torch.zeros(3, 2, 64, dtype=bf16), k, slots, pages, page_size=16),
        lambda: L.kv4_attention(Dev, Gpu(3, 3, 64, dtype=bf16), Gpu(3, 3, 64, dtype=bf16), Gpu(3), Gpu(2), Gpu(2, 5), pages, page_size=16, workspace=Gpu(1 << 20)),
        lambda: L.kv4_attention(Dev, k, Gpu(3, 2, 64, dtype=f32), Gpu(3), Gpu(2), Gpu(2, 5), pages, page_size=16, workspace=Gpu(1 << 20)),
        lambda: L.kv4_attention(Dev, k, k, Gpu(2), Gpu(2), Gpu(2, 5), pages, page_size=16, workspace=Gpu(1 << 20)),
        lambda: L.kv4_attention(Dev, k, k, Gpu(3), Gpu(2), Gpu(2, 5, contiguous=False), pages, page_size=16, workspace=Gpu(1 << 20)),
        lambda: L.kv_reserve(Dev, Gpu(2), Gpu(1), Gpu(2, 4), Gpu(9), Gpu(1), page_size=16, lens_out=Gpu(2), n_free_out=Gpu(1), cu_rows=Gpu(3), slots=Gpu(5), status=Gpu(1)),
        lambda: L.kv_reserve(Dev, Gpu(2), Gpu(2), Gpu(2, 4), Gpu(9), Gpu(1), page_size=16, lens_out=Gpu(2), n_free_out=Gpu(1), cu_rows=Gpu(2), slots=Gpu(5), status=Gpu(1)),
        lambda: L.kv_shrink(Dev, Gpu(2), Gpu(2), Gpu(1, 4), Gpu(9), Gpu(1), page_size=16, lens_out=Gpu(2), n_free_out=Gpu(1)),
        lambda: L.verify_drafts(Dev, Gpu(3, 50, dtype=f32), Gpu(3, 49, dtype=f32), Gpu(2), Gpu(3), None, None, None, Gpu(3), Gpu(1), Gpu(1), workspace=Gpu(1 << 20)),
        lambda: L.verify_drafts(Dev, Gpu(3, 50, dtype=f32), None, Gpu(2), Gpu(3), Gpu(1, dtype=bf16), Gpu(3, dtype=f32), Gpu(1, dtype=f32), Gpu(3), Gpu(1), Gpu(1), workspace=Gpu(1 << 20)),
        lambda: L.verify_drafts(Dev, Gpu(3, 50, dtype=f32), None, Gpu(2), Gpu(3), Gpu(1, dtype=f32), Gpu(2, dtype=f32), Gpu(1, dtype=f32), Gpu(3), Gpu(1), Gpu(1), workspace=Gpu(1 << 20)),
        lambda: L.verify_drafts(Dev, Gpu(3, 50, dtype=f32), None, Gpu(2), Gpu(2), None, None, None, Gpu(3), Gpu(1), Gpu(1), workspace=Gpu(1 << 20)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, L.LuminalB200Error)):
            f()
            pytest.fail(f"call {i} was not refused")


def test_wrappers_refuse_arrays_of_another_gpu(lib_built):
    import torch
    L = lib_built

    class Dev:
        handle, ordinal = FakeContext().handle, 0

    class On:
        def __init__(self, gpu, *shape, dtype=torch.int32):
            self.gpu, self.shape, self.dtype, self.is_cuda = gpu, shape, dtype, True

        def get_device(self): return self.gpu
        def data_ptr(self): return 256
        def numel(self): return int(np.prod(self.shape))
        def is_contiguous(self): return True
        def element_size(self): return 4

    def calls(g):
        i = iter(g)
        a = lambda *shape, dtype=torch.int32: On(next(i), *shape, dtype=dtype)  # noqa: E731
        f = torch.float32
        yield 4, lambda: L.kv4_append(Dev, a(3, 2, 64, dtype=f), a(3, 2, 64, dtype=f), a(3), a(4, 2, 1, 320), page_size=16)
        yield 4, lambda: L.kv4_read(Dev, a(3, 2, 64, dtype=f), a(3, 2, 64, dtype=f), a(3), a(4, 2, 1, 320), page_size=16)
        yield 10, lambda: L.kv_reserve(Dev, a(2), a(2), a(2, 4), a(9), a(1), page_size=16, lens_out=a(2), n_free_out=a(1), cu_rows=a(3), slots=a(5), status=a(1))
        yield 7, lambda: L.kv_shrink(Dev, a(2), a(2), a(2, 4), a(9), a(1), page_size=16, lens_out=a(2), n_free_out=a(1))
        yield 7, lambda: L.kv4_attention(Dev, a(3, 4, 64, dtype=f), a(3, 4, 64, dtype=f), a(3), a(2), a(2, 5), a(4, 2, 1, 320), page_size=16, workspace=a(1 << 20))
        yield 11, lambda: L.verify_drafts(Dev, a(3, 50, dtype=f), a(3, 50, dtype=f), a(2), a(3), a(1, dtype=f), a(3, dtype=f), a(1, dtype=f), a(3), a(1), a(1), workspace=a(1 << 20))

    for which, (n, _) in enumerate(calls([])):
        for other in range(n):
            f = list(calls([int(k == other) for k in range(n)]))[which][1]
            with pytest.raises(ValueError, match="on GPU 1"):
                f()


# ---------------------------------------------------------------------------------------------------------------------
# on the GPU
# ---------------------------------------------------------------------------------------------------------------------
def cuda(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


@pytest.fixture
def on_torch(lib_built, device):
    """The device on torch's stream for the length of a test."""
    device.set_stream(1)
    yield lib_built, device
    device.sync()
    device.set_stream(0)


def filled(rng, n_pages, heads, page, D, spread=1.0):
    """Pages as raw bytes: any level, scales and minima of features around 0."""
    pages = rng.integers(0, 256, (n_pages, heads, page // 16, 20 * D), dtype=np.uint8)
    meta = pages[..., 16 * D:].view(np.float16).reshape(n_pages, heads, page // 16, 2, 2, D // 2)
    width = rng.uniform(2.5, 5.5, meta[..., 0, :].shape) * spread
    meta[..., 0, :] = width / 15
    meta[..., 1, :] = -width * rng.uniform(0.3, 0.7, width.shape)
    return pages


def tables(rng, lens, page, extra=2):
    held = [-(-int(l) // page) for l in lens]
    order = rng.permutation(sum(held) + extra).astype(np.int32)
    table = np.full((len(lens), max(held + [1])), -1, np.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
    return table, len(order)


TABLE_CASES = [
    # n_seq, page, lens, add
    (1, 16, [0], [1]), (1, 16, [16], [1]), (1, 16, [15], [1]), (1, 256, [255], [2]), (3, 16, [0, 5, 16], [0, 0, 0]), (4, 32, [0, 31, 32, 33], [33, 1, 32, 0]),
    (7, 64, None, 3), (33, 16, None, 40), (512, 128, None, 5), (513, 16, None, 1), (2000, 16, None, 9), (8192, 32, None, 2), (3, 16, [0, 7, 100000], [40000, 0, 1]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("n,page,lens,add", TABLE_CASES)
@pytest.mark.parametrize("in_place", [False, True])
def test_tables(on_torch, n, page, lens, add, in_place):
    import torch
    L, dev = on_torch
    rng = np.random.default_rng(n * 7 + page)
    lens = rng.integers(0, 400, n).astype(np.int32) if lens is None else np.array(lens, np.int32)
    add = rng.integers(0, add + 1, n).astype(np.int32) if isinstance(add, int) else np.array(add, np.int32)
    table, n_pages = tables(rng, lens, page, extra=int(sum(-(-(int(l) + int(a)) // page) for l, a in zip(lens, add))) + 3)
    width = max(table.shape[1], int(max(-(-(int(l) + int(a)) // page) for l, a in zip(lens, add))))
    table = np.concatenate([table, np.full((n, width - table.shape[1]), -1, np.int32)], 1)
    used = sorted(set(table[table >= 0].tolist()))
    free = np.full(n_pages, -7, np.int32)
    left = rng.permutation(np.setdiff1d(np.arange(n_pages), used)).astype(np.int32)
    free[:len(left)] = left
    rows = int(add.sum()) + 3
    status, lens2, table2, top2, cu2, slots2 = P.reserve(lens, add, table, free, len(left), page, rows)
    assert status == 0
    d_lens, d_add, d_table, d_free, d_top = cuda(lens), cuda(add), cuda(table), cuda(free), cuda(np.array([len(left)], np.int32))
    d_lens2, d_top2 = (d_lens, d_top) if in_place else (torch.empty_like(d_lens), torch.empty_like(d_top))
    cu, slots, st = torch.full((n + 1,), 77, dtype=torch.int32, device="cuda"), torch.full((rows,), 77, dtype=torch.int32, device="cuda"), torch.full((1,), 77, dtype=torch.int32, device="cuda")
    L.kv_reserve(dev, d_lens, d_add, d_table, d_free, d_top, page_size=page, lens_out=d_lens2, n_free_out=d_top2, cu_rows=cu, slots=slots, status=st)
    dev.sync()
    assert st.item() == 0 and d_top2.item() == top2
    for got, want in ((d_lens2, lens2), (d_table, table2), (cu, cu2), (slots, slots2), (d_free, free)):
        assert np.array_equal(got.cpu().numpy(), want)
    if not in_place:
        assert np.array_equal(d_lens.cpu().numpy(), lens) and d_top.item() == len(left)
    # the tokens of every second sequence leave again, some sequences end
    drop = np.where(np.arange(n) % 2 == 0, add, 0).astype(np.int32)
    drop[rng.random(n) < 0.2] = 2 ** 31 - 1
    drop[rng.random(n) < 0.1] = -5
    lens3, free3, top3 = P.shrink(lens2, drop, table2, free, top2, page)
    d_lens3, d_top3 = (d_lens2, d_top2) if in_place else (torch.empty_like(d_lens), torch.empty_like(d_top))
    L.kv_shrink(dev, d_lens2, cuda(drop), d_table, d_free, d_top2, page_size=page, lens_out=d_lens3, n_free_out=d_top3)
    dev.sync()
    assert np.array_equal(d_lens3.cpu().numpy(), lens3) and np.array_equal(d_free.cpu().numpy(), free3) and d_top3.item() == top3


@pytest.mark.gpu
@pytest.mark.parametrize("change,status", [(dict(add=[1, 17, 1]), 1), (dict(rows=4), 2), (dict(lens=[64, 3, 1]), 4 + 0), (dict(lens=[-1, 3, 0]), 8), (dict(add=[1, -1, 0]), 8), (dict(top=-1), 8),
                                           (dict(top=9), 8), (dict(add=[2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1]), 1 + 2 + 4), (dict(lens=[2 ** 31 - 1, 0, 0]), 4)])
def test_tables_that_do_not_fit_change_nothing(on_torch, change, status):
    import torch
    L, dev = on_torch
    a = dict(lens=[16, 3, 0], add=[1, 2, 2], rows=40, top=2)
    a.update(change)
    table = np.full((3, 4), -1, np.int32)
    table[0, 0], table[1, 0] = 4, 5
    free = np.array([0, 1, 2, 3, 6, 7, -1, -1], np.int32)
    lens, add = np.array(a["lens"], np.int32), np.array(a["add"], np.int32)
    want = P.reserve(lens, add, table, free, a["top"], 16, a["rows"])
    assert want[0] == status
    d_lens, d_table, d_free, top = cuda(lens), cuda(table), cuda(free), cuda(np.array([a["top"]], np.int32))
    cu, slots, st = torch.full((4,), 77, dtype=torch.int32, device="cuda"), torch.full((a["rows"],), 77, dtype=torch.int32, device="cuda"), torch.full((1,), 77, dtype=torch.int32, device="cuda")
    out = torch.empty_like(d_lens)
    L.kv_reserve(dev, d_lens, cuda(add), d_table, d_free, top, page_size=16, lens_out=out, n_free_out=top, cu_rows=cu, slots=slots, status=st)
    dev.sync()
    assert st.item() == status and top.item() == a["top"]
    for got, w in ((out, lens), (d_table, table), (cu, np.zeros(4, np.int32)), (slots, np.full(a["rows"], -1, np.int32)), (d_free, free)):
        assert np.array_equal(got.cpu().numpy(), w)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,top", [([16, 3, 0], 8), ([16, -3, 0], 1), ([16, 300, 0], 1), ([16, 3, 0], -1)])
def test_shrink_that_does_not_fit_is_an_error(on_torch, lens, top):
    L, dev = on_torch
    free, table = np.arange(8).astype(np.int32), np.zeros((3, 4), np.int32)
    d_lens, d_free, d_top = cuda(np.array(lens, np.int32)), cuda(free), cuda(np.array([top], np.int32))
    L.kv_shrink(dev, d_lens, cuda(np.full(3, 400, np.int32)), cuda(table), d_free, d_top, page_size=16, lens_out=d_lens, n_free_out=d_top)
    with pytest.raises(L.LuminalB200Error) as e:
        dev.sync()
    assert e.value.code == -1
    dev.sync()
    assert d_lens.tolist() == lens and d_top.item() == top and np.array_equal(d_free.cpu().numpy(), free)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,heads,D,page,pitch", [(1, 1, 32, 16, 0), (5, 2, 64, 16, 0), (33, 3, 96, 32, 64), (16, 8, 128, 64, 0), (130, 1, 256, 128, 8), (40, 5, 160, 256, 0), (300, 2, 128, 64, 0),
                                                    (257, 3, 64, 16, 0)])
def test_append_and_read(on_torch, dtype, rows, heads, D, page, pitch):
    import torch
    L, dev = on_torch
    rng = np.random.default_rng(rows + D)
    tdt = torch.float32 if dtype == "f32" else torch.bfloat16
    n_pages = rows // page + 3
    # runs of neighbouring slots that begin anywhere, some rows without one
    pages_of = rng.permutation(n_pages)[: rows // page + 2]
    at = np.arange(rows) + int(rng.integers(0, page))
    slots = (pages_of[at // page] * page + at % page).astype(np.int32)
    if rows > 4:
        slots[rng.random(rows) < 0.1] = -1
        part = rng.permutation(rows)[: rows // 3]
        slots[np.sort(part)] = slots[part]                            # and some out of order
    x = rng.standard_normal((2, rows, heads, D)).astype(np.float32) * 10.0 ** rng.uniform(-3, 3, (2, rows, heads, 1)).astype(np.float32)
    x[0, :, :, :32] = np.where(rng.random((rows, heads, 1)) < 0.1, x[0, :, :, :1], x[0, :, :, :32])      # groups of one value
    if rows > 20:
        x[0, 3, 0, 5], x[0, 4, 0, 31], x[1, 5, 0, 0], x[1, 6, 0, 1], x[1, 7, 0, 1], x[0, 8, 0, 2] = np.nan, np.inf, -np.inf, 7e4, -7e4, 2e6
        x[1, 9, 0, :32] = np.arange(32) / 2                          # quotients that end in a half
        x[1, 10, 0, :32] = 0
        x[1, 11, 0, :32] = -rng.random(32) * 1e-6                      # below the smallest half
    width = heads * D
    buf = torch.zeros(2, rows, width + pitch, dtype=tdt, device="cuda")
    buf[:, :, :width] = cuda(x.reshape(2, rows, width)).to(tdt)
    k, v = buf[0, :, :width].unflatten(1, (heads, D)), buf[1, :, :width].unflatten(1, (heads, D))
    xk, xv = k.float().cpu().numpy(), v.float().cpu().numpy()
    start = rng.integers(0, 256, (n_pages, heads, page // 16, 20 * D), dtype=np.uint8)
    want = start.copy()
    P.store(want, xk, xv, slots, page)
    pages = cuda(start)
    L.kv4_append(dev, k, v, cuda(slots), pages, page_size=page)
    dev.sync()
    got = pages.cpu().numpy()
    # NaN has many patterns: metadata is compared as halves
    D16 = 16 * D
    assert np.array_equal(got[..., :D16], want[..., :D16])
    a, b = got[..., D16:].copy().view(np.uint16), want[..., D16:].copy().view(np.uint16)
    nan = (a & 0x7fff) > 0x7c00
    assert np.array_equal(nan, (b & 0x7fff) > 0x7c00) and np.array_equal(a[~nan], b[~nan])
    live = slots >= 0
    rk, rv = (torch.full((rows, width + pitch), 9.0, dtype=tdt, device="cuda") for _ in range(2))
    L.kv4_read(dev, rk[:, :width].unflatten(1, (heads, D)), rv[:, :width].unflatten(1, (heads, D)), cuda(slots), pages, page_size=page)
    dev.sync()
    for r, side in zip((rk, rv), P.load(want, np.where(live, slots, 0), page, D)):
        with np.errstate(all="ignore"):
            exact = torch.from_numpy(side.astype(np.float32).reshape(rows, width)).to(tdt)
        g = r.cpu()
        assert (g[:, width:] == 9).all() and (g[~live] == 9).all()
        assert torch.equal(torch.nan_to_num(g[live][:, :width], nan=3.0e38), torch.nan_to_num(exact[live], nan=3.0e38))


@pytest.mark.gpu
def test_slots_outside_the_cache_are_left_out(on_torch):
    import torch
    L, dev = on_torch
    k = torch.ones(3, 1, 32, device="cuda")
    pages = torch.zeros(2, 1, 1, 640, dtype=torch.uint8, device="cuda")
    L.kv4_append(dev, k, k, cuda(np.array([32, 5, 2 ** 31 - 1], np.int32)), pages, page_size=16)
    with pytest.raises(L.LuminalB200Error):
        dev.sync()
    out = torch.zeros_like(k)
    L.kv4_read(dev, out, out.clone(), cuda(np.array([32, 5, 2 ** 31 - 1], np.int32)), pages, page_size=16)
    with pytest.raises(L.LuminalB200Error):
        dev.sync()
    assert out.sum(-1).flatten().tolist() == [0, 32, 0]


def attend(L, dev, q, cu, lens, table, pages, page, scale, window=0, ws=None, out=None):
    import torch
    out = torch.full_like(q, 7.0) if out is None else out
    ws = torch.zeros(L.kv4_attention_workspace(dev, q.shape[-1]), dtype=torch.uint8, device="cuda") if ws is None else ws
    L.kv4_attention(dev, q, out, cu, lens, table, pages, page_size=page, scale=scale, window=window, workspace=ws)
    return out, ws


def check(got, want, size, dtype):
    got = got.float().cpu().numpy().astype(np.float64)
    f32 = 4 * 2.0 ** -18 * size
    tol = f32 if dtype == "f32" else f32 + 2.0 ** -10 * size + 2.0 ** -8 * np.abs(want)
    off = np.abs(got - want) - tol
    fits = np.isfinite(got).all() and (off <= 0).all()
    assert fits, f"worst {np.abs(got - want).max()}, over its limit by {off.max()}"


ATTENTION_CASES = [
    # D, kv heads, group, page, new tokens, lengths, window
    (64, 1, 1, 16, [1], [1], 0), (128, 2, 4, 16, [1, 1, 1, 1], [1, 15, 16, 17], 0), (32, 3, 1, 16, [1, 1], [100, 3], 0), (96, 2, 4, 32, [1, 0, 1], [70, 5, 31], 0),
    (128, 8, 4, 64, [1] * 5, [333, 1, 700, 64, 65], 0), (128, 1, 7, 128, [1, 1], [129, 1000], 0), (128, 2, 8, 64, [3, 1, 8], [3, 90, 300], 0),
    (64, 2, 3, 256, [5, 2], [5, 513], 0), (256, 1, 2, 64, [1, 4], [50, 260], 0), (160, 2, 5, 32, [2, 1], [40, 200], 0), (192, 1, 16, 16, [1, 2], [33, 150], 0), (224, 1, 1, 16, [1], [35], 0),
    (128, 1, 40, 64, [2], [200], 0), (64, 1, 1, 64, [100], [100], 0), (128, 2, 4, 16, [70, 1], [200, 64], 0), (128, 2, 4, 64, [1, 3, 6], [500, 40, 300], 16),
    (64, 1, 2, 16, [4], [1000], 1), (96, 1, 4, 16, [20], [300], 100), (128, 1, 1, 64, [1], [20000], 0), (128, 1, 4, 16, [6, 1, 1], [9000, 5, 3000], 4000),
    (64, 4, 2, 16, [1] * 150, None, 0), (128, 1, 4, 64, [0, 0, 0], [5, 6, 7], 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,heads,G,page,new,lens,window", ATTENTION_CASES)
def test_attention(on_torch, dtype, D, heads, G, page, new, lens, window):
    import torch
    L, dev = on_torch
    rng = np.random.default_rng(D + heads * G + len(new))
    lens = np.array(lens if lens is not None else rng.integers(1, 200, len(new)), np.int32)
    table, n_pages = tables(rng, lens, page)
    pages = filled(rng, n_pages, heads, page, D)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    rows = int(cu[-1]) + 2
    tdt = torch.float32 if dtype == "f32" else torch.bfloat16
    q = cuda(rng.standard_normal((rows, heads * G, D)).astype(np.float32), tdt)
    want, size = P.attention(q.float().cpu().numpy(), cu, lens, table, pages, page, D ** -0.5, window)
    out, ws = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(pages), page, D ** -0.5, window)
    dev.sync()
    assert (out[cu[-1]:] == 7).all()                                     # rows behind the last sequence
    check(out[:cu[-1]], want[:cu[-1]], size[:cu[-1]], dtype)
    # the workspace is as the first call wants it: the same bits again
    again, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(pages), page, D ** -0.5, window, ws=ws)
    dev.sync()
    assert torch.equal(out, again)


def one_case(rng, dtype, D=128, heads=2, G=4, page=16, lens=(70, 300), new=(2, 1), spread=1.0):
    import torch
    lens = np.array(lens, np.int32)
    table, n_pages = tables(rng, lens, page)
    pages = filled(rng, n_pages, heads, page, D, spread)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = cuda(rng.standard_normal((int(cu[-1]), heads * G, D)).astype(np.float32), torch.float32 if dtype == "f32" else torch.bfloat16)
    return q, cu, lens, table, pages


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_ignores_what_no_row_may_see(on_torch, dtype):
    """NaN and infinities behind a sequence's last token, in its last page and in pages of others, change nothing; nor do stale table entries."""
    import torch
    L, dev = on_torch
    q, cu, lens, table, pages = one_case(np.random.default_rng(1), dtype, lens=(70, 300, 3), new=(2, 1, 2))
    clean, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(pages), 16, 0.1)
    dirty, D = pages.copy(), 128
    seen = np.zeros((pages.shape[0], 16), bool)
    for b, l in enumerate(lens):
        for t in range(l):
            seen[table[b, t // 16], t % 16] = True
    _, _, _, km, vm = P.places(D)
    for value, m in ((np.nan, km), (np.inf, vm), (np.nan, vm + D // 2), (-np.inf, km + D // 2)):
        for p, t in zip(*np.nonzero(~seen)):
            dirty[p, :, 0, 16 * D:].view(np.float16)[:, m[t]] = value
    bad = np.concatenate([table, np.full((3, 3), 2 ** 30, np.int32)], 1)
    bad[bad < 0] = 10 ** 6
    got, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(bad), cuda(dirty), 16, 0.1)
    dev.sync()
    assert torch.equal(got, clean)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_nan_that_is_seen_reaches_its_rows_alone(on_torch, dtype):
    import torch
    L, dev = on_torch
    q, cu, lens, table, pages = one_case(np.random.default_rng(2), dtype)
    clean, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(pages), 16, 0.1)
    _, _, _, km, vm = P.places(128)
    key, value = pages.copy(), pages.copy()
    key[table[0, 1], 0, 0, 16 * 128:].view(np.float16)[km[3, 1]] = np.nan                 # a key of sequence 0, kv head 0
    value[table[1, 2], 1, 0, 16 * 128:].view(np.float16)[vm[7, 2] + 64] = np.nan           # a value of sequence 1, kv head 1, features 64..95
    a, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(key), 16, 0.1)
    b, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(value), 16, 0.1)
    dev.sync()
    assert torch.isnan(a[:2, :4]).all()
    a[:2, :4] = clean[:2, :4]
    assert torch.equal(a, clean)
    assert torch.isnan(b[2, 4:, 64:96]).all()
    b[2, 4:, 64:96] = clean[2, 4:, 64:96]
    assert torch.equal(b, clean)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("what", ["large values", "small values", "one large value", "constant groups", "large queries", "small queries", "sharp", "one query of zeros", "rising scores"])
def test_attention_over_the_numbers_range(on_torch, dtype, what):
    import torch
    L, dev = on_torch
    rng = np.random.default_rng(3)
    q, cu, lens, table, pages = one_case(rng, dtype, lens=(70, 600), new=(3, 1))
    D, scale = 128, 128 ** -0.5
    meta = pages[..., 16 * D:].view(np.float16).reshape(*pages.shape[:3], 2, 2, D // 2)
    if what == "large values":
        meta[..., 1, :, :] = np.clip(meta[..., 1, :, :].astype(np.float32) * 9000, -60000, 60000)
    elif what == "small values":
        meta[..., 1, :, :] = meta[..., 1, :, :].astype(np.float32) * 1e-3
    elif what == "one large value":
        meta[table[0, 1], :, :, 1, :, :] = meta[table[0, 1], :, :, 1, :, :].astype(np.float32) * 2000
        meta[table[1, 9], :, :, 1, :, :] = np.clip(meta[table[1, 9], :, :, 1, :, :].astype(np.float32) * 20000, -60000, 60000)   # append writes no infinity
    elif what == "constant groups":
        meta[..., 0, ::2] = 0
    elif what == "large queries":
        q = (q.float() * 1e18).to(q.dtype)
        scale = 1e-18 * scale
    elif what == "small queries":
        q = (q.float() * 1e-20).to(q.dtype)
        scale = 1e18 * scale
    elif what == "sharp":
        scale = 4.0
    elif what == "one query of zeros":
        q[0, 1] = 0
    elif what == "rising scores":                            # every block brings a larger maximum
        q = q.abs()
        for b in range(2):
            for i, p in enumerate(table[b][table[b] >= 0]):
                meta[p, :, :, 0, 1, :] = -2 + 0.2 * i
    want, size = P.attention(q.float().cpu().numpy(), cu, lens, table, pages, 16, scale)
    out, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(pages), 16, scale)
    dev.sync()
    check(out, want, size, dtype)


@pytest.mark.gpu
def test_attention_pages_that_are_not_there(on_torch):
    """A page outside the cache takes no part, and the call's error is told by the next synchronising call."""
    L, dev = on_torch
    q, cu, lens, table, pages = one_case(np.random.default_rng(4), "f32")
    for entry in (-1, pages.shape[0], 2 ** 31 - 1):
        bad = table.copy()
        bad[1, 3] = entry
        out, ws = attend(L, dev, q, cuda(cu), cuda(lens), cuda(bad), cuda(pages), 16, 0.1)
        with pytest.raises(L.LuminalB200Error) as e:
            dev.sync()
        assert e.value.code == -1
        whole, size = P.attention(q.cpu().numpy(), cu, lens, table, pages, 16, 0.1)
        check(out[:2], whole[:2], size[:2], "f32")
        keep = np.r_[0:48, 64:300]
        k, v = P.load(pages, table[1, keep // 16] * 16 + keep % 16, 16, 128)
        s = np.einsum("hd,khd->hk", q[2].cpu().numpy().astype(np.float64), k.repeat(4, 1)) * 0.1
        e = np.exp(s - s.max(1, keepdims=True))
        check(out[2], np.einsum("hk,khd->hd", e / e.sum(1, keepdims=True), v.repeat(4, 1)), size[2], "f32")
        good, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(pages), 16, 0.1, ws=ws)
        dev.sync()
        check(good, whole, size, "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("cu,lens", [([0, 2, 1], [70, 300]), ([0, 2, 9], [70, 300]), ([-1, 2, 3], [70, 300]), ([0, 2, 3], [-4, 300]), ([0, 2, 3], [70, 2 ** 31 - 1]), ([1, 2, 3], [70, 300])])
def test_attention_row_offsets_and_lengths_that_do_not_fit(on_torch, cu, lens):
    """They touch no memory outside the arrays; where they cannot be meant the next synchronising call says so."""
    L, dev = on_torch
    q, _, _, table, pages = one_case(np.random.default_rng(5), "bf16")
    attend(L, dev, q, cuda(np.array(cu, np.int32)), cuda(np.array(lens, np.int32)), cuda(table), cuda(pages), 16, 0.1)
    if cu == [1, 2, 3]:                                       # rows before the first sequence are nobody's
        dev.sync()
        return
    with pytest.raises(L.LuminalB200Error) as e:
        dev.sync()
    assert e.value.code == -1


@pytest.mark.gpu
@pytest.mark.parametrize("cu", [[0, 3, 1, 3], [0, 1, 2, 4], [0, 3, 0, 3]])
def test_attention_offsets_that_descend_or_leave_the_rows_write_nothing(on_torch, cu):
    """Overlapping sequences would be more work than the rows can hold, so the whole call is left out; the workspace stays usable."""
    import torch
    L, dev = on_torch
    q, good, lens, table, pages = one_case(np.random.default_rng(5), "bf16", lens=(70, 300, 40), new=(1, 1, 1))
    out, ws = attend(L, dev, q, cuda(np.array(cu, np.int32)), cuda(lens), cuda(table), cuda(pages), 16, 0.1)
    with pytest.raises(L.LuminalB200Error) as e:
        dev.sync()
    assert e.value.code == -1 and (out == 7).all()
    a, _ = attend(L, dev, q, cuda(good), cuda(lens), cuda(table), cuda(pages), 16, 0.1, ws=ws)
    b, _ = attend(L, dev, q, cuda(good), cuda(lens), cuda(table), cuda(pages), 16, 0.1)
    dev.sync()
    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [2 ** 31 - 1, 320, 304, 303])
def test_attention_windows_that_reach_past_everything(on_torch, window):
    """A window as long as the table or longer is none, also for rows before a sequence's first token."""
    import torch
    L, dev = on_torch
    q, cu, _, table, pages = one_case(np.random.default_rng(7), "bf16", new=(2, 5))
    assert table.shape[1] * 16 == 304
    lens = np.array([1, 2], np.int32)
    none, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(pages), 16, 0.1)
    out, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(pages), 16, 0.1, window=window)
    dev.sync()
    assert torch.equal(out, none) and (out[[0, 2, 3, 4]] == 0).all() and (out[[1, 5, 6]] != 0).any(-1).any(-1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_an_infinite_scale_spoils_its_features_alone(on_torch, dtype):
    """Beside scales that want the second pass: those are scaled down by the largest number among them."""
    L, dev = on_torch
    q, cu, lens, table, pages = one_case(np.random.default_rng(8), dtype, lens=(70, 600), new=(3, 1))
    meta = pages[..., 16 * 128:].view(np.float16).reshape(*pages.shape[:3], 2, 2, 64)
    meta[..., 1, :, :] = np.clip(meta[..., 1, :, :].astype(np.float32) * 9000, -60000, 60000)
    want, size = P.attention(q.float().cpu().numpy(), cu, lens, table, pages, 16, 128 ** -0.5)
    _, _, _, _, vm = P.places(128)
    pages[table[1, 2], :, 0, 16 * 128:].view(np.float16)[:, vm[7, 2]] = np.inf
    out, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(pages), 16, 128 ** -0.5)
    dev.sync()
    assert not out[3, :, 64:96].isfinite().any()
    out[3, :, 64:96] = 0
    want[3, :, 64:96] = 0
    check(out, want, size, dtype)


@pytest.mark.gpu
def test_attention_more_new_tokens_than_the_cache_holds(on_torch):
    """Rows before a sequence's first token see nothing and are 0."""
    L, dev = on_torch
    q, cu, _, table, pages = one_case(np.random.default_rng(6), "bf16", new=(2, 5))
    lens = np.array([0, 3], np.int32)
    want, size = P.attention(q.float().cpu().numpy(), cu, lens, table, pages, 16, 0.1)
    out, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(pages), 16, 0.1)
    dev.sync()
    assert (out[:4] == 0).all()
    check(out, want, size, "bf16")


@pytest.mark.gpu
def test_attention_strided_rows_and_places_beyond_32_bits(on_torch):
    """q and out inside wider rows; the same pages at the far end of a cache of more than 4 GiB give the same bits."""
    import torch
    L, dev = on_torch
    q, cu, lens, table, pages = one_case(np.random.default_rng(7), "bf16", page=64)
    clean, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(pages), 64, 0.1)
    wide, out = torch.zeros(3, 8 * 128 + 64, dtype=q.dtype, device="cuda"), torch.full((3, 8 * 128 + 256), 5.0, dtype=q.dtype, device="cuda")
    wide[:, 64:] = q.flatten(1)
    attend(L, dev, wide[:, 64:].unflatten(1, (8, 128)), cuda(cu), cuda(lens), cuda(table), cuda(pages), 64, 0.1, out=out[:, :1024].unflatten(1, (8, 128)))
    dev.sync()
    assert torch.equal(out[:, :1024].unflatten(1, (8, 128)), clean) and (out[:, 1024:] == 5).all()
    each = L.kv4_page_bytes(64, 2, 128)
    n = (1 << 32) // each + 400
    far = torch.empty(n, 2, 4, 20 * 128, dtype=torch.uint8, device="cuda")
    base = n - pages.shape[0]
    far[base:] = cuda(pages)
    moved = np.where(table >= 0, table + base, -1).astype(np.int32)
    got, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(moved), far, 64, 0.1)
    x = torch.randn(40, 2, 128, device="cuda")
    slots = cuda((np.arange(40) + (n - 1) * 64 + 7).astype(np.int32))
    a, b = torch.zeros_like(x), torch.zeros_like(x)
    L.kv4_append(dev, x, x, slots, far, page_size=64)
    L.kv4_read(dev, a, b, slots, far, page_size=64)
    dev.sync()
    assert torch.equal(got, clean)
    y = P.values(*P.quantise(x.cpu().numpy())).astype(np.float32)
    assert np.array_equal(a.cpu().numpy(), y) and np.array_equal(b.cpu().numpy(), y)


VERIFY_CASES = [
    # vocab, rows of each sequence, greedy share
    (1, [1, 3], 0.5), (7, [1, 2, 0, 4], 0.0), (100, [5, 1, 9], 0.5), (1000, [3] * 40, 0.3), (4096, [5, 2], 0.0), (4097, [6, 1, 3], 0.0), (32064, [5], 0.0), (51865, [4, 4, 1], 0.3),
    (128256, [5, 0, 3], 0.0), (200003, [2, 2], 0.0), (333, [70], 0.0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("draft_logits", [True, False])
@pytest.mark.parametrize("vocab,of,greedy", VERIFY_CASES)
def test_verify(on_torch, dtype, draft_logits, vocab, of, greedy):
    import torch
    L, dev = on_torch
    rng = np.random.default_rng(vocab + len(of))
    tdt = torch.float32 if dtype == "f32" else torch.bfloat16
    n, cu = len(of), np.concatenate([[0], np.cumsum(of)]).astype(np.int32)
    rows = int(cu[-1]) + 2
    target = rng.standard_normal((rows, vocab)).astype(np.float32) * 2 + 6 * (rng.random((rows, vocab)) < 8 / vocab)
    draft = target + 0.3 * rng.standard_normal((rows, vocab)).astype(np.float32)
    if vocab > 50:
        target[:, rng.random(vocab) < 0.1] = -np.inf
        draft[rng.random((rows, vocab)) < 0.02] = -np.inf
        target[1, 3], target[2, 5] = np.nan, np.inf
        target[0, :20] = target[0, 20:40].max()                # equal largest ones
    pitch = vocab + (3 if vocab % 2 else 0)
    wide = torch.zeros(2, rows, pitch, dtype=tdt, device="cuda")
    wide[0, :, :vocab], wide[1, :, :vocab] = cuda(target), cuda(draft)
    d_target, d_draft = wide[0, :, :vocab], wide[1, :, :vocab]
    target, draft = d_target.float().cpu().numpy(), d_draft.float().cpu().numpy()
    temperature = np.where(rng.random(n) < greedy, 0, rng.uniform(0.3, 1.5, n)).astype(np.float32)
    tokens = np.array([rng.integers(0, vocab) if rng.random() < 0.1 else np.nanargmax(draft[max(0, r - 1)] + rng.gumbel(size=vocab)) for r in range(rows)], np.int32)
    accept_u, sample_u = rng.random(rows).astype(np.float32), rng.random(n).astype(np.float32)
    before = np.full(rows, 55, np.int32)
    want = P.verify(target, draft if draft_logits else None, cu, tokens, temperature, accept_u, sample_u, before)
    out, n_out, drop = cuda(before), torch.full((n,), 9, dtype=torch.int32, device="cuda"), torch.full((n,), 9, dtype=torch.int32, device="cuda")
    ws = torch.full((L.verify_drafts_workspace(rows),), 255, dtype=torch.uint8, device="cuda")
    L.verify_drafts(dev, d_target, d_draft if draft_logits else None, cuda(cu), cuda(tokens), cuda(temperature), cuda(accept_u), cuda(sample_u), out, n_out, drop, workspace=ws)
    dev.sync()
    for got, w in zip((n_out, drop, out), (want[1], want[2], want[0])):
        assert np.array_equal(got.cpu().numpy(), w)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_verify_at_its_edges(on_torch, dtype):
    """Rows of -infinity, tokens outside the vocabulary, random numbers of 0 and just below 1, equal distributions, extreme temperatures, no temperatures."""
    import torch
    L, dev = on_torch
    tdt = torch.float32 if dtype == "f32" else torch.bfloat16
    rng = np.random.default_rng(8)
    V, n, per = 6000, 14, 3
    rows, cu = n * per, (np.arange(n + 1) * per).astype(np.int32)
    target = cuda(rng.standard_normal((rows, V)).astype(np.float32) * 3).to(tdt)
    draft = target.clone()                                     # equal: every draft is taken
    tokens = rng.integers(0, V, rows).astype(np.int32)
    temperature = np.ones(n, np.float32)
    accept_u, sample_u = np.full(rows, np.float32(1 - 2 ** -24)), np.linspace(0, 1 - 2 ** -24, n).astype(np.float32)
    target[3], draft[6] = -np.inf, -np.inf                     # sequence 1's first row; sequence 2's draft
    target[9] = -np.inf
    target[9, 17] = 1.0                                        # one choice
    target[14] = -np.inf                                       # sequence 4's last row
    tokens[16], tokens[19] = -1, V                             # sequences 5, 6
    temperature[7], temperature[8], temperature[9], temperature[10] = 1e-40, 1e30, np.inf, np.nan
    target[33:36, 5000] = np.inf                               # sequence 11
    tokens[37] = 5
    draft[36, 5] = 50.0                                        # sequence 12: a sure draft that the target refuses
    temperature[13] = -1
    t, d = target.float().cpu().numpy(), draft.float().cpu().numpy()
    before = np.full(rows, 55, np.int32)
    ws = torch.zeros(L.verify_drafts_workspace(rows), dtype=torch.uint8, device="cuda")
    for use in (d, None):
        for temp in (temperature, None):
            want = P.verify(t, use, cu, tokens, temp, accept_u, sample_u, before)
            out, n_out, drop = cuda(before), torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
            L.verify_drafts(dev, target, None if use is None else draft, cuda(cu), cuda(tokens), None if temp is None else cuda(temp), cuda(accept_u), cuda(sample_u), out, n_out, drop,
                            workspace=ws)
            dev.sync()
            for got, w in zip((out, n_out, drop), want):
                assert np.array_equal(got.cpu().numpy(), w)


@pytest.mark.gpu
def test_verify_row_offsets_that_do_not_fit(on_torch):
    import torch
    L, dev = on_torch
    target = torch.randn(4, 50, device="cuda")
    ints = lambda *v: cuda(np.array(v, np.int32))  # noqa: E731
    ws = torch.zeros(L.verify_drafts_workspace(4), dtype=torch.uint8, device="cuda")
    for cu in (ints(0, 2, 9), ints(-3, 2, 4), ints(0, 3, 2)):
        out, n_out, drop = ints(5, 5, 5, 5), ints(9, 9), ints(9, 9)
        L.verify_drafts(dev, target, None, cu, ints(1, 2, 3, 4), None, None, None, out, n_out, drop, workspace=ws)
        with pytest.raises(L.LuminalB200Error):
            dev.sync()
    L.verify_drafts(dev, target[:0], None, ints(0, 0, 0), ints(), None, None, None, ints(), n_out, drop, workspace=ws)       # no rows at all
    dev.sync()
    assert n_out.tolist() == [0, 0] and drop.tolist() == [0, 0]


@pytest.mark.gpu
def test_verify_follows_the_target(on_torch):
    """Over many random numbers the first token has the target's distribution although the drafts come from another: 40000 draws of 6 tokens; a share is off by at most five standard
    deviations, 5 sqrt(p (1 - p) / n) <= 5 x 0.0025."""
    import torch
    L, dev = on_torch
    n, V = 20000, 6
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    base = torch.tensor([1.0, 0.2, -1.0, 0.5, -0.3, 0.0], device="cuda")
    other = torch.tensor([0.0, 1.0, 0.3, -0.5, 0.2, -2.0], device="cuda")
    target, draft = base.expand(2 * n, V).contiguous(), other.expand(2 * n, V).contiguous()
    shares = torch.zeros(V, device="cuda")
    ws = torch.zeros(L.verify_drafts_workspace(2 * n), dtype=torch.uint8, device="cuda")
    for _ in range(2):
        tokens = torch.zeros(2 * n, dtype=torch.int32, device="cuda")
        tokens[1::2] = torch.multinomial(torch.softmax(other / 0.8, 0), n, replacement=True, generator=g).int()
        u = torch.rand(3 * n, generator=g, device="cuda")
        out, n_out, drop = (torch.zeros(k, dtype=torch.int32, device="cuda") for k in (2 * n, n, n))
        L.verify_drafts(dev, target, draft, (torch.arange(n + 1, device="cuda") * 2).int(), tokens, torch.full((n,), 0.8, device="cuda"), u[:2 * n].contiguous(), u[2 * n:].contiguous(), out, n_out,
                        drop, workspace=ws)
        dev.sync()
        shares += torch.bincount(out[0::2].long(), minlength=V).float()
    assert torch.allclose(shares / (2 * n), torch.softmax(base / 0.8, 0), atol=5 * 0.0025, rtol=0)


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_serving_loop(on_torch, captured):
    """reserve -> append -> attention -> verify -> shrink, as a server runs them, eight steps of five sequences of which some stand still and some end; with `captured` a step is recorded once
    and replayed with other contents.  Every step is checked against the oracle, and at the end all pages are free again."""
    import torch
    L, dev = on_torch
    rng = np.random.default_rng(10)
    n, heads, G, D, page, n_pages, max_pages, rows, V = 5, 2, 4, 64, 16, 40, 12, 32, 500
    if captured:
        stream = torch.cuda.Stream()                           # the legacy stream cannot be recorded
        dev.set_stream(stream.cuda_stream)
    i32 = dict(dtype=torch.int32, device="cuda")
    lens, add, table, free, top = torch.zeros(n, **i32), torch.zeros(n, **i32), torch.full((n, max_pages), -1, **i32), torch.arange(n_pages, **i32), torch.full((1,), n_pages, **i32)
    cu, slots, status, drop, n_out, out = torch.zeros(n + 1, **i32), torch.zeros(rows, **i32), torch.zeros(1, **i32), torch.zeros(n, **i32), torch.zeros(n, **i32), torch.zeros(rows, **i32)
    tokens, temperature, au, su = torch.zeros(rows, **i32), torch.tensor([0.0, 1.0, 0.7, 0.0, 1.3], device="cuda"), torch.zeros(rows, device="cuda"), torch.zeros(n, device="cuda")
    bf = dict(dtype=torch.bfloat16, device="cuda")
    qkv = torch.zeros(rows, (heads * G + 2 * heads) * D, **bf)
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split([heads * G * D, heads * D, heads * D], 1))
    att, target, draft = torch.zeros(rows, heads * G, D, **bf), torch.zeros(rows, V, device="cuda"), torch.zeros(rows, V, device="cuda")
    pages = torch.zeros(n_pages, heads, 1, 20 * D, dtype=torch.uint8, device="cuda")
    ws, vws = torch.zeros(L.kv4_attention_workspace(dev, D), dtype=torch.uint8, device="cuda"), torch.zeros(L.verify_drafts_workspace(rows), dtype=torch.uint8, device="cuda")
    end = torch.zeros(n, **i32)

    def step():
        L.kv_reserve(dev, lens, add, table, free, top, page_size=page, lens_out=lens, n_free_out=top, cu_rows=cu, slots=slots, status=status)
        L.kv4_append(dev, k, v, slots, pages, page_size=page)
        L.kv4_attention(dev, q, att, cu, lens, table, pages, page_size=page, workspace=ws)
        L.verify_drafts(dev, target, draft, cu, tokens, temperature, au, su, out, n_out, drop, workspace=vws)
        L.kv_shrink(dev, lens, drop, table, free, top, page_size=page, lens_out=lens, n_free_out=top)
        L.kv_shrink(dev, lens, end, table, free, top, page_size=page, lens_out=lens, n_free_out=top)

    torch.cuda.synchronize()
    graph = dev.capture(step) if captured else None
    o = dict(lens=np.zeros(n, np.int32), table=np.full((n, max_pages), -1, np.int32), free=np.arange(n_pages).astype(np.int32), top=n_pages, pages=np.zeros(pages.shape, np.uint8),
             out=np.zeros(rows, np.int32))
    for i in range(8):
        a = np.array([[9, 1, 4, 0, 17][b] if o["lens"][b] == 0 else rng.integers(0, 6) for b in range(n)], np.int32)
        ended = np.where(rng.random(n) < (0.2 if i < 7 else 2), 2 ** 31 - 1, 0).astype(np.int32)
        add.copy_(cuda(a))
        end.copy_(cuda(ended))
        qkv.copy_(torch.randn(qkv.shape, device="cuda"))
        target.copy_(torch.randn(target.shape, device="cuda") * 3)
        draft.copy_(target + 0.3 * torch.randn(target.shape, device="cuda"))
        tokens.copy_(torch.where(torch.rand(rows, device="cuda") < 0.8, draft.argmax(1).roll(1), torch.randint(0, V, (rows,), device="cuda")).int())
        au.uniform_()
        su.uniform_()
        att.fill_(3.0)
        torch.cuda.synchronize()
        dev.graph_launch(graph) if captured else step()
        dev.sync()
        st, o["lens"], o["table"], o["top"], ocu, oslots = P.reserve(o["lens"], a, o["table"], o["free"], o["top"], page, rows)
        assert st == 0 and status.item() == 0
        assert np.array_equal(cu.cpu().numpy(), ocu) and np.array_equal(slots.cpu().numpy(), oslots) and np.array_equal(table.cpu().numpy(), o["table"])
        P.store(o["pages"], k.float().cpu().numpy(), v.float().cpu().numpy(), oslots, page)
        assert np.array_equal(pages.cpu().numpy(), o["pages"])
        want, size = P.attention(q.float().cpu().numpy(), ocu, o["lens"], o["table"], o["pages"], page, D ** -0.5)
        assert (att[ocu[-1]:] == 3).all()
        check(att[:ocu[-1]], want[:ocu[-1]], size[:ocu[-1]], "bf16")
        o["out"], on, od = P.verify(target.cpu().numpy(), draft.cpu().numpy(), ocu, tokens.cpu().numpy(), temperature.cpu().numpy(), au.cpu().numpy(), su.cpu().numpy(), o["out"])
        assert np.array_equal(out.cpu().numpy(), o["out"]) and np.array_equal(n_out.cpu().numpy(), on) and np.array_equal(drop.cpu().numpy(), od)
        for d in (od, ended):
            o["lens"], o["free"], o["top"] = P.shrink(o["lens"], d, o["table"], o["free"], o["top"], page)
        assert np.array_equal(lens.cpu().numpy(), o["lens"]) and np.array_equal(free.cpu().numpy(), o["free"]) and top.item() == o["top"]
    assert top.item() == n_pages and sorted(free.tolist()) == list(range(n_pages))
    if captured:
        dev.graph_destroy(graph)


@pytest.mark.gpu
def test_calls_at_the_same_time_with_a_workspace_each(lib_built):
    """Two contexts on two streams, sixty calls each without waiting, give what each gives alone."""
    import torch
    L = lib_built
    devs = [L.B200Device(0), L.B200Device(0)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    cases = []
    for i, (d, s) in enumerate(zip(devs, streams)):
        d.set_stream(s.cuda_stream)
        q, cu, lens, table, pages = one_case(np.random.default_rng(20 + i), "bf16", heads=8, lens=(2000, 900, 10), new=(1, 3, 1))
        cases.append([q, cuda(cu), cuda(lens), cuda(table), cuda(pages), torch.zeros(L.kv4_attention_workspace(d, 128), dtype=torch.uint8, device="cuda")])
    torch.cuda.synchronize()
    alone = []
    for d, c in zip(devs, cases):
        alone.append(attend(L, d, *c[:5], 16, 0.1, ws=c[5])[0])
        torch.cuda.synchronize()
    outs = [[torch.full_like(c[0], 7.0) for _ in range(60)] for c in cases]
    torch.cuda.synchronize()
    for i in range(60):
        for d, c, o in zip(devs, cases, outs):
            attend(L, d, *c[:5], 16, 0.1, ws=c[5], out=o[i])
    for d in devs:
        d.sync()
    for a, o in zip(alone, outs):
        assert all(torch.equal(a, x) for x in o)
    for d in devs:
        d.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,heads,D,page,offset", [(600, 8, 128, 64, 0), (600, 8, 128, 64, 5), (2100, 3, 96, 16, 15), (700, 12, 64, 32, 16), (333, 7, 256, 256, 9), (5000, 8, 32, 128, 1),
                                                      (512, 9, 160, 16, 0), (4096, 1, 192, 64, 63)])
def test_append_many_rows(on_torch, dtype, rows, heads, D, page, offset):
    """Enough rows that whole blocks are written at once: sequences that begin anywhere, end anywhere, rows left out in between, the places around them untouched."""
    import torch
    L, dev = on_torch
    rng = np.random.default_rng(rows + D + offset)
    tdt = torch.float32 if dtype == "f32" else torch.bfloat16
    slots, at, n_pages = [], 0, 0
    while len(slots) < rows:                                   # runs of one sequence each
        n = int(min(rows - len(slots), rng.choice([1, 3, 15, 16, 17, 40, 200, 700])))
        first = offset if not slots else int(rng.integers(0, page))
        pages_of = n_pages + rng.permutation(-(-(first + n) // page))
        n_pages += len(pages_of)
        pos = first + np.arange(n)
        slots += list(pages_of[pos // page] * page + pos % page)
    slots = np.array(slots, np.int32)
    slots[rng.random(rows) < 0.01] = -1
    x = rng.standard_normal((2, rows, heads, D)).astype(np.float32) * 10.0 ** rng.uniform(-3, 3, (2, rows, heads, 1)).astype(np.float32)
    x[0, 40:56, 0, :32] = np.arange(32) / 2                    # quotients that end in a half
    x[1, 40:56, 0, :32] = -np.arange(32) / 2
    x[0, 60, 0, 5], x[0, 61, 0, 31], x[1, 62, 0, 0], x[1, 63, 0, 1], x[1, 64, 0, 1], x[0, 65, 0, 2] = np.nan, np.inf, -np.inf, 7e4, -7e4, 2e6
    x[1, 70, 0, :32], x[1, 71, 0, :32] = 0, 1.5
    k, v = cuda(x[0]).to(tdt), cuda(x[1]).to(tdt)
    start = rng.integers(0, 256, (n_pages, heads, page // 16, 20 * D), dtype=np.uint8)
    want = start.copy()
    P.store(want, k.float().cpu().numpy(), v.float().cpu().numpy(), slots, page)
    pages = cuda(start)
    L.kv4_append(dev, k, v, cuda(slots), pages, page_size=page)
    rk, rv = torch.full_like(k, 9.0), torch.full_like(v, 9.0)
    L.kv4_read(dev, rk, rv, cuda(slots), pages, page_size=page)
    dev.sync()
    got = pages.cpu().numpy()
    assert np.array_equal(got[..., :16 * D], want[..., :16 * D])
    a, b = got[..., 16 * D:].copy().view(np.uint16), want[..., 16 * D:].copy().view(np.uint16)
    nan = (a & 0x7fff) > 0x7c00
    assert np.array_equal(nan, (b & 0x7fff) > 0x7c00) and np.array_equal(a[~nan], b[~nan])
    live = slots >= 0
    for r, side in zip((rk, rv), P.load(want, np.where(live, slots, 0), page, D)):
        with np.errstate(all="ignore"):
            exact = torch.from_numpy(side.astype(np.float32)).to(tdt)
        g = r.cpu()
        assert (g[~live] == 9).all()
        assert torch.equal(torch.nan_to_num(g[live], nan=3.0e38), torch.nan_to_num(exact[live], nan=3.0e38))
    # the last slots lie outside a cache of one page less: those rows are left out, and told of
    short = pages[:n_pages - 1].contiguous()
    before = short.clone()
    L.kv4_append(dev, k, v, cuda(slots), short, page_size=page)
    with pytest.raises(L.LuminalB200Error):
        dev.sync()
    assert torch.equal(short[..., :16 * D], before[..., :16 * D])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_over_its_own_queries(on_torch, dtype):
    """out = q: what is written is read by no one else, in triples that many CTAs share as well."""
    import torch
    L, dev = on_torch
    q, cu, lens, table, pages = one_case(np.random.default_rng(9), dtype, lens=(9000, 300, 5000), new=(9, 1, 3))
    want, ws = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(pages), 16, 0.1)
    for _ in range(3):
        own = q.clone()
        attend(L, dev, own, cuda(cu), cuda(lens), cuda(table), cuda(pages), 16, 0.1, ws=ws, out=own)
        dev.sync()
        assert torch.equal(own, want)


@pytest.mark.gpu
def test_attention_of_the_most_sequences(on_torch):
    """8192 sequences, some of them without rows, some without tokens."""
    L, dev = on_torch
    rng = np.random.default_rng(10)
    lens = rng.integers(0, 40, 8192).astype(np.int32)
    new = rng.integers(0, 3, 8192)
    table, n_pages = tables(rng, lens, 16)
    pages = filled(rng, n_pages, 1, 16, 32)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = cuda(rng.standard_normal((int(cu[-1]), 1, 32)).astype(np.float32))
    want, size = P.attention(q.cpu().numpy(), cu, lens, table, pages, 16, 0.2)
    out, _ = attend(L, dev, q, cuda(cu), cuda(lens), cuda(table), cuda(pages), 16, 0.2)
    dev.sync()
    check(out, want, size, "f32")


@pytest.mark.gpu
def test_append_and_read_of_millions_of_rows(on_torch):
    """More windows of rows than one dimension of a grid takes: the same bits as in pieces."""
    import torch
    L, dev = on_torch
    rows, page = 2200011, 256
    n_pages = -(-rows // page) + 1
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(rows, 1, 32, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    slots = torch.arange(rows, dtype=torch.int32, device="cuda") + 5
    whole, pieces = (torch.zeros(n_pages, 1, page // 16, 640, dtype=torch.uint8, device="cuda") for _ in range(2))
    L.kv4_append(dev, k, v, slots, whole, page_size=page)
    for a in range(0, rows, 100000):
        L.kv4_append(dev, k[a:a + 100000], v[a:a + 100000], slots[a:a + 100000], pieces, page_size=page)
    dev.sync()
    assert torch.equal(whole, pieces)
    outs = [torch.full_like(k, 9) for _ in range(4)]
    L.kv4_read(dev, outs[0], outs[1], slots, whole, page_size=page)
    for a in range(0, rows, 100000):
        L.kv4_read(dev, outs[2][a:a + 100000], outs[3][a:a + 100000], slots[a:a + 100000], whole, page_size=page)
    dev.sync()
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
    spread = k.float().amax(-1, keepdim=True) - k.float().amin(-1, keepdim=True)
    # half a level, 1/30 of the spread; the minimum's and the scale's roundings to halves (2^-12 each of values below 8: 16 roundings at most), and the result's to bf16
    assert ((outs[0].float() - k.float()).abs() <= spread / 30 + 16 * 8 * 2.0 ** -12 + 8 * 2.0 ** -8).all()


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [None, 1.0])
def test_verify_the_most_sequences(on_torch, temperature):
    """65535 sequences of one row each: the largest logit, or for so peaked ones the same by chance."""
    import torch
    L, dev = on_torch
    n, vocab = 65535, 5
    best = torch.from_numpy(np.random.default_rng(11).integers(0, vocab, n)).cuda()
    logits = torch.nn.functional.one_hot(best, vocab).float() * 200
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    ints = [torch.full((n,), 7, dtype=torch.int32, device="cuda") for _ in range(4)]
    u = torch.rand(n, device="cuda")
    t = None if temperature is None else torch.full((n,), temperature, device="cuda")
    ws = torch.empty(L.verify_drafts_workspace(n), dtype=torch.uint8, device="cuda")
    L.verify_drafts(dev, logits, None, cu, ints[0], t, u, u, ints[1], ints[2], ints[3], workspace=ws)
    dev.sync()
    assert torch.equal(ints[1].long(), best) and (ints[2] == 1).all() and (ints[3] == 0).all()
