"""A paged key / value cache in 4 bits, its block tables on the device, and the verification of drafted tokens: the entry points of that section of
include/luminal_b200.h, where the formats and rules stand.

Arrays are device memory of the caller, as DeviceArrays or as anything with `data_ptr()` and `shape` (torch tensors); a DeviceArray of int32 is one of dtype I32, and a cache is any
array whose first axis counts its pages (of three axes or more the second counts kv heads).  Calls are asynchronous on the device's stream: `device.set_stream(...)` puts them on the stream that made the arrays (1: the
legacy default stream)."""
from __future__ import annotations

import ctypes as C
import math

from . import _lib
from ._lib import BF16, F32, I32
from .device import DeviceArray

_functions = {}


def _call(name, *args):
    f = _functions.get(name)
    if f is None:
        f = _functions[name] = getattr(_lib.load(), name)
    status = f(*args)
    if status:
        _lib.check(status)


_NAMES = {"torch.float32": F32, "torch.bfloat16": BF16, "torch.int32": I32}
_CODES = {F32: F32, BF16: BF16, I32: I32}     # dtype, of a DeviceArray or as torch spells it -> code


def _code(a):
    try:
        return _CODES[a.dtype]
    except KeyError:
        return _CODES.setdefault(a.dtype, _NAMES.get(str(a.dtype), -1))


def _count(a):
    try:
        return a.numel()
    except AttributeError:
        return math.prod(a.shape)


def _address(what, a, on):
    """Address of an array on GPU `on`: a kernel would fault on another one's."""
    if isinstance(a, DeviceArray):
        gpu, address = a.device.ordinal, a.ptr
    elif not a.is_cuda:
        raise ValueError(f"{what}: not in device memory")
    else:
        gpu, address = a.get_device(), a.data_ptr()
    if gpu != on:
        raise ValueError(f"{what}: an array on GPU {gpu} for a device on GPU {on}")
    return address


def _plain(what, a, least, on):
    """Address of a contiguous array of at least `least` elements."""
    if _count(a) < least:
        raise ValueError(f"{what}: {_count(a)} elements, at least {least} are needed")
    if not isinstance(a, DeviceArray) and not a.is_contiguous():
        raise ValueError(f"{what}: not contiguous")
    return _address(what, a, on)


def _ints(what, a, least, on):
    try:                                       # a step names a dozen of these: torch's own answers first
        if _CODES[a.dtype] == I32 and a.numel() >= least and a.get_device() == on and a.is_contiguous():
            return a.data_ptr()
    except (KeyError, AttributeError):
        pass
    if _code(a) != I32:
        raise ValueError(f"{what}: {a.dtype}, expected int32")
    return _plain(what, a, least, on)


def _float(what, a, on):
    """(address, dtype code) of a float32 or bfloat16 array."""
    code = _code(a)
    if code != F32 and code != BF16:
        raise ValueError(f"{what}: {a.dtype}, expected float32 or bfloat16")
    return _address(what, a, on), code


def _rows(what, a, inner):
    """Row pitch in elements of an array [rows, ...] whose rows are contiguous and `inner` long."""
    rows = a.shape[0]
    if _count(a) != rows * inner:
        raise ValueError(f"{what}: {_count(a)} elements for {rows} rows of {inner}")
    if isinstance(a, DeviceArray) or a.is_contiguous():
        return inner
    step, strides = 1, a.stride()
    for i in range(len(strides) - 1, 0, -1):
        if a.shape[i] > 1 and strides[i] != step:
            raise ValueError(f"{what}: the elements of a row must be contiguous")
        step *= a.shape[i]
    return strides[0] if rows > 1 else inner


def kv4_page_bytes(page_size, n_kv_heads, head_dim):
    """Bytes of one page of one layer's cache."""
    n = C.c_int64(0)
    _call("lmb200_kv4_page_bytes", int(page_size), int(n_kv_heads), int(head_dim), C.byref(n))
    return n.value


_PAGE_BYTES = {}


def _bytes(a):
    return _count(a) * ((2 if a.dtype == BF16 else 4) if isinstance(a, DeviceArray) else a.element_size())


def _pool(pages, page_size, heads, dim, on):
    n_pages, shape = pages.shape[0], (page_size, heads, dim)
    each = _PAGE_BYTES.get(shape)
    if each is None:
        each = _PAGE_BYTES[shape] = kv4_page_bytes(*shape)
    if _bytes(pages) < n_pages * each:
        raise ValueError(f"pages: {_bytes(pages)} bytes for {n_pages} pages of {each}")
    return _plain("pages", pages, 0, on), n_pages


def _kv_heads(pages, page_size, dim):
    """kv heads of a cache [pages, kv heads, ...], or [pages, bytes of a page in any dtype]."""
    if len(pages.shape) > 2:
        return pages.shape[1]
    head, held = kv4_page_bytes(page_size, 1, dim), _bytes(pages) // max(1, pages.shape[0])
    if held < head or held % head:
        raise ValueError(f"pages: {held} bytes a page are no number of kv heads of {head}")
    return held // head


def kv_reserve(device, lens, add, table, free_list, n_free, *, page_size, lens_out, n_free_out, cu_rows, slots, status):
    """Pages, slots and lengths for add[b] more tokens of every sequence (lmb200_kv_reserve).  lens_out may be lens, n_free_out n_free."""
    n, rows, on = lens.shape[0], slots.shape[0], device.ordinal
    _call("lmb200_kv_reserve", device.handle, n, page_size, table.shape[1], free_list.shape[0], rows, _ints("lens", lens, n, on), _ints("add", add, n, on),
              _ints("table", table, n * table.shape[1], on), _ints("free_list", free_list, 1, on), _ints("n_free", n_free, 1, on), _ints("lens_out", lens_out, n, on),
              _ints("n_free_out", n_free_out, 1, on), _ints("cu_rows", cu_rows, n + 1, on), _ints("slots", slots, 0, on), _ints("status", status, 1, on))


def kv_shrink(device, lens, drop, table, free_list, n_free, *, page_size, lens_out, n_free_out):
    """The last drop[b] tokens of every sequence leave the cache and their pages go back (lmb200_kv_shrink)."""
    n, on = lens.shape[0], device.ordinal
    _call("lmb200_kv_shrink", device.handle, n, page_size, table.shape[1], free_list.shape[0], _ints("lens", lens, n, on), _ints("drop", drop, n, on),
              _ints("table", table, n * table.shape[1], on), _ints("free_list", free_list, 1, on), _ints("n_free", n_free, 1, on), _ints("lens_out", lens_out, n, on),
              _ints("n_free_out", n_free_out, 1, on))


def _store(name, device, k, v, slots, pages, page_size):
    rows, heads, dim = k.shape
    on = device.ordinal
    (kp, code), (vp, v_code) = _float("k", k, on), _float("v", v, on)
    if code != v_code or v.shape != k.shape:
        raise ValueError(f"k {k.dtype} {tuple(k.shape)} and v {v.dtype} {tuple(v.shape)} differ")
    pool, n_pages = _pool(pages, page_size, heads, dim, on)
    _call(name, device.handle, code, kp, vp, _rows("k", k, heads * dim), _rows("v", v, heads * dim), rows, heads, dim, _ints("slots", slots, rows, on), pool, n_pages,
              page_size)


def kv4_append(device, k, v, slots, pages, *, page_size):
    """Stores k and v [rows, kv heads, head_dim] in 4 bits at slots [rows] (lmb200_kv4_append)."""
    _store("lmb200_kv4_append", device, k, v, slots, pages, page_size)


def kv4_read(device, k_out, v_out, slots, pages, *, page_size):
    """The values that the cache holds at slots [rows] (lmb200_kv4_read)."""
    _store("lmb200_kv4_read", device, k_out, v_out, slots, pages, page_size)


def kv4_attention_workspace(device, head_dim):
    """Bytes of workspace that kv4_attention takes; zero before the first call."""
    n = C.c_int64(0)
    _call("lmb200_kv4_attention_workspace", device.handle, int(head_dim), C.byref(n))
    return n.value


def kv4_attention(device, q, out, cu_rows, lens, table, pages, *, page_size, workspace, scale=None, window=0):
    """Causal attention of the sequences' last tokens, q and out [rows, heads, head_dim], over the cache (lmb200_kv4_attention)."""
    rows, n_heads, dim = q.shape
    n, on = lens.shape[0], device.ordinal
    (qp, code), (op, out_code) = _float("q", q, on), _float("out", out, on)
    if code != out_code or out.shape != q.shape:
        raise ValueError(f"q {q.dtype} {tuple(q.shape)} and out {out.dtype} {tuple(out.shape)} differ")
    heads = _kv_heads(pages, page_size, dim)
    if n_heads % heads:
        raise ValueError(f"{n_heads} query heads over {heads} kv heads")
    pool, n_pages = _pool(pages, page_size, heads, dim, on)
    _call("lmb200_kv4_attention", device.handle, code, qp, _rows("q", q, n_heads * dim), op, _rows("out", out, n_heads * dim), rows, n, _ints("cu_rows", cu_rows, n + 1, on),
              _ints("lens", lens, n, on), _ints("table", table, n * table.shape[1], on), table.shape[1], pool, n_pages, page_size, heads, n_heads // heads, dim,
              dim ** -0.5 if scale is None else scale, window, _plain("workspace", workspace, 0, on), _bytes(workspace))


def verify_drafts_workspace(rows):
    """Bytes of workspace that verify_drafts takes for so many rows."""
    n = C.c_int64(0)
    _call("lmb200_verify_drafts_workspace", int(rows), C.byref(n))
    return n.value


def verify_drafts(device, target, draft, cu_rows, tokens, temperature, accept_u, sample_u, tokens_out, n_out, drop, *, workspace):
    """Judges drafted tokens by the target's logits [rows, vocab] (lmb200_verify_drafts).  draft: the draft model's logits, or None for drafts that were certain;
    temperature: one per sequence, or None for the largest logit everywhere."""
    rows, vocab = target.shape
    n, on = n_out.shape[0], device.ordinal
    tp, code = _float("target", target, on)
    dp, d_stride = None, 0
    if draft is not None:
        dp, d_code = _float("draft", draft, on)
        if d_code != code or draft.shape != target.shape:
            raise ValueError(f"target {target.dtype} {tuple(target.shape)} and draft {draft.dtype} {tuple(draft.shape)} differ")
        d_stride = _rows("draft", draft, vocab)
    randoms = []
    for what, a, least in (("temperature", temperature, n), ("accept_u", accept_u, rows), ("sample_u", sample_u, n)):
        if a is None:
            randoms.append(None)
            continue
        if _float(what, a, on)[1] != F32:
            raise ValueError(f"{what}: {a.dtype}, expected float32")
        randoms.append(_plain(what, a, least, on))
    _call("lmb200_verify_drafts", device.handle, code, tp, _rows("target", target, vocab), dp, d_stride, vocab, rows, n, _ints("cu_rows", cu_rows, n + 1, on),
              _ints("tokens", tokens, rows, on), *randoms, _ints("tokens_out", tokens_out, rows, on), _ints("n_out", n_out, n, on), _ints("drop", drop, n, on),
              _plain("workspace", workspace, 0, on), _bytes(workspace))


__all__ = ["kv4_page_bytes", "kv_reserve", "kv_shrink", "kv4_append", "kv4_read", "kv4_attention_workspace", "kv4_attention", "verify_drafts_workspace", "verify_drafts"]
