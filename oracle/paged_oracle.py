"""Oracle of the paged 4-bit cache, its block tables and the verification of drafts: plain NumPy in 64 bits, one sequence at a time, from the rules in
include/luminal_b200.h.  The reference has none of these (its cache is one dense array, src/Whisper.jl:519-541)."""
import numpy as np


# ---- block tables ---------------------------------------------------------------------------------------------------
def reserve(lens, add, table, free_list, n_free, page, rows):
    """(status, lens, table, n_free, cu_rows, slots) after room for add[b] more tokens was made; nothing changes where status is not 0."""
    n, max_pages = table.shape
    table = table.copy()
    before = [-(-int(l) // page) for l in lens]
    after = [-(-(int(l) + int(a)) // page) for l, a in zip(lens, add)]
    status = 0
    if any(l < 0 or a < 0 for l, a in zip(lens, add)) or not 0 <= n_free <= len(free_list):
        status |= 8
    fine = [b for b in range(n) if lens[b] >= 0 and add[b] >= 0]
    need = sum(after[b] - before[b] for b in fine)
    if 0 <= n_free <= len(free_list) and need > n_free:
        status |= 1
    if sum(int(add[b]) for b in fine) > rows:
        status |= 2
    if any(after[b] > max_pages for b in fine):
        status |= 4
    cu, slots = np.zeros(n + 1, np.int32), np.full(rows, -1, np.int32)
    if status:
        return status, np.array(lens, np.int32), table, n_free, cu, slots
    top = n_free
    for b in range(n):
        for place in range(before[b], after[b]):
            top -= 1
            table[b, place] = free_list[top]
        cu[b + 1] = cu[b] + add[b]
        for i in range(int(add[b])):
            pos = int(lens[b]) + i
            slots[cu[b] + i] = table[b, pos // page] * page + pos % page
    return 0, np.array(lens, np.int32) + np.array(add, np.int32), table, top, cu, slots


def shrink(lens, drop, table, free_list, n_free, page):
    """(lens, free_list, n_free) after the last drop[b] tokens left."""
    free_list = free_list.copy()
    left = [max(0, int(l) - max(0, int(d))) for l, d in zip(lens, drop)]
    for b in reversed(range(len(lens))):
        for place in reversed(range(-(-left[b] // page), -(-int(lens[b]) // page))):
            free_list[n_free] = table[b, place]
            n_free += 1
    return np.array(left, np.int32), free_list, n_free


# ---- 4-bit values ---------------------------------------------------------------------------------------------------
def quantise(x):
    """x [..., D] float32 -> (n, s, m): levels [..., D], float16 scales and minima [..., D / 32]."""
    f = np.asarray(x, np.float32)
    f = f.reshape(*f.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        low, high = f.min(-1), f.max(-1)
        m = low.astype(np.float16)
        s = ((high - low) / np.float32(15)).astype(np.float16)
        bad = ~np.isfinite(m) | ~np.isfinite(s) | np.isnan(f).any(-1)
        sf, mf = s.astype(np.float32)[..., None], m.astype(np.float32)[..., None]
        n = np.where((sf > 0) & ~bad[..., None], np.clip(np.rint((f - mf) / np.where(sf > 0, sf, 1)), 0, 15), 0)
    n = np.where(bad[..., None], 0, n)
    m, s = np.where(bad, np.float16(np.nan), m), np.where(bad, np.float16(np.nan), s)
    return n.astype(np.uint8).reshape(x.shape), s.astype(np.float16), m.astype(np.float16)


def values(n, s, m):
    """The numbers they stand for, in 64 bits."""
    f = n.astype(np.float64).reshape(*n.shape[:-1], -1, 32)
    return (m.astype(np.float64)[..., None] + f * s.astype(np.float64)[..., None]).reshape(n.shape)


def places(D):
    """Of key / value (token % 16, feature): byte and shift in a block; of (token % 16, group): index among the block's 2 D halves."""
    t, d, g = np.arange(16)[:, None], np.arange(D)[None, :], np.arange(D // 32)[None, :]
    kb = ((((d // 32) * 8 + t % 8) * 4 + d % 8 // 2) * 2 + d // 16 % 2) * 4 + 2 * (d % 2) + t // 8
    vb = 8 * D + ((((d // 32) * 8 + d % 8) * 4 + t % 8 // 2) * 2 + d // 16 % 2) * 4 + 2 * (t % 2) + t // 8
    shift = np.broadcast_to(np.where(d % 16 < 8, 0, 4), (16, D))
    km = (g * 8 + t % 8) * 2 + t // 8
    vm = D + ((g * 4 + t % 8 // 2) * 2 + t // 8) * 2 + t % 2
    return kb, vb, shift, km, vm


def store(pages, k, v, slots, page):
    """k, v [rows, heads, D] into pages [n, heads, page / 16, 20 D] (uint8, in place) at slots."""
    D = k.shape[-1]
    kb, vb, shift, km, vm = places(D)
    for side, byte, meta in ((k, kb, km), (v, vb, vm)):
        n, s, m = quantise(side)
        for r, slot in enumerate(slots):
            if slot < 0:
                continue
            t = slot % 16
            for h in range(k.shape[1]):
                block = pages[slot // page, h, slot % page // 16]
                low = shift[t] == 0
                block[byte[t][low]] = n[r, h][low] | n[r, h][~low] << 4
                halves = block[16 * D:].view(np.float16)
                halves[meta[t]] = s[r, h]
                halves[meta[t] + D // 2] = m[r, h]


def load(pages, slots, page, D, size=False):
    """Values m + n s [rows, heads, D] in 64 bits of keys and values at slots; with `size` |m| + n s instead."""
    kb, vb, shift, km, vm = places(D)
    out = []
    for byte, meta in ((kb, km), (vb, vm)):
        slots = np.asarray(slots)
        t = slots % 16
        block = pages[slots // page, :, slots % page // 16]                      # [rows, heads, 20 D]
        n = np.take_along_axis(block, np.broadcast_to(byte[t][:, None], block.shape[:2] + (D,)), -1) >> shift[t][:, None] & 15
        halves = block[..., 16 * D:].copy().view(np.float16)
        at = np.broadcast_to(meta[t][:, None], block.shape[:2] + (D // 32,))
        m = np.take_along_axis(halves, at + D // 2, -1)
        out.append(values(n, np.take_along_axis(halves, at, -1), np.abs(m) if size else m))
    return out


def attention(q, cu, lens, table, pages, page, scale, window=0):
    """(out, size): q [rows, H, D] over the cache; size = sum p (|m| + s n) and 1 + the scores' absolute sums, which bound what rounding can do."""
    rows, H, D = q.shape
    heads = pages.shape[1]
    G = H // heads
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(len(lens)):
        new, held = int(cu[b + 1] - cu[b]), int(lens[b])
        if new == 0 or held == 0:
            continue
        pos = np.arange(held)
        slots = table[b, pos // page].astype(np.int64) * page + pos % page
        k, v = load(pages, slots, page, D)
        kn, vn = load(pages, slots, page, D, size=True)
        for t in range(new):
            p0 = held - new + t
            if p0 < 0:
                continue
            first = max(0, p0 - window + 1) if window > 0 else 0
            for h in range(H):
                qq = q[cu[b] + t, h].astype(np.float64)
                with np.errstate(all="ignore"):
                    s = k[first:p0 + 1, h // G] @ qq * scale
                    e = np.exp(s - s.max())
                    e /= e.sum()
                    out[cu[b] + t, h] = e @ v[first:p0 + 1, h // G]
                    x = 1 + abs(scale) * (kn[first:p0 + 1, h // G] @ np.abs(qq)).max()
                    size[cu[b] + t, h] = x * (e @ vn[first:p0 + 1, h // G])
    return out, size


# ---- drafts ---------------------------------------------------------------------------------------------------------
def _clean(x):
    x = np.asarray(x, np.float32).astype(np.float64)
    return np.where(np.isnan(x), -np.inf, np.minimum(x, float(np.finfo(np.float32).max)))


def probabilities(logits, T):
    """softmax(logits / T); all 0 where no logit is above -infinity."""
    x = _clean(logits)
    if not (x > -np.inf).any():
        return np.zeros(len(x))
    with np.errstate(all="ignore"):
        e = np.where(x > -np.inf, np.exp((x - x.max()) / float(np.float32(T))), 0.0)
    return e / e.sum()


def verify(target, draft, cu, tokens, temperature, accept_u, sample_u, tokens_out):
    """(tokens_out, n_out, drop); rows behind cu[-1] keep what tokens_out has."""
    out, n = tokens_out.copy(), len(cu) - 1
    n_out, drop = np.zeros(n, np.int32), np.zeros(n, np.int32)
    V = target.shape[1]
    for b in range(n):
        r0, r1 = int(cu[b]), int(cu[b + 1])
        if r1 <= r0:
            continue
        T = 0.0 if temperature is None else float(temperature[b])
        greedy, stop = not T > 0, r1 - 1
        for r in range(r0, r1 - 1):
            t = int(tokens[r + 1])
            known = 0 <= t < V
            if greedy:
                x = _clean(target[r])
                takes = known and int(np.argmax(x)) == t and x[t] > -np.inf
            else:
                p = probabilities(target[r], T)
                q = (probabilities(draft[r], T)[t] if known else 0.0) if draft is not None else 1.0
                takes = float(accept_u[r]) * q < (p[t] if known else 0.0)
            if not takes:
                stop = r
                break
        x = _clean(target[stop])
        if not (x > -np.inf).any():
            token = -1
        elif greedy:
            token = int(np.argmax(x))
        else:
            p = probabilities(target[stop], T)
            w = p
            if stop < r1 - 1:
                t = int(tokens[stop + 1])
                if draft is not None:
                    w = np.maximum(p - probabilities(draft[stop], T), 0)
                elif 0 <= t < V:
                    w = p.copy()
                    w[t] = 0
                if not w.sum() > 0:
                    w = p
            c = np.cumsum(w)
            above = np.nonzero((c > float(sample_u[b]) * c[-1]) & (w > 0))[0]
            token = int(above[0]) if len(above) else int(np.nonzero(w > 0)[0][-1])
        out[r0:r1] = -1
        out[r0:stop] = tokens[r0 + 1:stop + 1]
        out[stop] = token
        n_out[b], drop[b] = stop - r0 + 1, r1 - 1 - stop
    return out, n_out, drop
