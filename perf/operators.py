"""The operators of a paged 4-bit key/value cache and of speculative decoding, as cases that can be timed and compared.

`kind` says which operator a case runs:
  reserve    block tables, slot maps and lengths for a step's new tokens, from the sequences' lengths on the GPU
  shrink     the way back: refused drafts leave the cache, finished requests give their pages back
  append     new keys and values are quantised into their pages and, as a prompt's attention does, read back by their slots
  attention  the new tokens of every sequence attend to its pages
  verify     drafted tokens are judged by the target's probabilities with given random numbers

A page holds `page` tokens of every kv head; per head its tokens come in blocks of 16, each 640 bytes per 32 features ("group"):
  keys    [group][key % 8][d % 8 / 2][d / 16 % 2] of 4 bytes; byte 2 (d % 2) + key / 8, low half d % 16 < 8, high half the others
  values  [group][d % 8][key % 8 / 2][d / 16 % 2] of 4 bytes; byte 2 (key % 2) + key / 8, low half d % 16 < 8, high half the others
  then float16: key scales and key minima [group][key % 8][key / 8], value scales and value minima [group][key % 8 / 2][key / 8][key % 2]
"""
import math
import random

import numpy as np
import torch

own = False


def listed():
    return [
        # one user's next token: the smallest call
        dict(name="reserve_one", kind="reserve", n_seq=1, page=16, context=1031, add=1, prompts=0.0),
        # a serving step: most sequences take a token, some arrive with a prompt
        dict(name="reserve_mixed", kind="reserve", n_seq=256, page=64, context=4096, add=2048, prompts=0.06),
        # many short requests and many long prompts at once
        dict(name="reserve_wide", kind="reserve", n_seq=2048, page=16, context=2000, add=500, prompts=0.1),
        # after a verification: most sequences lose some drafts, some have ended
        dict(name="shrink_mixed", kind="shrink", n_seq=512, page=32, context=3000, drafts=7, ended=0.05),
        # the keys and values of one decoding step
        dict(name="append_step", kind="append", rows=32, n_kv_heads=8, dim=128, page=64, dtype="bf16", skip=0.0),
        # a batch of prompts
        dict(name="append_prompts", kind="append", rows=32768, n_kv_heads=8, dim=128, page=64, dtype="bf16", skip=0.0),
        # a small float32 model: one sequence, one token
        dict(name="attend_small_f32", kind="attention", n_seq=1, context=1024, ragged=0.0, new=1, n_kv_heads=8, group=1, dim=64, page=16, dtype="f32", window=0),
        # a serving batch at a middling context, heads of 96
        dict(name="attend_b16_d96", kind="attention", n_seq=16, context=2052, ragged=0.5, new=1, n_kv_heads=8, group=4, dim=96, page=32, dtype="bf16", window=0),
        # full batch, full context
        dict(name="attend_b32", kind="attention", n_seq=32, context=8184, ragged=0.0, new=1, n_kv_heads=8, group=4, dim=128, page=64, dtype="bf16", window=0),
        # drafted tokens of eight sequences of unequal lengths
        dict(name="attend_drafts", kind="attention", n_seq=8, context=16000, ragged=0.7, new=6, n_kv_heads=8, group=4, dim=128, page=64, dtype="bf16", window=0),
        # one sequence's drafts, judged one step at a time: where latency counts
        dict(name="verify_one", kind="verify", n_seq=1, drafts=4, vocab=32064, dtype="f32", draft_logits=True, greedy=0.0),
        # a serving batch with the largest vocabulary, some requests greedy
        dict(name="verify_b32", kind="verify", n_seq=32, drafts=4, vocab=128256, dtype="f32", draft_logits=True, greedy=0.2),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["reserve", "shrink", "append", "attention", "attention", "attention", "verify", "verify"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "reserve":
        n = _log_int(rng, 1, 2048)
        return dict(kind=kind, n_seq=n, page=page, context=_log_int(rng, 1, min(32768, 4096000 // n)), add=_log_int(rng, 1, min(4096, 204800 // n + 1)),
                    prompts=round(rng.uniform(0, 0.5), 3))
    if kind == "shrink":
        n = _log_int(rng, 1, 2048)
        return dict(kind=kind, n_seq=n, page=page, context=_log_int(rng, 1, min(32768, 4096000 // n)), drafts=rng.randint(0, 15), ended=round(rng.uniform(0, 0.5), 3))
    if kind == "append":
        heads, dim, dtype = _log_int(rng, 1, 16), rng.choice([32, 64, 96, 128, 192, 256]), rng.choice(["bf16", "bf16", "f32"])
        most = 32768 * 8 * 128 * 2 // (heads * dim * (4 if dtype == "f32" else 2))
        return dict(kind=kind, rows=_log_int(rng, 1, min(32768, most)), n_kv_heads=heads, dim=dim, page=page, dtype=dtype, skip=rng.choice([0.0, 0.0, 0.1]))
    if kind == "attention":
        n, heads, dim = _log_int(rng, 1, 64), _log_int(rng, 1, 16), rng.choice([32, 64, 96, 128, 192, 256])
        group, new = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16]), rng.choice([1, 1, 1, 2, 4, 5, 8])
        most = 32 * 8184 * 8 * 128 // (n * heads * dim) // max(1, group * new // 8)
        return dict(kind=kind, n_seq=n, context=max(new, _log_int(rng, 1, max(2, min(131072, most)))), ragged=rng.choice([0.0, 0.3, 0.9]), new=new, n_kv_heads=heads,
                    group=group, dim=dim, page=page, dtype=rng.choice(["bf16", "bf16", "f32"]), window=rng.choice([0, 0, 0, 500, 1024]))
    n, drafts, vocab = _log_int(rng, 1, 64), rng.randint(0, 8), rng.choice([1024, 4096, 32064, 51865, 128256])
    while n * (drafts + 1) * vocab > 32 * 5 * 128256:
        n = max(1, n // 2)
    return dict(kind="verify", n_seq=n, drafts=drafts, vocab=vocab, dtype=rng.choice(["f32", "bf16"]), draft_logits=rng.random() < 0.6, greedy=rng.choice([0.0, 0.3, 1.0]))


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
_DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}
_BIG = (1 << 31) - 1


def _lengths(case, rng):
    """How many tokens every sequence holds: `ragged` spreads them downwards from the context."""
    ragged = case.get("ragged", 0.5)
    return [max(1, int(case["context"] * (1 - ragged * rng.random()))) for _ in range(case["n_seq"])]


def _shape(case, seed):
    """The host's side of a case: lengths, new tokens, pages.  A case has one collection of requests; a seed brings them in another order."""
    rng, page, n = random.Random(1), case["page"], case["n_seq"]
    lens = _lengths(case, rng)
    if case["kind"] == "reserve":
        arrives = [rng.random() < case["prompts"] for _ in range(n)]
        lens = [0 if a else x for a, x in zip(arrives, lens)]
        change = [rng.randint((case["add"] + 1) // 2, case["add"]) if a else (0 if rng.random() < 0.03 and n > 1 else 1) for a in arrives]
        after = [x + c for x, c in zip(lens, change)]
    elif case["kind"] == "shrink":
        change = [_BIG if rng.random() < case["ended"] else rng.randint(0, case["drafts"]) for _ in range(n)]
        after = lens
    else:
        change = [min(case["new"], x) if rng.random() < 0.75 or n == 1 else rng.randint(1, min(case["new"], x)) for x in lens]
        after = lens
    order = list(range(n))
    random.Random(seed * 7 + 1).shuffle(order)
    lens, change, after = [lens[i] for i in order], [change[i] for i in order], [after[i] for i in order]
    held = [-(-x // page) for x in lens]
    return dict(lens=lens, change=change, held=held, max_pages=max(-(-x // page) for x in after) + 1, n_pages=sum(-(-x // page) for x in after) + n + 8)


def _table(s, g):
    """Pages handed out in no order, as they are after some hours of service; the rest is the free list."""
    order = torch.randperm(s["n_pages"], generator=g, device="cuda").to(torch.int32)
    held = torch.tensor(s["held"], device="cuda")
    place = torch.arange(s["max_pages"], device="cuda")[None, :]
    at = held.cumsum(0)[:, None] - held[:, None] + place
    table = torch.where(place < held[:, None], order[at.clamp(max=s["n_pages"] - 1)], torch.full((), -1, dtype=torch.int32, device="cuda"))
    used = sum(s["held"])
    free = torch.full((s["n_pages"],), -1, dtype=torch.int32, device="cuda")
    free[:s["n_pages"] - used] = order[used:]
    return table.contiguous(), free, torch.tensor([s["n_pages"] - used], dtype=torch.int32, device="cuda")


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, out = case["kind"], dict(case)
    if kind in ("reserve", "shrink"):
        s = _shape(case, seed)
        table, free, n_free = _table(s, g)
        n = case["n_seq"]
        out.update(lens=_ints(s["lens"]), change=_ints(s["change"]), table=table, free=free, n_free=n_free, lens_out=torch.zeros(n, dtype=torch.int32, device="cuda"),
                   n_free_out=torch.zeros(1, dtype=torch.int32, device="cuda"))
        if kind == "reserve":
            rows = sum(s["change"]) + 5                    # a step's buffers are a little larger than its tokens
            out.update(rows=rows, cu_rows=torch.zeros(n + 1, dtype=torch.int32, device="cuda"), slots=torch.zeros(rows, dtype=torch.int32, device="cuda"),
                       status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    elif kind == "append":
        rows, heads, dim, page = case["rows"], case["n_kv_heads"], case["dim"], case["page"]
        n_pages = -(-rows // page) + 3
        pages = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        at = torch.arange(rows, device="cuda") + (5 if rows > 5 else 0)          # the first token continues a sequence
        slots = pages[at // page] * page + (at % page).to(torch.int32)
        slots[torch.rand(rows, generator=g, device="cuda") < case["skip"]] = -1  # rows of sequences that stand still
        # keys have a few strong features, values are even
        strong = 1 + 6 * (torch.rand(heads, dim, generator=g, device="cuda") < 0.05)
        k = (torch.randn(rows, heads, dim, generator=g, device="cuda") * strong).to(_DTYPE[case["dtype"]])
        v = torch.randn(rows, heads, dim, generator=g, device="cuda").to(_DTYPE[case["dtype"]])
        out.update(slots=slots, k=k, v=v, n_pages=n_pages, pages=torch.zeros(n_pages, heads, page // 16, 20 * dim, dtype=torch.uint8, device="cuda"),
                   k_read=torch.zeros_like(k), v_read=torch.zeros_like(v))
    elif kind == "attention":
        s = _shape(case, seed)
        table, _, _ = _table(s, g)
        heads, dim = case["n_kv_heads"], case["dim"]
        rows = sum(s["change"])
        cu = [0]
        for c in s["change"]:
            cu.append(cu[-1] + c)
        # every value of 4 bits is as likely as another; scales and minima as of features spread over about four deviations
        pages = torch.randint(0, 256, (s["n_pages"], heads, case["page"] // 16, 20 * dim), generator=g, device="cuda", dtype=torch.uint8)
        meta = pages[..., 16 * dim:].view(torch.float16).view(*pages.shape[:3], 2, 2, dim // 2)
        spread = torch.rand(*pages.shape[:3], 2, dim // 2, generator=g, device="cuda") * 3 + 2.5
        meta[..., 0, :] = (spread / 15).half()
        meta[..., 1, :] = (-spread * (0.4 + 0.2 * torch.rand(spread.shape, generator=g, device="cuda"))).half()
        q = (torch.randn(rows, heads * case["group"], dim, generator=g, device="cuda") * 1.5).to(_DTYPE[case["dtype"]])
        out.update(table=table, lens=_ints(s["lens"]), cu_rows=_ints(cu), pages=pages, q=q, out=torch.zeros_like(q), longest=max(s["lens"]), most_new=max(s["change"]),
                   scale=dim ** -0.5)
    else:
        n, vocab, rng = case["n_seq"], case["vocab"], random.Random(1)
        drafts = [case["drafts"] if rng.random() < 0.75 or n == 1 else rng.randint(0, case["drafts"]) for _ in range(n)]
        rng = random.Random(seed * 7 + 3)
        rng.shuffle(drafts)
        cu = [0]
        for d in drafts:
            cu.append(cu[-1] + d + 1)
        rows = cu[-1]
        temperature = torch.tensor([0.0 if rng.random() < case["greedy"] else rng.uniform(0.5, 1.2) for _ in range(n)], device="cuda")
        # a few likely tokens over a long tail, the draft near the target, ids behind the tokenizer's masked
        target = torch.randn(rows, vocab, generator=g, device="cuda") * 2
        target += 7 * (torch.rand(rows, vocab, generator=g, device="cuda") < 12 / vocab)
        draft = target + 0.6 * torch.randn(rows, vocab, generator=g, device="cuda")
        target[:, vocab - vocab // 50:] = -math.inf
        draft[:, vocab - vocab // 50:] = -math.inf
        target, draft = target.to(_DTYPE[case["dtype"]]), draft.to(_DTYPE[case["dtype"]])
        seq = torch.repeat_interleave(torch.arange(n, device="cuda"), _ints(drafts) + 1)
        noise = -torch.log(-torch.log(torch.rand(rows, vocab, generator=g, device="cuda").clamp(1e-20, 1 - 1e-7)))
        drawn = (draft.float() + noise * (temperature[seq, None] if case["draft_logits"] else 0.0)).argmax(1).to(torch.int32)
        tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        first = torch.zeros(rows, dtype=torch.bool, device="cuda")
        first[_ints(cu[:-1]).long()] = True
        tokens = torch.where(first, tokens, drawn.roll(1))
        u = torch.rand(rows + n, generator=g, device="cuda")
        out.update(target=target, draft=draft if case["draft_logits"] else None, cu_rows=_ints(cu), tokens=tokens, temperature=temperature, accept_u=u[:rows].clone(),
                   sample_u=u[rows:].clone(), tokens_out=torch.zeros(rows, dtype=torch.int32, device="cuda"), n_out=torch.zeros(n, dtype=torch.int32, device="cuda"),
                   drop=torch.zeros(n, dtype=torch.int32, device="cuda"))
    return out


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
_lib = []


def _framework():
    """The framework and its device, on torch's stream."""
    if not _lib:
        import luminal_jl_b200 as L
        dev = L.get_device()
        dev.set_stream(torch.cuda.current_stream().cuda_stream or 1)        # 1: the legacy default stream
        _lib.extend((L, dev))
    return _lib


def _run_own(s):
    L, dev = _framework()
    kind = s["kind"]
    if kind == "reserve":
        L.kv_reserve(dev, s["lens"], s["change"], s["table"], s["free"], s["n_free"], page_size=s["page"], lens_out=s["lens_out"], n_free_out=s["n_free_out"],
                     cu_rows=s["cu_rows"], slots=s["slots"], status=s["status"])
        return s["table"], s["lens_out"], s["n_free_out"], s["cu_rows"], s["slots"], s["status"]
    if kind == "shrink":
        L.kv_shrink(dev, s["lens"], s["change"], s["table"], s["free"], s["n_free"], page_size=s["page"], lens_out=s["lens_out"], n_free_out=s["n_free_out"])
        return s["free"], s["lens_out"], s["n_free_out"]
    if kind == "append":
        L.kv4_append(dev, s["k"], s["v"], s["slots"], s["pages"], page_size=s["page"])
        L.kv4_read(dev, s["k_read"], s["v_read"], s["slots"], s["pages"], page_size=s["page"])
        return s["k_read"], s["v_read"]
    if kind == "attention":
        if "workspace" not in s:
            s["workspace"] = torch.zeros(L.kv4_attention_workspace(dev, s["dim"]), dtype=torch.uint8, device="cuda")
        L.kv4_attention(dev, s["q"], s["out"], s["cu_rows"], s["lens"], s["table"], s["pages"], page_size=s["page"], scale=s["scale"], window=s["window"],
                        workspace=s["workspace"])
        return s["out"]
    if "workspace" not in s:
        s["workspace"] = torch.empty(L.verify_drafts_workspace(s["tokens"].shape[0]), dtype=torch.uint8, device="cuda")
    L.verify_drafts(dev, s["target"], s["draft"], s["cu_rows"], s["tokens"], s["temperature"], s["accept_u"], s["sample_u"], s["tokens_out"], s["n_out"], s["drop"],
                    workspace=s["workspace"])
    return s["tokens_out"], s["n_out"], s["drop"]


def _pages_of(lens, page):
    return (lens + page - 1) // page


def _plain_reserve(s):
    page, n = s["page"], s["lens"].shape[0]
    lens, add = s["lens"].long(), s["change"].long()
    have = _pages_of(lens, page)
    need = _pages_of(lens + add, page) - have
    before, cu = need.cumsum(0) - need, torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), add.cumsum(0)])
    short = need.sum() > s["n_free"][0]
    wide = _pages_of(lens + add, page).max() > s["table"].shape[1]
    long = cu[-1] > s["rows"]
    status = short * 1 + long * 2 + wide * 4
    ok = status == 0
    place = torch.arange(s["table"].shape[1], device="cuda")[None, :]
    fresh = (place >= have[:, None]) & (place < (have + need)[:, None]) & ok
    at = s["n_free"][0] - 1 - (before[:, None] + place - have[:, None])
    s["table"].copy_(torch.where(fresh, s["free"][at.clamp(0, s["free"].shape[0] - 1)], s["table"]))
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(cu, row, right=True) - 1
    used = (row < cu[-1]) & ok
    seq = seq.clamp(max=n - 1)
    pos = (lens[seq] + row - cu[seq]).clamp(min=0)
    slots = torch.where(used, s["table"][seq, (pos // page).clamp(max=s["table"].shape[1] - 1)].long() * page + pos % page, -1)
    s["lens_out"].copy_(torch.where(ok, lens + add, lens))
    s["n_free_out"].copy_(s["n_free"] - torch.where(ok, need.sum(), 0))
    s["cu_rows"].copy_(torch.where(ok, cu, 0))
    s["slots"].copy_(slots)
    s["status"].copy_(status)
    return s["table"], s["lens_out"], s["n_free_out"], s["cu_rows"], s["slots"], s["status"]


def _plain_shrink(s):
    page = s["page"]
    lens = s["lens"].long()
    left = (lens - s["change"]).clamp(min=0)
    have, keep = _pages_of(lens, page), _pages_of(left, page)
    back = have - keep
    behind = back.flip(0).cumsum(0).flip(0) - back               # pages that later sequences give back
    place = torch.arange(s["table"].shape[1], device="cuda")[None, :]
    gone = (place >= keep[:, None]) & (place < have[:, None])
    at = s["n_free"][0] + behind[:, None] + (have[:, None] - 1 - place)
    s["free"][at[gone]] = s["table"][gone]
    s["lens_out"].copy_(left)
    s["n_free_out"].copy_(s["n_free"] + back.sum())
    return s["free"], s["lens_out"], s["n_free_out"]


def _quantised(x):
    """Every 32 features to 16 levels, and back."""
    f = x.float().reshape(*x.shape[:-1], -1, 32)
    low, high = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    m = low.half().float()
    s = ((high - low).double() / 15).float().half().float()
    n = ((f - m).double() / torch.where(s == 0, 1.0, s).double()).float().round().clamp(0, 15)
    return (m + torch.where(s == 0, 0.0, n) * s).reshape(x.shape).to(x.dtype)


def _plain_append(s):
    live = (s["slots"] >= 0)[:, None, None]
    s["k_read"].copy_(torch.where(live, _quantised(s["k"]), s["k_read"]))
    s["v_read"].copy_(torch.where(live, _quantised(s["v"]), s["v_read"]))
    return s["k_read"], s["v_read"]


def _values(blocks, dim):
    """Keys and values [.., 16, dim] in float32 of blocks [.., 20 dim] of bytes."""
    lead, groups = blocks.shape[:-1], dim // 32
    data = blocks[..., :16 * dim].reshape(*lead, 2, groups, 8, 4, 2, 2, 2, 1)
    n = torch.cat([data & 15, data >> 4], -1)                    # [.., kv, group, 8, 4, d / 16, pair, key / 8, d % 16 / 8]
    meta = blocks[..., 16 * dim:].contiguous().view(torch.float16).float().reshape(*lead, 4, groups, 16)
    b = len(lead)
    lead_axes = list(range(b))
    k = n[..., 0, :, :, :, :, :, :, :].permute(*lead_axes, b + 5, b + 1, b, b + 3, b + 6, b + 2, b + 4).reshape(*lead, 16, groups, 32)
    v = n[..., 1, :, :, :, :, :, :, :].permute(*lead_axes, b + 5, b + 2, b + 4, b, b + 3, b + 6, b + 1).reshape(*lead, 16, groups, 32)
    by_key = meta[..., :2, :, :].reshape(*lead, 2, groups, 8, 2).transpose(-1, -2).reshape(*lead, 2, groups, 16, 1).transpose(-2, -3)
    by_value = meta[..., 2:, :, :].reshape(*lead, 2, groups, 4, 2, 2).transpose(-2, -3).reshape(*lead, 2, groups, 16, 1).transpose(-2, -3)
    k = k.float() * by_key[..., 0, :, :, :] + by_key[..., 1, :, :, :]
    v = v.float() * by_value[..., 0, :, :, :] + by_value[..., 1, :, :, :]
    return k.reshape(*lead, 16, dim), v.reshape(*lead, 16, dim)


def _plain_attention(s):
    n, heads, group, dim, page = s["n_seq"], s["n_kv_heads"], s["group"], s["dim"], s["page"]
    pages = -(-s["longest"] // page)
    k, v = _values(s["pages"][s["table"][:, :pages].clamp(min=0).long()], dim)         # [n, pages, heads, blocks, 16, dim]
    k = k.transpose(1, 2).reshape(n, heads, pages * page, dim)
    v = v.transpose(1, 2).reshape(n, heads, pages * page, dim)
    cu, lens = s["cu_rows"].long(), s["lens"].long()
    new = cu[1:] - cu[:-1]
    t = torch.arange(s["most_new"], device="cuda")[None, :]
    row = (cu[:-1, None] + t).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].float().reshape(n, s["most_new"], heads, group, dim).permute(0, 2, 1, 3, 4).reshape(n, heads, -1, dim)
    score = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    at = torch.arange(pages * page, device="cuda")[None, None, :]
    position = (lens - new)[:, None] + t
    seen = at <= position[:, :, None]
    if s["window"] > 0:
        seen = seen & (at > position[:, :, None] - s["window"])
    seen = seen[:, None, :, None, :].expand(n, 1, s["most_new"], group, -1).reshape(n, 1, -1, pages * page)
    score = score.masked_fill(~seen, -math.inf)
    high = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(high == -math.inf, 0.0, high))
    out = torch.matmul(e, v) / e.sum(-1, keepdim=True)
    out = out.reshape(n, heads, s["most_new"], group, dim).permute(0, 2, 1, 3, 4).reshape(n, s["most_new"], heads * group, dim)
    s["out"].copy_(out[t.expand(n, -1) < new[:, None]].to(s["out"].dtype))
    return s["out"]


def _probabilities(logits, temperature):
    x = logits.double() / temperature[:, None].double()
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_verify(s):
    cu, rows, vocab = s["cu_rows"].long(), s["tokens"].shape[0], s["vocab"]
    n = cu.shape[0] - 1
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(cu, row, right=True) - 1
    last = row == cu[seq + 1] - 1
    greedy = s["temperature"] <= 0
    warm = torch.where(greedy, 1.0, s["temperature"])
    target = s["target"].float()
    high = target.amax(-1, keepdim=True)
    best = torch.where(target == high, torch.arange(vocab, device="cuda"), vocab).amin(-1)
    p = _probabilities(s["target"], warm[seq])
    judged = s["tokens"].long().roll(-1)[:, None]                  # the draft that a row's distribution judges
    if s["draft"] is not None:
        q = _probabilities(s["draft"], warm[seq])
    else:
        q = torch.zeros_like(p).scatter_(1, judged, 1.0)
    takes = s["accept_u"].double() * q.gather(1, judged)[:, 0] < p.gather(1, judged)[:, 0]
    takes = torch.where(greedy[seq], judged[:, 0] == best, takes) & ~last
    stops = torch.where(takes, rows, row)
    stop = torch.full((n,), rows, device="cuda").scatter_reduce(0, seq, stops, "amin")
    pick, ends = p[stop], last[stop]
    rest = (pick - torch.where(ends[:, None], 0.0, q[stop])).clamp(min=0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, pick)
    c = rest.cumsum(-1)
    chosen = (c <= s["sample_u"].double()[:, None] * c[:, -1:]).sum(-1)
    some = torch.where(rest > 0, torch.arange(vocab, device="cuda"), 0).amax(-1)
    chosen = torch.where(greedy, best[stop], torch.minimum(chosen, some))
    out = torch.where(row < stop[seq], judged[:, 0], torch.where(row == stop[seq], chosen[seq], -1))
    s["tokens_out"].copy_(out)
    s["n_out"].copy_(stop - cu[:-1] + 1)
    s["drop"].copy_(cu[1:] - 1 - stop)
    return s["tokens_out"], s["n_out"], s["drop"]


def run(state):
    if own:
        return _run_own(state)
    return dict(reserve=_plain_reserve, shrink=_plain_shrink, append=_plain_append, attention=_plain_attention, verify=_plain_verify)[state["kind"]](state)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and what it should return
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind in ("reserve", "shrink"):
        s = _shape(case, 0)
        if kind == "reserve":
            taken = sum(-(-(x + c) // case["page"]) + (-x // case["page"]) for x, c in zip(s["lens"], s["change"]))
            # lengths and requests in, lengths and offsets out, pages from the list into the table, a page's place read once and its slots written
            return {"bytes": 16 * case["n_seq"] + 8 * taken + 4 * sum(s["change"]) + 4 * sum(c > 0 for c in s["change"]) + 16, "flops": 0}
        left = [max(0, x - c) for x, c in zip(s["lens"], s["change"])]
        given = sum(-(-x // case["page"]) + (-y // case["page"]) for x, y in zip(s["lens"], left))
        return {"bytes": 12 * case["n_seq"] + 8 * given + 8, "flops": 0}
    if kind == "append":
        elements, size = case["rows"] * case["n_kv_heads"] * case["dim"] * 2, 4 if case["dtype"] == "f32" else 2
        # rows in and out, the 4-bit form written and read
        return {"bytes": elements * (2 * size + 2 * 0.625) + 8 * case["rows"], "flops": 6 * elements}
    if kind == "attention":
        s = _shape(case, 0)
        heads, dim, size = case["n_kv_heads"], case["dim"], 4 if case["dtype"] == "f32" else 2
        keys = [min(x, case["window"] + c - 1) if case["window"] > 0 else x for x, c in zip(s["lens"], s["change"])]
        rows = sum(s["change"])
        return {"bytes": sum(keys) * heads * dim * 1.25 + 2 * rows * heads * case["group"] * dim * size,
                "flops": 4 * sum(k * c for k, c in zip(keys, s["change"])) * heads * case["group"] * dim}
    rows, size = case["n_seq"] * (case["drafts"] + 1), 4 if case["dtype"] == "f32" else 2
    # the target's rows, and the draft's behind which a draft was made
    drafts = case["n_seq"] * case["drafts"] if case["draft_logits"] else 0
    return {"bytes": (rows + drafts) * case["vocab"] * size, "flops": 3 * (rows + drafts) * case["vocab"]}


def _exact_append(case, s):
    live = (s["slots"] >= 0).cpu().numpy()
    out = []
    for x in (s["k"], s["v"]):
        a = x.float().cpu().numpy().reshape(-1, 32)
        low, high = a.min(1), a.max(1)
        m = low.astype(np.float16).astype(np.float64)
        step = ((high - low) / np.float32(15)).astype(np.float16).astype(np.float64)
        level = np.zeros(a.shape)
        some = step > 0
        apart = (a[some] - m[some, None].astype(np.float32)).astype(np.float32)
        level[some] = np.clip(np.rint(apart / step[some, None].astype(np.float32)), 0, 15)
        y = (m[:, None] + level * step[:, None]).reshape(x.shape)
        y[~live] = 0
        out.append(torch.from_numpy(y))
    return tuple(out)


def _exact_attention(case, s):
    """A sequence and a kv head at a time, every value looked up by its place in its block."""
    heads, group, dim, page = case["n_kv_heads"], case["group"], case["dim"], case["page"]
    cu, lens = s["cu_rows"].tolist(), s["lens"].tolist()
    key, d = torch.arange(16)[:, None], torch.arange(dim)[None, :]
    tile = d // 16 % 2
    k_byte = (d // 32) * 256 + ((key % 8) * 4 + d % 8 // 2) * 8 + tile * 4 + 2 * (d % 2) + key // 8
    v_byte = 8 * dim + (d // 32) * 256 + ((d % 8) * 4 + key % 8 // 2) * 8 + tile * 4 + 2 * (key % 2) + key // 8
    high = (d % 16 // 8 * 4).expand(16, dim).cuda()
    k_meta = ((d // 32) * 16 + (key % 8) * 2 + key // 8).cuda()
    v_meta = ((d // 32) * 16 + (key % 8 // 2) * 4 + key // 8 * 2 + key % 2).cuda()
    k_byte, v_byte = k_byte.cuda(), v_byte.cuda()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["n_seq"]):
        new, held = cu[b + 1] - cu[b], lens[b]
        mine = s["table"][b, :-(-held // page)].long()
        for h in range(heads):
            blocks = s["pages"][mine, h].reshape(-1, 20 * dim)
            meta = blocks[:, 16 * dim:].contiguous().view(torch.float16).double().reshape(-1, 4, dim // 2)
            k = ((blocks[:, k_byte] >> high) & 15).double() * meta[:, 0][:, k_meta] + meta[:, 1][:, k_meta]
            v = ((blocks[:, v_byte] >> high) & 15).double() * meta[:, 2][:, v_meta] + meta[:, 3][:, v_meta]
            k, v = k.reshape(-1, dim)[:held], v.reshape(-1, dim)[:held]
            q = s["q"][cu[b]:cu[b + 1], h * group:(h + 1) * group].double()
            score = torch.einsum("tgd,kd->tgk", q, k) * case["dim"] ** -0.5
            at = torch.arange(held, device="cuda")
            for t in range(new):
                position = held - new + t
                hidden = (at > position) | ((at <= position - case["window"]) if case["window"] > 0 else (at < 0))
                score[t][:, hidden] = -math.inf
            out[cu[b]:cu[b + 1], h * group:(h + 1) * group] = torch.softmax(score, -1) @ v
    return out


def exact(case, seed):
    if case["kind"] not in ("append", "attention"):
        return None                                                # whole numbers
    s = prepare(case, seed)
    return _exact_append(case, s) if case["kind"] == "append" else _exact_attention(case, s)
