"""Verification of drafts where probabilities leave every number's range."""
import numpy as np
import pytest

import paged_oracle as P
from test_paged import cuda, on_torch  # noqa: F401  (a fixture)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [6, 5000, 50000])
@pytest.mark.parametrize("draft_logits", [True, False])
@pytest.mark.parametrize("top,T", [(10000, 1e-6), (1000, 7e-8), (20, 2e-9), (1.0, 3e-10), (-50, 4e-9), (3.0e38, 1e28)])
def test_verify_logits_one_step_apart_at_temperatures_near_0(on_torch, vocab, draft_logits, top, T):
    """Two logits that are neighbours among the floats, so cold that the lower one's probability is far below any number: the higher one is the token, as a draft and as the new token."""
    import torch
    L, dev = on_torch
    top = np.float32(top)
    below = np.nextafter(top, np.float32(-np.inf))
    n, per = 6, 2
    rows = n * per
    rng = np.random.default_rng(41)
    target = np.full((rows, vocab), -np.inf, np.float32)
    draft = target.copy()
    best = rng.integers(0, vocab, rows)
    other = (best + rng.integers(1, vocab, rows)) % vocab
    r = np.arange(rows)
    target[r, best], target[r, other] = top, below
    draft[r, other], draft[r, best] = top, below                                 # the draft model takes the two the other way round
    cu = (np.arange(n + 1) * per).astype(np.int32)
    tokens = np.zeros(rows, np.int32)
    tokens[1::2] = np.where(np.arange(n) % 2 == 0, best[0::2], other[0::2])            # every second draft is refused
    temperature = np.full(n, T, np.float32)
    accept_u, sample_u = np.full(rows, 0.5, np.float32), np.linspace(0, 1 - 2 ** -24, n).astype(np.float32)
    use = draft if draft_logits else None
    want = P.verify(target, use, cu, tokens, temperature, accept_u, sample_u, np.full(rows, 55, np.int32))
    out, n_out, drop = (torch.full((k,), 55, dtype=torch.int32, device="cuda") for k in (rows, n, n))
    ws = torch.zeros(L.verify_drafts_workspace(rows), dtype=torch.uint8, device="cuda")
    L.verify_drafts(dev, cuda(target), None if use is None else cuda(draft), cuda(cu), cuda(tokens), cuda(temperature), cuda(accept_u), cuda(sample_u), out, n_out, drop, workspace=ws)
    dev.sync()
    for got, w in zip((out, n_out, drop), want):
        assert np.array_equal(got.cpu().numpy(), w)
    assert (want[0] >= 0).sum() >= n and (want[1] == np.where(np.arange(n) % 2 == 0, 2, 1)).all()
