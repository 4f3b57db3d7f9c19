"""What a call of the paged 4-bit cache's operators leaves out and tells of later does not end the waits of kernels behind it on the same context."""
import numpy as np
import pytest

import luminal_oracle as O
from test_decode_parity import make_model
from test_llama_step import config
from test_paged import cuda, on_torch  # noqa: F401  (a fixture)


def leave_out(L, dev):
    """Enqueues a call one of whose rows goes nowhere."""
    import torch
    k = torch.ones(3, 1, 32, device="cuda")
    pages = torch.zeros(2, 1, 1, 640, dtype=torch.uint8, device="cuda")
    slots = cuda(np.array([1, 99, 2], np.int32))                # of a cache of 32
    torch.cuda.synchronize()
    L.kv4_append(dev, k, k, slots, pages, page_size=16)
    return k, pages, slots                                     # to be kept until it has run


@pytest.mark.gpu
def test_steps_of_one_launch(on_torch):
    """A step whose CTAs wait for one another, many times over, behind a slot outside its cache: the tokens of a step alone, and the refusal."""
    import torch
    L, dev = on_torch
    dev.set_stream(0)                                          # the legacy stream cannot be recorded, as a session does
    cfg = config(512, 8, 2, 1408, 3001, layers=4)
    model = make_model(L, dev, cfg, O.synth_llama_weights(cfg, seed=5), "f32")
    prompt = O.synth_tokens(5, 1000, (2, 20), cfg["vocab"])
    sess = L.Session(model, 2, 96)
    first = sess.prefill(prompt).argmax(-1).astype(np.int32)
    want = sess.decode_n(first, 40)
    sess.reset()
    sess.prefill(prompt)
    tokens, got = cuda(first), torch.zeros(40, 2, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    kept = leave_out(L, dev)                                   # noqa: F841
    sess.decode_n_device(tokens.data_ptr(), 40, got.data_ptr())
    with pytest.raises(L.LuminalB200Error) as e:
        dev.sync()
    assert e.value.code == -1
    dev.sync()
    assert np.array_equal(got.cpu().numpy(), want)
    sess.close(); model.close()


@pytest.mark.gpu
def test_recorded_steps_as_one_kernel(on_torch, monkeypatch):
    import torch
    monkeypatch.setenv("LMB200_GRAPH_KERNEL", "1")
    L, dev = on_torch
    stream = torch.cuda.Stream()                               # the legacy stream cannot be recorded
    dev.set_stream(stream.cuda_stream)
    g, reg = L.Graph(), {}
    net = L.nn.Llama(g, reg, vocab_size=300, n_layers=2, hidden=256, n_heads=8, n_kv_heads=8, intermediate=688)
    tok = L.tensor(g, [1, 33])
    out = net(tok, 0)
    inputs = {t.id: O.synth_normal(3, t.id, t.shape, 0.3) for t in reg.values()}
    inputs[tok.id] = O.synth_tokens(5, 999, (1, 33), 300).astype(np.float32)
    cg = L.compile(g, dev, outputs=[out.id])
    cg(inputs)
    want = cg.results[out.id].numpy()
    cg(inputs)
    torch.cuda.synchronize()
    kept = leave_out(L, dev)                                   # noqa: F841
    try:
        cg(inputs)                                             # may synchronise, and is then the call that tells
        dev.sync()
        raised = False
    except L.LuminalB200Error as e:
        raised = e.code == -1
    assert raised
    assert np.array_equal(cg.results[out.id].numpy(), want)
    cg.close()
