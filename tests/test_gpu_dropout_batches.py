"""Training with dropout on batches of more than 512 tokens (the boundary's
gradient then keeps partial sums in the workspace and joins them): every
gradient against float64 autograd of the same model and masks."""
import numpy as np
import pytest
import torch

import dropout_model
from test_gpu_dropout_train import dlogits, open_train
from test_gpu_train import check_grads, effective_weights, small_cfg, train_batch, weights_for

pytestmark = pytest.mark.gpu

# 673 tokens, and 1,073 (the fp32 GeGLU's gradient in the product's epilogue starts above 1,024).
BATCHES = {673: [(200, [20, 30, 25], True), (180, [40, 41], False), (108, [9, 17], True)],
           1073: [(400, [50, 30, 25], True), (280, [40, 41], False), (178, [9, 17], True)]}


def make(cfg, tokens):
    batch = train_batch(cfg.vocab, 399, specs=BATCHES[tokens])
    assert sum(len(s.ids) for s in batch) == tokens
    return batch


@pytest.mark.parametrize("tokens", [673, 1073])
@pytest.mark.parametrize("prec", ["fp32", "bf16"])
@pytest.mark.parametrize("train_from", [0, 1, 3])
def test_gradients_with_dropout(prec, train_from, tokens):
    """Bars: those of training without dropout (test_gpu_train.py) on logits and gradients."""
    cfg = small_cfg()
    w, batch = weights_for(cfg), make(cfg, tokens)
    p, seed, step = 0.2, 0x9876543210FEDCBA, 7
    dl = dlogits(batch)
    P = dropout_model.parameters(effective_weights(w, prec))
    want = dropout_model.logits(cfg, P, batch, p, seed, step)
    (want * torch.from_numpy(dl.astype(np.float64))).sum().backward()
    grads = {n: P[n].grad.numpy().reshape(np.shape(w[n])) for n in w}
    with open_train(cfg, w, prec, train_from=train_from, train_emb=train_from == 0) as eng:
        eng.set_dropout(p, seed, step)
        eng.zero_grad()
        got = eng.forward(batch)
        tol = 1e-4 if prec == "fp32" else 5e-2
        assert np.all(np.abs(got - want.detach().numpy()) <= tol * (1 + np.abs(want.detach().numpy())))
        eng.backward(dl)
        check_grads(eng, grads, prec, train_from=train_from, train_emb=train_from == 0, label="dropout")


@pytest.mark.parametrize("prec", ["fp32", "bf16"])
def test_micro_batches_add_up(prec):
    """Gradients of two micro-batches, each with its own masks, add up in every tensor, the norms' weights among
    them, and no tensor's are those of one mask."""
    cfg = small_cfg()
    w, batch = weights_for(cfg), make(cfg, 673)
    dl = dlogits(batch)
    with open_train(cfg, w, prec) as eng:
        single = []
        for step in (0, 1):
            eng.set_dropout(0.1, 11, step)
            eng.zero_grad()
            eng.forward(batch)
            eng.backward(dl)
            single.append({n: eng.download(n, "grad").astype(np.float64) for n in w})
        eng.set_dropout(0.1, 11, 0)
        eng.zero_grad()
        for _ in (0, 1):
            eng.forward(batch)
            eng.backward(dl)
        for n in w:
            a, b = single[0][n], single[1][n]
            # Sums that accumulate into the first micro-batch's: each of at most 1,073 + 16 additions in fp32 may
            # round at the size of the running sum, which the two and their difference bound.
            both, size = eng.download(n, "grad"), np.abs(a) + np.abs(b)
            assert np.all(np.abs(both - (a + b)) <= 1100 * 2.0 ** -24 * size.max()), n
            if n.endswith(("mlp_norm.weight", "attn_norm.weight", "Wo.weight", "Wqkv.weight")):
                assert np.linalg.norm(a - b) > 0.05 * np.linalg.norm(a), n


def test_a_call_without_tokens_does_not_count():
    """Nor does a refused one: the masks that follow are those of the step that was set."""
    from decide_amd import InvalidArgument, native

    cfg = small_cfg(2)
    none = np.zeros(1, np.int32), np.zeros(1, np.float32)
    w, batch = weights_for(cfg), make(cfg, 673)
    with open_train(cfg, w, "fp32") as eng:
        eng.set_dropout(0.3, 5, 4)
        want = eng.forward(batch)
        eng.set_dropout(0.3, 5, 4)
        assert native.lib.dn_forward_train(eng.handle, 0, *[none[0].ctypes.data] * 6,
                                           none[1].ctypes.data, 1) == native.DN_OK
        bad = train_batch(cfg.vocab, 399, specs=BATCHES[673])
        bad[0].ids[3] = cfg.vocab + 5
        with pytest.raises(InvalidArgument):
            eng.forward(bad)
        assert np.array_equal(eng.forward(batch), want)


def test_training_without_dropout_after_training_with_it():
    """A backward pass without dropout in a context whose first ones had it: the bits of one that never had."""
    cfg = small_cfg()
    w, batch = weights_for(cfg), make(cfg, 673)
    dl = dlogits(batch)
    got = []
    for ps in ((0.0,), (0.2, 0.0)):
        with open_train(cfg, w, "bf16") as eng:
            for p in ps:
                eng.set_dropout(p, 3)
                eng.zero_grad()
                logits = eng.forward(batch)
                eng.backward(dl)
            got.append([logits] + [eng.download(n, "grad") for n in w])
    assert all(np.array_equal(a, b) for a, b in zip(*got))
