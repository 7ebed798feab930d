"""Training with dropout on the GPU (dn_set_dropout): the forward's logits and
every gradient against float64 autograd of the same model and masks, replayed
and resumed masks, and training without dropout left as it was."""
import numpy as np
import pytest
import torch

import dropout_model
from test_gpu_train import check_grads, effective_weights, small_cfg, train_batch, weights_for

pytestmark = pytest.mark.gpu


def open_train(cfg, w, prec, **kw):
    from decide_amd import NoGPUError
    from decide_amd.train import TrainEngine

    try:
        return TrainEngine(cfg, w, precision=prec, **kw)
    except NoGPUError:
        pytest.skip("no GPU")


def dlogits(batch, seed=5):
    rng = np.random.default_rng(seed)
    n = sum(len(s.mask_pos) for s in batch)
    return (rng.standard_normal(n) / n).astype(np.float32)


@pytest.mark.parametrize("prec", ["fp32", "bf16"])
@pytest.mark.parametrize("train_from", [0, 1])
def test_gradients_with_dropout(prec, train_from):
    """Bars: those of training without dropout (test_gpu_train.py) on logits and gradients."""
    cfg = small_cfg()
    w, batch = weights_for(cfg), train_batch(cfg.vocab, 399)
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
        # fp32: the forward tests' bar. bf16: rounding of the operands, as without dropout.
        tol = 1e-4 if prec == "fp32" else 5e-2
        assert np.all(np.abs(got - want.detach().numpy()) <= tol * (1 + np.abs(want.detach().numpy())))
        eng.backward(dl)
        check_grads(eng, grads, prec, train_from=train_from, train_emb=train_from == 0, label="dropout")


@pytest.mark.parametrize("prec", ["fp32", "bf16"])
def test_masks_follow_the_step(prec):
    """The step advances with every training forward; the same step gives the same logits and gradients to
    the bit; the backward pass uses its own forward's masks whatever is set between; inference drops nothing."""
    cfg = small_cfg()
    w, batch = weights_for(cfg), train_batch(cfg.vocab, 399)
    dl = dlogits(batch)
    names = [f"model.layers.{i}.{n}.weight" for i in range(3) for n in ("attn.Wo", "mlp.Wo", "mlp_norm", "attn.Wqkv")]

    def grads(eng):
        eng.zero_grad()
        eng.backward(dl)
        return [eng.download(n, "grad") for n in names]

    with open_train(cfg, w, prec) as eng:
        plain = eng.infer(batch)
        none = eng.forward(batch)
        g0 = grads(eng)
        eng.set_dropout(0.1, 3, 0)
        assert np.array_equal(eng.infer(batch), plain)
        a0 = eng.forward(batch)
        ga = grads(eng)
        a1 = eng.forward(batch)
        g1 = grads(eng)
        assert not np.array_equal(a0, a1) and not np.array_equal(a0, none)
        eng.set_dropout(0.1, 3, 1)  # a resumed run
        assert np.array_equal(eng.forward(batch), a1)
        eng.set_dropout(0.5, 4, 9)
        assert all(np.array_equal(x, y) for x, y in zip(grads(eng), g1))
        eng.set_dropout(0.1, 3, 0)
        assert np.array_equal(eng.forward(batch), a0)
        assert all(np.array_equal(x, y) for x, y in zip(grads(eng), ga))
        eng.set_dropout(0.0)
        assert np.array_equal(eng.forward(batch), none)
        assert all(np.array_equal(x, y) for x, y in zip(grads(eng), g0))


def test_larger_batch_accumulates():
    """ModernBERT-base width, 1,100 tokens in bf16 (the GEMMs' other tiles and the fused GeGLU backward):
    gradients of two micro-batches add up, each with its own masks; a step of AdamW runs on them."""
    from decide_amd.nn import Config
    from decide_amd.synth import random_weights

    cfg = Config(hidden=768, intermediate=1152, heads=12, layers=2, vocab=500, half_window=64,
                 layer_types=["full_attention", "sliding_attention"])
    w = random_weights(cfg, seed=2)
    batch = train_batch(cfg.vocab, 499, specs=[(300, [20, 30, 25], True), (500, [40, 41], True), (120, [9, 8], True)])
    dl = dlogits(batch)
    with open_train(cfg, w, "bf16") as eng:
        name = "model.layers.1.mlp.Wo.weight"
        single = []
        for step in (0, 1):
            eng.set_dropout(0.1, 11, step)
            eng.zero_grad()
            eng.forward(batch)
            eng.backward(dl)
            single.append(eng.download(name, "grad").astype(np.float64))
        eng.set_dropout(0.1, 11, 0)
        eng.zero_grad()
        for _ in (0, 1):
            eng.forward(batch)
            eng.backward(dl)
        both = eng.download(name, "grad")
        want = single[0] + single[1]
        # one more fp32 addition per element, of terms of either's size
        assert np.all(np.abs(both - want) <= 4 * 2.0 ** -24 * (np.abs(single[0]) + np.abs(single[1]) + np.abs(want)))
        assert np.linalg.norm(single[0] - single[1]) > 0.05 * np.linalg.norm(single[0])
        before = eng.download(name)
        eng.update(1e-3, 1e-3, 0.01)
        assert np.all(np.isfinite(eng.download(name))) and not np.array_equal(before, eng.download(name))


def test_refusals():
    from decide_amd import Engine, InvalidArgument, NoGPUError, native

    cfg = small_cfg(1)
    with open_train(cfg, weights_for(cfg), "fp32") as eng:
        for p in (-0.1, 1.5, float("nan")):
            with pytest.raises(InvalidArgument, match="probability"):
                eng.set_dropout(p)
    try:
        eng = Engine(cfg, weights_for(cfg), precision="fp32")
    except NoGPUError:
        pytest.skip("no GPU")
    with eng:
        assert native.lib.dn_set_dropout(eng.handle, 0.1, 0, 0) == native.DN_INVALID_ARG
