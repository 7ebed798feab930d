"""CPU checks of the dropout model the GPU's training is compared with: without
dropout it is the oracle's model, forward and backward."""
import numpy as np
import torch

import dropout_model
from conftest import rel_err
from test_gpu_train import oracle_grads, small_cfg, train_batch, weights_for


def test_without_dropout_it_is_the_oracle():
    cfg = small_cfg()
    w, batch = weights_for(cfg), train_batch(cfg.vocab, 399)
    logits, dl, grads = oracle_grads(cfg, w, batch)
    P = dropout_model.parameters(w)
    got = dropout_model.logits(cfg, P, batch)
    assert np.allclose(got.detach().numpy(), logits, rtol=1e-5, atol=1e-5)
    (got * torch.from_numpy(np.asarray(dl, np.float64))).sum().backward()
    for name, g in grads.items():
        # the bars of the fp32 device gradients against the same oracle
        assert rel_err(P[name].grad.numpy().reshape(g.shape), g) <= 5e-4, name


def test_dropout_changes_the_logits_and_its_masks_differ_by_site():
    cfg = small_cfg(layers=2)
    w, batch = weights_for(cfg), train_batch(cfg.vocab, 399, specs=[(20, [5, 6], True)])
    P = dropout_model.parameters(w)
    with torch.no_grad():
        a = [dropout_model.logits(cfg, P, batch, p, seed, step) for p, seed, step in
             ((0.0, 1, 0), (0.3, 1, 0), (0.3, 1, 1), (0.3, 2, 0))]
    assert all(float((a[i] - a[j]).abs().max()) > 1e-3 for i in range(4) for j in range(i))
    offsets = [dropout_model.dropout_offset(cfg, step, layer, site) for step in range(3) for layer in range(2)
               for site in range(2)]
    assert len(set(offsets)) == len(offsets)


def test_set_dropout_needs_a_context():
    from decide_amd import native

    assert native.lib.dn_set_dropout(None, 0.1, 1, 2) == native.DN_INVALID_ARG
