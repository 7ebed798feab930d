"""The model's training forward with dropout, in float64 torch operations on
the CPU: autograd gives the gradients that the device's are held to."""
import numpy as np
import torch

import block_reference as ref


def dropout_offset(cfg, step, layer, site):
    """The generator's offset of a site (0 attention, 1 MLP) in training forward `step`."""
    return step * 2 * cfg.layers + 2 * layer + site


def parameters(weights):
    return {n: torch.from_numpy(np.asarray(a, np.float64).copy()).requires_grad_() for n, a in weights.items()}


def norm(x, w, eps, b=None):
    d = x - x.mean(-1, keepdim=True)
    y = d / (d.square().mean(-1, keepdim=True) + eps).sqrt() * w
    return y if b is None else y + b


def rope(x, pos, theta):
    half = x.shape[-1] // 2
    inv = 1.0 / theta ** (2.0 * np.arange(half) / (2 * half))
    f = torch.from_numpy(np.float32(pos[:, None] * inv).astype(np.float64))[:, None, :]  # the angle is rounded to fp32
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * f.cos() - b * f.sin(), b * f.cos() + a * f.sin()], -1)


def allowed(s):
    n = len(s.ids)
    if s.opt is None:
        return np.ones((n, n), bool)
    o = np.asarray(s.opt)
    return ((o[:, None] == -1) & (o[None] == -1)) | ((o[:, None] != -1) & ((o[None] == -1) | (o[:, None] == o[None])))


def logits(cfg, P, batch, p=0.0, seed=0, step=0):
    T = sum(len(s.ids) for s in batch)
    H, D = cfg.hidden, cfg.head_dim

    def dropped(x, layer, site):
        if p == 0.0:
            return x
        keep, scale = ref.keep_scale(T, H, p, seed, dropout_offset(cfg, step, layer, site))
        return x * torch.from_numpy(keep * scale)

    def linear(x, name):
        w = P[name]
        return x @ w.reshape(-1, x.shape[-1]).T

    ids = torch.from_numpy(np.concatenate([np.asarray(s.ids, np.int64) for s in batch]))
    h = norm(P["model.embeddings.tok_embeddings.weight"][ids], P["model.embeddings.norm.weight"], cfg.eps)
    for layer in range(cfg.layers):
        pre = f"model.layers.{layer}."
        x = h if layer == 0 else norm(h, P[pre + "attn_norm.weight"], cfg.eps)
        qkv = linear(x, pre + "attn.Wqkv.weight").reshape(T, 3, cfg.heads, D)
        sliding, out, off = cfg.is_sliding(layer), [], 0
        for s in batch:
            n = len(s.ids)
            pos = np.asarray(s.pos, np.float64)
            theta = cfg.local_theta if sliding else cfg.global_theta
            part = qkv[off: off + n]
            q, k = rope(part[:, 0], pos, theta), rope(part[:, 1], pos, theta)
            mask = allowed(s)
            if sliding:
                mask &= np.abs(pos[:, None] - pos[None]) <= cfg.half_window
            score = torch.stack([q[:, i] @ k[:, i].T for i in range(cfg.heads)]) / D ** 0.5
            score = score.masked_fill(~torch.from_numpy(mask), -torch.inf).softmax(-1)
            out.append(torch.cat([score[i] @ part[:, 2, i] for i in range(cfg.heads)], 1))
            off += n
        h = h + dropped(linear(torch.cat(out), pre + "attn.Wo.weight"), layer, 0)
        wi = linear(norm(h, P[pre + "mlp_norm.weight"], cfg.eps), pre + "mlp.Wi.weight")
        value, gate = wi[:, :cfg.intermediate], wi[:, cfg.intermediate:]
        act = 0.5 * value * (1 + torch.erf(value / 2 ** 0.5)) * gate
        h = h + dropped(linear(act, pre + "mlp.Wo.weight"), layer, 1)
    rows, off = [], 0
    for s in batch:
        rows += [off + int(m) for m in s.mask_pos]
        off += len(s.ids)
    x = norm(h[rows], P["model.final_norm.weight"], cfg.eps)
    x = norm(x, P["scorer.input_norm.weight"], 1e-5, P["scorer.input_norm.bias"])
    x = linear(x, "scorer.dense.weight") + P["scorer.dense.bias"]
    x = norm(0.5 * x * (1 + torch.erf(x / 2 ** 0.5)), P["scorer.norm.weight"], 1e-5, P["scorer.norm.bias"])
    return (x * P["scorer.out_proj.weight"].reshape(-1)).sum(1) + P["scorer.out_proj.bias"].reshape(())
