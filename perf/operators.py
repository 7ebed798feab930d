"""The training-block operators as timed cases: LayerNorm, dropout and the
residual boundary made of both, each with its backward pass.

  norm           LayerNorm of every row, with the row statistics the backward
                 pass reads (Engine.layer_norm_device).
  norm_grad      its gradients: input, weight, bias
                 (Engine.layer_norm_backward_device).
  dropout        dropout by a counter-based generator, optionally added to a
                 residual (Engine.dropout_device). Its own backward pass.
  boundary       h = res + dropout(x), y = LayerNorm(h): the end of one
                 sub-layer and the norm of the next
                 (Engine.dropout_add_norm_device).
  boundary_grad  the gradients of both its inputs, weight and bias
                 (Engine.dropout_add_norm_backward_device).

The generator is Philox4x32-10: the mask is a function of (seed, offset, row,
column), so the seed and the offset are inputs and every implementation gives
the same mask. Column c of a row takes 16 bits: half c % 2 of word (c % 8) / 2
of the block with counter (c / 8, row, offset low, offset high) and key (seed
low, seed high). It is kept where they are at least t = round(65536 p), scaled
by 65536 / (65536 - t).

Widths are the model's (768, its MLP's 1152, the scorer's 384), and generic
and odd ones; activations have a residual stream's statistics: every row with
a scale and an offset of its own, a few columns much larger than the rest.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-5


def listed():
    return [
        # The final norm of one question's tokens: pure latency.
        {"name": "norm 64x768 fp32-fp16", "kind": "norm", "rows": 64, "cols": 768, "stream": "fp32", "out": "fp16",
         "pad": 0, "bias": False},
        # The norm before a projection at the serving batch: fp32 residual stream in, operands out.
        {"name": "norm 32768x768 fp32-bf16", "kind": "norm", "rows": 32768, "cols": 768, "stream": "fp32",
         "out": "bf16", "pad": 0, "bias": False},
        # A norm with a bias over the scorer's width, the options of a training batch: the smallest gradient.
        {"name": "norm grad 203x384 fp32", "kind": "norm_grad", "rows": 203, "cols": 384, "stream": "fp32",
         "grad": "fp32", "pad": 0, "bias": True, "accumulate": False},
        # The gradient of the model's norm at a micro-batch of 12,288 tokens.
        {"name": "norm grad 12288x768 bf16", "kind": "norm_grad", "rows": 12288, "cols": 768, "stream": "fp32",
         "grad": "bf16", "pad": 0, "bias": False, "accumulate": True},
        # Embedding dropout of one short request.
        {"name": "dropout 112x768 bf16", "kind": "dropout", "rows": 112, "cols": 768, "x": "bf16", "out": "bf16",
         "pad": 0, "p": 0.1, "residual": False},
        # Dropout of the MLP's activations at the serving batch.
        {"name": "dropout 32768x1152 bf16", "kind": "dropout", "rows": 32768, "cols": 1152, "x": "bf16",
         "out": "bf16", "pad": 0, "p": 0.1, "residual": False},
        # A block boundary of one 64-token request in a fine-tuning step.
        {"name": "boundary 64x768 bf16", "kind": "boundary", "rows": 64, "cols": 768, "x": "bf16", "stream": "fp32",
         "out": "bf16", "pad": 0, "bias": False, "p": 0.1},
        # A micro-batch of 32 x 384 tokens: 16-bit sub-layer output, fp32 residual stream.
        {"name": "boundary 12288x768 bf16", "kind": "boundary", "rows": 12288, "cols": 768, "x": "bf16",
         "stream": "fp32", "out": "bf16", "pad": 0, "bias": False, "p": 0.1},
        # A wide model all in fp16, odd width, rows of a larger buffer.
        {"name": "boundary 4001x4099 fp16", "kind": "boundary", "rows": 4001, "cols": 4099, "x": "fp16",
         "stream": "fp16", "out": "fp16", "pad": 5, "bias": True, "p": 0.15},
        # The gradients of the first of these.
        {"name": "boundary grad 64x768 bf16", "kind": "boundary_grad", "rows": 64, "cols": 768, "grad": "bf16",
         "stream": "fp32", "x": "bf16", "pad": 0, "bias": False, "p": 0.1, "accumulate": False},
        # The gradients of the micro-batch, added to an earlier one's.
        {"name": "boundary grad 12288x768 bf16", "kind": "boundary_grad", "rows": 12288, "cols": 768, "grad": "bf16",
         "stream": "fp32", "x": "bf16", "pad": 0, "bias": False, "p": 0.1, "accumulate": True},
        # A wide model's gradients, everything in bf16.
        {"name": "boundary grad 4096x8192 bf16", "kind": "boundary_grad", "rows": 4096, "cols": 8192, "grad": "bf16",
         "stream": "bf16", "x": "bf16", "pad": 0, "bias": True, "p": 0.1, "accumulate": False},
    ]


_MOST = 4096 * 8192  # elements of a case


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "dropout", "boundary", "boundary_grad"])
    cols = rng.choice([384, 768, 768, 1152, 1024, 2304, 4096, _log_int(rng, 5, 8192), _log_int(rng, 5, 8192)])
    rows = _log_int(rng, 1, min(40000, (_MOST if kind.endswith("grad") else _MOST // 2) // cols))
    half = rng.choice(["bf16", "fp16"])
    case = {"kind": kind, "rows": rows, "cols": cols, "pad": rng.choice([0, 0, 8, rng.randint(1, 40)])}
    p = rng.choice([0.1, round(rng.uniform(0.01, 0.5), 3)])
    if kind == "norm":
        s, o = rng.choice([("fp32", "fp32"), ("fp32", half), (half, half)])
        return {**case, "stream": s, "out": o, "bias": rng.random() < 0.5}
    if kind == "norm_grad":
        g, s = rng.choice([("fp32", "fp32"), (half, "fp32"), (half, half)])
        return {**case, "stream": s, "grad": g, "bias": rng.random() < 0.5, "accumulate": rng.random() < 0.5}
    if kind == "dropout":
        x, o = rng.choice([("fp32", "fp32"), (half, half), (half, "fp32"), ("fp32", half)])
        return {**case, "x": x, "out": o, "p": p, "residual": rng.random() < 0.5}
    a, s, b = rng.choice([("fp32", "fp32", "fp32"), (half, half, half), (half, "fp32", half), ("fp32", "fp32", half)])
    if kind == "boundary":
        return {**case, "x": a, "stream": s, "out": b, "bias": rng.random() < 0.5, "p": p}
    return {**case, "grad": a, "stream": s, "x": b, "bias": rng.random() < 0.5, "p": p,
            "accumulate": rng.random() < 0.5}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, cols, ld = case["rows"], case["cols"], case["cols"] + case["pad"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def empty(dtype):
        return torch.empty(rows, ld, dtype=_TYPES[dtype], device="cuda")[:, :cols]

    def placed(values, dtype):
        t = empty(dtype)
        t.copy_(values)
        return t

    def stream():
        """A residual stream's rows: a scale and an offset each, every 97th column ten times as large."""
        v = normal(rows, cols) * (0.5 + normal(rows, 1).abs()) + 0.3 * normal(rows, 1)
        v[:, ::97] *= 10
        return v

    kind = case["kind"]
    # The stream that made the inputs; the calls on them go there too.
    st = {"case": case, "rows": rows, "cols": cols, "ld": ld, "stream": torch.cuda.current_stream().cuda_stream}
    if "p" in case:
        bits = torch.randint(0, 2 ** 31, (4,), generator=gen, device="cuda").tolist()
        st["seed"], st["offset"] = bits[0] << 32 | bits[1] << 1, bits[2] << 20 | bits[3] & 0xFFFFF
    if kind != "dropout":
        st["w"] = 1 + 0.1 * normal(cols)
        st["b"] = 0.1 * normal(cols) if case["bias"] else None
    if kind == "norm":
        st["x"], st["y"] = placed(stream(), case["stream"]), empty(case["out"])
    elif kind == "dropout":
        st["x"], st["y"] = placed(normal(rows, cols), case["x"]), empty(case["out"])
        st["res"] = placed(stream(), case["out"]) if case["residual"] else None
    elif kind == "boundary":
        st["x"], st["res"] = placed(normal(rows, cols), case["x"]), placed(stream(), case["stream"])
        st["h"], st["y"] = empty(case["stream"]), empty(case["out"])
    else:
        # The forward's kept stream and its statistics, and gradients of a loss summed over the batch.
        st["h"] = placed(stream(), case["stream"])
        h = st["h"].double()
        mean = h.mean(1, keepdim=True)
        st["mean"] = mean[:, 0].float()
        st["rstd"] = ((h - mean).square().mean(1) + EPS).rsqrt().float()
        st["dy"] = placed(0.02 * normal(rows, cols) * (1 + normal(rows, 1).abs()), case["grad"])
        st["dres"] = empty(case["stream"])
        if kind == "boundary_grad":
            st["dh"] = placed(0.02 * normal(rows, cols), case["stream"])
            st["dx"] = empty(case["x"])
        st["dw0"], st["db0"] = normal(cols), normal(cols)  # what earlier micro-batches left
    if kind in ("norm", "boundary"):
        st["mean"], st["rstd"] = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    return st


# The plain forms.


def _keep(seed, offset, rows, cols, p):
    """(keep [rows, cols], scale) of the mask: Philox4x32-10 on int64 tensors, whose products wrap modulo 2^64."""
    low = 0xFFFFFFFF
    blocks = (cols + 7) // 8
    c0 = torch.arange(blocks, device="cuda").expand(rows, blocks)
    c1 = torch.arange(rows, device="cuda")[:, None].expand(rows, blocks)
    c2 = torch.full((1, 1), offset & low, device="cuda").expand(rows, blocks)
    c3 = torch.full((1, 1), offset >> 32, device="cuda").expand(rows, blocks)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32 & low) ^ c1 ^ k0, b & low, (a >> 32 & low) ^ c3 ^ k1, a & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    words = torch.stack([c0, c1, c2, c3], 2)
    halves = torch.stack([words & 0xFFFF, words >> 16], 3).reshape(rows, blocks * 8)[:, :cols]
    t = round(65536 * p)
    return halves >= t, 65536.0 / (65536 - t) if t < 65536 else 0.0


def _dropped(v, keep, scale):
    return torch.where(keep, v * scale, torch.zeros_like(v))


def _norm(v, w, b, dtype):
    mean = v.mean(1, keepdim=True)
    d = v - mean
    rstd = (d * d).mean(1, keepdim=True).add(EPS).rsqrt()
    y = d * rstd * w
    if b is not None:
        y = y + b
    return y.to(dtype), mean[:, 0], rstd[:, 0]


def _norm_grad(st):
    """(input gradient, weight gradient, bias gradient) in 32 bits."""
    dy, xh = st["dy"].float(), (st["h"].float() - st["mean"][:, None]) * st["rstd"][:, None]
    g = dy * st["w"]
    dx = st["rstd"][:, None] * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    dw, db = (dy * xh).sum(0), dy.sum(0) if st["b"] is not None else None
    if st["case"]["accumulate"]:
        dw, db = st["dw0"] + dw, st["db0"] + db if db is not None else None
    return dx, dw, db


def _plain(st):
    case, kind = st["case"], st["case"]["kind"]
    if kind == "norm":
        return _norm(st["x"].float(), st["w"], st["b"], _TYPES[case["out"]])
    if kind == "norm_grad":
        dx, dw, db = _norm_grad(st)
        return dx.to(_TYPES[case["stream"]]), dw, db
    keep, scale = _keep(st["seed"], st["offset"], st["rows"], st["cols"], case["p"])
    if kind == "dropout":
        y = _dropped(st["x"].float(), keep, scale)
        if st["res"] is not None:
            y = st["res"].float() + y
        return y.to(_TYPES[case["out"]])
    if kind == "boundary":
        # The backward pass reads h as it is stored, so the norm is of that too.
        h = (st["res"].float() + _dropped(st["x"].float(), keep, scale)).to(_TYPES[case["stream"]])
        return (h, *_norm(h.float(), st["w"], st["b"], _TYPES[case["out"]]))
    g, dw, db = _norm_grad(st)
    g = st["dh"].float() + g
    return g.to(_TYPES[case["stream"]]), _dropped(g, keep, scale).to(_TYPES[case["x"]]), dw, db


# The framework's calls.

_kept = {}


def _engine(stream):
    if "engine" not in _kept:
        from decide_amd.nn import Config, Engine

        cfg = Config(hidden=256, intermediate=384, heads=4, layers=1, vocab=8, layer_types=["full_attention"])
        _kept["engine"] = Engine(cfg, None, precision="fp32")
    if _kept.get("stream") != stream:
        _kept["engine"].set_stream(stream)
        _kept["stream"] = stream
    return _kept["engine"]


def _at(t):
    return None if t is None else t.data_ptr()


def _sums(st, eng):
    """The weight and bias gradients' buffers, holding what earlier micro-batches left, and the workspace."""
    if "work" not in st:
        st["work"] = torch.empty(max(1, eng.norm_backward_workspace(st["rows"], st["cols"])), dtype=torch.uint8,
                                 device="cuda")
    dw = st["dw0"].clone() if st["case"]["accumulate"] else torch.empty_like(st["dw0"])
    if st["b"] is None:
        return dw, None, st["work"]
    return dw, st["db0"].clone() if st["case"]["accumulate"] else torch.empty_like(st["db0"]), st["work"]


def _own(st):
    case, kind, eng = st["case"], st["case"]["kind"], _engine(st["stream"])
    rows, cols, ld = st["rows"], st["cols"], st["ld"]
    if kind == "norm":
        eng.layer_norm_device(case["stream"], case["out"], rows, cols, _at(st["x"]), ld, _at(st["w"]), _at(st["b"]),
                              EPS, _at(st["y"]), ld, _at(st["mean"]), _at(st["rstd"]))
        return st["y"], st["mean"], st["rstd"]
    if kind == "dropout":
        eng.dropout_device(case["x"], case["out"], rows, cols, _at(st["x"]), ld, _at(st["res"]), ld, case["p"],
                           st["seed"], st["offset"], _at(st["y"]), ld)
        return st["y"]
    if kind == "boundary":
        eng.dropout_add_norm_device(case["x"], case["stream"], case["out"], rows, cols, _at(st["x"]), ld,
                                    _at(st["res"]), ld, case["p"], st["seed"], st["offset"], _at(st["w"]),
                                    _at(st["b"]), EPS, _at(st["h"]), ld, _at(st["y"]), ld, _at(st["mean"]),
                                    _at(st["rstd"]))
        return st["h"], st["y"], st["mean"], st["rstd"]
    dw, db, work = _sums(st, eng)
    if kind == "norm_grad":
        eng.layer_norm_backward_device(case["grad"], case["stream"], rows, cols, _at(st["dy"]), ld, _at(st["h"]), ld,
                                       _at(st["w"]), _at(st["mean"]), _at(st["rstd"]), _at(st["dres"]), ld, _at(dw),
                                       _at(db), case["accumulate"], _at(work), work.numel())
        return st["dres"], dw, db
    eng.dropout_add_norm_backward_device(case["grad"], case["stream"], case["x"], rows, cols, _at(st["dy"]), ld,
                                         _at(st["dh"]), ld, _at(st["h"]), ld, case["p"], st["seed"], st["offset"],
                                         _at(st["w"]), _at(st["mean"]), _at(st["rstd"]), _at(st["dres"]), ld,
                                         _at(st["dx"]), ld, _at(dw), _at(db), case["accumulate"], _at(work),
                                         work.numel())
    return st["dres"], st["dx"], dw, db


def run(st):
    return _own(st) if own else _plain(st)


def work(case):
    n, vec, kind = case["rows"] * case["cols"], 4 * case["cols"], case["kind"]
    size = {k: _SIZE[case[k]] for k in ("x", "stream", "out", "grad") if k in case}
    vectors = 1 + bool(case.get("bias"))
    if kind == "norm":
        return {"bytes": n * (size["stream"] + size["out"]) + 8 * case["rows"] + vectors * vec, "flops": 8 * n}
    if kind == "dropout":
        return {"bytes": n * (size["x"] + size["out"] * (2 if case["residual"] else 1)), "flops": 2 * n}
    if kind == "boundary":
        return {"bytes": n * (size["x"] + 2 * size["stream"] + size["out"]) + 8 * case["rows"] + vectors * vec,
                "flops": 10 * n}
    sums = vec * (1 + vectors * (2 if case["accumulate"] else 1))
    if kind == "norm_grad":
        return {"bytes": n * (size["grad"] + 2 * size["stream"]) + 8 * case["rows"] + sums, "flops": 14 * n}
    return {"bytes": n * (size["grad"] + 3 * size["stream"] + size["x"]) + 8 * case["rows"] + sums, "flops": 17 * n}


# The definition in 64 bits.


def _mask64(seed, offset, rows, cols, p):
    """Column by column of the definition, with NumPy's unsigned integers, 4,096 rows at a time."""
    import numpy as np

    u32, u64 = np.uint32, np.uint64
    blocks, threshold, parts = -(-cols // 8), round(65536 * p), []
    for first in range(0, rows, 4096):
        some = min(4096, rows - first)
        ctr = np.empty((4, some, blocks), u32)
        ctr[0], ctr[1] = np.arange(blocks, dtype=u32), np.arange(first, first + some, dtype=u32)[:, None]
        ctr[2], ctr[3] = u32(offset % 2 ** 32), u32(offset // 2 ** 32)
        for r in range(10):
            key = [(seed % 2 ** 32 + r * 0x9E3779B9) % 2 ** 32, (seed // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32]
            even, odd = ctr[0].astype(u64) * u64(0xD2511F53), ctr[2].astype(u64) * u64(0xCD9E8D57)
            ctr[0] = (odd >> u64(32)).astype(u32) ^ ctr[1] ^ u32(key[0])
            ctr[2] = (even >> u64(32)).astype(u32) ^ ctr[3] ^ u32(key[1])
            ctr[1], ctr[3] = odd.astype(u32), even.astype(u32)
        bits = np.ascontiguousarray(np.moveaxis(ctr, 0, -1)).astype("<u4").view("<u2").reshape(some, -1)[:, :cols]
        parts.append(torch.from_numpy(bits >= threshold))
    return torch.cat(parts).cuda().double() * (65536 / (65536 - threshold) if threshold < 65536 else 0.0)


def exact(case, seed):
    st = prepare(case, seed)
    kind, n = case["kind"], case["cols"]

    def norm(v):
        mean = v.sum(1) / n
        var = (v - mean[:, None]).pow(2).sum(1) / n
        rstd = 1 / torch.sqrt(var + EPS)
        y = (v - mean[:, None]) * rstd[:, None] * st["w"].double()
        return y if st["b"] is None else y + st["b"].double(), mean, rstd

    if kind == "norm":
        return norm(st["x"].double())
    mask = _mask64(st["seed"], st["offset"], case["rows"], n, case["p"]) if "p" in case else None
    if kind == "dropout":
        y = st["x"].double() * mask
        return y if st["res"] is None else y + st["res"].double()
    if kind == "boundary":
        h = st["res"].double() + st["x"].double() * mask
        return (h, *norm(h.to(_TYPES[case["stream"]]).double()))
    rstd = st["rstd"].double()[:, None]
    centred = (st["h"].double() - st["mean"].double()[:, None]) * rstd
    dy = st["dy"].double()
    through = dy * st["w"].double()
    along = (through * centred).sum(1, keepdim=True) / n
    dx = (through - through.sum(1, keepdim=True) / n - centred * along) * rstd
    dw, db = torch.einsum("rc,rc->c", dy, centred), dy.sum(0)
    if case["accumulate"]:
        dw, db = dw + st["dw0"].double(), db + st["db0"].double()
    db = db if st["b"] is not None else None
    if kind == "norm_grad":
        return dx, dw, db
    dres = st["dh"].double() + dx
    return dres, dres * mask, dw, db
