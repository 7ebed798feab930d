"""The 8-bit projection operators as timed cases: what a block whose products
run in 8-bit floating point calls, forward and backward.

  rms       h = res + x, y = RMSNorm(h), and y in 8 bits with a scale for each
            row and 128 columns, the operand of the product that follows
            (Engine.add_rms_norm_device).
  rms_grad  the gradients of both inputs and the weight
            (Engine.add_rms_norm_backward_device).
  quant     an array in 8 bits with a scale for each 1 x 128 or 128 x 128
            block, and its transpose's (Engine.quantize_blocks_device).
  gemm      C = A . B^T of such arrays (Engine.gemm_fp8_device).

A block's scale is its largest magnitude (at least 2^-100) over the type's
largest value, 448 (e4m3) or 57344 (e5m2); its elements are divided by the
scale and rounded to nearest. Scales are held block by block: the scale of
row r and columns 128 b .. 128 b + 127 at [b, r], of a 128 x 128 block at
[column block, row block].

Widths are the model's (768, its QKV's 2304, its MLP's 1152, the scorer's 384)
and generic and odd ones. Activations have a residual stream's statistics:
every row with a scale of its own, a few columns much larger than the rest.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn,
          "e5m2": torch.float8_e5m2}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2, "e4m3": 1, "e5m2": 1}
_LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
EPS = 1e-5
BLOCK = 128


def listed():
    return [
        # The norm in front of QKV of one 64-token request: pure latency.
        {"name": "rms 64x768", "kind": "rms", "rows": 64, "cols": 768, "x": "bf16", "stream": "fp32", "y": None,
         "q": "e4m3", "pad": 0, "residual": True},
        # The same at the serving batch, fp32 residual stream.
        {"name": "rms 32768x768", "kind": "rms", "rows": 32768, "cols": 768, "x": "bf16", "stream": "fp32", "y": None,
         "q": "e4m3", "pad": 0, "residual": True},
        # A wide model all in bf16, odd width, rows of a larger buffer, y kept for the weight gradient.
        {"name": "rms 4001x4099 bf16", "kind": "rms", "rows": 4001, "cols": 4099, "x": "bf16", "stream": "bf16",
         "y": "bf16", "q": "e4m3", "pad": 5, "residual": True},
        # The gradient of a norm over the scorer's width, the options of a training batch.
        {"name": "rms grad 203x384 fp32", "kind": "rms_grad", "rows": 203, "cols": 384, "dy": "fp32",
         "stream": "fp32", "x": None, "pad": 0, "accumulate": False},
        # The gradient at a micro-batch of 32 x 384 tokens, added to an earlier one's.
        {"name": "rms grad 12288x768 bf16", "kind": "rms_grad", "rows": 12288, "cols": 768, "dy": "bf16",
         "stream": "fp32", "x": "bf16", "pad": 0, "accumulate": True},
        # The MLP's activations of a request of 112 tokens, in front of its second product.
        {"name": "quant 112x1152 bf16", "kind": "quant", "rows": 112, "cols": 1152, "x": "bf16", "q": "e4m3",
         "block_rows": 1, "plain": True, "transposed": False, "pad": 0},
        # QKV's gradient of a micro-batch: rows for the input's gradient, columns for the weight's.
        {"name": "quant 12288x2304 bf16 both", "kind": "quant", "rows": 12288, "cols": 2304, "x": "bf16",
         "q": "e5m2", "block_rows": 1, "plain": True, "transposed": True, "pad": 0},
        # One token through QKV.
        {"name": "gemm 1x2304x768", "kind": "gemm", "M": 1, "N": 2304, "K": 768, "a": "e4m3", "b": "e4m3",
         "c": "bf16", "b_rows": 128, "pad": 0, "accumulate": False},
        # A short request through a wide model's product: the weights' bytes.
        {"name": "gemm 64x8192x4096", "kind": "gemm", "M": 64, "N": 8192, "K": 4096, "a": "e4m3", "b": "e4m3",
         "c": "bf16", "b_rows": 128, "pad": 0, "accumulate": False},
        # QKV of the serving batch.
        {"name": "gemm 32768x2304x768", "kind": "gemm", "M": 32768, "N": 2304, "K": 768, "a": "e4m3", "b": "e4m3",
         "c": "bf16", "b_rows": 128, "pad": 0, "accumulate": False},
        # A wide model's product, every size odd or ending inside a block.
        {"name": "gemm 4001x4099x8200", "kind": "gemm", "M": 4001, "N": 4099, "K": 8200, "a": "e4m3", "b": "e4m3",
         "c": "fp16", "b_rows": 128, "pad": 0, "accumulate": False},
        # QKV's weight gradient of a micro-batch, added to an earlier one's: a long sum, few outputs.
        {"name": "wgrad 2304x768x12288", "kind": "gemm", "M": 2304, "N": 768, "K": 12288, "a": "e5m2", "b": "e4m3",
         "c": "fp32", "b_rows": 1, "pad": 0, "accumulate": True},
    ]


_MOST = 4096 * 8192  # elements of a case's largest array
_MOST_FLOPS = 4001 * 4099 * 8200


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng):
    return rng.choice([384, 768, 768, 1152, 2304, 1024, 4096, 8192, _log_int(rng, 5, 8192), _log_int(rng, 5, 8192)])


def draw(rng):
    kind = rng.choice(["rms", "rms_grad", "quant", "gemm", "gemm", "gemm"])
    # Row strides: whole vectors of 16 mostly, as a program that chooses them would have them, or any.
    pad = rng.choice([0, 0, 0, 16, rng.randint(1, 40)])
    half = rng.choice(["bf16", "fp16"])
    if kind == "gemm":
        wgrad = rng.random() < 0.3
        M, N, K = (_width(rng), _width(rng), _log_int(rng, 1, 40000)) if wgrad else \
            (_log_int(rng, 1, 40000), _width(rng), _width(rng))
        if wgrad:
            K = max(1, min(K, _MOST // max(M, N), _MOST_FLOPS // (M * N)))
        else:
            M = max(1, min(M, 4 * _MOST // max(N, K), _MOST_FLOPS // (N * K)))
        return {"kind": kind, "M": M, "N": N, "K": K, "a": "e5m2" if wgrad else rng.choice(["e4m3", "e4m3", "e5m2"]),
                "b": "e4m3", "c": "fp32" if wgrad else rng.choice([half, half, "fp32"]), "b_rows": 1 if wgrad else 128,
                "pad": pad, "accumulate": wgrad and rng.random() < 0.5}
    cols = _width(rng)
    rows = _log_int(rng, 1, min(40000, _MOST // cols))
    case = {"kind": kind, "rows": rows, "cols": cols, "pad": pad}
    if kind == "quant":
        plain, transposed = rng.choice([(True, False), (True, True), (False, True)])
        return {**case, "x": rng.choice([half, half, "fp32"]), "q": rng.choice(["e4m3", "e5m2"]),
                "block_rows": rng.choice([1, 1, 128]), "plain": plain, "transposed": transposed}
    x, s = rng.choice([("fp32", "fp32"), (half, "fp32"), (half, half)])
    if kind == "rms":
        residual = rng.random() < 0.8
        return {**case, "x": x, "stream": s if residual else x, "y": rng.choice([None, None, x]), "q": "e4m3",
                "residual": residual}
    return {**case, "dy": x, "stream": s, "x": rng.choice([None, x]), "accumulate": rng.random() < 0.5}


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _wide(n, pad):
    """The row stride of an array of n columns: whole vectors of 16, or `pad` more elements than the row has."""
    return (n + 15) // 16 * 16 if pad == 0 else n + pad


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, pad = case["kind"], case["pad"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def empty(rows, cols, dtype):
        return torch.empty(rows, _wide(cols, pad), dtype=_TYPES[dtype], device="cuda")[:, :cols]

    def placed(values, dtype):
        t = empty(*values.shape, dtype)
        t.copy_(values)
        return t

    def stream(rows, cols):
        """A residual stream's rows: a scale each, every 97th column ten times as large."""
        v = normal(rows, cols) * (0.5 + normal(rows, 1).abs())
        v[:, ::97] *= 10
        return v

    def scales(rows, cols, block_rows=1):
        return torch.empty(_blocks(cols), rows if block_rows == 1 else _blocks(rows), device="cuda")

    st = {"case": case, "stream": torch.cuda.current_stream().cuda_stream}
    if kind == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        if case["b_rows"] == 128:  # activations by a weight
            a, b = stream(M, K), 0.02 * normal(N, K)
        else:  # a weight's gradient: both factors transposed, the sum over the tokens
            a, b = 0.01 * normal(M, K) * (1 + normal(1, K).abs()), stream(K, N).t()
        for name, v, block_rows in (("a", a, 1), ("b", b, case["b_rows"])):
            q, scale = _quantised(v, case[name], block_rows)
            st[name], st["s" + name] = empty(*v.shape, case[name]), scale
            st[name].view(torch.uint8).copy_(q.view(torch.uint8))
        st["c"] = empty(M, N, case["c"])
        st["c0"] = normal(M, N) if case["accumulate"] else None  # what earlier micro-batches left
        return st
    rows, cols = case["rows"], case["cols"]
    if kind == "quant":
        st["x"] = placed(0.02 * stream(rows, cols), case["x"])
        r = case["block_rows"]
        if case["plain"]:
            st["q"], st["scale"] = empty(rows, cols, case["q"]), scales(rows, cols, r)
        if case["transposed"]:
            st["qt"], st["scalet"] = empty(cols, rows, case["q"]), scales(cols, rows, r)
        return st
    st["w"] = 1 + 0.1 * normal(cols)
    if kind == "rms":
        st["x"] = placed(normal(rows, cols) if case["residual"] else stream(rows, cols), case["x"])
        if case["residual"]:
            st["res"], st["h"] = placed(stream(rows, cols), case["stream"]), empty(rows, cols, case["stream"])
        st["y"] = empty(rows, cols, case["y"]) if case["y"] else None
        st["q"], st["scale"] = empty(rows, cols, case["q"]), scales(rows, cols)
        st["rstd"] = torch.empty(rows, device="cuda")
        return st
    # The forward's kept stream and its statistics, and gradients of a loss summed over the batch.
    st["h"] = placed(stream(rows, cols), case["stream"])
    st["rstd"] = (st["h"].double().square().mean(1) + EPS).rsqrt().float()
    st["dy"] = placed(0.02 * normal(rows, cols) * (1 + normal(rows, 1).abs()), case["dy"])
    st["dh"], st["dres"] = placed(0.02 * normal(rows, cols), case["stream"]), empty(rows, cols, case["stream"])
    st["dx"] = empty(rows, cols, case["x"]) if case["x"] else None
    st["dw0"] = normal(cols)  # what earlier micro-batches left
    return st


# The plain forms.


def _spread(scale, rows, cols, block_rows):
    """The scale of every element, [rows, cols]."""
    s = scale.t().repeat_interleave(BLOCK, 1)[:, :cols]
    return s if block_rows == 1 else s.repeat_interleave(BLOCK, 0)[:rows]


def _quantised(v, dtype, block_rows=1):
    """(8-bit values, scales) of v in 32 bits."""
    rows, cols = v.shape
    tall = rows if block_rows == 1 else _blocks(rows) * BLOCK
    padded = torch.zeros(tall, _blocks(cols) * BLOCK, device=v.device)
    padded[:rows, :cols] = v.abs()
    largest = padded.view(tall // block_rows, block_rows, -1, BLOCK).amax((1, 3)).clamp(min=2.0 ** -100)
    scale = (largest / _LARGEST[dtype]).t().contiguous()
    return (v / _spread(scale, rows, cols, block_rows)).to(_TYPES[dtype]), scale


def _plain(st):
    case, kind = st["case"], st["case"]["kind"]
    if kind == "gemm":
        a = st["a"].float() * _spread(st["sa"], case["M"], case["K"], 1)
        b = st["b"].float() * _spread(st["sb"], case["N"], case["K"], case["b_rows"])
        c = a @ b.t()
        return (st["c0"] + c if case["accumulate"] else c).to(_TYPES[case["c"]])
    if kind == "quant":
        x = st["x"].float()
        return (_quantised(x, case["q"], case["block_rows"]) if case["plain"] else None,
                _quantised(x.t(), case["q"], case["block_rows"]) if case["transposed"] else None)
    if kind == "rms":
        h = st["x"].float()
        if case["residual"]:
            # The backward pass reads h as it is stored, so the norm is of that too.
            h = (st["res"].float() + h).to(_TYPES[case["stream"]]).float()
        rstd = ((h * h).mean(1, keepdim=True) + EPS).rsqrt()
        y = h * rstd * st["w"]
        return (h.to(_TYPES[case["stream"]]) if case["residual"] else None, *_quantised(y, case["q"]),
                y.to(_TYPES[case["y"]]) if case["y"] else None, rstd[:, 0])
    dy, rstd = st["dy"].float(), st["rstd"][:, None]
    xh, g = st["h"].float() * rstd, dy * st["w"]
    dres = st["dh"].float() + rstd * (g - xh * (g * xh).mean(1, keepdim=True))
    dw = (dy * xh).sum(0)
    return (dres.to(_TYPES[case["stream"]]), dres.to(_TYPES[case["x"]]) if case["x"] else None,
            st["dw0"] + dw if case["accumulate"] else dw)


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
    """(address, row stride) of an array; what the state lacks is not there."""
    return (None, 0) if t is None else (t.data_ptr(), t.stride(0))


def _work(st, size):
    """A workspace that the program keeps with its arrays."""
    if "work" not in st:
        st["work"] = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
    return st["work"].data_ptr(), st["work"].numel()


def _own(st):
    case, kind, eng = st["case"], st["case"]["kind"], _engine(st["stream"])
    if kind == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        c = st["c"]
        if case["accumulate"]:
            c.copy_(st["c0"])
        eng.gemm_fp8_device(case["a"], case["b"], case["c"], M, N, K, *_at(st["a"]), *_at(st["sa"]), *_at(st["b"]),
                            case["b_rows"], *_at(st["sb"]), *_at(c), case["accumulate"],
                            *_work(st, eng.gemm_fp8_workspace(M, N, K)))
        return c
    rows, cols = case["rows"], case["cols"]
    if kind == "quant":
        q, scale, qt, scalet = (st.get(k) for k in ("q", "scale", "qt", "scalet"))
        eng.quantize_blocks_device(case["x"], case["q"], rows, cols, case["block_rows"], *_at(st["x"]), *_at(q),
                                   *_at(scale), *_at(qt), *_at(scalet))
        return (q, scale) if case["plain"] else None, (qt, scalet) if case["transposed"] else None
    if kind == "rms":
        eng.add_rms_norm_device(case["x"], case["stream"], case["y"] or case["x"], case["q"], rows, cols,
                                *_at(st["x"]), *_at(st.get("res")), st["w"].data_ptr(), EPS, *_at(st.get("h")),
                                *_at(st["y"]), *_at(st["q"]), *_at(st["scale"]), st["rstd"].data_ptr())
        return st.get("h"), st["q"], st["scale"], st["y"], st["rstd"]
    dw = st["dw0"].clone() if case["accumulate"] else torch.empty_like(st["dw0"])
    eng.add_rms_norm_backward_device(case["dy"], case["stream"], case["x"] or case["dy"], rows, cols, *_at(st["dy"]),
                                     *_at(st["dh"]), *_at(st["h"]), st["w"].data_ptr(), st["rstd"].data_ptr(),
                                     *_at(st["dres"]), *_at(st["dx"]), dw.data_ptr(), case["accumulate"],
                                     *_work(st, eng.norm_backward_workspace(rows, cols)))
    return st["dres"], st["dx"], dw


def run(st):
    return _own(st) if own else _plain(st)


def work(case):
    kind = case["kind"]
    if kind == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        scales = _blocks(K) * (M + (N if case["b_rows"] == 1 else _blocks(N)))
        out = M * N * _SIZE[case["c"]] * (2 if case["accumulate"] else 1)
        return {"bytes": M * K + N * K + 4 * scales + out, "flops": 2 * M * N * K}
    rows, cols = case["rows"], case["cols"]
    n = rows * cols
    if kind == "quant":
        sides = case["plain"] + case["transposed"]
        each = n // (BLOCK * case["block_rows"])
        return {"bytes": n * (_SIZE[case["x"]] + sides) + 4 * sides * each, "flops": (1 + 2 * sides) * n}
    if kind == "rms":
        size = _SIZE[case["x"]] + 1 + (2 * _SIZE[case["stream"]] if case["residual"] else 0)
        size += _SIZE[case["y"]] if case["y"] else 0
        return {"bytes": n * size + 4 * rows * (_blocks(cols) + 1) + 4 * cols, "flops": 7 * n}
    size = _SIZE[case["dy"]] + 3 * _SIZE[case["stream"]] + (_SIZE[case["x"]] if case["x"] else 0)
    return {"bytes": n * size + 4 * rows + 4 * cols * (3 if case["accumulate"] else 2), "flops": 11 * n}


# The definition in 64 bits.


def _nearest(v, dtype):
    """v at the type's nearest values, ties to the even one: 3 or 2 bits behind the leading one, exponents from -6 or
    -14 on."""
    bits, least = (3, -6) if dtype == "e4m3" else (2, -14)
    step = torch.exp2(torch.frexp(v)[1].sub(1).clamp(min=least).double() - bits)
    return torch.round(v / step) * step


def _split(v, dtype, block_rows):
    """(values in units of the scale, scales), block by block."""
    rows, cols = v.shape
    q, scales = torch.empty_like(v), []
    for c in range(0, cols, BLOCK):
        part = v[:, c:c + BLOCK]
        m = part.abs().max(1).values
        if block_rows > 1:
            m = torch.stack([p.max() for p in m.split(block_rows)])
        s = torch.clamp(m, min=2.0 ** -100) / _LARGEST[dtype]
        each = s if block_rows == 1 else torch.cat([s[i].expand(p) for i, p in enumerate(
            [min(block_rows, rows - r) for r in range(0, rows, block_rows)])])
        q[:, c:c + BLOCK] = _nearest(part / each[:, None], dtype)
        scales.append(s)
    return q, torch.stack(scales)


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        c = st["c0"].double() if case["accumulate"] else torch.zeros(M, N, dtype=torch.float64, device="cuda")
        column = torch.arange(N, device="cuda") // case["b_rows"]
        for b in range(_blocks(K)):
            at = slice(b * BLOCK, min(K, (b + 1) * BLOCK))
            a = st["a"][:, at].double() * st["sa"][b].double()[:, None]
            c += torch.mm(a, (st["b"][:, at].double() * st["sb"][b].double()[column][:, None]).t().contiguous())
        return c
    if kind == "quant":
        x, r = st["x"].double(), case["block_rows"]
        return (_split(x, case["q"], r) if case["plain"] else None,
                _split(x.t().contiguous(), case["q"], r) if case["transposed"] else None)
    n = case["cols"]
    if kind == "rms":
        h = st["x"].double()
        kept = None
        if case["residual"]:
            kept = h + st["res"].double()
            h = kept.to(_TYPES[case["stream"]]).double()
        rstd = 1 / torch.sqrt(h.pow(2).sum(1) / n + EPS)
        y = h * st["w"].double() * rstd[:, None]
        return (kept, *_split(y, case["q"], 1), y if case["y"] else None, rstd)
    rstd, dy = st["rstd"].double()[:, None], st["dy"].double()
    unit = st["h"].double() * rstd
    through = dy * st["w"].double()
    dres = st["dh"].double() + (through - unit * ((through * unit).sum(1, keepdim=True) / n)) * rstd
    dw = torch.einsum("rc,rc->c", dy, unit)
    return dres, dres if case["x"] else None, dw + st["dw0"].double() if case["accumulate"] else dw
