"""The work of a ray head's operators, as cases for measuring it.

A ray head is a small network behind the tracer: it takes what was traced (or
stored) for each ray, pixel or cell and gives corrected colours, features or
scores.  Its operators hold numbers in microscaled formats, blocks of 32
consecutive values of a row under one power of two:

* ``store``: rows quantised to 4 bits (e2m1 values, e8m0 scales) and read back;
* ``linear``: a product with weights held in 4 bits, its rows quantised on the
  way or already stored;
* ``mlp``: a whole head of such layers with ReLU between them;
* ``activation``: an activation that keeps its input in 8 bits (e4m3 values,
  e8m0 scales) for the backward pass, and that backward pass;
* ``weights``: the gradient of the weights and the bias of the layer behind
  such an activation, from the 8-bit checkpoint.

The plain forms are elementary torch operations in 32 bits; ``exact`` states
the operators again in 64.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
BLOCK = 32
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
RAYS_FRAME = 1237 * 822  # the evaluation render
RAYS_BATCH = 800 * 600  # a training batch
CELLS = 1048576


def listed():
    return [
        # Features of a few picked cells put away, and read back for display: the smallest call.
        dict(name="store picks", kind="store", rows=7, width=100, dtype="f32"),
        # Features of every cell of the million-site scene, quantised when the scene is prepared for serving.
        dict(name="store cells", kind="store", rows=CELLS, width=256, dtype="bf16"),
        # One picked ray through a layer: a single row, where latency counts.
        dict(name="linear pick", kind="linear", rows=1, width=512, out=768, dtype="bf16", stored=False, relu=False,
             result="bf16"),
        # Scores of every stored cell against a few dozen queries: reads the store once.
        dict(name="linear scores", kind="linear", rows=CELLS, width=512, out=48, dtype="f32", stored=True, relu=False,
             result="f32"),
        # A hidden layer over the pixels of the evaluation render.
        dict(name="linear frame", kind="linear", rows=RAYS_FRAME, width=256, out=256, dtype="bf16", stored=False,
             relu=True, result="bf16"),
        # A wide layer over a 128x128 image, bound by its products.
        dict(name="linear wide", kind="linear", rows=16384, width=2048, out=2048, dtype="f16", stored=False, relu=False,
             result="f16"),
        # A small head for the rays of one click.
        dict(name="mlp picks", kind="mlp", rows=13, width=60, hidden=128, layers=3, out=33, dtype="f32", result="f32"),
        # The head over the evaluation render, per frame.
        dict(name="mlp frame", kind="mlp", rows=RAYS_FRAME, width=64, hidden=256, layers=4, out=64, dtype="bf16",
             result="bf16"),
        # A training patch of odd width with a smooth activation.
        dict(name="activation patch", kind="activation", rows=1000, width=77, dtype="f32", act="silu"),
        # The hidden activations of a training batch of 480,000 rays.
        dict(name="activation batch", kind="activation", rows=RAYS_BATCH, width=256, dtype="bf16", act="relu"),
        # Weight gradients of an odd layer over a small ragged batch.
        dict(name="weights patch", kind="weights", rows=5009, width=333, out=200, dtype="f16", act="gelu"),
        # Weight gradients of a hidden layer over the training batch: a long sum into a small result.
        dict(name="weights batch", kind="weights", rows=RAYS_BATCH, width=256, out=256, dtype="bf16", act="relu"),
    ]


def _log(rng, lo, hi):
    """A size spread over the logarithm of its range, odd as often as not."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "linear", "mlp", "activation", "weights"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "store":
        width = _log(rng, 1, 1024)
        return dict(kind=kind, rows=_log(rng, 1, min(CELLS, CELLS * 128 // width)), width=width, dtype=dtype)
    if kind == "linear":
        width, out = _log(rng, 24, 2048), _log(rng, 8, 2048)
        rows = _log(rng, 1, min(RAYS_FRAME, 16384 * 2048 * 1024 // (width * out), RAYS_FRAME * 256 // (width + out)))
        return dict(kind=kind, rows=rows, width=width, out=out, dtype=dtype, stored=rng.random() < 0.3,
                    relu=rng.random() < 0.5, result=rng.choice(["f32", dtype]))
    if kind == "mlp":
        return dict(kind=kind, rows=_log(rng, 1, RAYS_FRAME // 2), width=_log(rng, 3, 256), hidden=_log(rng, 16, 256),
                    layers=rng.randint(2, 5), out=_log(rng, 1, 256), dtype=dtype,
                    result="bf16" if dtype == "f32" else dtype)
    act = rng.choice(["none", "relu", "silu", "gelu"])
    if kind == "activation":
        width = _log(rng, 8, 1024)
        return dict(kind=kind, rows=_log(rng, 1, min(RAYS_BATCH, RAYS_BATCH * 128 // width)), width=width, dtype=dtype,
                    act=act)
    width, out = _log(rng, 8, 1024), _log(rng, 8, 1024)
    rows = _log(rng, 1, min(RAYS_BATCH, RAYS_BATCH * 256 * 128 // (width * out), RAYS_BATCH * 128 // (width + out)))
    return dict(kind=kind, rows=rows, width=width, out=out, dtype=dtype, act=act)


# ---- the plain forms


def _blocks(x):
    """x (rows, width) f32 as (rows, blocks, 32), the last block filled up with zeros, and the exponent of each
    block's largest magnitude (floor(log2), far below any for a block of zeros)."""
    pad = -x.shape[1] % BLOCK
    b = torch.nn.functional.pad(x, (0, pad)).reshape(x.shape[0], -1, BLOCK)
    top = b.abs().amax(-1, keepdim=True)
    return b, torch.where(top > 0, torch.frexp(top).exponent - 1, -300)


def _exp2(e):
    """2^e in f32 for whole e from -127 to 127."""
    return torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)


def _mx4(x):
    """Rows in 4 bits: the values (rows, blocks, 32) in units of their scale, and the exponents of the scales."""
    b, top = _blocks(x)
    e = (top - 2).clamp(-127, 127)
    v = b * _exp2(-e)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign((torch.round(a / step) * step).clamp(max=6.0), v), e


def _mx4_pack(x):
    """Codes and scales as they are stored: e2m1 nibbles, the lower one first, and e8m0 bytes."""
    v, e = _mx4(x)
    a = v.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code + torch.signbit(v).to(torch.uint8) * 8
    code = code.reshape(x.shape[0], -1, 2)
    return code[..., 0] + code[..., 1] * 16, (e + 127).to(torch.uint8).reshape(x.shape[0], -1)


def _mx4_read(codes, scales, width):
    """The values that codes and scales stand for, (rows, width) f32."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    table = torch.cat([table, -table])
    n = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1, BLOCK)
    v = table[n.to(torch.int32)] * _exp2(scales.to(torch.int32) - 127)[..., None]
    return v.reshape(codes.shape[0], -1)[:, :width]


def _mx4_round(x):
    v, e = _mx4(x)
    return (v * _exp2(e)).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _ckpt8_pack(x):
    """The 8-bit checkpoint of x: e4m3 bytes (rows, width) and e8m0 scales.  Nothing but zero becomes zero."""
    b, top = _blocks(x)
    e = (top - 7).clamp(-127, 127)
    v = b * _exp2(-e)
    q = v.to(torch.float8_e4m3fn).to(torch.float32)
    q = torch.where((q == 0) & (b != 0), torch.copysign(torch.full_like(q, 2.0 ** -9), b), q)
    q = q.to(torch.float8_e4m3fn).view(torch.uint8).reshape(x.shape[0], -1)[:, :x.shape[1]]
    return q.contiguous(), (e + 127).to(torch.uint8).reshape(x.shape[0], -1)


def _ckpt8_read(codes, scales):
    v = codes.view(torch.float8_e4m3fn).to(torch.float32)
    return v * _exp2(scales.to(torch.int32) - 127).repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]


def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


# ---- inputs


def _rows(g, rows, width, dtype):
    """Values of a hidden layer: rows of unlike size, and zeros where a ray met nothing (one in sixteen)."""
    x = torch.randn(rows, width, generator=g, device=DEV)
    size = torch.exp2(2 * torch.rand(rows, 1, generator=g, device=DEV) - 1)
    met = (torch.rand(rows, 1, generator=g, device=DEV) > 1 / 16) | (torch.arange(rows, device=DEV)[:, None] == 0)
    return (x * size * met).to(dtype)


def _layer(g, width, out):
    codes, scales = _mx4_pack(torch.randn(out, width, generator=g, device=DEV) / math.sqrt(width))
    return codes, scales, width, 0.1 * torch.randn(out, generator=g, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    state = dict(case=case, result=TYPES[case.get("result", case["dtype"])])
    x = _rows(g, case["rows"], case["width"], dtype)
    if case["kind"] == "linear":
        state["layers"] = [_layer(g, case["width"], case["out"])]
        if case["stored"]:
            state["x"] = _mx4_pack(x.to(torch.float32))
            return state
    elif case["kind"] == "mlp":
        widths = [case["width"]] + [case["hidden"]] * (case["layers"] - 1) + [case["out"]]
        state["layers"] = [_layer(g, a, b) for a, b in zip(widths, widths[1:])]
    elif case["kind"] == "activation":
        state["dy"] = (0.01 * torch.randn(x.shape, generator=g, device=DEV)).to(dtype)
    elif case["kind"] == "weights":
        state["dy"] = (0.01 * torch.randn(case["rows"], case["out"], generator=g, device=DEV)).to(dtype)
        x = _ckpt8_pack(x.to(torch.float32))
    state["x"] = x
    return state


# ---- one pass


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from vorotracing_amd import micro

    case, x = state["case"], state["x"]
    kind = case["kind"]
    if kind == "store":
        return micro.quantize_mx4(x).dequantize(x.dtype)
    if kind == "linear":
        codes, scales, width, bias = state["layers"][0]
        x = micro.Mx4(*x, case["width"]) if case["stored"] else x
        return micro.linear_mx4(x, micro.Mx4(codes, scales, width), bias, relu=case["relu"], dtype=state["result"])
    if kind == "mlp":
        layers = [(micro.Mx4(codes, scales, width), bias) for codes, scales, width, bias in state["layers"]]
        return micro.mlp_mx4(x, layers, dtype=state["result"])
    if kind == "activation":
        y, kept = micro.checkpoint_activation(x, case["act"])
        return {"y": y, "dz": kept.input_grad(state["dy"])}
    dw, db = micro.Checkpoint8(*x, case["act"]).weight_grad(state["dy"])
    return {"dw": dw, "db": db}


def _run_plain(state):
    case, x = state["case"], state["x"]
    kind = case["kind"]
    if kind == "store":
        return _mx4_round(x.to(torch.float32)).to(x.dtype)
    if kind in ("linear", "mlp"):
        h = _mx4_read(*x, case["width"]) if case.get("stored") else _mx4_round(x.to(torch.float32))
        for codes, scales, width, bias in state["layers"][:-1]:
            h = _mx4_round(torch.clamp(h @ _mx4_read(codes, scales, width).T + bias, min=0))
        codes, scales, width, bias = state["layers"][-1]
        y = h @ _mx4_read(codes, scales, width).T + bias
        return (torch.clamp(y, min=0) if case.get("relu") else y).to(state["result"])
    if kind == "activation":
        z = x.to(torch.float32)
        kept = _ckpt8_read(*_ckpt8_pack(z))
        dz = state["dy"].to(torch.float32) * _act_slope(kept, case["act"])
        return {"y": _act(z, case["act"]).to(x.dtype), "dz": dz.to(x.dtype)}
    dy = state["dy"].to(torch.float32)
    return {"dw": dy.T @ _act(_ckpt8_read(*x), case["act"]), "db": dy.sum(0)}


# ---- what a pass cannot do without


def work(case):
    rows, width = case["rows"], case["width"]
    size = 4 if case["dtype"] == "f32" else 2
    result = 4 if case.get("result", case["dtype"]) == "f32" else 2
    kept4 = lambda r, w: r * -(-w // BLOCK) * 17  # noqa: E731
    kept8 = rows * (width + -(-width // BLOCK))
    if case["kind"] == "store":  # in, the store, out
        return {"bytes": 2 * rows * width * size + kept4(rows, width), "flops": 2 * rows * width}
    if case["kind"] == "linear":
        out = case["out"]
        read = kept4(rows, width) if case["stored"] else rows * width * size
        return {"bytes": read + kept4(out, width) + 4 * out + rows * out * result, "flops": 2 * rows * width * out}
    if case["kind"] == "mlp":
        widths = [width] + [case["hidden"]] * (case["layers"] - 1) + [case["out"]]
        pairs = list(zip(widths, widths[1:]))
        return {"bytes": rows * (width * size + case["out"] * result) + sum(kept4(b, a) + 4 * b for a, b in pairs),
                "flops": 2 * rows * sum(a * b for a, b in pairs)}
    if case["kind"] == "activation":  # z and dy in, y and dz out, the checkpoint kept
        return {"bytes": 4 * rows * width * size + kept8, "flops": 8 * rows * width}
    out = case["out"]
    return {"bytes": kept8 + rows * out * size + 4 * out * (width + 1), "flops": 2 * rows * width * out}


# ---- the same from the definitions, in 64 bits


def _exact_scaled(x, largest):
    """x (f64) by blocks of 32 over 2^e, the scale under which the block's largest magnitude lies in
    [2^largest, 2^(largest + 1)): (quotients, scales)."""
    rows, width = x.shape
    n = -(-width // BLOCK)
    b = torch.zeros(rows, n * BLOCK, dtype=torch.float64, device=x.device)
    b[:, :width] = x
    b = b.view(rows, n, BLOCK)
    top = b.abs().amax(2, keepdim=True)
    mantissa, exponent = torch.frexp(torch.where(top > 0, top, torch.ones_like(top)))
    e = torch.where(top > 0, exponent - 1 - largest, -127).clamp(-127, 127).to(torch.float64)
    return b / torch.exp2(e), torch.exp2(e)


def _exact_mx4(x):
    q, s = _exact_scaled(x, 2)
    # the midpoints between 0, 1/2, 1, 3/2, 2, 3, 4, 6; at a midpoint the value of even code is taken
    values = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    middle = (values[1:] + values[:-1]) / 2
    a = q.abs().contiguous()
    below = torch.searchsorted(middle, a, right=False)  # a midpoint goes down
    above = torch.searchsorted(middle, a, right=True)  # a midpoint goes up
    code = torch.where(below % 2 == 0, below, above)
    out = torch.sign(q) * values[code] * s
    return out.reshape(x.shape[0], -1)[:, :x.shape[1]]


def _exact_weights(codes, scales, width):
    magnitude = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], dtype=torch.float64, device=codes.device) / 2
    out = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device=codes.device)
    for half, nibble in enumerate((codes % 16, codes // 16)):
        out[:, half::2] = magnitude[(nibble % 8).long()] * (1 - 2 * (nibble // 8).double())
    out = out * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, dim=1)
    return out[:, :width]


def _exact_kept(x):
    """x by its 8-bit checkpoint: three bits behind the leading one, 2^-9 of the scale at least."""
    q, s = _exact_scaled(x, 7)
    a = q.abs()
    _, exponent = torch.frexp(a)
    step = torch.exp2((exponent - 1).clamp(min=-6).double() - 3)
    near = torch.round(a / step) * step  # half to even
    near = torch.where((a > 0) & (near == 0), torch.full_like(near, 2.0 ** -9), near)
    return (torch.sign(q) * near * s).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _exact_kept_read(codes, scales):
    exponent, mantissa = (codes // 8 % 16).double(), (codes % 8).double()
    v = torch.where(exponent > 0, torch.exp2(exponent - 7) * (1 + mantissa / 8), mantissa * 2.0 ** -9)
    v = v * (1 - 2 * (codes // 128).double())
    return v * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, dim=1)[:, :codes.shape[1]]


def _exact_act(z, act):
    """(value, slope) of the activation."""
    if act == "relu":
        return torch.maximum(z, torch.zeros_like(z)), torch.heaviside(z, torch.zeros_like(z))
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    if act == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def exact(case, seed):
    state = prepare(case, seed)
    x = state["x"]
    if case["kind"] == "store":
        return _exact_mx4(x.double())
    if case["kind"] in ("linear", "mlp"):
        h = _exact_weights(*x, case["width"]) if case.get("stored") else _exact_mx4(x.double())
        last = len(state["layers"]) - 1
        for i, (codes, scales, width, bias) in enumerate(state["layers"]):
            h = torch.matmul(h, _exact_weights(codes, scales, width).t()) + bias.double()
            if i < last:
                h = _exact_mx4(h.clamp_(min=0))
        return h.clamp_(min=0) if case.get("relu") else h
    if case["kind"] == "activation":
        z = x.double()
        return {"y": _exact_act(z, case["act"])[0],
                "dz": state["dy"].double() * _exact_act(_exact_kept(z), case["act"])[1]}
    dy = state["dy"].double()
    return {"dw": torch.matmul(dy.t(), _exact_act(_exact_kept_read(*x), case["act"])[0]), "db": dy.sum(dim=0)}
