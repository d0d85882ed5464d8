"""The calls of the microscaled operators (``lich_amd.microscale``) by which their speed is judged.

Microscaled storage (OCP MX): 32 consecutive values of a row share one
power-of-two scale.  Two element formats: ``fp4`` (E2M1, weights and the
operands of a product) and ``int8`` (states kept for the backward pass).

Four kinds of call, each in its plain form (elementary torch operations in 32
bits) and, with ``own`` set, through the package's entry points:

* ``pack``     a matrix into microscaled storage and back: 8-bit checkpoints
               of states restored, weights laid out in 4 bits;
* ``product``  one kernel family of the training step with both operands in 4
               bits: f(X) (and E) quantised in the call, W kept quantised,
               the product and its fused epilogue;
* ``serve``    a forward pass of few samples: 4-bit weights, 16- or 32-bit
               states;
* ``backward`` the state X kept in 8 bits, then the weight update and the
               state gradient that read it there.

Quantisation picks among discrete values: an activation whose last bit differs
between two correct evaluations can pick another one.  The timed calls that
quantise take relu or identity, which are exact; the others take any.
"""
from __future__ import annotations

import math
from collections import namedtuple

import torch

own = False

BLOCK = 32
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ACTIVATIONS = ("relu", "tanh", "sigmoid", "silu", "gelu")
ALPHA, GAMMA = 1e-2, 0.5
Packed = namedtuple("Packed", "codes scales")


# ------------------------------------------------------------------ the cases
def _pack(name, rows, cols, storage, fmt, axis, activation="identity"):
    return {"name": name, "kind": "pack", "rows": rows, "cols": cols, "storage": storage, "format": fmt, "axis": axis,
            "activation": activation}


def _layer(name, kind, op, M, K, B, storage, activation):
    return {"name": name, "kind": kind, "op": op, "M": M, "K": K, "batch": B, "storage": storage,
            "activation": activation}


def listed():
    return [
        # The states of one hidden layer of the wide net into an 8-bit checkpoint and back.
        _pack("pack_states", 4096, 1024, "bf16", "int8", 1),
        # A wide layer's fp32 weights laid out in 4 bits for the product that reads them transposed.
        _pack("pack_weights_transposed", 4096, 4096, "fp32", "fp4", 0),
        # The first layer of the image nets: latency and launches.
        _layer("product_first_layer", "product", "pred", 64, 784, 128, "fp32", "relu"),
        # A layer of the wide net: prediction error of a training batch.
        _layer("product_wide_pred", "product", "pred", 4096, 4096, 1024, "bf16", "relu"),
        # A weight update at odd sizes over fp32 master weights.
        _layer("product_ragged_weight", "product", "weight", 1000, 1531, 300, "fp32", "relu"),
        # The inference update of a large layer.
        _layer("product_large_infer", "product", "infer", 8192, 8192, 2048, "bf16", "identity"),
        # Scoring a large batch with a large layer.  The largest work there is.
        _layer("product_large_forward", "product", "forward", 8192, 8192, 8192, "bf16", "relu"),
        # One sample through a wide layer: the online path's latency, bound by the weights' bytes.
        _layer("serve_one", "serve", "predict", 4096, 4096, 1, "bf16", "tanh"),
        # A few samples through the wide net's output layer, states in fp32.
        _layer("serve_few", "serve", "predict", 1000, 4096, 12, "fp32", "gelu"),
        # The first layer of the image nets in the reference's own storage type.
        _layer("backward_first_layer", "backward", "both", 64, 784, 128, "fp16", "tanh"),
        # Odd sizes, everything in fp32.
        _layer("backward_ragged", "backward", "both", 1000, 1531, 300, "fp32", "silu"),
        # A layer of the wide net at its batch.
        _layer("backward_wide", "backward", "both", 4096, 4096, 1024, "bf16", "tanh"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limit = work(listed()[6])["flops"]
    while True:
        kind = rng.choice(("pack", "product", "product", "serve", "backward", "backward"))
        storage = rng.choice(("fp32", "fp16", "bf16", "bf16"))
        even = rng.random() < 0.5  # half of the sizes are as even as real nets are
        def size(lo, hi):
            v = _log_int(rng, lo, hi)
            return max(lo, v // 64 * 64) if even else v
        if kind == "pack":
            fmt = rng.choice(("fp4", "int8"))
            case = _pack("", size(1, 8192), size(1, 8192), storage, fmt, rng.choice((0, 1)),
                         rng.choice(("identity", "relu")))
        elif kind == "product":
            case = _layer("", kind, rng.choice(("pred", "forward", "infer", "weight")), size(16, 8192), size(16, 8192),
                          size(1, 8192), storage, rng.choice(("identity", "relu")))
        elif kind == "serve":
            case = _layer("", kind, "predict", size(16, 8192), size(16, 8192), _log_int(rng, 1, 64), storage,
                          rng.choice(ACTIVATIONS))
        else:
            case = _layer("", kind, "both", size(16, 8192), size(16, 8192), size(1, 4096), storage,
                          rng.choice(ACTIVATIONS))
        # backward passes on fp32 operands run at a sixteenth of the 16-bit matrix rate
        cost = work(case)["flops"] * (8 if kind == "backward" and storage == "fp32" else 1)
        if cost <= limit / 2:
            del case["name"]
            return case


# ------------------------------------------------------------------ microscaled storage in plain torch
def _quantise(x, fmt):
    """The values that blocks of 32 along the last dimension of x (its length a
    multiple of 32) stand for, as (elements, exponents): value = element * 2^exponent."""
    b = x.reshape(x.shape[0], -1, BLOCK)
    m, e = torch.frexp(b.abs().amax(-1))
    # the exponent of the largest magnitude once that is rounded to the element's precision
    up = (m >= (0.875 if fmt == "fp4" else 1 - 2.0 ** -8)).to(e.dtype)
    e = (e - 1 + up - (2 if fmt == "fp4" else 0)).clamp(-126, 127)
    v = torch.ldexp(b, -e[..., None])
    if fmt == "fp4":
        a = v.abs()
        r = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2))
        v = torch.copysign(r.clamp(max=6.0), v)
    else:
        v = torch.round(v * 64).clamp(-127, 127) / 64
    return v, e


def _pad(x, multiple):
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % multiple))


def _quantised_values(x, fmt):
    v, e = _quantise(_pad(x.float(), BLOCK), fmt)
    return torch.ldexp(v, e[..., None]).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _pack_fp4(x):
    """x [rows, n] in the package's layout: rows padded with zeros to a multiple of
    128 values, two codes a byte (the lower value in the lower half); one scale
    byte (exponent + 127, 0 for a block of zeros) a block, [n / 128][rows][4]."""
    v, e = _quantise(_pad(x.float(), 128), "fp4")
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=x.device)
    code = torch.bucketize(v.abs(), grid) + 8 * (v < 0)
    code = code.reshape(x.shape[0], -1, 2).to(torch.uint8)
    zero = v.reshape(x.shape[0], e.shape[1], BLOCK).abs().amax(-1) == 0
    scales = torch.where(zero, 0, e + 127).to(torch.uint8).reshape(x.shape[0], -1, 4)
    return Packed((code[..., 0] | (code[..., 1] << 4)).contiguous(), scales.transpose(0, 1).contiguous())


def _unpack_fp4(packed, n):
    codes, scales = packed.codes, packed.scales.transpose(0, 1).reshape(packed.codes.shape[0], -1)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    grid = torch.cat([grid, -grid])
    v = grid[torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1).int()]
    v = torch.ldexp(v.reshape(*scales.shape, BLOCK), (scales.int() - 127)[..., None])
    return v.reshape(codes.shape[0], -1)[:, :n]


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt = DTYPES[case["storage"]]

    def normal(rows, cols, size=1.0):
        return (torch.randn((rows, cols), generator=g, device="cuda") * size).to(dt)

    if case["kind"] == "pack":
        return {"x": normal(case["rows"], case["cols"])}
    M, K, B = case["M"], case["K"], case["batch"]

    def weights(rows, cols):  # Xavier uniform, as the trainer's
        bound = math.sqrt(6.0 / (M + K))
        return ((torch.rand((rows, cols), generator=g, device="cuda") * 2 - 1) * bound).to(dt)

    if case["op"] == "pred":
        return {"x": normal(K, B), "w": weights(M, K), "x_lower": normal(M, B)}
    if case["op"] == "infer":  # W_lower [K, M]; errors a tenth of the states
        return {"x": normal(M, B), "e": normal(M, B, 0.1), "w": weights(K, M), "e_lower": normal(K, B, 0.1)}
    if case["op"] in ("weight", "both"):
        return {"x": normal(K, B), "w": weights(M, K), "e": normal(M, B, 0.1)}
    return {"x": normal(K, B), "w": weights(M, K)}


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    # products and serving keep their weights quantised (along the contraction), laid out once
    if case["kind"] in ("product", "serve") and case["op"] != "weight":
        w = state.pop("w")
        state["w4"] = _pack_fp4(w.T.contiguous() if case["op"] == "infer" else w)
    if case["kind"] == "pack":
        state["out"] = torch.empty_like(state["x"].T.contiguous() if case["axis"] == 0 else state["x"])
    elif case["op"] in ("pred", "forward", "predict"):
        state["out"] = torch.empty((case["M"], case["batch"]), dtype=DTYPES[case["storage"]], device="cuda")
    elif case["op"] == "both":
        state["grad"] = torch.empty_like(state["x"])
    return state


# ------------------------------------------------------------------ plain forms
def _f(name, x):
    if name == "relu":
        return torch.clamp(x, min=0)
    if name == "tanh":
        return torch.tanh(x)
    if name == "sigmoid":
        return torch.sigmoid(x)
    if name == "silu":
        return x * torch.sigmoid(x)
    if name == "gelu":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    return x


def _df(name, x):
    if name == "relu":
        return (x > 0).to(x.dtype)
    if name == "tanh":
        return 1 - torch.tanh(x) ** 2
    if name == "sigmoid":
        s = torch.sigmoid(x)
        return s * (1 - s)
    if name == "silu":
        s = torch.sigmoid(x)
        return s * (1 + x * (1 - s))
    if name == "gelu":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (x + 0.044715 * x ** 3))
        return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * k * (1 + 3 * 0.044715 * x * x)
    return torch.ones_like(x)


def _run_plain(s):
    case, act = s["case"], s["case"]["activation"]
    if case["kind"] == "pack":
        x = _f(act, s["x"].float())
        s["out"].copy_(_quantised_values(x.T if case["axis"] == 0 else x, case["format"]))
        return s["out"]
    if case["kind"] == "serve":
        s["out"].copy_(_unpack_fp4(s["w4"], case["K"]) @ _f(act, s["x"].float()))
        return s["out"]
    if case["kind"] == "backward":
        x8, e = _quantised_values(s["x"], "int8"), s["e"].float()
        s["grad"].copy_(_df(act, x8) * (s["w"].float().T @ e))
        s["w"].copy_(s["w"].float() + ALPHA * (e @ _f(act, x8).T))
        return {"w": s["w"], "grad": s["grad"]}
    if case["op"] in ("pred", "forward"):
        x4 = _quantised_values(_f(act, s["x"].float()).T, "fp4")
        y = _unpack_fp4(s["w4"], case["K"]) @ x4.T
        s["out"].copy_(s["x_lower"].float() - y if case["op"] == "pred" else y)
        return s["out"]
    if case["op"] == "infer":
        x = s["x"].float()
        up = _unpack_fp4(s["w4"], case["K"]) @ _quantised_values(s["e_lower"].T, "fp4").T
        s["x"].copy_(x + GAMMA * (_df(act, x) * up - s["e"].float()))
        return s["x"]
    e4, a4 = _quantised_values(s["e"], "fp4"), _quantised_values(_f(act, s["x"].float()), "fp4")
    s["w"].copy_(s["w"].float() + ALPHA * (e4 @ a4.T))
    return s["w"]


# ------------------------------------------------------------------ the package's calls
def _run_own(s):
    from lich_amd import microscale as mx

    case, act, dt = s["case"], s["case"]["activation"], DTYPES[s["case"]["storage"]]
    if case["kind"] == "pack":
        quantize = mx.build_mx_quantize(case["rows"], case["cols"], act, dt, format=case["format"], axis=case["axis"])
        packed = quantize.new_output(s["x"].device)
        quantize(s["x"], packed)
        mx.build_mx_dequantize(*s["out"].shape, dt, format=case["format"])(packed, s["out"])
        return s["out"]
    M, K, B, op = case["M"], case["K"], case["batch"], case["op"]
    if case["kind"] == "serve":
        predict = mx.build_mx_predict(M, K, B, act, dt)
        predict(s["x"], mx.MXMatrix(*s["w4"]), s["out"], workspace=predict.new_workspace(s["x"].device))
        return s["out"]
    if case["kind"] == "backward":
        save = mx.build_checkpoint_save(K, B, dt)
        x8 = save.new_output(s["x"].device)
        save(s["x"], x8)
        gradient = mx.build_checkpoint_gradient(K, M, B, act, dt)
        gradient(s["w"], s["e"], x8, s["grad"], workspace=gradient.new_workspace(s["x"].device))
        update = mx.build_checkpoint_weight_update(M, K, B, act, dt, ALPHA)
        update(s["w"], s["e"], x8, workspace=update.new_workspace(s["x"].device))
        return {"w": s["w"], "grad": s["grad"]}

    def packed4(x, rows, cols, activation, axis):
        quantize = mx.build_mx_quantize(rows, cols, activation, dt, format="fp4", axis=axis)
        out = quantize.new_output(x.device)
        quantize(x, out)
        return out

    if op == "weight":
        e4, a4 = packed4(s["e"], M, B, "identity", 1), packed4(s["x"], K, B, act, 1)
        mx.build_mx_weight_update(M, K, B, dt, ALPHA)(s["w"], e4, a4)
        return s["w"]
    w4 = mx.MXMatrix(*s["w4"])
    if op == "infer":
        e4 = packed4(s["e_lower"], K, B, "identity", 0)
        mx.build_mx_inference_update(M, K, B, act, dt, GAMMA)(s["x"], s["e"], w4, e4)
        return s["x"]
    x4 = packed4(s["x"], K, B, act, 0)
    if op == "pred":
        mx.build_mx_prediction_error(M, K, B, dt)(x4, w4, s["x_lower"], s["out"])
    else:
        mx.build_mx_forward(M, K, B, dt)(x4, w4, s["out"])
    return s["out"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ what they cost
def work(case):
    size = 4 if case["storage"] == "fp32" else 2
    if case["kind"] == "pack":
        n = case["rows"] * case["cols"]
        kept = n * (0.5 if case["format"] == "fp4" else 1) + n / BLOCK
        return {"bytes": 2 * size * n + 2 * kept, "flops": 0}
    M, K, B, op = case["M"], case["K"], case["batch"], case["op"]
    w4 = M * K * (0.5 + 1 / BLOCK)
    flops = 2.0 * M * K * B
    if case["kind"] == "backward":  # X, E and W in, W and the gradient out
        return {"bytes": size * (2 * K * B + M * B + 2 * M * K), "flops": 2 * flops}
    if op == "weight":
        return {"bytes": size * (M * B + K * B + 2 * M * K), "flops": flops}
    states = {"pred": K * B + 2 * M * B, "infer": K * B + 3 * M * B}.get(op, K * B + M * B)
    return {"bytes": w4 + size * states, "flops": flops}


# ------------------------------------------------------------------ the same in 64 bits
def _nearest(x, fmt, dim):
    """x rounded to its microscaled values, blocks of 32 along `dim`, by comparing
    magnitudes with the midpoints between neighbouring elements (a midpoint itself
    goes to the neighbour with the even code)."""
    if dim == 0:
        return _nearest(x.T, fmt, 1).T
    rows, n = x.shape
    b = torch.zeros((rows, -(-n // BLOCK) * BLOCK), dtype=torch.float64, device=x.device)
    b[:, :n] = x
    b = b.view(rows, -1, BLOCK)
    top = b.abs().max(-1, keepdim=True).values
    whole = torch.floor(torch.log2(top.clamp(min=2.0 ** -140)))  # log2 may be a unit off next to a power of two
    whole = whole + (top >= 2.0 ** (whole + 1)) - (top < 2.0 ** whole).double()
    limit = 7.0 / 4 if fmt == "fp4" else 255.0 / 128  # from here on the largest magnitude rounds to the next power
    scale = 2.0 ** ((whole + (top >= limit * 2.0 ** whole).double()) - (2 if fmt == "fp4" else 0)).clamp(-126, 127)
    a = b.abs() / scale
    if fmt == "fp4":
        q = torch.zeros_like(a)
        for middle, step, up in ((0.25, 0.5, 0), (0.75, 0.5, 1), (1.25, 0.5, 0), (1.75, 0.5, 1), (2.5, 1, 0),
                                 (3.5, 1, 1), (5, 2, 0)):
            q += step * ((a > middle) | (bool(up) & (a == middle)))
    else:
        low = torch.floor(a * 64)
        rest = a * 64 - low
        q = (low + ((rest > 0.5) | ((rest == 0.5) & (low % 2 == 1))).double()).clamp(max=127) / 64
    return (torch.sign(b) * q * scale).view(rows, -1)[:, :n]


def exact(case, seed):
    v, act = {k: t.double() for k, t in _inputs(case, seed).items()}, case["activation"]
    if case["kind"] == "pack":
        got = _nearest(_f(act, v["x"]), case["format"], case["axis"])
        return got.T.contiguous() if case["axis"] == 0 else got
    if case["kind"] == "backward":
        x8 = _nearest(v["x"], "int8", 1)
        return {"w": v["w"] + ALPHA * torch.mm(v["e"], _f(act, x8).T.contiguous()),
                "grad": _df(act, x8) * torch.mm(v["w"].T.contiguous(), v["e"])}
    if case["op"] == "weight":
        a4 = _nearest(_f(act, v["x"]), "fp4", 1)
        return v["w"] + ALPHA * torch.mm(_nearest(v["e"], "fp4", 1), a4.T.contiguous())
    if case["op"] == "infer":
        up = torch.mm(_nearest(v["w"], "fp4", 0).T.contiguous(), _nearest(v["e_lower"], "fp4", 0))
        return v["x"] + GAMMA * (-v["e"] + _df(act, v["x"]) * up)
    f = _f(act, v["x"])
    y = torch.mm(_nearest(v["w"], "fp4", 1), f if case["kind"] == "serve" else _nearest(f, "fp4", 0))
    return v["x_lower"] - y if case["op"] == "pred" else y
