"""The operators of a pre-norm training step and of serving it, beside the per-tensor scaled linears: the linear whose operands
are e4m3 with a power-of-two scale for each block of 128 (``blockwise_linear``; ``quantize_to_float8`` with
``ActivationCasting.BLOCKWISE``), layer norm (``layer_norm``), and the global norm of the gradients with their clipping
(``clip_grad_norm_``, ``clip_grads``).

A block is 128 neighbouring values of one row along the contraction (activations, gradients of outputs) or 128 x 128 values (weights); the
last of a row or column may be shorter.  Its scale 2^S has the smallest S >= -126 with max|block| <= 448 * 2^S; its values are
kept as e4m3 of value / 2^S, rounded to nearest even.  A product multiplies what is kept and adds in 32 bits or more:
  y = q(x) q(w)^T + bias,  dx = q(dy) q(w),  dw = q'(dy)^T q'(x),  dbias = columns of dy summed
where q' has its blocks along the tokens.  Layer norm: y = (x - mean) / sqrt(var + eps) * weight + bias over the last dimension, var without
Bessel's correction.  Clipping: every gradient times min(1, max_norm / (norm + 1e-6)), norm over all values of all of them.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _linear(name, what, m, k, n, dtype="bf16", bias=False):
    return {"name": name, "what": what, "m": m, "k": k, "n": n, "dtype": dtype, "bias": bias}


def _norm(name, rows, cols, dtype="bf16", train=True, params="same"):
    return {"name": name, "what": "norm", "rows": rows, "cols": cols, "dtype": dtype, "train": train, "params": params}


def _clip(name, shapes, layers, dtype="bf16", to="", seldom=False):
    return {"name": name, "what": "clip", "shapes": shapes, "layers": layers, "dtype": dtype, "to": to, "seldom": seldom}


# gradients of one decoder block (4096 wide, 1024 of keys and values, 14336 in its feed-forward part), its two norms in fp32
_DECODER = "4096x4096 1024x4096 1024x4096 4096x4096 14336x4096 14336x4096 4096x14336 4096f 4096f"


def listed():
    return [
        # a small layer, the size of the unit tests and of a first experiment: launches and host time are all there is
        _linear("linear_small", "train", 512, 1024, 1024),
        # one projection of a 4096-wide model at 2048 tokens: the first benchmark configuration
        _linear("linear_4096", "train", 2048, 4096, 4096),
        # sizes that are multiples of nothing (the padding configuration), with a bias: a last block of 1, of 3 and of 127
        _linear("linear_ragged", "train", 4099, 4097, 11007, bias=True),
        # the feed-forward projection of the 70B shapes at half of its tokens: where such a model spends its step
        _linear("linear_70b_w13", "train", 8192, 8192, 28672),
        # one token through one linear of a large model: the weight is read once, everything else is latency
        _linear("decode", "infer", 1, 8192, 8192),
        # a prompt through the up projection of the inference tests (d = 4096, ffn = 14336)
        _linear("prefill", "infer", 2048, 4096, 14336, dtype="fp16", bias=True),
        # the norm of one decoded token
        _norm("norm_token", 1, 4096, train=False),
        # the norm in front of a block of the 4096-wide model at 8192 tokens, weights kept in fp32
        _norm("norm_train", 8192, 4096, params="fp32"),
        # multiples of nothing, in fp32
        _norm("norm_ragged", 4099, 4097, dtype="fp32"),
        # a model of a first experiment: many small gradients (weights and biases), a step whose norm is below the limit, as most are
        _clip("clip_small", "1024x1024 1024 1000x1024 1000 77x33 1", 8, seldom=True),
        # two decoder blocks whose optimizer takes fp32 gradients: norm, then the clipped copies
        _clip("clip_to_fp32", _DECODER, 2, to="fp32"),
        # six of them in place, a step that is not clipped
        _clip("clip_in_place", _DECODER, 6, seldom=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size between lo and hi, spread over the logarithm; half of them are multiples of 128, as in most models."""
    v = _log_int(rng, lo, hi)
    return max(lo, v // 128 * 128) if rng.random() < 0.5 else v


def draw(rng):
    most = work(_linear("", "train", 8192, 8192, 28672))["flops"]
    while True:
        kind = rng.random()
        if kind < 0.35:
            case = _linear("", "train", _size(rng, 128, 16384), _size(rng, 256, 16384), _size(rng, 256, 28672),
                           dtype=rng.choice(["bf16", "bf16", "fp16"]), bias=rng.random() < 0.3)
        elif kind < 0.55:
            m = _log_int(rng, 1, 64) if rng.random() < 0.6 else _size(rng, 65, 8192)
            case = _linear("", "infer", m, _size(rng, 512, 16384), _size(rng, 512, 28672),
                           dtype=rng.choice(["bf16", "bf16", "fp16"]), bias=rng.random() < 0.3)
        elif kind < 0.8:
            train = rng.random() < 0.6
            case = _norm("", _log_int(rng, 16, 32768) if train else _log_int(rng, 1, 32768), _size(rng, 64, 20000),
                         dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), train=train, params=rng.choice(["same", "fp32"]))
            if case["rows"] * case["cols"] > 3e8:
                continue
        else:
            shapes = ["%dx%d" % (_log_int(rng, 1, 16384), _log_int(rng, 1, 16384)) if rng.random() < 0.6 else
                      "%d%s" % (_log_int(rng, 1, 20000), rng.choice(["", "f"])) for _ in range(rng.randint(1, 10))]
            case = _clip("", " ".join(shapes), rng.randint(1, 6), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                         to=rng.choice(["", "fp32", "same"]))
            case["seldom"] = not case["to"]  # in place, a second pass over clipped gradients would clip nothing
            if case["layers"] * sum(math.prod(s) for s, _ in _shapes(case)) > 1.2e9:
                continue
        if work(case)["flops"] <= most:
            del case["name"]
            return case


def _shapes(case):
    """[(shape, its dtype)] of one layer's gradients: "4096x1024" in the case's type, "4096f" in fp32."""
    return [(tuple(int(v) for v in s.rstrip("f").split("x")), "fp32" if s.endswith("f") else case["dtype"]) for s in case["shapes"].split()]


def _made(case, seed):
    """The tensors of a case, from its seed."""
    torch.manual_seed(seed)
    normal = lambda *shape, dtype=torch.float32, std=1.0: torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, std)
    dtype = _DTYPES[case["dtype"]]
    if case["what"] == "clip":
        std = 1e-4 if case["seldom"] else 3e-2
        return {"grads": [normal(*shape, dtype=_DTYPES[kind], std=std) for _ in range(case["layers"]) for shape, kind in _shapes(case)]}
    if case["what"] == "norm":
        d, params = case["cols"], dtype if case["params"] == "same" else torch.float32
        # a residual stream: a few channels are larger than the rest, rows have a mean
        x = normal(case["rows"], d, dtype=dtype).mul_(normal(d).exp_().to(dtype)).add_(0.5)
        made = {"x": x, "weight": normal(d, dtype=params, std=0.1).add_(1.0), "bias": normal(d, dtype=params, std=0.1)}
        if case["train"]:
            made["dy"] = normal(case["rows"], d, dtype=dtype, std=1e-2)
        return made
    m, k, n = case["m"], case["k"], case["n"]
    # activations whose channels differ in size, weights as they are initialised
    made = {"x": normal(m, k, dtype=dtype).mul_(normal(k).exp_().to(dtype)), "weight": normal(n, k, dtype=dtype, std=k ** -0.5),
            "bias": normal(n, dtype=dtype, std=0.1) if case["bias"] else None}
    if case["what"] == "train":
        made["dy"] = normal(m, n, dtype=dtype, std=1e-2).mul_(normal(m, 1).exp_().to(dtype))
    return made


def prepare(case, seed):
    state = _made(case, seed)
    if case["what"] == "train" or case.get("train"):
        for name in ("x", "weight", "bias"):
            if state[name] is not None:
                state[name].requires_grad_()
    elif case["what"] == "infer":
        # a program that serves a model quantises its weights once
        if own:
            from float8_experimental_amd.inference import ActivationCasting, QuantConfig, quantize_to_float8

            layer = torch.nn.Linear(case["k"], case["n"], bias=case["bias"], device="meta")
            layer.weight = torch.nn.Parameter(state["weight"])
            if case["bias"]:
                layer.bias = torch.nn.Parameter(state["bias"])
            state["layer"] = quantize_to_float8(layer, QuantConfig(ActivationCasting.BLOCKWISE))
        else:
            state["kept"] = _kept(state["weight"].float(), 128, 128)
        del state["weight"]
    elif case["what"] == "clip":
        state["params"] = [torch.nn.Parameter(torch.empty_like(g)) for g in state["grads"]]
        for p, g in zip(state["params"], state["grads"]):
            p.grad = g
    state["case"] = case
    return state


# ---- plain forms


def _kept(t, rows, cols):
    """What is kept of t [m, k] in blocks of rows x cols: e4m3 values and the power-of-two scales, each in its block's shape."""
    m, k = t.shape
    t = torch.nn.functional.pad(t, (0, -k % cols, 0, -m % rows)).view(-(-m // rows), rows, -(-k // cols), cols)
    bits = t.abs().amax((1, 3), keepdim=True).view(torch.int32)
    power = ((bits >> 23) - 135 + ((bits & 0x7FFFFF) > 0x600000)).clamp(min=-126)  # 448 is 1.75 * 2^8
    return (t * ((127 - power) << 23).view(torch.float32)).to(torch.float8_e4m3fn), ((127 + power) << 23).view(torch.float32), (m, k)


def _stands_for(kept):
    """The values that are kept, in 32 bits."""
    values, scales, (m, k) = kept
    t = values.float() * scales
    return t.view(t.shape[0] * t.shape[1], -1)[:m, :k]


def _plain_train(x, weight, bias, dy):
    dtype = x.dtype
    x, w, g = x.float(), _stands_for(_kept(weight.float(), 128, 128)), dy.float()
    y = _stands_for(_kept(x, 1, 128)) @ w.t()
    if bias is not None:
        y += bias.float()
    dx = _stands_for(_kept(g, 1, 128)) @ w
    dw = _stands_for(_kept(g, 128, 1)).t() @ _stands_for(_kept(x, 128, 1))
    out = {"y": y.to(dtype), "dx": dx.to(dtype), "dw": dw.to(dtype)}
    return out if bias is None else {**out, "db": g.sum(0).to(dtype)}


def _plain_infer(x, kept, bias):
    y = _stands_for(_kept(x.float(), 1, 128)) @ _stands_for(kept).t()
    return (y if bias is None else y + bias.float()).to(x.dtype)


def _plain_norm(x, weight, bias, dy=None):
    v, w = x.float(), weight.float()
    centred = v - v.mean(1, keepdim=True)
    rstd = (centred.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    normed = centred * rstd
    y = (normed * w + bias.float()).to(x.dtype)
    if dy is None:
        return y
    g = dy.float()
    gw = g * w
    dx = (gw - gw.mean(1, keepdim=True) - normed * (gw * normed).mean(1, keepdim=True)) * rstd
    return {"y": y, "dx": dx.to(x.dtype), "dw": (g * normed).sum(0).to(weight.dtype), "db": g.sum(0).to(bias.dtype)}


def _plain_clip(grads, max_norm, to):
    norm = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()
    factor = (max_norm / (norm + 1e-6)).clamp(max=1.0)
    if not to:
        return {"norm": norm, "grads": [g.copy_(g.float() * factor) for g in grads]}
    return {"norm": norm, "grads": [(g.float() * factor).to(g.dtype if to == "same" else torch.float32) for g in grads]}


# ---- one pass


def run(state):
    case = state["case"]
    if case["what"] == "clip":
        return _run_clip(state, case["to"])
    if case["what"] == "norm":
        return _run_norm(state, case["train"])
    if case["what"] == "infer":
        if not own:
            return _plain_infer(state["x"], state["kept"], state["bias"])
        with torch.no_grad():
            return state["layer"](state["x"])
    x, weight, bias, dy = (state[name] for name in ("x", "weight", "bias", "dy"))
    if not own:
        with torch.no_grad():
            return _plain_train(x, weight, bias, dy)
    import float8_experimental_amd as f8

    x.grad = weight.grad = None
    if bias is not None:
        bias.grad = None
    y = f8.blockwise_linear(x, weight, bias)
    y.backward(dy)
    out = {"y": y, "dx": x.grad, "dw": weight.grad}
    return out if bias is None else {**out, "db": bias.grad}


def _run_norm(state, train):
    x, weight, bias = state["x"], state["weight"], state["bias"]
    if not own:
        with torch.no_grad():
            return _plain_norm(x, weight, bias, state.get("dy"))
    import float8_experimental_amd as f8

    if not train:
        with torch.no_grad():
            return f8.layer_norm(x, (x.shape[1],), weight, bias)
    x.grad = weight.grad = bias.grad = None
    y = f8.layer_norm(x, (x.shape[1],), weight, bias)
    y.backward(state["dy"])
    return {"y": y, "dx": x.grad, "dw": weight.grad, "db": bias.grad}


def _run_clip(state, to):
    if not own:
        return _plain_clip(state["grads"], _MAX_NORM, to)
    import float8_experimental_amd as f8

    if to:
        norm, grads = f8.clip_grads(state["grads"], _MAX_NORM, out_dtype=None if to == "same" else torch.float32)
        return {"norm": norm, "grads": grads}
    norm = f8.clip_grad_norm_(state["params"], _MAX_NORM)
    return {"norm": norm, "grads": [p.grad for p in state["params"]]}


_MAX_NORM = 8.0


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["what"] == "clip":
        sizes = [(math.prod(s), 4 if kind == "fp32" else 2) for s, kind in _shapes(case)]
        n = case["layers"] * sum(v for v, _ in sizes)
        read = case["layers"] * sum(v * b for v, b in sizes)
        # below the limit gradients that are clipped in place are left as they are
        written = 0 if not case["to"] else 4 * n if case["to"] == "fp32" else read
        return {"bytes": float(read + written + 4), "flops": (3.0 if case["to"] else 2.0) * n}
    if case["what"] == "norm":
        n, d, p = case["rows"] * case["cols"], case["cols"], size if case["params"] == "same" else 4
        # forward: x, weight and bias read, y written; backward: dy read, dx and the gradients of weight and bias written.  About 8
        # operations a value forward, 12 backward
        return {"bytes": float(size * n * (4 if case["train"] else 2) + p * d * (4 if case["train"] else 2)), "flops": (20.0 if case["train"] else 8.0) * n}
    m, k, n = case["m"], case["k"], case["n"]
    bias = size * n if case["bias"] else 0
    if case["what"] == "infer":  # a byte for each weight, a scale of one byte for each 128 x 128 of them
        return {"bytes": float(n * k + -(-n // 128) * -(-k // 128) + size * (m * k + m * n) + bias), "flops": 2.0 * m * k * n}
    # x, weight and dy read, y and the three gradients written
    return {"bytes": float(size * (2 * m * k + 2 * n * k + 2 * m * n) + 2 * bias), "flops": 6.0 * m * k * n}


# ---- the definition in 64 bits


def _power64(exponent):
    """2^exponent in 64 bits, from its bits (torch.ldexp takes a power that may be off in the last place: every sixteenth value is a tie)."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _e4m3(v):
    """v rounded to nearest even among the e4m3 values (at most 448 in size, a step of 2^-9 near zero), in 64 bits."""
    exponent = torch.frexp(v)[1].clamp(min=-5) - 4  # of the last of the four significant bits
    return torch.round(v * _power64(-exponent)) * _power64(exponent)


def _quantised64(t, along, both=False):
    """t in 64 bits as blocks of 128 along a dimension (or both) stand for it."""
    t = t.double()
    most = t.abs()
    for dim in (0, 1) if both else (along,):
        parts = [p.amax(dim, keepdim=True).expand_as(p) for p in most.split(128, dim)]
        most = torch.cat(parts, dim)
    fraction, exponent = torch.frexp(most)  # most = fraction * 2^exponent, fraction in [0.5, 1)
    power = (exponent - 9 + (fraction > 0.875)).clamp(min=-126)
    return _e4m3(t * _power64(-power)) * _power64(power)


def exact(case, seed):
    made = _made(case, seed)
    if case["what"] == "clip":
        norm = sum(g.double().square().sum() for g in made["grads"]).sqrt()
        factor = min(1.0, _MAX_NORM / (float(norm) + 1e-6))
        return {"norm": norm, "grads": [g.double() * factor for g in made["grads"]]}
    if case["what"] == "norm":
        v, w = made["x"].double(), made["weight"].double()
        var, mean = torch.var_mean(v, 1, correction=0, keepdim=True)
        normed = (v - mean) / (var + 1e-5).sqrt()
        y = normed * w + made["bias"].double()
        if not case["train"]:
            return y
        g = made["dy"].double()
        gw = g * w
        dx = (gw - gw.mean(1, keepdim=True) - normed * (gw * normed).mean(1, keepdim=True)) / (var + 1e-5).sqrt()
        return {"y": y, "dx": dx, "dw": (g * normed).sum(0), "db": g.sum(0)}
    x, w, bias = made["x"], _quantised64(made["weight"], 1, both=True), made["bias"]
    y = _quantised64(x, 1) @ w.t()
    if bias is not None:
        y += bias.double()
    if case["what"] == "infer":
        return y
    out = {"y": y, "dx": _quantised64(made["dy"], 1) @ w}
    del w
    out["dw"] = _quantised64(made["dy"], 0).t() @ _quantised64(x, 0)
    return out if bias is None else {**out, "db": made["dy"].double().sum(0)}
