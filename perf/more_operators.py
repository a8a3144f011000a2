"""The operators of fine-tuning a pre-norm model with low-rank adapters and of serving it: RMS norm with the residual's addition
(``rms_norm``; ``rms_norm_blockwise`` in front of ``Float8BlockwiseInferenceLinear``), low-rank adapters of many requests beside a shared
projection (``low_rank_adapters``), and dropout whose mask is not stored (``dropout``).

RMS norm: s = x + residual, rounded to their type; y = s / sqrt(mean(s^2) + eps) * weight over the last dimension.  With block scales y is not
rounded to 16 bits but kept as e4m3 with a power-of-two scale 2^S for each 128 neighbouring values of a row, S >= -126 the smallest with max|block| <= 448 *
2^S; the projections behind it multiply what is kept by weights that are kept the same way in blocks of 128 x 128.
Adapters: out_i = y_i + scale_e * B_e (A_e x_i) with the adapter e of row i; a row without one keeps y_i.
Dropout: out = residual + (x / (1 - p) where kept, else 0).  Element i is kept if word i % 4 of the Philox block 4x32 of 7 rounds, with
the counter i / 4 and the 64-bit seed as its key, is at least p * 2^32.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-6


def _rms(name, rows, cols, dtype="bf16", residual=True, train=True, params="same"):
    return {"name": name, "what": "rms", "rows": rows, "cols": cols, "dtype": dtype, "residual": residual, "train": train, "params": params}


def _cast(name, rows, cols, outs, dtype="bf16", residual=True):
    return {"name": name, "what": "cast", "rows": rows, "cols": cols, "outs": outs, "dtype": dtype, "residual": residual, "params": "same"}


def _adapters(name, rows, k, n, rank, count, requests=0, without=False, train=False, dtype="bf16"):
    """``requests``: the rows are that many runs of one request each (0: every row is one of its own, in any order); ``without``: some have no adapter."""
    return {"name": name, "what": "adapters", "rows": rows, "k": k, "n": n, "rank": rank, "count": count, "requests": requests, "without": without, "train": train,
            "dtype": dtype}


def _dropout(name, rows, cols, p, dtype="bf16", residual=True):
    return {"name": name, "what": "dropout", "rows": rows, "cols": cols, "p": p, "dtype": dtype, "residual": residual}


def listed():
    return [
        # the norm of one decoded token: launches and host time are all there is
        _rms("norm_token", 1, 4096, train=False),
        # the norm in front of a block of the 4096-wide model at 8192 tokens, both passes, weights kept in fp32
        _rms("norm_train", 8192, 4096, params="fp32"),
        # multiples of nothing, in fp32, without a residual
        _rms("norm_ragged", 4099, 4097, dtype="fp32", residual=False),
        # one decoding step of 16 requests: the norm and the query, key and value projections of an 8192-wide model behind it
        _cast("norm_decode", 16, 8192, "8192 1024 1024"),
        # a prompt through the norm and the output projection's width of the same model: as many values to norm as to multiply with
        _cast("norm_prefill", 8192, 8192, "1024"),
        # one token with one adapter among eight beside a 4096-wide projection
        _adapters("adapters_token", 1, 4096, 4096, 8, 8),
        # a decoding step of 64 requests that each have an adapter of their own
        _adapters("adapters_decode", 64, 8192, 8192, 16, 64),
        # prompts of 24 requests, a few without an adapter, beside the up projection of the inference tests
        _adapters("adapters_prefill", 8192, 4096, 14336, 64, 8, requests=24, without=True),
        # fine-tuning four adapters at once on 8192 tokens, both passes
        _adapters("adapters_train", 8192, 4096, 4096, 16, 4, requests=16, train=True),
        # sizes that are multiples of nothing, both passes
        _adapters("adapters_ragged", 4099, 1000, 4097, 12, 3, requests=7, without=True, train=True, dtype="fp16"),
        # dropout on the branch of a small layer, both passes
        _dropout("dropout_small", 512, 1024, 0.1),
        # dropout on the residual branch of the 8192-wide model at 8192 tokens, both passes
        _dropout("dropout_train", 8192, 8192, 0.1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size between lo and hi, spread over the logarithm; half of them are multiples of 128, as in most models."""
    v = _log_int(rng, lo, hi)
    return max(lo, v // 128 * 128) if rng.random() < 0.5 else v


def draw(rng):
    most = {kind: max(work(c)["bytes"] for c in listed() if c["what"] == kind) for kind in ("rms", "cast", "adapters", "dropout")}
    while True:
        kind = rng.random()
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if kind < 0.25:
            train = rng.random() < 0.6
            case = _rms("", _log_int(rng, 16, 32768) if train else _log_int(rng, 1, 32768), _size(rng, 64, 20000), dtype=dtype, residual=rng.random() < 0.7, train=train,
                        params=rng.choice(["same", "fp32"]))
        elif kind < 0.45:
            outs = " ".join(str(_size(rng, 512, 16384)) for _ in range(rng.randint(1, 3)))
            rows = _log_int(rng, 1, 64) if rng.random() < 0.5 else _size(rng, 65, 8192)
            case = _cast("", rows, _size(rng, 512, 16384), outs, dtype=rng.choice(["bf16", "bf16", "fp16"]), residual=rng.random() < 0.7)
        elif kind < 0.8:
            train = rng.random() < 0.5
            rows = _log_int(rng, 16, 16384) if train else _log_int(rng, 1, 16384)
            requests = 0 if rows <= 256 and rng.random() < 0.7 else _log_int(rng, 1, min(rows, 64))
            count = _log_int(rng, 1, 64) if not train else _log_int(rng, 1, 16)
            case = _adapters("", rows, _size(rng, 64, 16384), _size(rng, 64, 16384), rng.choice([4, 8, 16, 16, 32, 64, 128, rng.randint(1, 128)]), count,
                             requests=requests, without=rng.random() < 0.4, train=train, dtype=dtype)
        else:
            case = _dropout("", _log_int(rng, 1, 16384), _log_int(rng, 1, 16384), round(rng.uniform(0.02, 0.6), 3), dtype=dtype, residual=rng.random() < 0.7)
        if work(case)["bytes"] <= most[case["what"]] and work(case)["flops"] <= 4e11:
            del case["name"]
            return case


def _outs(case):
    return [int(n) for n in case["outs"].split()]


def _of_requests(case):
    """The adapter of each of the case's requests, -1 for those without: every adapter has one while there are enough."""
    requests = case["requests"] or case["rows"]
    return [-1 if case["without"] and i % 8 == 5 else (i - (i + 2) // 8 * case["without"]) % case["count"] for i in range(requests)]


def _made(case, seed):
    """The tensors of a case, from its seed."""
    torch.manual_seed(seed)
    normal = lambda *shape, dtype=torch.float32, std=1.0: torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, std)
    dtype = _DTYPES[case["dtype"]]
    if case["what"] in ("rms", "cast"):
        rows, d, params = case["rows"], case["cols"], dtype if case["params"] == "same" else torch.float32
        made = {"x": normal(rows, d, dtype=dtype), "weight": normal(d, dtype=params, std=0.1).add_(1.0)}
        # a residual stream: a few channels are larger than the rest
        stream = made["x"] if not case["residual"] else made.setdefault("residual", normal(rows, d, dtype=dtype))
        stream.mul_(normal(d).exp_().to(dtype))
        if case["what"] == "cast":
            made["linears"] = [normal(n, d, dtype=dtype, std=d ** -0.5) for n in _outs(case)]
        elif case["train"]:
            made["dy"] = normal(rows, d, dtype=dtype, std=1e-2)
            if case["residual"]:
                made["ds"] = normal(rows, d, dtype=dtype, std=1e-2)
        return made
    if case["what"] == "dropout":
        shape = (case["rows"], case["cols"])
        made = {"x": normal(*shape, dtype=dtype), "seed": torch.randint(-2 ** 62, 2 ** 62, (1,), device="cuda"), "dout": normal(*shape, dtype=dtype, std=1e-2)}
        if case["residual"]:
            made["residual"] = normal(*shape, dtype=dtype, std=2.0)
        return made
    m, k, n, r, count = (case[name] for name in ("rows", "k", "n", "rank", "count"))
    ids = _of_requests(case)
    if case["requests"]:  # runs of uneven length
        cuts = sorted(torch.randperm(m - 1)[:len(ids) - 1].add(1).tolist())
        ids = [e for e, first, end in zip(ids, [0] + cuts, cuts + [m]) for _ in range(end - first)]
    else:
        ids = [ids[i] for i in torch.randperm(m).tolist()]
    # activations whose channels differ in size; adapters as they are after some training; what the projection gave
    made = {"x": normal(m, k, dtype=dtype).mul_(normal(k).exp_().to(dtype)), "a": normal(count, r, k, dtype=dtype, std=k ** -0.5),
            "b": normal(count, n, r, dtype=dtype, std=0.5 * r ** -0.5), "y": normal(m, n, dtype=dtype), "scale": normal(count, std=0.1).add_(1.0),
            "ids": torch.tensor(ids, device="cuda")}
    if case["train"]:
        made["dout"] = normal(m, n, dtype=dtype, std=1e-2)
    return made


def prepare(case, seed):
    state = _made(case, seed)
    if case["what"] == "cast":
        # a program that serves a model quantises its weights once
        if own:
            from float8_experimental_amd.inference import ActivationCasting, QuantConfig, quantize_to_float8

            layers = []
            for w in state["linears"]:
                layer = torch.nn.Linear(w.shape[1], w.shape[0], bias=False, device="meta")
                layer.weight = torch.nn.Parameter(w)
                layers.append(quantize_to_float8(layer, QuantConfig(ActivationCasting.BLOCKWISE)))
            state["linears"] = layers
        else:
            state["linears"] = [_kept(w.float(), 128, 128) for w in state["linears"]]
    elif case["what"] == "adapters":
        # which rows an adapter has is the same for every layer of a model, and known to the program that put the batch together
        ids = state.pop("ids")
        if own:
            import float8_experimental_amd as f8

            state["rows"] = f8.AdapterRows(ids, case["count"])
        elif case["rows"] <= 256 and not case["train"]:
            state["ids"] = ids
        else:
            state["rows"] = [(e, (ids == e).nonzero().flatten()) for e in sorted(set(ids.tolist())) if e >= 0]
    if case.get("train") or case["what"] == "dropout":
        for name in ("x", "weight", "a", "b"):
            if name in state:
                state[name].requires_grad_()
    state["case"] = case
    return state


# ---- plain forms


def _kept(t, rows, cols):
    """What is kept of t [m, k] in blocks of rows x cols, as the values that it stands for."""
    m, k = t.shape
    t = torch.nn.functional.pad(t, (0, -k % cols, 0, -m % rows)).view(-(-m // rows), rows, -(-k // cols), cols)
    bits = t.abs().amax((1, 3), keepdim=True).view(torch.int32)
    power = ((bits >> 23) - 135 + ((bits & 0x7FFFFF) > 0x600000)).clamp(min=-126)  # 448 is 1.75 * 2^8
    scaled = (t * ((127 - power) << 23).view(torch.float32)).to(torch.float8_e4m3fn).float()
    t = scaled * ((127 + power) << 23).view(torch.float32)
    return t.view(t.shape[0] * t.shape[1], -1)[:m, :k]


def _plain_rms(x, weight, residual=None, dy=None, ds=None):
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    v = s.float()
    rstd = (v.square().mean(1, keepdim=True) + _EPS).rsqrt()
    normed = v * rstd
    out = {"y": (normed * weight.float()).to(x.dtype)}
    if residual is not None:
        out["s"] = s
    if dy is None:
        return out
    g = dy.float()
    gw = g * weight.float()
    dx = rstd * (gw - normed * (gw * normed).mean(1, keepdim=True))
    if ds is not None:
        dx = dx + ds.float()
    return {**out, "dx": dx.to(x.dtype), "dw": (g * normed).sum(0).to(weight.dtype)}


def _plain_cast(x, weight, linears, residual=None):
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    v = s.float()
    kept = _kept(v * (v.square().mean(1, keepdim=True) + _EPS).rsqrt() * weight.float(), 1, 128)
    return {"y%d" % i: (kept @ w.t()).to(x.dtype) for i, w in enumerate(linears)} | ({} if residual is None else {"s": s})


def _plain_adapters(x, a, b, y, scale, ids=None, rows=None, dout=None):
    if ids is not None:  # few rows: each with its adapter's matrices
        at, factor = ids.clamp(min=0), torch.where(ids >= 0, scale[ids.clamp(min=0)], 0.0)
        h = (a[at].float() * x.float()[:, None, :]).sum(2)
        return {"out": (y.float() + factor[:, None] * (b[at].float() * h[:, None, :]).sum(2)).to(y.dtype)}
    out = y.float()
    grads = {} if dout is None else {"dx": torch.zeros_like(x, dtype=torch.float32), "da": torch.zeros_like(a), "db": torch.zeros_like(b)}
    for e, at in rows:
        xe, ae, be, f = x[at].float(), a[e].float(), b[e].float(), scale[e]
        h = xe @ ae.t()
        out.index_add_(0, at, (h @ be.t()).mul_(f))
        if dout is not None:
            ge = dout[at].float() * f
            dh = ge @ be
            grads["dx"][at] = dh @ ae
            grads["da"][e] = (dh.t() @ xe).to(a.dtype)
            grads["db"][e] = (ge.t() @ h).to(b.dtype)
    if grads:
        grads["dx"] = grads["dx"].to(x.dtype)
    return {"out": out.to(y.dtype), **grads}


_MULTIPLIERS, _WEYL = (0xD2511F53, 0xCD9E8D57), (0x9E3779B9, 0xBB67AE85)


def _plain_words(seed, count):
    """The first ``count`` random words of a seed (a tensor), as whole numbers in 64 bits."""
    low = 0xFFFFFFFF
    i = torch.arange(-(-count // 4), device=seed.device)
    c = [i & low, i >> 32, torch.zeros_like(i), torch.zeros_like(i)]
    key = [seed & low, seed >> 32 & low]
    for _ in range(7):
        p, q = c[0] * _MULTIPLIERS[0], c[2] * _MULTIPLIERS[1]  # (the sign goes with the shift's mask)
        c = [(q >> 32 & low) ^ c[1] ^ key[0], q & low, (p >> 32 & low) ^ c[3] ^ key[1], p & low]
        key = [key[0] + _WEYL[0] & low, key[1] + _WEYL[1] & low]
    return torch.stack(c, 1).view(-1)[:count]


def _plain_dropout(x, seed, p, dout, residual=None):
    keep = (_plain_words(seed, x.numel()) >= round(p * 2 ** 32)).view(x.shape)
    out, factor = torch.where(keep, x.float() * (1 / (1 - p)), 0.0), 1 / (1 - p)
    if residual is not None:
        out = out + residual.float()
    return {"out": out.to(x.dtype), "dx": torch.where(keep, dout.float() * factor, 0.0).to(x.dtype)}


# ---- one pass


def run(state):
    case = state["case"]
    of = lambda *names: {name: state[name] for name in names if name in state}
    if not own:
        with torch.no_grad():
            if case["what"] == "rms":
                return _plain_rms(**of("x", "weight", "residual", "dy", "ds"))
            if case["what"] == "cast":
                return _plain_cast(**of("x", "weight", "linears", "residual"))
            if case["what"] == "adapters":
                return _plain_adapters(**of("x", "a", "b", "y", "scale", "ids", "rows", "dout"))
            return _plain_dropout(**of("x", "seed", "dout", "residual"), p=case["p"])
    import float8_experimental_amd as f8

    x, residual = state["x"], state.get("residual")
    if case["what"] == "cast":
        with torch.no_grad():
            kept = f8.rms_norm_blockwise(x, (x.shape[1],), state["weight"], _EPS, residual=residual)
            kept, *s = kept if residual is not None else (kept,)
            return {**{"y%d" % i: layer(kept) for i, layer in enumerate(state["linears"])}, **({"s": s[0]} if s else {})}
    if case["what"] == "dropout":
        x.grad = None
        out = f8.dropout(x, case["p"], seed=state["seed"], residual=residual)
        out.backward(state["dout"])
        return {"out": out, "dx": x.grad}
    if case["what"] == "rms":
        weight = state["weight"]
        if not case["train"]:
            with torch.no_grad():
                out = f8.rms_norm(x, (x.shape[1],), weight, _EPS, residual=residual)
            return {"y": out} if residual is None else {"y": out[0], "s": out[1]}
        x.grad = weight.grad = None
        if residual is None:
            y = f8.rms_norm(x, (x.shape[1],), weight, _EPS)
            y.backward(state["dy"])
            return {"y": y, "dx": x.grad, "dw": weight.grad}
        y, s = f8.rms_norm(x, (x.shape[1],), weight, _EPS, residual=residual)
        torch.autograd.backward([y, s], [state["dy"], state["ds"]])
        return {"y": y, "s": s, "dx": x.grad, "dw": weight.grad}
    a, b = state["a"], state["b"]
    if not case["train"]:
        with torch.no_grad():
            return {"out": f8.low_rank_adapters(x, a, b, state["rows"], state["y"], state["scale"])}
    x.grad = a.grad = b.grad = None
    out = f8.low_rank_adapters(x, a, b, state["rows"], state["y"], state["scale"])
    out.backward(state["dout"])
    return {"out": out, "dx": x.grad, "da": a.grad, "db": b.grad}


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["what"] == "rms":
        n, d, p = case["rows"] * case["cols"], case["cols"], size if case["params"] == "same" else 4
        # forward: x, the residual and the weight read, y and their sum written; backward: dy and the sum's gradient read, dx and the gradient of the
        # weight written.  About 6 operations a value forward, 10 backward
        tensors = (4 if case["residual"] else 2) + (0 if not case["train"] else 3 if case["residual"] else 2)
        return {"bytes": float(size * n * tensors + p * d * (2 if case["train"] else 1)), "flops": (16.0 if case["train"] else 6.0) * n}
    if case["what"] == "cast":
        m, k, outs = case["rows"], case["cols"], _outs(case)
        # x, the residual and the norm's weight read, their sum written; a byte for each weight of the linears and one for each 128 x 128 of them
        read = size * (m * k * (3 if case["residual"] else 1) + k) + sum(n * k + -(-n // 128) * -(-k // 128) for n in outs)
        return {"bytes": float(read + size * m * sum(outs)), "flops": 2.0 * m * k * sum(outs) + 6.0 * m * k}
    if case["what"] == "dropout":
        n = case["rows"] * case["cols"]
        # x and the residual read, out written; dout read, dx written.  A fourth of 7 rounds of 2 products and 4 other operations, both passes
        return {"bytes": float(size * n * (5 if case["residual"] else 4) + 8), "flops": 2 * (7 * 6 / 4 + 3.0) * n}
    m, k, n, r = (case[name] for name in ("rows", "k", "n", "rank"))
    ids = _of_requests(case)
    adapters = size * len(set(ids) - {-1}) * r * (k + n)
    with_one = m * sum(e >= 0 for e in ids) / len(ids)  # rows; about, where runs are uneven
    # x and y read, out written, the adapters that are in use read; backward dout read, dx and the adapters' gradients written
    if not case["train"]:
        return {"bytes": float(size * (with_one * k + 2 * m * n) + adapters), "flops": 2.0 * with_one * r * (k + n)}
    return {"bytes": float(size * (with_one * k + m * k + 3 * m * n) + adapters + size * case["count"] * r * (k + n)), "flops": 6.0 * with_one * r * (k + n)}


# ---- the definition in 64 bits


def _power64(exponent):
    """2^exponent in 64 bits, from its bits."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _e4m3(v):
    """v rounded to nearest even among the e4m3 values (at most 448 in size, a step of 2^-9 near zero), in 64 bits."""
    exponent = torch.frexp(v)[1].clamp(min=-5) - 4  # of the last of the four significant bits
    return torch.round(v * _power64(-exponent)) * _power64(exponent)


def _quantised64(t, both=False):
    """t in 64 bits as blocks of 128 of a row (or of 128 x 128) stand for it."""
    t = t.double()
    most = t.abs()
    for dim in (0, 1) if both else (1,):
        most = torch.cat([p.amax(dim, keepdim=True).expand_as(p) for p in most.split(128, dim)], dim)
    fraction, exponent = torch.frexp(most)  # most = fraction * 2^exponent, fraction in [0.5, 1)
    power = (exponent - 9 + (fraction > 0.875)).clamp(min=-126)
    return _e4m3(t * _power64(-power)) * _power64(power)


def _kept64(seed, p, count):
    """Which of ``count`` elements are kept: the same generator, its products in parts of 16 bits that no word of 64 bits loses."""
    key = int(seed) % 2 ** 64
    key = [key % 2 ** 32, key // 2 ** 32]
    n = torch.arange((count + 3) // 4, device="cuda")
    words = [n.remainder(2 ** 32), n.div(2 ** 32, rounding_mode="floor"), torch.zeros_like(n), torch.zeros_like(n)]

    def product(v, factor):  # (upper, lower) 32 bits
        low, high = v.remainder(65536) * factor, v.div(65536, rounding_mode="floor") * factor  # below 2^48 each
        total = low + high.remainder(65536) * 65536
        return high.div(65536, rounding_mode="floor") + total.div(2 ** 32, rounding_mode="floor"), total.remainder(2 ** 32)

    for turn in range(7):
        up0, low0 = product(words[0], 0xD2511F53)
        up2, low2 = product(words[2], 0xCD9E8D57)
        words = [up2.bitwise_xor(words[1]).bitwise_xor((key[0] + turn * 0x9E3779B9) % 2 ** 32), low2,
                 up0.bitwise_xor(words[3]).bitwise_xor((key[1] + turn * 0xBB67AE85) % 2 ** 32), low0]
    kept = torch.empty(4 * len(n), dtype=torch.bool, device="cuda")
    for i, w in enumerate(words):
        kept[i::4] = w >= round(p * 2 ** 32)
    return kept[:count]


def exact(case, seed):
    made = _made(case, seed)
    x = made["x"]
    if case["what"] == "dropout":
        keep = _kept64(made["seed"], case["p"], x.numel()).view(x.shape)
        out = x.double() / (1 - case["p"]) * keep
        if case["residual"]:
            out += made["residual"].double()
        return {"out": out, "dx": made["dout"].double() / (1 - case["p"]) * keep}
    if case["what"] in ("rms", "cast"):
        s = x.double()
        if case["residual"]:
            s = (s + made["residual"].double()).to(x.dtype).double()
        rms = ((s * s).sum(1, keepdim=True) / s.shape[1] + _EPS).sqrt()
        w = made["weight"].double()
        sums = {"s": s} if case["residual"] else {}
        if case["what"] == "cast":
            kept = _quantised64(s / rms * w)
            return {**{"y%d" % i: kept @ _quantised64(v, both=True).t() for i, v in enumerate(made["linears"])}, **sums}
        out = {"y": s / rms * w, **sums}
        if not case["train"]:
            return out
        g = made["dy"].double()
        # of y_j = s_j w_j / rms, and d rms / d s_i = s_i / (cols * rms)
        dx = g * w / rms - s * (g * w * s).sum(1, keepdim=True) / (s.shape[1] * rms ** 3)
        if case["residual"]:
            dx += made["ds"].double()
        return {**out, "dx": dx, "dw": (g * s / rms).sum(0)}
    a, b, ids = made["a"], made["b"], made["ids"]
    out = made["y"].double()
    grads = {"dx": torch.zeros_like(x, dtype=torch.float64), "da": torch.zeros_like(a, dtype=torch.float64), "db": torch.zeros_like(b, dtype=torch.float64)}
    for e in range(case["count"]):
        here = ids == e
        # the adapter as one matrix would be n x k: kept as its two factors
        left, right, xe = b[e].double() * made["scale"][e].double(), a[e].double(), x[here].double()
        inner = xe.mm(right.t())
        out[here] += inner.mm(left.t())
        if case["train"]:
            g = made["dout"][here].double()
            grads["dx"][here] = g.mm(left).mm(right)
            grads["da"][e] = g.mm(left).t().mm(xe)
            grads["db"][e] = g.t().mm(inner) * made["scale"][e].double()
    return {"out": out, **(grads if case["train"] else {})}
