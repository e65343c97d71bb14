"""What a refiner with feed-forward layers trains and streams with, as a program calls it.

Three operators beside those of ``operators.py``: the linear layer (matrix product with bias,
activation and residual in its epilogue; serving and training), the global norm of many
gradients with clipping (alone, in place, and inside the splats' optimizer step), and the
attention of one new token a stream over a window's cache that is held in 4 bits. ``run``
computes a case in plain torch operations, or, where ``own`` is true, through this package's
entry points.
"""

import math
import random

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
_CLIP_EPS = 1e-6
_SPLAT_ROWS = (3, 4, 3, 1, 48)  # floats a splat: mean, rotation, scale, opacity, color (degree 3)
_SPLAT_NAMES = ("mean", "rotation", "scale", "opacity", "color")
_BETAS, _ADAM_EPS, _RATE = (0.9, 0.999), 1e-15, 1e-3


def listed():
    return [
        # A causal refiner's feed-forward for one new splat: latency counts.
        _linear("linear, one token", 1, 256, 1024, "gelu", "bfloat16", "bfloat16", "none", False),
        # A wide layer for a batch of streams: the weights are read for a few rows.
        _linear("linear, many streams", 96, 2048, 8192, "silu", "float16", "float32", "none",
                False),
        # The first layer over a large scene, splat parameters as they come: 59 of them.
        _linear("linear, large scene, 59 parameters", 500000, 59, 256, "none", "bfloat16",
                "float32", "none", False),
        # The feed-forward's way up over one scene of 16,384 splats and 4 scene tokens.
        _linear("linear train, one scene, up", 16388, 256, 1024, "gelu", "bfloat16", "bfloat16",
                "none", True),
        # Its way down over a ragged batch of scenes, added to a 32-bit residual stream.
        _linear("linear train, ragged batch, down", 131101, 1024, 256, "none", "bfloat16",
                "bfloat16", "float32", True),
        # A wide refiner: the products themselves count.
        _linear("linear train, wide", 65536, 1024, 4096, "gelu", "float16", "float16", "none",
                True),
        # The gradients of a refiner after its backward pass, clipped in place.
        _clip("clip, a refiner's gradients", "refiner", 256, 2, "bfloat16", True),
        # The norm that a trainer watches, over the gradients of 6,000,000 splats.
        _clip("norm, a large scene's gradients", "splats", 6000000, 5, "float32", False),
        # The optimizer step of 1,000,000 splats with their gradients clipped on the way.
        {"name": "clipped step, one scene", "op": "adam", "splats": 1000000, "clip": 0.25},
        # One stream emitting splats, every tenth of which is dead.
        _step("4-bit step, one stream", 1, 8, 2, 64, 1023, 4, 1.0, "bfloat16", 0.1),
        # Many streams with full windows.
        _step("4-bit step, many streams", 96, 16, 4, 128, 4095, 4, 1.0, "bfloat16", 0.0),
        # Few streams with long memories, partly filled.
        _step("4-bit step, long memories", 3, 24, 8, 96, 131071, 1, 0.5, "float16", 0.0),
    ]


def _linear(name, rows, inputs, outputs, activation, dtype, bias, residual, train):
    return {"name": name, "op": "linear", "rows": rows, "inputs": inputs, "outputs": outputs,
            "activation": activation, "dtype": dtype, "bias": bias, "residual": residual,
            "train": train}


def _clip(name, layout, size, count, dtype, clip):
    return {"name": name, "op": "clip", "layout": layout, "size": size, "count": count,
            "dtype": dtype, "clip": clip}


def _step(name, batch, heads, kv_heads, dim, left, first, fill, dtype, dead):
    return {"name": name, "op": "step", "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "left": left, "first": first, "fill": fill, "dtype": dtype, "dead": dead}


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "clip", "clip", "adam", "step", "step"])
    if op == "linear":
        dtype = rng.choice(["bfloat16", "float16"])
        c = _linear("", _log(rng, 1, 500000), _log(rng, 24, 4096), _log(rng, 24, 8192),
                    rng.choice(["none", "relu", "gelu", "silu"]), dtype,
                    rng.choice(["none", dtype, "float32"]),
                    rng.choice(["none", "none", dtype, "float32"]), rng.random() < 0.6)
        for side in ("inputs", "outputs"):
            if rng.random() < 0.7:
                c[side] = max(8, c[side] // 8 * 8)
        while c["rows"] > 1 and (
                c["rows"] * c["inputs"] * c["outputs"] > 65536 * 1024 * 4096 or
                c["rows"] * (c["inputs"] + c["outputs"]) > 131072 * 2048):
            c["rows"] = c["rows"] // 2 + 1 if c["rows"] > 2 else 1
        return _unnamed(c)
    if op == "clip":
        layout = rng.choice(["refiner", "splats", "mixed", "mixed"])
        dtype = rng.choice(["bfloat16", "float16", "float32"])
        if layout == "refiner":
            return _unnamed(_clip("", layout, rng.choice([64, 128, 256, 512]), rng.randint(1, 12),
                                  dtype, rng.random() < 0.7))
        if layout == "splats":
            return _unnamed(_clip("", layout, _log(rng, 100, 3000000), 5, "float32",
                                  rng.random() < 0.5))
        c = _clip("", layout, _log(rng, 10, 4000000), _log(rng, 1, 400), dtype, rng.random() < 0.7)
        while c["size"] * c["count"] > 200000000:
            c["count"] = c["count"] // 2 + 1
        return _unnamed(c)
    if op == "adam":
        return {"op": op, "splats": _log(rng, 100, 1000000), "clip": rng.choice([0.01, 0.25, 4.0])}
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
    c = _step("", _log(rng, 1, 256), kv_heads * group, kv_heads,
              rng.choice([32, 40, 64, 64, 96, 128, 128]), _log(rng, 20, 200000),
              rng.choice([0, 1, 4, 16]), rng.choice([0.5, 1.0]),
              rng.choice(["bfloat16", "float16"]), rng.choice([0.0, 0.0, 0.1]))
    while c["batch"] * c["left"] * kv_heads * c["dim"] > 96 * 4096 * 4 * 128:
        if c["batch"] > 1:
            c["batch"] //= 2
        else:
            c["left"] //= 2
    return _unnamed(c)


def _unnamed(case):
    return {key: value for key, value in case.items() if key != "name"}


def _gradients(case):
    """The shapes and types of a clipping case's gradients."""
    layout, size, count = case["layout"], case["size"], case["count"]
    if layout == "splats":
        return [((size, n), "float32") for n in _SPLAT_ROWS]
    if layout == "refiner":  # `count` blocks of width `size`, hidden layers four times as wide
        t = case["dtype"]
        block = [((size,), t), ((size,), t), ((2 * size, size), t), ((size, size), t),
                 ((2 * size, size), t), ((size, size), t), ((4 * size, size), t), ((4 * size,), t),
                 ((size, 4 * size), t), ((size,), t)]
        ends = [((4, size), "float32"), ((size, 59), "float32"), ((size,), "float32"),
                ((size,), t), ((59, size), "float32"), ((59,), "float32")]
        return block * count + ends
    rng = random.Random(size * 512 + count)
    return [((_log(rng, 1, size),), rng.choice([case["dtype"], case["dtype"], "float32"]))
            for _ in range(count)]


def work(case):
    if case["op"] == "linear":
        rows, inputs, outputs = case["rows"], case["inputs"], case["outputs"]
        size, out = _BYTES[case["dtype"]], _BYTES[_output(case)]
        residual = 0 if case["residual"] == "none" else _BYTES[case["residual"]]
        bias = 0 if case["bias"] == "none" else _BYTES[case["bias"]]
        move = size * (rows * inputs + inputs * outputs) + outputs * bias + \
            rows * outputs * (out + residual)
        if case["train"]:  # the gradient read; x's, the weight's, the bias's written
            move += rows * outputs * out + size * (rows * inputs + inputs * outputs) + \
                outputs * bias
        return {"bytes": move, "flops": (6 if case["train"] else 2) * rows * inputs * outputs}
    if case["op"] == "clip":
        total = sum(math.prod(shape) * _BYTES[t] for shape, t in _gradients(case))
        n = sum(math.prod(shape) for shape, _ in _gradients(case))
        return {"bytes": (2 if case["clip"] else 1) * total, "flops": 3 * n}
    if case["op"] == "adam":
        n = case["splats"] * sum(_SPLAT_ROWS)
        return {"bytes": 28 * n, "flops": 15 * n}
    slots = (case["left"] + 1 + case["first"]) * case["fill"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    held = case["batch"] * kv * slots * (dim + 8)  # two codes a byte and two ranges a row
    new = 2 * case["batch"] * (2 * heads + 2 * kv) * dim
    return {"bytes": held + new, "flops": 4 * dim * heads * case["batch"] * slots}


def _output(case):
    return case["dtype"] if case["residual"] == "none" else case["residual"]


def _randn(shape, generator, dtype, scale=1.0):
    x = torch.randn(shape, generator=generator, device="cuda", dtype=torch.float32)
    return x.mul_(scale).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "linear":
        rows, inputs, outputs = case["rows"], case["inputs"], case["outputs"]
        dtype, train = _DTYPES[case["dtype"]], case["train"]
        s["x"] = _randn((rows, inputs), g, dtype).requires_grad_(train)
        s["weight"] = _randn((outputs, inputs), g, dtype, inputs ** -0.5).requires_grad_(train)
        s["bias"] = s["residual"] = None
        if case["bias"] != "none":
            s["bias"] = _randn((outputs,), g, _DTYPES[case["bias"]], 0.5).requires_grad_(train)
        if case["residual"] != "none":
            s["residual"] = _randn((rows, outputs), g, _DTYPES[case["residual"]],
                                   2.0).requires_grad_(train)
        if train:
            s["grad"] = _randn((rows, outputs), g, _DTYPES[_output(case)])
    elif case["op"] == "clip":
        s["original"] = [_randn(shape, g, _DTYPES[t], 0.01) for shape, t in _gradients(case)]
        if case["clip"]:  # parameters as an optimizer holds them, with their gradients
            s["parameters"] = [torch.nn.Parameter(torch.zeros_like(t)) for t in s["original"]]
            for p in s["parameters"]:
                p.grad = torch.zeros_like(p)
            s["grads"] = [p.grad for p in s["parameters"]]
            total = sum(t.numel() for t in s["original"])
            s["max_norm"] = 0.01 * math.sqrt(total) / 3.0
    elif case["op"] == "adam":
        s["parameters"] = [torch.nn.Parameter(_randn((case["splats"], n), g, torch.float32))
                           for n in _SPLAT_ROWS]
        s["parameters"][4].data = s["parameters"][4].data.unflatten(1, (-1, 3))
        for p in s["parameters"]:
            p.grad = _randn(p.shape, g, torch.float32, 0.01)
        total = sum(p.numel() for p in s["parameters"])
        s["max_norm"] = case["clip"] * 0.01 * math.sqrt(total)
        s["m"] = [_randn(p.shape, g, torch.float32, 0.002) for p in s["parameters"]]
        s["v"] = [_randn(p.shape, g, torch.float32, 0.01).square_() for p in s["parameters"]]
        s["step"] = 100
        if own:
            from gaussian_splats_b200.optim import FusedAdam

            groups = [{"params": [p], "name": name, "lr": _RATE}
                      for name, p in zip(_SPLAT_NAMES, s["parameters"])]
            s["optimizer"] = FusedAdam(groups, betas=_BETAS, eps=_ADAM_EPS)
            for p, m, v in zip(s["parameters"], s["m"], s["v"]):
                s["optimizer"].state[p] = {"step": torch.tensor(float(s["step"])), "exp_avg": m,
                                           "exp_avg_sq": v}
    else:
        dtype, batch, dim, kv = (_DTYPES[case["dtype"]], case["batch"], case["dim"],
                                 case["kv_heads"])
        slots = case["left"] + 1 + case["first"]
        s["q"] = _randn((batch, case["heads"], dim), g, dtype)
        s["k"] = _randn((batch, kv, dim), g, dtype)
        s["v"] = _randn((batch, kv, dim), g, dtype)
        for name in ("k", "v"):  # the streams' earlier tokens, as the cache holds them
            held = [_held(_randn((kv, slots, dim), g, dtype)) for _ in range(batch)]
            s[name + "_codes"] = torch.stack([codes for codes, _ in held])
            s[name + "_range"] = torch.stack([ranges for _, ranges in held])
        low, high = (slots, 4 * slots) if case["fill"] == 1.0 else (slots // 4, 3 * slots // 4)
        s["positions"] = torch.randint(low, max(high, low + 1), (batch,), generator=g,
                                       device="cuda")
        s["cache_valid"] = s["valid"] = None
        if case["dead"]:
            s["cache_valid"] = torch.rand((batch, slots), generator=g, device="cuda") >= \
                case["dead"]
            s["valid"] = torch.rand(batch, generator=g, device="cuda") >= case["dead"]
    return s


def _held(x):
    """Rows ``x`` [..., dim] in 4 bits: two codes a byte, and each row's step and middle in its
    type. Codes are nearest in 64 bits, ties to the even one."""
    top, low = x.float().amax(-1), x.float().amin(-1)
    step, middle = ((top - low) / 15.0).to(x.dtype), ((top * 0.5 + low * 0.5)).to(x.dtype)
    place = (x.double() - middle.double()[..., None]) / step.double()[..., None] + 7.5
    code = place.round().clamp(0.0, 15.0)
    code = torch.where(step[..., None] > 0, code, 8.0).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, torch.stack((step, middle), -1)


def run(s):
    op = s["case"]["op"]
    if own:
        return {"linear": _linear_own, "clip": _clip_own, "adam": _adam_own,
                "step": _step_own}[op](s)
    with torch.no_grad():
        return {"linear": _linear_plain, "clip": _clip_plain, "adam": _adam_plain,
                "step": _step_plain}[op](s)


# ---------------------------------------------------------------- this package's operators


def _linear_own(s):
    from gaussian_splats_b200.linear import linear

    c = s["case"]
    activation = None if c["activation"] == "none" else c["activation"]
    y = linear(s["x"], s["weight"], s["bias"], s["residual"], activation=activation)
    if not c["train"]:
        return {"y": y}
    names = [n for n in ("x", "weight", "bias", "residual") if s[n] is not None]
    grads = torch.autograd.grad(y, [s[n] for n in names], s["grad"])
    return {"y": y, **{"d" + n: t for n, t in zip(names, grads)}}


def _clip_own(s):
    from gaussian_splats_b200.optim import clip_grad_norm, grad_norm

    if not s["case"]["clip"]:
        return {"norm": grad_norm(s["original"])}
    torch._foreach_copy_(s["grads"], s["original"])  # a backward pass's, each time
    return {"norm": clip_grad_norm(s["parameters"], s["max_norm"]), "grads": s["grads"]}


def _adam_own(s):
    s["optimizer"].step(max_norm=s["max_norm"])
    return {"norm": s["optimizer"].grad_norm, "parameters": [p.data for p in s["parameters"]],
            "m": s["m"], "v": s["v"]}


def _step_own(s):
    from gaussian_splats_b200.attention import FourBitCache, window_attention_step_4bit

    cache = FourBitCache(s["k_codes"], s["k_range"], s["v_codes"], s["v_range"])
    out = window_attention_step_4bit(s["q"], s["k"], s["v"], cache, s["positions"],
                                     first=s["case"]["first"], valid=s["valid"],
                                     cache_valid=s["cache_valid"])
    return _step_outputs(s, out)


def _step_outputs(s, out):
    """The output and the cache: its codes, two whole numbers a byte, and its ranges."""
    kept = {n: s[n] for n in ("k_codes", "k_range", "v_codes", "v_range")}
    if s["cache_valid"] is not None:
        kept["cache_valid"] = s["cache_valid"]
    return {"out": out, **kept}


# ------------------------------------------------------------------------------ plain forms


def _linear_plain(s):
    c = s["case"]
    dtype, out, kind = _DTYPES[c["dtype"]], _DTYPES[_output(c)], c["activation"]
    x, w = s["x"].float(), s["weight"].float()
    z = torch.matmul(x, w.t())
    if s["bias"] is not None:
        z += s["bias"].float()
    if kind == "none":
        y, slope = z, None
    elif kind == "relu":
        y, slope = z.clamp(min=0.0), (z > 0).float()
    elif kind == "gelu":
        half = 0.5 * torch.erfc(z * -(0.5 ** 0.5))
        y = z * half
        slope = half + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5 if c["train"] else None
    else:
        gate = torch.sigmoid(z)
        y = z * gate
        slope = gate * (1.0 + z * torch.sigmoid(-z)) if c["train"] else None
    if s["residual"] is not None:
        y = y + s["residual"].float()
    result = {"y": y.to(out)}
    if not c["train"]:
        return result
    dz = s["grad"].float()
    if slope is not None:
        dz = dz * slope
    result.update(dx=torch.matmul(dz, w).to(dtype), dweight=torch.matmul(dz.t(), x).to(dtype))
    if s["bias"] is not None:
        result["dbias"] = dz.sum(0, dtype=torch.float64).to(s["bias"].dtype)
    if s["residual"] is not None:
        result["dresidual"] = s["grad"]
    return result


def _clip_plain(s):
    if not s["case"]["clip"]:
        return {"norm": _norm_plain(s["original"]).float()}
    torch._foreach_copy_(s["grads"], s["original"])
    norm = _norm_plain(s["grads"])
    scale = (s["max_norm"] / (norm + _CLIP_EPS)).clamp(max=1.0).float()
    for t in s["grads"]:
        t.copy_(t.float() * scale)
    return {"norm": norm.float(), "grads": s["grads"]}


def _norm_plain(tensors):
    return torch.stack([t.double().square().sum() for t in tensors]).sum().sqrt()


def _adam_plain(s):
    norm = _norm_plain([p.grad for p in s["parameters"]])
    scale = (s["max_norm"] / (norm + _CLIP_EPS)).clamp(max=1.0).float()
    s["step"] += 1
    right1, right2 = 1.0 - _BETAS[0] ** s["step"], 1.0 - _BETAS[1] ** s["step"]
    for p, m, v in zip(s["parameters"], s["m"], s["v"]):
        g = p.grad * scale
        m.add_((g - m) * (1.0 - _BETAS[0]))
        v.mul_(_BETAS[1]).add_(g * g * (1.0 - _BETAS[1]))
        p.data.sub_(m / (v.sqrt() / math.sqrt(right2) + _ADAM_EPS) * (_RATE / right1))
    return {"norm": norm.float(), "parameters": [p.data for p in s["parameters"]], "m": s["m"],
            "v": s["v"]}


def _open(codes, ranges):
    """What codes stand for, [..., dim] in 32 bits."""
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    return (code - 7.5) * ranges[..., :1].float() + ranges[..., 1:].float()


def _step_plain(s):
    c = s["case"]
    first, kv, dim = c["first"], c["kv_heads"], c["dim"]
    batch, _, slots = s["k_codes"].shape[:3]
    p = s["positions"]
    slot = torch.where(p < first, p, first + (p - first) % (slots - first))
    at = torch.arange(batch, device=p.device)
    for name in ("k", "v"):
        codes, ranges = _held(s[name])
        s[name + "_codes"][at, :, slot] = codes
        s[name + "_range"][at, :, slot] = ranges
    filled = torch.arange(slots, device=p.device) <= p[:, None]
    if s["cache_valid"] is not None:
        s["cache_valid"][at, slot] = s["valid"]
        filled = filled & s["cache_valid"]
    out = torch.empty_like(s["q"])
    piece = max(1, (1 << 28) // (kv * slots * dim))  # streams whose opened cache fits in memory
    for lo in range(0, batch, piece):
        part = slice(lo, lo + piece)
        k, v = (_open(s[n + "_codes"][part], s[n + "_range"][part]) for n in ("k", "v"))
        q = s["q"][part].float().unflatten(1, (kv, -1))
        score = torch.matmul(q, k.transpose(-1, -2)) * dim ** -0.5
        score = score.masked_fill(~filled[part, None, None], float("-inf"))
        top = score.amax(-1, keepdim=True)
        e = (score - torch.where(top == float("-inf"), 0.0, top)).exp()
        total = e.sum(-1, keepdim=True)
        e = e * torch.where(total > 0, 1.0 / total, 0.0)
        out[part] = torch.matmul(e, v).flatten(1, 2).to(out.dtype)
    return _step_outputs(s, out)


# --------------------------------------------------------- the definitions, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"linear": _linear_exact, "clip": _clip_exact, "adam": _adam_exact,
                "step": _step_exact}[case["op"]](s)


def _linear_exact(s):
    """In pieces of rows, whose gradients of the weight and the bias add up."""
    c = s["case"]
    w = s["weight"].detach().double()
    b = None if s["bias"] is None else s["bias"].detach().double()
    ys, dxs, dw, db = [], [], torch.zeros_like(w), w.new_zeros(len(w))
    for lo in range(0, c["rows"], 16384):
        rows = slice(lo, lo + 16384)
        x = s["x"].detach()[rows].double()
        z = x @ w.mT if b is None else torch.addmm(b, x, w.mT)
        if c["activation"] == "gelu":
            y, slope = 0.5 * z * torch.erfc(-z / math.sqrt(2.0)), 0.5 * torch.erfc(
                -z / math.sqrt(2.0)) + z * (-z.pow(2) / 2.0).exp() / math.sqrt(2.0 * math.pi)
        elif c["activation"] == "silu":
            down = (-z).exp() + 1.0
            y, slope = z / down, (down + z * (down - 1.0)) / down.pow(2)
            slope = torch.where(z < -300.0, 0.0, slope)
        elif c["activation"] == "relu":
            y, slope = torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0).double()
        else:
            y, slope = z, None
        if s["residual"] is not None:
            y = s["residual"].detach()[rows].double() + y
        ys.append(y)
        if c["train"]:
            dz = s["grad"][rows].double()
            dz = dz if slope is None else slope * dz
            dxs.append(dz @ w)
            dw += dz.mT @ x
            db += torch.einsum("rn->n", dz)
    result = {"y": torch.cat(ys)}
    if c["train"]:
        result.update(dx=torch.cat(dxs), dweight=dw)
        if b is not None:
            result["dbias"] = db
        if s["residual"] is not None:
            result["dresidual"] = s["grad"].double()
    return result


def _length(tensors):
    """The length of all tensors' elements together, tensor by tensor."""
    total = 0.0
    for t in tensors:
        flat = t.detach().reshape(-1)
        for lo in range(0, flat.numel(), 1 << 26):
            part = flat[lo:lo + (1 << 26)].double()
            total += float(torch.dot(part, part))
    return math.sqrt(total)


def _clip_exact(s):
    norm = _length(s["original"])
    result = {"norm": torch.tensor(norm, dtype=torch.float64, device="cuda")}
    if s["case"]["clip"]:
        factor = min(1.0, s["max_norm"] / (norm + _CLIP_EPS))
        result["grads"] = [factor * t.double() for t in s["original"]]
    return result


def _adam_exact(s):
    grads = [p.grad for p in s["parameters"]]
    norm = _length(grads)
    factor = min(1.0, s["max_norm"] / (norm + _CLIP_EPS))
    n, (b1, b2) = s["step"] + 1, _BETAS
    ps, ms, vs = [], [], []
    for p, g, m, v in zip(s["parameters"], grads, s["m"], s["v"]):
        g = factor * g.double()
        m = b1 * m.double() + (1.0 - b1) * g
        v = b2 * v.double() + (1.0 - b2) * g.pow(2)
        rate = _RATE * (m / (1.0 - b1 ** n)) / ((v / (1.0 - b2 ** n)).sqrt() + _ADAM_EPS)
        ps.append(p.detach().double() - rate)
        ms.append(m)
        vs.append(v)
    return {"norm": torch.tensor(norm, dtype=torch.float64, device="cuda"), "parameters": ps,
            "m": ms, "v": vs}


def _step_exact(s):
    """Stream by stream and head by head, over the slots that count."""
    c = s["case"]
    first, ring, kv = c["first"], c["left"] + 1, c["kv_heads"]
    group = c["heads"] // kv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    kept = {n: s[n].clone() for n in ("k_codes", "k_range", "v_codes", "v_range")}
    valid = None if s["cache_valid"] is None else s["cache_valid"].clone()
    for b, p in enumerate(s["positions"].tolist()):
        slot = p if p < first else first + (p - first) % ring
        n = min(p + 1, first + ring)
        if valid is not None:
            valid[b, slot] = s["valid"][b]
        seen = slice(0, n) if valid is None else valid[b, :n].nonzero()[:, 0]
        for h in range(kv):
            opened = {}
            for name in ("k", "v"):
                x = s[name][b, h].double()
                step = ((x.max() - x.min()) / 15.0).to(s[name].dtype)
                middle = ((x.max() + x.min()) / 2.0).to(s[name].dtype)
                distance = (x[:, None] - middle.double()).sub(
                    (torch.arange(16, device=x.device) - 7.5) * step.double()).abs()
                best = distance.amin(1, keepdim=True)
                even = torch.arange(16, device=x.device) % 2
                code = (torch.where(distance == best, 0, 2) + even).argmin(1)
                code = (code if float(step) > 0 else torch.full_like(code, 8)).to(torch.uint8)
                codes, ranges = kept[name + "_codes"], kept[name + "_range"]
                codes[b, h, slot] = code[0::2] + 16 * code[1::2]
                ranges[b, h, slot, 0], ranges[b, h, slot, 1] = step, middle
                row, span = codes[b, h, :n][seen], ranges[b, h, :n][seen].double()
                value = torch.empty((len(row), c["dim"]), dtype=torch.float64, device=x.device)
                value[:, 0::2], value[:, 1::2] = (row % 16).double(), (row // 16).double()
                opened[name] = value.sub_(7.5).mul_(span[:, :1]).add_(span[:, 1:])
            if len(opened["k"]):
                q = s["q"][b, h * group:(h + 1) * group].double()
                weight = (q @ opened["k"].mT / math.sqrt(c["dim"])).softmax(-1)
                out[b, h * group:(h + 1) * group] = weight @ opened["v"]
    if valid is not None:
        kept["cache_valid"] = valid
    return {"out": out, **kept}
