"""The sequence operators over splats, as a program that trains and serves a refiner calls them.

A refiner is a sequence model whose tokens are Gaussians in a space-filling order. Its
operators: attention in a window of neighbours plus a few first tokens (training, and one new
token against a cache), a gated linear recurrence along the order (training, and one new
token), and the root-mean-square norm with the residual's addition (training, and an 8-bit
output for serving). ``run`` computes a case in plain torch operations, or, where ``own`` is
true, through this package's entry points.
"""

import math
import random

import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
_EPS = 1e-6
_E4M3_MAX = 448.0


def listed():
    return [
        # One small object, refined alone: latency counts.
        _attention("attention train, one object", 1000, 1, 4, 2, 64, 128, 128, 4, "bfloat16"),
        # A scene of 16,384 splats, window on both sides along the order, some dead splats.
        _attention("attention train, one scene", 16384, 1, 8, 8, 64, 256, 256, 16, "float16",
                   dead=0.1),
        # A batch of scenes of different sizes, causal (splats emitted one after the other).
        _attention("attention train, ragged batch", 131072, 8, 8, 4, 128, 1024, 0, 4, "bfloat16"),
        # Inference over a whole large scene.
        _attention("attention forward, large scene", 500000, 1, 4, 2, 64, 512, 512, 16,
                   "bfloat16", train=False),
        # One stream emitting splats.
        _step("attention step, one stream", 1, 8, 2, 64, 1023, 4, 1.0, "bfloat16"),
        # Many streams, caches partly filled.
        _step("attention step, many streams", 96, 16, 4, 128, 4095, 4, 1.0, "bfloat16"),
        # The recurrence over one small object.
        _scan("scan train, one object", 1000, 1, 256, "float32"),
        # One long scene with few channels: the sequence itself has to be split.
        _scan("scan train, long scene", 1000000, 1, 64, "bfloat16"),
        # A batch of scenes with many channels.
        _scan("scan train, ragged batch", 100003, 24, 1024, "bfloat16"),
        # One new token of many streams.
        {"name": "scan step, many streams", "op": "scan_step", "batch": 512, "channels": 2048,
         "dtype": "bfloat16"},
        # Training: every token of a batch, 16-bit activations on a 32-bit residual stream.
        _norm("norm train, large batch", 262144, 1024, "bfloat16", "float32", "train"),
        # Serving: a few tokens, 8-bit output for the next product.
        _norm("norm to 8 bits, few tokens", 16, 2048, "bfloat16", "bfloat16", "e4m3"),
    ]


def _attention(name, tokens, sequences, heads, kv_heads, dim, left, right, first, dtype, dead=0.0,
               train=True):
    return {"name": name, "op": "attention", "tokens": tokens, "sequences": sequences,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "left": left, "right": right,
            "first": first, "dtype": dtype, "dead": dead, "train": train}


def _step(name, batch, heads, kv_heads, dim, left, first, fill, dtype):
    return {"name": name, "op": "attention_step", "batch": batch, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "left": left, "first": first, "fill": fill,
            "dtype": dtype}


def _scan(name, tokens, sequences, channels, dtype):
    return {"name": name, "op": "scan", "tokens": tokens, "sequences": sequences,
            "channels": channels, "dtype": dtype}


def _norm(name, tokens, channels, dtype, residual, output):
    return {"name": name, "op": "norm", "tokens": tokens, "channels": channels, "dtype": dtype,
            "residual": residual, "output": output}


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention_step", "scan", "scan", "norm", "norm",
                     "scan_step"])
    if op == "attention":
        kv_heads, group = rng.choice([1, 2, 4]), rng.choice([1, 2, 4])
        left = _log(rng, 16, 2000)
        c = _attention("", _log(rng, 300, 300000), 1, kv_heads * group, kv_heads,
                       rng.choice([32, 64, 64, 96, 128, 128]), left, rng.choice([0, left]),
                       rng.choice([0, 1, 4, 16, 40]), rng.choice(["bfloat16", "float16"]),
                       rng.choice([0.0, 0.1]), rng.random() < 0.75)
        c["sequences"] = rng.choice([1, 1, min(40, max(1, c["tokens"] // 200))])
        limit = 131072 * 8 * 128 * 1100
        while c["tokens"] * c["heads"] * c["dim"] * (left + c["right"] + 100) > limit:
            c["tokens"] = c["tokens"] // 2 + 1
    elif op == "attention_step":
        kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
        c = _step("", _log(rng, 1, 256), kv_heads * group, kv_heads, rng.choice([32, 64, 96, 128]),
                  _log(rng, 30, 16000), rng.choice([0, 1, 4, 16]), rng.choice([0.5, 1.0]),
                  rng.choice(["bfloat16", "float16"]))
        while c["batch"] > 1 and c["batch"] * c["left"] * kv_heads * c["dim"] > 96 * 4096 * 4 * 128:
            c["batch"] = c["batch"] // 2
    elif op == "scan":
        c = _scan("", _log(rng, 60, 1000000), 1, _log(rng, 24, 4000),
                  rng.choice(["bfloat16", "float16", "float32"]))
        c["channels"] = max(8, c["channels"] // 8 * 8) if rng.random() < 0.7 else c["channels"]
        c["sequences"] = rng.choice([1, min(50, max(1, c["tokens"] // 50))])
        while c["tokens"] * c["channels"] > 100000000:
            c["tokens"] = c["tokens"] // 2 + 1
    elif op == "norm":
        c = _norm("", _log(rng, 1, 262144), _log(rng, 60, 8192),
                  rng.choice(["bfloat16", "float16", "float32"]), "", rng.choice(["train", "e4m3"]))
        c["residual"] = rng.choice([c["dtype"], "float32", "none"])
        c["channels"] = max(8, c["channels"] // 8 * 8) if rng.random() < 0.7 else c["channels"]
        while c["tokens"] * c["channels"] > 262144 * 1024:
            c["tokens"] = c["tokens"] // 2 + 1
    else:
        c = {"op": op, "batch": _log(rng, 1, 2000), "channels": _log(rng, 64, 4096),
             "dtype": rng.choice(["bfloat16", "float16", "float32"])}
    c.pop("name", None)
    return c


def _lengths(case):
    """The sequences' lengths: one, or a ragged split of the tokens with an empty sequence."""
    count = case["sequences"]
    if count == 1:
        return [case["tokens"]]
    rng = random.Random(case["tokens"] * 64 + count)
    cuts = sorted(rng.randint(0, case["tokens"]) for _ in range(count - 1))
    lengths = [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]
    if count >= 4:
        lengths[0], lengths[1] = lengths[0] + lengths[1], 0
    return lengths


def _pairs(case):
    """Visible (query, key) pairs of one head, dead keys not counted."""
    left, right, first, total = case["left"], case["right"], case["first"], 0
    for n in _lengths(case):
        i = torch.arange(n, dtype=torch.int64)
        low, high = (i - left).clamp(min=0), (i + right + 1).clamp(max=n)
        total += int((high - low + torch.minimum(low, torch.full_like(low, first))).sum())
    return total * (1.0 - case["dead"])


def work(case):
    op, size = case["op"], _BYTES[case["dtype"]]
    if op == "attention":
        tokens, dim = case["tokens"], case["dim"]
        q, kv = tokens * case["heads"] * dim * size, tokens * case["kv_heads"] * dim * size
        # forward: q, k, v read, out written; training: also grad_out read, dq, dk, dv written
        move = (4 * q + 4 * kv) if case["train"] else (2 * q + 2 * kv)
        flops = (14 if case["train"] else 4) * dim * case["heads"] * _pairs(case)
        return {"bytes": move, "flops": flops}
    if op == "attention_step":
        slots = (case["left"] + 1 + case["first"]) * case["fill"]
        kv = case["batch"] * case["kv_heads"] * case["dim"] * size
        q = case["batch"] * case["heads"] * case["dim"] * size
        return {"bytes": 2 * kv * (slots + 2) + 2 * q,
                "flops": 4 * case["dim"] * case["heads"] * case["batch"] * slots}
    if op == "scan":
        # x, gate, grad_y read; y, grad_x, grad_gate written
        n = case["tokens"] * case["channels"]
        return {"bytes": 6 * n * size, "flops": 16 * n}
    if op == "scan_step":
        n = case["batch"] * case["channels"]
        return {"bytes": n * (3 * size + 8), "flops": 4 * n}
    n, rows = case["tokens"] * case["channels"], case["tokens"]
    residual = 0 if case["residual"] == "none" else _BYTES[case["residual"]]
    if case["output"] == "e4m3":
        return {"bytes": n * (size + 2 * residual + 1) + 4 * rows, "flops": 6 * n}
    # x, residual, grad_y, grad_sum read; y, sum, grad_x, grad_residual written
    return {"bytes": n * (4 * size + 4 * residual), "flops": 16 * n}


def _randn(shape, seed_generator, dtype, scale=1.0):
    x = torch.randn(shape, generator=seed_generator, device="cuda", dtype=torch.float32)
    return x.mul_(scale).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], _DTYPES[case["dtype"]]
    s = {"case": case}
    if op in ("attention", "scan"):
        lengths = _lengths(case)
        s["lengths"] = lengths
        starts = [0]
        for n in lengths:
            starts.append(starts[-1] + n)
        s["offsets"] = torch.tensor(starts, dtype=torch.int64, device="cuda")
        s["packed"] = None
        if own:
            from gaussian_splats_b200.sequences import PackedSequences

            s["packed"] = PackedSequences(lengths, device="cuda")
    if op == "attention":
        tokens, dim = case["tokens"], case["dim"]
        train = case["train"]
        # the products of one projection, as a model has them: slices of one tensor
        width = (case["heads"] + 2 * case["kv_heads"]) * dim
        qkv = _randn((tokens, width), g, dtype)
        a, b = case["heads"] * dim, (case["heads"] + case["kv_heads"]) * dim
        for name, t, heads in (("q", qkv[:, :a], case["heads"]), ("k", qkv[:, a:b], case["kv_heads"]),
                               ("v", qkv[:, b:], case["kv_heads"])):
            s[name] = t.unflatten(1, (heads, dim)).detach().requires_grad_(train)
        s["valid"] = None
        if case["dead"]:
            s["valid"] = torch.rand(tokens, generator=g, device="cuda") >= case["dead"]
        if train:
            s["grad"] = _randn((tokens, case["heads"], dim), g, dtype)
    elif op == "attention_step":
        batch, dim, slots = case["batch"], case["dim"], case["left"] + 1 + case["first"]
        s["q"] = _randn((batch, case["heads"], dim), g, dtype)
        s["k"] = _randn((batch, case["kv_heads"], dim), g, dtype)
        s["v"] = _randn((batch, case["kv_heads"], dim), g, dtype)
        s["cache_k"] = _randn((batch, slots, case["kv_heads"], dim), g, dtype)
        s["cache_v"] = _randn((batch, slots, case["kv_heads"], dim), g, dtype)
        low, high = (slots, 4 * slots) if case["fill"] == 1.0 else (0, slots)
        s["positions"] = torch.randint(low, high, (batch,), generator=g, device="cuda")
    elif op == "scan":
        tokens, channels = case["tokens"], case["channels"]
        both = _randn((tokens, 2 * channels), g, dtype)
        both[:, channels:] -= 2.0  # a memory of about ten tokens
        s["x"] = both[:, :channels].detach().requires_grad_()
        s["gate"] = both[:, channels:].detach().requires_grad_()
        s["initial"] = _randn((len(s["lengths"]), channels), g, torch.float32).requires_grad_()
        s["grad"] = _randn((tokens, channels), g, dtype)
        s["grad_last"] = _randn((len(s["lengths"]), channels), g, torch.float32)
    elif op == "scan_step":
        shape = (case["batch"], case["channels"])
        s["x"] = _randn(shape, g, dtype)
        s["gate"] = _randn(shape, g, dtype) - 2.0
        s["start"] = _randn(shape, g, torch.float32)
    else:
        shape = (case["tokens"], case["channels"])
        train = case["output"] == "train"
        s["x"] = _randn(shape, g, dtype).requires_grad_(train)
        s["weight"] = (1.0 + 0.1 * torch.randn(shape[1], generator=g, device="cuda")).to(
            dtype).requires_grad_(train)
        s["residual"] = None
        if case["residual"] != "none":
            s["residual"] = _randn(shape, g, _DTYPES[case["residual"]], 2.0).requires_grad_(train)
        if train:
            s["grad"] = _randn(shape, g, dtype)
            if s["residual"] is not None:
                s["grad_sum"] = _randn(shape, g, _DTYPES[case["residual"]])
    return s


def run(s):
    op = s["case"]["op"]
    if own:
        return {"attention": _attention_own, "attention_step": _step_own, "scan": _scan_own,
                "scan_step": _scan_step_own, "norm": _norm_own}[op](s)
    with torch.no_grad():
        return {"attention": _attention_plain, "attention_step": _step_plain, "scan": _scan_plain,
                "scan_step": _scan_step_plain, "norm": _norm_plain}[op](s)


# ---------------------------------------------------------------- this package's operators


def _attention_own(s):
    from gaussian_splats_b200.attention import window_attention

    c = s["case"]
    out = window_attention(s["q"], s["k"], s["v"], s["packed"], left=c["left"], right=c["right"],
                           first=c["first"], valid=s["valid"])
    if not c["train"]:
        return {"out": out}
    dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["grad"])
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _step_own(s):
    from gaussian_splats_b200.attention import window_attention_step

    out = window_attention_step(s["q"], s["k"], s["v"], s["cache_k"], s["cache_v"],
                                s["positions"], first=s["case"]["first"])
    return {"out": out, "cache_k": s["cache_k"], "cache_v": s["cache_v"]}


def _scan_own(s):
    from gaussian_splats_b200.recurrence import gated_scan

    y, last = gated_scan(s["x"], s["gate"], s["packed"], initial=s["initial"])
    dx, dgate, dinitial = torch.autograd.grad((y, last), (s["x"], s["gate"], s["initial"]),
                                              (s["grad"], s["grad_last"]))
    return {"y": y, "last": last, "dx": dx, "dgate": dgate, "dinitial": dinitial}


def _scan_step_own(s):
    from gaussian_splats_b200.recurrence import gated_scan_step

    state = s["start"].clone()  # kept, so that the pass can be repeated
    y = gated_scan_step(s["x"], s["gate"], state)
    return {"y": y, "state": state}


def _norm_own(s):
    from gaussian_splats_b200.norm import rms_norm, rms_norm_e4m3

    c, residual = s["case"], s["residual"]
    if c["output"] == "e4m3":
        q, scale, *total = rms_norm_e4m3(s["x"], s["weight"], residual, eps=_EPS)
        return {"q": q, "scale": scale, "sum": total}
    if residual is None:
        y = rms_norm(s["x"], s["weight"], eps=_EPS)
        dx, dw = torch.autograd.grad(y, (s["x"], s["weight"]), s["grad"])
        return {"y": y, "dx": dx, "dw": dw}
    y, total = rms_norm(s["x"], s["weight"], residual, eps=_EPS)
    dx, dr, dw = torch.autograd.grad((y, total), (s["x"], residual, s["weight"]),
                                     (s["grad"], s["grad_sum"]))
    return {"y": y, "sum": total, "dx": dx, "dr": dr, "dw": dw}


# ------------------------------------------------------------------------------ plain forms


def _attention_plain(s):
    """Blocks of queries against their gathered band of keys, and against the first keys."""
    c = s["case"]
    left, right, first = c["left"], c["right"], c["first"]
    heads, kv, dim, dtype = c["heads"], c["kv_heads"], c["dim"], _DTYPES[c["dtype"]]
    group, scale = heads // kv, dim ** -0.5
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    tokens, batch, block = c["tokens"], len(s["lengths"]), 256
    blocks = max(1, -(-max(s["lengths"]) // block))
    start = s["offsets"][:-1, None]
    length = s["offsets"][1:, None] - start
    live = torch.ones(tokens, dtype=torch.bool, device=q.device) if s["valid"] is None else s["valid"]

    def place(position):  # the packed index of sequence positions, and which of them exist
        return (start + position).clamp(0, tokens - 1), (position >= 0) & (position < length)

    row = torch.arange(blocks * block, device=q.device)
    row_at, row_in = place(row[None])
    rel = torch.arange(block + left + right, device=q.device) - left
    key = (torch.arange(blocks, device=q.device)[:, None] * block + rel).reshape(-1)
    key_at, key_in = place(key[None])
    key_in = key_in & live[key_at] & (key >= first)
    head = torch.arange(first, device=q.device)
    head_at, head_in = place(head[None])
    head_in = head_in & live[head_at]

    def rows(x, n):  # tokens of the queries as [batch, blocks, kv, group * block, dim]
        return (x[row_at] * row_in[..., None, None]).reshape(batch, blocks, block, kv, group, dim).permute(
            0, 1, 3, 4, 2, 5).reshape(batch, blocks, kv, group * block, dim)

    def keys(x):  # [batch, blocks, kv, band, dim]
        return (x[key_at] * key_in[..., None, None]).reshape(batch, blocks, -1, kv, dim).transpose(2, 3)

    def heads_of(x):  # [batch, 1, kv, first, dim]
        return (x[head_at] * head_in[..., None, None]).transpose(1, 2)[:, None]

    qb, kb, vb, kh, vh = rows(q, block), keys(k), keys(v), heads_of(k), heads_of(v)
    i = row.reshape(blocks, 1, 1, block, 1)
    j = key.reshape(blocks, 1, 1, 1, -1)
    see = ((j >= i - left) & (j <= i + right)) & key_in.reshape(batch, blocks, 1, 1, 1, -1)
    see = see.expand(batch, blocks, 1, group, block, -1).reshape(batch, blocks, 1, group * block, -1)
    see_head = (head <= i + right) & head_in.reshape(batch, 1, 1, 1, 1, first)
    see_head = see_head.expand(batch, blocks, 1, group, block, -1).reshape(
        batch, blocks, 1, group * block, first)

    low = float("-inf")
    a = torch.matmul(qb, kb.transpose(-1, -2)).mul_(scale).masked_fill_(~see, low)
    b = torch.matmul(qb, kh.transpose(-1, -2)).mul_(scale).masked_fill_(~see_head, low)
    top = a.amax(-1, keepdim=True)
    if first:
        top = torch.maximum(top, b.amax(-1, keepdim=True))
    top = torch.where(top == low, 0.0, top)
    a, b = a.sub_(top).exp_(), b.sub_(top).exp_()
    total = a.sum(-1, keepdim=True) + b.sum(-1, keepdim=True)
    inverse = torch.where(total > 0, 1.0 / total, 0.0)
    a, b = a.mul_(inverse), b.mul_(inverse)
    out = torch.matmul(a, vb) + torch.matmul(b, vh)

    def unrows(x):
        x = x.reshape(batch, blocks, kv, group, block, dim).permute(0, 1, 4, 2, 3, 5)
        return x.reshape(batch, blocks * block, heads, dim)[row_in]

    result = {"out": unrows(out).to(dtype)}
    if not c["train"]:
        return result
    g = rows(s["grad"].float(), block)
    delta = (g * out).sum(-1, keepdim=True)
    dv, dvh = torch.matmul(a.transpose(-1, -2), g), torch.matmul(b.transpose(-1, -2), g).sum(1)
    da = torch.matmul(g, vb.transpose(-1, -2)).sub_(delta).mul_(a).mul_(scale)
    db = torch.matmul(g, vh.transpose(-1, -2)).sub_(delta).mul_(b).mul_(scale)
    dq = torch.matmul(da, kb) + torch.matmul(db, kh)
    dk, dkh = torch.matmul(da.transpose(-1, -2), qb), torch.matmul(db.transpose(-1, -2), qb).sum(1)

    def unkeys(band, few):
        t = torch.zeros((tokens, kv, dim), device=q.device)
        band = band.transpose(2, 3).reshape(batch, -1, kv, dim) * key_in[..., None, None]
        t.index_add_(0, key_at.reshape(-1), band.reshape(-1, kv, dim))
        few = few.transpose(1, 2) * head_in[..., None, None]
        return t.index_add_(0, head_at.reshape(-1), few.reshape(-1, kv, dim))

    result.update(dq=unrows(dq).to(dtype), dk=unkeys(dk, dkh).to(dtype), dv=unkeys(dv, dvh).to(dtype))
    return result


def _step_plain(s):
    c = s["case"]
    first, kv, dim = c["first"], c["kv_heads"], c["dim"]
    batch, slots = s["cache_k"].shape[:2]
    p = s["positions"]
    slot = torch.where(p < first, p, first + (p - first) % (slots - first))
    at = torch.arange(batch, device=p.device)
    s["cache_k"][at, slot] = s["k"]
    s["cache_v"][at, slot] = s["v"]
    k, v = s["cache_k"].float().transpose(1, 2), s["cache_v"].float().transpose(1, 2)
    q = s["q"].float().reshape(batch, kv, -1, dim)
    score = torch.matmul(q, k.transpose(-1, -2)) * dim ** -0.5
    filled = torch.arange(slots, device=p.device) <= p[:, None]
    score = score.masked_fill(~filled[:, None, None], float("-inf"))
    e = (score - score.amax(-1, keepdim=True)).exp()
    out = torch.matmul(e / e.sum(-1, keepdim=True), v)
    return {"out": out.reshape(s["q"].shape).to(s["q"].dtype), "cache_k": s["cache_k"],
            "cache_v": s["cache_v"]}


def _scan_doubling(a, b):
    """The inclusive scan of h <- a h + b along dimension 0, by doubling."""
    span = 1
    while span < a.shape[0]:
        b = torch.cat((b[:span], torch.addcmul(b[span:], a[span:], b[:-span])))
        a = torch.cat((a[:span], a[span:] * a[:-span]))
        span *= 2
    return b


def _scan_plain(s):
    x, gate, initial = s["x"].float(), s["gate"].float(), s["initial"]
    dtype = s["x"].dtype
    alpha, keep = torch.sigmoid(gate), torch.sigmoid(-gate)
    begin, end = s["offsets"][:-1], s["offsets"][1:]
    full = end > begin
    begin, tail, initial_full = begin[full], end[full] - 1, initial[full]
    first_keep = keep[begin]
    chain, push = keep.clone(), alpha * x
    push[begin] += first_keep * initial_full
    chain[begin] = 0
    h = _scan_doubling(chain, push)
    last = initial.clone()
    last[full] = h[tail]
    before = torch.cat((h[:1], h[:-1]))
    before[begin] = initial_full
    # back: l_t = grad_t + keep_{t+1} l_{t+1}
    grad, grad_last = s["grad"].float().clone(), s["grad_last"]
    grad[tail] += grad_last[full]
    chain = torch.cat((keep[1:], keep[:1]))
    chain[tail] = 0
    back = _scan_doubling(chain.flip(0), grad.flip(0)).flip(0)
    dinitial = grad_last.clone()
    dinitial[full] = first_keep * back[begin]
    dx = alpha * back
    dgate = back * (x - before) * alpha * keep
    return {"y": h.to(dtype), "last": last, "dx": dx.to(dtype), "dgate": dgate.to(dtype),
            "dinitial": dinitial}


def _scan_step_plain(s):
    alpha, keep = torch.sigmoid(s["gate"].float()), torch.sigmoid(-s["gate"].float())
    state = keep * s["start"] + alpha * s["x"].float()
    return {"y": state.to(s["x"].dtype), "state": state}


def _norm_plain(s):
    c, dtype = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    total = x if s["residual"] is None else x + s["residual"].float()
    inverse = torch.rsqrt(total.square().mean(-1, keepdim=True) + _EPS)
    hat = total * inverse
    y = hat * w
    kept = [] if s["residual"] is None else [total.to(s["residual"].dtype)]
    if c["output"] == "e4m3":
        top = y.abs().amax(-1, keepdim=True)
        scale = torch.where(top > 0, top / _E4M3_MAX, 1.0)
        q = (y / scale).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)
        return {"q": q, "scale": scale[:, 0], "sum": kept}
    g = s["grad"].float()
    gw = g * w
    d = inverse * (gw - hat * (gw * hat).mean(-1, keepdim=True))
    dw = (g * hat).sum(0).to(s["weight"].dtype)
    if s["residual"] is None:
        return {"y": y.to(dtype), "dx": d.to(dtype), "dw": dw}
    d = d + s["grad_sum"].float()
    return {"y": y.to(dtype), "sum": kept[0], "dx": d.to(dtype), "dr": d.to(s["residual"].dtype),
            "dw": dw}


# --------------------------------------------------------- the definitions, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _attention_exact, "attention_step": _step_exact, "scan": _scan_exact,
                "scan_step": _scan_step_exact, "norm": _norm_exact}[case["op"]](s)


def _attention_exact(s):
    """Row by row of the definition: 256 queries of a sequence against every key they may see."""
    c = s["case"]
    left, right, first, scale = c["left"], c["right"], c["first"], c["dim"] ** -0.5
    if _pairs(c) * c["heads"] * c["dim"] > 3e11:
        return None
    q, k, v = (s[n].detach().double().transpose(0, 1) for n in ("q", "k", "v"))  # [heads, tokens, dim]
    group = c["heads"] // c["kv_heads"]
    q = q.reshape(c["kv_heads"], group, c["tokens"], c["dim"])
    out, train = torch.zeros_like(q), c["train"]
    if train:
        g = s["grad"].double().transpose(0, 1).reshape(q.shape)
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    at = 0
    for n in s["lengths"]:
        for lo in range(0, n, 256):
            hi = min(n, lo + 256)
            js = torch.arange(max(0, lo - left), min(n, hi + right), device=q.device)
            js = torch.cat((torch.arange(min(first, int(js[0])), device=q.device), js))
            i = torch.arange(lo, hi, device=q.device)[:, None]
            see = (js <= i + right) & ((js >= i - left) | (js < first))
            if s["valid"] is not None:
                see &= s["valid"][at + js]
            kk, vv, qq = k[:, at + js][:, None], v[:, at + js][:, None], q[:, :, at + lo:at + hi]
            p = torch.where(see, scale * (qq @ kk.mT), -math.inf).softmax(-1)
            p = torch.where(see, p, 0.0)
            out[:, :, at + lo:at + hi] = p @ vv
            if train:
                gg = g[:, :, at + lo:at + hi]
                dp = gg @ vv.mT
                ds = scale * p * (dp - (p * dp).sum(-1, keepdim=True))
                dq[:, :, at + lo:at + hi] = ds @ kk
                dk.index_add_(1, at + js, (ds.mT @ qq).sum(1))
                dv.index_add_(1, at + js, (p.mT @ gg).sum(1))
        at += n
    whole = lambda t: t.reshape(-1, c["tokens"], c["dim"]).transpose(0, 1)  # noqa: E731
    result = {"out": whole(out)}
    if train:
        result.update(dq=whole(dq), dk=whole(dk), dv=whole(dv))
    return result


def _step_exact(s):
    c = s["case"]
    first, ring = c["first"], c["left"] + 1
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    ck, cv = s["cache_k"].double(), s["cache_v"].double()
    for b, p in enumerate(s["positions"].tolist()):
        slot = p if p < first else first + (p - first) % ring
        ck[b, slot], cv[b, slot] = s["k"][b].double(), s["v"][b].double()
        n = min(p + 1, first + ring)
        q = s["q"][b].double().reshape(c["kv_heads"], -1, c["dim"])
        w = torch.einsum("hgd,nhd->hgn", q, ck[b, :n]).mul(c["dim"] ** -0.5).softmax(-1)
        out[b] = torch.einsum("hgn,nhd->hgd", w, cv[b, :n]).reshape(-1, c["dim"])
    return {"out": out, "cache_k": ck, "cache_v": cv}


def _scan_exact(s):
    """Token by token, in pieces that are walked side by side and then joined in order."""
    x, gate, initial = s["x"].detach().double(), s["gate"].detach().double(), s["initial"].detach().double()
    tokens, channels = x.shape
    alpha, keep = gate.sigmoid(), (-gate).sigmoid()
    starts, ends = s["offsets"][:-1].tolist(), s["offsets"][1:].tolist()

    def walk(chain, push):
        size = max(1, int(math.isqrt(tokens)))
        pieces = -(-tokens // size)
        pad = pieces * size - tokens
        chain = torch.cat((chain, chain.new_ones(pad, channels))).reshape(pieces, size, channels)
        push = torch.cat((push, push.new_zeros(pad, channels))).reshape(pieces, size, channels)
        h, a = torch.zeros_like(push), torch.zeros_like(push)
        now, through = push.new_zeros(pieces, channels), push.new_ones(pieces, channels)
        for t in range(size):
            now = chain[:, t] * now + push[:, t]
            through = chain[:, t] * through
            h[:, t], a[:, t] = now, through
        state = push.new_zeros(channels)
        for piece in range(pieces):
            h[piece] += a[piece] * state
            state = h[piece, -1]
        return h.reshape(-1, channels)[:tokens]

    chain, push = keep.clone(), alpha * x
    for b, (lo, hi) in enumerate(zip(starts, ends)):
        if hi > lo:
            push[lo] += keep[lo] * initial[b]
            chain[lo] = 0.0
    h = walk(chain, push)
    last, before = initial.clone(), torch.zeros_like(h)
    before[1:] = h[:-1]
    grad = s["grad"].double()
    grad_last, dinitial = s["grad_last"].double(), s["grad_last"].double()
    chain = torch.zeros_like(keep)
    chain[:-1] = keep[1:]
    for b, (lo, hi) in enumerate(zip(starts, ends)):
        if hi > lo:
            last[b], before[lo] = h[hi - 1], initial[b]
            grad[hi - 1] += grad_last[b]
            chain[hi - 1] = 0.0
    back = walk(chain.flip(0), grad.flip(0)).flip(0)
    for b, (lo, hi) in enumerate(zip(starts, ends)):
        if hi > lo:
            dinitial[b] = keep[lo] * back[lo]
    return {"y": h, "last": last, "dx": alpha * back, "dgate": back * (x - before) * alpha * keep,
            "dinitial": dinitial}


def _scan_step_exact(s):
    alpha = s["gate"].double().sigmoid()
    state = s["start"].double() + alpha * (s["x"].double() - s["start"].double())
    return {"y": state, "state": state}


def _norm_exact(s):
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    r = None if s["residual"] is None else s["residual"].detach().double()
    z = x if r is None else x + r
    norm = (z.pow(2).sum(-1, keepdim=True) / z.shape[1] + _EPS).sqrt()
    y = z / norm * w
    if s["case"]["output"] == "e4m3":
        scale = y.abs().max(-1, keepdim=True).values / _E4M3_MAX
        return {"q": _nearest_e4m3(y / scale), "scale": scale[:, 0], "sum": [] if r is None else [z]}
    g = s["grad"].double()
    proj = (g * w * z).sum(-1, keepdim=True) / (z.shape[1] * norm ** 3)
    d = g * w / norm - z * proj
    dw = torch.einsum("tc,tc->c", g, z / norm)
    if r is None:
        return {"y": y, "dx": d, "dw": dw}
    d = d + s["grad_sum"].double()
    return {"y": y, "sum": z, "dx": d, "dr": d, "dw": dw}


def _nearest_e4m3(y):
    """The nearest value with 4 significant bits and exponents from -6 (below: steps of 2**-9)."""
    exponent = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20))).clamp(min=-6.0)
    step = torch.exp2(exponent - 3.0)
    return torch.round(y / step) * step
