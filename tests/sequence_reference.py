"""The sequence operators' definitions in 64 bits, token by token, with bounds on
what rounding may change: the oracle of their tests."""

import torch


def attention(q, k, v, lengths, left, right=0, first=0, valid=None, scale=None, grad=None):
    """Dense attention of every sequence and, with ``grad``, its gradients.
    Returns a dict of float64 tensors: out, lse, (dq, dk, dv), and for each a
    ``*_spread``: the sum of the absolute values that a relative error of one
    unit in every weight (probability, or score gradient) would add up to."""
    q, k, v = q.double(), k.double(), v.double()
    tokens, heads, dim = q.shape
    group = heads // k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    r = {n: torch.zeros_like(q) for n in ("out", "out_spread", "dq", "dq_spread")}
    r |= {n: torch.zeros_like(k) for n in ("dk", "dk_spread", "dv", "dv_spread")}
    r["lse"] = torch.full((heads, tokens), -torch.inf, dtype=torch.float64, device=q.device)
    at = 0
    for n in lengths:
        i, j = torch.arange(n, device=q.device)[:, None], torch.arange(n, device=q.device)[None]
        see = (j <= i + right) & ((j >= i - left) | (j < first))
        rows = slice(at, at + n)
        if valid is not None:
            see = see & valid[rows]
        seen = see.any(0)  # rows that no query sees are left out, whatever they hold
        for h in range(heads if n else 0):
            kk = torch.where(seen[:, None], k[rows, h // group], 0.0)
            vv = torch.where(seen[:, None], v[rows, h // group], 0.0)
            qq = q[rows, h]
            s = torch.where(see, scale * (qq @ kk.T), -torch.inf)
            lse = torch.logsumexp(s, 1)
            p = torch.where(see, (s - lse[:, None]).exp(), 0.0)
            r["lse"][h, rows] = lse
            o = p @ vv
            r["out"][rows, h], r["out_spread"][rows, h] = o, p @ vv.abs()
            if grad is None:
                continue
            g = grad[rows, h].double()
            d = (g * o).sum(1, keepdim=True)
            e = p * (g @ vv.T - d)
            # one unit in each score gradient, and one in each rounded output behind d
            w = e.abs() + p * (g.abs() * o.abs()).sum(1, keepdim=True)
            r["dq"][rows, h], r["dq_spread"][rows, h] = scale * e @ kk, scale * w @ kk.abs()
            r["dk"][rows, h // group] += scale * e.T @ qq
            r["dk_spread"][rows, h // group] += scale * w.T @ qq.abs()
            r["dv"][rows, h // group] += p.T @ g
            r["dv_spread"][rows, h // group] += p.T @ g.abs()
        at += n
    return r


def gated_scan(x, gate, lengths, initial=None, grad=None, grad_last=None):
    """The recurrence token by token; gradients with ``grad`` and ``grad_last``."""
    x, gate = x.double(), gate.double()
    a, keep = gate.sigmoid(), (-gate).sigmoid()
    channels = x.shape[1]
    y, before = torch.zeros_like(x), torch.zeros_like(x)
    last = torch.zeros(len(lengths), channels, dtype=torch.float64, device=x.device)
    if initial is not None:
        last = last + initial.double()
    at = 0
    for b, n in enumerate(lengths):
        h = last[b]
        for t in range(at, at + n):
            before[t] = h
            h = keep[t] * h + a[t] * x[t]
            y[t] = h
        last[b] = h
        at += n
    r = {"y": y, "last": last}
    if grad is None:
        return r
    message = torch.zeros_like(last) if grad_last is None else grad_last.double().clone()
    back = torch.zeros_like(x)
    for b, n in enumerate(lengths):
        at = sum(lengths[:b])
        u = message[b]
        for t in range(at + n - 1, at - 1, -1):
            back[t] = grad[t].double() + u
            u = keep[t] * back[t]
        message[b] = u
    r |= {"dx": a * back, "dgate": back * (x - before) * a * keep, "dinitial": message}
    return r


def rms_norm(x, weight, residual=None, eps=1e-6, grad=None, grad_sum=None):
    """The norm and, with ``grad``, its gradients by the quotient rule."""
    z = x.double() if residual is None else x.double() + residual.double()
    w = weight.double()
    root = (z.square().mean(-1, keepdim=True) + eps).sqrt()
    r = {"y": z / root * w, "sum": z}
    if grad is not None:
        gw = grad.double() * w
        r["dz"] = gw / root - z * (gw * z).mean(-1, keepdim=True) / root ** 3
        if grad_sum is not None:
            r["dz"] = r["dz"] + grad_sum.double()
        r["dw"] = (grad.double() * z / root).reshape(-1, z.shape[-1]).sum(0)
    return r
