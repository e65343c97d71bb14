"""The linear layer, gradient clipping and the 4-bit step from their definitions in
64 bits, on whatever device the tensors are."""

import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def activate(kind, z):
    """act(z) and act'(z)."""
    if kind is None:
        return z, torch.ones_like(z)
    if kind == "relu":
        return z.clamp(min=0.0), (z > 0).to(z.dtype)
    if kind == "gelu":
        half = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * half, half + z * (-0.5 * z * z).exp() / math.sqrt(2.0 * math.pi)
    gate = torch.sigmoid(z)
    return z * gate, gate * (1.0 + z * torch.sigmoid(-z))


def linear(x, weight, bias, residual, activation, grad=None):
    """y and, with ``grad``, the gradients; magnitudes for bounds beside them."""
    x, w = x.double(), weight.double()
    z = x @ w.t()
    size = x.abs() @ w.abs().t()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    y, slope = activate(activation, z)
    out = {"z": z, "size": size, "act": y, "slope": slope,
           "y": y if residual is None else y + residual.double()}
    if grad is not None:
        dz = grad.double() * slope
        out.update(dz=dz, dx=dz @ w, dweight=dz.t() @ x, dbias=dz.sum(0))
    return out


def norm(tensors):
    return math.sqrt(sum(float(t.double().square().sum()) for t in tensors))


def factor(norm_value, max_norm):
    return min(1.0, max_norm / (norm_value + 1e-6))


def held(x):
    """Rows [..., dim] as the 4-bit cache holds them: codes [..., dim], step, middle."""
    top, low = x.double().amax(-1), x.double().amin(-1)
    step, middle = ((top - low) / 15.0).to(x.dtype), ((top + low) / 2.0).to(x.dtype)
    place = (x.double() - middle.double()[..., None]) / step.double()[..., None] + 7.5
    code = place.round().clamp(0.0, 15.0)
    code = torch.where((step > 0)[..., None], code, torch.full_like(code, 8.0))
    return code.to(torch.uint8), step, middle


def packed(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


class Streams:
    """The 4-bit caches of a batch of streams, and their attention."""

    def __init__(self, batch, slots, first, kv_heads, dim, dtype, device):
        self.first, self.slots = first, slots
        self.k = torch.zeros(batch, kv_heads, slots, dim, dtype=torch.float64, device=device)
        self.v = torch.zeros_like(self.k)
        self.codes = [torch.zeros(batch, kv_heads, slots, dim // 2, dtype=torch.uint8,
                                  device=device) for _ in range(2)]
        self.ranges = [torch.zeros(batch, kv_heads, slots, 2, dtype=dtype, device=device)
                       for _ in range(2)]
        self.seen = torch.zeros(batch, slots, dtype=torch.bool, device=device)

    def step(self, q, k, v, positions, scale, valid=None):
        """The output, and beside it what its bound needs: sum p |v - middle| with
        the weights p, sum p |v|, and the size of the scores."""
        batch, heads, dim = q.shape
        kv = k.shape[1]
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        sizes = [torch.zeros_like(out) for _ in range(2)]
        score_size = torch.zeros(batch, heads, dtype=torch.float64, device=q.device)
        for b, p in enumerate(positions.tolist()):
            if p < 0:
                continue
            s = p if p < self.first else self.first + (p - self.first) % (self.slots - self.first)
            self.seen[b, s] = True if valid is None else bool(valid[b])
            for i, (x, kept) in enumerate(((k[b], self.k), (v[b], self.v))):
                code, step, middle = held(x)
                self.codes[i][b, :, s] = packed(code)
                self.ranges[i][b, :, s] = torch.stack((step, middle), -1)
                kept[b, :, s] = (code.double() - 7.5) * step.double()[:, None] + \
                    middle.double()[:, None]
            at = self.seen[b].nonzero()[:, 0]
            if len(at) == 0:
                continue
            kk, vv = (t[b][:, at].repeat_interleave(heads // kv, 0) for t in (self.k, self.v))
            middle = self.ranges[1][b][:, at, 1].double().repeat_interleave(heads // kv, 0)
            qq = q[b].double()
            score = scale * torch.einsum("hd,htd->ht", qq, kk)
            w = score.softmax(-1)
            out[b] = torch.einsum("ht,htd->hd", w, vv)
            sizes[0][b] = torch.einsum("ht,htd->hd", w, (vv - middle[..., None]).abs())
            sizes[1][b] = torch.einsum("ht,htd->hd", w, vv.abs())
            # a score's parts: q times codes (|c - 7.5| < 2^7 with the offset that
            # the products carry) and q times the middle
            step = self.ranges[0][b][:, at].double().repeat_interleave(heads // kv, 0)
            score_size[b] = scale * (qq.abs().sum(-1)[:, None] *
                                     (151.0 * step[..., 0] + step[..., 1].abs())).amax(-1)
        return out, sizes[0], sizes[1], score_size
