"""The norm with the residual's addition against its definition in 64 bits."""

import pytest
import torch

import sequence_reference as R

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
         (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
         (torch.float16, torch.float32), (torch.float32, None), (torch.bfloat16, None)]
SHAPES = [(1, 1), (3, 7), (1, 64), (17, 64), (5, 100), (300, 136), (33, 1000), (40, 1024),
          (700, 256), (9, 2048), (4, 4100), (3, 8192), (2, 16384), (2, 16383)]


def make(rows, channels, dtype, residual, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    return dict(x=rand(rows, channels).to(dtype), w=(1 + 0.2 * rand(channels)).to(dtype),
                r=None if residual is None else (2 * rand(rows, channels)).to(residual),
                g=rand(rows, channels).to(dtype),
                h=None if residual is None else rand(rows, channels).to(residual))


def call(s, eps=1e-6):
    from gaussian_splats_b200.norm import rms_norm

    x, w = s["x"].detach().requires_grad_(), s["w"].detach().requires_grad_()
    if s["r"] is None:
        y = rms_norm(x, w, eps=eps)
        dx, dw = torch.autograd.grad(y, (x, w), s["g"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    r = s["r"].detach().requires_grad_()
    y, z = rms_norm(x, w, r, eps=eps)
    dx, dr, dw = torch.autograd.grad((y, z), (x, r, w), (s["g"], s["h"]))
    return {"y": y.detach(), "sum": z.detach(), "dx": dx, "dr": dr, "dw": dw}


def check(got, s, eps=1e-6):
    """One rounding to the result's type; in front of it float sums over the
    channels or the rows (a few units of their largest terms), and, in the
    backward, the rounding of the stored sum: relative U of its type in each z,
    which reaches dz through z mean(g w z) / root**3 (each of three factors)
    and dw term by term."""
    ref = R.rms_norm(s["x"], s["w"], s["r"], eps, s["g"], s["h"])
    z, gw = ref["sum"], (s["g"].double() * s["w"].double()).abs()
    root = (z.square().mean(-1, keepdim=True) + eps).sqrt()
    stored = U[s["r"].dtype] if s["r"] is not None else 0.0
    pull = (gw * z.abs()).mean(-1, keepdim=True) * z.abs() / root ** 3
    inner = {"y": 4e-6 * ref["y"].abs(), "sum": 0.0,
             "dx": 4e-6 * (gw / root + pull) + stored * (4 * pull + gw / root),
             "dw": (4e-6 + 2 * stored) * (s["g"].double() * z / root).abs().sum(0) + 1e-6}
    inner["dr"] = inner["dx"]
    ref["dx"] = ref["dr"] = ref["dz"]
    if s["h"] is not None:
        inner["dx"] = inner["dr"] = inner["dx"] + 1e-6 * s["h"].double().abs()
    for name, t in got.items():
        bound = 1.01 * U[t.dtype] * ref[name].abs() + inner[name] + 2.0 ** -25
        error = (t.double() - ref[name]).abs()
        assert (error <= bound).all(), f"{name}: {(error - bound).max().item():.3g} beyond"


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("rows,channels", SHAPES)
def test_against_the_definition(rows, channels, types):
    s = make(rows, channels, *types)
    check(call(s), s)


@pytest.mark.parametrize("types", [(torch.bfloat16, torch.float32), (torch.float32, None)], ids=str)
def test_many_rows(types):
    s = make(5003, 320, *types)
    check(call(s), s)


def test_small_and_large_values():
    for size in (1e-4, 1e4):
        s = make(30, 256, torch.float32, torch.float32)
        s["x"], s["r"] = s["x"] * size, s["r"] * size
        check(call(s), s)
    s = make(6, 256, torch.float32, None)
    s["x"][2] = 0.0  # a token of zeros
    got = call(s)
    assert torch.isfinite(got["dx"]).all() and torch.count_nonzero(got["y"][2]) == 0
    check(got, s)


def test_a_bad_token_stays_alone():
    s = make(20, 512, torch.bfloat16, torch.bfloat16)
    clean = call(s)
    s["x"][7, 3], s["g"][7, 5] = float("nan"), float("inf")
    got = call(s)
    keep = torch.arange(20, device="cuda") != 7
    for n in ("y", "sum", "dx", "dr"):
        assert torch.equal(got[n][keep], clean[n][keep]), n
    assert torch.isnan(got["y"][7]).all()


@pytest.mark.parametrize("channels", [96, 97])
def test_strides_shapes_and_streams(channels):
    from gaussian_splats_b200.norm import rms_norm

    s = make(60, channels, torch.bfloat16, torch.float32)
    expected = call(s)
    wide = torch.cat((s["x"], s["x"]), 1)
    views = {**s, "x": wide[:, channels:], "r": s["r"].t().contiguous().t(),
             "g": s["g"].t().contiguous().t()}
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = call(views)
    torch.cuda.current_stream().wait_stream(stream)
    for n in got:
        torch.testing.assert_close(got[n], expected[n], rtol=0, atol=0)
    cube = {n: t.view(5, 12, channels) if n != "w" else t for n, t in s.items()}
    got = call(cube)
    for n in got:
        torch.testing.assert_close(got[n].view_as(expected[n]), expected[n], rtol=0, atol=0)
    assert rms_norm(s["x"][0], s["w"]).shape == (channels,)


def test_partial_gradients():
    from gaussian_splats_b200.norm import rms_norm

    s = make(10, 64, torch.float32, torch.float32)
    full = call(s)
    x, r = s["x"].requires_grad_(), s["r"].requires_grad_()
    y, z = rms_norm(x, s["w"], r)
    by_y = torch.autograd.grad(y, x, s["g"], retain_graph=True)[0]
    by_z = torch.autograd.grad(z, r, s["h"])[0]
    torch.testing.assert_close(by_y + by_z, full["dx"], rtol=1e-5, atol=1e-6)


def test_gradient_against_differences():
    s = make(40, 72, torch.float32, torch.float32, seed=3)
    got = call(s)

    def value(t):
        r = call({**s, **t})
        return sum((r[n].double() * s[k].double()).sum() for n, k in (("y", "g"), ("sum", "h")))

    for name, grad in (("x", "dx"), ("r", "dr"), ("w", "dw")):
        d = got[grad] / got[grad].norm()
        up, down = value({name: s[name] + 0.05 * d}), value({name: s[name] - 0.05 * d})
        assert abs((up - down) / 0.1 / got[grad].double().norm() - 1) < 2e-3, name


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("rows,channels", [(1, 1), (5, 100), (16, 2048), (300, 136), (3, 8192),
                                           (2, 16383)])
def test_eight_bits(rows, channels, types):
    from gaussian_splats_b200.norm import rms_norm_e4m3

    s = make(rows, channels, *types)
    if rows > 2:
        s["x"][1] = 0.0
        if s["r"] is not None:
            s["r"][1] = 0.0
    q, scale, *total = rms_norm_e4m3(s["x"], s["w"], s["r"])
    ref = R.rms_norm(s["x"], s["w"], s["r"])
    top = ref["y"].abs().amax(-1)
    expected = torch.where(top > 0, top / 448.0, 1.0)
    assert ((scale.double() - expected).abs() <= 4e-6 * expected).all()
    # half a step: 2**-4 of the value, or half the smallest step, 2**-10 of the scale
    error = (q.double() * scale.double()[:, None] - ref["y"]).abs()
    assert (error <= 1.0001 * torch.maximum(ref["y"].abs() * 2.0 ** -4,
                                            expected[:, None] * 2.0 ** -10)).all()
    if s["r"] is not None:
        assert torch.equal(total[0], (s["x"].float() + s["r"].float()).to(s["r"].dtype))


def test_refusals():
    from gaussian_splats_b200.norm import rms_norm, rms_norm_e4m3

    x, w = torch.zeros(4, 8, device="cuda"), torch.ones(8, device="cuda")
    for op in (rms_norm, rms_norm_e4m3):
        for error, match, args, more in [
            (RuntimeError, "CUDA devices only", (x.cpu(), w.cpu()), {}),
            (ValueError, "weight", (x, w[:4]), {}),
            (ValueError, "does not match", (x, w, x[:2]), {}),
            (ValueError, "residual must be", (x, w, x.half()), {}),
            (ValueError, "float64 is not supported", (x.double(), w), {}),
            (ValueError, "channels in its last axis",
             (torch.zeros(1, 16385, device="cuda"), torch.zeros(16385, device="cuda")), {}),
            (ValueError, "eps must be", (x, w), {"eps": -1.0}),
        ]:
            with pytest.raises(error, match=match):
                op(*args, **more)


def test_no_rows():
    s = make(0, 64, torch.bfloat16, torch.float32)
    got = call(s)
    assert got["y"].shape == (0, 64) and torch.count_nonzero(got["dw"]) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("rows,channels", SHAPES + [(5003, 320)])
def test_gradients_are_those_of_the_unrounded_sum(rows, channels, dtype):
    """With a 16-bit residual the sum is returned rounded, but its rounding is in no
    gradient: one rounding of the result, and float sums."""
    s = make(rows, channels, dtype, dtype, seed=5)
    got, ref = call(s), R.rms_norm(s["x"], s["w"], s["r"], 1e-6, s["g"], s["h"])
    z, gw = ref["sum"], (s["g"].double() * s["w"].double()).abs()
    root = (z.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    pull = (gw * z.abs()).mean(-1, keepdim=True) * z.abs() / root ** 3
    dz = 4e-6 * (gw / root + pull) + 1e-6 * s["h"].double().abs()
    dw = 4e-6 * (s["g"].double() * z / root).abs().sum(0) + 1e-6
    for name, expected, inner in (("dx", "dz", dz), ("dr", "dz", dz), ("dw", "dw", dw)):
        bound = 1.01 * U[dtype] * ref[expected].abs() + inner + 2.0 ** -25
        error = (got[name].double() - ref[expected]).abs()
        assert (error <= bound).all(), f"{name}: {(error - bound).max().item():.3g} beyond"


def test_a_16_bit_sum_with_rows_of_their_own_strides():
    s = make(60, 96, torch.bfloat16, torch.bfloat16)
    expected = call(s)
    wide = torch.cat((s["x"], s["r"], s["r"]), 1)
    for x, r in ((wide[:, :96], wide[:, 96:192]), (s["x"].t().contiguous().t(), wide[:, 192:])):
        got = call({**s, "x": x, "r": r})
        assert all(torch.equal(got[n], expected[n]) for n in got)


@pytest.mark.parametrize("channels", [30, 32], ids=["any", "words"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32],
                         ids=["bf16", "f16", "f32"])
def test_eight_bits_halfway_between_two_codes(dtype, channels):
    """Values whose quotient by the scale is a halfway point go to the even code. The
    largest value is 448 n, so value h n is h in units of the scale; n is odd, and for
    all but the first a product with the rounded 1 / n misses some of the points."""
    from gaussian_splats_b200.norm import rms_norm_e4m3

    halves = [17, 19, 21, 23, 25, 27, 29, 31, 8.5, 9.5, 1.0625, 1.1875, 104, 120, 2.0 ** -10,
              3 * 2.0 ** -10, 5 * 2.0 ** -10, 7 * 2.0 ** -10]
    even = [16, 20, 20, 24, 24, 28, 28, 32, 8, 10, 1, 1.25, 104, 120, 0, 2 * 2.0 ** -9,
            2 * 2.0 ** -9, 4 * 2.0 ** -9]  # 104 and 120 are codes
    x = torch.tensor([448.0] + halves + [0.0] * (channels - 1 - len(halves)), device="cuda")
    expected = torch.tensor([448.0] + even, device="cuda")
    assert torch.equal(x.to(dtype).float(), x)
    for n in (1, 49, 75, 77, 91, 93):
        weight = torch.full((channels,), float(n), dtype=dtype, device="cuda")
        for sign in (1, -1):
            q, _ = rms_norm_e4m3((sign * x[None]).to(dtype), weight)
            assert torch.equal(q.float()[0, :len(expected)], sign * expected), (n, sign)
