"""The linear layer with its epilogue against its definition in 64 bits."""

import pytest
import torch

import operator_reference as R

pytestmark = pytest.mark.gpu

U = R.U
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
SHAPES = [(1, 1, 1), (1, 8, 8), (2, 64, 128), (3, 59, 11), (5, 7, 9), (16, 2048, 24),
          (33, 136, 520), (96, 256, 1024), (127, 256, 96), (128, 64, 256), (129, 65, 257),
          (300, 520, 136), (700, 1030, 264), (1000, 72, 1000), (4097, 24, 40)]
# type, bias, residual, activation
FORMS = [(BF, None, None, None), (BF, BF, None, "gelu"), (BF, FL, FL, "silu"),
         (HF, HF, HF, "relu"), (HF, FL, None, "gelu"), (HF, None, FL, None),
         (BF, FL, BF, "silu"), (HF, HF, None, "silu"), (BF, BF, FL, "gelu"), (BF, BF, BF, None)]


def make(rows, inputs, outputs, dtype, bias, residual, seed=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    out = dtype if residual is None else residual
    return dict(x=(size * rand(rows, inputs)).to(dtype),
                weight=(inputs ** -0.5 * rand(outputs, inputs)).to(dtype),
                bias=None if bias is None else (0.5 * rand(outputs)).to(bias),
                residual=None if residual is None else (2 * rand(rows, outputs)).to(residual),
                grad=rand(rows, outputs).to(out))


def call(s, activation, train=True):
    from gaussian_splats_b200.linear import linear

    names = [n for n in ("x", "weight", "bias", "residual") if s[n] is not None]
    leaves = {n: s[n].detach().requires_grad_(train) for n in names}
    y = linear(leaves["x"], leaves["weight"], leaves.get("bias"), leaves.get("residual"),
               activation=activation)
    got = {"y": y.detach()}
    if train:
        grads = torch.autograd.grad(y, [leaves[n] for n in names], s["grad"])
        got.update({"d" + n: t for n, t in zip(names, grads)})
    return got


def bounds(s, ref, activation):
    """A float sum of n products, 16 at a time: (n / 16 + 5) units 2^-23 of the sum
    of their sizes, and one more for a float32 bias or residual. The activations' slopes
    are below 1.13 and their own errors below 1e-5 of what they return and 1e-7 of z.
    dz is rounded to the inputs' type (U), its slope to steps of 1 / 49152 before that,
    and inherits z's error through act'' (below 0.8; relu's slope may jump where z is 0
    within its error)."""
    x, w, dtype = s["x"].double().abs(), s["weight"].double().abs(), s["x"].dtype
    rows, inputs = x.shape
    outputs = len(w)
    unit = 2.0 ** -23
    z_error = (inputs / 16 + 6) * unit * ref["size"]
    out = {"y": 1.13 * z_error + 1e-5 * ref["act"].abs() + 1e-7 * ref["z"].abs() +
           unit * ref["y"].abs()}
    if "dz" not in ref:
        return out
    g = s["grad"].double().abs()
    slope_error = 0.0 if activation is None else \
        1e-5 * ref["slope"].abs() + 1.02e-5 + 1e-6 + 0.8 * z_error
    if activation == "relu":
        slope_error = slope_error + (ref["z"].abs() <= z_error)
    # subnormal float16 dz: half a step of 2^-24
    dz_error = U[dtype] * (ref["dz"].abs() + g * slope_error) + g * slope_error + 2.0 ** -25
    dz = ref["dz"].abs() + dz_error
    out["dx"] = dz_error @ w + (outputs / 16 + 6) * unit * (dz @ w) + 2.0 ** -25
    out["dweight"] = dz_error.t() @ x + (rows / 16 + 40) * unit * (dz.t() @ x) + 2.0 ** -25
    out["dbias"] = dz_error.sum(0) + (rows / 16 + 40) * unit * dz.sum(0) + 2.0 ** -25
    out["dresidual"] = 0.0
    return out


def check(got, s, activation, train=True):
    ref = R.linear(s["x"], s["weight"], s["bias"], s["residual"], activation,
                   s["grad"] if train else None)
    if train:
        ref["dresidual"] = s["grad"].double()
    inner = bounds(s, ref, activation)
    for name, t in got.items():
        assert t.shape == ref[name].shape
        bound = 1.01 * U[t.dtype] * ref[name].abs() + 1.01 * inner[name]
        error = (t.double() - ref[name]).abs()
        assert (error <= bound).all(), f"{name}: {(error - bound).max().item():.3g} beyond"


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_definition(shape, form):
    dtype, bias, residual, activation = form
    s = make(*shape, dtype, bias, residual)
    check(call(s, activation), s, activation)
    check(call(s, activation, train=False), s, activation, train=False)


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("shape", [(20003, 72, 520), (9001, 520, 300)], ids=str)
def test_many_tiles(shape, form):
    """Several tiles a block, in every form of the epilogue; with 520 inputs in pairs."""
    dtype, bias, residual, activation = form
    s = make(*shape, dtype, bias, residual)
    check(call(s, activation), s, activation)
    check(call(s, activation, train=False), s, activation, train=False)


@pytest.mark.parametrize("rows,inputs,outputs", [(40003, 264, 40), (20000, 512, 512),
                                                 (3, 4096, 2056), (70000, 8, 256),
                                                 (40003, 64, 280), (20001, 72, 281)])
def test_larger(rows, inputs, outputs):
    s = make(rows, inputs, outputs, BF, FL, FL)
    check(call(s, "gelu"), s, "gelu")


@pytest.mark.parametrize("activation", ["relu", "gelu", "silu"])
def test_far_sums(activation):
    """Sums of up to +-200, where slopes are 0 or 1 and exponentials leave their range."""
    s = make(64, 64, 64, HF, FL, None, size=60.0)
    check(call(s, activation), s, activation)


@pytest.mark.parametrize("inputs", [1, 2, 7, 10, 59, 62, 63, 64, 65, 70, 131])
@pytest.mark.parametrize("rows,outputs", [(1, 8), (130, 300), (40000, 24)])
def test_rows_that_lie_anyhow(rows, inputs, outputs):
    """Without gradients x is read in place, wherever its rows begin; what lies around
    them does not matter."""
    from gaussian_splats_b200.linear import linear

    s = make(rows, inputs, outputs, BF, FL, None)
    want = call(s, "silu", train=False)["y"]
    check({"y": want}, s, "silu", train=False)
    for offset, pitch in ((1, inputs + 3), (2, inputs + 4), (3, inputs + 2), (1, inputs)):
        whole = torch.full((rows * pitch + offset + 1,), float("nan"), device="cuda", dtype=BF)
        x = whole.as_strided((rows, inputs), (pitch, 1), offset)
        x.copy_(s["x"])
        with torch.no_grad():
            y = linear(x, s["weight"], s["bias"], activation="silu")
        assert torch.equal(y, want), (offset, pitch)


def test_special_values():
    """A row's infinities and NaN stay in that row of y and dx."""
    from gaussian_splats_b200.linear import linear

    s = make(300, 64, 72, BF, BF, FL)
    clean = call(s, "silu")
    x = s["x"].clone()
    x[17, 3], x[200, 0] = float("nan"), float("inf")
    leaf = x.requires_grad_()
    y = linear(leaf, s["weight"], s["bias"], s["residual"], activation="silu")
    dx, = torch.autograd.grad(y, leaf, s["grad"])
    rows = torch.ones(300, dtype=torch.bool, device="cuda")
    rows[17] = rows[200] = False
    assert torch.equal(y[rows], clean["y"][rows]) and torch.equal(dx[rows], clean["dx"][rows])
    assert y[17].isnan().all() and not y[200].isfinite().all()
    big = linear(torch.full((1, 8), 60000.0, device="cuda", dtype=HF),
                 torch.tensor([[1.0] * 8, [-1.0] * 8], device="cuda", dtype=HF),
                 residual=torch.zeros(1, 2, device="cuda"), activation="gelu")
    assert big.tolist() == [[480000.0, 0.0]]


@pytest.mark.parametrize("bias", [BF, FL], ids=str)
@pytest.mark.parametrize("activation", ["gelu", "silu"])
def test_nan_reaches_the_gradients(activation, bias):
    """A channel whose sums are NaN has NaN gradients, and the others theirs."""
    s = make(300, 64, 72, BF, bias, None)
    clean = call(s, activation)
    s["bias"][5] = float("nan")
    got = call(s, activation)
    others = torch.arange(72, device="cuda") != 5
    assert got["y"][:, 5].isnan().all() and got["dx"].isnan().all()
    assert got["dweight"][5].isnan().all() and got["dbias"][5].isnan()
    for name in ("dweight", "dbias"):
        assert torch.equal(got[name][others], clean[name][others])


def test_strides_and_offsets():
    """Slices of a projection, odd offsets and pitches, a transposed weight, three axes."""
    from gaussian_splats_b200.linear import linear

    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(BF)  # noqa: E731
    wide, weight = rand(200, 300), rand(80, 64)
    residual = rand(200, 160).float()
    for x in (wide[:, 8:72], wide[:, 5:69], wide[::2, 8:72], wide[1:, 1:65],
              rand(64, 200).t(), wide[:1, :64].expand(200, 64)):
        for w in (weight, rand(64, 80).t(), rand(80, 72)[:, 3:67]):
            for res in (None, residual[:len(x), 3:83], residual[:len(x), ::2],
                        residual[:1, :80].expand(len(x), 80)):
                y = linear(x, w, None, res, activation="gelu")
                whole = linear(x.contiguous(), w.contiguous(), None,
                               None if res is None else res.contiguous(), activation="gelu")
                assert torch.equal(y, whole)
    x = rand(4, 50, 64).requires_grad_()
    w = weight.clone().requires_grad_()
    y = linear(x, w, activation="silu")
    flat = linear(x.reshape(200, 64), w, activation="silu")
    assert y.shape == (4, 50, 80) and torch.equal(y.reshape(200, 80), flat)
    up = rand(4, 80, 50).transpose(1, 2)
    got = torch.autograd.grad(y, (x, w), up)
    whole = torch.autograd.grad(flat, (x, w), up.reshape(200, 80))
    assert got[0].shape == x.shape and all(torch.equal(a, b) for a, b in zip(got, whole))
    one = linear(x[0, 0], w)
    assert one.shape == (80,) and torch.equal(one, linear(x[0, :1], w)[0])


@pytest.mark.parametrize("wanted", range(1, 16))
def test_gradients_asked_for(wanted):
    from gaussian_splats_b200.linear import linear

    s = make(130, 72, 40, BF, FL, FL)
    whole = call(s, "gelu")
    names = ("x", "weight", "bias", "residual")
    leaves = {n: s[n].detach().requires_grad_(bool(wanted >> i & 1)) for i, n in enumerate(names)}
    y = linear(*leaves.values(), activation="gelu")
    some = [n for n in names if leaves[n].requires_grad]
    for n, t in zip(some, torch.autograd.grad(y, [leaves[n] for n in some], s["grad"])):
        assert torch.equal(t, whole["d" + n]), n


@pytest.mark.parametrize("wanted", range(1, 8))
def test_gradients_asked_for_without_activation(wanted):
    """The gradient itself is an operand then, and needs no copy."""
    from gaussian_splats_b200.linear import linear

    s = make(1030, 136, 200, HF, HF, None)
    whole = call(s, None)
    names = ("x", "weight", "bias")
    leaves = {n: s[n].detach().requires_grad_(bool(wanted >> i & 1)) for i, n in enumerate(names)}
    y = linear(*leaves.values())
    some = [n for n in names if leaves[n].requires_grad]
    wide = torch.empty(1030 * 200 + 1, device="cuda", dtype=HF)
    for up in (s["grad"], wide[1:].view(1030, 200).copy_(s["grad"])):  # off its 16-byte borders
        grads = torch.autograd.grad(y, [leaves[n] for n in some], up, retain_graph=True)
        for n, t in zip(some, grads):
            assert torch.equal(t, whole["d" + n]), n


def test_no_rows():
    s = make(0, 24, 16, BF, FL, FL)
    got = call(s, "gelu")
    assert got["y"].shape == (0, 16) and got["dx"].shape == (0, 24)
    assert got["dweight"].abs().max() == 0 and got["dbias"].abs().max() == 0


def test_repeats_and_leaves_the_rest_alone():
    """Bit for bit the same; rows behind the last one stay as they were."""
    import ctypes

    from gaussian_splats_b200 import native
    from gaussian_splats_b200.sequences import call as library

    s = make(5000, 136, 264, BF, BF, FL)
    a, b = call(s, "gelu"), call(s, "gelu")
    assert all(torch.equal(a[n], b[n]) for n in a)
    y = torch.full((5100, 264), 7.0, device="cuda")
    slope = torch.full((5100, 264), 7, device="cuda", dtype=torch.int16)
    args = native.LinearArgs(
        rows=5000, inputs=136, outputs=264, dtype=1, bias_dtype=1, residual_dtype=0, activation=2,
        x=s["x"].data_ptr(), weight=s["weight"].data_ptr(), bias=s["bias"].data_ptr(),
        residual=s["residual"].data_ptr(), x_stride=136, weight_stride=136, residual_stride=264,
        y=y.data_ptr(), slope=slope.data_ptr())
    library("gs_linear", y.device, ctypes.byref(args))
    assert torch.equal(y[:5000], a["y"]) and (y[5000:] == 7.0).all()
    assert (slope[5000:] == 7).all() and (slope[:5000] != 7).float().mean() > 0.99


def test_other_stream_and_graph():
    """On another stream, and captured: a replay with new inputs is a call with them."""
    from gaussian_splats_b200.linear import linear

    sets = [make(300, 72, 264, HF, FL, FL, seed=i) for i in range(3)]
    want = [call(s, "silu") for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(sets[1], "silu")
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[1][n]) for n in got)
    names = ("x", "weight", "bias", "residual")
    held = {n: sets[0][n].clone().requires_grad_() for n in names}
    up = sets[0]["grad"].clone()

    def run():
        y = linear(*held.values(), activation="silu")
        return (y, *torch.autograd.grad(y, list(held.values()), up))

    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for s, w in zip(sets[1:], want[1:]):
        with torch.no_grad():
            for n in names:
                held[n].copy_(s[n])
            up.copy_(s["grad"])
        graph.replay()
        torch.cuda.synchronize()
        for n, t in zip(("y", "dx", "dweight", "dbias", "dresidual"), out):
            assert torch.equal(t.detach(), w[n]), n


def test_arrays_past_32_bits():
    """Results, slopes and gradients of more than 2^31 elements: their last rows are those
    of a call with these rows alone, and all that reaches the weight's gradient."""
    from gaussian_splats_b200.linear import linear

    rows, tail = 2_200_003, 5001
    s = make(tail, 8, 1000, BF, BF, None)
    want = call(s, "gelu")
    x = torch.zeros(rows, 8, device="cuda", dtype=BF)
    x[-tail:] = s["x"]
    leaves = [x.requires_grad_(), s["weight"].requires_grad_()]
    y = linear(*leaves, s["bias"], activation="gelu")
    assert y.numel() > 2 ** 31
    up = torch.ones_like(y)
    up[-tail:] = s["grad"]
    dx, dw = torch.autograd.grad(y, leaves, up)
    assert torch.equal(y[-tail:], want["y"]) and torch.equal(dx[-tail:], want["dx"])
    assert torch.equal(y[0], y[-tail - 1]) and torch.equal(dx[0], dx[-tail - 1])
    # Both are sums of the same products in another order, each rounded: dz is at most 1.13 grad.
    sizes = 1.13 * s["grad"].double().abs().t() @ s["x"].double().abs()
    bound = 2 * (tail / 16 + 40) * 2.0 ** -23 * sizes + 1.01 * U[BF] * 2 * want["dweight"].double().abs()
    assert ((dw.double() - want["dweight"].double()).abs() <= 1.01 * bound + 2.0 ** -25).all()


def test_calls_at_once():
    """Products of all kinds on four streams at the same time, with nothing between them."""
    sets = [(make(3001, 264, 520, BF, FL, FL, seed=1), "gelu"),
            (make(40, 1030, 300, HF, HF, None, seed=2), "silu"),
            (make(5000, 59, 72, BF, BF, None, seed=3), "relu"),
            (make(2000, 1024, 640, HF, None, None, seed=4), None)]
    want = [call(s, a) for s, a in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for turn in range(5):
        for i, stream in enumerate(streams):
            s, activation = sets[(i + turn) % len(sets)]
            with torch.cuda.stream(stream):
                got.append(((i + turn) % len(sets), call(s, activation)))
    torch.cuda.synchronize()
    for i, results in got:
        assert all(torch.equal(results[n], want[i][n]) for n in results), i


def test_saved_tensors_may_move():
    """Hooks that take the saved tensors to the host and bring them back otherwise laid out."""
    from gaussian_splats_b200.linear import linear

    s = make(100, 72, 40, BF, FL, None)
    want = call(s, "gelu")

    def unpack(t):
        t = t.cuda()
        return t.t().contiguous().t() if t.dim() == 2 else t

    leaves = [s[n].detach().requires_grad_() for n in ("x", "weight", "bias")]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), unpack):
        y = linear(*leaves, activation="gelu")
    for n, t in zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, leaves, s["grad"])):
        assert torch.equal(t, want[n]), n


def test_refusals():
    from gaussian_splats_b200.linear import linear

    x, w = torch.zeros(4, 16, device="cuda", dtype=BF), torch.zeros(8, 16, device="cuda", dtype=BF)
    for bad in (lambda: linear(x, w.half()), lambda: linear(x.float(), w.float()),
                lambda: linear(x, w[:, :8]), lambda: linear(x, w[0]),
                lambda: linear(x, w, x[0]), lambda: linear(x, w, w[:, 0].half()),
                lambda: linear(x, w, residual=x), lambda: linear(x, w, activation="tanh"),
                lambda: linear(x, w, residual=torch.zeros(4, 8, device="cuda", dtype=HF)),
                lambda: linear(x, w[:0]), lambda: linear(x[:, :0], w[:, :0])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        linear(x, w.cpu())


@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
@pytest.mark.parametrize("rows,inputs,outputs", [
    (1, 136, 32), (96, 136, 1024), (300, 59, 128), (640, 64, 4096), (5000, 136, 264),
    (20003, 72, 520), (9001, 520, 300), (4000, 59, 260), (70, 136, 37), (1280, 136, 640),
    (1280, 59, 640), (9000, 59, 256), (18944, 59, 256)])
def test_float_results_without_a_residual(rows, inputs, outputs, dtype):
    """Which only a C caller asks for: rows by TMA and gathered, by pairs of blocks, tiles
    of every width, results that TMA takes and others."""
    import ctypes

    from gaussian_splats_b200 import native
    from gaussian_splats_b200.linear import _operand
    from gaussian_splats_b200.sequences import call as library

    for bias, activation in ((None, None), (dtype, None), (FL, None), (FL, "gelu")):
        s = make(rows, inputs, outputs, dtype, bias, None)
        w = _operand(s["weight"])
        whole = torch.full((rows * outputs + 4,), 7.0, device="cuda")
        for offset in (0, 1):  # 1: off its 16-byte borders
            y = whole[offset:offset + rows * outputs].view(rows, outputs)
            args = native.LinearArgs(
                rows=rows, inputs=inputs, outputs=outputs, dtype=1 if dtype == BF else 2,
                bias_dtype=0 if bias == FL else 1 if dtype == BF else 2, residual_dtype=0,
                activation=0 if activation is None else 2, x=s["x"].data_ptr(),
                weight=w.data_ptr(), bias=None if bias is None else s["bias"].data_ptr(),
                x_stride=inputs, weight_stride=w.stride(0), y=y.data_ptr())
            library("gs_linear", y.device, ctypes.byref(args))
            check({"y": y}, s, activation, train=False)


@pytest.mark.parametrize("name", ["x", "weight", "bias", "residual"])
def test_forward_mode_is_refused(name):
    """A tangent is refused, with reverse-mode gradients or without, and not dropped."""
    from torch.autograd import forward_ad

    from gaussian_splats_b200.linear import linear

    s = make(5, 16, 8, BF, BF, FL)
    given = {n: s[n] for n in ("x", "weight", "bias", "residual")}
    want = linear(*given.values(), activation="silu")
    with forward_ad.dual_level():
        assert torch.equal(linear(*given.values(), activation="silu"), want)  # no tangent in it
        given[name] = forward_ad.make_dual(given[name], torch.ones_like(given[name]))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(NotImplementedError):
                linear(*given.values(), activation="silu")
    assert torch.equal(linear(*(s[n] for n in given), activation="silu"), want)


@pytest.mark.parametrize("bias", [None, BF, FL], ids=str)
def test_backward_without_the_bias(bias):
    """A C caller's backward need not have the bias, whose values it does not read; the
    arguments say how the slopes are held."""
    import ctypes

    from gaussian_splats_b200 import native
    from gaussian_splats_b200.sequences import call as library

    rows, inputs, outputs = 700, 136, 264
    s = make(rows, inputs, outputs, BF, bias, None)
    want = call(s, "gelu")
    for slope_float in (0, 1):
        slope = torch.empty(rows, outputs, device="cuda", dtype=FL if slope_float else torch.int16)
        y = torch.empty(rows, outputs, device="cuda", dtype=BF)
        args = native.LinearArgs(
            rows=rows, inputs=inputs, outputs=outputs, dtype=1, bias_dtype=1 if bias == BF else 0,
            residual_dtype=1, activation=2, x=s["x"].data_ptr(), weight=s["weight"].data_ptr(),
            bias=None if bias is None else s["bias"].data_ptr(), x_stride=inputs,
            weight_stride=inputs, y=y.data_ptr(), slope=slope.data_ptr(), slope_float=slope_float)
        library("gs_linear", y.device, ctypes.byref(args))
        assert torch.equal(y, want["y"])
        grads = {"dx": torch.empty_like(s["x"]), "dweight": torch.empty_like(s["weight"]),
                 "dbias": torch.empty(outputs, device="cuda", dtype=BF if bias == BF else FL)}
        args.bias = None
        args.grad_y, args.grad_x = s["grad"].data_ptr(), grads["dx"].data_ptr()
        args.grad_weight, args.grad_bias = grads["dweight"].data_ptr(), grads["dbias"].data_ptr()
        size = native.lib().gs_linear_workspace_size(ctypes.byref(args))
        workspace = torch.empty(size, device="cuda", dtype=torch.uint8)
        args.workspace, args.workspace_size = workspace.data_ptr(), size
        library("gs_linear_backward", y.device, ctypes.byref(args))
        if bias is None:  # its gradient is written all the same
            check({n: grads[n] for n in ("dx", "dweight")}, s, "gelu")
        else:
            check(grads, s, "gelu")
            if slope_float == (bias == FL):  # as the function holds them
                assert all(torch.equal(grads[n], want[n]) for n in grads)


@pytest.mark.parametrize("dtype,bias", [(BF, FL), (HF, FL), (BF, BF), (HF, HF)], ids=str)
@pytest.mark.parametrize("activation", [None, "gelu", "silu"])
@pytest.mark.parametrize("rows,inputs,outputs", [(1, 8, 1000), (1, 8, 1001), (300, 24, 264)])
def test_gradient_of_the_bias(rows, inputs, outputs, activation, dtype, bias):
    """It is a sum of dz before its rounding to the inputs' type, with slopes that are exact
    to their own errors where the bias is float32: exponentials and reciprocals of 2^-22,
    a polynomial of 1.6e-7 and a dozen roundings of 2^-24, times 1.13 at most, less than
    2e-6 together; 1.02e-5 more where slopes are held in 16 bits. The sum is `rows` floats'.
    A float16 result below 2^-14 is rounded to steps of 2^-24."""
    s = make(rows, inputs, outputs, dtype, bias, None)
    got = call(s, activation)["dbias"]
    ref = R.linear(s["x"], s["weight"], s["bias"], None, activation, s["grad"])
    g, unit = s["grad"].double().abs(), 2.0 ** -23
    slope = 0.0 if activation is None else \
        2e-6 + 0.8 * (inputs / 16 + 6) * unit * ref["size"] + (0.0 if bias == FL else 1.02e-5)
    inner = (g * slope).sum(0) + (0.0 if rows == 1 else rows * unit / 2) * \
        (ref["dz"].abs() + g * slope).sum(0) + unit * ref["dz"].abs().sum(0)
    limit = 1.01 * (inner + U[bias] * ref["dbias"].abs() + (2.0 ** -25 if bias == HF else 0.0))
    error = (got.double() - ref["dbias"]).abs()
    assert (error <= limit).all(), f"{(error - limit).max().item():.3g} beyond"
    if bias == FL and activation:  # neither rounded dz nor slopes in 16 bits would do
        rounded = (ref["dz"].to(dtype).double().sum(0) - ref["dbias"]).abs()
        assert (rounded > limit).any()
        if rows == 1:
            codes = ((ref["slope"] + 1 / 6) * 49152).round() / 49152 - 1 / 6
            assert (((s["grad"].double() * codes).sum(0) - ref["dbias"]).abs() > limit).any()


@pytest.mark.parametrize("rows", [300, 1000])
def test_weight_gradients_of_several_turns(rows):
    """More tiles of the weight's gradient than multiprocessors, or pairs of them, and a last
    turn and last tiles that are not full."""
    s = make(rows, 2500, 5130, BF, BF, None)
    check(call(s, "gelu"), s, "gelu")


def test_no_rows_of_any_strides():
    from gaussian_splats_b200.linear import linear

    whole = torch.zeros(4, 17, 3, device="cuda", dtype=BF)
    weight = torch.ones(8, 16, device="cuda", dtype=BF, requires_grad=True)
    for x in (whole[:0, :16, 0], whole[:0, 1:, 1], whole[0, :16, :0].t(), whole[:0, 0, :1].expand(0, 16)):
        x = x.detach().requires_grad_()
        y = linear(x, weight, activation="gelu")
        dx, dw = torch.autograd.grad(y.sum(), (x, weight))
        assert y.shape == (0, 8) and dx.shape == x.shape and (dw == 0).all()
        with torch.no_grad():
            assert linear(x, weight).shape == (0, 8)
