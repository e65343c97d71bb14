"""The gated recurrence against its definition in 64 bits."""

import pytest
import torch

import sequence_reference as R

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(lengths, channels, dtype, seed=0, bias=-2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens, rand = sum(lengths), lambda *s: torch.randn(s, generator=g, device="cuda")
    both = rand(tokens, 2 * channels)
    both[:, channels:] += bias
    both = both.to(dtype)
    return dict(x=both[:, :channels], gate=both[:, channels:],
                initial=rand(len(lengths), channels), grad=rand(tokens, channels).to(dtype),
                grad_last=rand(len(lengths), channels))


def call(s, lengths, initial=True):
    from gaussian_splats_b200.recurrence import gated_scan
    from gaussian_splats_b200.sequences import PackedSequences

    leaves = [s[n].detach().requires_grad_() for n in ("x", "gate", "initial")]
    packed = None if len(lengths) == 1 else PackedSequences(lengths)
    y, last = gated_scan(leaves[0], leaves[1], packed, initial=leaves[2] if initial else None)
    grads = torch.autograd.grad((y, last), leaves if initial else leaves[:2],
                                (s["grad"], s["grad_last"]))
    return dict(zip(("y", "last", "dx", "dgate", "dinitial"), (y.detach(), last.detach(), *grads)))


def check(got, ref, dtype):
    """The states and messages are averages of what went in, so their float
    error is a few units (gates, exponentials, folds: 2e-6 in all) of the
    largest input that they hold, 8 here; then one rounding to the type."""
    for name, t in got.items():
        u = U[dtype] if t.dtype == dtype else U[torch.float32]
        bound = 1.01 * u * ref[name].abs() + 8 * 2e-6
        if dtype == torch.float16:
            bound = bound + 2.0 ** -25
        error = (t.double() - ref[name]).abs()
        assert (error <= bound).all(), f"{name}: {(error - bound).max().item():.3g} beyond"


CASES = [
    ([1], 1), ([1], 64), ([2, 0, 1], 3), ([127], 33), ([128], 64), ([129], 70),
    ([0, 300, 0, 0, 5, 128, 256, 1, 0], 40), ([1000], 256), ([3, 2500, 77], 97),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16],
                         ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("lengths,channels", CASES, ids=str)
def test_against_the_definition(lengths, channels, dtype):
    s = make(lengths, channels, dtype)
    ref = R.gated_scan(s["x"], s["gate"], lengths, s["initial"], s["grad"], s["grad_last"])
    check(call(s, lengths), ref, dtype)


@pytest.mark.parametrize("bias", [-30.0, -9.0, 0.0, 9.0, 100.0])
def test_gates_that_are_almost_shut_or_open(bias):
    s = make([700], 34, torch.float32, bias=bias)
    ref = R.gated_scan(s["x"], s["gate"], [700], s["initial"], s["grad"], s["grad_last"])
    got = call(s, [700])
    # shut gates: the messages add up 700 gradients, so the sums' error grows with them
    for name, t in got.items():
        bound = 2e-6 * (8 + 40 * ref[name].abs().max()) + 1e-5 * ref[name].abs()
        assert ((t.double() - ref[name]).abs() <= bound).all(), name


def test_long_sequence():
    """The tiles' scan over many tiles, against a walk in 64 bits."""
    lengths, channels = [70001], 8
    s = make(lengths, channels, torch.float32)
    h, keep, push = s["initial"][0].double().cpu(), None, None
    gate = s["gate"].double().cpu()
    keep, push = (-gate).sigmoid(), gate.sigmoid() * s["x"].double().cpu()
    rows = []
    for t in range(lengths[0]):
        h = keep[t] * h + push[t]
        rows.append(h)
    got = call(s, lengths)
    assert (got["y"].double().cpu() - torch.stack(rows)).abs().max() <= 8 * 2e-6


def test_without_initial_state_and_partial_gradients():
    from gaussian_splats_b200.recurrence import gated_scan

    s = make([300], 20, torch.float32)
    ref = R.gated_scan(s["x"], s["gate"], [300], None, s["grad"], s["grad_last"])
    got = call(s, [300], initial=False)
    check(got, {n: ref[n] for n in got}, torch.float32)
    x = s["x"].detach().requires_grad_()
    y, last = gated_scan(x, s["gate"])
    alone = torch.autograd.grad(last, x, s["grad_last"], retain_graph=True)[0]
    rest = torch.autograd.grad(y, x, s["grad"])[0]
    torch.testing.assert_close(alone + rest, got["dx"], rtol=1e-5, atol=1e-5)


def test_repeats_bit_for_bit_and_on_another_stream():
    s = make([5000, 300], 130, torch.bfloat16)
    a = call(s, [5000, 300])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        b = call(s, [5000, 300])
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_strides(dtype):
    s = make([260], 18, dtype)
    expected = call({n: t.contiguous() for n, t in s.items()}, [260])
    odd = torch.randn(260, 41, device="cuda").to(dtype)
    odd[:, 1:19], odd[:, 20:38] = s["x"], s["gate"]
    for x, gate in ((s["x"], s["gate"]), (odd[:, 1:19], odd[:, 20:38]),
                    (s["x"].t().contiguous().t(), s["gate"].t().contiguous().t())):
        got = call({**s, "x": x, "gate": gate,
                    "grad": s["grad"].t().contiguous().t()}, [260])
        for n in got:
            torch.testing.assert_close(got[n], expected[n], rtol=0, atol=0)


def test_a_bad_sequence_stays_alone():
    lengths = [150, 200, 90]
    s = make(lengths, 36, torch.float32)
    clean = call(s, lengths)
    s = {n: t.clone() for n, t in s.items()}
    s["x"][150:350], s["grad"][150:350] = float("nan"), float("inf")
    got = call(s, lengths)
    for n in ("y", "dx", "dgate"):
        assert torch.equal(got[n][:150], clean[n][:150])
        assert torch.equal(got[n][350:], clean[n][350:])


@pytest.mark.parametrize("channels", [64, 33], ids=["boxes", "plain"])
def test_infinite_gates_and_nan(channels):
    """A gate of minus infinity keeps the state, one of plus infinity takes the
    input; a NaN is in its own channel's states from there on and in the
    gradients up to there."""
    s = make([300], channels, torch.float32, bias=0.0)
    s["gate"][100, 1], s["gate"][150, 2], s["gate"][200, 3] = -torch.inf, torch.inf, torch.nan
    got = call(s, [300])
    y, x = got["y"], s["x"]
    assert y[100, 1] == y[99, 1] and got["dx"][100, 1] == 0 and got["dgate"][100, 1] == 0
    torch.testing.assert_close(y[150, 2], x[150, 2], rtol=1e-6, atol=1e-6)
    assert got["dgate"][150, 2] == 0
    assert y[200:, 3].isnan().all() and got["last"][0, 3].isnan()
    assert got["dx"][:201, 3].isnan().all() and got["dinitial"][0, 3].isnan()
    y[200:, 3] = 0
    assert y.isfinite().all() and got["dx"][201:].isfinite().all()
    other = [c for c in range(channels) if c != 3]
    assert all(t[..., other].isfinite().all() for t in got.values())


def test_step_with_infinite_gates_and_nan():
    from gaussian_splats_b200.recurrence import gated_scan_step

    x, state = torch.tensor([[1.0, 2.0, 3.0]], device="cuda"), torch.full((1, 3), 5.0, device="cuda")
    gate = torch.tensor([[-torch.inf, torch.inf, torch.nan]], device="cuda")
    y = gated_scan_step(x, gate, state)
    assert y[0, 0] == 5 and y[0, 1] == 2 and y[0, 2].isnan() and state[0, 2].isnan()


def test_gradient_against_differences():
    s = make([200, 61], 24, torch.float32, seed=2)
    got = call(s, [200, 61])

    def value(t):
        r = call({**s, **t}, [200, 61])
        return (r["y"].double() * s["grad"].double()).sum() + \
            (r["last"].double() * s["grad_last"].double()).sum()

    for name, grad in (("x", "dx"), ("gate", "dgate"), ("initial", "dinitial")):
        d = got[grad] / got[grad].norm()
        up, down = value({name: s[name] + 0.1 * d}), value({name: s[name] - 0.1 * d})
        # the third order of the step, and float rounding of a few thousand outputs
        assert abs((up - down) / 0.2 / got[grad].double().norm() - 1) < 2e-3, name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16],
                         ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("batch,channels", [(1, 1), (1, 2069), (7, 33), (130, 512)])
def test_step(batch, channels, dtype):
    from gaussian_splats_b200.recurrence import gated_scan_step

    g = torch.Generator(device="cuda").manual_seed(4)
    both = torch.randn((batch, 2 * channels), generator=g, device="cuda").to(dtype)
    state = torch.randn((batch, channels), generator=g, device="cuda")
    x, gate, a = both[:, :channels], both[:, channels:], both[:, channels:].double().sigmoid()
    expected = (1 - a) * state.double() + a * x.double()
    y = gated_scan_step(x, gate, state)
    assert (state.double() - expected).abs().max() <= 1e-5
    assert torch.equal(y, state.to(dtype))


def test_steps_follow_the_whole_sequence():
    from gaussian_splats_b200.recurrence import gated_scan, gated_scan_step

    s = make([140], 48, torch.float32)
    y, last = gated_scan(s["x"], s["gate"], initial=s["initial"])
    state = s["initial"].clone()
    for t in range(140):
        out = gated_scan_step(s["x"][t:t + 1], s["gate"][t:t + 1], state)
        torch.testing.assert_close(out[0], y[t], rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(state, last, rtol=1e-5, atol=1e-5)


def test_refusals():
    from gaussian_splats_b200.recurrence import gated_scan, gated_scan_step
    from gaussian_splats_b200.sequences import PackedSequences

    x = torch.zeros(10, 4, device="cuda")
    state = torch.zeros(1, 4, device="cuda")
    for error, match, args, more in [
        (RuntimeError, "CUDA devices only", (x.cpu(), x.cpu()), {}),
        (ValueError, "expected x and gate", (x, x[:5]), {}),
        (ValueError, "expected x and gate", (x[0], x[0]), {}),
        (ValueError, "gate is", (x, x.half()), {}),
        (ValueError, "float64 is not supported", (x.double(), x.double()), {}),
        (ValueError, "initial must be", (x, x), {"initial": state.half()}),
        (ValueError, "initial must be", (x, x), {"initial": x}),
        (ValueError, "hold 9 tokens", (x, x, PackedSequences([4, 5])), {}),
    ]:
        with pytest.raises(error, match=match):
            gated_scan(*args, **more)
    with pytest.raises(ValueError, match="contiguous float32"):
        gated_scan_step(x, x, x.half())
    with pytest.raises(ValueError, match="contiguous float32"):
        gated_scan_step(x, x, torch.zeros(4, 10, device="cuda").t())


def test_no_tokens():
    s = make([0, 0], 6, torch.bfloat16)
    got = call(s, [0, 0])
    assert torch.equal(got["last"], s["initial"]) and torch.equal(got["dinitial"], s["grad_last"])
    assert got["y"].shape == (0, 6)


def test_no_wait_ran_out():
    from gaussian_splats_b200 import native

    s = make([3000, 5], 64, torch.bfloat16)
    call(s, [3000, 5])
    assert native.lib().gs_gated_scan_status(torch.cuda.current_stream().cuda_stream) == 0


def tiles_of_a_span(lengths, channels, dtype):
    """How many tiles a block walks: what spans_of in recurrence.cu makes of these sizes."""
    tiles = sum(-(-n // 128) for n in lengths)
    boxes = channels % (16 // dtype.itemsize) == 0
    columns = -(-channels // (128 // dtype.itemsize if boxes else 32))
    return min(max(tiles * columns // (8 * 148), 1), 8)


SPANS = [
    # lengths, channels, type, tiles of a span; sequences end inside spans and inside tiles
    ([5000, 0, 1, 1029, 3500], 1024, torch.float32, 2),
    ([5000, 0, 1, 1029, 3500], 4096, torch.bfloat16, 4),
    ([9000, 127, 0, 10400], 4096, torch.float16, 8),
    ([5000, 0, 1, 1029, 3500], 1001, torch.bfloat16, 2),
    ([4700, 300, 0, 4600], 4001, torch.float32, 8),
]


@pytest.mark.parametrize("lengths,channels,dtype,span", SPANS, ids=str)
def test_spans_of_several_tiles(lengths, channels, dtype, span):
    """Loads into places that were used before, the carry from tile to tile, and the
    walk back through a span, for copied boxes and for plain loads."""
    assert tiles_of_a_span(lengths, channels, dtype) == span
    s = make(lengths, channels, dtype, seed=9)
    ref = R.gated_scan(s["x"], s["gate"], lengths, s["initial"], s["grad"], s["grad_last"])
    check(call(s, lengths), ref, dtype)


def one_sequence(s):
    """The definition for one long sequence: pieces of its length's root walked side by
    side in 64 bits, then joined in order."""
    x, gate = s["x"].double(), s["gate"].double()
    a, keep = gate.sigmoid(), (-gate).sigmoid()
    n, channels = x.shape

    def walk(chain, push, start):
        size = int(n ** 0.5)
        pieces = -(-n // size)
        fill = torch.zeros(pieces * size - n, channels, dtype=x.dtype, device=x.device)
        chain = torch.cat((chain, fill)).view(pieces, size, channels)
        push = torch.cat((push, fill)).view(pieces, size, channels)
        h, through = torch.zeros_like(push), torch.zeros_like(push)
        now, factor = torch.zeros_like(push[:, 0]), torch.ones_like(push[:, 0])
        for t in range(size):
            now, factor = chain[:, t] * now + push[:, t], chain[:, t] * factor
            h[:, t], through[:, t] = now, factor
        for piece in range(pieces):
            h[piece] += through[piece] * start
            start = h[piece, -1]
        return h.view(-1, channels)[:n]

    h = walk(keep, a * x, s["initial"][0].double())
    before = torch.cat((s["initial"].double(), h[:-1]))
    # u_t = keep_t (g_t + u_{t+1}), from the end
    u = walk(keep.flip(0), (keep * s["grad"].double()).flip(0), s["grad_last"][0].double()).flip(0)
    back = s["grad"].double() + torch.cat((u[1:], s["grad_last"].double()))
    return {"y": h, "last": h[-1:], "dx": a * back, "dgate": back * (x - before) * a * keep,
            "dinitial": u[:1]}


def test_the_pieces_give_the_definition():
    s = make([157], 5, torch.float32, seed=10)
    ref = R.gated_scan(s["x"], s["gate"], [157], s["initial"], s["grad"], s["grad_last"])
    for name, t in one_sequence(s).items():
        torch.testing.assert_close(t, ref[name], rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("tokens,channels,span", [(70001, 8, 1), (70001, 7, 1), (310001, 8, 2),
                                                  (310001, 7, 2), (1310001, 16, 8)])
def test_long_narrow_sequences(tokens, channels, span, dtype):
    """More than 128 spans of a sequence: the scan that shares them out to 1024 threads,
    in both directions."""
    assert tiles_of_a_span([tokens], channels, dtype) == span
    assert -(-tokens // 128) // span > 128
    s = make([tokens], channels, dtype, seed=11)
    check(call(s, [tokens]), one_sequence(s), dtype)
