"""What the sequence operators share: saved tensors, layouts, graphs, streams."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def operators(tokens=300):
    """For each operator a call on slices of one projection and its gradients:
    name -> (function, leaves, gradients of its outputs)."""
    from gaussian_splats_b200.attention import window_attention
    from gaussian_splats_b200.norm import rms_norm
    from gaussian_splats_b200.recurrence import gated_scan
    from gaussian_splats_b200.sequences import PackedSequences

    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    half = rand(tokens, 512).to(torch.bfloat16)
    packed = PackedSequences([tokens - 100, 0, 100])
    valid = rand(tokens) > -1.0

    def leaves(*parts):
        return [t.detach().requires_grad_() for t in parts]

    def slices(*widths):
        return half[:, :sum(widths)].split(widths, 1)

    q, k, v = (t.unflatten(1, (-1, 64)) for t in slices(256, 128, 128))
    x, gate = slices(128, 128)
    odd_x, odd_gate = half[:, 1:98], half[:, 101:198]
    weight, initial = rand(128).to(torch.bfloat16), rand(3, 128)
    return {
        "attention": (lambda q, k, v: [window_attention(q, k, v, packed, left=40, right=9, first=3,
                                                        valid=valid)],
                      leaves(q, k, v), [rand(tokens, 4, 64).to(torch.bfloat16)]),
        "scan": (lambda x, gate, initial: gated_scan(x, gate, packed, initial=initial),
                 leaves(x, gate, initial), [rand(tokens, 128).to(torch.bfloat16), rand(3, 128)]),
        "scan, odd": (lambda x, gate: gated_scan(x, gate, packed), leaves(odd_x, odd_gate),
                      [rand(tokens, 97).to(torch.bfloat16), rand(3, 97)]),
        "norm": (lambda x, w: [rms_norm(x, w)], leaves(x, weight),
                 [rand(tokens, 128).to(torch.bfloat16)]),
        "norm, residual": (lambda x, w, r: rms_norm(x, w, r), leaves(x, weight, gate.float()),
                           [rand(tokens, 128).to(torch.bfloat16), rand(tokens, 128)]),
        "norm, 16-bit residual": (lambda x, w, r: rms_norm(x, w, r), leaves(x, weight, gate),
                                  [rand(tokens, 128).to(torch.bfloat16) for _ in range(2)]),
    }


NAMES = ["attention", "scan", "scan, odd", "norm", "norm, residual",
         "norm, 16-bit residual"]


def run(function, inputs, grads):
    outputs = function(*inputs)
    return [*outputs, *torch.autograd.grad(outputs, inputs, grads)]


@pytest.mark.parametrize("pinned", [False, True], ids=["pageable", "pinned"])
@pytest.mark.parametrize("name", NAMES)
def test_saved_tensors_kept_on_the_host(name, pinned):
    """Offloading brings strided inputs back contiguous."""
    function, inputs, grads = operators()[name]
    expected = run(function, inputs, grads)
    with torch.autograd.graph.save_on_cpu(pin_memory=pinned):
        outputs = function(*inputs)
    got = [*outputs, *torch.autograd.grad(outputs, inputs, grads)]
    assert all(torch.equal(a, b) for a, b in zip(got, expected))


def test_a_layout_dropped_while_another_stream_reads_it():
    """The tables' memory is not given out again before that stream is done."""
    from gaussian_splats_b200.recurrence import gated_scan
    from gaussian_splats_b200.sequences import PackedSequences

    x = torch.randn(700, 64, device="cuda")
    expected, _ = gated_scan(x, x, PackedSequences([300, 400]))  # and the kernels are loaded
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    packed = PackedSequences([300, 400])
    sizes = [(t.data_ptr(), t.numel()) for t in (packed.tiles, packed.tile_starts)]
    with torch.cuda.stream(stream):
        torch.cuda._sleep(1_000_000_000)  # 0.5 s
        y, _ = gated_scan(x, x, packed)
    del packed
    for pointer, numel in sizes:
        others = [torch.empty(numel, dtype=torch.int32, device="cuda") for _ in range(50)]
        assert all(t.data_ptr() != pointer for t in others)
    assert not stream.query(), "the stream was done before the test was"
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(y, expected)


@pytest.mark.parametrize("name", NAMES)
def test_captured_in_a_graph(name):
    """A pass, forward and backward, is captured and gives the same again."""
    function, inputs, grads = operators()[name]
    expected = [t.detach().clone() for t in run(function, inputs, grads)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(function, inputs, grads)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = run(function, inputs, grads)
    for _ in range(2):
        with torch.no_grad():
            for t in outputs:
                t.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outputs, expected))


def test_steps_captured_in_a_graph():
    """Single-token forms: replays advance the cache and the state in place."""
    from gaussian_splats_b200.attention import window_attention_step, window_cache
    from gaussian_splats_b200.norm import rms_norm_e4m3
    from gaussian_splats_b200.recurrence import gated_scan_step

    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    tokens = rand(12, 3, 4, 64).to(torch.bfloat16)
    weight = torch.ones(64, device="cuda")

    def fresh():
        return (*window_cache(3, 6, 1, 2, 64), torch.zeros(3, 256, device="cuda"),
                torch.zeros(3, dtype=torch.int64, device="cuda"), tokens[0].clone())

    def step(cache_k, cache_v, state, positions, token):
        out = window_attention_step(token, token[:, :2], token[:, 2:], cache_k, cache_v, positions,
                                    first=1)
        y = gated_scan_step(token.flatten(1), out.flatten(1), state)
        positions += 1
        return out, y, *rms_norm_e4m3(out, weight)

    eager, called = fresh(), []
    for t in tokens:
        eager[4].copy_(t)
        called.append([x.clone() for x in step(*eager)])
    held = fresh()
    step(*held)  # warm
    for a, b in zip(held, fresh()):
        a.copy_(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step(*held)
    for t, expected in zip(tokens, called):
        held[4].copy_(t)
        graph.replay()
        for a, b in zip(results, expected):
            assert torch.equal(a.float(), b.float())
