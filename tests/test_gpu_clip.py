"""The global gradient norm and clipping against their definitions in 64 bits."""

import pytest
import torch

import operator_reference as R

pytestmark = pytest.mark.gpu

U = R.U
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
# 128 bytes of elements squared in float (at most 64 squares and sums, half a step
# each; the root halves that) and the result rounded to float
NORM = 2.0 ** -24 + 32 * 2.0 ** -24


def rand(seed, *shape, dtype=FL, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (size * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def parameters(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros(g.shape, dtype=g.dtype, device=g.device))
        p.grad = g
        out.append(p)
    return out


def check(grads, max_norm):
    """Clips clones of ``grads`` that lie as they do."""
    from gaussian_splats_b200.optim import clip_grad_norm, grad_norm

    want = R.norm(grads)
    assert abs(grad_norm(grads).item() - want) <= NORM * want
    kept = [g.double() for g in grads]
    norm = clip_grad_norm(parameters(grads), max_norm)
    assert norm.shape == () and norm.dtype == FL and abs(norm.item() - want) <= NORM * want
    f = R.factor(want, max_norm)
    for g, k in zip(grads, kept):
        # the factor's error, its rounding to float and the product's, the result's
        bound = (NORM + 2.0 ** -23) * (f * k).abs() + U[g.dtype] * (f * k).abs() + \
            (2.0 ** -25 if g.dtype == HF else 2.0 ** -149)
        assert ((g.double() - f * k).abs() <= 1.01 * bound).all()


SIZES = [1, 2, 3, 7, 8, 9, 255, 1000, 2048, 4096, 8192, 8193, 16384, 40000, 123457]


@pytest.mark.parametrize("dtype", [FL, BF, HF], ids=str)
@pytest.mark.parametrize("n", SIZES)
def test_one_tensor(n, dtype):
    check([rand(n, n, dtype=dtype)], 0.5)
    check([rand(n, n, dtype=dtype)], 1e9)


@pytest.mark.parametrize("count", [2, 26, 80, 81, 300, 1024, 1025, 2500])
def test_many_tensors(count):
    types = (FL, BF, HF)
    check([rand(i, 1 + (i * 7919) % 611, i % 3 + 1, dtype=types[i % 3]) for i in range(count)], 1.0)


@pytest.mark.parametrize("dtype", [FL, BF], ids=str)
@pytest.mark.parametrize("offset", range(0, 9))
def test_offsets(offset, dtype):
    """Elements in front of the first 16-byte border and behind the last; neighbours stay."""
    for n in (1, 2, 5, 8193, 20011):
        whole = rand(n, n + 20, dtype=dtype)
        before = whole.clone()
        check([whole[offset:offset + n]], 0.25)
        assert torch.equal(whole[:offset], before[:offset])
        assert torch.equal(whole[offset + n:], before[offset + n:])


def test_large():
    """More chunks than blocks, in several types."""
    check([rand(1, 12_000_001), rand(2, 9_000_003, dtype=BF), rand(3, 5, dtype=HF)], 10.0)


def test_strides():
    check([rand(1, 40, 50).t(), rand(2, 4, 5, 6).permute(2, 0, 1)], 0.5)
    whole = rand(3, 60, 64)
    before = whole.clone()
    check([whole[::2, 3:50], whole[1::2, :9]], 0.5)  # neither dense, nor overlapping
    untouched = torch.ones_like(whole, dtype=torch.bool)
    untouched[::2, 3:50] = untouched[1::2, :9] = False
    assert torch.equal(whole[untouched], before[untouched])
    check([rand(4, 0), rand(5, 3, 0, 2), rand(6, 10)], 0.5)


def test_zero_and_small_norms():
    from gaussian_splats_b200.optim import clip_grad_norm

    zeros = [torch.zeros(1000, device="cuda"), torch.zeros(3, device="cuda", dtype=BF)]
    assert clip_grad_norm(parameters(zeros), 1.0).item() == 0.0
    assert all((t == 0).all() for t in zeros)
    check([rand(1, 5000, size=1e-30)], 1e-28)
    check([rand(1, 5000, size=1e-30), torch.zeros(5000, device="cuda")], 0.0)
    g = [rand(2, 100), rand(3, 7, dtype=BF)]
    kept = [t.clone() for t in g]
    clip_grad_norm(parameters(g), 1e6)
    clip_grad_norm(parameters(g), float("inf"))
    assert all(torch.equal(a, b) for a, b in zip(g, kept))


def test_large_values():
    """Squares beyond float's range; a norm beyond it still gives the right factor."""
    check([rand(1, 5000, size=1e25), rand(2, 300)], 1.0)
    from gaussian_splats_b200.optim import clip_grad_norm

    g = torch.full((400,), 3e38, device="cuda")
    assert clip_grad_norm(parameters([g]), 10.0).item() == float("inf")
    assert ((g - 0.5).abs() <= 1e-6).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_not_finite(bad):
    from gaussian_splats_b200.optim import clip_grad_norm, grad_norm

    g = [rand(1, 9000), rand(2, 500, dtype=BF)]
    g[0][8191] = bad
    kept = [t.clone() for t in g]
    with pytest.raises(RuntimeError, match="norm is"):
        clip_grad_norm(parameters(g), 1.0, error_if_nonfinite=True)
    assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(g, kept))
    assert not grad_norm(g).isfinite()
    norm = clip_grad_norm(parameters(g), 1.0)
    if bad != bad:
        assert norm.isnan() and all(t.isnan().all() for t in g)
    else:  # factor 0: an infinity times it is NaN
        assert norm.item() == float("inf") and g[0][8191].isnan()
        assert (g[0][:8191] == 0).all() and (g[1] == 0).all()


def test_which_parameters():
    from gaussian_splats_b200.optim import clip_grad_norm

    a, b = parameters([rand(1, 100), rand(2, 50)])
    c = torch.nn.Parameter(torch.zeros(5, device="cuda"))
    want = R.norm([a.grad, b.grad])
    kept = a.grad.clone()
    norm = clip_grad_norm(iter([a, c, b, a]), 1.0)  # a once
    assert abs(norm.item() - want) <= NORM * want
    assert torch.allclose(a.grad, kept / (want + 1e-6), rtol=1e-6, atol=0)
    assert clip_grad_norm([c], 1.0).item() == 0.0
    assert clip_grad_norm(b, 1.0).item() <= 1.0 + 1e-6  # one tensor; it was clipped already
    base = torch.ones(20, device="cuda")
    norm = clip_grad_norm(parameters([base[:11], base[10:]]), 1.0)  # one element in both
    assert abs(norm.item() - 21 ** 0.5) <= NORM * 5
    assert torch.allclose(base, torch.full_like(base, 21 ** -0.5), rtol=1e-5, atol=0)
    with pytest.raises(ValueError, match="shares memory"):
        clip_grad_norm(parameters([base[:1].expand(4)]), 1.0)
    for bad in (lambda: clip_grad_norm([], 1.0), lambda: clip_grad_norm([a], -1.0),
                lambda: clip_grad_norm([a], float("nan")),
                lambda: clip_grad_norm(parameters([torch.ones(4, device="cuda").double()]), 1.0)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        clip_grad_norm(parameters([torch.ones(4), torch.ones(4, device="cuda")]), 1.0)


def test_autograd_sees_the_write():
    from gaussian_splats_b200.optim import clip_grad_norm

    p = parameters([rand(1, 10)])[0]
    leaf = torch.ones(10, device="cuda", requires_grad=True)
    product = (leaf * p.grad).sum()
    clip_grad_norm([p], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()


def test_repeats_streams_and_graph():
    from gaussian_splats_b200.optim import clip_grad_norm, grad_norm

    source = [rand(1, 300_001), rand(2, 77_777, dtype=BF), rand(3, 5, dtype=HF)]
    g = [t.clone() for t in source]
    norm = clip_grad_norm(parameters(g), 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h = [t.clone() for t in source]
        again = clip_grad_norm(parameters(h), 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(norm, again) and all(torch.equal(a, b) for a, b in zip(g, h))
    torch.cuda.synchronize()
    static, ps = [t.clone() for t in source], None
    ps = parameters(static)
    graphs = []
    for _ in range(2):  # two captures of the same gradients
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = clip_grad_norm(ps, 1.0), grad_norm(static)
        graphs.append((graph, out))
    for turn in range(4):
        for t, s in zip(static, source):
            t.copy_(s * (turn + 1))
        want = R.norm(static)
        graph, (before, after) = graphs[turn % 2]
        graph.replay()
        torch.cuda.synchronize()
        assert abs(before.item() - want) <= NORM * want
        assert abs(after.item() - 1.0) <= 1e-3  # bfloat16's roundings


@pytest.mark.parametrize("n", [1, 37, 1000])
@pytest.mark.parametrize("max_norm", [0.0, 0.3, 1e9])
def test_clipped_step(n, max_norm):
    """FusedAdam's step with a max_norm is that of gradients clipped before it, bit for
    bit, and leaves them alone."""
    from gaussian_splats_b200.optim import GROUP_NAMES, FusedAdam, clip_grad_norm

    shapes = [(n, 3), (n, 4), (n, 3), (n, 1), (n, 16, 3)]

    def optimizer():
        ps = parameters([rand(10 + i, *s) for i, s in enumerate(shapes)])
        return ps, FusedAdam([{"params": [p], "name": name, "lr": 1e-2}
                              for p, name in zip(ps, GROUP_NAMES)], eps=1e-15)

    (ps, fused), (qs, plain) = optimizer(), optimizer()
    for turn in range(3):
        for p, q in zip(ps, qs):
            q.grad = p.grad.clone()
        kept = [p.grad.clone() for p in ps]
        want = clip_grad_norm(qs, max_norm)
        plain.step()
        fused.step(max_norm=max_norm)
        assert torch.equal(fused.grad_norm, want)
        for p, q, k in zip(ps, qs, kept):
            assert torch.equal(p, q) and torch.equal(p.grad, k)
            assert torch.equal(fused.state[p]["exp_avg"], plain.state[q]["exp_avg"])
            p.grad = rand(turn, *p.shape)
    for p in ps:
        p.grad = None
    fused.step(max_norm=1.0)
    assert fused.grad_norm is None
    with pytest.raises(ValueError):
        fused.step(max_norm=-1.0)


def test_parameters_with_one_gradient():
    """Two parameters whose gradient is one tensor: it counts twice and is multiplied once."""
    from gaussian_splats_b200.optim import clip_grad_norm

    g, other = rand(1, 1000), rand(2, 50, dtype=BF)
    kept, kept_other = g.double(), other.double()
    a, b, c = parameters([g, g, other])
    want = R.norm([g, g, other])
    norm = clip_grad_norm([a, b, c, b], 1.0)
    assert abs(norm.item() - want) <= NORM * want
    f = R.factor(want, 1.0)
    for t, k in ((g, kept), (other, kept_other)):
        assert ((t.double() - f * k).abs() <= 1.01 * (NORM + 2.0 ** -23 + U[t.dtype]) *
                (f * k).abs()).all()


def test_clipped_step_with_noise_and_skipped_groups():
    """Beside the position noise and with gradients that are not there, the step is that of
    the clipped ones too."""
    from gaussian_splats_b200.optim import GROUP_NAMES, FusedAdam, clip_grad_norm

    shapes = [(333, 3), (333, 4), (333, 3), (333, 1), (333, 4, 3)]

    def optimizer():
        ps = parameters([rand(10 + i, *s) for i, s in enumerate(shapes)])
        return ps, FusedAdam([{"params": [p], "name": name, "lr": 1e-2}
                              for p, name in zip(ps, GROUP_NAMES)], eps=1e-15)

    (ps, fused), (qs, plain) = optimizer(), optimizer()
    for turn, missing in enumerate(((), (1, 4), (0,))):
        for i, (p, q) in enumerate(zip(ps, qs)):
            p.grad = None if i in missing else rand(20 + 5 * turn + i, *p.shape)
            q.grad = None if i in missing else p.grad.clone()
        want = clip_grad_norm(qs, 0.5)
        torch.manual_seed(turn)
        plain.step(noise=(5e5, 5e-4))
        torch.manual_seed(turn)
        fused.step(noise=(5e5, 5e-4), max_norm=0.5)
        assert torch.equal(fused.grad_norm, want)
        assert all(torch.equal(p, q) for p, q in zip(ps, qs))
