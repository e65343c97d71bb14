"""A refiner with feed-forward layers: the linear layer, clipping and 4-bit caches run with
the other sequence operators, as they are meant to be used."""

import pytest
import torch

import operator_reference as R
from gaussian_splats_b200.refine import RefinerShape, SplatRefiner, morton_order
from gaussian_splats_b200.splats import GaussianSplat
from test_gpu_refine import GaussianLike, scene, shaken

pytestmark = pytest.mark.gpu

NAMES = ("mean", "rotation", "scale", "opacity", "color")
SHAPE = dict(width=128, heads=2, kv_heads=1, left=40, right=20, hidden=512)


def plain_linear(x, weight, bias=None, residual=None, *, activation=None):
    z = torch.nn.functional.linear(x.float(), weight.float(), None if bias is None else bias.float())
    y, _ = R.activate(activation, z)
    y = y if residual is None else y + residual.float()
    return y.to(x.dtype if residual is None else residual.dtype)


def made(seed=0, **shape):
    torch.manual_seed(seed)
    refiner = shaken(SplatRefiner(shape=RefinerShape(**{**SHAPE, **shape})))
    with torch.no_grad():
        for block in refiner.blocks:
            torch.nn.init.normal_(block.feed.up_bias, std=0.3)
    return refiner


def test_no_feed_forward_by_default():
    torch.manual_seed(0)
    refiner = SplatRefiner()
    assert all(block.feed is None for block in refiner.blocks)
    assert not any("feed" in name for name in refiner.state_dict())


def test_follows_the_plain_layer(monkeypatch):
    """Values and gradients with the plain layer in its place: the bfloat16 results'
    roundings differ here and there by a unit (2^-8), which two blocks carry on."""
    from gaussian_splats_b200 import refine

    refiner, scenes = made(), [scene(300, 1, dead=30), scene(1, 2), scene(777, 3)]

    def values():
        return torch.cat([torch.cat([t.flatten() for t in s.values()]) for s in refiner(scenes)])

    def run():
        out = values()
        return out, torch.autograd.grad(out.square().sum(), list(refiner.parameters()))

    out, grads = run()
    with monkeypatch.context() as m:
        m.setattr(refine, "linear", plain_linear)
        want, want_grads = run()
    torch.testing.assert_close(out, want, rtol=0, atol=3e-2)
    for (name, p), a, b in zip(refiner.named_parameters(), grads, want_grads):
        # sums over a thousand tokens of terms that are 2^-8 off
        assert (a.float() - b.float()).norm() <= 0.05 * b.float().norm() + 1e-6, name
    assert any("feed" in n for n, _ in refiner.named_parameters())
    with monkeypatch.context() as m:
        m.setattr(refine._FeedForward, "forward", lambda self, y, x: x)
        assert not torch.equal(values(), want)  # the layers matter


@pytest.mark.parametrize("max_norm", [1e-3, 1e6])
def test_clipped_training_step(max_norm):
    """Rendered loss, gradients, clipping, step: the clipped gradients are the unclipped
    ones times the factor, whatever their types."""
    from gaussian_splats_b200 import scenes as S
    from gaussian_splats_b200.losses import l1_loss
    from gaussian_splats_b200.optim import clip_grad_norm
    from gaussian_splats_b200.rasterize import rasterize

    s = S.config1(num_points=2000, image=128)
    camera = s.cameras[0]
    given = GaussianSplat.from_tensors(*(t.cuda() for t in s.tensors()))
    with torch.no_grad():
        target = rasterize(given, camera, tile_size=16) * 0.5
    refiner = made(left=64, right=64)
    optimizer = torch.optim.Adam(refiner.parameters(), lr=1e-3)
    for _ in range(2):
        out = refiner([given])[0]
        loss = l1_loss(rasterize(GaussianLike(out), camera, tile_size=16), target)
        optimizer.zero_grad()
        loss.backward()
        grads = [p.grad.clone() for p in refiner.parameters()]
        assert all(torch.isfinite(g).all() for g in grads)
        want = R.norm(grads)
        norm = clip_grad_norm(refiner.parameters(), max_norm)
        assert abs(norm.item() - want) <= 33 * 2.0 ** -24 * want
        f = R.factor(want, max_norm)
        for p, g in zip(refiner.parameters(), grads):
            bound = (R.U[g.dtype] + 2.0 ** -20) * (f * g.double()).abs() + 2.0 ** -126
            assert ((p.grad.double() - f * g.double()).abs() <= bound).all()
            if f == 1.0:
                assert torch.equal(p.grad, g)
        optimizer.step()
    assert all(torch.isfinite(p).all() for p in refiner.parameters())


def test_captured_step():
    """Forward, backward and clipping captured once and replayed."""
    from gaussian_splats_b200.optim import clip_grad_norm

    refiner, splats = made(blocks=1), scene(200, 4)
    features = torch.randn(200, refiner.shape.width, device="cuda")
    block = refiner.blocks[0]
    valid = torch.ones(200, dtype=torch.bool, device="cuda")

    def step():
        for p in block.parameters():
            p.grad = None
        x, residual = block(torch.zeros_like(features, dtype=torch.bfloat16), features, None, valid)
        (x.float() * residual).sum().backward()
        return clip_grad_norm(block.parameters(), 0.1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = step()
    held = [p.grad for p in block.parameters()]
    for seed in (5, 6):
        features.copy_(torch.randn(features.shape, generator=torch.Generator("cuda").manual_seed(seed),
                                   device="cuda"))
        graph.replay()
        got = [g.clone() for g in held]
        got_norm = norm.clone()
        want_norm = step()
        assert torch.equal(got_norm, want_norm)
        for g, p in zip(got, block.parameters()):
            assert torch.equal(g, p.grad)
        for p, g in zip(block.parameters(), held):
            p.grad = g
    assert len(splats.mean) == 200


def test_eight_bit_products():
    refiner, splats = made(left=64, right=64), scene(600, 6)
    with torch.no_grad():
        full = refiner([splats])[0]
        refiner.quantize()
        small = refiner([splats])[0]
    change = torch.cat([(full[n] - getattr(splats, n)).flatten() for n in full])
    error = torch.cat([(full[n] - small[n]).flatten() for n in full])
    # two roundings of 2**-4 at most in each of six products
    assert 0 < error.norm() < 0.3 * change.norm()


def one_of(splats, at, batch):
    return GaussianSplat.from_tensors(*(getattr(splats, n)[at:at + 1].detach().expand(
        batch, *getattr(splats, n).shape[1:]).contiguous() for n in NAMES))


def test_streams_with_four_bit_caches(monkeypatch):
    """Streams against 4-bit caches, and the same with the step from its definition."""
    from gaussian_splats_b200 import refine

    refiner, splats = made(left=16, right=0, first=3), scene(60, 5, dead=20)
    oracles = {}

    def defined(q, k, v, cache, positions, *, first, valid, cache_valid):
        ref = oracles.setdefault(cache.k_codes.data_ptr(), R.Streams(
            len(q), cache.k_codes.shape[2], first, k.shape[1], k.shape[2], k.dtype, "cuda"))
        valid = torch.ones(len(q), dtype=torch.bool) if valid is None else valid
        out = ref.step(q, k, v, positions, k.shape[2] ** -0.5, valid)[0]
        cache_valid.copy_(ref.seen)
        return out.to(q.dtype)

    with torch.no_grad():
        order = morton_order(splats.mean).tolist()
        state, plain, want = (refiner.stream(2, four_bit=True), refiner.stream(2), None)
        with monkeypatch.context() as m:
            m.setattr(refine, "window_attention_step_4bit", defined)
            want = refiner.stream(2, four_bit=True)
        for at in order:
            one = one_of(splats, at, 2)
            out = refiner.step(one, state)
            with monkeypatch.context() as m:
                m.setattr(refine, "window_attention_step_4bit", defined)
                reference = refiner.step(one, want)
            close = refiner.step(one, plain)
            for name in NAMES:
                assert torch.equal(out[name][0], out[name][1])
                # a unit of bfloat16 here and there, and codes that it moves by a step
                torch.testing.assert_close(out[name], reference[name], rtol=0, atol=0.1)
                torch.testing.assert_close(out[name], close[name], rtol=0, atol=0.5)
        assert torch.equal(state["alive"], want["alive"])
    held = sum(t.numel() * t.element_size() for cache, _ in state["blocks"] for t in cache)
    whole = sum(t.numel() * t.element_size() for cache, _ in plain["blocks"] for t in cache)
    assert held < 0.29 * whole


def test_quantized_refiner_keeps_its_feed_forward(monkeypatch):
    """8-bit products are those of the attention then: both ways of the feed-forward layer
    run through the linear layer, whatever its size, as before."""
    from gaussian_splats_b200 import refine

    for hidden in (512, 40):
        refiner, splats, calls = made(hidden=hidden), scene(100, 6), []
        refiner.quantize()

        def recorded(x, *args, **more):
            calls.append(more.get("activation"))
            return plain_linear(x, *args, **more)

        with torch.no_grad(), monkeypatch.context() as m:
            m.setattr(refine, "linear", recorded)
            out = refiner([splats])[0]
        assert calls == ["gelu", None] * len(refiner.blocks)
        assert all(t.isfinite().all() for t in out.values())
        assert all(block.qkv.codes is not None for block in refiner.blocks)
