"""The splat refiner: the sequence operators together, up to the rendered image."""

import pytest
import torch

from gaussian_splats_b200.refine import RefinerShape, SplatRefiner
from gaussian_splats_b200.splats import GaussianSplat

pytestmark = pytest.mark.gpu


def scene(points, seed, dead=0):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    opacity = rand(points, 1)
    opacity[:dead] = -9.0
    return GaussianSplat.from_tensors(*(t.cuda() for t in (
        rand(points, 3), rand(points, 4), 0.3 * rand(points, 3) - 3.0, opacity,
        0.5 * rand(points, 1, 3))))


def shaken(refiner):
    """The refiner with an output layer that does something."""
    with torch.no_grad():
        torch.nn.init.normal_(refiner.head.weight, std=2.5,
                              generator=torch.Generator("cuda").manual_seed(1))
    return refiner


def test_untrained_refiner_changes_nothing():
    splats = scene(500, 0)
    out = SplatRefiner()([splats])[0]
    for name, t in out.items():
        assert torch.equal(t, getattr(splats, name)), name


def test_a_batch_gives_what_its_scenes_give():
    torch.manual_seed(0)
    refiner = shaken(SplatRefiner(shape=RefinerShape(width=128, heads=2, kv_heads=1, left=40,
                                                     right=20)))
    scenes = [scene(300, 1, dead=30), scene(1, 2), scene(777, 3)]
    together = refiner(scenes)
    for splats, out in zip(scenes, together):
        alone = refiner([splats])[0]
        for name in alone:  # bfloat16 products of other sizes may add in another order
            torch.testing.assert_close(out[name], alone[name], rtol=0, atol=2e-2)


def test_dead_splats_do_not_reach_the_others():
    torch.manual_seed(0)
    refiner = shaken(SplatRefiner(shape=RefinerShape(width=128, heads=2, kv_heads=1, blocks=1,
                                                     left=40, right=20)))
    # attention only: with the gates shut the recurrence passes nothing on
    splats = scene(400, 4, dead=50)
    packed_grad = torch.autograd.grad(refiner([splats])[0]["mean"][50:].square().sum(),
                                      refiner.embed.weight)[0]
    assert torch.isfinite(packed_grad).all()


def test_training_through_the_rasterizer():
    """A refiner learns to undo a shift of a scene's colours and opacities from a
    rendered view: a few steps of the whole path."""
    from gaussian_splats_b200 import scenes as S
    from gaussian_splats_b200.losses import l1_loss
    from gaussian_splats_b200.rasterize import rasterize

    torch.manual_seed(0)
    s = S.config1(num_points=2000, image=128)
    camera = s.cameras[0]
    true = GaussianSplat.from_tensors(*(t.cuda() for t in s.tensors()))
    with torch.no_grad():
        target = rasterize(true, camera, tile_size=16)
        given = GaussianSplat.from_tensors(*(t.cuda().clone() for t in s.tensors()))
        given.color += 0.3
        given.opacity -= 1.0
    refiner = SplatRefiner(shape=RefinerShape(width=128, heads=2, kv_heads=1, left=64, right=64))
    optimizer = torch.optim.Adam(refiner.parameters(), lr=1e-2)
    losses = []
    for _ in range(40):
        out = refiner([given])[0]
        image = rasterize(GaussianLike(out), camera, tile_size=16)
        loss = l1_loss(image, target)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    assert all(torch.isfinite(p.grad).all() for p in refiner.parameters())
    assert losses[-1] < 0.6 * losses[0], losses


class GaussianLike:
    """The refined tensors as the rasterizer takes splats (no parameters of their own)."""

    def __init__(self, tensors):
        self.__dict__.update(tensors)
        self.normals = torch.zeros_like(self.mean)


def test_stream_follows_the_whole_scene():
    torch.manual_seed(0)
    shape = RefinerShape(width=128, heads=2, kv_heads=1, left=16, right=0, first=3)
    refiner = shaken(SplatRefiner(shape=shape))
    from gaussian_splats_b200.refine import morton_order

    splats = scene(90, 5)
    with torch.no_grad():
        whole = refiner([splats])[0]
        state = refiner.stream(2)
        for at in morton_order(splats.mean).tolist():
            one = GaussianSplat.from_tensors(*(getattr(splats, n)[at:at + 1].detach().expand(
                2, *getattr(splats, n).shape[1:]).contiguous()
                for n in ("mean", "rotation", "scale", "opacity", "color")))
            out = refiner.step(one, state)
            for name in whole:
                torch.testing.assert_close(out[name][0], whole[name][at], rtol=0, atol=3e-2)
                assert torch.equal(out[name][0], out[name][1])


def test_eight_bit_products():
    torch.manual_seed(0)
    refiner = shaken(SplatRefiner(shape=RefinerShape(width=128, heads=2, kv_heads=1, left=64,
                                                     right=64)))
    splats = scene(600, 6)
    with torch.no_grad():
        full = refiner([splats])[0]
        refiner.quantize()
        small = refiner([splats])[0]
    change = torch.cat([(full[n] - getattr(splats, n)).flatten() for n in full])
    error = torch.cat([(full[n] - small[n]).flatten() for n in full])
    # two roundings of 2**-4 at most in each of four products
    assert 0 < error.norm() < 0.25 * change.norm()


def test_refusals():
    with pytest.raises(ValueError, match="do not divide"):
        SplatRefiner(shape=RefinerShape(width=100, heads=3))
    with pytest.raises(ValueError, match="cannot take splats"):
        SplatRefiner(sh_degree=1)([scene(10, 0)])
    with pytest.raises(ValueError, match="causal"):
        SplatRefiner().stream(1)


def test_stream_follows_a_scene_with_dead_splats():
    """A causal refiner is one model: dead splats are no keys in either form."""
    from gaussian_splats_b200.refine import morton_order

    torch.manual_seed(0)
    shape = RefinerShape(width=128, heads=2, kv_heads=1, left=16, right=0, first=3)
    refiner = shaken(SplatRefiner(shape=shape))
    splats = scene(90, 5, dead=40)
    with torch.no_grad():
        splats.mean[:40] *= 30  # far out: keys that would be seen, were they seen
        whole = refiner([splats])[0]
        state = refiner.stream(2)
        for at in morton_order(splats.mean).tolist():
            one = GaussianSplat.from_tensors(*(getattr(splats, n)[at:at + 1].detach().expand(
                2, *getattr(splats, n).shape[1:]).contiguous()
                for n in ("mean", "rotation", "scale", "opacity", "color")))
            out = refiner.step(one, state)
            for name in whole:
                torch.testing.assert_close(out[name][0], whole[name][at], rtol=0, atol=3e-2)


def test_dead_splats_are_no_keys(monkeypatch):
    """With a recurrence that passes nothing on, what dead splats hold is seen by
    themselves alone; what live ones hold is seen by others."""
    from gaussian_splats_b200 import refine

    monkeypatch.setattr(refine, "gated_scan", lambda x, gate, packed: (torch.zeros_like(x), None))
    torch.manual_seed(0)
    refiner = shaken(SplatRefiner(shape=RefinerShape(width=128, heads=2, kv_heads=1, left=40,
                                                     right=20)))
    splats, changes = scene(400, 4, dead=50), scene(400, 7)

    def refined(rows):
        """The live splats' results with the rows' parameters replaced, order and
        opacity kept."""
        with torch.no_grad():
            tensors = {n: getattr(splats, n).detach().clone()
                       for n in ("mean", "rotation", "scale", "opacity", "color")}
            for n in ("rotation", "scale", "color"):
                tensors[n][rows] = 5 * getattr(changes, n)[rows]
            out = refiner([GaussianSplat.from_tensors(*tensors.values())])[0]
        return torch.cat([out[n][100:].flatten(1) for n in out], 1)

    plain = refined(slice(0, 0))
    assert torch.equal(refined(slice(0, 50)), plain)          # dead ones
    assert not torch.equal(refined(slice(50, 100)), plain)    # live ones
    attention = refine.window_attention
    monkeypatch.setattr(refine, "window_attention",
                        lambda *a, valid, **k: attention(*a, valid=None, **k))
    assert not torch.equal(refined(slice(0, 50)), refined(slice(0, 0)))  # were they keys
