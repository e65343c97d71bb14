"""Host side of the linear layer, gradient clipping and the 4-bit step: refusals, argument
checks, and the oracle's own gradients and codes. No GPU."""

import ctypes

import pytest
import torch

import operator_reference as R


def test_no_cpu_path():
    from gaussian_splats_b200.attention import window_attention_step_4bit, window_cache_4bit
    from gaussian_splats_b200.linear import linear
    from gaussian_splats_b200.optim import clip_grad_norm, grad_norm

    t = torch.zeros(8, 8, dtype=torch.bfloat16)
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    h = torch.zeros(4, 1, 8, dtype=torch.bfloat16)
    cache = window_cache_4bit(4, 3, 0, 1, 8, device="cpu")
    for call in (lambda: linear(t, t), lambda: grad_norm([p.grad]),
                 lambda: clip_grad_norm([p], 1.0),
                 lambda: window_attention_step_4bit(h, h, h, cache,
                                                    torch.zeros(4, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="CUDA devices only"):
            call()
    with pytest.raises(ValueError):
        window_cache_4bit(1, -1, 0, 1, 8, device="cpu")
    with pytest.raises(ValueError):
        window_cache_4bit(1, 3, 0, 1, 12, device="cpu")


def test_linear_checks_arguments():
    """Bad arguments come back as statuses before anything touches a device."""
    from gaussian_splats_b200 import native

    lib, a = native.lib(), 256  # an address that passes the alignment checks, never read
    good = dict(rows=300, inputs=64, outputs=72, dtype=1, bias_dtype=0, residual_dtype=0,
                activation=2, x=a, weight=a, bias=a, residual=a, x_stride=64, weight_stride=64,
                residual_stride=72, y=a, slope=a, grad_y=a, grad_x=a, grad_weight=a, grad_bias=a,
                workspace=a, workspace_size=1 << 40)
    for status, bad in [(-1, dict(rows=-1)), (-1, dict(rows=2 ** 31)), (-1, dict(inputs=0)),
                        (-1, dict(outputs=65537)), (-1, dict(activation=4)), (-4, dict(dtype=0)),
                        (-1, dict(bias_dtype=2)), (-1, dict(residual_dtype=2)), (-1, dict(x=None)),
                        (-1, dict(weight=None)), (-1, dict(x_stride=-1)), (-5, dict(x=a + 1)),
                        (-1, dict(weight_stride=56)), (-5, dict(weight_stride=68))]:
        args = native.LinearArgs(**{**good, **bad})
        assert lib.gs_linear(ctypes.byref(args), None) == status, bad
        assert lib.gs_linear_backward(ctypes.byref(args), None) == status, bad
    for status, bad in ((-1, dict(y=None)), (-5, dict(y=a + 2)), (-5, dict(residual=a + 2)),
                        (-5, dict(bias=a + 2)), (-5, dict(slope=a + 8)),
                        (-5, dict(y=a + 1, residual_dtype=1)), (-5, dict(bias=a + 1, bias_dtype=1))):
        args = native.LinearArgs(**{**good, **bad})
        assert lib.gs_linear(ctypes.byref(args), None) == status, bad
    for status, bad in ((-1, dict(grad_y=None)), (-1, dict(slope=None)), (-1, dict(workspace=None)),
                        (-3, dict(workspace_size=0)), (-5, dict(x=a + 8)), (-5, dict(x_stride=60)),
                        (-5, dict(grad_x=a + 1)), (-5, dict(grad_weight=a + 4)),
                        (-5, dict(grad_bias=a + 2)), (-5, dict(workspace=a + 128))):
        args = native.LinearArgs(**{**good, **bad})
        assert lib.gs_linear_backward(ctypes.byref(args), None) == status, bad
    assert lib.gs_linear(None, None) == -1 and lib.gs_linear_backward(None, None) == -1
    assert lib.gs_linear_workspace_size(None) == 0
    args = native.LinearArgs(**{**good, "rows": 0})
    assert lib.gs_linear_workspace_size(ctypes.byref(args)) == 0
    assert lib.gs_linear(ctypes.byref(args), None) == 0
    args = native.LinearArgs(**{**good, "rows": 2 ** 31 - 512, "inputs": 65536, "outputs": 65536,
                                "x_stride": 65536, "weight_stride": 65536})
    assert lib.gs_linear_workspace_size(ctypes.byref(args)) > 2 ** 47


def test_align_rows_checks_arguments():
    from gaussian_splats_b200 import native

    lib, a = native.lib(), 256
    for status, bad in [(-1, (-1, 8, a, 8, a)), (-1, (4, 0, a, 8, a)), (-1, (4, 8, a, -8, a)),
                        (-1, (4, 8, None, 8, a)), (-1, (4, 65537, a, 8, a)), (-5, (4, 8, a + 1, 8, a)),
                        (-5, (4, 8, a, 8, a + 8)), (0, (0, 8, a, 8, a))]:
        assert lib.gs_align_rows(*bad, None) == status, bad


def test_clip_checks_arguments():
    from gaussian_splats_b200 import native

    lib, a, inf = native.lib(), 256, float("inf")

    def call(tensors=1, max_norm=1.0, result=a, workspace=a, size=1 << 30, **entry):
        entry = native.Gradient(**{**dict(data=a, count=10, dtype=0), **entry})
        return lib.gs_clip_grad_norm(tensors, ctypes.byref(entry), max_norm, 1, result, workspace,
                                     size, None)

    for status, bad in [(-1, dict(tensors=0)), (-1, dict(tensors=2 ** 20 + 1)),
                        (-1, dict(max_norm=-1.0)), (-1, dict(max_norm=inf - inf)),
                        (-1, dict(result=None)), (-1, dict(workspace=None)), (-3, dict(size=8)),
                        (-1, dict(count=-1)), (-1, dict(data=None)), (-1, dict(dtype=3)),
                        (-5, dict(data=a + 2)), (-5, dict(workspace=a + 4))]:
        assert call(**bad) == status, bad
    assert lib.gs_clip_grad_norm(1, None, 1.0, 1, a, a, 1 << 30, None) == -1
    assert lib.gs_clip_grad_norm_workspace_size(0) == 0
    assert lib.gs_clip_grad_norm_workspace_size(5000) > lib.gs_clip_grad_norm_workspace_size(5) > 0


def test_copied_optimizer_has_a_norm():
    import copy
    import pickle

    from gaussian_splats_b200.optim import GROUP_NAMES, FusedAdam

    shapes = [(4, 3), (4, 4), (4, 3), (4, 1), (4, 1, 3)]
    opt = FusedAdam([{"params": [torch.nn.Parameter(torch.zeros(*shape))], "name": name}
                     for shape, name in zip(shapes, GROUP_NAMES)])
    assert opt.grad_norm is None
    assert copy.deepcopy(opt).grad_norm is None and pickle.loads(pickle.dumps(opt)).grad_norm is None


def test_4bit_step_checks_arguments():
    from gaussian_splats_b200 import native

    lib, a = native.lib(), 256
    good = dict(batch=2, heads=4, kv_heads=2, dim=64, dtype=1, slots=10, first=2, scale=0.1, q=a,
                k=a, v=a, q_stride=64, q_head_stride=64, k_stride=64, k_head_stride=64,
                v_stride=64, v_head_stride=64, k_codes=a, v_codes=a, k_range=a, v_range=a,
                positions=a, out=a, workspace=a, workspace_size=1 << 40)
    for status, bad in [(-1, dict(heads=3)), (-1, dict(dim=12)), (-4, dict(dim=136)),
                        (-4, dict(dtype=0)), (-1, dict(batch=-1)), (-1, dict(first=10)),
                        (-1, dict(slots=0)), (-1, dict(batch=2 ** 30)),
                        (-1, dict(scale=float("nan"))), (-1, dict(k_codes=None)),
                        (-1, dict(v_range=None)), (-1, dict(valid=a)), (-5, dict(k=a + 2)),
                        (-5, dict(v_stride=4)), (-5, dict(v_codes=a + 4)),
                        (-1, dict(workspace=None)), (-3, dict(workspace_size=16))]:
        args = native.WindowAttentionStep4BitArgs(**{**good, **bad})
        assert lib.gs_window_attention_step_4bit(ctypes.byref(args), None) == status, bad
    assert lib.gs_window_attention_step_4bit(None, None) == -1


@pytest.mark.parametrize("activation", [None, "relu", "gelu", "silu"])
def test_oracle_gradients(activation):
    """The linear layer's gradients against differences of its values."""
    g = torch.Generator().manual_seed(0)
    rand = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    x, w, b, up = rand(5, 7), rand(4, 7), rand(4), rand(5, 4)
    grads = R.linear(x, w, b, None, activation, up)
    for name, t in (("dx", x), ("dweight", w), ("dbias", b)):
        way, h = rand(*t.shape), 1e-6
        ends = []
        for sign in (1, -1):
            moved = {"dx": x, "dweight": w, "dbias": b}
            moved[name] = t + sign * h * way
            ends.append((R.linear(*moved.values(), None, activation)["y"] * up).sum())
        want = (grads[name] * way).sum()
        assert abs((ends[0] - ends[1]) / (2 * h) - want) < 1e-7 * (1 + abs(want))


def test_oracle_codes():
    """A row's codes are the nearest of its sixteen values, ties to the even code."""
    g = torch.Generator().manual_seed(1)
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.randn(200, 24, generator=g).to(dtype)
        code, step, middle = R.held(x)
        steps = (torch.arange(16) - 7.5) * step.double()[:, None, None] + \
            middle.double()[:, None, None]
        distance = (x.double()[..., None] - steps).abs()
        best = distance.amin(-1)
        assert torch.equal(distance.gather(-1, code.long()[..., None])[..., 0], best)
        ties = (distance == best[..., None]).sum(-1) > 1
        assert (code[ties] % 2 == 0).all()
        both = R.packed(code)
        assert torch.equal(both & 15, code[:, 0::2]) and torch.equal(both >> 4, code[:, 1::2])
    code, step, middle = R.held(torch.tensor([[0.0, 1.0, 15.0, 0.5, 2.5, 7.5]]).half())
    assert step.item() == 1.0 and middle.item() == 7.5
    assert code.tolist() == [[0, 1, 15, 0, 2, 8]]
    assert R.held(torch.full((1, 4), 3.0).half())[0].tolist() == [[8] * 4]


def test_linear_workspace_holds_what_is_used():
    """The gradient of the sums where a product reads it from there, and the splits' sums
    where there are several."""
    from gaussian_splats_b200 import native

    def size(rows, inputs, outputs, wanted="xwb", **more):
        a = 256
        args = native.LinearArgs(**{**dict(
            rows=rows, inputs=inputs, outputs=outputs, dtype=1, bias_dtype=1, residual_dtype=1,
            activation=2, x=a, weight=a, x_stride=inputs, weight_stride=inputs,
            grad_x=a if "x" in wanted else None, grad_weight=a if "w" in wanted else None,
            grad_bias=a if "b" in wanted else None), **more})
        return native.lib().gs_linear_workspace_size(ctypes.byref(args))

    dz, strips = 1000 * 8192 * 2, 1000 * 8192 * 4 // 4  # four rows a strip at least
    assert dz < size(1000, 8192, 8192) <= dz + strips + 1024
    assert size(1000, 65536, 65536) < 2 ** 30
    assert size(1000, 8192, 8192, "b") <= strips + 1024
    assert size(1000, 8192, 8192, "") == size(1000, 8192, 8192) == size(1000, 8192, 8192, "x")
    assert size(1000, 8192, 8192, activation=0) <= strips + 1024  # grad_y is read in its place
    assert size(100000, 256, 256, "w", activation=0) >= 18 * 256 * 256 * 4


def test_operands_are_copied_once(monkeypatch):
    """A transposed operand by torch, where that makes it whole 16-byte words, and by the
    kernel that aligns rows only where it does not."""
    from gaussian_splats_b200 import linear as L

    calls = []
    monkeypatch.setattr(L, "call", lambda name, *args: calls.append(name))
    t = torch.zeros(64, 48, dtype=torch.bfloat16)
    assert L._operand(t) is t and L._operand(t[:, 8:24]).data_ptr() == t[:, 8:].data_ptr()
    turned = L._operand(t.t())
    assert calls == [] and turned.shape == (48, 64) and turned.is_contiguous()
    for other in (t[:, 1:9], t.view(-1)[:45].view(9, 5), t[:5].t(), t[:1].expand(9, 48)):
        assert L._operand(other).shape == other.shape
        assert calls.pop() == "gs_align_rows" and calls == []


def test_refiner_saved_before_it_had_feed_forward_layers():
    """A whole module, saved by a version whose blocks and shapes knew of none."""
    import pickle

    from gaussian_splats_b200.refine import RefinerShape, SplatRefiner

    refiner = SplatRefiner(shape=RefinerShape(width=64, heads=2, kv_heads=1), device="cpu")
    for block in refiner.blocks:
        del block.feed
    del refiner.shape.__dict__["hidden"]
    loaded = pickle.loads(pickle.dumps(refiner))
    assert loaded.shape.hidden == 0 and all(block.feed is None for block in loaded.blocks)
    x = torch.zeros(3, 64)
    assert loaded.blocks[0]._fed(x, (x,)) is x
    loaded.quantize()
