"""Host side of the sequence operators: layouts, refusals, argument checks, and
the oracle's own gradients. No GPU."""

import ctypes

import pytest
import torch

import sequence_reference as R
from gaussian_splats_b200.sequences import PackedSequences


def test_packed_sequences_tables():
    p = PackedSequences([0, 128, 300, 0, 1], device="cpu")
    assert p.total == 429 and len(p) == 5 and p.num_tiles == 5
    assert p.offsets.tolist() == [0, 0, 128, 428, 428, 429]
    assert p.tile_starts.tolist() == [0, 0, 1, 4, 4, 5]
    assert p.tiles.tolist() == [[0, 128, 0, 1], [128, 428, 128, 2], [128, 428, 256, 2],
                                [128, 428, 384, 2], [428, 429, 428, 4]]
    assert p.tiles.dtype == torch.int32 and p.tiles.is_contiguous()
    assert PackedSequences([0], device="cpu").tiles.shape == (0, 4)


@pytest.mark.parametrize("lengths", [[], [3, -1], [2 ** 30, 2 ** 30]])
def test_packed_sequences_refuses(lengths):
    with pytest.raises(ValueError):
        PackedSequences(lengths, device="cpu")


def test_no_cpu_path():
    from gaussian_splats_b200.attention import window_attention, window_attention_step
    from gaussian_splats_b200.norm import rms_norm, rms_norm_e4m3
    from gaussian_splats_b200.recurrence import gated_scan, gated_scan_step

    t, h = torch.zeros(4, 8), torch.zeros(4, 1, 8, dtype=torch.bfloat16)
    for call in (lambda: window_attention(h, h, h, left=1),
                 lambda: window_attention_step(h, h, h, h[:, None], h[:, None],
                                               torch.zeros(4, dtype=torch.int64)),
                 lambda: gated_scan(t, t), lambda: gated_scan_step(t, t, t),
                 lambda: rms_norm(t, t[0]), lambda: rms_norm_e4m3(t, t[0])):
        with pytest.raises(RuntimeError, match="CUDA devices only"):
            call()


def test_library_checks_arguments():
    """Bad arguments come back as statuses before anything touches a device."""
    from gaussian_splats_b200 import native

    lib, a = native.lib(), 256  # an address that passes the alignment checks, never read
    good = dict(tokens=300, num_tiles=3, heads=4, kv_heads=2, dim=64, dtype=1, left=3, right=0,
                first=2, scale=0.1, q=a, k=a, v=a, q_stride=64, q_head_stride=64, k_stride=64,
                k_head_stride=64, v_stride=64, v_head_stride=64, out=a)
    for status, bad in [(-1, dict(heads=3)), (-1, dict(dim=12)), (-4, dict(dim=136)),
                        (-4, dict(dtype=0)), (-1, dict(left=-1)), (-1, dict(first=129)),
                        (-1, dict(scale=float("nan"))), (-1, dict(num_tiles=2)),
                        (-1, dict(q=None)), (-5, dict(k=a + 2)), (-5, dict(v_stride=4)),
                        (-5, dict(tiles=a + 4)), (-1, dict(tokens=-1))]:
        args = native.WindowAttentionArgs(**{**good, **bad})
        assert lib.gs_window_attention(ctypes.byref(args), None) == status, bad
    args = native.WindowAttentionArgs(**good)
    assert lib.gs_window_attention_backward(ctypes.byref(args), None) == -1  # no gradients
    assert lib.gs_window_attention_workspace_size(ctypes.byref(args)) >= 4 * 4 * 300
    step = dict(batch=1, heads=4, kv_heads=2, dim=64, dtype=1, slots=9, first=2, scale=0.1, q=a,
                k=a, v=a, q_stride=64, q_head_stride=64, k_stride=64, k_head_stride=64,
                v_stride=64, v_head_stride=64, cache_k=a, cache_v=a, positions=a, out=a)
    for status, bad in [(-1, dict(slots=2)), (-1, dict(positions=None)), (-5, dict(cache_v=a + 8)),
                        (-1, dict(batch=-1)), (-4, dict(dtype=0))]:
        args = native.WindowAttentionStepArgs(**{**step, **bad})
        assert lib.gs_window_attention_step(ctypes.byref(args), None) == status, bad
    scan = dict(tokens=300, sequences=1, num_tiles=3, channels=8, dtype=0, x=a, gate=a, x_stride=8,
                gate_stride=8, y=a, last=a, entering=a, workspace=a, workspace_size=1 << 20)
    for status, bad in [(-1, dict(channels=0)), (-1, dict(num_tiles=4)), (-1, dict(sequences=2)),
                        (-3, dict(workspace_size=8)), (-1, dict(x=None)), (-1, dict(dtype=5)),
                        (-1, dict(tiles=a)), (-1, dict(last=None))]:
        args = native.GatedScanArgs(**{**scan, **bad})
        assert lib.gs_gated_scan(ctypes.byref(args), None) == status, bad
    assert lib.gs_gated_scan_step(-1, 8, 0, a, 8, a, 8, a, a, None) == -1
    assert lib.gs_gated_scan_step(1, 8, 7, a, 8, a, 8, a, a, None) == -1
    norm = dict(rows=4, channels=8, dtype=1, residual_dtype=0, weight_dtype=1, eps=1e-6, x=a,
                weight=a, x_stride=8, y=a)
    for status, bad in [(-1, dict(channels=0)), (-1, dict(channels=16385)), (-1, dict(y=None)),
                        (-1, dict(weight=None)), (-4, dict(residual_dtype=2)),
                        (-1, dict(q=a)), (-1, dict(weight_dtype=3))]:
        args = native.RmsNormArgs(**{**norm, **bad})
        assert lib.gs_rms_norm(ctypes.byref(args), None) == status, bad
    args = native.RmsNormArgs(**norm, sum=a, sum_stride=8, grad_y=a, grad_x=a, grad_weight=a,
                              workspace=a)
    assert lib.gs_rms_norm_backward(ctypes.byref(args), None) == -3  # workspace too small
    for entry in (lib.gs_window_attention, lib.gs_gated_scan, lib.gs_rms_norm):
        assert entry(None, None) == -1


def _difference(f, t, grad, step=1e-5):
    d = torch.randn_like(t)
    return (f(t + step * d) - f(t - step * d)) / (2 * step), (grad * d).sum()


def test_the_oracles_gradients_against_differences():
    torch.manual_seed(0)
    lengths = [9, 0, 14]
    t = dict(q=torch.randn(23, 4, 8), k=torch.randn(23, 2, 8), v=torch.randn(23, 2, 8))
    t = {n: x.double() for n, x in t.items()}
    grad, valid = torch.randn(23, 4, 8).double(), torch.rand(23) > 0.3
    window = dict(left=3, right=1, first=2, valid=valid)
    ref = R.attention(**t, lengths=lengths, grad=grad, **window)
    for name in t:
        f = lambda x: (R.attention(**{**t, name: x}, lengths=lengths, **window)["out"] *  # noqa
                       grad).sum()
        torch.testing.assert_close(*_difference(f, t[name], ref["d" + name]), rtol=1e-6, atol=1e-8)
    s = dict(x=torch.randn(23, 5), gate=torch.randn(23, 5), initial=torch.randn(3, 5))
    s = {n: x.double() for n, x in s.items()}
    g, gl = torch.randn(23, 5).double(), torch.randn(3, 5).double()

    def total(r):
        return (r["y"] * g).sum() + (r["last"] * gl).sum()

    ref = R.gated_scan(**s, lengths=lengths, grad=g, grad_last=gl)
    for name in s:
        f = lambda x: total(R.gated_scan(**{**s, name: x}, lengths=lengths))  # noqa: E731
        torch.testing.assert_close(*_difference(f, s[name], ref["d" + name]), rtol=1e-6, atol=1e-8)
    x, w = torch.randn(6, 9).double(), torch.randn(9).double()
    ref = R.rms_norm(x, w, eps=1e-3, grad=(gy := torch.randn(6, 9).double()))
    f = lambda x, w: (R.rms_norm(x, w, eps=1e-3)["y"] * gy).sum()  # noqa: E731
    torch.testing.assert_close(*_difference(lambda u: f(u, w), x, ref["dz"]), rtol=1e-6, atol=1e-8)
    torch.testing.assert_close(*_difference(lambda u: f(x, u), w, ref["dw"]), rtol=1e-6, atol=1e-8)


@pytest.mark.parametrize("plant", ["window", "first", "scale", "group"])
def test_the_oracle_tells_wrong_windows_apart(plant):
    """A planted mistake moves the oracle's result by far more than any bound."""
    torch.manual_seed(1)
    q, k, v = torch.randn(40, 4, 8), torch.randn(40, 2, 8), torch.randn(40, 2, 8)
    right = R.attention(q, k, v, [25, 15], left=4, right=2, first=2)["out"]
    wrong = {"window": dict(left=5, right=2, first=2), "first": dict(left=4, right=2, first=1),
             "scale": dict(left=4, right=2, first=2, scale=0.3),
             "group": dict(left=4, right=2, first=2)}[plant]
    if plant == "group":
        k, v = k.flip(1), v.flip(1)
    assert (R.attention(q, k, v, [25, 15], **wrong)["out"] - right).abs().max() > 0.05


def test_morton_order():
    from gaussian_splats_b200.refine import morton_order

    corners = torch.tensor([[x, y, z] for z in (0.0, 1.0) for y in (0.0, 1.0) for x in (0.0, 1.0)])
    shuffled = torch.randperm(8, generator=torch.Generator().manual_seed(0))
    assert torch.equal(shuffled[morton_order(corners[shuffled])], torch.arange(8))
    points = torch.rand(4000, 3, generator=torch.Generator().manual_seed(1))
    order = morton_order(points)
    assert torch.equal(order.sort().values, torch.arange(4000))
    # neighbours along the order are near: far nearer than random pairs (0.66 apart)
    assert (points[order][1:] - points[order][:-1]).norm(dim=1).mean() < 0.12
    assert torch.equal(morton_order(torch.ones(5, 3)), torch.arange(5))  # ties by index
    assert morton_order(torch.empty(0, 3)).shape == (0,)
    with pytest.raises(ValueError):
        morton_order(torch.zeros(3, 2))


def _backward_calls(monkeypatch, build, hooks):
    """The arguments that a backward passes to the library, and the tensors that the
    hooks gave it; the library itself is not called."""
    from gaussian_splats_b200 import attention, norm, recurrence

    seen, unpacked = {}, []

    def record(name, device, args):
        if name.endswith("backward"):
            seen["args"] = type(args._obj).from_buffer_copy(args._obj)

    for module in (attention, norm, recurrence):
        monkeypatch.setattr(module, "call", record)

    def unpack(t):
        unpacked.append(hooks[1](t))
        return unpacked[-1]

    with torch.autograd.graph.saved_tensors_hooks(hooks[0], unpack):
        outputs, inputs = build()
    torch.autograd.grad(outputs, inputs, [torch.ones_like(t) for t in outputs])
    return seen["args"], {t.data_ptr(): t for t in unpacked}


@pytest.mark.parametrize("packed", ["as it is", "contiguous", "wider"])
@pytest.mark.parametrize("operator", ["attention", "scan", "norm"])
def test_backward_goes_by_the_tensors_it_gets(monkeypatch, operator, packed):
    """Saved-tensor hooks may hand back other strides than the forward's."""
    wide = torch.randn(40, 4 * 64)
    half = wide.to(torch.bfloat16)

    def build():
        from gaussian_splats_b200 import attention, norm, recurrence

        if operator == "attention":
            leaves = [half[:, s].unflatten(1, (-1, 64)).detach().requires_grad_()
                      for s in (slice(0, 128), slice(128, 192), slice(192, 256))]
            return [attention._WindowAttention.apply(*leaves, None, 3, 0, 0, None, 0.1, 1, True)], leaves
        leaves = [wide[:, s].detach().requires_grad_() for s in (slice(0, 128), slice(128, 256))]
        if operator == "scan":
            return [recurrence._GatedScan.apply(*leaves, None, None, 0)[0]], leaves
        weight = torch.ones(128, requires_grad=True)
        return [norm._RmsNorm.apply(leaves[0], weight, None, 1e-6)], [leaves[0], weight]

    def wider(t):
        if t.dim() != 2 and t.dim() != 3:
            return t.detach().clone()
        return torch.cat((t, t, t), -1)[..., :t.shape[-1]].detach()

    pack = {"as it is": lambda t: t.detach(), "contiguous": lambda t: t.detach().clone(
        memory_format=torch.contiguous_format), "wider": wider}[packed]
    args, tensors = _backward_calls(monkeypatch, build, (pack, lambda t: t))
    fields = {"attention": ("q", "k", "v"), "scan": ("x", "gate"), "norm": ("sum",)}[operator]
    for name in fields:
        t = tensors[getattr(args, name)]
        assert getattr(args, name + "_stride") == t.stride(0), name
        if operator == "attention":
            assert getattr(args, name + "_head_stride") == t.stride(1), name
    for name in {"attention": ("out", "lse"), "scan": ("entering",), "norm": ("weight",)}[operator]:
        t = tensors.get(getattr(args, name))  # or a contiguous copy of it
        assert t is None or t.is_contiguous(), name


def test_library_refuses_half_a_layout():
    """A table of tiles without the sequences' first tiles, first tiles without a
    table, or no sequences: never walked."""
    from gaussian_splats_b200 import native

    lib, a = native.lib(), 256
    attention = dict(tokens=300, num_tiles=3, heads=4, kv_heads=2, dim=64, dtype=1, left=3, first=2,
                     scale=0.1, q=a, k=a, v=a, q_stride=64, q_head_stride=64, k_stride=64,
                     k_head_stride=64, v_stride=64, v_head_stride=64, out=a, lse=a, grad_out=a,
                     grad_q=a, grad_k=a, grad_v=a, workspace=a, workspace_size=1 << 40)
    scan = dict(tokens=300, num_tiles=3, channels=8, x=a, gate=a, x_stride=8, gate_stride=8, y=a,
                last=a, entering=a, grad_y=a, grad_x=a, grad_gate=a, workspace=a,
                workspace_size=1 << 40)
    for layout in (dict(tile_starts=a, sequences=2), dict(tiles=a, sequences=2),
                   dict(tiles=a, tile_starts=a, sequences=0),
                   dict(tiles=a, tile_starts=a, sequences=-3),
                   dict(tiles=a, tile_starts=a, sequences=2 ** 62),
                   dict(tiles=a, tile_starts=a, sequences=2, num_tiles=2 ** 61)):
        args = native.WindowAttentionArgs(**{**attention, **layout})
        assert lib.gs_window_attention(ctypes.byref(args), None) == -1, layout
        assert lib.gs_window_attention_backward(ctypes.byref(args), None) == -1, layout
        args = native.GatedScanArgs(**{**scan, **layout})
        assert lib.gs_gated_scan(ctypes.byref(args), None) == -1, layout
        assert lib.gs_gated_scan_backward(ctypes.byref(args), None) == -1, layout
    args = native.WindowAttentionArgs(**{**attention, "tiles": a, "tile_starts": a})
    assert lib.gs_window_attention_workspace_size(ctypes.byref(args)) == 0


def test_positions_end_before_32_bits_do():
    """The last tile of a walk reaches up to 256 tokens past the last one: lengths for
    which that position has no 32-bit number are refused."""
    from gaussian_splats_b200 import native

    lib, a, longest = native.lib(), 256, native.MAX_SEQUENCE_TOKENS
    assert longest + 511 <= 2 ** 31 - 1
    for tokens in (longest + 1, 2 ** 31 - 1):
        with pytest.raises(ValueError, match="at most"):
            PackedSequences([tokens], device="cpu")
        args = native.WindowAttentionArgs(
            tokens=tokens, num_tiles=-(-tokens // 128), heads=1, kv_heads=1, dim=8, dtype=1,
            scale=0.1, q=a, k=a, v=a, q_stride=8, q_head_stride=8, k_stride=8, k_head_stride=8,
            v_stride=8, v_head_stride=8, out=a)
        assert lib.gs_window_attention(ctypes.byref(args), None) == -1
        args = native.GatedScanArgs(
            tokens=tokens, sequences=1, num_tiles=-(-tokens // 128), channels=8, dtype=1, x=a,
            gate=a, x_stride=8, gate_stride=8, y=a, last=a, entering=a, workspace=a,
            workspace_size=1 << 50)
        assert lib.gs_gated_scan(ctypes.byref(args), None) == -1
        args = native.WindowAttentionStepArgs(
            batch=1, heads=1, kv_heads=1, dim=8, dtype=1, slots=tokens, scale=0.1, q=a, k=a, v=a,
            q_stride=8, q_head_stride=8, k_stride=8, k_head_stride=8, v_stride=8, v_head_stride=8,
            cache_k=a, cache_v=a, positions=a, out=a)
        assert lib.gs_window_attention_step(ctypes.byref(args), None) == -1


def test_library_refuses_validity_without_a_place_for_it():
    from gaussian_splats_b200 import native

    a = 256
    args = native.WindowAttentionStepArgs(
        batch=1, heads=1, kv_heads=1, dim=8, dtype=1, slots=4, scale=0.1, q=a, k=a, v=a, q_stride=8,
        q_head_stride=8, k_stride=8, k_head_stride=8, v_stride=8, v_head_stride=8, cache_k=a,
        cache_v=a, positions=a, out=a, valid=a)
    assert native.lib().gs_window_attention_step(ctypes.byref(args), None) == -1


def test_eight_bit_weights_follow_the_weights(monkeypatch):
    """After further training or a loaded checkpoint the codes are those of the new
    weights; they move with the module and are not saved."""
    from gaussian_splats_b200.refine import _Product

    used = []
    monkeypatch.setattr(torch, "_scaled_mm", lambda a, b, sa, sb, out_dtype: used.append(
        b.float() * sb))
    x, scale = torch.zeros(4, 32).to(torch.float8_e4m3fn), torch.ones(4)
    p = _Product(32, 48)
    names = set(p.state_dict())
    p.quantize()
    codes = p.codes
    p.eight_bit(x, scale)
    assert p.codes is codes  # not rounded again without need
    optimizer = torch.optim.SGD(p.parameters(), lr=1.0)
    p.weight.grad = torch.randn_like(p.weight)
    optimizer.step()
    p.eight_bit(x, scale)
    other = _Product(32, 48)
    p.load_state_dict(other.state_dict())
    p.eight_bit(x, scale)
    for got, weight in ((used[1], None), (used[2], other.weight)):
        if weight is not None:  # half a step of e4m3 (2**-4), or half its smallest (2**-10)
            w = weight.detach().float().t()
            assert ((got - w).abs() <= 1.01 * torch.maximum(
                w.abs() * 2.0 ** -4, w.abs().amax(0) / 448 * 2.0 ** -10)).all()
        assert not torch.equal(got, used[0])
    assert set(p.state_dict()) == names
    assert p.to("meta").codes.is_meta and p.scales.is_meta


def test_steps_tell_autograd_what_they_write(monkeypatch):
    """A graph that saved a cache or a state must not go on with what a step wrote."""
    from gaussian_splats_b200 import attention, recurrence

    for module in (attention, recurrence):
        monkeypatch.setattr(module, "call", lambda *arguments: None)
        monkeypatch.setattr(module, "check_cuda", lambda what, **tensors: torch.device("cpu"))
    h = torch.zeros(4, 1, 8, dtype=torch.bfloat16)
    k, v = torch.zeros(4, 5, 1, 8, dtype=torch.bfloat16), torch.zeros(4, 5, 1, 8, dtype=torch.bfloat16)
    seen, state, x = torch.zeros(4, 5, dtype=torch.bool), torch.zeros(4, 8), torch.zeros(4, 8)
    at = torch.zeros(4, dtype=torch.int64)
    for written, step in (
            ([k, v, seen], lambda: attention.window_attention_step(h, h, h, k, v, at,
                                                                   cache_valid=seen)),
            ([k, v], lambda: attention.window_attention_step(h, h, h, k, v, at)),
            ([state], lambda: recurrence.gated_scan_step(x, x, state))):
        for t in written:
            factor = torch.ones_like(t, dtype=torch.float32, requires_grad=True)
            product = factor * t  # saves t
            with torch.no_grad():
                step()
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                product.sum().backward()


def test_threads_share_the_entry_points():
    """The library's first calls from many threads at once (autograd has its own):
    without a GPU all come back with the same status, and none crashes."""
    from concurrent.futures import ThreadPoolExecutor

    from gaussian_splats_b200 import native

    if torch.cuda.is_available():
        pytest.skip("the addresses are not to be read")
    lib, a = native.lib(), 256
    args = native.WindowAttentionArgs(
        tokens=300, num_tiles=3, heads=4, kv_heads=2, dim=64, dtype=1, left=3, scale=0.1, q=a, k=a,
        v=a, q_stride=64, q_head_stride=64, k_stride=64, k_head_stride=64, v_stride=64,
        v_head_stride=64, out=a)
    with ThreadPoolExecutor(16) as pool:
        got = set(pool.map(lambda _: lib.gs_window_attention(ctypes.byref(args), None), range(200)))
    assert len(got) == 1 and got.pop() < 0
