"""Windowed attention against its definition in 64 bits."""

import pytest
import torch

import sequence_reference as R

pytestmark = pytest.mark.gpu

# Half a unit in the last place, relative: an output is rounded once, and the
# weights of a sum (probabilities, score gradients) may be rounded once to the
# same type before the product, so |error| <= U (|result| + spread), with a
# quarter more for float sums and exponentials. Weights under float16's normal
# range are off by at most 2**-25 each instead.
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def make(lengths, heads, kv_heads, dim, dtype, seed=0, dead=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens = sum(lengths)
    qkv = torch.randn((tokens, (heads + 2 * kv_heads) * dim), generator=g, device="cuda").to(dtype)
    q, k, v = (t.unflatten(1, (-1, dim)) for t in
               qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
    grad = torch.randn((tokens, heads, dim), generator=g, device="cuda").to(dtype)
    valid = torch.rand(tokens, generator=g, device="cuda") >= dead if dead else None
    return q, k, v, grad, valid


def call(q, k, v, grad, lengths, **window):
    from gaussian_splats_b200.attention import window_attention
    from gaussian_splats_b200.sequences import PackedSequences

    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    packed = None if len(lengths) == 1 else PackedSequences(lengths)
    out = window_attention(*leaves, packed, **window)
    grads = torch.autograd.grad(out, leaves, grad)
    return dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)))


def check(got, ref, dtype, rows, large):
    """``rows``: how many weights a sum may have; ``large``: the largest factor
    that a weight meets (for the weights that fall under the normal range)."""
    for name, t in got.items():
        bound = 1.25 * U[dtype] * (ref[name].abs() + ref[name + "_spread"]) + 1e-5
        bound = bound + TINY[dtype] * rows * large
        excess = ((t.double() - ref[name]).abs() - bound).max()
        assert torch.isfinite(t).all(), name
        assert excess <= 0, f"{name}: {excess.item():.3g} beyond its bound"


CASES = [
    # lengths, heads, kv_heads, dim, left, right, first, dead
    ([1], 1, 1, 8, 0, 0, 0, 0.0),
    ([1], 4, 2, 64, 5, 5, 3, 0.0),
    ([2, 0, 1, 3], 2, 1, 64, 1, 0, 1, 0.0),
    ([128], 2, 2, 64, 127, 0, 0, 0.0),
    ([129], 2, 1, 64, 16, 16, 4, 0.0),
    ([257], 3, 1, 72, 300, 300, 0, 0.0),           # wider than the sequence: no window
    ([0, 5, 0, 130, 384, 0], 4, 4, 64, 40, 0, 7, 0.0),
    ([700], 2, 1, 128, 100, 0, 128, 0.0),          # all first tokens allowed
    ([700], 2, 1, 96, 0, 0, 0, 0.0),               # each token sees itself
    ([640], 8, 2, 64, 200, 200, 16, 0.1),
    ([333, 444], 4, 1, 128, 130, 64, 4, 0.5),
    ([500], 2, 2, 32, 64, 0, 2, 0.97),             # most keys dead: rows that see nothing
    ([1100], 2, 1, 64, 2, 700, 1, 0.0),            # wider after than before
    ([1500, 33], 2, 2, 128, 1000, 0, 40, 0.0),
    ([300], 1, 1, 40, 2 ** 31 - 1, 2 ** 31 - 1, 5, 0.0),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_the_definition(case, dtype):
    lengths, heads, kv_heads, dim, left, right, first, dead = case
    q, k, v, grad, valid = make(lengths, heads, kv_heads, dim, dtype, dead=dead)
    window = dict(left=left, right=right, first=first, valid=valid)
    got = call(q, k, v, grad, lengths, **window)
    ref = R.attention(q, k, v, lengths, grad=grad, **window)
    check(got, ref, dtype, max(lengths) * heads // kv_heads, 6.0)


def test_forward_alone_gives_the_same():
    from gaussian_splats_b200.attention import window_attention

    q, k, v, grad, _ = make([700], 4, 2, 64, torch.bfloat16)
    with torch.no_grad():
        alone = window_attention(q, k, v, left=64, right=64, first=4)
    assert torch.equal(alone, call(q, k, v, grad, [700], left=64, right=64, first=4)["out"])


def test_repeats_bit_for_bit():
    q, k, v, grad, valid = make([900, 300], 8, 2, 64, torch.bfloat16, dead=0.1)
    a = call(q, k, v, grad, [900, 300], left=128, right=30, first=8, valid=valid)
    b = call(q, k, v, grad, [900, 300], left=128, right=30, first=8, valid=valid)
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_all_keys_dead():
    q, k, v, grad, _ = make([200, 60], 2, 1, 64, torch.bfloat16)
    valid = torch.ones(260, dtype=torch.bool, device="cuda")
    valid[200:] = False
    got = call(q, k, v, grad, [200, 60], left=30, right=30, first=2, valid=valid)
    for t in got.values():
        assert torch.count_nonzero(t[200:]) == 0 and torch.isfinite(t).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_dead_rows_may_hold_anything(bad):
    """Keys, values of dead tokens; the sequences beside a sequence."""
    lengths = [190, 300, 77]
    q, k, v, grad, valid = make(lengths, 2, 1, 64, torch.bfloat16, dead=0.2)
    window = dict(left=50, right=20, first=3)
    clean = call(q, k, v, grad, lengths, valid=valid, **window)
    k, v = k.clone(), v.clone()
    k[~valid], v[~valid] = bad, bad
    got = call(q, k, v, grad, lengths, valid=valid, **window)
    for n in got:
        assert torch.equal(got[n], clean[n]), n
    # a whole bad sequence in the middle leaves the others as they were
    q, grad = q.clone(), grad.clone()
    for t in (q, k, v, grad):
        t[190:490] = bad
    got = call(q, k, v, grad, lengths, valid=valid, **window)
    for n in got:
        assert torch.equal(got[n][:190], clean[n][:190]), n
        assert torch.equal(got[n][490:], clean[n][490:]), n


def test_a_seen_nan_shows():
    q, k, v, grad, _ = make([100], 1, 1, 64, torch.bfloat16)
    k = k.clone()
    k[:] = float("nan")
    assert torch.isnan(call(q, k, v, grad, [100], left=5)["out"]).all()


def test_large_scores():
    """Scores in the thousands: the running maximum carries them."""
    q, k, v, grad, _ = make([400], 2, 2, 64, torch.bfloat16)
    q, k = q * 30, k * 30
    ref = R.attention(q, k, v, [400], left=150, first=2)
    got = call(q, k, v, grad, [400], left=150, first=2)
    # float scores of this size are exact to 2**-23 of 5e3 or so: exp is off by 1e-3 at most
    bound = 1.25 * (U[torch.bfloat16] + 2e-3) * (ref["out"].abs() + ref["out_spread"]) + 1e-5
    assert ((got["out"].double() - ref["out"]).abs() <= bound).all()


@pytest.mark.parametrize("layout", ["heads first", "odd rows", "expanded", "offset"])
def test_strides(layout):
    q, k, v, grad, _ = make([200], 4, 2, 64, torch.float16)
    window = dict(left=40, right=8, first=1)
    if layout == "expanded":
        k, v = k[:, :1].expand(-1, 2, -1), v[:1].expand(200, -1, -1)
    expected = call(q.contiguous(), k.contiguous(), v.contiguous(), grad, [200], **window)
    if layout == "heads first":
        q, k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    elif layout == "odd rows":
        q, k, v = (torch.cat((t.flatten(1), t.flatten(1)[:, :3]), 1)[:, :-3].unflatten(1, (-1, 64))
                   for t in (q, k, v))
    elif layout == "offset":
        q, k, v = (torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape) for t in (q, k, v))
    grad = grad.transpose(0, 1).contiguous().transpose(0, 1)
    got = call(q, k, v, grad, [200], **window)
    assert all(torch.equal(got[n], expected[n]) for n in got)


def test_gradient_against_differences():
    q, k, v, grad, _ = make([96], 2, 1, 32, torch.float16, seed=3)
    window = dict(left=30, right=10, first=2)
    grads = call(q, k, v, grad, [96], **window)
    for name, at in (("dq", 0), ("dk", 1), ("dv", 2)):
        d = grads[name].double()
        d = 4.0 * d / d.norm()  # about 0.06 in each element
        sides = []
        for sign in (1, -1):
            inputs = [q, k, v]
            inputs[at] = (inputs[at].double() + sign * d).half()
            out = call(*inputs, grad, [96], **window)["out"]
            sides.append(((out.double() * grad.double()).sum(), inputs[at].double()))
        expected = (grads[name].double() * (sides[0][1] - sides[1][1])).sum()
        # the third order of a step of 0.1 in a score, and the outputs' rounding
        assert abs((sides[0][0] - sides[1][0]) / expected - 1) < 0.03


def test_on_another_stream():
    from gaussian_splats_b200.attention import window_attention

    q, k, v, grad, _ = make([3000], 4, 2, 64, torch.bfloat16)
    expected = call(q, k, v, grad, [3000], left=100, first=4)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = window_attention(*leaves, left=100, first=4)
        grads = torch.autograd.grad(out, leaves, grad)
    torch.cuda.current_stream().wait_stream(stream)
    for t, n in zip((out, *grads), ("out", "dq", "dk", "dv")):
        assert torch.equal(t, expected[n])


# ------------------------------------------------------------------ one new token


STEPS = [
    # batch, heads, kv_heads, dim, left, first
    (1, 1, 1, 8, 0, 0),
    (1, 8, 2, 64, 1023, 4),
    (3, 4, 4, 128, 30, 1),
    (5, 6, 1, 96, 200, 16),
    (2, 16, 1, 64, 700, 0),
    (70, 8, 8, 32, 129, 3),
    (2, 7, 7, 120, 5000, 4),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("case", STEPS, ids=str)
def test_step_against_the_definition(case, dtype):
    from gaussian_splats_b200.attention import window_attention_step

    batch, heads, kv_heads, dim, left, first = case
    g = torch.Generator(device="cuda").manual_seed(1)
    slots, rand = first + left + 1, lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)
    q, k, v = rand(batch, heads, dim), rand(batch, kv_heads, dim), rand(batch, kv_heads, dim)
    cache_k, cache_v = rand(batch, slots, kv_heads, dim), rand(batch, slots, kv_heads, dim)
    positions = torch.randint(0, 3 * slots, (batch,), generator=g, device="cuda")
    positions[0] = slots - 1
    if batch > 1:
        positions[1] = -1
    if batch > 2:
        positions[2] = 0
    ck, cv = cache_k.clone(), cache_v.clone()
    for b, p in enumerate(positions.tolist()):  # what no token has filled may hold anything
        cache_k[b, p + 1:], cache_v[b, p + 1:] = float("nan"), float("nan")
        if p < slots:
            ck[b, p + 1:], cv[b, p + 1:] = float("nan"), float("nan")
    out = window_attention_step(q, k, v, cache_k, cache_v, positions, first=first)
    for b, p in enumerate(positions.tolist()):
        if p >= 0:
            slot = p if p < first else first + (p - first) % (left + 1)
            ck[b, slot], cv[b, slot] = k[b], v[b]
            n = min(p + 1, slots)
            kk, vv = (t[b, :n].double().repeat_interleave(heads // kv_heads, 1) for t in (ck, cv))
            w = (torch.einsum("hd,nhd->hn", q[b].double(), kk) * dim ** -0.5).softmax(1)
            o, spread = torch.einsum("hn,nhd->hd", w, vv), torch.einsum("hn,nhd->hd", w, vv.abs())
            bound = 1.25 * U[dtype] * (o.abs() + spread) + 1e-5 + TINY[dtype] * n * 6.0
            assert ((out[b].double() - o).abs() <= bound).all(), b
        else:
            assert torch.count_nonzero(out[b]) == 0
    for got, expected in ((cache_k, ck), (cache_v, cv)):
        assert torch.equal(got.view(torch.int16), expected.view(torch.int16))


def test_steps_follow_the_whole_sequence():
    """A stream token by token gives the rows of the whole sequence's attention."""
    from gaussian_splats_b200.attention import (window_attention, window_attention_step,
                                                window_cache)

    q, k, v, _, _ = make([150], 4, 2, 64, torch.float16, seed=5)
    whole = window_attention(q, k, v, left=20, first=3)
    cache = window_cache(1, 20, 3, 2, 64, torch.float16)
    for t in range(150):
        out = window_attention_step(q[t:t + 1], k[t:t + 1], v[t:t + 1], *cache,
                                    torch.tensor([t], device="cuda"), first=3)
        torch.testing.assert_close(out[0], whole[t], rtol=2 * 2.0 ** -10, atol=2e-3)


# ------------------------------------------------------------------------ refusals


def test_refusals():
    from gaussian_splats_b200.attention import window_attention, window_attention_step
    from gaussian_splats_b200.sequences import PackedSequences

    q, k, v, _, _ = make([64], 4, 2, 64, torch.bfloat16)
    for error, match, args, window in [
        (RuntimeError, "CUDA devices only", (q.cpu(), k.cpu(), v.cpu()), {}),
        (ValueError, "not a multiple of 2 key-value", (q[:, :3], k, v), {}),
        (ValueError, "does not go with", (q, k[:10], v[:10]), {}),
        (ValueError, "does not go with", (q, k, v[:, :1]), {}),
        (ValueError, "different types", (q, k.half(), v), {}),
        (ValueError, "float32 is not supported", (q.float(), k.float(), v.float()), {}),
        (ValueError, "head dim 60", (q[..., :60], k[..., :60], v[..., :60]), {}),
        (ValueError, r"expected \[tokens", (q[0], k[0], v[0]), {}),
        (ValueError, "left and right", (q, k, v), {"left": -1}),
        (ValueError, "first must be", (q, k, v), {"first": 129}),
        (ValueError, "scale must be", (q, k, v), {"scale": 0.0}),
        (ValueError, "valid must be", (q, k, v), {"valid": torch.ones(64, device="cuda")}),
        (ValueError, "hold 65 tokens", (q, k, v, PackedSequences([60, 5])), {}),
        (RuntimeError, "packed sequences on cpu", (q, k, v, PackedSequences([64], "cpu")), {}),
    ]:
        with pytest.raises(error, match=match):
            window_attention(*args, **{"left": 4, **window})
    wide = torch.zeros((8, 1, 136), dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="head dim 136"):
        window_attention(wide, wide, wide, left=1)
    cache = torch.zeros((64, 9, 2, 64), dtype=torch.bfloat16, device="cuda")
    at = torch.zeros(64, dtype=torch.int64, device="cuda")
    for match, args, first in [
        ("positions must be int64", (cache, cache.clone(), at.int()), 0),
        ("are not", (cache, cache[:, :5], at), 0),
        ("caches of", (cache.half(), cache.half(), at), 0),
        ("contiguous", (cache.transpose(1, 2).contiguous().transpose(1, 2), cache, at), 0),
        ("first must be", (cache, cache.clone(), at), 9),
    ]:
        with pytest.raises(ValueError, match=match):
            window_attention_step(q, k, v, *args, first=first)


def test_no_tokens():
    q, k, v, grad, _ = make([0], 2, 1, 64, torch.bfloat16)
    assert call(q, k, v, grad, [0], left=3)["out"].shape == (0, 2, 64)
    assert call(q, k, v, grad, [0, 0], left=3)["dk"].shape == (0, 1, 64)


def test_no_wait_ran_out():
    """The status call: every bounded wait of the kernels came back."""
    from gaussian_splats_b200 import native

    q, k, v, grad, valid = make([700, 0, 129], 4, 2, 128, torch.float16, dead=0.3)
    call(q, k, v, grad, [700, 0, 129], valid=valid, left=200, right=9, first=5)
    assert native.lib().gs_window_attention_status(torch.cuda.current_stream().cuda_stream) == 0


def test_outputs_end_where_the_sequence_ends():
    """Rows are written side by side: none of a neighbour's, none past the end."""
    import ctypes

    from gaussian_splats_b200 import native
    from gaussian_splats_b200.attention import _arguments
    from gaussian_splats_b200.sequences import (PackedSequences, call as run, element_type,
                                                tile_arguments)

    lengths, heads, kv_heads, dim = [130, 1, 255, 66], 3, 3, 72
    q, k, v, grad, _ = make(lengths, heads, kv_heads, dim, torch.bfloat16)
    tokens, packed = sum(lengths), PackedSequences(lengths)
    spare = {n: torch.full((tokens + 300, heads, dim), 7.0, dtype=q.dtype, device="cuda")
             for n in ("out", "grad_q", "grad_k", "grad_v")}
    lse = torch.empty((heads, tokens), device="cuda")
    q, k, v, grad = (t.contiguous() for t in (q, k, v, grad))
    args = _arguments(native.WindowAttentionArgs, q, k, v, tokens=tokens,
                      **tile_arguments(packed, tokens), heads=heads, kv_heads=kv_heads, dim=dim,
                      dtype=element_type(q.dtype, "q"), left=40, right=3, first=2,
                      scale=0.1, lse=lse.data_ptr(), grad_out=grad.data_ptr(),
                      **{n: t.data_ptr() for n, t in spare.items()})
    size = native.lib().gs_window_attention_workspace_size(ctypes.byref(args))
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    args.workspace, args.workspace_size = workspace.data_ptr(), size
    run("gs_window_attention", q.device, ctypes.byref(args))
    run("gs_window_attention_backward", q.device, ctypes.byref(args))
    want = call(q, k, v, grad, lengths, left=40, right=3, first=2, scale=0.1)
    for name, other in (("out", "out"), ("grad_q", "dq"), ("grad_k", "dk"), ("grad_v", "dv")):
        assert torch.equal(spare[name][:tokens], want[other]), name
        assert (spare[name][tokens:] == 7).all(), name


@pytest.mark.parametrize("size", [2.0 ** -9, 2.0 ** 10], ids=["small", "large"])
@pytest.mark.parametrize("dim,left,right,first", [(64, 300, 200, 5), (128, 700, 0, 0),
                                                  (64, 1, 1, 2)], ids=str)
def test_float16_gradients_of_any_size(dim, left, right, first, size):
    """Gradients under a loss scale, or far below one: powers of two times the unit
    ones, so the bounds are those of the unit ones times the size, and half a unit of
    the subnormal results. Peaked weights (scores of deviation 3) make score
    gradients of several thousand at the larger size, where the results fit."""
    lengths = [900, 0, 270]
    q, k, v, grad, valid = make(lengths, 4, 2, dim, torch.float16, seed=7, dead=0.1)
    q, grad = 3 * q, size * grad
    window = dict(left=left, right=right, first=first, valid=valid)
    ref = R.attention(q, k, v, lengths, grad=grad, **window)
    got = call(q, k, v, grad, lengths, **window)
    for name in ("dq", "dk", "dv"):
        assert ref[name].abs().max() < torch.finfo(torch.float16).max
        bound = 1.25 * U[torch.float16] * (ref[name].abs() + ref[name + "_spread"])
        bound = bound + size * (1e-5 + TINY[torch.float16] * 900 * 2 * 18.0) + 2.0 ** -25
        assert torch.isfinite(got[name]).all(), name
        excess = ((got[name].double() - ref[name]).abs() - bound).max()
        assert excess <= 0, f"{name}: {excess.item():.3g} beyond its bound"


def test_float16_gradients_of_one_query_leave_the_others_theirs():
    """One query's gradient of 2**15 times the others' size, in another sequence and in
    the same one out of reach: those that it does not meet keep their bits."""
    lengths = [400, 900]
    q, k, v, grad, _ = make(lengths, 2, 1, 64, torch.float16, seed=8)
    grad = grad * 2.0 ** -6
    window = dict(left=20, right=20)
    clean = call(q, k, v, grad, lengths, **window)
    grad[450] *= 2.0 ** 15
    got = call(q, k, v, grad, lengths, **window)
    for name in ("dq", "dk", "dv"):
        assert torch.isfinite(got[name]).all()
        assert torch.equal(got[name][:400], clean[name][:400]), name
        assert torch.equal(got[name][900:], clean[name][900:]), name


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dim", [64, 128])
def test_queries_that_see_nothing_may_hold_anything(dim, bad):
    """A run of dead tokens longer than the window: those inside it see nothing, and no
    gradient flows through them, whatever they and their output's gradient hold."""
    q, k, v, grad, _ = make([500], 4, 2, dim, torch.bfloat16)
    valid = torch.ones(500, dtype=torch.bool, device="cuda")
    valid[200:240] = False
    window = dict(left=6, right=3, valid=valid)
    clean = call(q, k, v, grad, [500], **window)
    q, grad = q.clone(), grad.clone()
    q[206:237], grad[206:237] = bad, bad
    got = call(q, k, v, grad, [500], **window)
    for name in got:
        assert torch.equal(got[name], clean[name]), name
    assert torch.count_nonzero(got["dq"][206:237]) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("case", STEPS, ids=str)
def test_step_leaves_slots_out(case, dtype):
    """Slots that are not valid, the new token's own among them, whatever they hold."""
    from gaussian_splats_b200.attention import window_attention_step

    batch, heads, kv_heads, dim, left, first = case
    g = torch.Generator(device="cuda").manual_seed(2)
    slots, rand = first + left + 1, lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)
    q, k, v = rand(batch, heads, dim), rand(batch, kv_heads, dim), rand(batch, kv_heads, dim)
    cache_k, cache_v = rand(batch, slots, kv_heads, dim), rand(batch, slots, kv_heads, dim)
    positions = torch.randint(0, 3 * slots, (batch,), generator=g, device="cuda")
    if batch > 4:
        positions[1], positions[2] = -1, 0
    seen = torch.rand(batch, slots, generator=g, device="cuda") > 0.4
    valid = torch.rand(batch, generator=g, device="cuda") > 0.5
    seen[-1] = False  # nothing but the token itself, or not even that
    at, expected = positions.tolist(), seen.clone()
    for b, p in enumerate(at):
        if p >= 0:
            expected[b, p if p < first else first + (p - first) % (left + 1)] = valid[b]
    for t in (cache_k, cache_v):
        t[~seen] = float("nan")
    bad = ~valid[:, None, None]
    k, v = torch.where(bad, float("inf"), k), torch.where(bad, float("nan"), v)
    cache_valid = seen.clone()
    out = window_attention_step(q, k, v, cache_k, cache_v, positions, first=first, valid=valid,
                                cache_valid=cache_valid)
    assert torch.equal(cache_valid, expected)
    for b, p in enumerate(at):
        keys = expected[b].clone()
        keys[max(p + 1, 0):] = False
        if p < 0 or not keys.any():
            assert torch.count_nonzero(out[b]) == 0, b
            continue
        kk, vv = (t[b, keys].double().repeat_interleave(heads // kv_heads, 1)
                  for t in (cache_k, cache_v))
        w = (torch.einsum("hd,nhd->hn", q[b].double(), kk) * dim ** -0.5).softmax(1)
        o, spread = torch.einsum("hn,nhd->hd", w, vv), torch.einsum("hn,nhd->hd", w, vv.abs())
        bound = 1.25 * U[dtype] * (o.abs() + spread) + 1e-5 + TINY[dtype] * len(kk) * 6.0
        assert ((out[b].double() - o).abs() <= bound).all(), b


def test_step_without_valid_fills_cache_valid():
    from gaussian_splats_b200.attention import window_attention_step, window_cache

    q, k, v, _, _ = make([3], 2, 2, 64, torch.bfloat16)
    cache, positions = window_cache(3, 4, 1, 2, 64), torch.tensor([0, -1, 7], device="cuda")
    seen = torch.zeros(3, 6, dtype=torch.bool, device="cuda")
    out = window_attention_step(q, k, v, *cache, positions, first=1, cache_valid=seen)
    assert seen.nonzero().tolist() == [[0, 0], [2, 2]]
    assert torch.equal(out[0], v[0]) and torch.equal(out[2], v[2])


def test_step_refuses_validity_that_does_not_fit():
    from gaussian_splats_b200.attention import window_attention_step, window_cache

    q, k, v, _, _ = make([3], 2, 2, 64, torch.bfloat16)
    cache, at = window_cache(3, 4, 1, 2, 64), torch.zeros(3, dtype=torch.int64, device="cuda")
    seen = torch.ones(3, 6, dtype=torch.bool, device="cuda")
    for match, valid, cache_valid in [
        ("without cache_valid", seen[:, 0], None), ("valid must be bool", seen[:2, 0], seen),
        ("valid must be bool", at, seen), ("cache_valid must be", seen[:, 0], seen[:, :5]),
        ("cache_valid must be", None, seen.int()),
        ("cache_valid must be", None, seen.t().contiguous().t()),
    ]:
        with pytest.raises(ValueError, match=match):
            window_attention_step(q, k, v, *cache, at, first=1, valid=valid,
                                  cache_valid=cache_valid)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("tokens,dim,left,right,first", [
    (2600, 64, 2300, 0, 0),    # more than 32 tiles of 64 keys: the plan's second batch
    (2700, 64, 1200, 1400, 70),
    (4700, 128, 4500, 0, 3),   # more than 32 tiles of 128 keys
    (6000, 64, 50, 0, 9),      # six chunks of first tokens' later queries
    (6200, 128, 30, 40, 128),
], ids=str)
def test_long_walks(tokens, dim, left, right, first, dtype):
    if max(left, right) > 1000:
        seen = min(left, tokens) + right + 1
        assert seen > 32 * (64 if dim == 64 else 128)
    else:
        assert tokens > 5 * 8 * 128 and left + right < 7 * 128  # chunks of 8 tiles
    q, k, v, grad, _ = make([tokens], 2, 1, dim, dtype, seed=12)
    window = dict(left=left, right=right, first=first)
    got = call(q, k, v, grad, [tokens], **window)
    ref = R.attention(q, k, v, [tokens], grad=grad, **window)
    check(got, ref, dtype, tokens * 2, 6.0)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("depth", [20.5, 25.2], ids=str)
def test_float16_keeps_many_small_weights(dim, depth):
    """One key holds nearly all of the weight, thousands have 2**-depth of it each: the
    sum of these is kept, not cut off under float16's smallest number. Stored times
    2**7 they are off by at most 2**-32, 4096 of them by 2**-20 of a value."""
    from gaussian_splats_b200.attention import window_attention, window_attention_step

    n = 4096
    q = torch.zeros(n, 1, dim, dtype=torch.float16, device="cuda")
    k, v = q.clone(), torch.ones_like(q)
    q[..., 0], k[0, 0, 0], v[0] = 1.0, 32.0, 0.0
    scale = depth * 0.6931471805599453 / 32.0
    small = torch.arange(n, device="cuda").double() * 2.0 ** -depth
    expected = small / (1.0 + small)
    bound = 1.25 * 2 * U[torch.float16] * expected + 2.0 ** -20 + 2.0 ** -25
    out = window_attention(q, k, v, left=n, scale=scale)
    assert ((out[:, 0].double() - expected[:, None]).abs() <= bound[:, None]).all()
    step = window_attention_step(q[:1], k[-1:], v[-1:], k[None].clone(), v[None].clone(),
                                 torch.tensor([n - 1], device="cuda"), scale=scale)
    assert ((step[0, 0].double() - expected[-1]).abs() <= bound[-1]).all()
