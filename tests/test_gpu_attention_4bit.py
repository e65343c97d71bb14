"""The step against a 4-bit cache, from its definition in 64 bits."""

import pytest
import torch

import operator_reference as R

pytestmark = pytest.mark.gpu

U = R.U
BF, HF = torch.bfloat16, torch.float16


def rand(g, *shape, dtype, size=1.0):
    return (size * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def bound(dtype, dim, out, spread, size, scores):
    """The result's rounding; the weights times the steps rounded to the inputs' type
    (a weight's rounding error meets a value's distance from its middle) and, for their
    sum with the middles, float sums; a score's error shifts its weight by as much:
    (dim + 8) units 2^-23 of its parts' sizes, twice for the ratio of two weights."""
    shift = 2.0 * (dim + 8) * 2.0 ** -23 * scores[..., None] + 2.0 ** -20
    return 1.01 * (U[dtype] * out.abs() + U[dtype] * spread + shift * 2.0 * size +
                   2.0 ** -18 * (spread + size) + 2.0 ** -25)


def compare(got, ref, dtype, dim):
    out = ref[0]
    error = (got.double() - out).abs()
    limit = bound(dtype, dim, *ref)
    # Rows at float16's limit: the step, 131008 / 15 rounded to 8736, holds 65504 as 7.5
    # steps, 65520, which is where rounding to float16 gives infinity.
    if dtype == HF:
        error[(got == out.sign() * float("inf")) & (out.abs() + limit >= 65520.0)] = 0.0
    assert (error <= limit).all(), f"{(error - limit).max().item():.3g} beyond"


@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 8), (2, 1, 64), (8, 2, 64), (6, 2, 40),
                                                (4, 4, 96), (16, 4, 128), (24, 2, 128),
                                                (9, 1, 32), (40, 2, 16), (3, 3, 120)])
def test_streams(heads, kv_heads, dim, dtype):
    """From empty caches past their wrap, streams at different positions, one idle now
    and then, dead tokens."""
    from gaussian_splats_b200.attention import window_attention_step_4bit, window_cache_4bit

    g = torch.Generator(device="cuda").manual_seed(heads * 1000 + dim)
    for left, first, masked in ((0, 0, False), (6, 0, True), (20, 3, False), (20, 3, True)):
        batch, slots = 4, first + left + 1
        cache = window_cache_4bit(batch, left, first, kv_heads, dim, dtype)
        ref = R.Streams(batch, slots, first, kv_heads, dim, dtype, "cuda")
        cache_valid = torch.zeros(batch, slots, dtype=torch.bool, device="cuda") if masked else None
        at = torch.zeros(batch, dtype=torch.int64)
        for turn in range(2 * slots + 3):
            busy = torch.tensor([True, turn % 2 == 0, turn % 3 > 0, turn > slots])
            positions = torch.where(busy, at, -1).cuda()
            at = at + busy
            q = rand(g, batch, heads, dim, dtype=dtype)
            k = rand(g, batch, kv_heads, dim, dtype=dtype)
            v = rand(g, batch, kv_heads, dim, dtype=dtype, size=3.0) + 1.0
            valid = torch.rand(batch, generator=g, device="cuda") < 0.6 if masked else None
            out = window_attention_step_4bit(q, k, v, cache, positions, first=first, valid=valid,
                                             cache_valid=cache_valid)
            want = ref.step(q, k, v, positions, dim ** -0.5, valid)
            compare(out, want, dtype, dim)
            for i, (codes, ranges) in enumerate((cache[:2], cache[2:])):
                assert torch.equal(codes, ref.codes[i]) and torch.equal(ranges, ref.ranges[i])
            if masked:
                assert torch.equal(cache_valid, ref.seen)


def fill(ref, g, dtype, batch, kv_heads, slots, dim, full=True):
    """Caches as earlier tokens left them."""
    for i, kept in enumerate((ref.k, ref.v)):
        code, step, middle = R.held(rand(g, batch, kv_heads, slots, dim, dtype=dtype, size=1 + i))
        ref.codes[i][:], ref.ranges[i][:] = R.packed(code), torch.stack((step, middle), -1)
        kept[:] = (code.double() - 7.5) * step.double()[..., None] + middle.double()[..., None]
    ref.seen[:] = full


@pytest.mark.parametrize("batch,heads,kv_heads,dim,left,first,dtype", [
    (1, 8, 2, 64, 1023, 4, BF), (3, 4, 1, 128, 5000, 0, HF), (2, 6, 2, 96, 2047, 16, BF),
    (1, 16, 1, 128, 20000, 1, HF), (5, 3, 3, 32, 700, 2, BF), (2, 20, 1, 72, 3001, 0, HF),
    (64, 4, 4, 64, 130, 0, BF)])
def test_long_caches(batch, heads, kv_heads, dim, left, first, dtype):
    from gaussian_splats_b200.attention import FourBitCache, window_attention_step_4bit

    g = torch.Generator(device="cuda").manual_seed(left)
    slots = first + left + 1
    for masked in (False, True):
        ref = R.Streams(batch, slots, first, kv_heads, dim, dtype, "cuda")
        positions = torch.randint(slots, 5 * slots, (batch,), generator=g, device="cuda")
        fill(ref, g, dtype, batch, kv_heads, slots, dim)
        if masked:  # stream 0 sees its own token at most
            ref.seen[:] = torch.rand(batch, slots, generator=g, device="cuda") < 0.5
            ref.seen[0] = False
        cache = FourBitCache(ref.codes[0].clone(), ref.ranges[0].clone(), ref.codes[1].clone(),
                             ref.ranges[1].clone())
        q = rand(g, batch, heads, dim, dtype=dtype)
        k, v = (rand(g, batch, kv_heads, dim, dtype=dtype) for _ in range(2))
        cache_valid = ref.seen.clone() if masked else None
        valid = torch.arange(batch, device="cuda") % 3 != 0 if masked else None
        out = window_attention_step_4bit(q, k, v, cache, positions, first=first, valid=valid,
                                         cache_valid=cache_valid)
        want = ref.step(q, k, v, positions, dim ** -0.5, valid)
        compare(out, want, dtype, dim)
        if masked:
            assert (out[0] == 0).all() and torch.equal(cache_valid, ref.seen)
        assert torch.equal(cache.k_codes, ref.codes[0]) and torch.equal(cache.v_codes, ref.codes[1])
        # partly filled: what lies past the token's position is not looked at
        few = torch.full((batch,), slots // 3, device="cuda")
        nan = [t.clone() for t in cache]
        nan[1][:, :, slots // 3 + 1:] = float("nan")
        nan[3][:, :, slots // 3 + 1:] = float("nan")
        ref.seen[:, slots // 3 + 1:] = False
        if masked:  # nor what is left out
            cache_valid = ref.seen.clone()
            out_of = ~ref.seen[:, None, :, None].expand_as(nan[1])
            nan[1][out_of] = nan[3][out_of] = float("nan")
            out_of = out_of[..., :1].expand_as(nan[0])
            nan[0][out_of] = nan[2][out_of] = 255
        else:
            ref.seen[:, :slots // 3] = True
        out = window_attention_step_4bit(q, k, v, FourBitCache(*nan), few, first=first,
                                         valid=valid, cache_valid=cache_valid)
        compare(out, ref.step(q, k, v, few, dim ** -0.5, valid), dtype, dim)


def test_many_streams():
    """More streams than are counted first, some idle, at different places; and one head
    that many query heads share."""
    from gaussian_splats_b200.attention import FourBitCache, window_attention_step_4bit

    for batch, heads, kv_heads, dim, slots in ((1025, 2, 1, 16, 70), (1500, 3, 3, 8, 40),
                                               (1024, 1, 1, 64, 65)):
        g = torch.Generator(device="cuda").manual_seed(batch)
        ref = R.Streams(batch, slots, 2, kv_heads, dim, BF, "cuda")
        fill(ref, g, BF, batch, kv_heads, slots, dim)
        positions = torch.randint(-1, 2 * slots, (batch,), generator=g, device="cuda")
        ref.seen[:] = torch.arange(slots, device="cuda") < positions[:, None]
        cache = FourBitCache(ref.codes[0].clone(), ref.ranges[0].clone(), ref.codes[1].clone(),
                             ref.ranges[1].clone())
        q = rand(g, batch, heads, dim, dtype=BF)
        k, v = (rand(g, batch, kv_heads, dim, dtype=BF) for _ in range(2))
        out = window_attention_step_4bit(q, k, v, cache, positions, first=2)
        compare(out, ref.step(q, k, v, positions, dim ** -0.5), BF, dim)
        assert (out[positions < 0] == 0).all() and (positions < 0).any()
        for i, (codes, ranges) in enumerate((cache[:2], cache[2:])):
            assert torch.equal(codes, ref.codes[i]) and torch.equal(ranges, ref.ranges[i])


def test_all_idle():
    from gaussian_splats_b200.attention import window_attention_step_4bit, window_cache_4bit

    g = torch.Generator(device="cuda").manual_seed(1)
    for batch in (3, 2000):
        cache = window_cache_4bit(batch, 5, 0, 1, 32)
        q = rand(g, batch, 2, 32, dtype=BF)
        out = window_attention_step_4bit(q, q[:, :1], q[:, 1:], cache,
                                         torch.full((batch,), -1, device="cuda"))
        assert (out == 0).all() and all((t == 0).all() for t in cache)


def test_status():
    import ctypes

    from gaussian_splats_b200 import native

    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert native.lib().gs_window_attention_status(stream) == 0
    assert native.lib().gs_linear_status(stream) == 0


def test_rows_that_are_special():
    """Rows of one value, of zeros, of subnormals, of the type's limits, and not finite."""
    from gaussian_splats_b200.attention import window_attention_step_4bit, window_cache_4bit

    for dtype in (BF, HF):
        top = torch.finfo(dtype).max if dtype == HF else 1e30
        rows = [torch.zeros(32), torch.full((32,), 3.5), torch.full((32,), -2.0 ** -20),
                torch.linspace(-1, 1, 32) * 2.0 ** -22, torch.linspace(-1, 1, 32) * top,
                torch.tensor([0.0] * 31 + [1.0]), torch.arange(32) / 31.0 * 15.0]
        batch = len(rows)
        k = torch.stack(rows).to(dtype).cuda()[:, None]
        v = k.clone()
        cache = window_cache_4bit(batch, 4, 0, 1, 32, dtype)
        ref = R.Streams(batch, 5, 0, 1, 32, dtype, "cuda")
        q = torch.full((batch, 1, 32), 2.0 ** -10, device="cuda", dtype=dtype)
        positions = torch.zeros(batch, dtype=torch.int64, device="cuda")
        out = window_attention_step_4bit(q, k, v, cache, positions)
        want = ref.step(q, k, v, positions, 32 ** -0.5)
        for i, (codes, ranges) in enumerate((cache[:2], cache[2:])):
            assert torch.equal(codes, ref.codes[i]) and torch.equal(ranges, ref.ranges[i])
        compare(out, want, dtype, 32)
        for bad in (float("nan"), float("inf")):
            v2 = v.clone()
            v2[:, :, 5] = bad
            out = window_attention_step_4bit(q, k, v2, cache, positions + 1)
            assert not out.isfinite().any()


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes of codes: its last slots are where they belong."""
    from gaussian_splats_b200.attention import FourBitCache, window_attention_step_4bit

    kv_heads, dim, slots = 8, 128, 9_000_001
    codes = [torch.full((1, kv_heads, slots, dim // 2), 0x88, dtype=torch.uint8, device="cuda")
             for _ in range(2)]
    ranges = [torch.zeros(1, kv_heads, slots, 2, dtype=BF, device="cuda") for _ in range(2)]
    ranges[0][..., 0] = 0.125  # keys (8 - 7.5) / 8
    codes[0][:, :, -3] = 0xff
    ranges[0][:, :, -3, 0] = 64.0  # one key that outweighs all others
    ranges[1][:, :, -3, 1] = torch.arange(1, kv_heads + 1, device="cuda").to(BF)
    q = torch.ones(1, kv_heads, dim, device="cuda", dtype=BF)
    token = torch.zeros(1, kv_heads, dim, device="cuda", dtype=BF)
    out = window_attention_step_4bit(q, token, token, FourBitCache(codes[0], ranges[0], codes[1],
                                                                   ranges[1]),
                                     torch.tensor([slots * 3 + 5], device="cuda"))
    want = torch.arange(1, kv_heads + 1, device="cuda").to(BF)[None, :, None].expand_as(out)
    assert torch.equal(out, want)
    assert (codes[0][0, :, 5] == 0x88).all() and (ranges[0][0, :, 5] == 0).all()


def test_repeats_streams_and_graph():
    from gaussian_splats_b200.attention import window_attention_step_4bit, window_cache_4bit

    g = torch.Generator(device="cuda").manual_seed(5)
    tokens = [(rand(g, 3, 8, 64, dtype=BF), rand(g, 3, 2, 64, dtype=BF), rand(g, 3, 2, 64, dtype=BF))
              for _ in range(12)]
    caches = [window_cache_4bit(3, 6, 1, 2, 64) for _ in range(3)]
    positions = torch.zeros(3, dtype=torch.int64, device="cuda")
    plain = [window_attention_step_4bit(*t, caches[0], positions + i, first=1)
             for i, t in enumerate(tokens)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [window_attention_step_4bit(*t, caches[1], positions + i, first=1)
                 for i, t in enumerate(tokens)]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    held, at = [t.clone() for t in tokens[0]], positions.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = window_attention_step_4bit(*held, caches[2], at, first=1)
        at += 1
    for i, t in enumerate(tokens):
        for h, x in zip(held, t):
            h.copy_(x)
        graph.replay()
        assert torch.equal(out, plain[i]) and torch.equal(other[i], plain[i])
    for a, b, c in zip(*caches):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_steps_at_once():
    """Steps of three batches on three streams at the same time, each its own caches."""
    from gaussian_splats_b200.attention import window_attention_step_4bit, window_cache_4bit

    shapes = [(1, 8, 2, 64, 200), (40, 16, 4, 128, 300), (7, 3, 3, 96, 1000)]

    def run(streams):
        g = torch.Generator(device="cuda").manual_seed(5)
        caches = [window_cache_4bit(b, left, 1, kv, d) for b, _, kv, d, left in shapes]
        tokens = [[(rand(g, b, h, d, dtype=BF), rand(g, b, kv, d, dtype=BF),
                    rand(g, b, kv, d, dtype=BF)) for b, h, kv, d, _ in shapes] for _ in range(6)]
        places = [[torch.full((shape[0],), p, device="cuda") for p in range(6)] for shape in shapes]
        torch.cuda.synchronize()
        out = []
        for p, step in enumerate(tokens):
            for i, (q, k, v) in enumerate(step):
                with torch.cuda.stream(streams[i]):
                    out.append(window_attention_step_4bit(q, k, v, caches[i], places[i][p], first=1))
        torch.cuda.synchronize()
        return out + [t for cache in caches for t in cache]

    apart = run([torch.cuda.Stream() for _ in shapes])
    assert all(torch.equal(a, b) for a, b in zip(run([torch.cuda.current_stream()] * 3), apart))


def test_strided_tokens_and_refusals():
    from gaussian_splats_b200.attention import (FourBitCache, window_attention_step_4bit,
                                                window_cache_4bit)

    g = torch.Generator(device="cuda").manual_seed(6)
    both = rand(g, 3, 12 * 64 + 3, dtype=HF)
    parts = [both[:, 3 + a:3 + b].unflatten(1, (-1, 64)) for a, b in ((0, 512), (512, 640), (640, 768))]
    positions = torch.tensor([0, 5, 900], device="cuda")
    caches = [window_cache_4bit(3, 6, 1, 2, 64, HF) for _ in range(2)]
    a = window_attention_step_4bit(*parts, caches[0], positions, first=1, scale=0.3)
    b = window_attention_step_4bit(*(t.contiguous() for t in parts), caches[1], positions, first=1,
                                   scale=0.3)
    assert torch.equal(a, b)
    none = window_attention_step_4bit(*(t[:0] for t in parts), window_cache_4bit(0, 6, 1, 2, 64, HF),
                                      positions[:0], first=1)
    assert none.shape == (0, 8, 64)
    c = caches[0]
    for bad in (dict(cache=FourBitCache(c[0], c[1], c[2], c[3].bfloat16())),
                dict(cache=FourBitCache(c[0][:, :, :3], c[1], c[2], c[3])),
                dict(cache=FourBitCache(c[0].transpose(1, 2), c[1], c[2], c[3])),
                dict(first=8), dict(positions=positions.int()), dict(scale=0.0),
                dict(valid=torch.ones(3, device="cuda", dtype=torch.bool)),
                dict(cache_valid=torch.ones(3, 7, device="cuda", dtype=torch.bool))):
        args = {**dict(cache=c, positions=positions, first=1), **bad}
        with pytest.raises(ValueError):
            window_attention_step_4bit(*parts, **args)
    with pytest.raises(RuntimeError):
        window_attention_step_4bit(*parts, FourBitCache(c[0].cpu(), *c[1:]), positions)


def test_positions_to_the_last():
    """The greatest position that there is counts a full cache, in both steps."""
    from gaussian_splats_b200.attention import (window_attention_step, window_attention_step_4bit,
                                                window_cache, window_cache_4bit)

    g = torch.Generator(device="cuda").manual_seed(11)
    last, first, left = 2 ** 63 - 1, 2, 40
    near = first + left + 1 + (last - first) % (left + 1)  # the same slot, the cache full too
    q = rand(g, 2, 4, 64, dtype=BF)
    k, v = (rand(g, 2, 2, 64, dtype=BF) for _ in range(2))
    results = []
    for place in (near, last):
        positions = torch.tensor([place, 5], device="cuda")
        four, whole = window_cache_4bit(2, left, first, 2, 64), window_cache(2, left, first, 2, 64)
        gen = torch.Generator(device="cuda").manual_seed(12)
        for t in (*four, *whole):
            t.copy_(torch.randint(0, 256, t.shape, generator=gen, device="cuda") if
                    t.dtype == torch.uint8 else torch.randn(t.shape, generator=gen, device="cuda"))
        results.append([window_attention_step_4bit(q, k, v, four, positions, first=first),
                        window_attention_step(q, k, v, *whole, positions, first=first), *four, *whole])
    assert all(torch.equal(a, b) for a, b in zip(*results)) and (results[0][0] != 0).any()


def test_values_of_the_whole_range():
    """Values next to bfloat16's limits, alone and among small ones, and rows without a
    spread: finite wherever the definition is."""
    from gaussian_splats_b200.attention import FourBitCache, window_attention_step_4bit

    g = torch.Generator(device="cuda").manual_seed(9)
    top = torch.finfo(BF).max
    sizes = [2.0 ** -126, 1e-30, 1.0, 1e30, 1e33, 1e36, 0.4 * top]
    for heads, kv_heads, dim, slots in ((4, 2, 64, 70), (16, 1, 128, 300), (3, 3, 40, 33)):
        batch = len(sizes) + 2
        v = 2.0 * torch.rand(batch, kv_heads, slots, dim, generator=g, device="cuda").double() - 1.0
        for b, size in enumerate(sizes):
            v[b] *= size
        v[-2] = 1e37  # no spread
        v[-1, :, ::2] *= 1e37  # large and small ones
        ref = R.Streams(batch, slots, 0, kv_heads, dim, BF, "cuda")
        for i, (x, kept) in enumerate(((rand(g, *v.shape, dtype=BF), ref.k), (v.to(BF), ref.v))):
            code, step, middle = R.held(x)
            ref.codes[i][:], ref.ranges[i][:] = R.packed(code), torch.stack((step, middle), -1)
            kept[:] = (code.double() - 7.5) * step.double()[..., None] + middle.double()[..., None]
        ref.seen[:] = True
        cache = FourBitCache(ref.codes[0].clone(), ref.ranges[0].clone(), ref.codes[1].clone(),
                             ref.ranges[1].clone())
        q = rand(g, batch, heads, dim, dtype=BF)
        k = rand(g, batch, kv_heads, dim, dtype=BF)
        positions = torch.full((batch,), 5 * slots + 2, device="cuda")
        out = window_attention_step_4bit(q, k, v[:, :, 1].to(BF), cache, positions)
        want = ref.step(q, k, v[:, :, 1].to(BF), positions, dim ** -0.5)
        for i, (codes, ranges) in enumerate((cache[:2], cache[2:])):
            assert torch.equal(codes, ref.codes[i]) and torch.equal(ranges, ref.ranges[i])
        assert out.isfinite().all()
        compare(out, want, BF, dim)


@pytest.mark.parametrize("side", ["keys", "values"])
def test_rows_of_the_whole_range(side):
    """A row whose greatest and least channel lie further apart than float32 reaches is
    held as the definition has it."""
    from gaussian_splats_b200.attention import window_attention_step_4bit, window_cache_4bit

    top = torch.finfo(BF).max
    wide = torch.stack([torch.linspace(-0.9, 0.9, 32).double() * top,
                        torch.tensor([-0.6 * top] * 31 + [0.6 * top]).double(),
                        torch.linspace(-1.0, 1.0, 32).double()]).to(BF).cuda()[:, None]
    one = torch.linspace(-1.0, 1.0, 32).to(BF).cuda().expand(3, 1, 32)
    k, v = (wide, one) if side == "keys" else (one, wide)
    cache = window_cache_4bit(3, 4, 0, 1, 32)
    ref = R.Streams(3, 5, 0, 1, 32, BF, "cuda")
    q = torch.zeros(3, 1, 32, device="cuda", dtype=BF)
    positions = torch.zeros(3, dtype=torch.int64, device="cuda")
    out = window_attention_step_4bit(q, k, v, cache, positions)
    want = ref.step(q, k, v, positions, 32 ** -0.5)
    for i, (codes, ranges) in enumerate((cache[:2], cache[2:])):
        assert torch.equal(codes, ref.codes[i]) and torch.equal(ranges, ref.ranges[i])
    compare(out, want, BF, 32)


@pytest.mark.parametrize("power", [-120, -64, 60, 64, 100, 112, 120, 126])
def test_queries_of_the_whole_range(power):
    """Queries of any size against keys of its inverse: the scores are those of 1 and 1."""
    from gaussian_splats_b200.attention import FourBitCache, window_attention_step_4bit

    g = torch.Generator(device="cuda").manual_seed(10)
    for heads, kv_heads, dim, slots in ((4, 2, 64, 70), (16, 1, 128, 300), (3, 3, 40, 33)):
        batch = 3
        q = (rand(g, batch, heads, dim, dtype=BF).clamp(-1.9, 1.9).double() * 2.0 ** power).to(BF)
        ref = R.Streams(batch, slots, 0, kv_heads, dim, BF, "cuda")
        fill(ref, g, BF, batch, kv_heads, slots, dim)
        keys = (rand(g, batch, kv_heads, slots, dim, dtype=BF).double() * 2.0 ** -power).to(BF)
        code, step, middle = R.held(keys)
        ref.codes[0][:], ref.ranges[0][:] = R.packed(code), torch.stack((step, middle), -1)
        ref.k[:] = (code.double() - 7.5) * step.double()[..., None] + middle.double()[..., None]
        cache = FourBitCache(ref.codes[0].clone(), ref.ranges[0].clone(), ref.codes[1].clone(),
                             ref.ranges[1].clone())
        k, v = keys[:, :, 0].contiguous(), rand(g, batch, kv_heads, dim, dtype=BF)
        positions = torch.full((batch,), 3 * slots + 2, device="cuda")
        out = window_attention_step_4bit(q, k, v, cache, positions)
        assert out.isfinite().all()
        compare(out, ref.step(q, k, v, positions, dim ** -0.5), BF, dim)


def test_large_queries_leave_their_groups_other_heads_alone():
    """A head whose scores leave float32's range, or whose query is not finite, has no
    finite output; the heads beside it have theirs, of large keys too."""
    from gaussian_splats_b200.attention import FourBitCache, window_attention_step_4bit

    g = torch.Generator(device="cuda").manual_seed(13)
    slots, heads, dim = 70, 12, 64
    for size in (2.0 ** 70, 2.0 ** 99, float("inf"), float("nan")):
        ref = R.Streams(1, slots, 0, 1, dim, BF, "cuda")
        fill(ref, g, BF, 1, 1, slots, dim)
        q = rand(g, 1, heads, dim, dtype=BF)
        many = 2.0 ** 66 if size < 2.0 ** 100 else 1.0
        keys = (rand(g, 1, 1, slots, dim, dtype=BF).double() * many).to(BF)
        code, step, middle = R.held(keys)
        ref.codes[0][:], ref.ranges[0][:] = R.packed(code), torch.stack((step, middle), -1)
        ref.k[:] = (code.double() - 7.5) * step.double()[..., None] + middle.double()[..., None]
        cache = FourBitCache(ref.codes[0].clone(), ref.ranges[0].clone(), ref.codes[1].clone(),
                             ref.ranges[1].clone())
        q = (q.double() / many).to(BF)
        q[:, 3] = size
        k, v = keys[:, :, 0].contiguous(), rand(g, 1, 1, dim, dtype=BF)
        positions = torch.full((1,), 3 * slots + 2, device="cuda")
        out = window_attention_step_4bit(q, k, v, cache, positions)
        others = torch.arange(heads, device="cuda") != 3
        want = ref.step(q[:, others], k, v, positions, dim ** -0.5)
        compare(out[:, others], want, BF, dim)
        assert not out[:, 3].isfinite().all() or size < 2.0 ** 100
