"""GPU tests of the rope operator against oracle/longctx_oracle.py (64 bits).

An output is a' = a c - b s in f32 with c and s rounded to f32 from 64 bits:
with |c|, |s| <= gain, two roundings of the factors, one of the product and one of
the fused sum, each 2^-24 of at most (|a| + |b|) * gain; the angle itself is off by
less than 2^-33 turns up to position 2^20. So ROUNDINGS * 2^-24 * (|a| + |b|) *
gain, and half a step of the type on top. Dims past the rotary part are equal.
"""
import numpy as np
import pytest

from oracle import longctx_oracle as L

pytestmark = pytest.mark.gpu

ROUNDINGS = 4
DTYPES = ("float32", "bfloat16", "float16")


def case(**kw):
    print("CASE", " ".join(f"{k}={v}" for k, v in kw.items()), flush=True)


@pytest.fixture(scope="module")
def env():
    import torch
    import engine_amd as E
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    return {"E": E, "ctx": E.AmdContext(0), "torch": torch}


def oracle(x, positions, spec):
    rotary = spec.rotary_dim or spec.head_dim
    turns, gain = L.rope_turns(rotary, spec.base, spec.scaling, spec.factor, spec.original_context, spec.beta_fast,
                               spec.beta_slow, spec.attention_factor, spec.freq_factors)
    return L.rope(x, positions, turns, gain, spec.layout), gain


def check(env, x, y, positions, spec):
    """y = rope(x), both [tokens][heads][dim] tensors."""
    torch = env["torch"]
    torch.cuda.synchronize()
    rotary = spec.rotary_dim or spec.head_dim
    xd, yd = x.double().cpu().numpy(), y.double().cpu().numpy()
    want, gain = oracle(xd, positions.cpu().numpy(), spec)
    n = rotary // 2
    a, b = (xd[..., :n], xd[..., n:rotary]) if spec.layout == "half" else (xd[..., 0:rotary:2], xd[..., 1:rotary:2])
    pair = (np.abs(a) + np.abs(b)) * gain
    size = np.zeros_like(want)
    if spec.layout == "half":
        size[..., :n] = size[..., n:rotary] = pair
    else:
        size[..., 0:rotary:2] = size[..., 1:rotary:2] = pair
    tol = ROUNDINGS * 2.0 ** -24 * size
    if x.dtype != torch.float32:
        tol = tol + (np.abs(want) + tol) * torch.finfo(x.dtype).eps / 2 + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    bad = np.abs(yd - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:3], np.abs(yd - want).max())
    assert torch.equal(y[..., rotary:], x[..., rotary:])


def rows(env, tokens, heads, dim, dtype, seed):
    torch = env["torch"]
    g = torch.Generator(device="cuda:0")
    g.manual_seed(seed)
    return torch.randn((tokens, heads, dim), device="cuda:0", generator=g).to(getattr(torch, dtype))


def positions(env, tokens, seed, far=131072):
    rng = np.random.default_rng(seed)
    return env["torch"].from_numpy(rng.integers(0, far, tokens).astype(np.int32)).to("cuda:0")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (128, 64), (64, 64), (80, 22), (96, 96), (256, 192), (2, 2), (4, 2), (1024, 1024), (130, 128), (128, 126),
                                        (1024, 2), (1022, 510)])
def test_layouts_and_sizes(env, dtype, layout, dim, rotary):
    case(test="sizes", dtype=dtype, layout=layout, dim=dim, rotary=rotary)
    E = env["E"]
    spec = E.AmdRopeSpec(head_dim=dim, rotary_dim=rotary, layout=layout, base=1.0e4)
    rope = E.AmdRope(env["ctx"], spec)
    for tokens, heads in ((1, 1), (1, 40), (3, 5), (33, 2), (200, 9)):
        x, pos = rows(env, tokens, heads, dim, dtype, tokens + heads), positions(env, tokens, tokens)
        y = env["torch"].full_like(x, 9.0)
        rope.execute(x, pos, y)
        check(env, x, y, pos, spec)


@pytest.mark.parametrize("kw", [dict(scaling="linear", factor=4.0), dict(scaling="yarn", factor=4.0, original_context=32768),
                                dict(scaling="yarn", factor=8.0, original_context=4096, attention_factor=1.3, rotary_dim=96),
                                dict(freq_factors=tuple(1.0 + 0.1 * i for i in range(64)))], ids=str)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_scalings(env, kw, layout):
    case(test="scalings", layout=layout)
    E = env["E"]
    spec = E.AmdRopeSpec(layout=layout, **kw)
    rope = E.AmdRope(env["ctx"], spec)
    x, pos = rows(env, 257, 3, 128, "float32", 1), positions(env, 257, 2)
    y = env["torch"].empty_like(x)
    rope.execute(x, pos, y)
    check(env, x, y, pos, spec)


def test_far_and_negative_positions(env):
    """Up to 2^20, and int32's ends: there an angle's 64-bit product is off by 2^31 *
    0.16 turns * 2^-53 = 3.8e-8 turns, 2.4e-7 radians, four more roundings."""
    case(test="far")
    E, torch = env["E"], env["torch"]
    spec = E.AmdRopeSpec()
    rope = E.AmdRope(env["ctx"], spec)
    pos = torch.tensor([0, 1, -1, -7, 1 << 20, (1 << 20) - 1, -(1 << 20), 999983], dtype=torch.int32, device="cuda:0")
    x = rows(env, 8, 4, 128, "float32", 3)
    y = torch.empty_like(x)
    rope.execute(x, pos, y)
    check(env, x, y, pos, spec)
    assert torch.equal(y[0], x[0])  # position 0: the identity
    ends = torch.tensor([2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda:0")
    rope.execute(x[:2], ends, y[:2])
    torch.cuda.synchronize()
    want, _ = oracle(x[:2].double().cpu().numpy(), ends.cpu().numpy(), spec)
    assert np.abs(y[:2].double().cpu().numpy() - want).max() <= 2 * float(x.abs().max()) * (2 * 2.4e-7 + ROUNDINGS * 2.0 ** -24)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides_and_places(env, dtype, layout):
    """Rows inside a fused projection, head-major rows, a broadcast input, starts
    that are not 16-byte aligned; in place and out of place; what lies between
    the rows stays as it is."""
    case(test="strides", dtype=dtype, layout=layout)
    E, torch = env["E"], env["torch"]
    spec = E.AmdRopeSpec(layout=layout, rotary_dim=96)
    rope = E.AmdRope(env["ctx"], spec)
    pos = positions(env, 37, 5)
    fused = rows(env, 37, 12, 128, dtype, 6)
    before = fused.clone()
    q, k = fused[:, :8], fused[:, 8:10]
    outs = [torch.empty((37, n, 128), dtype=fused.dtype, device="cuda:0") for n in (8, 2)]
    rope.execute_group([q, k], pos, outs)
    check(env, q, outs[0], pos, spec)
    check(env, k, outs[1], pos, spec)
    assert torch.equal(fused, before)
    rope.execute_group([q, k], pos, [q, k])  # in place
    torch.cuda.synchronize()
    assert torch.equal(q, outs[0]) and torch.equal(k, outs[1]) and torch.equal(fused[:, 10:], before[:, 10:])
    heads_first = rows(env, 5, 37, 128, dtype, 7)
    y = torch.empty_like(heads_first)
    rope.execute(heads_first.transpose(0, 1), pos, y.transpose(0, 1))
    check(env, heads_first.transpose(0, 1), y.transpose(0, 1), pos, spec)
    one = rows(env, 1, 3, 128, dtype, 8).expand(37, 3, 128)  # one row for every token
    y = torch.empty((37, 3, 128), dtype=one.dtype, device="cuda:0")
    rope.execute(one, pos, y)
    check(env, one, y, pos, spec)
    flat = torch.full((37 * 2 * 130 + 1,), 5.0, dtype=fused.dtype, device="cuda:0")
    view = flat[1:].view(37, 2, 130)[:, :, :128]  # odd start, odd strides
    view.copy_(rows(env, 37, 2, 128, dtype, 9))
    y = torch.empty((37, 2, 128), dtype=flat.dtype, device="cuda:0")
    rope.execute(view, pos, y)
    check(env, view, y, pos, spec)
    rope.execute(view, pos, view)
    torch.cuda.synchronize()
    assert torch.equal(view, y) and bool((flat[0] == 5.0).all()) and bool((flat[1:].view(37, 2, 130)[:, :, 128:] == 5.0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rotary", [(96, 42), (128, 14), (80, 68), (256, 2), (64, 62), (192, 190), (128, 6), (1024, 1022), (1024, 520)])
def test_rotary_parts_that_end_inside_a_piece(env, dtype, layout, dim, rotary):
    """Whole heads are in 16-byte pieces, the rotary part or its halves are not: three tensors of uneven heads
    out of a fused row, out of place and in place, the rest of the row as it was."""
    E, torch = env["E"], env["torch"]
    spec = E.AmdRopeSpec(head_dim=dim, rotary_dim=rotary, layout=layout, base=1.0e4)
    rope = E.AmdRope(env["ctx"], spec)
    for tokens, heads in ((1, (1, 1, 1)), (1, (40, 8, 3)), (7, (33, 1, 2)), (300, (9, 2, 1)), (1500, (3, 1, 1))):
        case(test="inside", dtype=dtype, layout=layout, dim=dim, rotary=rotary, tokens=tokens, heads=heads)
        fused, pos = rows(env, tokens, sum(heads) + 2, dim, dtype, tokens + heads[0]), positions(env, tokens, tokens)
        ends = np.cumsum(heads)
        parts = [fused[:, e - n:e] for e, n in zip(ends, heads)]
        outs = [torch.full((tokens, n, dim), 9.0, dtype=fused.dtype, device="cuda:0") for n in heads]
        rope.execute_group(parts, pos, outs)
        for x, y in zip(parts, outs):
            check(env, x, y, pos, spec)
        rest = fused[:, ends[-1]:].clone()
        rope.execute_group(parts, pos, parts)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(parts, outs)) and torch.equal(fused[:, ends[-1]:], rest)


def test_four_tensors_of_many_heads(env):
    case(test="four")
    E, torch = env["E"], env["torch"]
    spec = E.AmdRopeSpec(head_dim=64)
    rope = E.AmdRope(env["ctx"], spec)
    for tokens in (1, 2, 700):
        pos = positions(env, tokens, tokens)
        xs = [rows(env, tokens, h, 64, "bfloat16", h) for h in (1, 7, 128, 3)]
        ys = [torch.empty_like(x) for x in xs]
        rope.execute_group(xs, pos, ys)
        for x, y in zip(xs, ys):
            check(env, x, y, pos, spec)


def test_there_and_back(env):
    """Turning by p and then by -p gives the input back, whatever the layout."""
    case(test="back")
    E, torch = env["E"], env["torch"]
    for layout in ("half", "interleaved"):
        rope = E.AmdRope(env["ctx"], E.AmdRopeSpec(layout=layout, scaling="linear", factor=3.0))
        pos = positions(env, 100, 1)
        x = rows(env, 100, 4, 128, "float32", 2)
        y = torch.empty_like(x)
        rope.execute(x, pos, y)
        rope.execute(y, -pos, y)
        torch.cuda.synchronize()
        # two rotations: each within ROUNDINGS * 2^-24 * (|a| + |b|), |a| + |b| <= 2 max
        assert float((y - x).abs().max()) <= 2 * ROUNDINGS * 2.0 ** -24 * 2 * float(x.abs().max()) * 1.5


def test_values_that_are_not_finite_stay_in_their_pair(env):
    case(test="nonfinite")
    E, torch = env["E"], env["torch"]
    rope = E.AmdRope(env["ctx"], E.AmdRopeSpec(rotary_dim=64))
    x, pos = rows(env, 4, 2, 128, "float32", 2), positions(env, 4, 3)
    x[1, 0, 5] = float("nan")
    x[2, 1, 40] = float("inf")
    x[3, 0, 100] = float("nan")
    y = torch.empty_like(x)
    rope.execute(x, pos, y)
    torch.cuda.synchronize()
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    for t, h, dims in ((1, 0, (5, 37)), (2, 1, (8, 40)), (3, 0, (100,))):
        for d in dims:
            want[t, h, d] = True
    assert torch.equal(bad, want)


def test_captured_and_on_another_stream(env):
    case(test="capture")
    E, torch = env["E"], env["torch"]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = E.AmdContext(0, stream=stream)
        spec = E.AmdRopeSpec()
        rope = E.AmdRope(ctx, spec)
        x, pos = rows(env, 64, 8, 128, "float16", 2), positions(env, 64, 3)
        y = torch.empty_like(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            rope.execute(x, pos, y)
        for i in range(3):
            x.copy_(rows(env, 64, 8, 128, "float16", 10 + i))
            y.zero_()
            graph.replay()
            stream.synchronize()
            check(env, x, y, pos, spec)
            again = torch.empty_like(x)
            rope.execute(x, pos, again)
            stream.synchronize()
            assert torch.equal(again, y)


def test_a_rope_outlives_its_context(env):
    case(test="lifetime")
    E, torch = env["E"], env["torch"]
    ctx = E.AmdContext(0)
    spec = E.AmdRopeSpec()
    rope = E.AmdRope(ctx, spec)
    ctx.close()
    x, pos = rows(env, 4, 2, 128, "float32", 2), positions(env, 4, 3)
    y = torch.empty_like(x)
    rope.execute(x, pos, y)
    check(env, x, y, pos, spec)
    rope.close()
    rope.close()


def test_refusals(env):
    case(test="refusals")
    E, torch = env["E"], env["torch"]
    rope = E.AmdRope(env["ctx"], E.AmdRopeSpec())
    x, pos = rows(env, 4, 2, 128, "float32", 2), positions(env, 4, 3)
    y = torch.empty_like(x)

    def refused(kind, call):
        with pytest.raises(E.AmdModelKernelError) as e:
            call()
        assert e.value.kind == kind, str(e.value)

    refused("EmptyInput", lambda: rope.execute(x[:0], pos[:0], y[:0]))
    refused("InvalidArgument", lambda: rope.execute_group([], pos, []))
    refused("InvalidArgument", lambda: rope.execute_group([x] * 5, pos, [torch.empty_like(x) for _ in range(5)]))
    refused("InvalidArgument", lambda: rope.execute(x.cpu(), pos, y))
    refused("InvalidArgument", lambda: rope.execute(x, pos.cpu(), y))
    refused("InvalidArgument", lambda: rope.execute(x, pos, y[:1].expand(4, 2, 128)))               # rows that overlap
    refused("InvalidArgument", lambda: rope.execute(y[:2], pos[:2], y[:2].transpose(0, 1)))  # in place, other strides
    with pytest.raises(TypeError):
        rope.execute(x.double(), pos, y.double())
    with pytest.raises(TypeError):
        rope.execute(x, pos, y.half())
    with pytest.raises(TypeError):
        rope.execute(x, pos.long(), y)
    with pytest.raises(ValueError):
        rope.execute(x, pos[:3].contiguous(), y)
    with pytest.raises(ValueError):
        rope.execute(x[..., :64], pos, y[..., :64])
    with pytest.raises(ValueError):
        rope.execute(x, pos, y[:, :1])
    lib, name = env["ctx"]._lib, lambda st: E._lib.STATUS_NAMES[st]
    import ctypes

    def raw(tokens=4, dtype=0, **kw):
        r = E._lib.RopeRows(x.data_ptr(), 1024, 256, 128, y.data_ptr(), 1024, 256, 128, 2)
        for k, v in kw.items():
            setattr(r, k, v)
        return name(lib.ribn_amd_rope_execute(rope.handle, ctypes.c_void_p(pos.data_ptr()), tokens, ctypes.byref(r), 1, dtype))

    assert raw() == "Ok"
    assert raw(tokens=0) == "EmptyInput" and raw(heads=0) == "EmptyInput"
    assert raw(dtype=3) == "InvalidArgument"
    assert raw(input_len=1023) == "InputLength" and raw(output_len=1023) == "OutputLength"
    assert raw(tokens=1 << 32) == "ShapeOverflow" and raw(heads=70000) == "ShapeOverflow"
    assert raw(input_token_stride=1 << 63) == "ShapeOverflow"
    assert raw(output_head_stride=127) == "InvalidArgument" and raw(output_token_stride=128) == "InvalidArgument"
    assert raw(output=x.data_ptr(), output_token_stride=512, output_len=4096) == "InvalidArgument"  # in place, other strides
    assert raw(input=x.data_ptr() + 2) == "InvalidArgument"
    torch.cuda.synchronize()
