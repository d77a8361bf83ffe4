"""GPU tests of log probabilities, entropy and alternatives, through the public entry point, against
oracle/logprob_oracle.py (64 bits).

Tolerances. R, the sum beside the likeliest token, is of f32 terms 2^t: t = (x - M) log2 e is off by three roundings
of 2^-24 (difference, constant, product), so a term by 1.3e-7 |x - M| relatively, and by 2^-23 of the exponential; a
lane adds 16 terms, then up to 40 such sums (594 values a lane at 151,936 tokens, in 38 iterations): 54 roundings of
2^-24. With the terms' mean |x - M| under p at most 20 here: EPS = 1.3e-7 * 20 + 1.2e-7 + 54 * 6e-8 = 6e-6 at worst. Then log1p(R) is off by
EPS min(1, R), and a log probability by that and its own rounding to f32; the entropy, a sum of two positive terms each off
by at most 2 EPS of itself, by 2 EPS of itself (R in its denominator too) and a rounding. Tokens are equal."""
import ctypes

import numpy as np
import pytest

from oracle import logprob_oracle as P

pytestmark = pytest.mark.gpu

EPS = 6e-6
HALF_STEP = 2.0 ** -24


def case(**kw):
    print("CASE", " ".join(f"{k}={v}" for k, v in kw.items()), flush=True)


@pytest.fixture(scope="module")
def env():
    import torch
    import engine_amd as E
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    ctx = E.AmdContext(0)
    return {"E": E, "ctx": ctx, "ops": E.AmdQwenOps(ctx), "torch": torch}


def typed(env, x, dtype, pad=0, offset=0):
    """x [rows][n] on the device in `dtype`, in a wider buffer whose other values are +inf; and its values in 64 bits."""
    torch = env["torch"]
    rows, n = x.shape
    wide = torch.full((rows, offset + n + pad), float("inf"), dtype=getattr(torch, dtype))
    wide[:, offset:offset + n] = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(wide.dtype)
    wide = wide.to("cuda:0")
    view = wide[:, offset:offset + n]
    return view, view.double().cpu().numpy()


def run(env, logits, targets, top, ops=None):
    torch = env["torch"]
    rows = logits.shape[0]
    nan = lambda *s: torch.full(s, float("nan"), device="cuda:0")  # noqa: E731
    t = torch.from_numpy(np.asarray(targets, np.int64).astype(np.uint32).view(np.int32)).to("cuda:0")
    lp, h, ids, alt = nan(rows), nan(rows), torch.full((rows, top), -7, dtype=torch.int32, device="cuda:0"), nan(rows, top)
    (ops or env["ops"]).logprobs_into(logits, t, lp, h, ids if top else None, alt if top else None)
    torch.cuda.synchronize()
    return [v.cpu().numpy() for v in (lp, h, ids, alt)]


def check(got, x, targets, top):
    lp, h, ids, alt = got
    given, entropy, order, alternatives = P.logprobs(x, targets, top)
    np.testing.assert_array_equal(ids, order)
    first = P.logprobs(x, None, 1)[3][:, 0]
    rest = np.expm1(np.where(np.isfinite(first), -first, 0.0))  # R, of the likeliest token's -log1p(R)
    for have, want in ((lp, given), (alt, alternatives)):
        off = np.minimum(1.0, rest) * EPS
        off = off if have.ndim == 1 else off[:, None]
        finite = np.isfinite(want)
        np.testing.assert_array_equal(np.isfinite(have), finite)
        np.testing.assert_array_equal(have[~finite], want[~finite])
        err = np.abs(np.where(finite, have, 0) - np.where(finite, want, 0))
        bound = off + HALF_STEP * np.abs(np.where(finite, want, 0)) + 1e-37
        assert (err <= bound).all(), (err - bound).max()
    bound = (2 * EPS + HALF_STEP) * entropy + 1e-37
    assert (np.abs(h - entropy) <= bound).all(), (np.abs(h - entropy) - bound).max()


def bell(rng, rows, n, lift=24.0):
    x = 2.0 * rng.standard_normal((rows, n))
    at = rng.integers(0, n, rows)
    x[np.arange(rows), at] += lift * rng.random(rows)
    return x, np.where(rng.random(rows) < 0.7, at, rng.integers(0, n, rows))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("n", [1, 2, 3, 5, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 127, 255, 257, 1000, 1023, 1024, 1025, 4095, 4096, 4097, 8193,
                               32001, 151936])
def test_lengths(env, dtype, n):
    case(test="lengths", dtype=dtype, n=n)
    rng = np.random.default_rng(n)
    for rows in (1, 3, 5 if n > 30000 else 70):
        x, t = bell(rng, rows, n)
        view, values = typed(env, x, dtype)
        top = min(n, int(rng.choice([1, 5, 20, 32])))
        check(run(env, view, t, top), values, t, top)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("offset", [0, 1, 2, 3, 5, 7])
@pytest.mark.parametrize("pad", [0, 1, 6])
def test_rows_anywhere(env, dtype, offset, pad):
    """Rows of any alignment out of a wider buffer; what lies beside them is +inf."""
    case(test="anywhere", dtype=dtype, offset=offset, pad=pad)
    rng = np.random.default_rng(offset + 10 * pad)
    for rows, n in ((9, 5), (4, 13), (7, 1000), (3, 9001)):
        x, t = bell(rng, rows, n)
        view, values = typed(env, x, dtype, pad, offset)
        top = min(n, 7)
        check(run(env, view, t, top), values, t, top)


@pytest.mark.parametrize("rows,n", [(1, 151936), (8, 151936), (64, 40000), (257, 20011), (600, 5003), (1100, 4097), (2047, 301)])
@pytest.mark.parametrize("top", [0, 1, 20, 32])
def test_rows(env, rows, n, top):
    """One workgroup a row, and rows shared by several."""
    case(test="rows", rows=rows, n=n, top=top)
    rng = np.random.default_rng(rows)
    x, t = bell(rng, rows, n)
    x = x.astype(np.float32)
    view, values = typed(env, x, "float32")
    got = run(env, view, t, top)
    check(got, values, t, top)
    again = run(env, view, t, top)
    for a, b in zip(got, again):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("n", [40, 1025, 20000])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_orders_and_ties(env, n, dtype):
    """All alike, rising, falling, few distinct values, zeros of both signs, the best at the row's ends and in its
    last piece."""
    case(test="orders", n=n, dtype=dtype)
    rng = np.random.default_rng(n)
    x = np.zeros((9, n))
    x[1] = np.arange(n) / n * 20
    x[2] = -np.arange(n) / n * 20
    x[3] = rng.integers(0, 3, n)
    x[4] = np.where(rng.random(n) < 0.5, -0.0, 0.0)
    x[5, [0, n - 1]] = 9.0
    x[6, n - 1] = 9.0
    x[7, :: max(1, n // 30)] = 5.0
    x[8] = -1e4
    view, values = typed(env, x, dtype)
    t = rng.integers(0, n, 9)
    for top in (1, 20, 32):
        check(run(env, view, t, top), values, t, top)


@pytest.mark.parametrize("n", [33, 2000, 151936])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_masks_and_what_is_no_number(env, n, dtype):
    """Masks of -inf and of the type's lowest value, rows with nothing left, one token left, NaN, +inf."""
    case(test="masks", n=n, dtype=dtype)
    torch = env["torch"]
    rng = np.random.default_rng(n)
    low = float(torch.finfo(getattr(torch, dtype)).min)
    x = 2.0 * rng.standard_normal((14, n))
    x[0, rng.random(n) < 0.95] = -np.inf
    x[1, rng.random(n) < 0.95] = low
    x[2] = -np.inf
    x[3] = low
    x[4] = np.nan
    x[5] = -np.inf
    x[5, n // 2] = 1.5
    x[6, rng.random(n) < 0.5] = np.nan
    x[7, n - 1] = np.inf
    x[8, [3, n // 2, n - 1]] = np.inf
    x[9] = np.inf
    x[10, 0] = -np.inf
    x[11] = np.where(np.arange(n) % 2, np.nan, -np.inf)
    x[12, : n // 2], x[12, n // 2:] = -np.inf, np.where(rng.random(n - n // 2) < 0.5, np.inf, low)
    x[13] = np.where(rng.random(n) < 0.3, 6e4, low)
    view, values = typed(env, x, dtype)
    t = rng.integers(0, n, 14)
    t[5] = n // 2
    t[7] = n - 1
    for top in (0, 1, 20, 32):
        check(run(env, view, t, top), values, t, top)


def test_signaling_nans(env):
    case(test="signaling")
    torch = env["torch"]
    rng = np.random.default_rng(2)
    x = (2.0 * rng.standard_normal((4, 3000))).astype(np.float32)
    bits = x.view(np.uint32)
    bits[0, 5::7] = 0x7f800001
    bits[1, 1::3] = 0xff812345
    bits[2] = 0x7fa00000
    bits[3, [0, 1, 2, 2999]] = 0x7f800001
    view = torch.from_numpy(bits.view(np.int32)).to("cuda:0").view(torch.float32)
    t = [5, 0, 7, 100]
    check(run(env, view, t, 20), x.astype(np.float64), t, 20)


def test_the_top_moves_far(env):
    """A largest logit that moves by more than f32's exponents, at the row's end too, among values of 1e30."""
    case(test="far")
    rng = np.random.default_rng(5)
    x = rng.standard_normal((6, 30000))
    x[0, 25000:] += 200.0
    x[1, ::2] = -1.5e38
    x[1, 29999] = 1.5e38
    x[2] *= 1e30
    x[3] = np.linspace(-5000, 5000, 30000)
    x[4, 4096:8192] = 1000.0
    x[5] = 1e-40 * rng.integers(-5, 6, 30000)
    view, values = typed(env, x, "float32")
    t = rng.integers(0, 30000, 6)
    check(run(env, view, t, 32), values, t, 32)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_lowest_after_nothing(env, dtype):
    """A row of nothing but -inf for long, then of its type's lowest value only, one token or many."""
    case(test="lowest_after_nothing", dtype=dtype)
    torch = env["torch"]
    low = float(torch.finfo(getattr(torch, dtype)).min)
    x = np.full((4, 60000), -np.inf)
    x[0, 55001], x[1, 59999] = low, low
    x[2, 40000:], x[3, 40000::3] = low, low / 2
    view, values = typed(env, x, dtype)
    for top in (0, 1, 20):
        check(run(env, view, [55001, 59999, 50000, 1], top), values, [55001, 59999, 50000, 1], top)


def test_very_many_rows(env):
    """More rows than a grid's 32-bit count of threads has room for, two tokens each: log p by the logits' difference."""
    case(test="very_many_rows")
    torch = env["torch"]
    rows = 2 ** 24 + 5
    g = torch.Generator(device="cuda:0").manual_seed(3)
    x = (4 * torch.randn((rows, 2), device="cuda:0", generator=g)).half()
    t = torch.randint(0, 3, (rows,), device="cuda:0", generator=g, dtype=torch.int32)  # 2: outside
    lp, h = (torch.full((rows,), 7.0, device="cuda:0") for _ in range(2))
    ids, alt = torch.full((rows, 1), -7, dtype=torch.int32, device="cuda:0"), torch.full((rows, 1), 7.0, device="cuda:0")
    env["ops"].logprobs_into(x, t, lp, h, ids, alt)
    torch.cuda.synchronize()
    d = x[:, 0].double() - x[:, 1].double()
    both = torch.stack((-torch.log1p(torch.exp(-d)), -torch.log1p(torch.exp(d))), 1)
    want = torch.where(t == 0, both[:, 0], torch.where(t == 1, both[:, 1], torch.full_like(d, -float("inf"))))
    inside = t < 2
    assert torch.isinf(lp[~inside]).all()
    rest = torch.expm1(-both.max(1)[0])
    off = EPS * torch.clamp(rest, max=1.0) + HALF_STEP * want.abs()
    assert ((lp.double() - want)[inside].abs() <= off[inside]).all()
    assert torch.equal(ids[:, 0], (d < 0).int())
    assert ((alt[:, 0].double() - both.max(1)[0]).abs() <= EPS * torch.clamp(rest, max=1.0) + HALF_STEP * both.max(1)[0].abs()).all()
    entropy = -(both * torch.exp(both)).sum(1)
    assert ((h.double() - entropy).abs() <= (2 * EPS + HALF_STEP) * entropy).all()


def test_certain_models(env):
    """Log probabilities and entropies near 0 keep their digits."""
    case(test="certain")
    rng = np.random.default_rng(6)
    for gap in (10.0, 16.0, 20.0, 30.0, 60.0):
        x = rng.standard_normal((3, 50000))
        x[:, 777] = gap + 12.0
        view, values = typed(env, x, "float32")
        check(run(env, view, [777] * 3, 2), values, [777] * 3, 2)


def test_tokens_outside_the_vocabulary(env):
    case(test="outside")
    rng = np.random.default_rng(7)
    x, _ = bell(rng, 5, 1001)
    view, values = typed(env, x, "bfloat16", 3)
    t = np.array([1000, 1001, 0xffffffff, 0x80000000, 0])
    got = run(env, view, t, 3)
    check(got, values, t, 3)
    assert list(np.isinf(got[0])) == [False, True, True, True, False]


def test_each_result_alone(env):
    """Whatever is asked for, it has the bits it has among the others."""
    case(test="alone")
    torch, ops = env["torch"], env["ops"]
    rng = np.random.default_rng(8)
    for rows in (3, 1500):
        x, t = bell(rng, rows, 9000 if rows == 3 else 600)
        view, values = typed(env, x, "float32")
        want = run(env, view, t, 8)
        td = torch.from_numpy(t.astype(np.int32)).to("cuda:0")
        a, b = torch.zeros(rows, device="cuda:0"), torch.zeros(rows, device="cuda:0")
        ids, alt = torch.zeros((rows, 8), dtype=torch.int32, device="cuda:0"), torch.zeros((rows, 8), device="cuda:0")
        ops.logprobs_into(view, td, a)
        ops.logprobs_into(view, entropy=b)
        ops.logprobs_into(view, top_tokens=ids, top_logprobs=alt)
        torch.cuda.synchronize()
        for have, w in zip((a, b, ids, alt), want):
            np.testing.assert_array_equal(have.cpu().numpy(), w)
    one = run(env, view[:1], t[:1], 8)  # a row of its own, by several workgroups
    np.testing.assert_allclose(one[0], want[0][:1], rtol=1e-5)


# ------------------------------------------------- streams, graphs, several at once

def test_captured_calls_replay(env):
    """Captured and replayed between eager work: every replay gives the eager call's bits; new logits in the same
    buffer give theirs."""
    case(test="capture")
    E, torch = env["E"], env["torch"]
    stream = torch.cuda.Stream()
    ctx = E.AmdContext(0, stream=stream)
    ops = E.AmdQwenOps(ctx)
    rng = np.random.default_rng(9)
    sets = [bell(rng, 4, 50001) for _ in range(3)]
    with torch.cuda.stream(stream):
        x = torch.zeros((4, 50001), device="cuda:0")
        t = torch.zeros(4, dtype=torch.int32, device="cuda:0")
        out = [torch.zeros(4, device="cuda:0"), torch.zeros(4, device="cuda:0"), torch.zeros((4, 20), dtype=torch.int32, device="cuda:0"),
               torch.zeros((4, 20), device="cuda:0")]

        def put(i):
            x.copy_(torch.from_numpy(sets[i][0].astype(np.float32)))
            t.copy_(torch.from_numpy(sets[i][1].astype(np.int32)))

        put(0)
        ops.logprobs_into(x, t, *out)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.logprobs_into(x, t, *out)
        for i in (0, 1, 2, 1):
            put(i)
            for v in out:
                v.zero_()
            ops.logprobs_into(x, t, *out)
            stream.synchronize()
            want = [v.clone() for v in out]
            for v in out:
                v.zero_()
            graph.replay()
            stream.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b), i
            check([v.cpu().numpy() for v in out], x.double().cpu().numpy(), sets[i][1], 20)
    ctx.synchronize()


def test_two_contexts_at_once(env):
    case(test="two_contexts")
    E, torch = env["E"], env["torch"]
    rng = np.random.default_rng(10)
    lanes = []
    for i in range(2):
        ctx = E.AmdContext(0, stream=torch.cuda.Stream())
        x, t = bell(rng, 3, 60000)
        view, values = typed(env, x, "float16")
        lanes.append((E.AmdQwenOps(ctx), view, values, t))
    torch.cuda.synchronize()
    outs = []
    for _ in range(6):
        for ops, view, values, t in lanes:
            td = torch.from_numpy(t.astype(np.int32)).to("cuda:0")
            out = [torch.zeros(3, device="cuda:0"), torch.zeros(3, device="cuda:0"), torch.zeros((3, 9), dtype=torch.int32, device="cuda:0"),
                   torch.zeros((3, 9), device="cuda:0")]
            torch.cuda.synchronize()
            outs.append((ops, view, values, t, td, out))
    for ops, view, values, t, td, out in outs:
        ops.logprobs_into(view, td, *out)
    torch.cuda.synchronize()
    for ops, view, values, t, td, out in outs:
        check([v.cpu().numpy() for v in out], values, t, 9)


# ----------------------------------------------------------------------- refusals

def test_refusals(env):
    case(test="refusals")
    E, torch, ctx, ops = env["E"], env["torch"], env["ctx"], env["ops"]
    x = torch.zeros((3, 40), device="cuda:0")
    t, lp = torch.zeros(3, dtype=torch.int32, device="cuda:0"), torch.zeros(3, device="cuda:0")
    ids, alt = torch.zeros((3, 40), dtype=torch.int32, device="cuda:0"), torch.zeros((3, 40), device="cuda:0")

    def refused(kind, call):
        with pytest.raises(E.AmdModelKernelError) as e:
            call()
        assert e.value.kind == kind, str(e.value)

    refused("InvalidArgument", lambda: ops.logprobs_into(x))
    refused("InvalidArgument", lambda: ops.logprobs_into(x, t))
    refused("InvalidArgument", lambda: ops.logprobs_into(x, None, lp))
    refused("InvalidArgument", lambda: ops.logprobs_into(x, t, lp, None, ids[:, :5].contiguous()))
    refused("InvalidArgument", lambda: ops.logprobs_into(x, t, lp, None, ids, alt))                       # 40 > 32
    refused("InvalidArgument", lambda: ops.logprobs_into(x[:, :4], t, lp, None, ids[:, :5].contiguous(), alt[:, :5].contiguous()))
    refused("EmptyInput", lambda: ops.logprobs_into(x[:0], t[:0], lp[:0]))
    refused("EmptyInput", lambda: ops.logprobs_into(x[:, :0], t, lp))
    refused("InputLength", lambda: ops.logprobs_into(x[:1].expand(3, 40), t, lp))
    refused("InvalidArgument", lambda: ops.logprobs_into(x.cpu(), t, lp))
    refused("InvalidArgument", lambda: ops.logprobs_into(x, t.cpu(), lp))
    lib = ctx._lib
    name = lambda st: E._lib.STATUS_NAMES[st]  # noqa: E731
    p = lambda v, by=0: ctypes.c_void_p(v.data_ptr() + by)  # noqa: E731

    def call(logits=p(x), n=120, rows=3, length=40, stride=40, dtype=0, targets=p(t), out=p(lp)):
        return name(lib.ribn_amd_logprobs(ctx.handle, logits, n, rows, length, stride, dtype, targets, out, None, None, None, 0))

    assert call() == "Ok"
    assert call(dtype=3) == "InvalidArgument"
    assert call(n=119) == "InputLength"
    assert call(stride=39) == "InputLength"
    assert call(length=1 << 32, stride=1 << 32) == "ShapeOverflow"
    assert call(rows=1 << 32) == "ShapeOverflow"
    assert call(logits=None) == "InvalidArgument"
    assert call(logits=p(x, 2)) == "InvalidArgument"
    assert call(out=p(lp, 2)) == "InvalidArgument"
    assert call(logits=p(x, 2), dtype=1, n=239) == "Ok"
    env["torch"].cuda.synchronize()


@pytest.mark.parametrize("rows,n", [(6, 12300), (64, 100003), (520, 12300)])
def test_the_top_crosses_two_to_the_sixteen(env, rows, n):
    """Rows whose largest logit so far passes 65,536 or -65,536 by little, while many tokens lie at what it was before:
    one workgroup a row and several, one iteration of a wave and more. Each of at most six moves scales the sums by a factor
    off by 2^-23 and two roundings, 1.8e-6 in all, and |x - M| is 3 at most (4e-7): within EPS."""
    case(test="crosses", rows=rows, n=n)
    rng = np.random.default_rng(n)
    at = np.arange(n)
    x = np.zeros((rows, n))
    for r in range(rows):
        low, high = [(65535.5, 65536.0), (-65536.5, -65535.5), (65535.0, 65537.0), (-65537.0, -65534.5)][r % 4]
        kind = (r // 4) % 5
        if kind == 0:    # the last token alone
            x[r] = np.where(at == n - 1, high, low)
        elif kind == 1:  # halves
            x[r] = np.where(at < n // 2, low, high)
        elif kind == 2:  # 4,096 tokens in turn, as a workgroup takes them
            x[r] = np.where(at // 4096 % 2, high, low)
        elif kind == 3:  # in four steps
            x[r] = low + (high - low) / 4 * (5 * at // n)
        else:            # among others, over the border and back
            x[r] = np.where(at // 4096 % 2, high, low) - rng.integers(0, 64, n) / 64
    view, values = typed(env, x, "float32")
    np.testing.assert_array_equal(values, x)
    t = rng.integers(0, n, rows)
    for top in (0, 5):
        check(run(env, view, t, top), values, t, top)


@pytest.mark.parametrize("n", [3000, 20000])
@pytest.mark.parametrize("gap", [50, 65, 80, 86])
def test_far_runners_up_keep_their_digits(env, n, gap):
    """One token `gap` nats below the likeliest and no other: log p of the likeliest is -R = -2^t, t = (x - M) log2 e, with
    M = 0 and t all but free of rounding (x is chosen so), which leaves the exponential's last place (2^-23), log1p's two
    and R's rounding to f32: 3 * 2^-23 + 2^-24 = 4.2e-7 of it at any gap. The entropy (1 + gap) R: the same and
    its own rounding."""
    case(test="runner_up", n=n, gap=gap)
    rng = np.random.default_rng(gap)
    log2e = np.float64(np.float32(1.44269504088896341))
    x = -(gap + rng.random(40000)).astype(np.float32)
    exact = x.astype(np.float64) * log2e  # (48 bits)
    best = np.argsort(np.abs(exact.astype(np.float32).astype(np.float64) - exact), kind="stable")[:12]
    x = x[best].astype(np.float64)
    assert (np.abs((x * log2e).astype(np.float32) - x * log2e) < 2.0 ** -27).all()
    rows = np.full((12, n), -1000.0)
    rows[:, n // 3] = 0.0
    rows[np.arange(12), rng.permutation(n // 3)[:12]] = x
    view, values = typed(env, rows, "float32")
    lp, h, _, _ = run(env, view, [n // 3] * 12, 2)
    want = np.log1p(np.exp(x))
    print("CASE off", float(np.abs(-lp / want - 1).max()), float(np.abs(h / (want - x * np.exp(x) / (1 + np.exp(x))) - 1).max()))
    bound = 3 * 2.0 ** -23 + 2.0 ** -24 + 2.0 ** -27
    assert (np.abs(-lp.astype(np.float64) - want) <= bound * want).all()
    entropy = want - x * np.exp(x) / (1 + np.exp(x))
    assert (np.abs(h - entropy) <= (bound + 2.0 ** -24) * entropy).all()
