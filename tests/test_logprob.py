"""CPU tests of the log-probability operator: its oracle against the plain definition, and the
checks its Python entry point makes before the library is called."""
import ctypes

import numpy as np
import pytest

import engine_amd as E
from engine_amd import _lib
from oracle import logprob_oracle as P


def test_oracle_is_the_definition():
    rng = np.random.default_rng(0)
    x = 3 * rng.standard_normal((5, 300))
    x[1, :250] = -np.inf
    x[2] = 0.0
    x[3, 7] = 60.0
    targets = [3, 260, 299, 7, 0]
    p = np.exp(x) / np.exp(x).sum(1, keepdims=True)
    given, entropy, order, alt = P.logprobs(x, targets, 12)
    np.testing.assert_allclose(given[:3], np.log(p[np.arange(5), targets])[:3], rtol=1e-13)
    with np.errstate(divide="ignore", invalid="ignore"):
        want = -np.where(p > 0, p * np.log(p), 0.0).sum(1)
    np.testing.assert_allclose(entropy, want, rtol=1e-9, atol=1e-12)
    assert list(order[2]) == list(range(12))                       # ties: the lowest token first
    assert order[1].min() >= 250 and (np.diff(alt, axis=1) <= 0).all()
    # a certain row's log probability is the others' share
    assert abs(given[3] / -(np.exp(np.delete(x[3], 7) - 60.0).sum()) - 1) < 1e-9


def test_oracle_at_the_edges():
    inf, nan = np.inf, np.nan
    x = np.array([[nan, 1.0, -inf, 1.0], [-inf, -inf, nan, -inf], [inf, 3.0, inf, nan], [5.0, nan, nan, -inf]])
    given, entropy, order, alt = P.logprobs(x, [0, 1, 2, 0xffffffff], 4)
    np.testing.assert_allclose(entropy, [np.log(2), 0, np.log(2), 0], atol=1e-15)
    np.testing.assert_array_equal(given, [-inf, -inf, -np.log(2), -inf])
    assert [list(o) for o in order] == [[1, 3, 0, 2], [0, 1, 2, 3], [0, 2, 1, 3], [0, 1, 2, 3]]
    np.testing.assert_allclose(alt[0], [-np.log(2), -np.log(2), -inf, -inf])


class FakeLib:
    def __init__(self):
        self.calls = []

    def ribn_amd_logprobs(self, *args):
        self.calls.append(args)
        return 0


class FakeCtx:
    def __init__(self):
        self._lib = FakeLib()
        self.handle = ctypes.c_void_p(1)


def test_python_checks():
    import torch
    ctx = FakeCtx()
    ops = E.AmdQwenOps(ctx)
    x = torch.zeros((3, 40))
    t, lp, ids, alt = torch.zeros(3, dtype=torch.int32), torch.zeros(3), torch.zeros((3, 5), dtype=torch.int32), torch.zeros((3, 5))
    ops.logprobs_into(x[:, 2:33], t, lp, lp.clone(), ids, alt)
    (handle, data, length, rows, n, stride, dtype, *ptrs, top), = ctx._lib.calls
    assert (length, rows, n, stride, dtype, top) == (3 * 40 - 2, 3, 31, 40, 0, 5) and data == x.data_ptr() + 8 and all(ptrs)
    for kind, code in ((torch.bfloat16, 1), (torch.float16, 2)):
        ops.logprobs_into(x.to(kind), t, lp)
        assert ctx._lib.calls[-1][6] == code and ctx._lib.calls[-1][9:] == (None, None, None, 0)
    ops.logprobs_into(x[0], t[:1], lp[:1], None, ids[0], alt[0])  # one row
    assert ctx._lib.calls[-1][3:6] == (1, 40, 40)
    n = len(ctx._lib.calls)
    for bad in (lambda: ops.logprobs_into(x.double(), t, lp), lambda: ops.logprobs_into(x, t.long(), lp), lambda: ops.logprobs_into(x, t, lp.double()),
                lambda: ops.logprobs_into(x, t, lp, lp.half()), lambda: ops.logprobs_into(x, t, lp, None, alt, alt), lambda: ops.logprobs_into(x, t, lp, None, ids, ids)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: ops.logprobs_into(x.t(), t, lp), lambda: ops.logprobs_into(x[None], t, lp), lambda: ops.logprobs_into(x, t[:2], lp),
                lambda: ops.logprobs_into(x, t, torch.zeros(6)[::2]), lambda: ops.logprobs_into(x, t, lp, None, ids, alt[:, :4]),
                lambda: ops.logprobs_into(x, t, lp, None, ids[:2], alt)):
        with pytest.raises(ValueError):
            bad()
    assert len(ctx._lib.calls) == n


def test_no_context_is_refused():
    lib = _lib.load()
    assert _lib.STATUS_NAMES[lib.ribn_amd_logprobs(None, None, 0, 0, 0, 0, 0, None, None, None, None, None, 0)] == "InvalidArgument"


def test_no_decoder_is_refused():
    lib = _lib.load()
    one, out = (ctypes.c_uint32 * 1)(0), (ctypes.c_float * 1)()
    for status in (lib.ribn_amd_qwen3_logprobs(None, 1, None, out, None, None, None, 0),
                   lib.ribn_amd_qwen3_score_prompt(None, None, one, 1, 0, 0, one, out, None, None, None, 0)):
        assert _lib.STATUS_NAMES[status] == "InvalidArgument"
    assert out[0] == 0.0


class FakeDecoder(E.AmdQwen3Decode):
    def __init__(self):
        self.ctx, self.config, self.handle = FakeCtx(), E.AmdQwen3Config(vocab=40), ctypes.c_void_p(0)


def test_python_checks_of_a_decoder():
    dec, cache = FakeDecoder(), FakeCtx()
    for bad in (lambda: dec.logprobs(2, targets=[1]), lambda: dec.logprobs(1, top=41), lambda: dec.logprobs(1, top=-1),
                lambda: dec.score_prompt(cache, [1, 2, 3], 0, [2, 3]), lambda: dec.score_prompt(cache, [1], 0, [1], top=41),
                lambda: dec.score_prompt(cache, [1], 0, top=-1)):
        with pytest.raises(ValueError):
            bad()


class Recorder(FakeDecoder):
    """Host tokens as the library is given them."""

    def __init__(self):
        super().__init__()
        self.seen = []

        def words(at, n):
            return None if at is None else list((ctypes.c_uint32 * n).from_address(at))

        def score(handle, cache, tokens, count, position, chunk, targets, *rest):
            self.seen.append((words(tokens, count), words(targets, count)))
            return 0

        def step(handle, members, targets, *rest):
            self.seen.append(words(targets, members))
            return 0

        self.ctx._lib.ribn_amd_qwen3_score_prompt, self.ctx._lib.ribn_amd_qwen3_logprobs = score, step


OUTSIDE = [-1, -100, 2 ** 32 + 5, 2 ** 32, 40, -2 ** 32 + 3, 2 ** 32 - 1]


@pytest.mark.parametrize("as_", [list, tuple, lambda x: np.array(x, np.int64)], ids=("list", "tuple", "int64"))
def test_tokens_outside_32_bits(as_):
    """A target outside the vocabulary, -1 among them, has no probability: it must not become a token by its lower 32
    bits. A prompt's own token outside it reaches the library as one that it refuses."""
    dec, cache = Recorder(), FakeCtx()
    goal = as_([3, 39] + OUTSIDE)
    dec.score_prompt(cache, [1] * 9, 0, goal)
    (tokens, targets), = dec.seen
    assert tokens == [1] * 9 and targets[:2] == [3, 39] and min(targets[2:]) >= 40
    dec.logprobs(9, goal)
    assert dec.seen[1][:2] == [3, 39] and min(dec.seen[1][2:]) >= 40
    for bad in OUTSIDE:
        dec.score_prompt(cache, as_([1, bad, 2]), 0, [1, 2, 3])
        assert dec.seen[-1][0][::2] == [1, 2] and dec.seen[-1][0][1] >= 40


def test_tokens_are_whole_numbers():
    dec, cache = Recorder(), FakeCtx()
    for bad in (lambda: dec.score_prompt(cache, [1, 2], 0, [1.5, 2.0]), lambda: dec.logprobs(1, [0.5]), lambda: dec.score_prompt(cache, [1.5], 0, [1])):
        with pytest.raises(TypeError):
            bad()
    assert not dec.seen
    for kind in (np.int8, np.uint8, np.int32, np.uint32, np.int64, np.uint64):
        dec.score_prompt(cache, np.array([1, 2], kind), 0, np.array([3, 4], kind))
        assert dec.seen[-1] == ([1, 2], [3, 4])
    dec.score_prompt(cache, [], 0, [])
    assert dec.seen[-1] == ([], [])
