"""GPU tests of log probabilities, entropies and likeliest tokens against float64.

Tolerance.  Probabilities, sums and logarithms are float64 and rounded to f32
once: half a step, 2^-24 of the value; the float64 part is within 2^-40 of
max(1, |value|) (sums of 2^18 terms of 2^-51 (|y| + 2) each, a logarithm), which
counts near a log probability of 0, and 2^-149 more for numbers below f32's
normal ones.  Token ids are exact."""
import math
import sys

import numpy as np
import pytest

import paged_refs as ref
from atlas_amd import OperatorError

pytestmark = pytest.mark.gpu
f32, u32 = np.float32, np.uint32


def say(msg):
    print(f"[gpu-logprobs] {msg}", flush=True)
    sys.stdout.flush()


def run(rt, logits, vocab, tokens, inv, top, entropy=True):
    """logits [rows, stride]."""
    R, stride = logits.shape
    given = tokens.shape[1]
    dl, dt = rt.upload(logits), rt.upload(tokens) if given else None
    lp, en = rt.upload(np.full((R, max(given, 1)), 7, f32)), rt.upload(np.full(R, 7, f32))
    ids, tp = rt.upload(np.full((R, max(top, 1)), 7, u32)), rt.upload(np.full((R, max(top, 1)), 7, f32))
    n = rt.token_logprobs_workspace(R, vocab, top)
    ws = rt.alloc(n + 256)
    rt.memset(ws, 0xFF, n + 256)
    rt.token_logprobs(dl, stride, dt, given, lp if given else None, en if entropy else None, ids if top else None,
                      tp if top else None, R, vocab, top, inv, ws, n)
    rt.sync()
    assert (ws.download(n + 256, np.uint8)[n:] == 0xFF).all(), "wrote behind the workspace"
    got = (lp.download(R * max(given, 1)).reshape(R, -1)[:, :given], en.download(R), ids.download(R * max(top, 1)).reshape(R, -1)[:, :top],
           tp.download(R * max(top, 1)).reshape(R, -1)[:, :top])
    for b in (dl, lp, en, ids, tp, ws) + ((dt,) if given else ()):
        rt.free(b)
    return got


def close(name, got, exp):
    same = np.isinf(exp) | np.isinf(got)
    assert np.array_equal(got[same], exp[same].astype(f32)), name
    off = np.abs(got[~same].astype(np.float64) - exp[~same])
    tol = np.abs(exp[~same]) * 2.0 ** -24 + np.maximum(1.0, np.abs(exp[~same])) * 2.0 ** -40 + 2.0 ** -149
    assert (off <= tol).all(), f"{name}: {float((off / tol).max()):.3f} of the tolerance"


def check(rt, name, logits, vocab, tokens, inv, top):
    say(name)
    got = run(rt, logits, vocab, tokens, inv, top)
    exp = ref.logprobs(logits[:, :vocab], tokens, inv, top)
    assert np.array_equal(got[2], exp[2]), f"{name}: ids differ in rows {np.nonzero((got[2] != exp[2]).any(1))[0][:5]}"
    for what, g, e in (("logprobs", got[0], exp[0]), ("entropy", got[1], exp[1]), ("tops", got[3], exp[3])):
        close(f"{name}: {what}", g, e)


def rows(seed, R, stride, std=4.0):
    return (np.random.default_rng(seed).standard_normal((R, stride)) * std).astype(f32)


@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
@pytest.mark.parametrize("R,vocab,pad", [(1, 1, 0), (3, 2, 1), (2, 63, 0), (5, 64, 0), (2, 1000, 3), (3, 1023, 0), (3, 1024, 0),
                                         (3, 1025, 0), (2, 4097, 0), (2, 8191, 2), (1, 49152, 0), (4, 50257, 47), (3, 32001, 0),
                                         (2, 262144, 0), (300, 1500, 1)])
def test_rows_of_all_lengths(rt, R, vocab, pad, top):
    x = rows(vocab, R, vocab + pad)
    if pad:
        x[:, vocab:] = np.nan  # behind a row: anything
    tokens = np.random.default_rng(R).integers(0, vocab, (R, 3)).astype(u32)
    tokens[:, 1] = x[:, :vocab].argmax(1)
    check(rt, f"{R} x {vocab} + {pad}, {top}", x, vocab, tokens, 1.0 / 0.8, top)


@pytest.mark.parametrize("top", [5, 64])
@pytest.mark.parametrize("kind", ["equal", "two_values", "few_values", "rising", "falling", "block", "zeros"])
def test_ties_and_orders(rt, kind, top):
    """Equal logits: the lowest tokens; the likeliest ones all in one place."""
    for vocab in (700, 5000, 150001):
        x = rows(5, 3, vocab)
        at = np.arange(vocab)
        if kind == "equal":
            x[:] = 2.5
        elif kind == "two_values":
            x[:] = np.where(at % 3 == 1, 1.0, -1.0)
        elif kind == "few_values":
            x = np.round(x)
        elif kind == "rising":
            x[:] = at * 1e-3
        elif kind == "falling":
            x[:] = at * -1e-3
        elif kind == "block":
            x[:, vocab // 2:vocab // 2 + 600] += 50
        else:
            x[:] = np.where(at % 2, 0.0, -0.0)
        tokens = np.random.default_rng(1).integers(0, vocab, (3, 2)).astype(u32)
        check(rt, f"{kind} {vocab}, {top}", x, vocab, tokens, 1.0, top)


def test_infinite_and_missing_logits(rt):
    """-inf, NaN, the lowest number, +inf; rows of nothing; fewer tokens than asked for; tokens out of range."""
    huge = np.finfo(f32).min
    for vocab in (50, 3000, 20000):
        x = rows(9, 12, vocab)
        x[0] = -np.inf
        x[1] = np.nan
        x[2, :] = -np.inf
        x[2, vocab - 2] = -3.0
        x[3, 1:] = np.nan
        x[4, ::2] = -np.inf
        x[5, 3] = np.inf
        x[6, [3, 17, vocab - 1]] = np.inf
        x[7] = huge
        x[8, 5:] = huge
        x[9] = np.nan
        x[9, 7] = np.inf
        x[10, :] = -np.inf
        x[10, 10:40:3] = 1.5
        x[11] = np.finfo(f32).max
        tokens = np.array([[3, 17, vocab - 2, vocab, ref.NO]] * 12, u32)
        for top in (1, 20, 64):
            check(rt, f"{vocab}, {top}", x, vocab, tokens, 1.0, top)


@pytest.mark.parametrize("inv", [1e-6, 1.0, 1.0 / 0.3, 1e4, 1.7e308, 5e-324])
def test_temperatures(rt, inv):
    x = rows(3, 4, 9000)
    x[1, 77] = x[1].max()
    x[2] = 0.25
    tokens = np.argsort(-x, 1)[:, :4].astype(u32)
    got = run(rt, x, 9000, tokens, inv, 6)
    exp = ref.logprobs(x, tokens, inv, 6)
    with np.errstate(over="ignore"):
        for g, e in ((got[0], exp[0]), (got[1], exp[1]), (got[3], exp[3])):
            close(f"inv {inv}", g, e.astype(f32).astype(np.float64) if np.isinf(e.astype(f32)).any() else e)
    assert np.array_equal(got[2], exp[2])


@pytest.mark.parametrize("inv", [1e20, 1e30, 1e39, 1e46, 1e60, 1e300])
def test_cold_rows_around_zero(rt, inv):
    """A largest logit of zero or hardly more, and others nearer to it than a number of its size could tell, and farther."""
    x = np.zeros((5, 1500), f32)
    away = np.random.default_rng(6).uniform(0, 30, (5, 1500)) / inv
    x[0] = -away[0].astype(f32)
    x[0, 7] = 0.0
    x[1] = -1.0
    x[1, 700] = 0.0
    x[2] = -np.arange(1500, dtype=f32) * f32(2.0 ** -149)
    x[3] = -1e-30
    x[3, 3:40:9] = 1e-41
    x[4] = np.where(np.arange(1500) % 2, -1e-40, -2.0)
    tokens = np.argsort(-x, 1, kind="stable")[:, :5].astype(u32)
    got = run(rt, x, 1500, tokens, inv, 5)
    exp = ref.logprobs(x, tokens, inv, 5)
    assert np.array_equal(got[2], exp[2])
    with np.errstate(over="ignore"):
        for g, e in ((got[0], exp[0]), (got[1], exp[1]), (got[3], exp[3])):
            close(f"inv {inv}", g, np.where(np.isinf(e.astype(f32)), e.astype(f32), e))


def test_likely_tokens_keep_their_digits(rt):
    """Log probabilities down to -1e-30: the others' mass, not 1 less a sum."""
    x = np.zeros((4, 3000), f32)
    x[0, 5], x[1, 5], x[2, 5], x[3, 5] = 12.0, 25.0, 40.0, 70.0
    check(rt, "likely", x, 3000, np.full((4, 1), 5, u32), 1.0, 3)


def test_parts_alone_are_the_same(rt):
    x = rows(4, 7, 33333)
    tokens = np.random.default_rng(2).integers(0, 33333, (7, 2)).astype(u32)
    none = np.zeros((7, 0), u32)
    all_of = run(rt, x, 33333, tokens, 1.0, 10)
    assert np.array_equal(run(rt, x, 33333, tokens, 1.0, 0, entropy=False)[0], all_of[0])
    assert np.array_equal(run(rt, x, 33333, none, 1.0, 0)[1], all_of[1])
    alone = run(rt, x, 33333, none, 1.0, 10, entropy=False)
    assert np.array_equal(alone[2], all_of[2]) and np.array_equal(alone[3], all_of[3]) and (alone[1] == 7).all()
    for _ in range(2):
        again = run(rt, x, 33333, tokens, 1.0, 10)
        assert all(np.array_equal(a, b) for a, b in zip(all_of, again))


def test_refusals(rt):
    x, t, o = rt.empty(100), rt.empty(100, u32), rt.empty(100)
    n = rt.token_logprobs_workspace(2, 50, 3)
    ws = rt.alloc(n)
    with pytest.raises(OperatorError, match="too small") as e:
        rt.token_logprobs(x, 50, t, 1, o, None, None, None, 2, 50, 0, 1.0, ws, n - 1)
    assert e.value.kind == "InvalidInput"
    with pytest.raises(OperatorError, match="asked"):
        rt.token_logprobs(x, 50, None, 0, None, None, None, None, 2, 50, 0, 1.0, ws, n)
    with pytest.raises(OperatorError, match="inv_temperature"):
        rt.token_logprobs(x, 50, t, 1, o, None, None, None, 2, 50, 0, math.nan, ws, n)
    with pytest.raises(OperatorError, match="64"):
        rt.token_logprobs_workspace(2, 50, 65)


def test_replays(rt):
    """A recorded call follows its buffers from replay to replay, with eager work between."""
    R, V, top = 5, 40000, 7
    dl, dt = rt.empty(R * V), rt.empty(R, u32)
    lp, en, ids, tp = rt.empty(R), rt.empty(R), rt.empty(R * top, u32), rt.empty(R * top)
    n = rt.token_logprobs_workspace(R, V, top)
    ws = rt.alloc(n)
    rt.graph_begin()
    rt.argmax(dl, dt, R, V)
    rt.token_logprobs(dl, V, dt, 1, lp, en, ids, tp, R, V, top, 1.25, ws, n)
    graph = rt.graph_end()
    for step in range(4):
        x = rows(step, R, V)
        dl.upload(x)
        rt.sync()
        rt.graph_launch(graph)
        rt.sync()
        exp = ref.logprobs(x, dt.download(R).reshape(R, 1), 1.25, top)
        assert np.array_equal(ids.download().reshape(R, top), exp[2])
        close("logprobs", lp.download(R).reshape(R, 1), exp[0])
        close("entropy", en.download(R), exp[1])
        close("tops", tp.download().reshape(R, top), exp[3])
        rt.memset(ids, 0xEE, ids.nbytes)
        rt.argmax(dl, dt, R, V)
        rt.sync()
    rt.graph_destroy(graph)


@pytest.mark.parametrize("vocab,R", [(1, 3), (2, 3), (60, 3), (1000, 3), (3000, 3), (50257, 2), (16385, 600)])
@pytest.mark.parametrize("ahead", [0.5, 5.5, 9.0, 12.0, 25.0, 40.0, 70.0, 100.0])
def test_log_probabilities_near_zero(rt, vocab, R, ahead):
    """A token so likely that the others' mass is far below the last bit of 1: its log probability is that mass, of its own
    size, and so is the entropy.  f32's half a step; masses and sums are within 2^-38 (2^-45 a power, 2^-52 |y| its
    argument, 45 additions of 2^-53 each of sums 2^8 times as large as what is left)."""
    say(f"{R} x {vocab}, {ahead} ahead")
    x = rows(vocab, R, vocab, std=1.0)
    best = np.random.default_rng(int(ahead)).integers(0, vocab, R)
    best[0], best[-1] = 0, vocab - 1
    x[np.arange(R), best] = x.max(1) + f32(ahead)
    x[:, 7::50] = -np.inf
    x[np.arange(R), best] = np.where(np.isinf(x[np.arange(R), best]), f32(5 + ahead), x[np.arange(R), best])
    if R > 3:
        x[5, :] = -np.inf
        x[5, best[5]] = 3.0  # alone
        x[6, (best[6] + 1) % vocab] = x[6, best[6]]  # two of them
    tokens = best.reshape(R, 1).astype(u32)
    for inv in (1.0, 1.0 / 0.7):
        got, exp = run(rt, x, vocab, tokens, inv, 2), ref.logprobs(x, tokens, inv, 2)
        assert np.array_equal(got[2], exp[2])
        for what, g, e in (("logprobs", got[0], exp[0]), ("entropy", got[1], exp[1]), ("tops", got[3], exp[3])):
            same = np.isinf(e) | np.isinf(g)
            assert np.array_equal(g[same], e[same].astype(f32)), what
            assert not np.signbit(g[g == 0]).any(), f"{what}: -0"
            off, tol = np.abs(g[~same] - e[~same]), np.abs(e[~same]) * (2.0 ** -24 + 2.0 ** -38) + 2.0 ** -149
            assert (off <= tol).all(), f"{what}: {float((off / tol).max()):.3g} of the tolerance"
