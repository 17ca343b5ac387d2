"""GPU tests of every launch of the paged attention and of the log probabilities,
by the calls of paged_launches.py (test_paged_plans.py says which launch each
takes), against float64, within the bounds of test_gpu_paged_attention.py and
test_gpu_logprobs.py."""
import sys

import numpy as np
import pytest

import paged_refs as ref
import test_gpu_logprobs as lp
import test_gpu_paged_attention as at
from paged_launches import ATTENTION, FORMATS, LOGPROBS

pytestmark = pytest.mark.gpu
f32, u32 = np.float32, np.uint32


def say(msg):
    print(f"[gpu-paged-launches] {msg}", flush=True)
    sys.stdout.flush()


@pytest.mark.parametrize("name", list(ATTENTION))
def test_attention(rt, name):
    fmt, H, KH, D, ps, width, lengths, window, launch = ATTENTION[name]
    say(f"{name} {launch}")
    args = at.spread(len(lengths) + D, fmt, H, KH, D, ps, width, lengths)
    got = at.run(rt, fmt, *args, window, D ** -0.5)
    assert (got[args[3] == 0] == 0).all()
    at.check(name, fmt, *args, window, D ** -0.5, got)
    assert np.array_equal(got, at.run(rt, fmt, *args, window, D ** -0.5)), "not the same bits again"


@pytest.mark.parametrize("fmt", FORMATS)
def test_more_parts_than_stay(rt, fmt):
    """More units than 1024 a part of those that stay.  Every position the same key and value, so the result is the value:
    within (256 + 256 + 64) 2^-24 = 3.5e-5 by the count of roundings of sum and weights alike, and in effect 1e-5."""
    H, KH, D, ps, n, B = 8, 1, 64, 256, 1 << 20, 40
    pool = ref.Pool(fmt, 1, ps, KH, D).random(np.random.default_rng(4))
    for plane in range(2):
        row = np.random.default_rng(plane).standard_normal(D).astype(f32)
        for i in range(ps):
            pool.write(0, plane, 0, i, row)
    table = np.zeros((B, n // ps), u32)
    q = np.random.default_rng(2).standard_normal((B, H, D)).astype(f32)
    lengths = np.array([n - 7 * b for b in range(B)], u32)
    say(fmt)
    got = at.run(rt, fmt, pool, table, q, lengths, 0, 0.125).astype(np.float64)
    value = pool.values(0, 1, 0)[0]
    worst = float((np.abs(got - value) / np.maximum(np.abs(value), 1e-30)).max())
    say(f"{fmt}: {worst:.2e} of each value")
    assert worst <= 3.5e-5
    assert np.linalg.norm(got - value) <= 1e-5 * np.linalg.norm(np.broadcast_to(value, got.shape))


@pytest.mark.parametrize("kind", ["random", "ties"])
@pytest.mark.parametrize("name", list(LOGPROBS))
def test_log_probabilities(rt, name, kind):
    """With and without entropy and alternatives; ties: rows of few values, of one, and of a run at the end."""
    R, vocab, pad, *launch = LOGPROBS[name]
    say(f"{name} {kind} {launch}")
    x = lp.rows(vocab + R, R, vocab + pad)
    x[:, vocab:] = np.nan
    if kind == "ties":
        x = np.round(x)
        x[1] = 2.5
        x[2, :vocab - 3] = -np.inf
        x[R // 2, vocab // 2:vocab] = 9.0
        x[R - 2, :vocab] = -np.inf
        x[R - 1, :vocab - 1] = np.nan
    tokens = np.random.default_rng(R).integers(0, vocab, (R, 2)).astype(u32)
    tokens[:, 1] = np.where(np.isnan(x[:, :vocab]), -np.inf, x[:, :vocab]).argmax(1)
    exp = ref.logprobs(x[:, :vocab], tokens, 1.25, 64)
    for top, entropy in ((0, True), (20, False), (64, True)):
        got = lp.run(rt, x, vocab, tokens, 1.25, top, entropy)
        assert np.array_equal(got[2], exp[2][:, :top]), f"top {top}: ids differ in rows {np.nonzero((got[2] != exp[2][:, :top]).any(1))[0][:5]}"
        lp.close(f"top {top}: logprobs", got[0], exp[0])
        lp.close(f"top {top}: tops", got[3], exp[3][:, :top])
        if entropy:
            lp.close(f"top {top}: entropy", got[1], exp[1])
        else:
            assert (got[1] == 7).all()
