"""GPU tests of the shared-prompt attention where finite inputs lie far from
those of a model, against float64."""
import sys

import numpy as np
import pytest

import decode_refs as ref
from test_gpu_prefix_attention import check, run

pytestmark = pytest.mark.gpu
f32 = np.float32


def say(msg):
    print(f"[gpu-prefix-range] {msg}", flush=True)
    sys.stdout.flush()


# sequences of 8 heads, prompt, head_dim: f32 products throughout, f16 pieces, f16 pieces of a packed prompt
PATHS = {"few_rows": (1, 300, 128), "many_rows": (40, 300, 128), "packed": (70, 10915, 256)}


def one_dim(B, P, D, cap, seed, value):
    """A batch whose scores lie in dim 0 alone: q (dim 0 zero), prompt and own keys zero, values about N(0, value)."""
    r = np.random.default_rng(seed)
    q = np.zeros((B, 1, 8, D), f32)
    prefix, cache = np.zeros((2, P, D), f32), np.zeros((2, B * cap, D), f32)
    prefix[1] = r.standard_normal((P, D)) * value
    cache[1] = r.standard_normal((B * cap, D)) * value
    n = np.asarray([cap - i % (cap + 1) for i in range(B)], np.uint32)
    return q, prefix, cache, n


def as_bytes(a):
    return a.view(np.uint8).reshape(*a.shape[:-1], -1)


@pytest.mark.parametrize("path", list(PATHS))
@pytest.mark.parametrize("value", [1e-6, 1e-2, 1e3])
@pytest.mark.parametrize("e", [10, 24, 27, 28, 29, 31, 100])
def test_scores_of_any_size(rt, path, value, e):
    """Keys alike but one or three, whose scores are the only large ones, or the only small ones: every weight is 1, a
    third, or nothing, whatever the scores' spacing.  (Equal keys have equal scores: only the sums round.)"""
    B, P, D = PATHS[path]
    say(f"{path}, values {value}, scores of 2^{e}")
    q, prefix, cache, n = one_dim(B, P, D, 8, 3, value)
    q[..., 0] = 2.0 ** (e / 2)
    hot = [P // 3, P // 2, P - 1]
    for which, sign in (([P // 3], 1), (hot, 1), (hot, -1), (range(P), 1)):
        prefix[0] = 0.0
        prefix[0, list(which), 0] = sign * 2.0 ** (e / 2)
        exp, _, bound = ref.attention(q, as_bytes(prefix), P, as_bytes(cache), n, 8, 1, 1.0, "f32")
        got, _ = run(rt, "f32", q, as_bytes(prefix), P, as_bytes(cache), n, 8, 1, 1.0)
        # the weights are exact, so the bound has no part of the scores' rounding
        check(f"{path} {value} 2^{e} {len(list(which))} {sign}", got, exp, (bound[0], np.zeros_like(bound[1])), P + 8, D)


@pytest.mark.parametrize("path", list(PATHS))
@pytest.mark.parametrize("score", [20.0, 60.0, 75.0])
def test_a_row_of_zeros_that_draws_all_attention(rt, path, score):
    """What the other rows add is small and keeps its bits.  (Scores in dim 0, 75 = 108 in base 2 and exact but for the
    factor log2 e: 2^-24 of 108 moves a weight by 4.5e-6.)"""
    B, P, D = PATHS[path]
    say(f"{path}, score {score}")
    q, prefix, cache, n = one_dim(B, P, D, 8, 5, 1.0)
    q[..., 0] = 1.0
    prefix[0, P // 2, 0] = score
    prefix[1, P // 2] = 0.0
    cache[1] = 0.0
    exp, _, bound = ref.attention(q, as_bytes(prefix), P, as_bytes(cache), n, 8, 1, 1.0, "f32")
    got, _ = run(rt, "f32", q, as_bytes(prefix), P, as_bytes(cache), n, 8, 1, 1.0)
    check(f"{path} zeros {score}", got, exp, bound, P + 8, D)


@pytest.mark.parametrize("path", list(PATHS))
@pytest.mark.parametrize("q_exp,k_exp,v_exp", [(0, 0, -100), (0, 0, -106), (116, -118, 0), (-118, 116, 0), (110, -112, -100)])
def test_operands_at_the_ends_of_the_range(rt, path, q_exp, k_exp, v_exp):
    B, P, D = PATHS[path]
    say(f"{path}, q 2^{q_exp} k 2^{k_exp} v 2^{v_exp}")
    r = np.random.default_rng(7)
    q = np.ldexp(r.standard_normal((B, 1, 8, D)), q_exp).astype(f32)
    prefix = np.stack([np.ldexp(r.standard_normal((P, D)), k_exp), np.ldexp(r.standard_normal((P, D)), v_exp)]).astype(f32)
    n = np.zeros(B, np.uint32)
    exp, _, bound = ref.attention(q, as_bytes(prefix), P, None, n, 0, 1, 0.25, "f32")
    got, _ = run(rt, "f32", q, as_bytes(prefix), P, None, n, 0, 1, 0.25)
    check(f"{path} {q_exp} {k_exp} {v_exp}", got, exp, bound, P, D)


def test_weights_of_equal_keys_at_any_score(rt):
    """A third each, whatever the score's spacing: the rounding of a score shifts all three alike."""
    B, H, D, cap = 3, 2, 64, 4
    for e in (0, 10, 20, 24, 27, 60):
        q, cache = np.zeros((B, 1, H, D), f32), np.zeros((2, B * cap, D), f32)
        q[..., 0] = 1.375
        cache[0, :, 0] = 2.0 ** e
        cache[1] = 1.0
        n = np.full(B, 3, np.uint32)
        w = np.zeros((B, cap), f32)
        _, got = run(rt, "f32", q, None, 0, as_bytes(cache), n, cap, 1, 1.0, None, w)
        say(f"scores of 2^{e}: {got[0]}")
        # H shares of a third, each off by under 16 roundings of 2^-24
        assert np.allclose(got[:, :3], H / 3, rtol=16 * 2.0 ** -24, atol=0) and (got[:, 3] == 0).all()


@pytest.mark.parametrize("path", list(PATHS))
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 1e38])
def test_a_query_that_is_no_number_stays_alone(rt, path, bad):
    """A padded row of a batch: its own result may be anything, the others' are theirs."""
    B, P, D = PATHS[path]
    say(f"{path}, query {bad}")
    r = np.random.default_rng(13)
    q = (r.standard_normal((B, 1, 8, D)) * 2).astype(f32)
    prefix, cache = (as_bytes(r.standard_normal((2, rows, D)).astype(f32)) for rows in (P, B * 8))
    n = np.asarray([8 - i % 9 for i in range(B)], np.uint32)
    exp, _, bound = ref.attention(q, prefix, P, cache, n, 8, 1, 0.0625, "f32")
    q[0, 0, 3] = bad
    got, _ = run(rt, "f32", q, prefix, P, cache, n, 8, 1, 0.0625)
    got[0, 0, 3] = exp[0, 0, 3]
    check(f"{path} query {bad}", got, exp, bound, P + 8, D)
