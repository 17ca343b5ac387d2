"""GPU tests of the attention over a shared prompt and own caches (f32, Q8_0,
Q4_0) against float64, row by row.

Tolerance.  A score is a dot product of D f32 products whose operands carry at
most 2^-21 relative error (f32 rounding of q * scale, or the two-part f16 form of
an operand), summed in f32: |dx| <= (D + 8) 2^-24 S + 2^-20 S with S = sum |q k|
|scale|, since D products summed in any order round at most D times.  A weight
changes by a factor e^{dx}, a quotient of weights by e^{2 dx}; the two-part
forms of the weight and the value add 2^-20, the sums over n keys at most
n 2^-24 in any order, exp2 and the joins under 16 roundings.  So
|dout| <= ((e^{2 dx} - 1) + 2^-20 + (n + 16) 2^-24) * sum p |v|, elementwise;
and normwise, as the header promises, 1e-5 for values of about N(0, 1)."""
import sys

import numpy as np
import pytest

import decode_refs as ref
from atlas_amd import HipRuntime, OperatorError

pytestmark = pytest.mark.gpu
f32 = np.float32


def say(msg):
    print(f"[gpu-prefix-attention] {msg}", flush=True)
    sys.stdout.flush()


def make(seed, fmt, B, T, H, KH, D, P, pcap, cap, lengths, q_std=2.0, std=1.0):
    r = np.random.default_rng(seed)
    q = (r.standard_normal((B, T, H, D)) * q_std).astype(f32)
    prefix = ref.make_cache(r, fmt, pcap, KH * D, std) if pcap else None
    cache = ref.make_cache(r, fmt, B * cap, KH * D, std) if cap else None
    return q, prefix, cache, np.asarray(lengths, np.uint32)


def run(rt, fmt, q, prefix, P, cache, lengths, cap, KH, scale, w_in=None, w_out=None, alias=False):
    B, T, H, D = q.shape
    pcap = prefix.shape[1] if prefix is not None else 0
    up = lambda x: None if x is None else rt.upload(x)  # noqa: E731
    dq, dp, dc, dn, wi = up(q), up(prefix), up(cache), up(lengths) if cap else None, up(w_in)
    wo = wi if alias else up(w_out)
    out = rt.empty(q.size)
    rt.memset(out, 0xFF, q.nbytes)
    nbytes = rt.prefix_attention_workspace(fmt, B, T, H, KH, D, P, cap, wo is not None)
    ws = rt.alloc(nbytes + 256)
    rt.memset(ws, 0xFF, nbytes + 256)
    rt.prefix_attention(fmt, dq, dp, P, pcap, dc, dn, cap, out, wi, wo, B, T, H, KH, D, scale, ws, nbytes)
    rt.sync()
    got = out.download(q.size).reshape(q.shape)
    guard = ws.download(nbytes + 256, np.uint8)[nbytes:]
    assert (guard == 0xFF).all(), "wrote behind the workspace"
    weights = None if wo is None else wo.download(B * cap).reshape(B, cap)
    for b in (dq, dp, dc, dn, wi, out, ws) + (() if alias else (wo,)):
        if b is not None:
            rt.free(b)
    return got, weights


def check(name, got, exp, bound, keys, D):
    mass, dot = bound
    dx = (D + 8) * 2.0 ** -24 * dot + 2.0 ** -20 * dot
    tol = (np.expm1(2 * dx)[..., None] + 2.0 ** -20 + (keys + 16) * 2.0 ** -24) * mass + 1e-37
    off = np.abs(got.astype(np.float64) - exp)
    assert np.isfinite(got).all(), f"{name}: not finite"
    worst = float((off / tol).max())
    norm = float(np.linalg.norm(off) / max(np.linalg.norm(exp), 1e-300))
    say(f"{name}: normwise {norm:.2e}, of the elementwise bound {worst:.3f}")
    assert worst <= 1.0 and norm <= 1e-5, name


# name: B, T, H, KH, D, prefix, prefix capacity, capacity, lengths
SHAPES = {
    "one_token_one_key": (1, 1, 1, 1, 64, 1, 1, 0, []),
    "one_own_key": (1, 1, 8, 1, 256, 0, 0, 1, [1]),
    "empty_rows": (4, 1, 8, 1, 128, 0, 0, 40, [0, 1, 17, 40]),
    "smol": (1, 1, 9, 3, 64, 512, 512, 128, [77]),
    "no_own": (3, 1, 8, 2, 128, 65, 70, 0, []),
    "tile_edges": (5, 1, 8, 1, 256, 63, 64, 80, [15, 16, 17, 64, 65]),
    "clamped": (3, 1, 4, 2, 96, 16, 16, 20, [21, 4000000000, 20]),
    "drafts": (6, 5, 16, 4, 128, 257, 300, 90, [0, 1, 4, 5, 77, 90]),
    "drafts_alone": (4, 4, 8, 1, 256, 0, 0, 70, [0, 2, 3, 70]),
    "many_heads": (2, 3, 32, 1, 64, 100, 100, 50, [3, 50]),
    "no_groups": (2, 1, 32, 32, 64, 33, 40, 31, [31, 2]),
    "wide_heads": (2, 2, 6, 2, 160, 129, 129, 66, [66, 30]),
    "batch": (70, 1, 8, 1, 256, 1000, 1024, 64, [(7 * i) % 65 for i in range(70)]),
    "batch_128": (33, 2, 32, 4, 128, 333, 333, 16, [(5 * i) % 17 for i in range(33)]),
    "batch_64": (90, 1, 12, 2, 64, 700, 700, 9, [(5 * i) % 10 for i in range(90)]),
    "batch_96": (110, 1, 10, 2, 96, 65, 65, 9, [(5 * i) % 10 for i in range(110)]),
    "batch_160": (35, 2, 16, 2, 160, 129, 129, 40, [(5 * i) % 41 for i in range(35)]),
    "batch_256": (9, 1, 8, 1, 256, 300, 300, 40, [(5 * i) % 41 for i in range(9)]),
    "packed_64": (90, 1, 12, 2, 64, 21777, 21777, 9, [(5 * i) % 10 for i in range(90)]),
    "packed_96": (110, 1, 10, 2, 96, 10881, 10881, 9, [(5 * i) % 10 for i in range(110)]),
    "packed_128": (33, 2, 32, 4, 128, 5441, 5442, 16, [(5 * i) % 17 for i in range(33)]),
    "packed_160": (35, 2, 16, 2, 160, 5441, 5441, 40, [(5 * i) % 41 for i in range(35)]),
    "packed_256": (70, 1, 8, 1, 256, 10915, 11000, 64, [(7 * i) % 65 for i in range(70)]),
    "widest_rows": (2, 1, 128, 128, 256, 40, 41, 20, [20, 3]),
    "widest_batch": (18, 1, 128, 128, 256, 40, 41, 3, [i % 4 for i in range(18)]),
    "one_group": (1, 1, 128, 1, 128, 70, 70, 50, [50]),
    "prefill": (1, 300, 4, 2, 64, 100, 100, 301, [300]),
    "one_long_prompt": (1, 1, 8, 1, 256, 30001, 30001, 70, [70]),
    "one_long_own": (1, 2, 16, 4, 128, 0, 0, 20001, [20001]),
    "odd_segments": (37, 1, 28, 4, 128, 1500, 1500, 8, [i % 9 for i in range(37)]),
    "long": (2, 1, 8, 1, 256, 9001, 9001, 5000, [4999, 700]),
}


@pytest.mark.parametrize("fmt", ["f32", "q8_0", "q4_0"])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_prefix_attention_matches_float64(rt, shape, fmt):
    B, T, H, KH, D, P, pcap, cap, lengths = SHAPES[shape]
    say(f"{shape} {fmt}")
    q, prefix, cache, n = make(len(shape) + D, fmt, B, T, H, KH, D, P, pcap, cap, lengths)
    scale = float(f32(D ** -0.5))
    exp, weights, bound = ref.attention(q, prefix, P, cache, n, cap, KH, scale, fmt)
    got, _ = run(rt, fmt, q, prefix, P, cache, n, cap, KH, scale)
    check(f"{shape} {fmt}", got, exp, bound, P + cap, D)
    empty = np.array([[P + max(0, min(int(n[b]), cap) - (T - 1 - t)) == 0 for t in range(T)] for b in range(B)]) if cap else np.zeros((B, T), bool)
    assert (got[empty] == 0).all()
    if cap:
        r = np.random.default_rng(5)
        w_in, w_fill = r.uniform(0, 3, (B, cap)).astype(f32), np.full((B, cap), -7.0, f32)
        for with_in, alias in ((True, False), (False, False), (True, True)):
            got2, w = run(rt, fmt, q, prefix, P, cache, n, cap, KH, scale, w_in if with_in else None, w_fill, alias)
            assert np.array_equal(got2.view(np.uint32), got.view(np.uint32)), "the weights changed the output"
            before = w_in if with_in else np.zeros_like(w_in)
            rest = w_in if alias else w_fill
            there = np.arange(cap)[None, :] < np.minimum(n, cap)[:, None]
            assert np.array_equal(w[~there], rest[~there]), "a weight behind a sequence changed"
            # a weight is a sum of T * H shares p; each is off by (e^{2 dx} - 1 + (keys + 32) 2^-24) p
            dx = (D + 8) * 2.0 ** -24 * bound[1].max() + 2.0 ** -20 * bound[1].max()
            tol = (np.expm1(2 * dx) + (P + cap + 32 + T * H) * 2.0 ** -24) * weights + 2.0 ** -23 * (before + weights) + 1e-30
            off = np.abs(w.astype(np.float64) - (before.astype(np.float64) + weights))
            assert (off[there] <= tol[there]).all(), f"{shape} {fmt}: weights off {float((off / tol)[there].max()):.2f} of the bound"


def test_more_sequences_than_a_launch_has_rows_of_workgroups(rt):
    say("70001 sequences")
    B, D, cap = 70001, 4, 3
    q, prefix, cache, n = make(2, "f32", B, 1, 1, 1, D, 5, 5, cap, [i % 4 for i in range(B)])
    exp, weights, bound = ref.attention(q, prefix, 5, cache, n, cap, 1, 0.5, "f32")
    w = np.full((B, cap), 2.0, f32)
    got, w_got = run(rt, "f32", q, prefix, 5, cache, n, cap, 1, 0.5, w, w, alias=True)
    check("70001 sequences", got, exp, bound, 5 + cap, D)
    # one share of at most 1, off by under 16 roundings of 2^-24 (eight keys, exp2, log2), added to 2
    assert np.allclose(w_got, w + weights, rtol=2e-6, atol=0)


@pytest.mark.parametrize("D", [4, 20, 36, 68, 80, 132, 244])
def test_head_dims_that_fill_no_tile(rt, D):
    say(f"head_dim {D}")
    q, prefix, cache, n = make(D, "f32", 3, 2, 6, 2, D, 50, 50, 20, [20, 1, 9])
    exp, _, bound = ref.attention(q, prefix, 50, cache, n, 20, 2, 0.3, "f32")
    got, _ = run(rt, "f32", q, prefix, 50, cache, n, 20, 2, 0.3)
    check(f"head_dim {D}", got, exp, bound, 70, D)


@pytest.mark.parametrize("B", [1, 40])
def test_what_is_not_seen_never_matters(rt, B):
    """NaN, infinities and the type's extremes behind the prompt, behind each sequence, and in drafts that a token
    does not see yet."""
    say(f"unseen places, batch {B}")
    T, H, KH, D, P, cap = 4, 8, 1, 256, 70, 100
    lengths = [(13 * i + 30) % 97 + 4 for i in range(B)]
    q, prefix, cache, n = make(3, "f32", B, T, H, KH, D, P, 128, cap, lengths)
    clean, _ = run(rt, "f32", q, prefix, P, cache, n, cap, KH, 0.0625)
    for bad in (np.nan, np.inf, -np.inf, np.finfo(f32).max, np.finfo(f32).min):
        p2, c2 = prefix.copy(), cache.copy()
        p2.view(f32)[:, P:] = bad
        rows = c2.view(f32).reshape(2, B, cap, D)
        for b in range(B):
            rows[:, b, lengths[b]:] = bad
        got, _ = run(rt, "f32", q, p2, P, c2, n, cap, KH, 0.0625)
        assert np.array_equal(got.view(np.uint32), clean.view(np.uint32)), f"{bad} behind the rows"
        for b in range(B):
            rows[:, b, lengths[b] - 1:] = bad  # the last draft's own row: only the last token sees it
        w = np.zeros((B, cap), f32)
        got, _ = run(rt, "f32", q, p2, P, c2, n, cap, KH, 0.0625, None, w)
        assert np.isfinite(got[:, :T - 1]).all(), f"{bad} in a later draft"
        # with other arithmetic at most: the tile may be added key by key
        assert np.allclose(got[:, :T - 1], clean[:, :T - 1], rtol=2e-4, atol=2e-6), f"{bad} in a later draft"
        if not np.isfinite(bad):
            assert not np.isfinite(got[:, T - 1]).all()


@pytest.mark.parametrize("q_std,std", [(1e-12, 1e-12), (1e8, 1e-8), (30.0, 1.0), (1.0, 1e-25), (1e-15, 1e15)])
def test_values_of_any_scale(rt, q_std, std):
    say(f"q {q_std} cache {std}")
    for B in (1, 40):
        q, prefix, cache, n = make(17, "f32", B, 1, 8, 1, 128, 300, 300, 40, [40 - i % 40 for i in range(B)], q_std, std)
        exp, _, bound = ref.attention(q, prefix, 300, cache, n, 40, 1, 0.1, "f32")
        got, _ = run(rt, "f32", q, prefix, 300, cache, n, 40, 1, 0.1)
        check(f"q {q_std} cache {std} batch {B}", got, exp, bound, 340, 128)


def test_rows_of_very_different_scale(rt):
    """Rows of a cache from 1e-18 to 1e18 side by side: each weight and value keeps its own precision."""
    say("mixed scales")
    B, D, P = 40, 128, 257
    q, prefix, cache, n = make(23, "f32", B, 1, 8, 1, D, P, P, 8, [8] * B, 1.0)
    f = prefix.view(f32)
    r = np.random.default_rng(1)
    f[0] *= (10.0 ** r.uniform(-18, 0, (P, 1))).astype(f32)
    f[1] *= (10.0 ** r.uniform(-18, 18, (P, 1))).astype(f32)
    f[0, ::5] = 0.0
    f[1, ::7] = 0.0
    exp, _, bound = ref.attention(q, prefix, P, cache, n, 8, 1, 0.2, "f32")
    got, _ = run(rt, "f32", q, prefix, P, cache, n, 8, 1, 0.2)
    check("mixed scales", got, exp, bound, P + 8, D)


@pytest.mark.parametrize("B,P", [(3, 70), (1, 70), (40, 70), (70, 10915)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_seen_value_that_is_no_number_is_never_lost(rt, B, P, bad):
    """It may leave NaN in all dims of the rows that see it, and a number only where float64 has the same."""
    say(f"seen {bad}, batch {B}, prompt {P}")
    D, cap = 256, 20
    lengths = [(13 * i) % 20 + 1 for i in range(B)]
    q, prefix, cache, n = make(3, "f32", B, 1, 8, 1, D, P, P, cap, lengths)
    prefix.view(f32)[1, P // 3, 7] = bad
    cache.view(f32).reshape(2, B, cap, D)[1, B - 1, 0, 100] = bad
    exp, _, bound = ref.attention(q, prefix, P, cache, n, cap, 1, 0.0625, "f32")
    got, _ = run(rt, "f32", q, prefix, P, cache, n, cap, 1, 0.0625)
    assert not np.isfinite(got[..., 7]).any() and not np.isfinite(got[B - 1, ..., 100]).any()
    same = np.isfinite(got)
    assert np.isfinite(exp[same]).all()
    got, exp = np.where(same, got, 0), np.where(same, exp, 0)
    check(f"seen {bad} batch {B}", got, exp, (np.where(np.isfinite(bound[0]), bound[0], 0), bound[1]), P + cap, D)


def test_offsets_past_32_bits(rt):
    """The third sequence's rows and the whole V plane lie more than 2^32 bytes into the cache."""
    say("long cache")
    B, D, cap, n = 3, 256, 1 << 21, 33
    r = np.random.default_rng(9)
    rows = r.standard_normal((2, B, n, D)).astype(f32)
    big = rt.alloc(2 * B * cap * D * 4)
    for plane in range(2):
        for b in range(B):
            big.offset(((plane * B + b) * cap) * D * 4).upload(rows[plane, b])
    q = r.standard_normal((B, 1, 8, D)).astype(f32)
    lengths = np.full(B, n, np.uint32)
    nbytes = rt.prefix_attention_workspace("f32", B, 1, 8, 1, D, 0, cap)
    ws, out = rt.alloc(nbytes), rt.empty(q.size)
    rt.prefix_attention("f32", rt.upload(q), None, 0, 0, big, rt.upload(lengths), cap, out, None, None, B, 1, 8, 1, D, 0.0625,
                        ws, nbytes)
    rt.sync()
    small = rows.reshape(2, B * n, D).view(np.uint8)
    exp, _, bound = ref.attention(q, None, 0, small, lengths, n, 1, 0.0625, "f32")
    check("long cache", out.download(q.size).reshape(q.shape), exp, bound, n, D)
    rt.free(big)
    rt.free(ws)


def _program(rt, seed, B):
    T, H, KH, D, P, cap = 2, 8, 1, 256, 8 * B + 600, 64
    q, prefix, cache, n = make(seed, "q8_0", B, T, H, KH, D, P, P, cap, [(i * 11) % 65 for i in range(B)])
    d = {"q": rt.upload(q), "prefix": rt.upload(prefix), "cache": rt.upload(cache), "n": rt.upload(n),
         "out": rt.empty(q.size), "w": rt.empty(B * cap)}
    nbytes = rt.prefix_attention_workspace("q8_0", B, T, H, KH, D, P, cap, True)
    d["ws"] = rt.alloc(nbytes)

    def call():
        rt.prefix_attention("q8_0", d["q"], d["prefix"], P, P, d["cache"], d["n"], cap, d["out"], None, d["w"], B, T, H, KH, D,
                            0.0625, d["ws"], nbytes)

    return d, call, q, B * cap


@pytest.mark.parametrize("B", [2, 40, 300])
def test_graph_replays_equal_the_eager_call(rt, B):
    say(f"graph, batch {B}")
    d, call, q, weights = _program(rt, 31, B)
    rt.memset(d["w"], 0, weights * 4)
    call()
    rt.sync()
    eager = d["out"].download(q.size), d["w"].download(weights)
    rt.graph_begin()
    call()
    graph = rt.graph_end()
    for i in range(4):
        rt.memset(d["out"], 0xEE, q.nbytes)
        rt.memset(d["w"], 0, weights * 4)
        rt.graph_launch(graph)
        rt.sync()
        assert np.array_equal(d["out"].download(q.size), eager[0]) and np.array_equal(d["w"].download(weights), eager[1]), i
        other, call2, _, _ = _program(rt, 32 + i, 3)
        call2()  # eager work between the replays
        rt.sync()
    # the graph reads its inputs at replay
    q2 = -q
    d["q"].upload(q2)
    rt.graph_launch(graph)
    rt.sync()
    again = d["out"].download(q.size)
    call()
    rt.sync()
    assert np.array_equal(again, d["out"].download(q.size)) and not np.array_equal(again, eager[0])
    rt.graph_destroy(graph)


def test_two_contexts_at_once_and_another_stream(rt):
    say("two contexts")
    other = HipRuntime(0)
    try:
        a, call_a, qa, _ = _program(rt, 41, 24)
        b, call_b, qb, _ = _program(other, 42, 24)
        call_a()
        rt.sync()
        call_b()
        other.sync()
        alone = a["out"].download(qa.size), b["out"].download(qb.size)
        for _ in range(8):
            call_a()
            call_b()
        rt.sync()
        other.sync()
        assert np.array_equal(a["out"].download(qa.size), alone[0]) and np.array_equal(b["out"].download(qb.size), alone[1])
        rt.memset(a["out"], 0, qa.nbytes)
        rt.sync()
        rt._check(rt.lib.atlas_hip_set_stream(rt.ctx, other.lib.atlas_hip_get_stream(other.ctx)))
        try:
            call_a()
            rt.sync()
        finally:
            rt._check(rt.lib.atlas_hip_set_stream(rt.ctx, None))
        assert np.array_equal(a["out"].download(qa.size), alone[0])
    finally:
        other.close()


def test_refusals(rt):
    say("refusals")
    B, T, H, KH, D, P, cap = 2, 1, 8, 1, 64, 32, 16
    q, prefix, cache, n = make(1, "f32", B, T, H, KH, D, P, P, cap, [3, 4])
    dq, dp, dc, dn, out, w = rt.upload(q), rt.upload(prefix), rt.upload(cache), rt.upload(n), rt.empty(q.size), rt.empty(B * cap)
    nbytes = rt.prefix_attention_workspace("f32", B, T, H, KH, D, P, cap, True)
    ws = rt.alloc(nbytes)
    good = dict(fmt="f32", q=dq, prefix=dp, prefix_length=P, prefix_capacity=P, cache=dc, lengths=dn, capacity=cap, out=out,
                weights_in=None, weights_out=w, sequences=B, tokens=T, q_heads=H, kv_heads=KH, head_dim=D, scale=0.1,
                workspace=ws, workspace_bytes=nbytes)
    rt.prefix_attention(**good)
    rt.sync()
    bad = [dict(q=None), dict(out=None), dict(workspace=None), dict(prefix=None), dict(cache=None), dict(lengths=None),
           dict(sequences=0), dict(tokens=0), dict(q_heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(head_dim=0),
           dict(head_dim=260), dict(head_dim=62), dict(fmt="q8_0", head_dim=48), dict(prefix_length=P + 1),
           dict(prefix_length=0, capacity=0, weights_out=None), dict(capacity=0), dict(scale=float("nan")),
           dict(scale=float("inf")), dict(workspace_bytes=nbytes - 1), dict(q=dq.ptr + 4), dict(cache=dc.ptr + 8),
           dict(prefix=dp.ptr + 8), dict(workspace=ws.ptr + 8), dict(weights_out=w.ptr + 2), dict(out=dq.ptr + 16),
           dict(weights_in=w, weights_out=None), dict(weights_in=w.ptr + 4), dict(fmt="q4_0", prefix=dp.ptr + 1)]
    for change in bad:
        with pytest.raises(OperatorError) as e:
            rt.prefix_attention(**{**good, **change})
        assert e.value.kind == "InvalidInput", change
    for sizes in (("f32", 0, 1, 8, 1, 64, 1, 1), ("q8_0", 1, 1, 8, 1, 40, 1, 1), ("f32", 1, 1, 8, 3, 64, 1, 1)):
        with pytest.raises(OperatorError):
            rt.prefix_attention_workspace(*sizes)
    rt.prefix_attention(**good)  # the context is as good as before
    rt.sync()
