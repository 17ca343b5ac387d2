"""GPU tests of the cut of caches to a budget: every byte of the cache, every
weight, length and kept position against a plain restatement, in place and into
another cache."""
import sys

import numpy as np
import pytest

import decode_refs as ref
from atlas_amd import OperatorError

pytestmark = pytest.mark.gpu
f32 = np.float32


def say(msg):
    print(f"[gpu-kv-evict] {msg}", flush=True)
    sys.stdout.flush()


def run(rt, fmt, cache, weights, lengths, cap, width, budget, recent, in_place):
    B = len(lengths)
    fill = np.full_like(cache, 0x5A)
    w_fill = np.full_like(weights, -3.0)
    dc, dw, dn = rt.upload(cache), rt.upload(weights), rt.upload(lengths)
    oc, ow, on = (dc, dw, dn) if in_place else (rt.upload(fill), rt.upload(w_fill), rt.empty(B, np.uint32))
    kept = rt.empty(B * budget, np.uint32)
    rt.kv_evict(fmt, dc, oc, dw, ow, dn, on, kept, B, cap, width, budget, recent)
    rt.sync()
    got = (oc.download(cache.size, np.uint8).reshape(cache.shape), ow.download(weights.size).reshape(weights.shape),
           on.download(B, np.uint32), kept.download(B * budget, np.uint32).reshape(B, budget))
    exp = ref.evict(cache, weights, lengths, cap, budget, recent, cache if in_place else fill, weights if in_place else w_fill)
    if not in_place:
        assert np.array_equal(dc.download(cache.size, np.uint8).reshape(cache.shape), cache), "the input cache changed"
    for b in {id(x): x for x in (dc, dw, dn, oc, ow, on, kept)}.values():
        rt.free(b)
    return got, exp


def check(name, got, exp):
    for what, g, e in zip(("cache", "weights", "lengths", "kept"), got, exp):
        if what == "weights":
            g, e = g.view(np.uint32), e.view(np.uint32)
        assert np.array_equal(g, e), f"{name}: {what}, {int((g != e).sum())} differ, first {np.argwhere(g != e)[0]}"


def weights_of(r, kind, B, cap):
    if kind == "plain":
        return (r.standard_normal((B, cap)).clip(0) ** 4).astype(f32)
    if kind == "ties":
        return r.integers(0, 3, (B, cap)).astype(f32)
    if kind == "equal":
        return np.full((B, cap), 0.25, f32)
    if kind == "close":  # one binade, one step apart
        return (np.float32(1.0).view(np.uint32) + r.integers(0, 9, (B, cap), dtype=np.uint32)).view(f32)
    w = r.standard_normal((B, cap)).astype(f32)
    w[:, ::5] = np.nan
    w[:, 1::5] = -np.inf
    w[:, 2::7] = np.inf
    w[:, 3::4] = -0.0
    w[:, 4::9] = 0.0
    w.view(np.uint32)[:, 6::11] = 0xFFC00001  # NaN with its sign set
    return w


# B, capacity, lengths, budget, recent
SHAPES = {
    "one": (1, 1, [1], 1, 0),
    "empty": (3, 8, [0, 3, 8], 4, 2),
    "all_recent": (2, 50, [50, 41], 20, 20),
    "no_recent": (2, 50, [50, 41], 20, 0),
    "clamped": (2, 40, [41, 4000000000], 10, 3),
    "full_budget": (2, 64, [64, 30], 64, 8),
    "one_out": (3, 300, [300, 299, 257], 256, 17),
    "steps": (4, 3100, [3100, 2049, 1025, 2048], 1024, 100),
    "keep_one": (2, 2500, [2500, 2400], 1, 0),
    "batch": (130, 70, [(i * 17) % 71 for i in range(130)], 33, 5),
}


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind", ["plain", "ties", "equal", "close", "odd"])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_kv_evict_selects_and_moves(rt, shape, kind, in_place):
    B, cap, lengths, budget, recent = SHAPES[shape]
    say(f"{shape} {kind} in place {in_place}")
    r = np.random.default_rng(len(shape) * 7 + len(kind))
    n = np.asarray(lengths, np.uint32)
    cache = ref.make_cache(r, "f32", B * cap, 12)
    got, exp = run(rt, "f32", cache, weights_of(r, kind, B, cap), n, cap, 12, budget, recent, in_place)
    check(f"{shape} {kind}", got, exp)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("fmt,width", [("f32", 1), ("f32", 3), ("f32", 64), ("f32", 192), ("f32", 257), ("f32", 2048),
                                       ("q8_0", 32), ("q8_0", 64), ("q8_0", 256), ("q8_0", 1024), ("q4_0", 32),
                                       ("q4_0", 96), ("q4_0", 64), ("q4_0", 256), ("q4_0", 1024)])
def test_kv_evict_rows_of_every_format(rt, fmt, width, in_place):
    say(f"{fmt} {width} in place {in_place}")
    r = np.random.default_rng(width)
    B, cap = 3, 700
    n = np.asarray([700, 100, 555], np.uint32)
    cache = ref.make_cache(r, fmt, B * cap, width)
    got, exp = run(rt, fmt, cache, weights_of(r, "plain", B, cap), n, cap, width, 300, 40, in_place)
    check(f"{fmt} {width}", got, exp)


@pytest.mark.parametrize("in_place", [False, True])
def test_kv_evict_long_cache(rt, in_place):
    say(f"long, in place {in_place}")
    r = np.random.default_rng(77)
    n = np.asarray([140001, 131072], np.uint32)
    cache = ref.make_cache(r, "q4_0", 2 * 140001, 32)
    for kind in ("plain", "ties", "odd"):
        got, exp = run(rt, "q4_0", cache, weights_of(r, kind, 2, 140001), n, 140001, 32, 70001, 1000, in_place)
        check(f"long {kind}", got, exp)


@pytest.mark.parametrize("cap", [1024, 1025, 2049, 4096, 8000, 16384, 16385, 32768, 65536, 65537])
def test_kv_evict_capacities(rt, cap):
    """Every number of positions a lane of the selection holds, and the first that it reads anew."""
    say(f"capacity {cap}")
    r = np.random.default_rng(cap)
    n = np.asarray([cap, cap - 1, cap // 2 + 3, 1], np.uint32)
    cache = ref.make_cache(r, "f32", 4 * cap, 4)
    for kind in ("plain", "ties", "odd"):
        for budget, recent, in_place in ((cap // 2, cap // 8, True), (cap - 2, 1, False), (3, 3, True)):
            got, exp = run(rt, "f32", cache, weights_of(r, kind, 4, cap), n, cap, 4, budget, recent, in_place)
            check(f"{cap} {kind} {budget}", got, exp)


@pytest.mark.parametrize("in_place", [False, True])
def test_kv_evict_more_sequences_than_a_launch_moves(rt, in_place):
    say(f"22001 sequences, in place {in_place}")
    r = np.random.default_rng(8)
    n = r.integers(0, 5, 22001, dtype=np.uint32)
    cache = ref.make_cache(r, "f32", 4 * 22001, 4)
    got, exp = run(rt, "f32", cache, weights_of(r, "plain", 22001, 4), n, 4, 4, 2, 1, in_place)
    check("22001 sequences", got, exp)


def test_kv_evict_offsets_past_32_bits(rt):
    say("offsets past 32 bits")
    B, cap, width = 3, 1 << 21, 256
    big = rt.alloc(2 * B * cap * width * 4)
    r = np.random.default_rng(4)
    n, budget = 500, 100
    rows = r.standard_normal((2, B, n, width)).astype(f32)
    weights = r.uniform(0, 1, (B, n)).astype(f32)
    for plane in range(2):
        for b in range(B):
            big.offset((plane * B + b) * cap * width * 4).upload(rows[plane, b])
    dw = rt.alloc(B * cap * 4)
    for b in range(B):
        dw.offset(b * cap * 4).upload(weights[b])
    dn, kept = rt.upload(np.full(B, n, np.uint32)), rt.empty(B * budget, np.uint32)
    rt.kv_evict("f32", big, big, dw, dw, dn, dn, kept, B, cap, width, budget, 10)
    rt.sync()
    small = rows.reshape(2, B * n, width).view(np.uint8)
    exp = ref.evict(small, weights, np.full(B, n), n, budget, 10, small, weights)
    for plane in range(2):
        for b in range(B):
            got = big.offset((plane * B + b) * cap * width * 4, np.uint8).download(n * width * 4)
            assert np.array_equal(got.reshape(n, -1), exp[0].reshape(2, B, n, -1)[plane, b]), (plane, b)
    assert np.array_equal(kept.download(B * budget, np.uint32).reshape(B, budget), exp[3])
    rt.free(big)
    rt.free(dw)


def test_kv_evict_graph_replays(rt):
    """An in-place cut in a graph: each replay cuts what the cache then holds."""
    say("graph")
    r = np.random.default_rng(8)
    B, cap, width, budget = 5, 400, 64, 150
    dc, dw, dn = rt.empty(2 * B * cap * width), rt.empty(B * cap), rt.empty(B, np.uint32)
    kept = rt.empty(B * budget, np.uint32)
    rt.graph_begin()
    rt.kv_evict("f32", dc, dc, dw, dw, dn, dn, kept, B, cap, width, budget, 20)
    graph = rt.graph_end()
    for i in range(4):
        cache, w = ref.make_cache(r, "f32", B * cap, width), weights_of(r, "plain", B, cap)
        n = r.integers(0, cap + 1, B, dtype=np.uint32)
        dc.upload(cache), dw.upload(w), dn.upload(n)
        rt.graph_launch(graph)
        rt.sync()
        got = (dc.download(cache.size, np.uint8).reshape(cache.shape), dw.download(w.size).reshape(w.shape),
               dn.download(B, np.uint32), kept.download(B * budget, np.uint32).reshape(B, budget))
        exp = ref.evict(cache, w, n, cap, budget, 20, cache, w)
        check(f"replay {i}", got, exp)
        rt.graph_launch(graph)  # nothing is left to cut
        rt.sync()
        assert np.array_equal(dn.download(B, np.uint32), exp[2])
        assert np.array_equal(dc.download(cache.size, np.uint8).reshape(cache.shape), exp[0])
    rt.graph_destroy(graph)


def test_kv_evict_refusals(rt):
    say("refusals")
    B, cap, width = 2, 16, 64
    dc, oc, dw, dn = rt.empty(2 * B * cap * width), rt.empty(2 * B * cap * width), rt.empty(B * cap), rt.upload(np.asarray([5, 16], np.uint32))
    kept = rt.empty(B * 8, np.uint32)
    good = dict(fmt="f32", cache=dc, cache_out=oc, weights=dw, weights_out=dw, lengths=dn, lengths_out=dn, kept=kept,
                sequences=B, capacity=cap, kv_width=width, budget=8, recent=2)
    bad = [dict(cache=None), dict(cache_out=None), dict(weights=None), dict(weights_out=None), dict(lengths=None),
           dict(lengths_out=None), dict(kept=None), dict(sequences=0), dict(capacity=0), dict(kv_width=0),
           dict(budget=0), dict(budget=17), dict(recent=9), dict(fmt="q8_0", kv_width=48), dict(fmt="q4_0", kv_width=16),
           dict(cache=dc.ptr + 2), dict(cache_out=dc.ptr + 64), dict(weights_out=dw.ptr + 4), dict(lengths_out=dn.ptr + 4),
           dict(kept=kept.ptr + 1), dict(fmt="q8_0", cache=dc.ptr + 1), dict(sequences=1 << 31, capacity=16)]
    for change in bad:
        with pytest.raises(OperatorError) as e:
            rt.kv_evict(**{**good, **change})
        assert e.value.kind == "InvalidInput", change
