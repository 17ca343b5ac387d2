"""GPU tests of the attention of one token over a paged cache (f32, f16, Q8_0,
Q4_0) against float64, within the bound that paged_refs.attention_bound derives,
and normwise within 1e-5 as the header promises."""
import sys

import numpy as np
import pytest

import paged_refs as ref
from atlas_amd import HipRuntime, OperatorError

pytestmark = pytest.mark.gpu
f32, u32 = np.float32, np.uint32
FORMATS = ["f32", "f16", "q8_0", "q4_0"]


def say(msg):
    print(f"[gpu-paged-attention] {msg}", flush=True)
    sys.stdout.flush()


def make(seed, fmt, H, KH, D, ps, cap, lengths, missing=0.0, q_std=2.0, spare=3):
    r = np.random.default_rng(seed)
    B, width = len(lengths), -(-cap // ps)
    pages = B * width + spare
    pool = ref.Pool(fmt, pages, ps, KH, D).random(r)
    table = r.permutation(pages)[:B * width].reshape(B, width).astype(u32)
    table[r.random(table.shape) < missing] = ref.NO
    return pool, table, (r.standard_normal((B, H, D)) * q_std).astype(f32), np.asarray(lengths, u32)


def run(rt, fmt, pool, table, q, lengths, window, scale):
    B, H, D = q.shape
    dp, dt, dq, dn = rt.upload(pool.bytes), rt.upload(table), rt.upload(q), rt.upload(lengths)
    cache = rt.paged_cache(fmt, dp, pool.bytes.shape[0], pool.ps, pool.KH, D, dt, *table.shape)
    out = rt.empty(q.size)
    rt.memset(out, 0xFF, q.nbytes)
    nbytes = rt.paged_attention_workspace(cache, H)
    ws = rt.alloc(nbytes + 256)
    rt.memset(ws, 0xFF, nbytes + 256)
    rt.paged_attention(cache, dq, dn, out, H, scale, window, ws, nbytes)
    rt.sync()
    got = out.download(q.size).reshape(q.shape)
    assert (ws.download(nbytes + 256, np.uint8)[nbytes:] == 0xFF).all(), "wrote behind the workspace"
    for b in (dp, dt, dq, dn, out, ws):
        rt.free(b)
    return got


def check(name, fmt, pool, table, q, lengths, window, scale, got):
    exp = ref.attention(pool, table, q, lengths, window, scale)
    tol = ref.attention_bound(fmt, pool, table, q, lengths, window, scale, exp)
    assert np.isfinite(got).all(), f"{name}: not finite"
    off = np.abs(got.astype(np.float64) - exp[0])
    worst, norm = float((off / tol).max()), float(np.linalg.norm(off) / max(np.linalg.norm(exp[0]), 1e-300))
    say(f"{name}: normwise {norm:.2e}, of the elementwise bound {worst:.3f}")
    assert worst <= 1.0 and norm <= 1e-5, name


# name: q heads, KV heads, head_dim, page size, capacity, lengths, window
SHAPES = {
    "one_key": (1, 1, 32, 16, 16, [1], 0),
    "nothing": (8, 2, 64, 16, 32, [0, 0], 0),
    "empty_rows": (8, 1, 128, 16, 48, [0, 1, 17, 48], 0),
    "smol": (9, 3, 64, 16, 2048, [701], 0),
    "edges_16": (4, 1, 256, 16, 144, [15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 143, 144], 0),
    "clamped": (4, 2, 96, 16, 32, [33, 4000000000, 32], 0),
    "every_head": (16, 1, 192, 32, 200, [200, 3], 0),
    "more_than_16": (24, 1, 64, 16, 300, [300, 1, 77], 0),
    "more_than_32": (71, 1, 64, 16, 150, [150, 149], 0),
    "no_groups": (32, 32, 64, 16, 64, [61, 2], 0),
    "five_blocks": (8, 2, 160, 64, 300, [300, 5], 0),
    "six_blocks": (6, 1, 192, 64, 300, [299, 64], 0),
    "seven_blocks": (7, 1, 224, 16, 300, [298, 16], 0),
    "wide_rows": (16, 16, 256, 16, 48, [48, 40], 0),
    "big_pages": (8, 1, 256, 4096, 5000, [4999, 4097, 1], 0),
    "window": (8, 1, 256, 16, 400, [0, 1, 49, 50, 51, 100, 131, 400], 50),
    "window_of_one": (8, 2, 64, 16, 300, [0, 1, 2, 65, 300], 1),
    "window_wider": (4, 1, 128, 16, 100, [100, 7], 1000),
    "batch": (8, 1, 256, 32, 520, [(37 * i) % 521 for i in range(70)], 0),
    "many": (4, 4, 32, 16, 40, [(7 * i) % 41 for i in range(700)], 0),
    "one_long": (8, 1, 256, 64, 30001, [30001], 0),
    "long_window": (8, 2, 128, 16, 20000, [20000, 19999, 1234], 5000),
    "ragged": (32, 8, 128, 16, 3000, [1, 3000, 40, 2999, 0, 777], 0),
}


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", list(SHAPES))
def test_attention(rt, fmt, shape):
    H, KH, D, ps, cap, lengths, window = SHAPES[shape]
    args = make(len(shape) + D, fmt, H, KH, D, ps, cap, lengths)
    say(f"{shape} {fmt}")
    got = run(rt, fmt, *args, window, D ** -0.5)
    check(f"{shape} {fmt}", fmt, *args, window, D ** -0.5, got)


@pytest.mark.parametrize("fmt,D", [("f32", 4), ("f32", 20), ("f32", 36), ("f32", 72), ("f32", 100), ("f32", 252), ("f16", 8),
                                   ("f16", 40), ("f16", 72), ("f16", 200), ("f16", 248)])
def test_odd_head_sizes(rt, fmt, D):
    """Behind the last row of a part comes another head's, of numbers that are none."""
    pool, table, q, lengths = make(D, fmt, 6, 2, D, 16, 100, [100, 31, 16])
    kind = f32 if fmt == "f32" else np.float16
    x = pool.bytes.view(kind).reshape(*pool.bytes.shape[:3], 16, D)
    used = np.isin(np.arange(len(x)), table)
    x[~used] = np.nan
    for b, n in enumerate(lengths):
        for e in range(table.shape[1]):
            x[table[b, e], :, :, max(0, min(16, int(n) - 16 * e)):] = np.nan
    say(f"{fmt} {D}")
    got = run(rt, fmt, pool, table, q, lengths, 0, D ** -0.5)
    check(f"{fmt} {D}", fmt, pool, table, q, lengths, 0, D ** -0.5, got)


@pytest.mark.parametrize("fmt", FORMATS)
def test_what_is_not_seen_may_hold_anything(rt, fmt):
    """Rows behind a sequence's end and in front of its window, and pages of no sequence: NaN and infinities."""
    for window in (0, 21):
        pool, table, q, lengths = make(5, fmt, 8, 2, 64, 16, 120, [120, 33, 1, 0, 70])
        clean = pool.bytes.copy()
        got = run(rt, fmt, pool, table, q, lengths, window, 0.125)
        check(f"clean {fmt}", fmt, pool, table, q, lengths, window, 0.125, got)
        for worst in (0xFF, 0x7C):  # NaN; f16: 0x7c7c NaN, codes and scales of all kinds
            pool.bytes = np.full_like(clean, worst)
            if worst == 0x7C and fmt != "f32":
                half = pool.bytes.view(np.float16)
                half[...] = np.inf
            spots = ref.Pool(fmt, len(clean), 16, 2, 64)
            spots.bytes = clean
            for b, n in enumerate(lengths):
                lo = max(0, int(n) - window) if window else 0
                for p in range(lo, int(n)):
                    for part, src in zip(pool.bytes[table[b, p // 16]].reshape(4, -1), clean[table[b, p // 16]].reshape(4, -1)):
                        at, scales = spots._spots(p % 16)
                        part[at] = src[at]
                        if fmt in ("q8_0", "q4_0"):
                            for s in scales:
                                part[s:s + 2] = src[s:s + 2]
            again = run(rt, fmt, pool, table, q, lengths, window, 0.125)
            assert np.array_equal(got, again), (fmt, window, worst)


@pytest.mark.parametrize("fmt", FORMATS)
def test_missing_pages(rt, fmt):
    """Entries that name no page: some, the first, the last, all of a sequence's."""
    pool, table, q, lengths = make(6, fmt, 8, 2, 128, 16, 400, [400, 399, 100, 64, 17, 400], missing=0.4)
    table[2] = ref.NO
    table[3] = [len(pool.bytes), 0xFFFFFFFE] + [ref.NO] * (table.shape[1] - 2)
    table[4, 0] = ref.NO
    table[5, 1:] = ref.NO
    for window in (0, 40):
        got = run(rt, fmt, pool, table, q, lengths, window, 0.09)
        assert (got[2:4] == 0).all()
        check(f"{fmt} window {window}", fmt, pool, table, q, lengths, window, 0.09, got)


@pytest.mark.parametrize("fmt", FORMATS)
def test_shared_pages(rt, fmt):
    pool, table, q, lengths = make(7, fmt, 4, 1, 64, 16, 160, [160, 100, 90])
    table[1:, :5] = table[0, :5]
    table[2, 3] = table[2, 4]  # and one page twice
    got = run(rt, fmt, pool, table, q, lengths, 0, 0.125)
    check(fmt, fmt, pool, table, q, lengths, 0, 0.125, got)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kind", ["large", "small", "one_hot", "equal", "zero"])
def test_queries_of_all_sizes(rt, fmt, kind):
    """Scores of thousands and of almost nothing, a key that takes all, keys alike, no query at all; other heads stay as they
    are."""
    pool, table, q, lengths = make(8, fmt, 8, 2, 128, 64, 1000, [1000, 513])
    q[:, 1] *= {"large": 300.0, "small": 1e-20, "one_hot": 0.0, "equal": 0.0, "zero": 0.0}[kind]
    if kind == "one_hot":
        q[:, 1, 5] = 1e4
    if kind == "equal":
        q[:, 1, ::2] = 1e-3
    scale = 128 ** -0.5
    got = run(rt, fmt, pool, table, q, lengths, 0, scale)
    check(f"{fmt} {kind}", fmt, pool, table, q, lengths, 0, scale, got)


def test_queries_far_apart_in_size(rt):
    """A query's largest number where the keys are zero leaves the others their digits, within 2^-38 of it."""
    for fmt in FORMATS:
        pool, table, q, lengths = make(9, fmt, 4, 1, 64, 16, 200, [200])
        if fmt in ("f32", "f16"):
            pool.bytes.view(f32 if fmt == "f32" else np.float16).reshape(-1, 2, 1, 16, 64)[:, 0, :, :, 7] = 0
            q[:, :, 7] = 1e6
        got = run(rt, fmt, pool, table, q, lengths, 0, 0.125)
        check(fmt, fmt, pool, table, q, lengths, 0, 0.125, got)


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_query_that_is_no_number_stays_alone(rt, fmt):
    pool, table, q, lengths = make(10, fmt, 8, 2, 64, 16, 300, [300, 40, 0])
    got = run(rt, fmt, pool, table, q, lengths, 0, 0.125)
    q[0, 3] = np.nan
    q[1, 6, 5] = np.inf
    again = run(rt, fmt, pool, table, q, lengths, 0, 0.125)
    assert np.isnan(again[0, 3]).all() and not np.isfinite(again[1, 6]).any()
    again[0, 3], again[1, 6] = got[0, 3], got[1, 6]
    assert np.array_equal(got, again)


@pytest.mark.parametrize("fmt", FORMATS)
def test_scales_and_values_of_all_sizes(rt, fmt):
    """Numbers near the ends of the formats: f16's largest and smallest, f32's wide range."""
    for power in ((-40, -20, 40) if fmt == "f32" else (-13, 8)):
        pool, table, q, lengths = make(11, fmt, 4, 2, 64, 16, 300, [300, 33])
        if fmt in ("f32", "f16"):
            x = pool.bytes.view(f32 if fmt == "f32" else np.float16)
            x *= x.dtype.type(2.0) ** x.dtype.type(power)
            q = (q * 2.0 ** -power).astype(f32)
        else:
            n = 16 * ref.code_bytes(fmt, 64)
            d = np.ascontiguousarray(pool.bytes[..., n:]).view(np.float16) * np.float16(2.0) ** np.float16(power)
            pool.bytes[..., n:] = d.view(np.uint8)
            q = (q * 2.0 ** -power).astype(f32)
        got = run(rt, fmt, pool, table, q, lengths, 0, 0.125)
        check(f"{fmt} 2^{power}", fmt, pool, table, q, lengths, 0, 0.125, got)


@pytest.mark.parametrize("fmt", FORMATS)
def test_long_sums_of_keys_alike(rt, fmt):
    """Every position the same key and value: the sums' roundings all fall to one side.  The result is the value: within
    (256 + 256 + 64) 2^-24 = 3.5e-5 by the count of roundings of sum and weights alike, and in effect 1e-5."""
    H, KH, D, ps, n = 8, 1, 64, 256, 1 << 20
    pool = ref.Pool(fmt, 1, ps, KH, D).random(np.random.default_rng(4))
    for plane in range(2):
        row = np.random.default_rng(plane).standard_normal(D).astype(f32)
        for i in range(ps):
            pool.write(0, plane, 0, i, row)
    table = np.zeros((3, n // ps), u32)
    q = np.random.default_rng(2).standard_normal((3, H, D)).astype(f32)
    lengths = np.array([n, n - 1, 12345], u32)
    got = run(rt, fmt, pool, table, q, lengths, 0, 0.125).astype(np.float64)
    value = pool.values(0, 1, 0)[0]
    worst = float((np.abs(got - value) / np.maximum(np.abs(value), 1e-30)).max())
    say(f"{fmt}: {worst:.2e} of each value")
    assert worst <= 3.5e-5
    assert np.linalg.norm(got - value) <= 1e-5 * np.linalg.norm(np.broadcast_to(value, got.shape))


def test_the_same_bits_every_time_and_in_any_batch(rt):
    """A call's result does not depend on timing; the split does on the other sequences' lengths, within the bound."""
    for fmt in FORMATS:
        args = make(12, fmt, 8, 1, 256, 16, 3000, [3000, 100, 2000])
        first = run(rt, fmt, *args, 0, 0.0625)
        for _ in range(3):
            assert np.array_equal(first, run(rt, fmt, *args, 0, 0.0625))


def test_pages_behind_four_gigabytes(rt):
    KH, D, ps, pages = 8, 256, 4096, 66
    nbytes = rt.paged_cache_bytes("f32", pages, ps, KH, D)
    assert nbytes > 1 << 32
    dp = rt.alloc(nbytes)
    small, table, q, lengths = make(13, "f32", 16, KH, D, ps, 4096, [70], spare=0)
    page = nbytes // pages
    dp.offset((pages - 1) * page).upload(small.bytes)
    dt, dq, dn, out = rt.upload(np.array([[pages - 1]], u32)), rt.upload(q), rt.upload(lengths), rt.empty(q.size)
    cache = rt.paged_cache("f32", dp, pages, ps, KH, D, dt, 1, 1)
    n = rt.paged_attention_workspace(cache, 16)
    ws = rt.alloc(n)
    rt.paged_attention(cache, dq, dn, out, 16, 0.0625, 0, ws, n)
    rt.sync()
    check("far page", "f32", small, np.zeros((1, 1), u32), q, lengths, 0, 0.0625, out.download().reshape(q.shape))
    rt.free(dp)


def test_refusals(rt):
    pool, table, q, lengths = make(14, "f16", 8, 2, 64, 16, 64, [64])
    dp, dt, dq, dn, out = rt.upload(pool.bytes), rt.upload(table), rt.upload(q), rt.upload(lengths), rt.empty(q.size)
    cache = rt.paged_cache("f16", dp, len(pool.bytes), 16, 2, 64, dt, *table.shape)
    n = rt.paged_attention_workspace(cache, 8)
    ws = rt.alloc(n)
    for change, what in ((dict(bytes=n - 1), "too small"), (dict(scale=float("nan")), "finite"), (dict(out=dq), "overlaps"),
                         (dict(heads=7), "multiple"), (dict(q=None), "null")):
        with pytest.raises(OperatorError, match=what) as e:
            rt.paged_attention(cache, change.get("q", dq), dn, change.get("out", out), change.get("heads", 8),
                               change.get("scale", 0.1), 0, ws, change.get("bytes", n))
        assert e.value.kind == "InvalidInput"
    with pytest.raises(OperatorError, match="multiple"):
        rt.paged_attention_workspace(cache, 9)
    rt.paged_attention(cache, dq, dn, out, 8, 0.1, 0, ws, n)
    rt.sync()


def spread(seed, fmt, H, KH, D, ps, width, lengths):
    """Tables of `width` entries, of which the lengths need the first."""
    r = np.random.default_rng(seed)
    need = [-(-n // ps) for n in lengths]
    pool = ref.Pool(fmt, sum(need) + 2, ps, KH, D).random(r)
    order = iter(r.permutation(len(pool.bytes)))
    table = np.full((len(lengths), width), ref.NO, u32)
    for b, n in enumerate(need):
        table[b, :n] = [next(order) for _ in range(n)]
    return pool, table, (r.standard_normal((len(lengths), H, D)) * 2).astype(f32), np.asarray(lengths, u32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", range(32, 257, 32))
@pytest.mark.parametrize("how", ["split", "whole", "short"])
def test_rows_split_and_whole(rt, fmt, D, how):
    """Rows that may be long are split over workgroups and joined; many of some length, and short ones, are not.  Of 3, 8 and
    more than 16 query heads to a KV head, in each of the products' widths."""
    for group, KH in ((3, 2), (8, 1), (19, 1)):
        if how == "split":
            args = spread(D + group, fmt, group * KH, KH, D, 64, 800, [700, 33, 0, 129])
        elif how == "whole":
            args = spread(D + group, fmt, group * KH, KH, D, 16, 20, [(53 * i) % 321 for i in range(80 // KH)])
        else:
            args = spread(D + group, fmt, group * KH, KH, D, 16, 7, [112, 0, 17, 1, 64])
        for window in (0, 37) if how == "short" else (0,):
            say(f"{how} {fmt} {D} group {group} window {window}")
            got = run(rt, fmt, *args, window, D ** -0.5)
            assert (got[args[3] == 0] == 0).all()
            check(f"{how} {fmt} {D}", fmt, *args, window, D ** -0.5, got)


@pytest.mark.parametrize("fmt", FORMATS)
def test_windows_of_many_rows(rt, fmt):
    """A window bounds a row where the capacity does not: such rows are whole."""
    args = spread(3, fmt, 8, 2, 128, 16, 4000, [(211 * i) % 2001 for i in range(40)])
    got = run(rt, fmt, *args, 200, 0.09)
    check(f"{fmt}", fmt, *args, 200, 0.09, got)


def test_two_graphs_with_a_workspace_each():
    """Recorded calls of two contexts replayed together, with other lengths and tables from replay to replay."""
    rts = [HipRuntime(0), HipRuntime(0)]
    try:
        calls = []
        for i, rt in enumerate(rts):
            fmt = FORMATS[2 * i]
            pool, table, q, lengths = make(15 + i, fmt, 8, 2, 128, 16, 2000, [2000, 1, 700])
            dp, dt, dq, dn, out = rt.upload(pool.bytes), rt.upload(table), rt.upload(q), rt.upload(lengths), rt.empty(q.size)
            cache = rt.paged_cache(fmt, dp, len(pool.bytes), 16, 2, 128, dt, *table.shape)
            n = rt.paged_attention_workspace(cache, 8)
            ws = rt.alloc(n)
            rt.graph_begin()
            rt.paged_attention(cache, dq, dn, out, 8, 0.08, 0, ws, n)
            calls.append([rt, fmt, pool, table, q, lengths, dt, dn, out, rt.graph_end()])
        r = np.random.default_rng(3)
        for step in range(4):
            for c in calls:
                c[5] = r.integers(0, 2001, 3).astype(u32)
                c[3] = r.permutation(len(c[2].bytes))[:c[3].size].reshape(c[3].shape).astype(u32)
                c[6].upload(c[3])
                c[7].upload(c[5])
                c[0].memset(c[8], 0xEE, c[8].nbytes)
                c[0].sync()
            for c in calls:
                c[0].graph_launch(c[9])
            for c in calls:
                c[0].sync()
                got = c[8].download().reshape(c[4].shape)
                check(f"step {step} {c[1]}", c[1], c[2], c[3], c[4], c[5], 0, 0.08, got)
        for c in calls:
            c[0].graph_destroy(c[9])
    finally:
        for rt in rts:
            rt.close()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", range(32, 257, 32))
def test_more_rows_than_workgroups_at_once(rt, fmt, D):
    """More than 256 rows, whole and of several steps each, empty ones among them."""
    for group, KH in ((2, 3), (8, 2), (20, 1)):
        B = 320 // KH if group < 16 else 140  # 20 heads are two rows
        args = spread(D + group, fmt, group * KH, KH, D, 16, 20, [(53 * i) % 321 for i in range(B)])
        say(f"{fmt} {D} group {group}")
        got = run(rt, fmt, *args, 0, D ** -0.5)
        assert (got[args[3] == 0] == 0).all()
        check(f"{fmt} {D}", fmt, *args, 0, D ** -0.5, got)


def test_many_long_rows_of_small_heads(rt):
    """Rows of few bytes and many positions are cut where a wavefront would add too many of them up."""
    H, KH, D, ps, n = 257, 257, 4, 4096, 20000
    pool = ref.Pool("f32", 1, ps, KH, D)
    row = np.random.default_rng(1).standard_normal((2, KH, 1, D)).astype(f32)
    pool.bytes = np.ascontiguousarray(np.broadcast_to(row, (2, KH, ps, D))).view(np.uint8).reshape(pool.bytes.shape)
    table = np.zeros((1, -(-n // ps)), u32)
    q = np.random.default_rng(2).standard_normal((1, H, D)).astype(f32)
    got = run(rt, "f32", pool, table, q, np.array([n], u32), 0, 0.5).astype(np.float64)
    off = np.abs(got[0] - row[1, :, 0]) / np.abs(row[1, :, 0])
    say(f"{off.max():.2e} of each value")
    assert off.max() <= 3.5e-5 and np.linalg.norm(got[0] - row[1, :, 0]) <= 1e-5 * np.linalg.norm(row[1])


@pytest.mark.parametrize("fmt", ["q8_0", "q4_0"])
@pytest.mark.parametrize("D", range(32, 257, 32))
def test_scales_of_rows_behind_the_last(rt, fmt, D):
    """Whatever lies in a page behind a sequence's last row, scales that are no numbers too: any number of blocks, of 3, 8
    and 16 heads."""
    for group in (3, 8, 16):
        for n in (1, 5, 16, 20, 28):
            pool, table, q, lengths = spread(D + n, fmt, group * 2, 2, D, 16, 4, [n, 3])
            rows, clean = ref.Pool(fmt, len(pool.bytes), 16, 2, D), pool.bytes
            rows.bytes = np.full_like(clean, 0xFF)
            for b, length in enumerate(lengths):
                for p in range(int(length)):
                    for part, src in zip(rows.bytes[table[b, p // 16]].reshape(4, -1), clean[table[b, p // 16]].reshape(4, -1)):
                        at, scales = rows._spots(p % 16)
                        part[at] = src[at]
                        for s in scales:
                            part[s:s + 2] = src[s:s + 2]
            got = run(rt, fmt, rows, table, q, lengths, 0, D ** -0.5)
            assert np.array_equal(got, run(rt, fmt, pool, table, q, lengths, 0, D ** -0.5)), (group, n)


@pytest.mark.parametrize("n", [2, 32, 64, 700])
@pytest.mark.parametrize("most", [1, 60, 1023])
def test_f16_numbers_below_the_normal_ones(rt, n, most):
    """The matrix unit lines products up by their operands' exponents, which are 2^-14 for all f16 numbers below it, and
    drops what is 2^-24 below the largest: of a weight of 1, held as 2^15, and such a value 2^(15 - 14 - 24) = 2^-23, which
    is 2^-38 of the result for each of a step's 32 keys; of a query's largest number, held below 2^14, and such a key 2^-37
    of it for each dim."""
    r = np.random.default_rng(n + most)
    pool, table, q, lengths = make(n, "f16", 8, 2, 64, 16, max(16, n), [n] * 3)
    x = pool.bytes.view(np.float16).reshape(len(pool.bytes), 2, -1)
    small = lambda shape: (r.integers(-most, most + 1, shape) * 2.0 ** -24).astype(np.float16)  # noqa: E731
    keys = x[:, 0].copy()
    x[:, 1] = small(keys.shape)
    got = run(rt, "f16", pool, table, q, lengths, 0, 0.125)
    exp = ref.attention(pool, table, q, lengths, 0, 0.125)
    tol = ref.attention_bound("f16", pool, table, q, lengths, 0, 0.125, exp) + 2.0 ** -33
    off = np.abs(got.astype(np.float64) - exp[0])
    say(f"values {n} {most}: {float((off / tol).max()):.3f} of the bound, 2^{np.log2(off.max() + 1e-99):.1f}")
    assert (off <= tol).all()
    x[:, 0] = small(keys.shape)
    x[:, 1] = keys
    q *= f32(2.0 ** 14)
    got = run(rt, "f16", pool, table, q, lengths, 0, 0.125)
    exp = ref.attention(pool, table, q, lengths, 0, 0.125)
    dx = 64 * 2.0 ** -37 * 0.125 * np.abs(q.astype(np.float64)).max(2)[..., None]
    tol = ref.attention_bound("f16", pool, table, q, lengths, 0, 0.125, exp) + np.expm1(2 * dx) * exp[1]
    off = np.abs(got.astype(np.float64) - exp[0])
    say(f"keys {n} {most}: {float((off / tol).max()):.3f} of the bound")
    assert (off <= tol).all()
