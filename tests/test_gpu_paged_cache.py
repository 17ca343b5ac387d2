"""GPU tests of appending to a paged cache with rotation and of reading it back:
every byte of the pool against the layout's restatement (test_paged_checks.py
holds that against the headers), the rotation against the reference's, rounded
step by step; nothing else in the pool changes."""
import sys

import numpy as np
import pytest

import paged_refs as ref
from atlas_amd import HipRuntime, OperatorError

pytestmark = pytest.mark.gpu
f32, u32 = np.float32, np.uint32
FORMATS = ["f32", "f16", "q8_0", "q4_0"]


def say(msg):
    print(f"[gpu-paged-cache] {msg}", flush=True)
    sys.stdout.flush()


def angles(r, positions, D):
    a = r.uniform(-3, 3, (positions, D // 2))
    return np.cos(a).astype(f32), np.sin(a).astype(f32)


def make_table(r, B, width, pages, missing=0.0):
    table = r.permutation(pages)[:B * width].reshape(B, width).astype(u32)
    table[r.random((B, width)) < missing] = ref.NO
    return table


def device(rt, fmt, pool, table):
    dp, dt = rt.upload(pool.bytes), rt.upload(table)
    return dp, dt, rt.paged_cache(fmt, dp, pool.bytes.shape[0], pool.ps, pool.KH, pool.D, dt, *table.shape)


def run_append(rt, fmt, pool, table, key, value, query, cos, sin, ids, positions, in_place=False):
    """The pool's bytes and the queries after the call, and as they should be."""
    dp, dt, cache = device(rt, fmt, pool, table)
    up = lambda x: None if x is None else rt.upload(x)  # noqa: E731
    dk, dv, dq, dc, ds, di, dn = up(key), up(value), up(query), up(cos), up(sin), up(ids), up(positions)
    fill = None if query is None else (query.copy() if in_place else np.full_like(query, -7.0))
    dqo = None if query is None else (dq if in_place else rt.upload(fill))
    H = 0 if query is None else query.shape[1]
    rt.paged_append(cache, dk, dv, dq, dqo, dc, ds, 0 if cos is None else cos.shape[0], 0 if cos is None else cos.shape[1], di, dn,
                    len(positions), H)
    rt.sync()
    got = dp.download(pool.bytes.size, np.uint8).reshape(pool.bytes.shape)
    q_got = None if query is None else dqo.download(query.size).reshape(query.shape)
    if query is not None and not in_place:
        assert np.array_equal(dq.download(query.size).reshape(query.shape), query)
    ref.append(pool, table, key, value, query, fill, cos, sin, ids, positions)
    for b in {id(x): x for x in (dp, dt, dk, dv, dq, dc, ds, di, dn, dqo) if x is not None}.values():
        rt.free(b)
    return got, q_got, fill


def same(name, got, exp):
    assert np.array_equal(got, exp), f"{name}: {int((got != exp).sum())} of {exp.size} differ, first {np.argwhere(got != exp)[0]}"


# q heads, KV heads, head_dim
HEADS = [(1, 1, 32), (9, 3, 64), (12, 2, 96), (8, 2, 128), (8, 2, 160), (3, 1, 192), (7, 1, 224), (8, 1, 256)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "x".join(map(str, h)))
def test_append_writes_the_rows_and_nothing_else(rt, fmt, heads):
    """A decode step of a batch with padding, missing pages, and a prompt of consecutive positions over page borders."""
    H, KH, D = heads
    say(f"{fmt} {heads}")
    r = np.random.default_rng(D + H)
    ps, B, width = 16, 5, 4
    pool = ref.Pool(fmt, 23, ps, KH, D, fill=0xA5)
    table = make_table(r, B, width, 23)
    table[2, 1] = ref.NO
    table[3, 3] = 23  # the first number that names no page
    cos, sin = angles(r, width * ps, D)
    ids = np.array([0, 1, 2, 2, 4, 5, ref.NO, 3] + [1] * 21 + [4] * 30, u32)
    positions = np.array([63, 0, 16, 31, 64, 3, 3, 50] + list(range(5, 26)) + list(range(30)), u32)
    T = len(ids)
    key, value = r.standard_normal((2, T, KH, D)).astype(f32)
    query = r.standard_normal((T, H, D)).astype(f32)
    for in_place in (False, True):
        got, q, q_exp = run_append(rt, fmt, pool, table, key, value, query, cos, sin, ids, positions, in_place)
        same("queries", q.view(u32), q_exp.view(u32))
        same("pool", got, pool.bytes)
        key, value = -value, key * f32(0.37)


@pytest.mark.parametrize("fmt,D", [("f32", 4), ("f32", 20), ("f32", 36), ("f32", 72), ("f32", 252), ("f16", 8), ("f16", 40), ("f16", 200)])
def test_append_and_read_of_odd_head_sizes(rt, fmt, D):
    say(f"{fmt} {D}")
    r = np.random.default_rng(D)
    pool = ref.Pool(fmt, 9, 16, 3, D, fill=0x11)
    table = make_table(r, 3, 3, 9)
    cos, sin = angles(r, 48, D)
    key, value = r.standard_normal((2, 3, 3, D)).astype(f32)
    query = r.standard_normal((3, 5, D)).astype(f32)
    positions = np.array([47, 0, 17], u32)
    got, q, q_exp = run_append(rt, fmt, pool, table, key, value, query, cos, sin, None, positions)
    same("queries", q.view(u32), q_exp.view(u32))
    same("pool", got, pool.bytes)
    check_read(rt, fmt, pool, table, None, positions)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("ps", [16, 64, 4096])
def test_append_without_rotation_and_with_wide_tables(rt, fmt, ps):
    say(f"{fmt} pages of {ps}")
    r = np.random.default_rng(ps)
    KH, D, B = 2, 64, 2
    pool = ref.Pool(fmt, 4, ps, KH, D)
    table = make_table(r, B, 2, 4)
    positions = np.array([ps - 1, ps, 2 * ps - 1, 3], u32)
    ids = np.array([0, 1, 0, 1], u32)
    key, value = r.standard_normal((2, 4, KH, D)).astype(f32)
    got, _, _ = run_append(rt, fmt, pool, table, key, value, None, None, None, ids, positions)
    same("pool", got, pool.bytes)
    wide = [np.concatenate([a, np.full((2 * ps, 5), 9, f32)], 1) for a in angles(r, 2 * ps, D)]  # a stride of its own
    query = r.standard_normal((4, 6, D)).astype(f32)
    dp, dt, cache = device(rt, fmt, pool, table)
    dq = rt.upload(query)
    rt.paged_append(cache, rt.upload(key), rt.upload(value), dq, dq, rt.upload(wide[0]), rt.upload(wide[1]), 2 * ps, D // 2 + 5,
                    rt.upload(ids), rt.upload(positions), 4, 6)
    rt.sync()
    out = query.copy()
    ref.append(pool, table, key, value, query, out, wide[0][:, :D // 2], wide[1][:, :D // 2], ids, positions)
    same("queries", dq.download(query.size).reshape(query.shape), out)
    same("pool", dp.download(pool.bytes.size, np.uint8).reshape(pool.bytes.shape), pool.bytes)


@pytest.mark.parametrize("fmt", ["q8_0", "q4_0", "f16"])
def test_values_at_the_borders_of_the_encoders(rt, fmt):
    """Blocks of zeros, of equal magnitudes of both signs, of ties, of the largest and smallest numbers, infinite, NaN."""
    D, KH = 128, 1
    x = np.zeros((16, D), f32)
    x[1] = np.where(np.arange(D) % 2, 1.5, -1.5)
    x[2] = np.where(np.arange(D) % 2, -1.5, 1.5)
    x[3] = np.arange(D) - 63.5
    x[4] = np.where(np.arange(D) % 32 == 31, 127.0, np.arange(D) % 7 + 0.5)
    x[5] = 1e-45
    x[6] = np.where(np.arange(D) % 32 == 3, 3e38, 1.0)
    x[7] = 65519.0 + np.arange(D) * 0.25
    x[8, ::5] = np.nan
    x[8, 1::5] = 2.0
    x[9] = np.nan
    x[10] = -0.0
    x[11] = 2.0 ** -24 * (np.arange(D) - 64) / 2
    x[12, 7] = -8.0
    x[13, 7] = 8.0
    r = np.random.default_rng(3)
    x[14] = np.round(r.standard_normal(D) * 64) / 8 + 0.0625
    x[15, :64] = 4.0
    pool = ref.Pool(fmt, 1, 16, KH, D, fill=0xFF)
    table = np.zeros((1, 1), u32)
    rows = x[:, None]
    got, _, _ = run_append(rt, fmt, pool, table, rows, np.ascontiguousarray(rows[::-1]), None, None, None, np.zeros(16, u32),
                           np.arange(16, dtype=u32))
    if fmt == "f16":  # NaN of any bits
        g, e = got.view(np.float16), pool.bytes.view(np.float16)
        assert np.array_equal(np.isnan(g), np.isnan(e))
        got, pool.bytes = np.where(np.isnan(g), 0, g), np.where(np.isnan(e), 0, e)
    same("pool", got, pool.bytes)


def check_read(rt, fmt, pool, table, ids, positions):
    dp, dt, cache = device(rt, fmt, pool, table)
    n = len(positions)
    di, dn = None if ids is None else rt.upload(ids), rt.upload(positions)
    exp = np.zeros((2, n, pool.KH, pool.D))
    for t, p in enumerate(positions):
        b = t if ids is None else int(ids[t])
        if b < table.shape[0] and int(p) // pool.ps < table.shape[1] and table[b, int(p) // pool.ps] < pool.bytes.shape[0]:
            for plane in range(2):
                for h in range(pool.KH):
                    exp[plane, t, h] = pool.values(int(table[b, int(p) // pool.ps]), plane, h)[int(p) % pool.ps]
    for which in ((0, 1), (0,), (1,)):
        out = [rt.upload(np.full((n, pool.KH, pool.D), 5, f32)) for _ in range(2)]
        rt.paged_read(cache, di, dn, n, *(out[i] if i in which else None for i in range(2)))
        rt.sync()
        for plane in range(2):
            got = out[plane].download().reshape(exp[plane].shape)
            # a code times a scale is an f32 number: no rounding
            assert np.array_equal(got, exp[plane].astype(f32) if plane in which else np.full_like(got, 5)), (which, plane)
        for b in out:
            rt.free(b)
    for b in [dp, dt, dn] + ([] if di is None else [di]):
        rt.free(b)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "x".join(map(str, h)))
def test_read_gives_the_rows_back(rt, fmt, heads):
    _, KH, D = heads
    say(f"{fmt} {heads}")
    r = np.random.default_rng(D)
    pool = ref.Pool(fmt, 20, 16, KH, D).random(r)
    table = make_table(r, 4, 5, 20, missing=0.2)
    ids = r.integers(0, 5, 70).astype(u32)  # 4: no such sequence
    positions = r.integers(0, 85, 70).astype(u32)
    positions[::11] = ref.NO
    check_read(rt, fmt, pool, table, ids, positions)
    check_read(rt, fmt, pool, table, None, positions[:3])


def test_rows_behind_four_gigabytes(rt):
    """The last page of a pool of more than 2^32 bytes."""
    KH, D, ps, pages = 8, 256, 4096, 70
    nbytes = rt.paged_cache_bytes("f32", pages, ps, KH, D)
    assert nbytes == pages * 2 * KH * ps * D * 4 > 1 << 32
    dp = rt.alloc(nbytes)
    table = np.array([[pages - 1, 0]], u32)
    dt = rt.upload(table)
    cache = rt.paged_cache("f32", dp, pages, ps, KH, D, dt, 1, 2)
    r = np.random.default_rng(1)
    key, value = r.standard_normal((2, 3, KH, D)).astype(f32)
    ids, positions = rt.upload(np.zeros(3, u32)), rt.upload(np.array([0, ps - 1, ps], u32))
    rt.paged_append(cache, rt.upload(key), rt.upload(value), None, None, None, None, 0, 0, ids, positions, 3, 0)
    k, v = rt.empty(key.size), rt.empty(key.size)
    rt.paged_read(cache, ids, positions, 3, k, v)
    rt.sync()
    same("keys", k.download().reshape(key.shape), key)
    same("values", v.download().reshape(key.shape), value)
    head = dp.offset((pages - 1) * (nbytes // pages)).download(D)
    same("the page's first row", head, key[0, 0])
    rt.free(dp)


@pytest.mark.parametrize("fmt", ["f32", "q4_0"])
def test_more_rows_than_the_caches_hold(rt, fmt):
    """Rotated queries of 39 MB in a call, and rows of 39 MB read back: the same as a few."""
    r = np.random.default_rng(4)
    KH, D, H, T = 1, 64, 16, 9500
    pool = ref.Pool(fmt, 20, 1024, KH, D)
    table = make_table(r, 2, 5, 20)
    table[1, 2] = ref.NO
    cos, sin = angles(r, 5120, D)
    ids, positions = np.repeat(np.arange(2, dtype=u32), T // 2), np.tile(np.arange(T // 2, dtype=u32), 2)
    key, value = r.standard_normal((2, T, KH, D)).astype(f32)
    query = r.standard_normal((T, H, D)).astype(f32)
    got, q, q_exp = run_append(rt, fmt, pool, table, key, value, query, cos, sin, ids, positions)
    same("queries", q.view(u32), q_exp.view(u32))
    same("pool", got, pool.bytes)

    dp, dt, cache = device(rt, fmt, pool, table)
    n = 76000
    ids, positions = r.integers(0, 2, n).astype(u32), r.integers(0, 5120, n).astype(u32)
    di, dn, k, v = rt.upload(ids), rt.upload(positions), rt.empty(n * D), rt.empty(n * D)
    rt.paged_read(cache, di, dn, n, k, v)
    rt.sync()
    held = np.stack([np.concatenate([pool.values(int(p), plane, 0) if p != ref.NO else np.zeros((1024, D)) for p in table.reshape(-1)])
                     for plane in range(2)]).astype(f32)
    rows = ids.astype(np.int64) * 5120 + positions
    same("keys", k.download().reshape(n, D), held[0, rows])
    same("values", v.download().reshape(n, D), held[1, rows])
    for b in (dp, dt, di, dn, k, v):
        rt.free(b)


def test_refusals(rt):
    pool = ref.Pool("f32", 2, 16, 1, 64)
    dp, dt, cache = device(rt, "f32", pool, np.zeros((2, 1), u32))
    x, p = rt.empty(4 * 64), rt.upload(np.zeros(4, u32))
    with pytest.raises(OperatorError, match="more tokens than sequences") as e:
        rt.paged_append(cache, x, x, None, None, None, None, 0, 0, None, p, 3, 0)
    assert e.value.kind == "InvalidInput"
    with pytest.raises(OperatorError, match="power of two"):
        rt.paged_cache_bytes("f32", 2, 24, 1, 64)
    with pytest.raises(OperatorError, match="more rows than sequences"):
        rt.paged_read(cache, None, p, 3, x, None)
    with pytest.raises(OperatorError, match="overlap"):
        rt.paged_read(cache, None, p, 2, dp, None)
    with pytest.raises(OperatorError, match="null"):
        rt.paged_append(cache, None, x, None, None, None, None, 0, 0, None, p, 2, 0)
    rt.paged_read(cache, None, p, 2, x, None)
    rt.sync()


def test_two_contexts_and_replays_from_new_tables():
    """A recorded append and read follow the table, ids and positions as they are at each replay."""
    rt = HipRuntime(0)
    try:
        r = np.random.default_rng(8)
        pool = ref.Pool("q8_0", 12, 16, 2, 64)
        table = make_table(r, 3, 2, 12)
        dp, dt, cache = device(rt, "q8_0", pool, table)
        cos, sin = angles(r, 32, 64)
        dc, ds = rt.upload(cos), rt.upload(sin)
        key, value, query = (r.standard_normal((3, h, 64)).astype(f32) for h in (2, 2, 4))
        dk, dv, dq, dn = rt.upload(key), rt.upload(value), rt.upload(query), rt.empty(3, u32)
        qo, ko, vo = rt.empty(query.size), rt.empty(key.size), rt.empty(key.size)

        def enqueue():
            rt.paged_append(cache, dk, dv, dq, qo, dc, ds, 32, 32, None, dn, 3, 4)
            rt.paged_read(cache, None, dn, 3, ko, vo)

        rt.graph_begin()
        enqueue()
        graph = rt.graph_end()
        for step in range(4):
            positions = r.integers(0, 32, 3).astype(u32)
            table = make_table(r, 3, 2, 12, missing=0.2)
            key = r.standard_normal(key.shape).astype(f32)
            dn.upload(positions)
            dt.upload(table)
            dk.upload(key)
            rt.sync()
            rt.graph_launch(graph)
            rt.sync()
            q_exp = np.empty_like(query)
            ref.append(pool, table, key, value, query, q_exp, cos, sin, None, positions)
            same(f"pool {step}", dp.download(pool.bytes.size, np.uint8).reshape(pool.bytes.shape), pool.bytes)
            same(f"queries {step}", qo.download().reshape(query.shape), q_exp)
            first = [ko.download(), vo.download()]
            rt.memset(ko, 0xEE, ko.nbytes)
            enqueue()
            rt.sync()
            same(f"read {step}", np.concatenate(first), np.concatenate([ko.download(), vo.download()]))
        rt.graph_destroy(graph)
    finally:
        rt.close()
