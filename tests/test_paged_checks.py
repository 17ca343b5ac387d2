"""CPU tests of the paged decode ops: which calls are refused and that the calls
the documentation allows are not, and the layout of a page, compiled from their
headers by the host compiler; no device."""
import ctypes
import math
import os
import subprocess
from ctypes import c_char_p, c_double, c_float, c_int, c_uint32, c_uint64

import numpy as np
import pytest

import paged_refs as ref
from atlas_amd.chains import PagedDecode, PagedShape

HERE = os.path.dirname(os.path.abspath(__file__))
U32, U64 = c_uint32, c_uint64
CACHE_TYPES = [c_int, U64, U64] + [U32] * 6


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("checks") / "libpaged_checks.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__=1", "-I/opt/rocm/include",
                    "-o", so, os.path.join(HERE, "cpp", "paged_checks.cpp")], check=True)
    lib = ctypes.CDLL(so)
    lib.paged_bytes.argtypes, lib.paged_bytes.restype = CACHE_TYPES, U64
    lib.value_place.argtypes, lib.value_place.restype = [U32, U32], U32
    lib.check_append.argtypes = CACHE_TYPES + [U64] * 8 + [U32] * 4
    lib.check_read.argtypes = CACHE_TYPES + [U64] * 4 + [U32]
    lib.check_attention.argtypes = CACHE_TYPES + [U64] * 3 + [U32, U32, c_float, U64]
    lib.check_logprobs.argtypes = [U64] * 7 + [U32] * 4 + [c_double, U64]
    for f in (lib.check_append, lib.check_read, lib.check_attention, lib.check_logprobs):
        f.restype = c_char_p
    return lib


M = 1 << 40  # addresses far apart
CACHE = dict(format=0, pages=M, table=2 * M, page_count=100, page_size=16, kv_heads=2, head_dim=128, sequences=4, table_width=20)
APPEND = dict(CACHE, key=3 * M, value=4 * M, query=5 * M, query_out=6 * M, cosine=7 * M, sine=8 * M, ids=9 * M, positions=10 * M,
              rope_rows=320, rope_stride=64, tokens=7, q_heads=8)
READ = dict(CACHE, ids=3 * M, positions=4 * M, key=5 * M, value=6 * M, rows=9)
ATTEND = dict(CACHE, q=3 * M, lengths=4 * M, output=5 * M, q_heads=8, window=0, scale=0.1, workspace=6 * M)
LOGPROBS = dict(logits=M, row_stride=1000, tokens=2 * M, logprobs=3 * M, entropy=4 * M, top_ids=5 * M, top_logprobs=6 * M, rows=4,
                vocab=1000, given=1, top=5, inv_temperature=1.0, workspace=7 * M)
GOOD_CACHES = [{}, dict(format=3), dict(format=1), dict(format=2), dict(head_dim=4, rope_stride=2), dict(format=3, head_dim=8),
               dict(format=1, head_dim=256, rope_stride=128), dict(format=2, head_dim=96), dict(page_size=4096, rope_rows=81920),
               dict(kv_heads=1), dict(page_count=1), dict(page_count=1 << 20)]
BAD_CACHES = [dict(format=4), dict(format=-1), dict(pages=0), dict(table=0), dict(page_count=0), dict(page_count=0xFFFFFFFF),
              dict(page_size=0), dict(page_size=8), dict(page_size=48), dict(page_size=8192), dict(kv_heads=0),
              dict(kv_heads=257), dict(head_dim=0), dict(head_dim=6), dict(head_dim=260), dict(format=3, head_dim=12),
              dict(format=1, head_dim=48), dict(format=2, head_dim=16), dict(sequences=0), dict(sequences=(1 << 20) + 1),
              dict(table_width=0), dict(table_width=(1 << 25) + 1), dict(pages=M + 8), dict(table=2 * M + 2)]


def call(fn, base, change):
    return fn(*{**base, **{k: v for k, v in change.items() if k in base}}.values())


@pytest.mark.parametrize("change", GOOD_CACHES)
def test_caches_that_are_allowed(checks, change):
    assert call(checks.check_append, APPEND, change) is None
    assert call(checks.check_read, READ, change) is None
    assert call(checks.check_attention, ATTEND, change) is None


@pytest.mark.parametrize("change", BAD_CACHES)
def test_caches_that_are_refused(checks, change):
    for fn, base in ((checks.check_append, APPEND), (checks.check_read, READ), (checks.check_attention, ATTEND)):
        assert call(fn, base, change)


@pytest.mark.parametrize("change", [
    dict(query=0, query_out=0), dict(query=0, query_out=0, cosine=0, sine=0, rope_rows=0, rope_stride=0, q_heads=0),
    dict(query_out=5 * M), dict(ids=0, tokens=4), dict(tokens=1), dict(rope_rows=400, rope_stride=100), dict(q_heads=1),
    dict(cosine=7 * M + 4, sine=8 * M + 4), dict(tokens=(1 << 25) // 12),
])
def test_append_calls_that_are_allowed(checks, change):
    assert call(checks.check_append, APPEND, change) is None


@pytest.mark.parametrize("change", [
    dict(key=0), dict(value=0), dict(positions=0), dict(tokens=0), dict(ids=0, tokens=5), dict(cosine=0), dict(sine=0),
    dict(cosine=0, sine=0), dict(query_out=0), dict(query=0), dict(q_heads=0), dict(rope_rows=319), dict(rope_stride=63),
    dict(key=3 * M + 4), dict(value=4 * M + 8), dict(query=5 * M + 4), dict(query_out=6 * M + 4), dict(cosine=7 * M + 2),
    dict(positions=10 * M + 1), dict(ids=9 * M + 2), dict(query_out=5 * M + 16), dict(key=M + 1024), dict(value=M + 1024),
    dict(query=M + 1024), dict(query_out=M + 1024), dict(query_out=3 * M), dict(query_out=4 * M), dict(tokens=(1 << 25) // 12 + 1),
    dict(q_heads=0xFFFFFFFF),
])
def test_append_calls_that_are_refused(checks, change):
    assert call(checks.check_append, APPEND, change)


@pytest.mark.parametrize("change,fine", [
    ({}, True), (dict(key=0), True), (dict(value=0), True), (dict(ids=0, rows=4), True), (dict(rows=(1 << 25) // 4), True),
    (dict(key=0, value=0), False), (dict(positions=0), False), (dict(rows=0), False), (dict(ids=0, rows=5), False),
    (dict(key=5 * M + 4), False), (dict(value=6 * M + 4), False), (dict(key=M + 16), False), (dict(value=M + 16), False),
    (dict(value=5 * M), False), (dict(positions=4 * M + 2), False), (dict(ids=3 * M + 2), False), (dict(rows=(1 << 25) // 4 + 1), False),
])
def test_read_calls(checks, change, fine):
    assert (call(checks.check_read, READ, change) is None) == fine


@pytest.mark.parametrize("change,fine", [
    ({}, True), (dict(window=1), True), (dict(window=0xFFFFFFFF), True), (dict(q_heads=2), True), (dict(q_heads=64), True),
    (dict(scale=0.0), True), (dict(scale=-1.0), True), (dict(sequences=1 << 20, q_heads=8), True),
    (dict(q=0), False), (dict(lengths=0), False), (dict(output=0), False), (dict(workspace=0), False), (dict(q_heads=0), False),
    (dict(q_heads=7), False), (dict(scale=math.nan), False), (dict(scale=math.inf), False), (dict(q=3 * M + 4), False),
    (dict(output=5 * M + 8), False), (dict(workspace=6 * M + 8), False), (dict(lengths=4 * M + 2), False), (dict(output=3 * M), False),
    (dict(output=M + 16), False), (dict(sequences=1 << 20, q_heads=10), False),
    (dict(sequences=1 << 20, table_width=512), True), (dict(sequences=1 << 20, table_width=513), False),
    (dict(sequences=1 << 17, q_heads=64, table_width=2048), True), (dict(sequences=1 << 17, q_heads=64, table_width=2049), False),
    (dict(table_width=1 << 25), True), (dict(sequences=17, table_width=1 << 25), False),
])
def test_attention_calls(checks, change, fine):
    assert (call(checks.check_attention, ATTEND, change) is None) == fine


@pytest.mark.parametrize("change,fine", [
    ({}, True), (dict(given=0, tokens=0, logprobs=0), True), (dict(entropy=0), True), (dict(top=0, top_ids=0, top_logprobs=0), True),
    (dict(top=64), True), (dict(vocab=1), True), (dict(row_stride=1 << 40), True), (dict(vocab=1 << 29, row_stride=1 << 29), True),
    (dict(inv_temperature=5e-324), True), (dict(inv_temperature=1.7e308), True), (dict(rows=1 << 23), True),
    (dict(logits=0), False), (dict(workspace=0), False), (dict(tokens=0), False), (dict(logprobs=0), False), (dict(top_ids=0), False),
    (dict(top_logprobs=0), False), (dict(rows=0), False), (dict(vocab=0), False), (dict(top=65), False), (dict(row_stride=999), False),
    (dict(given=0, top=0, entropy=0), False), (dict(inv_temperature=0.0), False), (dict(inv_temperature=-1.0), False),
    (dict(inv_temperature=math.nan), False), (dict(inv_temperature=math.inf), False), (dict(logits=M + 2), False),
    (dict(tokens=2 * M + 2), False), (dict(workspace=7 * M + 8), False), (dict(rows=(1 << 23) + 1), False),
    (dict(vocab=(1 << 29) + 1, row_stride=1 << 30), False),
])
def test_logprob_calls(checks, change, fine):
    assert (call(checks.check_logprobs, LOGPROBS, change) is None) == fine


def test_pages_have_their_bytes(checks):
    for fmt, name in enumerate(("f32", "q8_0", "q4_0", "f16")):
        for ps in (16, 64, 4096):
            for D in (32, 96, 160, 224, 256):
                got = call(checks.paged_bytes, CACHE, dict(format=fmt, page_size=ps, head_dim=D, kv_heads=3, page_count=7))
                assert got == 7 * 2 * 3 * ref.part_bytes(name, ps, D)
                assert ref.part_bytes(name, ps, D) % 16 == 0  # every part is as aligned as the pool
    big = call(checks.paged_bytes, CACHE, dict(page_count=0xFFFFFFFE, page_size=4096, kv_heads=128, head_dim=256))
    assert big == 0xFFFFFFFE * 2 * 128 * 4096 * 1024


@pytest.mark.parametrize("D", range(32, 257, 32))
def test_a_values_codes_are_where_the_layout_says(checks, D):
    order = ref.value_order(D)
    assert sorted(order) == list(range(D))
    place = np.argsort(order)
    for d in range(0, D, 2):
        assert checks.value_place(D, d) == place[d] and place[d + 1] == place[d] + 1


def test_sequences_that_do_not_fit_change_nothing():
    """PagedDecode.begin takes all of its prompts or none, and set_step pages for all of the sequences."""
    class Runtime:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was called")

    chain = object.__new__(PagedDecode)
    chain.rt, chain.S = Runtime(), PagedShape(sequences=4, capacity=64, pages=6, page_size=16)
    chain.lengths, chain.table = np.array([16, 0, 0, 16], np.uint32), np.full((4, 4), PagedDecode.NO_PAGE, np.uint32)
    chain.table[0, 0], chain.table[3, 0] = 0, 1
    chain.free = [5]
    before = chain.lengths.copy(), chain.table.copy(), list(chain.free)

    def prompt(n):
        return [(np.zeros((n, 3, 64), np.float32),) * 2] * 3

    for prompts, what in (({1: prompt(16), 2: prompt(17)}, "no page left"), ({1: prompt(3), 0: prompt(1)}, "has a sequence"),
                          ({1: prompt(3), 2: prompt(65)}, "no room"), ({1: prompt(3), 2: prompt(0)}, "no token")):
        with pytest.raises(ValueError, match=what):
            chain.begin(prompts)
        assert (chain.lengths == before[0]).all() and (chain.table == before[1]).all() and chain.free == before[2], what
    with pytest.raises(ValueError, match="no page left"):
        chain.set_step(None)
    assert (chain.table == before[1]).all() and chain.free == before[2]


def test_a_failed_recording_leaves_no_graph_behind():
    """PagedDecode keeps no handle of the graph that a failed recording destroyed."""
    class Runtime:
        live, next = set(), 1

        def graph_begin(self):
            pass

        def graph_end(self):
            self.next += 1
            self.live.add(self.next)
            return self.next

        def graph_destroy(self, graph):
            self.live.remove(graph)  # KeyError: destroyed twice

    chain = object.__new__(PagedDecode)
    chain.rt, chain.graph = Runtime(), None
    chain.enqueue = lambda: None
    first = chain.capture()
    assert chain.graph == first and chain.rt.live == {first}

    def fails():
        raise ValueError("no")

    chain.enqueue = fails
    with pytest.raises(ValueError, match="no"):
        chain.capture()
    assert chain.graph is None and not chain.rt.live


class Nothing:
    """A runtime that no one may call."""

    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


def chain_of(rt, lengths, table, free, **shape):
    """A chain without a device: its sequences, their pages and the pool's."""
    chain = object.__new__(PagedDecode)
    chain.rt, chain.S = rt, PagedShape(sequences=len(lengths), **shape)
    chain.lengths, chain.table, chain.free = np.array(lengths, np.uint32), np.array(table, np.uint32), list(free)
    return chain


def rows_of(n, heads=3, dim=64, dtype=np.float32):
    return np.zeros((n, heads, dim), dtype)


@pytest.mark.parametrize("prompts,what", [
    ({0: [(rows_of(9), rows_of(9)), (rows_of(9), rows_of(8))]}, "every layer"),        # values of fewer tokens
    ({0: [(rows_of(9), rows_of(9)), (rows_of(8), rows_of(9))]}, "every layer"),        # keys of fewer
    ({0: [(rows_of(9), rows_of(9)), (rows_of(10), rows_of(10))]}, "every layer"),      # a layer of more
    ({0: [(rows_of(9), rows_of(9))]}, "every layer"),                                  # a layer less
    ({0: [(rows_of(9), rows_of(9))] * 3}, "every layer"),
    ({0: []}, "every layer"),
    ({0: [(rows_of(9),)] * 2}, "every layer"),
    ({0: [(rows_of(9, heads=2), rows_of(9, heads=2))] * 2}, "every layer"),
    ({0: [(rows_of(9, dim=32), rows_of(9, dim=32))] * 2}, "every layer"),
    # one prompt's more make up for the other's less
    ({0: [(rows_of(9), rows_of(9)), (rows_of(8), rows_of(8))], 1: [(rows_of(9), rows_of(9)), (rows_of(10), rows_of(10))]}, "every layer"),
    ({-1: [(rows_of(9), rows_of(9))] * 2}, "no place"),
    ({2: [(rows_of(9), rows_of(9))] * 2}, "no place"),
])
def test_prompts_that_do_not_match_are_refused(prompts, what):
    """What would be read behind a layer's rows, or stored for another sequence, changes nothing."""
    chain = chain_of(Nothing(), [0, 0], [[ref.NO] * 4] * 2, [3, 2, 1, 0], layers=2, capacity=64, pages=4)
    with pytest.raises(ValueError, match=what):
        chain.begin(prompts)
    assert not chain.lengths.any() and (chain.table == ref.NO).all() and chain.free == [3, 2, 1, 0]


@pytest.mark.parametrize("dtype", [np.float16, np.float32, np.float64])
def test_prompts_go_up_as_f32_rows(dtype):
    """Every buffer of an append has the bytes that the call reads, whatever the prompt's type."""
    class Runtime:
        def __init__(self):
            self.appended = []

        def upload(self, host):
            return np.ascontiguousarray(host)

        def paged_append(self, cache, key, value, query, query_out, cos, sin, rope_rows, rope_stride, ids, positions, tokens, heads):
            assert key.nbytes == value.nbytes == 4 * tokens * 3 * 64 and ids.nbytes == positions.nbytes == 4 * tokens
            self.appended.append((key, value))

        def sync(self):
            pass

        def free(self, buf):
            pass

    rt = Runtime()
    chain = chain_of(rt, [0, 0, 0], [[ref.NO] * 4] * 3, [5, 4, 3, 2, 1, 0], layers=2, capacity=64, pages=6)
    chain.width, chain.caches = 4, [None, None]
    chain.dev = {"table": type("Table", (), {"upload": lambda self, host: None})(), "cos": None, "sin": None}
    r = np.random.default_rng(1)
    first, second = ([tuple(r.integers(-9, 9, (n, 3, 64)).astype(dtype) for _ in range(2)) for _ in range(2)] for n in (17, 5))
    second = [tuple(x.reshape(5, 192) for x in pair) for pair in second]  # heads side by side
    chain.begin({2: first, 0: second})
    assert chain.lengths.tolist() == [5, 0, 17] and len(chain.free) == 3
    for layer, pair in enumerate(rt.appended):
        for i in range(2):
            exp = np.concatenate([first[layer][i], second[layer][i].reshape(5, 3, 64)])
            assert pair[i].dtype == np.float32 and np.array_equal(pair[i], exp.astype(np.float32))


@pytest.mark.parametrize("given,fine", [(1, True), (1 << 29, True), ((1 << 29) + 1, False), (0xFFFFFC00, False), (0xFFFFFFFF, False)])
def test_given_tokens_that_a_thread_can_count(checks, given, fine):
    """A count past 2^32 begins again at zero, and a loop up to a larger number never ends."""
    assert (call(checks.check_logprobs, LOGPROBS, dict(given=given)) is None) == fine


class Buffer:
    def upload(self, host):
        self.host = np.array(host)

    def download(self, count, dtype):
        return np.zeros(count, dtype)


def stepping_chain(lengths):
    chain = chain_of(Nothing(), lengths, [[i] + [ref.NO] * 3 if n else [ref.NO] * 4 for i, n in enumerate(lengths)], [9, 8, 7, 6, 5],
                     capacity=64, pages=10, vocab=10)
    chain.stepped = np.zeros(len(lengths), bool)
    chain.dev = {k: Buffer() for k in ("table", "positions", "lengths", "logits")}
    chain.out = {"tokens": Buffer()}
    return chain


def test_sequences_grow_by_the_steps_that_they_were_in():
    """A sequence that begins between set_step and advance has no row of that step, nor has one whose place another took; a
    second advance is of no step."""
    chain = stepping_chain([3, 0, 15, 7])
    chain.set_step(np.zeros((4, 10), np.float32))
    assert chain.dev["positions"].host.tolist() == [3, ref.NO, 15, 7] and chain.dev["lengths"].host.tolist() == [4, 0, 16, 8]
    chain.end(3)
    chain.lengths[1], chain.lengths[3] = 4, 6  # begun: prompts of 4 and 6
    chain.advance()
    assert chain.lengths.tolist() == [4, 4, 16, 6]
    chain.advance()
    assert chain.lengths.tolist() == [4, 4, 16, 6]
    chain.table[1, 0], chain.table[3, 0] = chain.free.pop(), chain.free.pop()
    chain.set_step(np.zeros((4, 10), np.float32))
    assert chain.dev["positions"].host.tolist() == [4, 4, 16, 6]
    chain.advance()
    assert chain.lengths.tolist() == [5, 5, 17, 7] and chain.lengths.dtype == np.uint32


@pytest.mark.parametrize("logits", [np.zeros((3, 10)), np.zeros((4, 9), np.float32), np.zeros((2, 4, 10), np.float32), np.zeros(0), None])
def test_a_step_without_its_logits_changes_nothing(logits):
    """Fewer numbers than the step has would leave the last step's logits of other sequences in their place."""
    chain = stepping_chain([16, 0, 5, 0])
    table = chain.table.copy()
    with pytest.raises(ValueError, match="logits"):
        chain.set_step(logits)
    assert (chain.table == table).all() and chain.free == [9, 8, 7, 6, 5] and not hasattr(chain.dev["table"], "host")


@pytest.mark.parametrize("dtype", [np.float16, np.float32, np.float64])
def test_a_steps_logits_go_up_as_f32(dtype):
    chain = stepping_chain([16, 0, 5, 0])
    x = (np.arange(40).reshape(4, 10) - 20).astype(dtype)
    chain.set_step(x)
    assert chain.dev["logits"].host.dtype == np.float32 and np.array_equal(chain.dev["logits"].host, x.astype(np.float32))
    assert chain.table[0].tolist() == [0, 5, ref.NO, ref.NO] and chain.free == [9, 8, 7, 6]


@pytest.mark.parametrize("call_that_fails", range(1, 10))
def test_prompts_that_could_not_be_stored_leave_no_sequence(call_that_fails):
    """A device without memory, or a call that fails half-way through the layers: pages and buffers come back."""
    class Runtime:
        calls, live = 0, 0

        def step(self):
            self.calls += 1
            if self.calls == call_that_fails:
                raise RuntimeError("no memory")

        def upload(self, host):
            self.step()
            self.live += 1
            return object()

        def paged_append(self, *args):
            self.step()

        def sync(self):
            self.step()

        def free(self, buf):
            self.live -= 1

    chain = chain_of(Runtime(), [0, 3, 0], [[ref.NO] * 4, [9, ref.NO, ref.NO, ref.NO], [ref.NO] * 4], [5, 4, 3, 2, 1, 0], layers=2,
                     capacity=64, pages=10)
    chain.width, chain.caches, chain.stepped = 4, [None, None], np.array([False, True, False])
    chain.dev = {"table": Buffer(), "cos": None, "sin": None}
    with pytest.raises(RuntimeError, match="no memory"):
        chain.begin({2: [(rows_of(17), rows_of(17))] * 2, 0: [(rows_of(5), rows_of(5))] * 2})
    assert chain.rt.live == 0 and chain.lengths.tolist() == [0, 3, 0] and sorted(chain.free) == list(range(6))
    assert chain.table[1].tolist() == [9] + [ref.NO] * 3 and (chain.table[[0, 2]] == ref.NO).all()
    assert chain.stepped.tolist() == [False, True, False]


@pytest.mark.parametrize("scale,fine", [(2.3e38, True), (-2.3e38, True), (2.4e38, False), (-3.4e38, False)])
def test_scales_that_are_no_number_with_their_logarithm(checks, scale, fine):
    """f32's largest number over log2(e) is 2.36e38: what is larger made infinities of every query and NaN of every zero."""
    assert (call(checks.check_attention, ATTEND, dict(scale=scale)) is None) == fine


@pytest.mark.parametrize("change", [
    dict(workspace=5 * M), dict(workspace=5 * M + 4096), dict(output=6 * M + 256), dict(output=4 * M), dict(output=2 * M),
    dict(workspace=3 * M), dict(workspace=4 * M), dict(workspace=2 * M), dict(workspace=M + 4096), dict(lengths=5 * M + 16),
    dict(table=6 * M), dict(workspace=2 * M - 16),
])
def test_attention_outputs_and_workspaces_lie_apart(checks, change):
    """The join takes its parts' numbers from the workspace: nothing else may write there, nor change the lengths."""
    assert call(checks.check_attention, ATTEND, change)
