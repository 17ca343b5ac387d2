"""CPU tests of the rules by which the paged attention and the log probabilities
are launched, compiled from their headers by the host compiler: the calls of
paged_launches.py take the launches that they are named for, and all that there
are."""
import ctypes
import os
import subprocess
from ctypes import c_int, c_uint32

import pytest

from paged_launches import ATTENTION, FORMATS, LOGPROBS

HERE = os.path.dirname(os.path.abspath(__file__))
NUMBER = {"f32": 0, "q8_0": 1, "q4_0": 2, "f16": 3}


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("plans") / "libpaged_plans.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__=1", "-I/opt/rocm/include",
                    "-o", so, os.path.join(HERE, "cpp", "paged_plans.cpp")], check=True)
    lib = ctypes.CDLL(so)
    lib.attention_plan.argtypes, lib.attention_plan.restype = [c_int] + [c_uint32] * 7 + [ctypes.c_void_p], None
    lib.logprobs_plan.argtypes, lib.logprobs_plan.restype = [c_uint32] * 2 + [ctypes.c_void_p], None
    return lib


def attention_plan(plans, fmt, H, KH, D, ps, width, sequences, window):
    out = (c_uint32 * 7)()
    plans.attention_plan(NUMBER[fmt], ps, KH, D, sequences, width, H, window, out)
    return list(out)


def launch_of(plans, case):
    fmt, H, KH, D, ps, width, lengths, window, _ = case
    units, waves, _, _, lanes, threads, groups = attention_plan(plans, fmt, H, KH, D, ps, width, len(lengths), window)
    if units:
        return ("whole", waves)
    assert groups * 4 * lanes >= D and (threads == 1024 or groups == 1)
    n = len(lengths)
    return ("split", "wave" if n <= 64 else "chunk" if n <= 256 else "chunks", (lanes, threads))


@pytest.mark.parametrize("name", list(ATTENTION))
def test_attention_takes_the_launch(plans, name):
    assert launch_of(plans, ATTENTION[name]) == ATTENTION[name][8]


def test_every_launch_of_the_attention_is_there():
    joins = {(16, 256), (32, 256), (64, 256), (8, 1024), (16, 1024)}
    for fmt in FORMATS:
        mine = [c for c in ATTENTION.values() if c[0] == fmt]
        split = [c for c in mine if c[8][0] == "split"]
        assert {c[8][2] for c in split} == joins and {c[8][1] for c in split} == {"wave", "chunk", "chunks"}
        assert {c[8][1] for c in mine if c[8][0] == "whole"} == {4, 16, 6 if fmt == "f16" else 8}
        assert {min(4 if -(-c[1] // c[2]) <= 4 else 8 if c[1] // c[2] <= 8 else 16, 16) for c in split} == {4, 8, 16}


def test_parts_of_the_largest_and_smallest_calls(plans):
    """At least as many parts as stay on the chip where there are units for them, 1024 units a part behind that."""
    assert attention_plan(plans, "q8_0", 8, 1, 64, 256, 4096, 40, 0)[2:4] == [1024, 1280]
    assert attention_plan(plans, "f32", 8, 1, 64, 256, 4096, 40, 0)[2:4] == [1024, 2560]
    assert attention_plan(plans, "f32", 8, 1, 64, 16, 1, 3, 0)[2:4] == [1024, 3]
    assert attention_plan(plans, "f16", 8, 1, 256, 64, 1 << 23, 16, 0)[2:4] == [512, 1 << 18]
    assert attention_plan(plans, "f32", 8, 1, 4, 16, 1 << 25, 32, 0)[3] == 1 << 20  # and 2^20 at most


@pytest.mark.parametrize("name", list(LOGPROBS))
def test_log_probabilities_take_the_launch(plans, name):
    rows, vocab, _, each, again, threads = LOGPROBS[name]
    out = (c_uint32 * 5)()
    plans.logprobs_plan(rows, vocab, out)
    strips, of_a_slice, slices, groups, row_threads = list(out)
    assert strips == -(-vocab // 1024) and slices == -(-strips // each) and groups == min(2048, -(-rows * slices // 4))
    assert (of_a_slice, rows * slices > 4 * groups, row_threads) == (each, again, threads)


def test_every_launch_of_the_log_probabilities_is_there(plans):
    cases = LOGPROBS.values()
    assert {(each, again) for _, _, _, each, again, _ in cases} == {(1, False), (2, False), (2, True)}
    assert {(each, threads) for _, _, _, each, _, threads in cases} == {(1, 1024), (2, 1024), (1, 256), (2, 256)}
    assert {-(-vocab // 1024) % 2 for _, vocab, _, each, again, _ in cases if again} == {0, 1}  # the last slice whole and not
    # a wavefront with one strip a slice never has a second one: 8192 slices stay at once
    for rows, vocab in ((8191, 1000), (1, 8191 << 10), (3, 2730 << 10), (4096, 1000)):
        out = (c_uint32 * 5)()
        plans.logprobs_plan(rows, vocab, out)
        assert out[1] == 1 and rows * out[2] <= 4 * out[3]
