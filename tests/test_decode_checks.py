"""CPU tests of the argument checks of the shared-prompt decode ops: which
calls are refused, and that the calls the documentation allows are not.  The
checks are compiled from their header by the host compiler; no device."""
import ctypes
import math
import os
import subprocess
from ctypes import c_char_p, c_double, c_float, c_int, c_uint32, c_uint64

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
U32, U64 = c_uint32, c_uint64


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("checks") / "libdecode_checks.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__=1", "-I/opt/rocm/include",
                    "-o", so, os.path.join(HERE, "cpp", "decode_checks.cpp")], check=True)
    lib = ctypes.CDLL(so)
    lib.check_prefix_attention.argtypes = [c_int, U64, U64, U32, U32, U64, U64, U32, U64, U64, U64, U32, U32, U32, U32, U32,
                                           c_float, U64]
    lib.check_kv_evict.argtypes = [c_int] + [U64] * 7 + [U32] * 5
    lib.check_verify_draft.argtypes = [U64] * 8 + [U32] * 3 + [c_double, U64]
    for f in (lib.check_prefix_attention, lib.check_kv_evict, lib.check_verify_draft):
        f.restype = c_char_p
    return lib


M = 1 << 32  # addresses far apart
ATTEND = dict(format=0, q=M, prefix=2 * M, prefix_length=100, prefix_capacity=128, cache=4 * M, lengths=6 * M, capacity=64,
              output=7 * M, weights_in=8 * M, weights_out=9 * M, sequences=4, tokens=2, q_heads=8, kv_heads=2, head_dim=128,
              scale=0.1, workspace=10 * M)
EVICT = dict(format=0, cache=M, cache_out=8 * M, weights=16 * M, weights_out=17 * M, lengths=18 * M, lengths_out=19 * M,
             kept=20 * M, sequences=4, capacity=1000, kv_width=96, budget=500, recent=100)
VERIFY = dict(target=M, draft=2 * M, draft_tokens=3 * M, draft_lengths=4 * M, accept=5 * M, sample=6 * M, accepted=7 * M,
              tokens=8 * M, sequences=4, drafts=3, vocab=1000, inv_temperature=1.0, workspace=9 * M)


def call(fn, base, change):
    return fn(*{**base, **change}.values())


@pytest.mark.parametrize("change", [
    {}, dict(prefix=0, prefix_length=0, prefix_capacity=0), dict(cache=0, lengths=0, capacity=0, weights_in=0, weights_out=0),
    dict(weights_in=0), dict(weights_in=0, weights_out=0), dict(weights_in=9 * M), dict(head_dim=4), dict(head_dim=256),
    dict(format=1, cache=4 * M + 2, prefix=2 * M + 2), dict(format=2, head_dim=96), dict(scale=-1.0), dict(scale=0.0),
    dict(sequences=1, tokens=1, q_heads=1, kv_heads=1), dict(tokens=4097), dict(prefix_length=128),
    dict(prefix_length=1 << 29, prefix_capacity=1 << 31), dict(sequences=7, capacity=1 << 29, weights_in=0), dict(kv_heads=128, q_heads=128, head_dim=256),
])
def test_attention_calls_that_are_allowed(checks, change):
    assert call(checks.check_prefix_attention, ATTEND, change) is None


@pytest.mark.parametrize("change", [
    dict(format=3), dict(format=-1), dict(q=0), dict(output=0), dict(workspace=0), dict(prefix=0), dict(cache=0), dict(lengths=0),
    dict(sequences=0), dict(tokens=0), dict(q_heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(kv_heads=16), dict(head_dim=0),
    dict(head_dim=2), dict(head_dim=130), dict(head_dim=260), dict(format=1, head_dim=100), dict(format=2, head_dim=80),
    dict(prefix_length=129), dict(prefix_length=0, capacity=0, weights_in=0, weights_out=0), dict(capacity=0),
    dict(weights_out=0), dict(weights_in=9 * M + 16), dict(scale=math.nan), dict(scale=math.inf), dict(q=M + 4),
    dict(output=7 * M + 8), dict(workspace=10 * M + 4), dict(prefix=2 * M + 4), dict(cache=4 * M + 8),
    dict(format=1, cache=4 * M + 1), dict(weights_out=9 * M + 2), dict(lengths=6 * M + 1), dict(output=M), dict(output=M + 16),
    dict(output=M - 16), dict(sequences=8, capacity=1 << 29), dict(prefix_length=(1 << 29) + 1, prefix_capacity=1 << 31),
    dict(sequences=1 << 20, tokens=1, q_heads=9, kv_heads=3),
    dict(sequences=1 << 31, capacity=1), dict(tokens=1 << 28), dict(kv_heads=256, q_heads=256, head_dim=256),
])
def test_attention_calls_that_are_refused(checks, change):
    assert call(checks.check_prefix_attention, ATTEND, change)


@pytest.mark.parametrize("change", [
    {}, dict(cache_out=M), dict(weights_out=16 * M), dict(lengths_out=18 * M), dict(budget=1000, recent=1000), dict(budget=1, recent=0),
    dict(kv_width=1), dict(kv_width=32768), dict(format=1, cache=M + 2), dict(format=2, kv_width=32),
    dict(cache_out=M + 2 * 4000 * 96 * 4), dict(sequences=7, capacity=1 << 29, cache_out=1 << 50, weights_out=16 * M)])
def test_evict_calls_that_are_allowed(checks, change):
    assert call(checks.check_kv_evict, EVICT, change) is None


@pytest.mark.parametrize("change", [
    dict(cache=0), dict(cache_out=0), dict(weights=0), dict(weights_out=0), dict(lengths=0), dict(lengths_out=0), dict(kept=0),
    dict(sequences=0), dict(capacity=0), dict(kv_width=0), dict(kv_width=32769), dict(budget=0), dict(budget=1001), dict(recent=501),
    dict(format=1, kv_width=48), dict(format=2, kv_width=100), dict(cache=M + 2), dict(format=1, cache=M + 1), dict(kept=20 * M + 2),
    dict(cache_out=M + 16), dict(cache_out=M + 2 * 4000 * 96 * 4 - 4), dict(cache_out=M - 4), dict(weights_out=16 * M + 4),
    dict(lengths_out=18 * M + 4), dict(sequences=8, capacity=1 << 29), dict(sequences=(1 << 20) + 1, capacity=1, budget=1, recent=0)])
def test_evict_calls_that_are_refused(checks, change):
    assert call(checks.check_kv_evict, EVICT, change)


@pytest.mark.parametrize("change", [
    {}, dict(draft=0), dict(draft_lengths=0), dict(drafts=0, draft=0, draft_tokens=0, accept=0), dict(vocab=1), dict(drafts=1024),
    dict(inv_temperature=1e-3), dict(vocab=1 << 29, drafts=1, sequences=1)])
def test_verify_calls_that_are_allowed(checks, change):
    assert call(checks.check_verify_draft, VERIFY, change) is None


@pytest.mark.parametrize("change", [
    dict(target=0), dict(draft_tokens=0), dict(accept=0), dict(sample=0), dict(accepted=0), dict(tokens=0), dict(workspace=0),
    dict(sequences=0), dict(vocab=0), dict(drafts=1025), dict(vocab=(1 << 29) + 1), dict(sequences=(1 << 20) + 1),
    dict(inv_temperature=0.0), dict(inv_temperature=-1.0), dict(inv_temperature=math.nan), dict(inv_temperature=math.inf),
    dict(target=M + 2), dict(draft=2 * M + 1), dict(tokens=8 * M + 2), dict(workspace=9 * M + 8),
    dict(sequences=1 << 20, drafts=1024, vocab=4096)])
def test_verify_calls_that_are_refused(checks, change):
    assert call(checks.check_verify_draft, VERIFY, change)


@pytest.mark.parametrize("scale,fine", [(2.3e38, True), (-2.3e38, True), (2.4e38, False), (-3.4e38, False)])
def test_scales_that_are_no_number_with_their_logarithm(checks, scale, fine):
    assert (call(checks.check_prefix_attention, ATTEND, dict(scale=scale)) is None) == fine
