"""GPU tests of the draft verification at the ends of its temperatures."""
import sys

import numpy as np
import pytest

import decode_refs as ref
from test_gpu_verify import run

pytestmark = pytest.mark.gpu
f32 = np.float32


@pytest.mark.parametrize("inv", [5e-324, 1e-300, 1e300, 3e306, 5e306, 1e308, np.finfo(np.float64).max])
@pytest.mark.parametrize("certain", [False, True])
def test_temperatures_near_zero_and_infinity(rt, inv, certain):
    """A temperature near zero leaves all mass on the largest logit, one near infinity the same mass on every finite one."""
    print(f"[gpu-verify-range] {inv} {certain}", flush=True)
    sys.stdout.flush()
    r = np.random.default_rng(12)
    B, T, V = 6, 2, 3001
    target = (r.standard_normal((B, T + 1, V)) * 4).astype(f32)
    draft = (target[:, :T] + r.standard_normal((B, T, V))).astype(f32)
    target[1, 0, 40] = target[1, 0, 900] = 50.0  # two largest
    target[2] = -np.inf
    target[3, :, 7] = np.inf
    tokens = target[:, :T].argmax(-1).astype(np.uint32)
    tokens[4] = 5
    accept, sample = r.random((B, T), dtype=f32), r.random(B, dtype=f32)
    with np.errstate(over="ignore"):
        acc, out, near = ref.verify(target, None if certain else draft, tokens, None, accept, sample, inv)
    assert near.min() > 1e-9, "an input lies on a border by chance"
    got = run(rt, target, None if certain else draft, tokens, None, accept, sample, inv)
    assert np.array_equal(got[0], acc) and np.array_equal(got[1], out), (got, acc, out)
