"""GPU tests of the shared-prompt attention's sums over many keys: alike, so that
all roundings fall to one side and the result is the one value that they hold,
and with maxima that move, against float64."""
import sys

import numpy as np
import pytest

import decode_refs as ref
from test_gpu_prefix_attention import check, run

pytestmark = pytest.mark.gpu
f32 = np.float32


def say(msg):
    print(f"[gpu-prefix-sums] {msg}", flush=True)
    sys.stdout.flush()


# Every key alike and every value one number c: the result is c, and each sum adds equal terms.  Values are
# written by memset: f32 0x3c3c3c3c = 0.0115; a block of Q8_0 or Q4_0 of bytes x has scale f16(0x3c3c) = 1.0586 and
# codes x.  Batches of as many (head, row tile) units as fill the chip, so that segments are few and long.
def constant(fmt, byte):
    if fmt == "f32":
        return float(np.full(4, byte, np.uint8).view(f32)[0])
    d = float(np.full(2, byte, np.uint8).view(np.float16)[0])
    # Q4_0: alternate dims hold the two nibbles; equal ones make one number
    return d * (float(np.int8(byte)) if fmt == "q8_0" else (byte & 15) - 8)


LONG = {  # sequences, heads, KV heads, head_dim, prompt, capacity
    "prompt": (448, 32, 32, 32, 60001, 0),
    "prompt_128": (448, 32, 32, 128, 30001, 0),
    "prompt_256": (448, 32, 32, 256, 20001, 0),
    "prompt_longer": (448, 32, 32, 4, 300001, 0),
    "prompt_packed": (1024, 32, 32, 32, 60001, 0),
    "prompt_packed_256": (2048, 16, 16, 256, 40001, 0),
    "prompt_1024": (448, 32, 32, 32, 1024, 0),
    "prompt_1025": (448, 32, 32, 32, 1025, 0),
    "prompt_few_rows": (1, 1, 1, 32, 3000001, 0),
    "own": (768, 1, 1, 32, 0, 40001),
    "own_128": (256, 1, 1, 128, 0, 40001),
    "own_256": (256, 1, 1, 256, 0, 30001),
    "own_longer": (8, 1, 1, 32, 0, 3000001),
    "own_longest": (1, 1, 1, 4, 0, 1 << 29),
}


FILLS = [("f32", 0x3C), ("f32", 0x3B), ("f32", 0x3A), ("q8_0", 0x3C), ("q4_0", 0x33)]


@pytest.mark.parametrize("shape,fmt,byte", [(shape, fmt, byte) for shape, (_, _, _, D, _, _) in LONG.items()
                                            for fmt, byte in FILLS if fmt == "f32" or D % 32 == 0])
def test_long_sums_of_equal_terms(rt, shape, fmt, byte):
    B, H, KH, D, P, cap = LONG[shape]
    width = KH * D
    c = constant(fmt, byte)
    say(f"{shape} {fmt} {byte:#x}: {c}")
    rows = max(P, B * cap)
    nbytes = 2 * rows * ref.row_bytes(fmt, width)
    data = rt.alloc(nbytes)
    rt.memset(data, byte, nbytes)
    # rows' scores differ, so that their weights, 2^(x - a whole number) in the prompt's kernels, take many values
    r = np.random.default_rng(9)
    q = np.repeat(r.uniform(0.0, 1.0, (B, 1, H, 1)), D, -1).astype(f32)
    scale = float(f32(2.0 / (abs(c) * D)))
    dq, out, n = rt.upload(q), rt.empty(q.size), rt.upload(np.full(B, cap, np.uint32))
    size = rt.prefix_attention_workspace(fmt, B, 1, H, KH, D, P, cap, False)
    ws = rt.alloc(size)
    rt.prefix_attention(fmt, dq, data if P else None, P, P, data if cap else None, n if cap else None, cap, out, None, None,
                        B, 1, H, KH, D, scale, ws, size)
    rt.sync()
    got = out.download(q.size).astype(np.float64)
    for b in (data, dq, out, n, ws):
        rt.free(b)
    worst = float(np.abs(got / c - 1).max())
    say(f"{shape} {fmt} {byte:#x}: off by {worst:.2e}")
    assert worst <= 1e-5


def test_weights_of_many_rows(rt):
    """131072 shares of about 1 / 60000 added up for each of a sequence's first rows."""
    T, H, D, P, cap = 2048, 64, 4, 60000, 2112
    say("131072 shares")
    q = np.zeros((1, T, H, D), f32)
    dq, zero, w = rt.upload(q), rt.alloc(2 * P * D * 4), rt.empty(cap)
    rt.memset(zero, 0, 2 * P * D * 4)
    out, n = rt.empty(q.size), rt.upload(np.asarray([cap], np.uint32))
    size = rt.prefix_attention_workspace("f32", 1, T, H, 1, D, P, cap, True)
    ws = rt.alloc(size)
    rt.prefix_attention("f32", dq, zero, P, P, zero, n, cap, out, None, w, 1, T, H, 1, D, 1.0, ws, size)
    rt.sync()
    got = w.download(cap).astype(np.float64)
    for b in (dq, zero, w, out, n, ws):
        rt.free(b)
    # token t sees the prompt and own rows below cap - (T - 1 - t), all with equal scores
    sees = cap - (T - 1 - np.arange(T))
    share = H / (P + sees.astype(np.float64))
    exp = np.array([share[sees > j].sum() for j in range(cap)])
    worst = float(np.abs(got / exp - 1).max())
    say(f"off by {worst:.2e}")
    assert worst <= 2e-6  # a share's sum of 62112 equal weights and under 32 roundings of 2^-24


@pytest.mark.parametrize("fmt", ["f32", "q8_0", "q4_0"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ramp", ["up", "down", "none"])
@pytest.mark.parametrize("B", [112, 129])
def test_segments_of_several_runs(rt, B, D, fmt, ramp):
    """Maxima that rise from run to run, or fall away behind the first: 1500 or more keys to a segment, unpacked (448 rows
    of each KV head) and packed (516)."""
    H, KH, P = 64, 16, 3001
    say(f"{B} {D} {fmt} {ramp}")
    r = np.random.default_rng(D)
    q = (r.standard_normal((B, 1, H, D)) * 2).astype(f32)
    prefix = ref.make_cache(r, fmt, P, KH * D)
    scale = np.ones(P) if ramp == "none" else np.linspace(0.1, 3.0, P)[:: 1 if ramp == "up" else -1]
    if fmt == "f32":
        prefix.view(f32).reshape(2, P, -1)[:] *= scale[None, :, None].astype(f32)
    else:
        size = {"q8_0": 34, "q4_0": 18}[fmt]
        b = prefix.reshape(2, P, KH * D // 32, size)
        d = np.ascontiguousarray(b[..., :2]).view(np.float16) * scale[None, :, None, None]
        b[..., :2] = d.astype(np.float16).view(np.uint8)
    lengths = np.zeros(B, np.uint32)
    some = np.arange(0, B, 16)  # of whose rows float64 is asked
    exp, _, bound = ref.attention(q[some], prefix, P, None, lengths[some], 0, KH, float(f32(D ** -0.5)), fmt)
    got, _ = run(rt, fmt, q, prefix, P, None, lengths, 0, KH, float(f32(D ** -0.5)))
    check(f"{B} {D} {fmt} {ramp}", got[some], exp, bound, P, D)
