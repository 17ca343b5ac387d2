"""GPU tests of the verification of drafted tokens: accepted counts and tokens
equal a float64 restatement's.  Inputs whose decision lies within 1e-9 of a
border in the restatement are refused by the test itself (none does)."""
import sys

import numpy as np
import pytest

import decode_refs as ref
from atlas_amd import OperatorError

pytestmark = pytest.mark.gpu
f32 = np.float32


def say(msg):
    print(f"[gpu-verify] {msg}", flush=True)
    sys.stdout.flush()


def run(rt, target, draft, tokens, lengths, accept, sample, inv):
    B, T1, V = target.shape
    T = T1 - 1
    up = lambda x: None if x is None or x.size == 0 else rt.upload(x)  # noqa: E731
    bufs = [up(x) for x in (target, draft, tokens, lengths, accept, sample)]
    acc, out = rt.empty(B, np.uint32), rt.empty(B * T1, np.uint32)
    nbytes = rt.verify_draft_workspace(B, T, V)
    ws = rt.alloc(nbytes + 256)
    rt.memset(ws, 0xFF, nbytes + 256)
    rt.verify_draft(*bufs, acc, out, B, T, V, inv, ws, nbytes)
    rt.sync()
    assert (ws.download(nbytes + 256, np.uint8)[nbytes:] == 0xFF).all(), "wrote behind the workspace"
    got = acc.download(B, np.uint32), out.download(B * T1, np.uint32).reshape(B, T1)
    for b in bufs + [acc, out, ws]:
        if b is not None:
            rt.free(b)
    return got


def both(rt, name, target, draft, tokens, lengths, accept, sample, inv, border=1e-9):
    acc, out, near = ref.verify(target, draft, tokens, lengths, accept, sample, inv)
    assert near.min() > border, "an input lies on a border by chance"
    got = run(rt, target, draft, tokens, lengths, accept, sample, inv)
    say(f"{name}: accepted {np.bincount(acc).tolist()}")
    assert np.array_equal(got[0], acc), (name, got[0], acc)
    assert np.array_equal(got[1], out), (name, np.argwhere(got[1] != out)[:4])


def make(seed, B, T, V, std=4.0, apart=1.0):
    r = np.random.default_rng(seed)
    target = (r.standard_normal((B, T + 1, V)) * std).astype(f32)
    draft = (target[:, :T] + r.standard_normal((B, T, V)) * apart).astype(f32)
    tokens = np.zeros((B, T), np.uint32)
    for b in range(B):
        for t in range(T):
            p = np.exp(draft[b, t].astype(np.float64) - draft[b, t].max())
            tokens[b, t] = r.choice(V, p=p / p.sum())
    return (r, target, draft, tokens, r.integers(0, T + 1, B, dtype=np.uint32), r.random((B, T), dtype=f32),
            r.random(B, dtype=f32))


@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (3, 1, 2), (2, 4, 3), (5, 2, 63), (4, 3, 257), (6, 2, 4095), (6, 2, 4096),
                                   (6, 2, 4097), (3, 5, 8193), (40, 3, 1000), (2, 4, 50257), (1, 2, 151936),
                                   (3, 16, 500), (4, 17, 500), (2, 70, 4097), (1, 3, 300000), (2, 1024, 7), (3000, 1, 5),
                                   (300, 17, 40)])
@pytest.mark.parametrize("certain", [False, True])
def test_verify_matches_float64(rt, B, T, V, certain):
    r, target, draft, tokens, lengths, accept, sample = make(B * 31 + V, B, T, V)
    for inv in (1.0, 1.0 / 0.7):
        both(rt, f"{B} {T} {V} certain {certain}", target, None if certain else draft, tokens, lengths, accept, sample, inv)
    both(rt, "all drafts", target, None if certain else draft, tokens, None, accept, sample, 1.0)


def test_no_drafts_is_sampling(rt):
    r, target, _, _, _, _, sample = make(5, 30, 0, 9000)
    both(rt, "sampling", target, None, np.zeros((30, 0), np.uint32), None, np.zeros((30, 0), f32), sample, 1.3)


def test_masked_rows_and_odd_logits(rt):
    r, target, draft, tokens, lengths, accept, sample = make(6, 24, 2, 5000)
    low = np.finfo(f32).min
    target[:, :, ::3], draft[:, :, 1::3] = low, -np.inf
    target[2:4, :, 5::7] = np.nan
    draft[3:5, :, 2::5] = np.nan
    target[5] = -np.inf                      # nothing can be drawn
    target[6] = np.nan
    target[7, :, 77] = np.inf                # all mass on one
    target[8, :, [3, 4999]] = np.inf         # or on two
    draft[9, :, 10] = np.inf
    draft[10] = -np.inf                      # a draft model without mass
    target[11] = -np.inf
    target[11, :, 4999] = low                # one finite logit, the last
    tokens[12] = 5000                        # no such token
    tokens[13] = 0xFFFFFFFF
    lengths[14] = 0
    lengths[15] = 4000000000                 # more than there are: all
    target[16] = 3.0                         # all equal, and equal to the draft's: nothing remains of p - q
    draft[16] = 3.0
    accept[16] = np.float32(1) - np.float32(2.0 ** -24)
    both(rt, "odd logits", target, draft, tokens, lengths, accept, sample, 1.0)
    both(rt, "odd logits, certain", target, None, tokens, lengths, accept, sample, 1.0)


def test_borders_fall_as_the_rule_says(rt):
    """Equal logits over 4 or 8192 tokens give powers of two: running sums and products are exact in float64."""
    say("borders")
    for V in (4, 8192):
        target = np.zeros((V, 1, V), f32)
        sample = (np.arange(V) / V).astype(f32)  # i / V: the first i with (i + 1) / V > sample
        got = run(rt, target, None, np.zeros((V, 0), np.uint32), None, np.zeros((V, 0), f32), sample, 1.0)
        assert np.array_equal(got[1][:, 0], np.arange(V)), V
    target, draft = np.zeros((3, 2, 4), f32), np.full((3, 1, 4), -np.inf, f32)
    draft[:, 0, :2] = 0.0  # q = 1/2, p = 1/4: accepted below 1/2
    accept = np.array([[0.5], [np.nextafter(f32(0.5), f32(0))], [0.0]], f32)
    got = run(rt, target, draft, np.ones((3, 1), np.uint32), None, accept, np.zeros(3, f32), 1.0)
    assert got[0].tolist() == [0, 1, 1]
    assert got[1][:, 0].tolist() == [2, 1, 1] and got[1][:, 1].tolist() == [ref.NO, 0, 0]


def test_sample_uniform_zero_takes_the_first_with_mass(rt):
    say("zero uniforms")
    r, target, draft, tokens, lengths, accept, sample = make(9, 12, 2, 6000)
    target[:, :, :37] = -np.inf
    both(rt, "zeros", target, draft, tokens, lengths, np.zeros_like(accept), np.zeros_like(sample), 1.0)


def test_drawn_tokens_follow_the_target(rt):
    """One row, many uniforms on a grid: the counts are the probabilities, to within one each."""
    say("grid")
    r = np.random.default_rng(11)
    V, N = 10, 4096
    row = r.standard_normal(V).astype(f32)
    target = np.broadcast_to(row, (N, 1, V)).copy()
    sample = ((np.arange(N) + 0.5) / N).astype(f32)
    got = run(rt, target, None, np.zeros((N, 0), np.uint32), None, np.zeros((N, 0), f32), sample, 1.0)
    p = np.exp(row.astype(np.float64))
    count = np.bincount(got[1][:, 0], minlength=V)
    assert (np.abs(count - p / p.sum() * N) <= 1.0).all()


def test_graph_replays_equal_the_eager_call(rt):
    say("graph")
    r, target, draft, tokens, lengths, accept, sample = make(21, 9, 3, 5001)
    bufs = [rt.upload(x) for x in (target, draft, tokens, lengths, accept, sample)]
    acc, out = rt.empty(9, np.uint32), rt.empty(36, np.uint32)
    nbytes = rt.verify_draft_workspace(9, 3, 5001)
    ws = rt.alloc(nbytes)
    rt.graph_begin()
    rt.verify_draft(*bufs, acc, out, 9, 3, 5001, 1.0, ws, nbytes)
    graph = rt.graph_end()
    for i in range(4):
        accept, sample = r.random((9, 3), dtype=f32), r.random(9, dtype=f32)
        bufs[4].upload(accept), bufs[5].upload(sample)
        rt.graph_launch(graph)
        rt.sync()
        a, o, near = ref.verify(target, draft, tokens, lengths, accept, sample, 1.0)
        assert near.min() > 1e-9
        assert np.array_equal(acc.download(9, np.uint32), a) and np.array_equal(out.download(36, np.uint32).reshape(9, 4), o)
        got = run(rt, target, draft, tokens, lengths, accept, sample, 1.0)  # eager, its own workspace
        assert np.array_equal(got[1], o)
    rt.graph_destroy(graph)


def test_refusals(rt):
    say("refusals")
    r, target, draft, tokens, lengths, accept, sample = make(2, 2, 1, 40)
    b = [rt.upload(x) for x in (target, draft, tokens, lengths, accept, sample)]
    acc, out = rt.empty(2, np.uint32), rt.empty(4, np.uint32)
    nbytes = rt.verify_draft_workspace(2, 1, 40)
    ws = rt.alloc(nbytes)
    good = dict(target_logits=b[0], draft_logits=b[1], draft_tokens=b[2], draft_lengths=b[3], accept_uniform=b[4],
                sample_uniform=b[5], accepted=acc, tokens=out, sequences=2, drafts=1, vocab=40, inv_temperature=1.0,
                workspace=ws, workspace_bytes=nbytes)
    rt.verify_draft(**good)
    rt.sync()
    bad = [dict(target_logits=None), dict(draft_tokens=None), dict(accept_uniform=None), dict(sample_uniform=None),
           dict(accepted=None), dict(tokens=None), dict(workspace=None), dict(sequences=0), dict(vocab=0), dict(drafts=1025),
           dict(inv_temperature=0.0), dict(inv_temperature=-1.0), dict(inv_temperature=float("nan")),
           dict(inv_temperature=float("inf")), dict(workspace_bytes=nbytes - 1), dict(workspace=ws.ptr + 8),
           dict(target_logits=b[0].ptr + 2), dict(tokens=out.ptr + 1), dict(vocab=1 << 31), dict(sequences=1 << 21)]
    for change in bad:
        with pytest.raises(OperatorError) as e:
            rt.verify_draft(**{**good, **change})
        assert e.value.kind == "InvalidInput", change
    for sizes in ((0, 1, 40), (1, 1, 0), (1 << 21, 1, 40)):
        with pytest.raises(OperatorError):
            rt.verify_draft_workspace(*sizes)
