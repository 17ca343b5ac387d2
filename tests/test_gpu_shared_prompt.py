"""A batch that decodes drafted tokens behind a shared prompt
(atlas_amd.chains.SharedPromptDecode) on the GPU, eager and as HIP-graph
replays: every step's rotated queries and keys, caches, attention, weights,
verification and, when the caches are full, cut, against the oracle's ops and
the float64 references, from the state the step began with."""
import sys

import numpy as np
import pytest

import decode_refs as ref
from atlas_amd import workloads as wl
from atlas_amd.chains import SharedPromptDecode, SharedPromptShape
from test_gpu_prefix_attention import check

pytestmark = pytest.mark.gpu
f32, u32 = np.float32, np.uint32


def say(msg):
    print(f"[gpu-shared-prompt] {msg}", flush=True)
    sys.stdout.flush()


def step_inputs(r, S):
    B, V = S.sequences, S.vocab
    logits = (r.standard_normal((B, S.drafts + 1, V)) * 6).astype(f32)
    draft = (logits[:, :S.drafts] + r.standard_normal((B, S.drafts, V)) * 0.5).astype(f32)
    tokens = draft.argmax(-1).astype(u32)
    return tokens, logits, draft, r.random((B, S.drafts), dtype=f32), r.random(B, dtype=f32)


def state_of(chain):
    return [(kv.download(chain.cache_bytes, np.uint8), w.download()) for kv, w in zip(chain.out["kv"], chain.out["weights"])]


def check_step(ora, chain, before, inputs, tag):
    S, fmt = chain.S, chain.kv_format
    B, T, QH, D, cap = S.sequences, S.drafts + 1, S.q_heads, S.head_dim, S.capacity
    got = chain.results()
    ahead = np.arange(T, dtype=u32)
    c, s = ora.rope_tables_gemma4((chain.positions[:, None] + ahead).reshape(-1).astype(u32), D // 2, D, 1e4)
    slots = (np.arange(B)[:, None] * cap + chain.lengths[:, None] + ahead).astype(u32)
    lengths = (chain.lengths + T).astype(u32)
    for layer, lay in enumerate(chain.layers):
        cache, w_in = before[layer]
        qo, ko = ora.qk_norm_rope(lay["q"], lay["k"], lay["qw"], lay["kw"], c, s, B * T, QH, True, D, D // 2, S.eps)
        assert np.array_equal(got["q_rot"][layer], np.asarray(qo).reshape(-1)), f"{tag}: queries {layer}"
        kv = np.asarray(ora.kv_append(fmt, ko, lay["v"], cache, D, B * cap, slots.reshape(-1), True, S.eps)).view(np.uint8)
        assert np.array_equal(got["kv"][layer], kv.reshape(-1)), f"{tag}: cache {layer}"
        prompt = chain.out["prompt"][layer].download(chain.prompt_bytes, np.uint8).reshape(2, S.prompt, -1)
        exp, drawn, bound = ref.attention(got["q_rot"][layer].reshape(B, T, QH, D), prompt, S.prompt, kv.reshape(2, B * cap, -1),
                                          lengths, cap, 1, float(chain.scale), fmt)
        check(f"{tag} layer {layer}", got["attention"][layer].reshape(exp.shape), exp, bound, S.prompt + cap, D)
        w_in = w_in.reshape(B, cap).copy()
        for b in range(B):
            w_in[b, chain.lengths[b]:lengths[b]] = 0
        dx = (D + 8) * 2.0 ** -24 * bound[1].max() + 2.0 ** -20 * bound[1].max()
        tol = (np.expm1(2 * dx) + (S.prompt + cap + 32 + T * QH) * 2.0 ** -24) * drawn + 2.0 ** -23 * (w_in + drawn) + 1e-30
        off = np.abs(got["weights"][layer].reshape(B, cap) - (w_in.astype(np.float64) + drawn))
        assert (off <= tol).all(), f"{tag}: weights {layer}"
    tokens, logits, draft, accept, sample = inputs
    assert np.array_equal(got["capped"], np.asarray(ora.softcap(logits.reshape(-1), S.softcap)).reshape(-1)), f"{tag}: logits"
    accepted, out, near = ref.verify(got["capped"].reshape(logits.shape), draft if S.drafts else None, tokens, None, accept, sample,
                                     1.0 / S.temperature)
    assert near.min() > 1e-9, "an input lies on a border by chance"
    assert np.array_equal(got["accepted"].view(u32), accepted) and np.array_equal(got["tokens"].view(u32).reshape(B, T), out), tag
    return accepted


@pytest.mark.parametrize("fmt", ["f32", "q8_0", "q4_0"])
@pytest.mark.parametrize("drafts", [3, 0])
def test_shared_prompt_decode_eager_graph_and_cut(rt, ora, fmt, drafts):
    """Steps until every cache has been cut: three eager, then replays of one recorded step with eager work between
    them, each against the references."""
    S = SharedPromptShape(drafts=drafts, layers=2, capacity=20, budget=8, recent=3)
    say(f"{fmt}, {drafts} drafts")
    chain = SharedPromptDecode(rt, S, fmt)
    r = wl.rng(99 + drafts)
    cuts, total = 0, 0
    try:
        for i in range(24):
            if chain.full:
                before = state_of(chain)
                n = chain.lengths.astype(u32)
                chain.cut()
                for layer, (cache, w) in enumerate(before):
                    cache = cache.reshape(2, S.sequences * S.capacity, -1)
                    w = w.reshape(S.sequences, S.capacity)
                    exp = ref.evict(cache, w, n, S.capacity, S.budget, S.recent, cache, w)
                    after = state_of(chain)[layer]
                    assert np.array_equal(after[0], exp[0].reshape(-1)) and np.array_equal(after[1], exp[1].reshape(-1)), "cut"
                    assert np.array_equal(chain.out["cut_lengths"][layer].download(), exp[2])
                    assert np.array_equal(chain.out["kept"][layer].download().reshape(exp[3].shape), exp[3])
                assert (chain.lengths <= S.budget).all()
                cuts += 1
            inputs = step_inputs(r, S)
            before = state_of(chain)
            chain.set_step(*inputs)
            if i < 3:
                chain.enqueue()
            else:
                if i == 3:
                    chain.capture()
                for b in chain.out["attention"]:
                    rt.memset(b, 0xEE, b.nbytes)  # eager work between the replays
                rt.sync()
                chain.replay()
            rt.sync()
            accepted = check_step(ora, chain, before, inputs, f"step {i}")
            assert np.array_equal(chain.advance()[0], accepted)
            total += int(accepted.sum())
        say(f"{cuts} cuts, {total} drafts accepted")
        assert cuts >= 1 and (drafts == 0 or total > 0)
    finally:
        chain.close()


def test_a_step_that_does_not_fit_is_refused(rt):
    S = SharedPromptShape(sequences=2, drafts=1, layers=1, prompt=16, capacity=4, budget=2, recent=1, vocab=64)
    chain = SharedPromptDecode(rt, S, "f32")
    r = wl.rng(5)
    chain.lengths = np.array([1, 3], u32)
    assert chain.full
    with pytest.raises(ValueError, match="cut"):
        chain.set_step(*step_inputs(r, S))
    chain.cut()
    assert chain.lengths.tolist() == [1, 2] and not chain.full
    chain.set_step(*step_inputs(r, S))
    chain.close()
