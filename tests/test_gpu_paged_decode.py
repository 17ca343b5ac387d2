"""A batch that decodes from a paged cache (atlas_amd.chains.PagedDecode) on the
GPU, eager and as HIP-graph replays, with sequences that begin, grow over page
borders, end and give their pages to others: every step's queries, pools,
attention, tokens and probabilities against the plain restatements."""
import sys

import numpy as np
import pytest

import paged_refs as ref
from atlas_amd import workloads as wl
from atlas_amd.chains import PagedDecode, PagedShape
from test_gpu_logprobs import close
from test_gpu_paged_attention import check

pytestmark = pytest.mark.gpu
f32, u32 = np.float32, np.uint32


def say(msg):
    print(f"[gpu-paged-decode] {msg}", flush=True)
    sys.stdout.flush()


class Pools:
    """The layers' pools as the references keep them."""

    def __init__(self, chain):
        S = chain.S
        self.chain = chain
        self.pools = [ref.Pool(chain.kv_format, S.pages, S.page_size, S.kv_heads, S.head_dim) for _ in range(S.layers)]
        self.cos = chain.dev["cos"].download().reshape(-1, S.head_dim // 2)
        self.sin = chain.dev["sin"].download().reshape(-1, S.head_dim // 2)

    def begin(self, prompts):
        for place, layers in prompts.items():
            for pool, (k, v) in zip(self.pools, layers):
                n = len(k)
                ref.append(pool, self.chain.table, k, v, None, None, self.cos, self.sin, np.full(n, place, u32), np.arange(n, dtype=u32))

    def step(self, tag, logits):
        c, S = self.chain, self.chain.S
        B, H, KH, D = S.sequences, S.q_heads, S.kv_heads, S.head_dim
        got = c.results()
        active = c.lengths > 0
        positions = np.where(active, c.lengths, ref.NO).astype(u32)
        lengths = np.where(active, c.lengths + 1, 0).astype(u32)
        for layer, (lay, pool) in enumerate(zip(c.layers, self.pools)):
            q = np.where(active[:, None, None], 0, got["q_rot"][layer].reshape(B, H, D)).astype(f32)
            ref.append(pool, c.table, lay["k"].reshape(B, KH, D), lay["v"].reshape(B, KH, D), lay["q"].reshape(B, H, D), q, self.cos,
                       self.sin, None, positions)
            assert np.array_equal(got["q_rot"][layer].reshape(B, H, D).view(u32), q.view(u32)), f"{tag}: queries {layer}"
            assert np.array_equal(got["pool"][layer], pool.bytes.reshape(-1)), f"{tag}: pool {layer}"
            out = got["attention"][layer].reshape(B, H, D)
            assert (out[~active] == 0).all()
            q[~active] = 0
            check(f"{tag} layer {layer}", c.kv_format, pool, c.table, q, lengths, c.window(layer), float(c.scale), out)
        tokens = got["tokens"].view(u32)
        assert np.array_equal(tokens, logits.shape[1] - 1 - logits[:, ::-1].argmax(1)), tag
        exp = ref.logprobs(logits, tokens.reshape(B, 1), 1.0 / S.temperature, S.alternatives)
        close(f"{tag}: logprobs", got["logprobs"].reshape(B, 1), exp[0])
        close(f"{tag}: entropy", got["entropy"], exp[1])
        assert np.array_equal(got["top_ids"].view(u32).reshape(B, -1), exp[2]), tag
        close(f"{tag}: tops", got["top_logprobs"].reshape(B, -1), exp[3])


def prompt(r, S, n):
    return [(r.standard_normal((n, S.kv_heads, S.head_dim)).astype(f32), r.standard_normal((n, S.kv_heads, S.head_dim)).astype(f32))
            for _ in range(S.layers)]


@pytest.mark.parametrize("fmt", ["f32", "f16", "q8_0", "q4_0"])
def test_paged_decode_eager_and_graph(rt, fmt):
    S = PagedShape(layers=5, vocab=3001, alternatives=4)
    say(fmt)
    chain = PagedDecode(rt, S, fmt)
    held = Pools(chain)
    r = wl.rng(77)
    try:
        first = {0: prompt(r, S, 1), 1: prompt(r, S, 15), 3: prompt(r, S, 61)}
        chain.begin(first)
        held.begin(first)
        for i in range(9):
            if i == 4:
                chain.end(3)
                other = {3: prompt(r, S, 33), 5: prompt(r, S, 90)}
                chain.begin(other)
                held.begin(other)
            if i == 7:
                chain.end(1)
            logits = (r.standard_normal((S.sequences, S.vocab)) * 4).astype(f32)
            chain.set_step(logits)
            if i < 2:
                chain.enqueue()
            else:
                if i == 2:
                    chain.capture()
                for b in chain.out["attention"]:
                    rt.memset(b, 0xEE, b.nbytes)  # eager work between the replays
                rt.sync()
                chain.replay()
            rt.sync()
            held.step(f"{fmt} step {i}", logits)
            chain.advance()
        used = {int(p) for p in chain.table.reshape(-1) if p != ref.NO}
        assert len(used) + len(chain.free) == S.pages and not used & set(chain.free)
    finally:
        chain.close()


def test_a_pool_or_a_sequence_that_is_full(rt):
    S = PagedShape(sequences=3, layers=1, capacity=32, pages=3, vocab=64, alternatives=0)
    chain = PagedDecode(rt, S, "f32")
    r = wl.rng(5)
    chain.begin({0: prompt(r, S, 32)})
    with pytest.raises(ValueError, match="no room"):
        chain.set_step(np.zeros((3, 64), f32))
    with pytest.raises(ValueError, match="has a sequence"):
        chain.begin({0: prompt(r, S, 1)})
    with pytest.raises(ValueError, match="no page left"):
        chain.begin({1: prompt(r, S, 17)})
    chain.end(0)
    chain.begin({1: prompt(r, S, 17)})
    chain.set_step(np.zeros((3, 64), f32))
    chain.enqueue()
    rt.sync()
    assert chain.advance().tolist() == [63, 63, 63] and chain.lengths.tolist() == [0, 18, 0]
    chain.close()
