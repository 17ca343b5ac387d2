"""Decoding a batch from a shared prompt, as cases to time.

Three operators that follow one another in a serving loop whose sequences all
begin with the same long prompt and are decoded by drafting and verifying:

    attend   attention of the new tokens of a batch: the keys and values of the
             shared prompt are held once (its cache is read once for all
             sequences), every sequence has a cache of its own behind it; with
             `weights`, the attention each own position received is added up
    evict    a sequence's cache is cut to a budget: the most recent positions
             and, of the others, the ones with the largest added-up weight
    verify   drafted tokens are accepted or rejected against the target's
             probabilities with given random numbers, and one token is drawn
             from what remains

Caches have the layout that the KV append writes, [K | V][position][row], f32,
Q8_0 or Q4_0; a batch's own caches are one such cache of sequences * capacity
positions, sequence b at b * capacity.  Head layouts, widths and vocabularies
are those of the benchmark configurations and tests, or generic ones.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

HUGE = torch.finfo(torch.float32).min
NO_TOKEN = -1  # 0xffffffff


def listed():
    return [
        # The smallest call: one sequence, one token, a small model's heads, behind a short system prompt.
        {"name": "attend_one", "kind": "attend", "fmt": "f32", "sequences": 1, "tokens": 1, "q_heads": 9, "kv_heads": 3,
         "head_dim": 64, "prefix": 512, "capacity": 128, "shortest": 77, "longest": 77, "weights": False},
        # A small batch behind a long prompt: the prompt's cache is what has to be read.
        {"name": "attend_8_long_prompt", "kind": "attend", "fmt": "q8_0", "sequences": 8, "tokens": 1, "q_heads": 8,
         "kv_heads": 1, "head_dim": 256, "prefix": 100003, "capacity": 512, "shortest": 1, "longest": 512,
         "weights": False},
        # The benchmark's batched decode step behind a long prompt: products over the prompt are most of the work.
        {"name": "attend_256", "kind": "attend", "fmt": "f32", "sequences": 256, "tokens": 1, "q_heads": 8,
         "kv_heads": 1, "head_dim": 256, "prefix": 32768, "capacity": 512, "shortest": 1, "longest": 512,
         "weights": False},
        # Five drafted tokens at a time, grouped heads, an odd prompt, ragged own lengths, Q4_0.
        {"name": "attend_24_drafts", "kind": "attend", "fmt": "q4_0", "sequences": 24, "tokens": 5, "q_heads": 16,
         "kv_heads": 4, "head_dim": 128, "prefix": 4097, "capacity": 1024, "shortest": 3, "longest": 1001,
         "weights": True},
        # Long own caches behind a short prompt, with their weights: every cache has to be read.
        {"name": "attend_64_long_own", "kind": "attend", "fmt": "f32", "sequences": 64, "tokens": 1, "q_heads": 8,
         "kv_heads": 1, "head_dim": 256, "prefix": 1000, "capacity": 8192, "shortest": 1000, "longest": 8192,
         "weights": True},
        # One sequence at its budget: latency.
        {"name": "evict_one", "kind": "evict", "fmt": "f32", "sequences": 1, "kv_width": 192, "capacity": 2048,
         "shortest": 2048, "longest": 2048, "budget": 1024, "recent": 256},
        # A batch's caches, ragged: some are below the budget and only copied.
        {"name": "evict_256", "kind": "evict", "fmt": "f32", "sequences": 256, "kv_width": 256, "capacity": 1024,
         "shortest": 300, "longest": 1024, "budget": 512, "recent": 128},
        # Long contexts halved, wide Q8_0 rows.
        {"name": "evict_8_long", "kind": "evict", "fmt": "q8_0", "sequences": 8, "kv_width": 1024, "capacity": 65536,
         "shortest": 40001, "longest": 65536, "budget": 30000, "recent": 4096},
        # One sequence, four drafts, a small vocabulary: latency.
        {"name": "verify_one", "kind": "verify", "sequences": 1, "drafts": 4, "vocab": 49152, "certain": False,
         "shortest": 4, "temperature": 1.0},
        # A batch over the full vocabulary, both models' logits.
        {"name": "verify_64", "kind": "verify", "sequences": 64, "drafts": 4, "vocab": 262144, "certain": False,
         "shortest": 1, "temperature": 0.8},
        # Drafts looked up in the prompt (proposed with certainty), an odd vocabulary.
        {"name": "verify_256_lookup", "kind": "verify", "sequences": 256, "drafts": 3, "vocab": 50257, "certain": True,
         "shortest": 0, "temperature": 1.0},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _most(kind):
    works = [work(c) for c in listed() if c["kind"] == kind]
    return max(w["bytes"] for w in works), max(w["flops"] for w in works)


HELD = 3e9  # bytes of a drawn batch's own caches, filled or not


def _held(case):
    if case["kind"] == "verify":
        return 0
    width = case["kv_width"] if case["kind"] == "evict" else case["kv_heads"] * case["head_dim"]
    return 2 * _row_bytes(width, case["fmt"]) * case["sequences"] * case["capacity"]


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "evict", "verify"])
    if kind == "attend":
        q_heads, kv_heads, head_dim = rng.choice([(8, 1, 256), (8, 1, 256), (9, 3, 64), (32, 32, 64), (16, 4, 128),
                                                  (32, 8, 128), (12, 2, 96), (8, 2, 160), (16, 2, 256), (7, 1, 128)])
        case = {"fmt": rng.choice(["f32", "q8_0", "q4_0"]), "sequences": _log(rng, 1, 256),
                "tokens": rng.choice([1, 1, 1, rng.randint(2, 8)]), "q_heads": q_heads, "kv_heads": kv_heads,
                "head_dim": head_dim, "prefix": rng.choice([0, _log(rng, 1, 131072), _log(rng, 64, 32768), _log(rng, 64, 32768)]),
                "capacity": _log(rng, 1, 8192), "shortest": 0, "longest": 0, "weights": rng.random() < 0.4}
        case["longest"] = rng.randint(1, case["capacity"])
        case["shortest"] = rng.randint(0, case["longest"])
        shrink = ("sequences", "prefix", "longest")
    elif kind == "evict":
        capacity = _log(rng, 2, 65536)
        case = {"fmt": rng.choice(["f32", "q8_0", "q4_0"]), "sequences": _log(rng, 1, 256),
                "kv_width": rng.choice([64, 192, 256, 512, 768, 1024, 2048]), "capacity": capacity,
                "shortest": rng.randint(0, capacity), "longest": capacity, "budget": rng.randint(1, capacity), "recent": 0}
        case["recent"] = rng.randint(0, case["budget"])
        shrink = ("sequences", "kv_width", "sequences")
    else:
        drafts = rng.randint(1, 8)
        case = {"sequences": _log(rng, 1, 256), "drafts": drafts,
                "vocab": rng.choice([32000, 32001, 49152, 50257, 128256, 151936, 262144]), "certain": rng.random() < 0.3,
                "shortest": rng.randint(0, drafts), "temperature": rng.choice([0.6, 0.8, 1.0, 1.3])}
        shrink = ("sequences", "drafts", "vocab")
    case = {"kind": kind, **case}
    most = _most(kind)
    step = 0
    while _held(case) > HELD:
        case["sequences"] = max(1, case["sequences"] * 3 // 4)
    while work(case)["bytes"] > most[0] or work(case)["flops"] > most[1]:
        at = shrink[step % 3]
        if at == "kv_width":
            case[at] = max(64, case[at] // 2)
        else:
            case[at] = max(1, case[at] * 3 // 4)
        case["shortest"] = min(case["shortest"], case.get("longest", case.get("drafts")))
        step += 1
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


class _Draw:
    """Inputs from a seed, made on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.g, device="cuda").mul_(std)

    def uniform(self, low, high, *shape):
        return torch.rand(shape, generator=self.g, device="cuda") * (high - low) + low

    def lengths(self, count, low, high):
        """Evenly spread over [low, high] (one: high), in an order of the seed's."""
        low = high if count == 1 else low
        i = torch.arange(count, device="cuda", dtype=torch.float64)
        even = low + torch.floor(i * (high - low) / max(1, count - 1) + 0.5)
        return even[torch.randperm(count, generator=self.g, device="cuda")].to(torch.int32)

    def cache(self, positions, width, fmt):
        """Both planes of `positions` rows of values of about N(0, 1), as the KV append leaves them."""
        if fmt == "f32":
            return self.normal(2, positions, width)
        size, low, high = {"q8_0": (34, 0.008, 0.016), "q4_0": (18, 0.15, 0.3)}[fmt]
        t = torch.randint(0, 256, (2, positions, width // 32, size), generator=self.g, device="cuda", dtype=torch.uint8)
        t[..., :2] = self.uniform(low, high, 2, positions, width // 32).to(torch.float16).view(torch.uint8).reshape(2, positions, -1, 2)
        return t.reshape(2, positions, -1)


def _row_bytes(width, fmt):
    return {"f32": width * 4, "q8_0": width // 32 * 34, "q4_0": width // 32 * 18}[fmt]


def _values(rows, fmt, dtype):
    """A cache's rows, [..., row], as numbers."""
    if fmt == "f32":
        return rows.to(dtype)
    size = {"q8_0": 34, "q4_0": 18}[fmt]
    blocks = rows.shape[-1] // size
    b = rows.reshape(*rows.shape[:-1], blocks, size)
    d = b[..., :2].contiguous().view(torch.float16).to(dtype)
    if fmt == "q8_0":
        codes = b[..., 2:].contiguous().view(torch.int8).to(dtype)
    else:
        codes = torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], -1).to(dtype) - 8.0
    return (codes * d).reshape(*rows.shape[:-1], blocks * 32)


def prepare(case, seed):
    state = {"attend": _attend_inputs, "evict": _evict_inputs, "verify": _verify_inputs}[case["kind"]](case, _Draw(seed))
    state["case"] = case
    torch.cuda.synchronize()
    return state


def _attend_inputs(c, d):
    width = c["kv_heads"] * c["head_dim"]
    n, cap = c["sequences"], c["capacity"]
    s = {"q": d.normal(n, c["tokens"], c["q_heads"], c["head_dim"], std=2.0),
         "prefix": d.cache(c["prefix"], width, c["fmt"]) if c["prefix"] else None,
         "cache": d.cache(n * cap, width, c["fmt"]), "lengths": d.lengths(n, c["shortest"], c["longest"]),
         "scale": c["head_dim"] ** -0.5, "weights": d.uniform(0.0, 1.0, n, cap) if c["weights"] else None}
    s["out"] = torch.empty_like(s["q"])
    s["weights_out"] = torch.zeros_like(s["weights"]) if c["weights"] else None
    return s


def _evict_inputs(c, d):
    n, cap = c["sequences"], c["capacity"]
    s = {"cache": d.cache(n * cap, c["kv_width"], c["fmt"]), "lengths": d.lengths(n, c["shortest"], c["longest"]),
         # a few positions take most of the attention; unvisited ones share a weight of zero
         "weights": torch.relu(d.normal(n, cap)).pow_(4)}
    s["cache_out"] = torch.zeros_like(s["cache"])
    s["weights_out"] = torch.zeros_like(s["weights"])
    s["lengths_out"] = torch.zeros_like(s["lengths"])
    s["kept"] = torch.zeros(n, c["budget"], dtype=torch.int32, device="cuda")
    return s


def _verify_inputs(c, d):
    n, t, v = c["sequences"], c["drafts"], c["vocab"]
    x = d.normal(n, t + 1, v, std=4.0)
    draft = 30.0 * torch.tanh((x[:, :t] + d.normal(n, t, v)) / 30.0)
    target = 30.0 * torch.tanh(x.mul_(1.0 / 30.0))
    banned = torch.arange(v, device="cuda") % 97 == 5
    target[:, :, banned] = HUGE
    draft[:, :, banned] = -math.inf
    # a draft is drawn from the draft model: the largest of its scaled logits with Gumbel noise
    noise = -torch.log(-torch.log(d.uniform(1e-7, 1.0 - 1e-6, n, t, v)))
    tokens = torch.argmax(draft / c["temperature"] + noise, -1).to(torch.int32)
    return {"target": target, "draft": None if c["certain"] else draft.contiguous(), "tokens": tokens,
            "draft_lengths": d.lengths(n, c["shortest"], t), "accept": d.uniform(0.0, 1.0, n, t),
            "sample": d.uniform(0.0, 1.0, n), "accepted": torch.zeros(n, dtype=torch.int32, device="cuda"),
            "chosen": torch.zeros(n, t + 1, dtype=torch.int32, device="cuda")}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attend": _attend_own, "evict": _evict_own, "verify": _verify_own}[kind](state)
    return {"attend": _attend_plain, "evict": _evict_plain, "verify": _verify_plain}[kind](state)


@functools.lru_cache(maxsize=None)
def _runtime():
    from atlas_amd import HipRuntime

    rt = HipRuntime(0)
    # the tensors are torch's: the library's launches join its stream (1 names the legacy default stream, whose handle is 0
    # and would ask for the context's own)
    rt._check(rt.lib.atlas_hip_set_stream(rt.ctx, torch.cuda.current_stream().cuda_stream or 1))
    return rt


@functools.lru_cache(maxsize=None)
def _workspace(nbytes):
    """The workspace that a program of these sizes allocates once."""
    return _runtime().alloc(nbytes)


def _p(t):
    return None if t is None else t.data_ptr()


def _attend_own(s):
    c, rt = s["case"], _runtime()
    nbytes = rt.prefix_attention_workspace(c["fmt"], c["sequences"], c["tokens"], c["q_heads"], c["kv_heads"],
                                           c["head_dim"], c["prefix"], c["capacity"], c["weights"])
    rt.prefix_attention(c["fmt"], _p(s["q"]), _p(s["prefix"]), c["prefix"], c["prefix"], _p(s["cache"]), _p(s["lengths"]),
                        c["capacity"], _p(s["out"]), _p(s["weights"]), _p(s["weights_out"]), c["sequences"], c["tokens"],
                        c["q_heads"], c["kv_heads"], c["head_dim"], s["scale"], _workspace(nbytes), nbytes)
    return {"out": s["out"], "weights": s["weights_out"]}


def _evict_own(s):
    c, rt = s["case"], _runtime()
    rt.kv_evict(c["fmt"], _p(s["cache"]), _p(s["cache_out"]), _p(s["weights"]), _p(s["weights_out"]), _p(s["lengths"]),
                _p(s["lengths_out"]), _p(s["kept"]), c["sequences"], c["capacity"], c["kv_width"], c["budget"], c["recent"])
    return {"cache": s["cache_out"], "weights": s["weights_out"], "lengths": s["lengths_out"], "kept": s["kept"]}


def _verify_own(s):
    c, rt = s["case"], _runtime()
    nbytes = rt.verify_draft_workspace(c["sequences"], c["drafts"], c["vocab"])
    rt.verify_draft(_p(s["target"]), _p(s["draft"]), _p(s["tokens"]), _p(s["draft_lengths"]), _p(s["accept"]),
                    _p(s["sample"]), _p(s["accepted"]), _p(s["chosen"]), c["sequences"], c["drafts"], c["vocab"],
                    1.0 / c["temperature"], _workspace(nbytes), nbytes)
    return {"accepted": s["accepted"], "tokens": s["chosen"]}


def _attend_plain(s):
    """softmax over the prompt's and the sequence's own keys together.  Token t of a sequence of length n sees the
    prompt and its own positions below n - (tokens - 1 - t); a row that sees nothing is zero."""
    c = s["case"]
    n, t, h, kh, hd, cap, p = (c[k] for k in ("sequences", "tokens", "q_heads", "kv_heads", "head_dim", "capacity", "prefix"))
    g = h // kh
    q = (s["q"] * s["scale"]).view(n, t, kh, g, hd).permute(2, 0, 1, 3, 4).reshape(kh, n * t * g, hd)
    k, v = _values(s["cache"], c["fmt"], torch.float32).view(2, n, cap, kh, hd).permute(0, 3, 1, 2, 4)
    at = torch.arange(cap, device="cuda")
    length = s["lengths"].long()
    v = torch.where((at < length[:, None])[None, :, :, None], v, 0.0)  # what lies behind a sequence is anything
    seen = at < length[:, None, None] - (t - 1 - torch.arange(t, device="cuda"))[None, :, None]
    scores = q.view(kh, n, t * g, hd) @ k.transpose(2, 3).contiguous()
    scores = torch.where(seen[None, :, :, None], scores.view(kh, n, t, g, cap), -math.inf).view(kh, n * t * g, cap)
    top = scores.amax(2, keepdim=True)
    if p:
        pk, pv = _values(s["prefix"], c["fmt"], torch.float32).view(2, p, kh, hd).permute(0, 2, 1, 3)
        pscores = q @ pk.transpose(1, 2).contiguous()
        top = torch.maximum(top, pscores.amax(2, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(scores - top)
    total = e.sum(2, keepdim=True)
    out = (e.view(kh, n, t * g, cap) @ v.contiguous()).view(kh, n * t * g, hd)
    if p:
        pe = torch.exp(pscores - top)
        total = total + pe.sum(2, keepdim=True)
        out = out + pe @ pv.contiguous()
    out = torch.where(total > 0, out / total, 0.0)
    out = out.view(kh, n, t, g, hd).permute(1, 2, 0, 3, 4).reshape(n, t, h, hd)
    weights = None
    if c["weights"]:
        share = torch.where(total > 0, e / total, 0.0).view(kh, n, t * g, cap).sum((0, 2))
        weights = torch.where(at < length[:, None], s["weights"] + share, s["weights_out"])
    return {"out": out, "weights": weights}


def _evict_plain(s):
    """A sequence longer than the budget keeps its `recent` last positions and the heaviest of the others (of equal
    weights the first), in their order; what lies behind the kept rows stays as it was."""
    c = s["case"]
    n, cap, budget = c["sequences"], c["capacity"], c["budget"]
    at = torch.arange(cap, device="cuda")
    length = s["lengths"].long()[:, None]
    recent = at >= length - c["recent"]
    rank = torch.where(recent, math.inf, s["weights"])
    rank = torch.where(at < length, rank, -math.inf)
    order = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :budget]
    keep = torch.zeros(n, cap, dtype=torch.bool, device="cuda").scatter_(1, order, True) & (at < length)
    kept = torch.sort(torch.where(keep, at, cap), dim=1).values[:, :budget]
    there = kept < cap
    source = torch.where(there, kept, 0)
    rows = (torch.arange(n, device="cuda")[:, None] * cap + source).reshape(-1)
    moved = s["cache"][:, rows].view(2, n, budget, -1)
    cache = s["cache_out"].clone()
    first = cache.view(2, n, cap, -1)[:, :, :budget]
    first.copy_(torch.where(there[None, :, :, None], moved, first))
    weights = s["weights_out"].clone()
    weights[:, :budget] = torch.where(there, torch.gather(s["weights"], 1, source), weights[:, :budget])
    return {"cache": cache, "weights": weights, "lengths": there.sum(1).to(torch.int32),
            "kept": torch.where(there, kept, NO_TOKEN).to(torch.int32)}


def _softmax64(x, temperature):
    x = x.double() * (1.0 / temperature)
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.amax(-1, keepdim=True)
    e = torch.where(x == top, 1.0, torch.exp(x - top))
    e = torch.where(top == -math.inf, 0.0, e)
    total = e.sum(-1, keepdim=True)
    return torch.where(total > 0, e / total, 0.0)


def _verify_plain(s):
    """Draft t is accepted while accept[t] * q(token) < p(token); after the first rejection a token is drawn from
    max(p - q, 0), after none from the target's next row: the first whose running sum exceeds sample * sum."""
    c = s["case"]
    n, t, v = c["sequences"], c["drafts"], c["vocab"]
    p = _softmax64(s["target"], c["temperature"])
    token = s["tokens"].long()
    if c["certain"]:
        q = torch.zeros(n, t, v, dtype=torch.float64, device="cuda").scatter_(2, token[:, :, None], 1.0)
    else:
        q = _softmax64(s["draft"], c["temperature"])
    pt = torch.gather(p[:, :t], 2, token[:, :, None])[:, :, 0]
    qt = torch.gather(q, 2, token[:, :, None])[:, :, 0]
    at = torch.arange(t, device="cuda")
    length = s["draft_lengths"].long()
    ok = (s["accept"].double() * qt < pt) & (at < length[:, None])
    accepted = torch.cumprod(ok.long(), 1).sum(1)
    row = accepted[:, None, None].expand(n, 1, v)
    p = torch.gather(p, 1, row)[:, 0]
    q = torch.gather(q, 1, torch.clamp(row, max=t - 1))[:, 0]
    rest = torch.where((accepted < length)[:, None], torch.clamp(p - q, min=0.0), p)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p)
    run_sum = torch.cumsum(rest, 1)
    goal = s["sample"].double() * run_sum[:, -1]
    drawn = torch.clamp((run_sum <= goal[:, None]).sum(1), max=v - 1)
    drawn = torch.where(run_sum[:, -1] > 0, drawn, NO_TOKEN)
    place = torch.arange(t + 1, device="cuda")
    tokens = torch.cat([token, token[:, :1]], 1)
    tokens = torch.where(place < accepted[:, None], tokens, NO_TOKEN)
    tokens = torch.where(place == accepted[:, None], drawn[:, None], tokens)
    return {"accepted": accepted.to(torch.int32), "tokens": tokens.to(torch.int32)}


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its results in 64 bits
# ---------------------------------------------------------------------------


def _mean_length(c):
    return c["longest"] if c["sequences"] == 1 else 0.5 * (c["shortest"] + c["longest"])


def work(case):
    c = case
    n = c["sequences"]
    if c["kind"] == "attend":
        row = _row_bytes(c["kv_heads"] * c["head_dim"], c["fmt"])
        mean = _mean_length(c)
        rows = n * c["tokens"] * c["q_heads"]
        own_keys = max(0.0, mean - 0.5 * (c["tokens"] - 1))
        return {"bytes": 8.0 * rows * c["head_dim"] + 2.0 * row * (c["prefix"] + n * mean) + 4.0 * n + (8.0 * n * mean if c["weights"] else 0.0),
                "flops": 4.0 * c["head_dim"] * rows * (c["prefix"] + own_keys)}
    if c["kind"] == "evict":
        row = _row_bytes(c["kv_width"], c["fmt"])
        mean = _mean_length(c)
        # lengths are spread evenly: the mean of min(length, budget)
        low, high, most = (c["longest"] if n == 1 else c["shortest"]), c["longest"], c["budget"]
        kept = min(most, mean) if low >= most or high <= most else (0.5 * (low + most) * (most - low) + most * (high - most)) / (high - low)
        return {"bytes": n * (4.0 * mean + 4.0 * row * kept + 4.0 * kept + 4.0 * most + 8.0), "flops": n * mean}
    rows = n * (c["drafts"] + 1 + (0 if c["certain"] else c["drafts"]))
    return {"bytes": 4.0 * rows * c["vocab"] + 4.0 * n * (4 * c["drafts"] + 4), "flops": 4.0 * rows * c["vocab"]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _attend_exact, "evict": _evict_exact, "verify": _verify_exact}[case["kind"]](s)


def _attend_exact(s):
    """Sequence by sequence, head by head: the definition over the keys that a token sees."""
    c = s["case"]
    n, t, h, kh, hd, cap, p = (c[k] for k in ("sequences", "tokens", "q_heads", "kv_heads", "head_dim", "capacity", "prefix"))
    g = h // kh
    if n * t * kh > 4096 or work(c)["flops"] > 1e11:
        return None
    f64 = torch.float64
    out = torch.zeros(n, t, h, hd, dtype=f64, device="cuda")
    weights = s["weights_out"].double() if c["weights"] else None
    lengths = s["lengths"].tolist()
    pk, pv = _values(s["prefix"], c["fmt"], f64).view(2, p, kh, hd) if p else torch.zeros(2, 0, kh, hd, dtype=f64, device="cuda")
    mine = s["cache"].view(2, n, cap, -1)
    for b in range(n):
        k, v = _values(mine[:, b, :lengths[b]], c["fmt"], f64).reshape(2, lengths[b], kh, hd)
        if c["weights"]:
            weights[b, :lengths[b]] = s["weights"][b, :lengths[b]].double()
        for i in range(t):
            see = max(0, lengths[b] - (t - 1 - i))
            if p + see == 0:
                continue
            for j in range(kh):
                keys, values = torch.cat([pk[:, j], k[:see, j]]), torch.cat([pv[:, j], v[:see, j]])
                x = torch.mv if g == 1 else torch.mm
                q = s["q"][b, i, j * g:(j + 1) * g].double()
                prob = torch.softmax((x(keys, q[0])[:, None] if g == 1 else x(keys, q.t().contiguous())) * s["scale"], 0)
                out[b, i, j * g:(j + 1) * g] = prob.t().contiguous() @ values
                if c["weights"]:
                    weights[b, :see] += prob[p:].sum(1)
    return {"out": out, "weights": weights}


def _evict_exact(s):
    c = s["case"]
    n, cap, budget = c["sequences"], c["capacity"], c["budget"]
    if work(c)["bytes"] > 3e9:
        return None
    cache, weights = s["cache_out"].clone().view(2, n, cap, -1), s["weights_out"].double()
    lengths = torch.zeros(n, dtype=torch.int32, device="cuda")
    kept = torch.full((n, budget), NO_TOKEN, dtype=torch.int32, device="cuda")
    source = s["cache"].view(2, n, cap, -1)
    for b, length in enumerate(s["lengths"].tolist()):
        w = s["weights"][b, :length].tolist()
        if length <= budget:
            stay = list(range(length))
        else:
            old = length - c["recent"]
            stay = sorted(sorted(range(old), key=lambda i: (-w[i], i))[:budget - c["recent"]]) + list(range(old, length))
        i = torch.tensor(stay, dtype=torch.long, device="cuda")
        cache[:, b, :len(stay)] = source[:, b, i]
        weights[b, :len(stay)] = s["weights"][b, i].double()
        lengths[b] = len(stay)
        kept[b, :len(stay)] = i.to(torch.int32)
    cache = cache.reshape(s["cache_out"].shape)
    return {"cache": cache.double() if c["fmt"] == "f32" else cache, "weights": weights, "lengths": lengths, "kept": kept}


def _verify_exact(s):
    """Sequence by sequence, draft by draft, as the rule is read aloud."""
    c = s["case"]
    n, t = c["sequences"], c["drafts"]

    def distribution(logits):
        return torch.softmax(logits.double() / c["temperature"], 0)

    accepted, tokens = [], []
    lengths, drafts = s["draft_lengths"].tolist(), s["tokens"].tolist()
    accept, sample = s["accept"].tolist(), s["sample"].tolist()
    for b in range(n):
        line, rest = [], None
        for i in range(lengths[b]):
            p, x = distribution(s["target"][b, i]), drafts[b][i]
            q = torch.zeros_like(p) if c["certain"] else distribution(s["draft"][b, i])
            if c["certain"]:
                q[x] = 1.0
            if accept[b][i] * float(q[x]) >= float(p[x]):
                rest = torch.relu(p - q)
                rest = rest if float(rest.sum()) > 0 else p
                break
            line.append(x)
        accepted.append(len(line))
        if rest is None:
            rest = distribution(s["target"][b, lengths[b]])
        total = torch.cumsum(rest, 0)
        line.append(int(torch.searchsorted(total, total[-1:] * sample[b], right=True)[0]))
        tokens.append(line + [NO_TOKEN] * (t + 1 - len(line)))
    return {"accepted": torch.tensor(accepted, dtype=torch.int32, device="cuda"),
            "tokens": torch.tensor(tokens, dtype=torch.int32, device="cuda")}
