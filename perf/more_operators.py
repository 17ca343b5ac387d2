"""Decoding a batch from a paged cache, as cases to time.

Four operators of a serving loop that keeps keys and values in pages of a pool
and answers with the probabilities of what it chose:

    append    new tokens' keys are rotated to their positions and stored with
              their values in the pages that a table names; their queries are
              rotated in the same pass
    attend    one new token of each sequence attends to the sequence's pages,
              to all of them or to a window of the last positions
    read      cached rows as f32, for products that are not this framework's
    logprobs  log probabilities of given tokens, a row's entropy and its most
              likely tokens

A pool is [page][K | V][KV head][part]; a part holds `page_size` rows of
head_dim values.  f32 and f16 parts are [row][head_dim].  A quantised part is
the codes, [row][codes], then the scales, f16 [row / 4][block][row % 4], a block
being 32 values: Q8_0 a byte a code, Q4_0 two codes a byte (the first one low;
value = (code - 8) * scale).  Codes of a key are in the order of its dims.
Codes of a value: its blocks in runs of 8, 4, 2 and 1 (the binary digits of
head_dim / 32, the largest first), a run as [16][block][2]: of dims
32 block + 2 i + e, e = 0, 1, the sixteen i's.  Entries of the table that name no page
of the pool (NO_PAGE) hold nothing.  Head layouts, widths and vocabularies are
those of the benchmark configurations and tests, or generic ones.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

NO_PAGE = -1   # 0xffffffff
NO_TOKEN = -1


def listed():
    return [
        # The smallest call: one sequence's next token, a small model's heads: latency.
        {"name": "append_one", "kind": "append", "fmt": "f32", "sequences": 1, "tokens": 1, "q_heads": 9, "kv_heads": 3,
         "head_dim": 64, "page_size": 16, "capacity": 2048},
        # The benchmark's batched decode step: 256 sequences at any position.
        {"name": "append_256", "kind": "append", "fmt": "q8_0", "sequences": 256, "tokens": 256, "q_heads": 8, "kv_heads": 1,
         "head_dim": 256, "page_size": 64, "capacity": 8192},
        # A prefill chunk of three prompts of different lengths.
        {"name": "append_4096", "kind": "append", "fmt": "f16", "sequences": 3, "tokens": 4096, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "page_size": 16, "capacity": 8192},
        # One sequence, the small model: latency.
        {"name": "attend_one", "kind": "attend", "fmt": "f32", "sequences": 1, "q_heads": 9, "kv_heads": 3, "head_dim": 64,
         "page_size": 16, "capacity": 2048, "shortest": 701, "longest": 701, "window": 0},
        # One very long context: the cache is split over the whole chip.
        {"name": "attend_one_long", "kind": "attend", "fmt": "q4_0", "sequences": 1, "q_heads": 8, "kv_heads": 1,
         "head_dim": 256, "page_size": 256, "capacity": 262144, "shortest": 261001, "longest": 261001, "window": 0},
        # A ragged batch of grouped heads.
        {"name": "attend_24_ragged", "kind": "attend", "fmt": "q8_0", "sequences": 24, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "page_size": 16, "capacity": 32768, "shortest": 1000, "longest": 30001, "window": 0},
        # A sliding-window layer of the batch in f16; pages behind the window are given back.
        {"name": "attend_256_window", "kind": "attend", "fmt": "f16", "sequences": 256, "q_heads": 8, "kv_heads": 1,
         "head_dim": 256, "page_size": 32, "capacity": 4096, "shortest": 0, "longest": 4096, "window": 512},
        # A short prompt that a next chunk attends to.
        {"name": "read_500", "kind": "read", "fmt": "f16", "sequences": 1, "rows": 500, "kv_heads": 3, "head_dim": 64,
         "page_size": 16, "capacity": 2048},
        # A long prompt's rows.
        {"name": "read_32768", "kind": "read", "fmt": "q4_0", "sequences": 2, "rows": 32768, "kv_heads": 8, "head_dim": 128,
         "page_size": 64, "capacity": 65536},
        # One sequence's chosen token and five alternatives: latency.
        {"name": "logprobs_one", "kind": "logprobs", "rows": 1, "vocab": 49152, "pad": 0, "given": 1, "top": 5,
         "entropy": False, "temperature": 1.0},
        # A batch over the full vocabulary, twenty alternatives.
        {"name": "logprobs_256", "kind": "logprobs", "rows": 256, "vocab": 262144, "pad": 0, "given": 1, "top": 20,
         "entropy": True, "temperature": 0.8},
        # Scoring a long prompt: no alternatives, an odd vocabulary.
        {"name": "logprobs_2048_prompt", "kind": "logprobs", "rows": 2048, "vocab": 50257, "pad": 0, "given": 1, "top": 0,
         "entropy": True, "temperature": 1.0},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


HEADS = [(8, 1, 256), (8, 1, 256), (9, 3, 64), (32, 32, 64), (16, 4, 128), (32, 8, 128), (12, 2, 96), (8, 2, 160),
         (16, 2, 256), (7, 1, 128), (16, 1, 192), (24, 1, 64), (4, 4, 32)]
HELD = 3e9    # bytes of a drawn pool
PLAIN = 8e9   # bytes of its rows as f32, padded to the longest


def _pool_pages(c):
    each = -(-c["capacity"] // c["page_size"])
    return c["sequences"] * each


def _held(c):
    return _pool_pages(c) * 2.0 * c["kv_heads"] * _part_bytes(c)


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "read", "logprobs", "logprobs"])
    if kind == "logprobs":
        case = {"rows": _log(rng, 1, 4096), "vocab": rng.choice([32000, 32001, 49152, 50257, 128256, 151936, 262144]),
                "pad": rng.choice([0, 0, 47]), "given": rng.choice([0, 1, 1, 4]), "top": rng.choice([0, 1, 5, 20, 64]),
                "entropy": rng.random() < 0.5, "temperature": rng.choice([0.6, 0.8, 1.0, 1.3])}
        if case["given"] + case["top"] + case["entropy"] == 0:
            case["top"] = 1
        shrink = ("rows", "vocab", "rows")
    else:
        q_heads, kv_heads, head_dim = rng.choice(HEADS)
        case = {"fmt": rng.choice(["f32", "f16", "q8_0", "q4_0"]), "sequences": _log(rng, 1, 256), "q_heads": q_heads,
                "kv_heads": kv_heads, "head_dim": head_dim, "page_size": rng.choice([16, 16, 32, 64, 128, 256]),
                "capacity": _log(rng, 16, 262144)}
        if case["fmt"] in ("f32", "f16") and rng.random() < 0.2:
            case["head_dim"] = rng.choice([72, 80, 200])
        if kind == "attend":
            case["longest"] = case["capacity"]
            case["shortest"] = rng.randint(0, case["longest"])
            case["window"] = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
            shrink = ("sequences", "capacity", "capacity")
        elif kind == "append":
            decode = rng.random() < 0.5
            case["tokens"] = case["sequences"] if decode else _log(rng, 1, 4096)
            shrink = ("tokens", "sequences", "capacity")
        else:
            case["rows"] = _log(rng, 1, 32768)
            case.pop("q_heads")
            shrink = ("rows", "sequences", "capacity")
    case = {"kind": kind, **case}
    works = [work(c) for c in listed() if c["kind"] == kind]
    most = max(w["bytes"] for w in works), max(w["flops"] for w in works)
    step = 0
    while (work(case)["bytes"] > most[0] or work(case)["flops"] > most[1] or
           (kind != "logprobs" and (_held(case) > HELD or _plain(case) > PLAIN)) or
           case.get("tokens", case.get("rows", 0)) > case.get("sequences", 1 << 30) * case.get("capacity", 1 << 30)):
        at = shrink[step % 3]
        if case.get("tokens", case.get("rows", 0)) > case.get("sequences", 1 << 30) * case.get("capacity", 1 << 30):
            at = "tokens" if "tokens" in case else "rows"
        case[at] = max(1, case[at] * 3 // 4)
        if kind == "attend":
            case["longest"] = case["capacity"]
            case["shortest"] = min(case["shortest"], case["longest"])
        step += 1
    return case


def _plain(c):
    if c["kind"] != "attend":
        return 0
    return 8.0 * c["sequences"] * c["capacity"] * c["kv_heads"] * c["head_dim"]


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

    def order(self, count):
        return torch.randperm(count, generator=self.g, device="cuda")

    def lengths(self, count, low, high):
        """Evenly spread over [low, high] (one: high), in an order of the seed's."""
        low = high if count == 1 else low
        i = torch.arange(count, device="cuda", dtype=torch.float64)
        return torch.floor(low + i * (high - low) / max(1, count - 1) + 0.5)[self.order(count)].to(torch.int32)

    def pool(self, c):
        """Pages of values of about N(0, 1)."""
        n, kh, ps, hd = _pool_pages(c), c["kv_heads"], c["page_size"], c["head_dim"]
        if c["fmt"] == "f32":
            return self.normal(n, 2, kh, ps, hd)
        if c["fmt"] == "f16":
            pool = torch.empty(n, 2, kh, ps, hd, dtype=torch.float16, device="cuda")
            return pool.normal_(generator=self.g)
        codes = ps * hd * (2 if c["fmt"] == "q8_0" else 1) // 2
        low, high = {"q8_0": (0.008, 0.016), "q4_0": (0.15, 0.3)}[c["fmt"]]
        pool = torch.randint(0, 256, (n, 2, kh, _part_bytes(c)), generator=self.g, device="cuda", dtype=torch.uint8)
        pool[..., codes:] = self.uniform(low, high, n, 2, kh, ps * hd // 32).to(torch.float16).view(torch.uint8)
        return pool


def _part_bytes(c):
    """Bytes of one head's rows of K or V in a page."""
    n = c["page_size"] * c["head_dim"]
    return {"f32": 4 * n, "f16": 2 * n, "q8_0": n // 32 * 34, "q4_0": n // 32 * 18}[c["fmt"]]


def _value_order(blocks):
    """The dims of a value's codes, in their order."""
    dims, first, run = [], 0, 1 << (blocks.bit_length() - 1)
    while first < blocks:
        if run <= blocks - first:
            dims += [32 * (first + j) + 2 * i + e for i in range(16) for j in range(run) for e in range(2)]
            first += run
        run //= 2
    return dims


def prepare(case, seed):
    state = {"append": _append_inputs, "attend": _attend_inputs, "read": _read_inputs,
             "logprobs": _logprobs_inputs}[case["kind"]](case, _Draw(seed))
    state["case"] = case
    torch.cuda.synchronize()
    return state


def _paged_inputs(c, d):
    n, width = c["sequences"], -(-c["capacity"] // c["page_size"])
    table = d.order(_pool_pages(c)).to(torch.int32).view(n, width)
    s = {"pool": d.pool(c), "table": table, "width": width}
    if c["fmt"] in ("q8_0", "q4_0"):
        order = torch.tensor(_value_order(c["head_dim"] // 32), device="cuda")
        s["value_order"], s["value_place"] = order, torch.argsort(order)
    return s


def _places(c, d, rows):
    """Sequences and positions of `rows` tokens: one each, or runs of consecutive positions."""
    n, cap = c["sequences"], c["capacity"]
    if rows == n:
        return torch.arange(n, device="cuda"), torch.floor(d.uniform(0, cap, n).double()).long().clamp(max=cap - 1)
    each = [rows // n + (1 if i < rows % n else 0) for i in range(n)]
    move = min(each[0] - 1, cap - each[0], each[-1] // 3)  # ragged: from the last sequence to the first
    if n > 1 and move > 0:
        each[0] += move
        each[-1] -= move
    count = torch.tensor(each, device="cuda")
    sequence = torch.repeat_interleave(torch.arange(n, device="cuda"), count)
    first = torch.floor(d.uniform(0, 1, n).double() * (cap - count + 1)).long().clamp(min=0)
    first = torch.minimum(first, cap - count)
    return sequence, torch.arange(rows, device="cuda") - (torch.cumsum(count, 0) - count)[sequence] + first[sequence]


def _append_inputs(c, d):
    s = _paged_inputs(c, d)
    t, h, kh, hd = c["tokens"], c["q_heads"], c["kv_heads"], c["head_dim"]
    sequence, position = _places(c, d, t)
    angle = torch.arange(s["width"] * c["page_size"], device="cuda", dtype=torch.float64)[:, None] * torch.pow(
        torch.tensor(1e4, device="cuda", dtype=torch.float64), -torch.arange(hd // 2, device="cuda", dtype=torch.float64) * 2.0 / hd)
    s.update(sequence=sequence.to(torch.int32), position=position.to(torch.int32), cos=torch.cos(angle).float(),
             sin=torch.sin(angle).float(), key=d.normal(t, kh, hd), value=d.normal(t, kh, hd), query=d.normal(t, h, hd))
    s["query_out"] = torch.zeros_like(s["query"])
    if c["fmt"] in ("q8_0", "q4_0"):
        s["key_out"], s["value_out"] = torch.zeros_like(s["key"]), torch.zeros_like(s["value"])
    return s


def _attend_inputs(c, d):
    s = _paged_inputs(c, d)
    s["lengths"] = d.lengths(c["sequences"], c["shortest"], c["longest"])
    first = torch.arange(s["width"], device="cuda") * c["page_size"]
    length = s["lengths"][:, None]
    gone = first >= length
    if c["window"]:
        gone |= first + c["page_size"] <= length - c["window"]
    s["table"] = torch.where(gone, NO_PAGE, s["table"]).contiguous()
    s["q"] = d.normal(c["sequences"], c["q_heads"], c["head_dim"], std=2.0)
    s["out"] = torch.empty_like(s["q"])
    s["scale"] = c["head_dim"] ** -0.5
    return s


def _read_inputs(c, d):
    s = _paged_inputs(c, d)
    sequence, position = _places(c, d, c["rows"])
    s.update(sequence=sequence.to(torch.int32), position=position.to(torch.int32))
    s["key_out"] = torch.zeros(c["rows"], c["kv_heads"], c["head_dim"], device="cuda")
    s["value_out"] = torch.zeros_like(s["key_out"])
    return s


def _logprobs_inputs(c, d):
    n, v = c["rows"], c["vocab"]
    x = torch.tanh(d.normal(n, v + c["pad"], std=4.0).mul_(1.0 / 30.0)).mul_(30.0)
    x[:, 5:v:97] = -math.inf  # banned tokens
    s = {"logits": x, "tokens": torch.randint(0, v, (n, c["given"]), generator=d.g, device="cuda", dtype=torch.int32)}
    if c["given"]:
        # mostly likely ones: the best of the row's next sixteen
        near = (s["tokens"][:, :1].long() + torch.arange(16, device="cuda")) % v
        s["tokens"][:, 0] = torch.gather(near, 1, torch.gather(x, 1, near).argmax(1, keepdim=True))[:, 0].to(torch.int32)
        s["tokens"] += (s["tokens"] % 97 == 5).to(torch.int32)  # a banned one was not chosen
        s["tokens"].clamp_(max=v - 1)
    s["logprobs"] = torch.zeros(n, c["given"], device="cuda") if c["given"] else None
    s["entropy"] = torch.zeros(n, device="cuda") if c["entropy"] else None
    s["top_ids"] = torch.zeros(n, c["top"], dtype=torch.int32, device="cuda") if c["top"] else None
    s["top_logprobs"] = torch.zeros(n, c["top"], device="cuda") if c["top"] else None
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"append": _append_own, "attend": _attend_own, "read": _read_own, "logprobs": _logprobs_own}[kind](state)
    return {"append": _append_plain, "attend": _attend_plain, "read": _read_plain, "logprobs": _logprobs_plain}[kind](state)


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


def _cache(s):
    c = s["case"]
    return _runtime().paged_cache(c["fmt"], _p(s["pool"]), _pool_pages(c), c["page_size"], c["kv_heads"], c["head_dim"],
                                  _p(s["table"]), c["sequences"], s["width"])


def _append_own(s):
    c, rt, cache = s["case"], _runtime(), _cache(s)
    rt.paged_append(cache, _p(s["key"]), _p(s["value"]), _p(s["query"]), _p(s["query_out"]), _p(s["cos"]), _p(s["sin"]),
                    s["cos"].shape[0], c["head_dim"] // 2, _p(s["sequence"]), _p(s["position"]), c["tokens"], c["q_heads"])
    if c["fmt"] in ("f32", "f16"):
        return {"query": s["query_out"], "pool": s["pool"]}
    rt.paged_read(cache, _p(s["sequence"]), _p(s["position"]), c["tokens"], _p(s["key_out"]), _p(s["value_out"]))
    return {"query": s["query_out"], "key": s["key_out"], "value": s["value_out"]}


def _attend_own(s):
    c, rt, cache = s["case"], _runtime(), _cache(s)
    nbytes = rt.paged_attention_workspace(cache, c["q_heads"])
    rt.paged_attention(cache, _p(s["q"]), _p(s["lengths"]), _p(s["out"]), c["q_heads"], s["scale"], c["window"],
                       _workspace(nbytes), nbytes)
    return s["out"]


def _read_own(s):
    c, rt = s["case"], _runtime()
    rt.paged_read(_cache(s), _p(s["sequence"]), _p(s["position"]), c["rows"], _p(s["key_out"]), _p(s["value_out"]))
    return {"key": s["key_out"], "value": s["value_out"]}


def _logprobs_own(s):
    c, rt = s["case"], _runtime()
    nbytes = rt.token_logprobs_workspace(c["rows"], c["vocab"], c["top"])
    rt.token_logprobs(_p(s["logits"]), c["vocab"] + c["pad"], _p(s["tokens"]) if c["given"] else None, c["given"],
                      _p(s["logprobs"]), _p(s["entropy"]), _p(s["top_ids"]), _p(s["top_logprobs"]), c["rows"], c["vocab"],
                      c["top"], 1.0 / c["temperature"], _workspace(nbytes), nbytes)
    return {"logprobs": s["logprobs"], "entropy": s["entropy"], "ids": s["top_ids"], "tops": s["top_logprobs"]}


def _codes_and_scales(pool, c):
    """Views of a quantised pool: codes [.., row, bytes] and scales [.., row / 4, block, 4]."""
    ps, hd = c["page_size"], c["head_dim"]
    row = hd if c["fmt"] == "q8_0" else hd // 2
    codes = pool[..., :ps * row].unflatten(-1, (ps, row))
    return codes, pool[..., ps * row:].view(torch.float16).unflatten(-1, (ps // 4, hd // 32, 4))


def _decode(codes, scales, order, c, dtype):
    """Rows as numbers from codes [.., bytes] and scales [.., blocks]; `order`: the place of each dim among the codes."""
    if c["fmt"] == "q8_0":
        x = codes.contiguous().view(torch.int8).to(dtype)
    else:
        x = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(dtype) - 8.0
    if order is not None:
        x = x[..., order]
    return (x.unflatten(-1, (-1, 32)) * scales[..., None].to(dtype)).flatten(-2)


def _pages(s, plane, table, dtype=torch.float32):
    """K (plane 0) or V (1) of pages `table` [..]: [.., KV head, row, head_dim]."""
    c = s["case"]
    if c["fmt"] in ("f32", "f16"):
        return s["pool"][table, plane].to(dtype)
    codes, scales = _codes_and_scales(s["pool"][table, plane], c)
    return _decode(codes, scales.transpose(-1, -2).flatten(-3, -2), s["value_place"] if plane else None, c, dtype)


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    x0, x1, cos, sin = x[..., :half], x[..., half:], cos[:, None], sin[:, None]
    return torch.cat([x0 * cos - x1 * sin, x0 * sin + x1 * cos], -1)


def _encode(x, c):
    """Codes [.., head_dim], in the order of the dims, and scales [.., blocks] of rows x."""
    b = x.unflatten(-1, (-1, 32))
    size = b.abs()
    top, at = size.amax(-1, keepdim=True), size.argmax(-1, keepdim=True)
    first = torch.where(size == top, torch.arange(32, device="cuda"), 32).amin(-1, keepdim=True)
    if c["fmt"] == "q8_0":
        scale = top / torch.full_like(top, 127.0)
        y = b / torch.where(scale == 0, 1.0, scale)
        codes = torch.sign(y) * torch.floor(y.clamp(-127.0, 127.0).abs().double() + 0.5)
        codes = codes.to(torch.int8).view(torch.uint8)
    else:
        scale = torch.gather(b, -1, torch.where(top == 0, at, first)) / torch.full_like(top, -8.0)
        y = b / torch.where(scale == 0, 1.0, scale) + 8.5
        codes = torch.where(scale == 0, 0.0, torch.trunc(y.clamp(0.0, 15.0))).to(torch.uint8)
    return codes.flatten(-2), scale[..., 0].to(torch.float16)


def _append_plain(s):
    """Row `position` of a sequence is row position % page_size of page table[sequence, position / page_size]."""
    c = s["case"]
    at = s["position"].long()
    page, row = s["table"][s["sequence"].long(), at // c["page_size"]].long(), at % c["page_size"]
    cos, sin = s["cos"][at], s["sin"][at]
    query, key, value = _rotate(s["query"], cos, sin), _rotate(s["key"], cos, sin), s["value"]
    if c["fmt"] in ("f32", "f16"):
        for plane, x in enumerate((key, value)):
            s["pool"][page, plane, :, row] = x.to(s["pool"].dtype)
        return {"query": query, "pool": s["pool"]}
    codes, scales = _codes_and_scales(s["pool"], c)
    out = {"query": query}
    for plane, x in enumerate((key, value)):
        code, scale = _encode(x, c)
        if plane:
            code = code[..., s["value_order"]]
        if c["fmt"] == "q4_0":
            code = code[..., ::2] | code[..., 1::2] << 4
        codes[page, plane, :, row] = code
        scales[page, plane, :, row // 4, :, row % 4] = scale
        out["value" if plane else "key"] = _decode(codes[page, plane, :, row], scales[page, plane, :, row // 4, :, row % 4],
                                                   s["value_place"] if plane else None, c, torch.float32)
    return out


def _attend_plain(s):
    """softmax over the positions of a sequence (its last `window` ones) whose page is there; nothing seen: zero."""
    c = s["case"]
    n, h, kh, hd = c["sequences"], c["q_heads"], c["kv_heads"], c["head_dim"]
    table = s["table"].long()
    at = torch.arange(s["width"] * c["page_size"], device="cuda")
    length = s["lengths"].long()[:, None]
    seen = (at < length) & (table >= 0).repeat_interleave(c["page_size"], 1)
    if c["window"]:
        seen &= at >= length - c["window"]
    table = table.clamp(min=0)

    def plane(i):
        return _pages(s, i, table).transpose(1, 2).reshape(n, kh, -1, hd)

    q = (s["q"] * s["scale"]).view(n, kh, h // kh, hd)
    scores = torch.where(seen[:, None, None], q @ plane(0).transpose(2, 3).contiguous(), -math.inf)
    top = scores.amax(3, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(3, keepdim=True)
    out = e @ torch.where(seen[:, None, :, None], plane(1), 0.0)
    return torch.where(total > 0, out / total, 0.0).reshape(n, h, hd)


def _read_plain(s):
    c = s["case"]
    at = s["position"].long()
    page, row = s["table"][s["sequence"].long(), at // c["page_size"]].long(), at % c["page_size"]
    if c["fmt"] in ("f32", "f16"):
        return {"key": s["pool"][page, 0, :, row].float(), "value": s["pool"][page, 1, :, row].float()}
    codes, scales = _codes_and_scales(s["pool"], c)
    key, value = (_decode(codes[page, i, :, row], scales[page, i, :, row // 4, :, row % 4], s["value_place"] if i else None,
                          c, torch.float32) for i in range(2))
    return {"key": key, "value": value}


def _logprobs_plain(s):
    """log p = x / temperature - log(sum of e^(x / temperature)); entropy = -sum of p log p."""
    c = s["case"]
    x = s["logits"][:, :c["vocab"]].double() * (1.0 / c["temperature"])
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    out = {"logprobs": None, "entropy": None, "ids": None, "tops": None}
    if c["given"]:
        out["logprobs"] = (torch.gather(x, 1, s["tokens"].long()) - top - log_total).float()
    if c["entropy"]:
        out["entropy"] = (log_total[:, 0] + torch.where(e > 0, e * (top - x), 0.0).sum(1) / total[:, 0]).float()
    if c["top"]:
        values, ids = torch.sort(s["logits"][:, :c["vocab"]], dim=1, descending=True, stable=True)
        out["ids"] = ids[:, :c["top"]].to(torch.int32)
        out["tops"] = (values[:, :c["top"]].double() * (1.0 / c["temperature"]) - top - log_total).float()
    return out


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its results in 64 bits
# ---------------------------------------------------------------------------


def _seen(c):
    """The mean number of positions that a token sees; lengths are spread evenly."""
    n, low, high = c["sequences"], c["shortest"], c["longest"]
    low = high if n == 1 else low
    w = c["window"]
    if w == 0 or w >= high:
        return 0.5 * (low + high)
    if w <= low:
        return float(w)
    return (0.5 * (low + w) * (w - low) + w * (high - w)) / (high - low)


def work(case):
    c = case
    if c["kind"] == "logprobs":
        n = c["rows"]
        return {"bytes": 4.0 * n * c["vocab"] + n * (8.0 * c["given"] + 8.0 * c["top"] + 4.0 * c["entropy"]),
                "flops": 4.0 * n * c["vocab"]}
    row = 2.0 * c["kv_heads"] * _part_bytes(c) / c["page_size"]
    wide = c["kv_heads"] * c["head_dim"]
    if c["kind"] == "append":
        t, back = c["tokens"], c["fmt"] in ("q8_0", "q4_0")
        # read back: the rows again, and as f32
        return {"bytes": t * (8.0 * c["q_heads"] * c["head_dim"] + 8.0 * wide + row + 4.0 * c["head_dim"] + 12.0 +
                              (row + 8.0 * wide if back else 0.0)),
                "flops": 3.0 * t * (c["q_heads"] + c["kv_heads"]) * c["head_dim"]}
    if c["kind"] == "read":
        return {"bytes": c["rows"] * (row + 8.0 * wide + 12.0), "flops": 2.0 * c["rows"] * wide}
    n, seen = c["sequences"], _seen(c)
    return {"bytes": n * (seen * row + 8.0 * c["q_heads"] * c["head_dim"] + 4.0 + 4.0 * math.ceil(seen / c["page_size"])),
            "flops": 4.0 * n * seen * c["q_heads"] * c["head_dim"]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _append_exact, "attend": _attend_exact, "read": _read_exact, "logprobs": _logprobs_exact}[case["kind"]](s)


def _rows64(s, b, positions):
    """Keys and values [KV head, positions, head_dim] of a sequence, number by number from the definition of a page."""
    c = s["case"]
    ps, hd = c["page_size"], c["head_dim"]
    page, row = s["table"][b, positions // ps].long(), positions % ps
    if c["fmt"] in ("f32", "f16"):
        return s["pool"][page, 0, :, row].double().transpose(0, 1), s["pool"][page, 1, :, row].double().transpose(0, 1)
    bits = 8 if c["fmt"] == "q8_0" else 4
    dims = torch.arange(hd, device="cuda")
    out = []
    for plane in range(2):
        place = dims
        if plane:
            blocks, first, place = hd // 32, 0, torch.empty(hd, dtype=torch.long, device="cuda")
            for run in (8, 4, 2, 1):
                if blocks & run:
                    block, i, e = dims // 32 - first, dims % 32 // 2, dims % 2
                    inside = (block >= 0) & (block < run)
                    place = torch.where(inside, 32 * first + i * 2 * run + 2 * block + e, place)
                    first += run
        part = s["pool"][page, plane]  # [position, KV head, bytes]
        byte = row[:, None] * (hd * bits // 8) + place * bits // 8
        code = torch.gather(part, 2, byte[:, None].expand(-1, c["kv_heads"], -1)).long()
        code = torch.where(code > 127, code - 256, code) if bits == 8 else (code >> 4 * (place % 2) & 15) - 8
        half = ps * hd * bits // 8 + 2 * ((row[:, None] // 4 * (hd // 32) + dims // 32) * 4 + row[:, None] % 4)
        pair = torch.stack([torch.gather(part, 2, (half + e)[:, None].expand(-1, c["kv_heads"], -1)) for e in (0, 1)], -1)
        scale = pair.contiguous().view(torch.float16)[..., 0].double()
        out.append((code.double() * scale).transpose(0, 1))
    return out


def _append_exact(s):
    c = s["case"]
    half = c["head_dim"] // 2
    at = s["position"].long()

    def rotated(x):
        x, cos, sin = x.double(), s["cos"][at].double()[:, None], s["sin"][at].double()[:, None]
        turned = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * torch.complex(cos, sin)
        return torch.cat([turned.real, turned.imag], -1)

    if c["fmt"] in ("q8_0", "q4_0"):
        return {"query": rotated(s["query"]), "key": None, "value": None}
    pool = s["pool"].double()
    key = rotated(s["key"])
    where = list(zip(s["sequence"].tolist(), s["position"].tolist()))
    table = s["table"].tolist()
    page = torch.tensor([table[b][p // c["page_size"]] for b, p in where], device="cuda")
    row = torch.tensor([p % c["page_size"] for _, p in where], device="cuda")
    pool[page, 0, :, row] = key
    pool[page, 1, :, row] = s["value"].double()
    return {"query": rotated(s["query"]), "pool": pool}


def _attend_exact(s):
    """Sequence by sequence, head by head: the definition over the positions that the token sees."""
    c = s["case"]
    n, h, kh, hd = c["sequences"], c["q_heads"], c["kv_heads"], c["head_dim"]
    if n * kh > 4096 or work(c)["flops"] > 3e10:
        return None
    out = torch.zeros(n, h, hd, dtype=torch.float64, device="cuda")
    for b, length in enumerate(s["lengths"].tolist()):
        first = max(0, length - c["window"]) if c["window"] else 0
        if length == first:
            continue
        k, v = _rows64(s, b, torch.arange(first, length, device="cuda"))
        for j in range(kh):
            for i in range(j * (h // kh), (j + 1) * (h // kh)):
                p = torch.softmax(torch.mv(k[j], s["q"][b, i].double()) * s["scale"], 0)
                out[b, i] = torch.mv(v[j].t(), p)
    return out


def _read_exact(s):
    c = s["case"]
    key = torch.zeros(c["rows"], c["kv_heads"], c["head_dim"], dtype=torch.float64, device="cuda")
    value = torch.zeros_like(key)
    if c["sequences"] > 4096:
        return {"key": None, "value": None}
    for b in range(c["sequences"]):
        mine = torch.nonzero(s["sequence"] == b)[:, 0]
        if len(mine):
            k, v = _rows64(s, b, s["position"][mine].long())
            key[mine], value[mine] = k.transpose(0, 1), v.transpose(0, 1)
    return {"key": key, "value": value}


def _logprobs_exact(s):
    c = s["case"]
    out = {"logprobs": None, "entropy": None, "ids": None, "tops": None}
    if c["rows"] * c["vocab"] * max(1, c["top"]) > 3e9:
        return None
    x = s["logits"][:, :c["vocab"]]
    y = torch.log_softmax(x.double() / c["temperature"], 1)
    if c["given"]:
        out["logprobs"] = torch.gather(y, 1, s["tokens"].long())
    if c["entropy"]:
        out["entropy"] = -torch.where(y == -math.inf, 0.0, y.exp() * y).sum(1)
    if c["top"]:
        # the largest, of equal ones the first, again and again
        x, ids = x.clone(), []
        at = torch.arange(c["vocab"], device="cuda")
        for _ in range(c["top"]):
            ids.append(torch.where(x == x.amax(1, keepdim=True), at, c["vocab"]).amin(1))
            x.scatter_(1, ids[-1][:, None], -math.inf)
        ids = torch.stack(ids, 1)
        out["ids"], out["tops"] = ids.to(torch.int32), torch.gather(y, 1, ids)
    return out
