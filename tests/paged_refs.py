"""Plain restatements of the paged decode ops: pages written and read number by
number as their layout is described, attention and log probabilities in float64."""
import numpy as np

f32 = np.float32
NO = 0xFFFFFFFF


def code_bytes(fmt, D):
    return {"f32": 4 * D, "f16": 2 * D, "q8_0": D, "q4_0": D // 2}[fmt]


def part_bytes(fmt, ps, D):
    return ps * (code_bytes(fmt, D) + (D // 32 * 2 if fmt in ("q8_0", "q4_0") else 0))


def value_order(D):
    """The dims of a value's codes, in their order."""
    blocks, first, dims = D // 32, 0, []
    for run in (8, 4, 2, 1):
        if blocks & run:
            dims += [32 * (first + j) + 2 * i + e for i in range(16) for j in range(run) for e in (0, 1)]
            first += run
    return np.array(dims)


def rotate(x, cos, sin):
    """[.., D] by [.., D / 2] angles, each product and sum rounded to f32."""
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return np.concatenate([a * cos - b * sin, a * sin + b * cos], -1).astype(f32)


def encode(x, fmt):
    """Codes [.., D] (Q4_0: 0 .. 15) and f16 scales [.., D / 32] of f32 rows, step by step in f32."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    size = np.abs(b)
    top = np.where(np.isnan(size), 0, size).max(-1, keepdims=True)
    if fmt == "q8_0":
        scale = top / f32(127)
        with np.errstate(all="ignore"):
            y = np.clip(b / scale, f32(-127), f32(127))
            y = np.where(np.isnan(y), f32(-127), y).astype(np.float64)
        codes = np.sign(y) * np.floor(np.abs(y) + 0.5)
        codes = np.where(scale == 0, 0, codes).astype(np.int8).view(np.uint8)
    else:
        first = (size == top).argmax(-1)[..., None]
        scale = np.where(top == 0, f32(0), np.take_along_axis(b, first, -1) / f32(-8))
        with np.errstate(all="ignore"):
            y = b / scale + f32(8.5)
        y = np.where(np.isnan(y), 0, np.clip(y, 0, 15))
        codes = np.where(scale == 0, 0, np.floor(y)).astype(np.uint8)
    with np.errstate(over="ignore"):
        return codes.reshape(x.shape), scale[..., 0].astype(np.float16)


class Pool:
    """Bytes of a pool, [page, plane, head, part]."""

    def __init__(self, fmt, pages, ps, KH, D, fill=0):
        self.fmt, self.ps, self.KH, self.D = fmt, ps, KH, D
        self.bytes = np.full((pages, 2, KH, part_bytes(fmt, ps, D)), fill, np.uint8)

    def random(self, r, std=1.0):
        n, D, ps = self.bytes.shape[0], self.D, self.ps
        if self.fmt in ("f32", "f16"):
            x = (r.standard_normal((n, 2, self.KH, ps, D)) * std).astype(f32 if self.fmt == "f32" else np.float16)
            self.bytes = x.view(np.uint8).reshape(self.bytes.shape)
        else:
            self.bytes = r.integers(0, 256, self.bytes.shape, dtype=np.uint8)
            low, high = {"q8_0": (0.008, 0.016), "q4_0": (0.15, 0.3)}[self.fmt]
            d = (r.uniform(low, high, (n, 2, self.KH, ps * D // 32)) * std).astype(np.float16)
            self.bytes[..., ps * code_bytes(self.fmt, D):] = d.view(np.uint8).reshape(n, 2, self.KH, -1)
        return self

    def _spots(self, row):
        cb = code_bytes(self.fmt, self.D)
        nb = self.D // 32
        return slice(row * cb, (row + 1) * cb), [self.ps * cb + 2 * ((row // 4 * nb + b) * 4 + row % 4) for b in range(nb)]

    def write(self, page, plane, head, row, x):
        """One head's f32 row."""
        part = self.bytes[page, plane, head]
        at, scales = self._spots(row)
        if self.fmt == "f32":
            part[at] = x.astype(f32).view(np.uint8)
        elif self.fmt == "f16":
            with np.errstate(over="ignore"):
                part[at] = x.astype(np.float16).view(np.uint8)
        else:
            codes, d = encode(x, self.fmt)
            if plane:
                codes = codes[value_order(self.D)]
            part[at] = codes if self.fmt == "q8_0" else codes[::2] | codes[1::2] << 4
            for s, v in zip(scales, d):
                part[s:s + 2] = np.frombuffer(v.tobytes(), np.uint8)

    def values(self, page, plane, head):
        """The part's rows as float64 [ps, D]."""
        part, ps, D = self.bytes[page, plane, head], self.ps, self.D
        if self.fmt in ("f32", "f16"):
            return part.view(f32 if self.fmt == "f32" else np.float16).reshape(ps, D).astype(np.float64)
        cb = code_bytes(self.fmt, D)
        codes = part[:ps * cb].reshape(ps, cb)
        codes = codes.view(np.int8).astype(np.float64) if self.fmt == "q8_0" else \
            np.stack([codes & 15, codes >> 4], -1).reshape(ps, D).astype(np.float64) - 8.0
        if plane:
            back = np.empty_like(codes)
            back[:, value_order(D)] = codes
            codes = back
        d = part[ps * cb:].copy().view(np.float16).astype(np.float64).reshape(ps // 4, D // 32, 4)
        d = d.transpose(0, 2, 1).reshape(ps, D // 32)
        with np.errstate(invalid="ignore"):
            return codes * np.repeat(d, 32, 1)


def append(pool, table, key, value, query, query_out, cos, sin, ids, positions):
    """The pool and query_out changed in place; cos, sin [positions, D / 2] or None."""
    count = pool.bytes.shape[0]
    for t, p in enumerate(positions):
        b = t if ids is None else int(ids[t])
        p = int(p)
        if b >= table.shape[0] or p // pool.ps >= table.shape[1]:
            continue
        turn = (lambda x: x) if cos is None else (lambda x: rotate(x, cos[p], sin[p]))  # noqa: B023
        if query is not None:
            query_out[t] = turn(query[t])
        page = int(table[b, p // pool.ps])
        if page >= count:
            continue
        k = turn(key[t])
        for h in range(pool.KH):
            pool.write(page, 0, h, p % pool.ps, k[h])
            pool.write(page, 1, h, p % pool.ps, value[t, h])


def rows(pool, table, b, head, lo, hi):
    """(keys, values, there) of positions lo .. hi - 1 of a sequence's KV head, in float64."""
    k, v = np.zeros((hi - lo, pool.D)), np.zeros((hi - lo, pool.D))
    there = np.zeros(hi - lo, bool)
    for e in range(lo // pool.ps, (hi + pool.ps - 1) // pool.ps):
        page = int(table[b, e])
        if page >= pool.bytes.shape[0]:
            continue
        a, z = max(lo, e * pool.ps), min(hi, (e + 1) * pool.ps)
        inside = slice(a - e * pool.ps, z - e * pool.ps)
        k[a - lo:z - lo], v[a - lo:z - lo] = pool.values(page, 0, head)[inside], pool.values(page, 1, head)[inside]
        there[a - lo:z - lo] = True
    return k, v, there


def attention(pool, table, q, lengths, window, scale):
    """(out, mass, dot): out [B, H, D] float64, sum_j p_j |v_j|, and each row's largest |scale| sum_i |q_i k_i|."""
    B, H, D = q.shape
    G = H // pool.KH
    cap = table.shape[1] * pool.ps
    out, mass, dot = np.zeros(q.shape), np.zeros(q.shape), np.zeros((B, H))
    for b in range(B):
        n = min(int(lengths[b]), cap)
        lo = n - window if window and n > window else 0
        for kh in range(pool.KH):
            if n == lo:
                continue
            k, v, there = rows(pool, table, b, kh, lo, n)
            k, v = k[there], v[there]
            if not len(k):
                continue
            mine = slice(kh * G, (kh + 1) * G)
            with np.errstate(invalid="ignore", over="ignore"):
                x = q[b, mine].astype(np.float64) @ k.T * scale
                dot[b, mine] = (np.abs(q[b, mine].astype(np.float64)) @ np.abs(k).T).max(1) * abs(scale)
                p = np.exp(x - x.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                out[b, mine], mass[b, mine] = p @ v, p @ np.abs(v)
    return out, mass, dot


def logprobs(logits, tokens, inv, top):
    """(logprobs, entropy, top ids, top logprobs) of rows of f32 logits, in float64."""
    R = logits.shape[0]
    given = np.full(tokens.shape, -np.inf)
    entropy, ids, tops = np.zeros(R), np.full((R, top), NO, np.uint32), np.full((R, top), -np.inf)
    for r in range(R):
        x = logits[r].astype(np.float64)
        x = np.where(np.isnan(x), -np.inf, x)
        order = np.lexsort((np.arange(len(x)), -x))
        order = order[x[order] > -np.inf][:top]
        best = x.max()
        y = np.full(len(x), -np.inf)
        if best == np.inf:
            y[x == np.inf] = -np.log((x == np.inf).sum())
        elif best > -np.inf:
            y = (x - best) * inv
            rest = np.exp(np.where(x == best, -np.inf, y)).sum()
            y = y - (np.log((x == best).sum()) + np.log1p(rest / (x == best).sum()))
        ids[r, :len(order)], tops[r, :len(order)] = order, y[order]
        for g, t in enumerate(tokens[r]):
            if t < len(x):
                given[r, g] = y[t]
        some = y > -np.inf
        entropy[r] = -(np.exp(y[some]) * y[some]).sum()
    return given, entropy, ids, tops


def attention_bound(fmt, pool, table, q, lengths, window, scale, exp):
    """Elementwise bound of |got - exp|; exp as attention() gives it.

    A score: D f32 products, each operand rounded once (q * scale) and once more as pieces (2^-24, or 2^-39 of the
    row's largest for f16 ones), summed in f32, a block's scale on its sum, and x - max: within (D + 24) 2^-24 dot, and
    for f16 pieces 2^-38 |scale| max|q| sum|k| besides.  A weight changes by e^dx, a quotient of weights by e^(2 dx).
    Weights: exp2 and pieces, 2^-22; f16 pieces besides 2^-40 of the largest weight, 1, times sum |v| / sum p <=
    sum |v|.  Sums: 32 products in a step, at most 256 additions of steps and as many changes of the maximum, 32
    roundings in the joins; never more than twice the keys."""
    out, mass, dot = exp
    B, H, D = q.shape
    G, cap = H // pool.KH, table.shape[1] * pool.ps
    tol = np.zeros(q.shape)
    for b in range(B):
        n = min(int(lengths[b]), cap)
        lo = n - window if window and n > window else 0
        for kh in range(pool.KH):
            mine = slice(kh * G, (kh + 1) * G)
            k, v, there = rows(pool, table, b, kh, lo, n)
            dx = (D + 24) * 2.0 ** -24 * dot[b, mine]
            floor = 0.0
            if fmt != "f32" and there.any():
                top = np.abs(q[b, mine].astype(np.float64)).max(1)
                dx = dx + 2.0 ** -38 * abs(scale) * top * np.abs(k[there]).sum(1).max()
            if fmt == "f16":
                floor = 2.0 ** -40 * np.abs(v[there]).sum(0)
            keys = int(there.sum())
            rel = np.expm1(2 * dx)[:, None] + 2.0 ** -22 + (min(2 * keys, 544) + 32) * 2.0 ** -24
            tol[b, mine] = rel * mass[b, mine] + floor
    return tol + 1e-37
