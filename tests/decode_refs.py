"""Plain float64 / integer restatements of the shared-prompt decode ops, one
row, one position, one token at a time, and the caches they read."""
import numpy as np

f32 = np.float32
NO = 0xFFFFFFFF


def row_bytes(fmt, width):
    return {"f32": 4 * width, "q8_0": width // 32 * 34, "q4_0": width // 32 * 18}[fmt]


def make_cache(r, fmt, positions, width, std=1.0):
    """[2, positions, row] bytes of values of about N(0, std)."""
    if fmt == "f32":
        return (r.standard_normal((2, positions, width)) * std).astype(f32).view(np.uint8).reshape(2, positions, 4 * width)
    size, low, high = {"q8_0": (34, 0.008, 0.016), "q4_0": (18, 0.15, 0.3)}[fmt]
    t = r.integers(0, 256, (2, positions, width // 32, size), dtype=np.uint8)
    d = (r.uniform(low, high, (2, positions, width // 32)) * std).astype(np.float16)
    t[..., :2] = d.view(np.uint8).reshape(2, positions, width // 32, 2)
    return t.reshape(2, positions, -1)


def cache_values(cache, fmt):
    """[..., row] bytes as float64 values."""
    if fmt == "f32":
        return np.ascontiguousarray(cache).view(f32).astype(np.float64)
    size = {"q8_0": 34, "q4_0": 18}[fmt]
    b = cache.reshape(*cache.shape[:-1], cache.shape[-1] // size, size)
    d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    if fmt == "q8_0":
        codes = np.ascontiguousarray(b[..., 2:]).view(np.int8).astype(np.float64)
    else:
        codes = np.concatenate([b[..., 2:] & 15, b[..., 2:] >> 4], -1).astype(np.float64) - 8.0
    return (codes * d).reshape(*cache.shape[:-1], b.shape[-2] * 32)


def attention(q, prefix, prefix_length, cache, lengths, capacity, kv_heads, scale, fmt):
    """(out, weight sums, bound): out [B, T, H, D] float64, the weights that own rows got [B, capacity], and per
    output sum_j p_j |v_j| with the largest sum_i |q_i k_i| * |scale| of the row, from which rounding is bounded."""
    B, T, H, D = q.shape
    G = H // kv_heads
    out, mass = np.zeros(q.shape), np.zeros(q.shape)
    dot = np.zeros((B, T, H))
    got = np.zeros((B, capacity))
    own = {}
    for b in range(B):
        n = min(int(lengths[b]), capacity) if capacity else 0
        if n:
            own[b] = cache_values(cache[:, b * capacity:b * capacity + n], fmt).reshape(2, n, kv_heads, D)
    if prefix_length:
        pk, pv = cache_values(prefix[:, :prefix_length], fmt).reshape(2, prefix_length, kv_heads, D)
    with np.errstate(invalid="ignore", over="ignore"):
        for kh in range(kv_heads):
            rows = q[:, :, kh * G:(kh + 1) * G].astype(np.float64).reshape(B * T * G, D)
            if prefix_length:  # every row sees the prompt
                k, v = np.ascontiguousarray(pk[:, kh]), np.ascontiguousarray(pv[:, kh])
                x = rows @ k.T * scale
                dots = (np.abs(rows) @ np.abs(k).T).max(1) * abs(scale)
            for i, row in enumerate(rows):
                b, t, h = i // (T * G), i // G % T, kh * G + i % G
                n = own[b].shape[1] if b in own else 0
                see = max(0, n - (T - 1 - t))
                if not see and not prefix_length:
                    continue
                xs = [x[i]] if prefix_length else []
                if see:
                    ok, ov = own[b][0, :see, kh], own[b][1, :see, kh]
                    xs.append(ok @ row * scale)
                    dot[b, t, h] = (np.abs(ok) @ np.abs(row)).max() * abs(scale)
                if prefix_length:
                    dot[b, t, h] = max(dot[b, t, h], dots[i])
                p = np.concatenate(xs)
                p = np.exp(p - p.max())
                p /= p.sum()
                if prefix_length:
                    x[i] = p[:prefix_length]
                if see:
                    mine = p[prefix_length:]
                    out[b, t, h], mass[b, t, h] = mine @ ov, mine @ np.abs(ov)
                    got[b, :see] += mine
            if prefix_length:
                out[:, :, kh * G:(kh + 1) * G] += (x @ v).reshape(B, T, G, D)
                mass[:, :, kh * G:(kh + 1) * G] += (x @ np.abs(v)).reshape(B, T, G, D)
    return out, got, (mass, dot)


def evict(cache, weights, lengths, capacity, budget, recent, cache_out, weights_out):
    """(cache, weights, lengths, kept); cache [2, B*capacity, row], the outputs' first contents given."""
    B = len(lengths)
    out, w_out = cache_out.copy(), weights_out.copy()
    n_out = np.zeros(B, np.uint32)
    kept = np.full((B, budget), NO, np.uint32)
    for b in range(B):
        n = min(int(lengths[b]), capacity)
        if n <= budget:
            stay = list(range(n))
        else:
            old = n - recent

            def rank(i):
                w = weights[b, i]
                return (-np.inf, 1) if np.isnan(w) else (float(w), 2)
            heavy = sorted(range(old), key=lambda i: (-rank(i)[0], -rank(i)[1], i))[:budget - recent]
            stay = sorted(heavy) + list(range(old, n))
        for i, j in enumerate(stay):
            out[:, b * capacity + i] = cache[:, b * capacity + j]
            w_out[b, i] = weights[b, j]
            kept[b, i] = j
        n_out[b] = len(stay)
    return out, w_out, n_out, kept


def _distribution(logits, inv):
    x = logits.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return np.zeros(len(x))
    e = np.where(x == top, 1.0, 0.0)
    rest = x != top
    if np.isfinite(top):
        e[rest] = np.exp((x[rest] - top) * inv)
    return e / e.sum()


def verify(target, draft, tokens, lengths, accept, sample, inv):
    """(accepted, tokens, distance): distance is how far, relative to the sum, each sequence's decisions were from
    falling the other way (a test refuses inputs that lie on a border by chance)."""
    B, T1, V = target.shape
    T = T1 - 1
    accepted, out = np.zeros(B, np.uint32), np.full((B, T1), NO, np.uint32)
    near = np.full(B, np.inf)
    for b in range(B):
        rest, n = None, min(int(lengths[b]), T) if lengths is not None else T
        for t in range(n):
            p, x = _distribution(target[b, t], inv), int(tokens[b, t])
            if draft is None:
                q = np.zeros(V)
                if x < V:
                    q[x] = 1.0
                qx = 1.0
            else:
                q = _distribution(draft[b, t], inv)
                qx = q[x] if x < V else 0.0
            px = p[x] if x < V else 0.0
            u = float(accept[b, t])
            if px > 0 and u > 0:
                near[b] = min(near[b], abs(u * qx - px) / px)
            if not u * qx < px:
                rest = np.maximum(p - q, 0.0)
                rest = rest if rest.sum() > 0 else p
                break
            out[b, t] = x
            accepted[b] += 1
        if rest is None:
            rest = _distribution(target[b, n], inv)
        total = np.cumsum(rest)
        if total[-1] > 0:
            goal = float(sample[b]) * total[-1]
            i = int(np.searchsorted(total, goal, side="right"))
            out[b, accepted[b]] = i
            if sample[b] > 0:
                near[b] = min(near[b], np.abs(total - goal).min() / total[-1])
    return accepted, out, near
