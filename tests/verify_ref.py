"""Draft verification stated in binary64 numpy, one sequence and one test at a time: the
definition the device results are held to (see rsc_verify in the C header)."""

import numpy as np


def scaled(x: np.ndarray, temperature: float) -> np.ndarray:
    """The sampler's scaled logits: NaN -> -inf, then one binary32 product with 1/T."""
    s = np.float32(1.0) / np.float32(temperature) if temperature > 0 else np.float32(1.0)
    x = np.where(np.isnan(x), np.float32(-np.inf), x).astype(np.float32)
    with np.errstate(over="ignore"):
        return (x * s).astype(np.float32)


def softmax(v: np.ndarray):
    """Binary64 softmax, or None where the row has no distribution."""
    m = v.max()
    if not np.isfinite(m):
        return None
    e = np.exp(v.astype(np.float64) - float(m))
    return e / e.sum()


def draw(w: np.ndarray, u: float) -> int:
    """First index whose running weight exceeds u times the sum, else the last of weight; -1
    without any weight."""
    c = np.cumsum(w)
    if not c[-1] > 0:
        return -1
    hit = np.nonzero(c > u * c[-1])[0]
    return int(hit[0]) if len(hit) else int(np.nonzero(w > 0)[0][-1])


def verify_one(p_rows, q_rows, tokens, n, u_tests, u_last):
    """p_rows(i), q_rows(i): distributions (q_rows None: one-hot drafts), arrays over the
    vocabulary or None. Returns (tokens, accepted, status, draws)."""
    for a in range(n + 1):
        p = p_rows(a)
        q = q_rows(a) if q_rows is not None and a < n else None
        if p is None or (a < n and q_rows is not None and q is None):
            return list(tokens[:a]), a, 1, a
        w = p
        if a < n:
            t = int(tokens[a])
            inside = 0 <= t < len(p)
            pt = p[t] if inside else 0.0
            qt = 1.0 if q is None else (q[t] if inside else 0.0)
            if float(u_tests[a]) * qt < pt:
                continue
            if q is None:
                w = p.copy()
                if inside:
                    w[t] = 0.0
            else:
                w = np.maximum(p - q, 0.0)
        last = draw(w, float(u_last(a + (a < n))))
        if last < 0:
            last = draw(p, float(u_last(a + (a < n))))
        return list(tokens[:a]) + [last], a, 0, a + (a < n) + 1
    raise AssertionError


def verify_batch(target, draft, tokens, n_draft, uniforms, temperature):
    """Arrays as rsc_verify takes them; returns (tokens, accepted, status) arrays."""
    b, d = tokens.shape
    out = np.full((b, d + 1), -1, np.int32)
    acc, st = np.zeros(b, np.int32), np.zeros(b, np.int32)
    for i in range(b):
        n = d if n_draft is None else int(np.clip(n_draft[i], 0, d))
        row, acc[i], st[i], _ = verify_one(
            lambda k: softmax(scaled(target[i, k], temperature)),
            None if draft is None else lambda k: softmax(scaled(draft[i, k], temperature)),
            tokens[i], n, uniforms[i], lambda k: uniforms[i, d])
        out[i, :len(row)] = row
    return out, acc, st


def verify_records(target, draft, vocab, tokens, n_draft, uniforms):
    """Records (n, ids, probs) of b * (d + 1) and b * d rows, as arrays."""
    b, d = tokens.shape

    def dense(rec, row):
        n, ids, probs = rec[:3]
        if n[row] == 0:
            return None
        p = np.zeros(vocab, np.float64)
        p[ids[row, :n[row]]] = probs[row, :n[row]]
        return p

    out = np.full((b, d + 1), -1, np.int32)
    acc, st = np.zeros(b, np.int32), np.zeros(b, np.int32)
    for i in range(b):
        n = d if n_draft is None else int(np.clip(n_draft[i], 0, d))
        row, acc[i], st[i], _ = verify_one(
            lambda k: dense(target, i * (d + 1) + k),
            None if draft is None else lambda k: dense(draft, i * d + k),
            tokens[i], n, uniforms[i], lambda k: uniforms[i, d])
        out[i, :len(row)] = row
    return out, acc, st


def greedy_batch(target, tokens, n_draft):
    b, d = tokens.shape
    out = np.full((b, d + 1), -1, np.int32)
    acc, st = np.zeros(b, np.int32), np.zeros(b, np.int32)
    for i in range(b):
        n = d if n_draft is None else int(np.clip(n_draft[i], 0, d))
        for a in range(n + 1):
            x = target[i, a]
            acc[i] = a
            if not np.isfinite(x).any():
                st[i] = 1
                break
            # f32::total_cmp, as rsc_greedy: -0 orders below +0.
            bits = np.where(np.isnan(x), np.float32(-np.inf), x).view(np.int32).astype(np.int64)
            key = np.where(bits < 0, -1 - (bits & 0x7fffffff), bits)
            best = int(np.nonzero(key == key.max())[0][-1])
            out[i, a] = best
            if a == n or tokens[i, a] != best:
                break
    return out, acc, st


_MASK = (1 << 64) - 1


def wyrand_uniforms(state: int, k: int):
    """The next k uniforms of a generator state (rsc_rng_seed) as binary32."""
    out = []
    for _ in range(k):
        state = (state + 0x2d358dccaa6c78a5) & _MASK
        x = state * (state ^ 0x8bb84b93962eacc9)
        bits = 0x3f800000 | ((((x >> 64) ^ x) & 0xffffffff) >> 9)
        out.append(np.array([bits], np.uint32).view(np.float32)[0] - np.float32(1.0))
    return out
