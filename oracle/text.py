"""The text decoder's operators in numpy float64, from their definitions (include/ocrhip.h)."""
import numpy as np

QMAX = {"i8": 127.0, "e4m3": 448.0}


def rotate(x, pos, rot, theta, pairs):
    """x [n][heads][dim] with its first rot values rotated by pos [n]."""
    y = x.copy()
    for i in range(rot // 2):
        a, b = (i, i + rot // 2) if pairs == "halves" else (2 * i, 2 * i + 1)
        ang = pos.astype(np.float64)[:, None] * theta ** (-2.0 * i / rot)
        y[..., a] = x[..., a] * np.cos(ang) - x[..., b] * np.sin(ang)
        y[..., b] = x[..., b] * np.cos(ang) + x[..., a] * np.sin(ang)
    return y


def norm(x, w, eps):
    return x if w is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def projections(qkv, q_heads, kv_heads, dim, pos, q_norm, k_norm, eps, rot, theta, pairs):
    """Queries, keys and values of qkv [n][(q_heads + 2 kv_heads) * dim]."""
    x = qkv.astype(np.float64).reshape(len(qkv), q_heads + 2 * kv_heads, dim)
    q, k, v = np.split(x, [q_heads, q_heads + kv_heads], 1)
    return rotate(norm(q, q_norm, eps), pos, rot, theta, pairs), rotate(norm(k, k_norm, eps), pos, rot, theta, pairs), v


def half_step(x, fmt):
    """How far a vector's values (last axis) may be from what an 8-bit cache holds of them: half a
    step of the code, and its scale."""
    scale = np.abs(x).max(-1, keepdims=True) / QMAX[fmt]
    if fmt == "i8":
        return 0.5 * scale + 0 * x
    y = np.abs(x) / np.where(scale > 0, scale, 1)
    return scale * 2.0 ** (np.floor(np.log2(np.maximum(y, 2.0 ** -6))) - 4)


def e4m3_value(code):
    code = np.asarray(code, np.uint8).astype(np.int64)
    sign, exp, man = code >> 7, (code >> 3) & 15, code & 7
    v = np.where(exp == 0, man * 2.0 ** -9, (8 + man) * 2.0 ** (exp.astype(np.float64) - 10))
    return np.where(sign == 1, -v, v)


def key_ranges(n, docs, prefix):
    """[lo, hi) of the keys that every token sees."""
    lo, hi = np.zeros(n, int), np.zeros(n, int)
    docs = [0, n] if docs is None else docs
    for d, (a, b) in enumerate(zip(docs, docs[1:])):
        for i in range(a, b):
            lo[i], hi[i] = a, min(max(i + 1, a + (0 if prefix is None else prefix[d])), b)
    return lo, hi


def weights(s, cap, bias):
    """Softmax of scores s (last axis); scores of minus infinity weigh nothing."""
    if cap:
        s = cap * np.tanh(s / cap)
    s = s + bias
    m = s.max(-1, keepdims=True, initial=-np.inf)
    e = np.exp(s - np.where(m == -np.inf, 0, m))
    t = e.sum(-1, keepdims=True)
    return e / np.where(t > 0, t, 1)


def attention(q, k, v, ranges, scale, cap=0.0, slopes=None, pos=None):
    """(o, sum of p |v|, largest |score|) for q [n][hq][d] over k, v [m][hk][d]: query i sees keys
    ranges[i] and stands at pos[i] (its own row by default)."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    out, size, top = np.zeros_like(q), np.zeros_like(q), 0.0
    g = q.shape[1] // max(1, k.shape[1])
    for i in range(len(q)):
        lo, hi = ranges[0][i], ranges[1][i]
        if hi <= lo:
            continue
        p = i if pos is None else pos[i]
        for h in range(q.shape[1]):
            s = k[lo:hi, h // g] @ q[i, h] * scale
            bias = 0.0 if slopes is None else -float(slopes[h]) * np.abs(p - np.arange(lo, hi))
            w = weights(s, cap, bias)
            vv = v[lo:hi, h // g]
            out[i, h] = w @ np.where(w[:, None] > 0, vv, 0)
            size[i, h] = w @ np.abs(np.where(w[:, None] > 0, vv, 0))
            top = max(top, np.abs(s[np.isfinite(s)]).max(initial=0))
    return out, size, top


def beam_select(logits, scores, finished, eos):
    """(scores, parents, tokens, finished) [groups][beams] after a step."""
    groups, beams = scores.shape
    x = np.asarray(logits, np.float64).reshape(groups, beams, -1)
    vocab = x.shape[2]
    x = np.where(np.isnan(x), -np.inf, x)
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max(-1, keepdims=True)
        rest = np.log(np.exp(x - m).sum(-1, keepdims=True))
        lse = m + rest
        b = lse - m
        lost = (m - (lse - b)) + (rest - b)  # all of rest, where a row's logits are very large
        s = x - lse - lost
    if finished is not None:
        s = np.where(finished[..., None] != 0, np.where(np.arange(vocab) == eos, 0.0, -np.inf), s)
    with np.errstate(invalid="ignore"):
        s = s + scores.astype(np.float64)[..., None]
    s = np.where(np.isfinite(s), s, -np.inf).reshape(groups, -1)
    at = np.argsort(-s, axis=1, kind="stable")[:, :beams]
    parents, tokens = at // vocab, at % vocab
    fin = np.zeros_like(parents) if finished is None else np.take_along_axis(finished, parents, 1)
    return np.take_along_axis(s, at, 1), parents, tokens, ((fin != 0) | (tokens == eos)).astype(np.int32)


def fork(table, lens, parents, spare, page):
    """(table, lens, used, copies): copies [(from page, to page, slots)]."""
    groups, beams = parents.shape
    out, new, used, copies = np.full_like(table, -1), np.zeros_like(lens), np.zeros_like(lens), []
    for g in range(groups):
        seen = set()
        for w in range(beams):
            r, p = g * beams + w, int(parents[g, w])
            if p < 0 or p >= beams:
                continue
            src = g * beams + p
            n = min(max(int(lens[src]), 0), table.shape[1] * page)
            new[r] = n
            full, tail = divmod(n, page)
            out[r, : full + (tail > 0)] = table[src, : full + (tail > 0)]
            if tail and p in seen:
                used[r] = 1
                copies.append((int(table[src, full]), int(spare[r]), tail))
                out[r, full] = spare[r]
            seen.add(p)
    return out, new, used, copies
