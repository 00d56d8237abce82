"""Plain 64-bit forms of the serving operators (test infrastructure only):
attention of single tokens and of chunks over a paged cache, the cache's
bookkeeping, position rotations, residual norms, logit adjustments and token
log probabilities.  numpy, one row at a time.

Each float result comes with `slack`, what 32-bit arithmetic may differ from it
by, from the sizes of the terms (u = 2^-24, a 32-bit rounding); rounding the
result to its type comes on top."""
import numpy as np

U = 2.0 ** -24


def attention(q, k, v, table, lengths, scale, softcap=0.0, window=0, sinks=None, split=0.0):
    """q (B, Hq, D), pools (pages, Hkv, page, D) as float64; (out, slack).
    split: a relative loss of each probability to allow for besides.

    Slack: a score of D products differs by (D + 8) u sum|q k| scale (its
    rounding, the cap and the change of base included); p then by twice the
    largest such difference relative, the sums over n keys by n u.
    """
    B, Hq, D = q.shape
    pages, Hkv, page, _ = k.shape
    out, slack = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), table.shape[1] * page)
        at = np.arange(max(0, n - window) if window else 0, n)
        if not len(at):
            continue
        ids = np.clip(table[b, at // page], 0, pages - 1)
        for h in range(Hq):
            kk, vv = k[ids, h // (Hq // Hkv), at % page], v[ids, h // (Hq // Hkv), at % page]
            s = kk @ q[b, h] * scale
            d = (D + 8) * U * (np.abs(kk) @ np.abs(q[b, h]) * abs(scale)).max()
            if softcap:
                s = softcap * np.tanh(s / softcap)
                d += 8 * U * softcap
            m = s.max() if sinks is None else max(s.max(), sinks[h])
            p = np.exp(s - m)
            total = p.sum() + (0 if sinks is None else np.exp(sinks[h] - m))
            d += 4 * U * np.abs(s).max()
            out[b, h] = p @ vv / total
            slack[b, h] = p @ np.abs(vv) / total * (2 * d + split + (len(at) + 32) * U)
    return out, slack


def pages_of(n, page):
    return -(-n // page)


def reserve(table, lengths, refs, counts, page):
    granted = []
    for r, c in enumerate(counts):
        a, b = pages_of(int(lengths[r]), page), pages_of(int(lengths[r]) + int(c), page)
        free = np.flatnonzero(refs == 0)[:max(b - a, 0)]
        ok = c >= 0 and lengths[r] >= 0 and int(lengths[r]) + int(c) <= table.shape[1] * page and len(free) == b - a
        if ok:
            table[r, a:b] = free
            refs[free] = 1
            lengths[r] += c
        granted.append(int(ok))
    return np.array(granted, np.int32)


def fork(pools, table, lengths, refs, src, dst, page):
    granted, was, seen = [], lengths.copy(), set()
    rows = len(lengths)
    start = [p.copy() for p in pools]
    for a, b in zip(src, dst):
        ok = 0 <= a < rows and 0 <= b < rows and was[b] == 0 and was[a] >= 0 and b not in seen
        seen.add(b)
        if ok:
            full, part = divmod(int(was[a]), page)
            free = np.flatnonzero(refs == 0)[:1]
            ok = not part or len(free) == 1
        if ok:
            for j in range(full):
                table[b, j] = table[a, j]
                refs[table[a, j]] += 1
            if part:
                table[b, full] = free[0]
                refs[free[0]] = 1
                for p, s in zip(pools, start):
                    p[free[0]] = s[table[a, full]]
            lengths[b] = was[a]
        granted.append(int(ok))
    return np.array(granted, np.int32)


def free(table, lengths, refs, rows, page):
    for r in rows:
        if 0 <= r < len(lengths):
            for p in table[r, :pages_of(int(lengths[r]), page)]:
                refs[p] -= 1
            lengths[r] = 0


def compact(pools, table, lengths, refs, page):
    n = int((refs > 0).sum())
    holes, movers = np.flatnonzero(refs[:n] <= 0), n + np.flatnonzero(refs[n:] > 0)
    to = dict(zip(movers.tolist(), holes.tolist()))
    for m, h in to.items():
        refs[h], refs[m] = refs[m], 0
        for p in pools:
            p[h] = p[m]
    for r in range(len(lengths)):
        for j in range(pages_of(int(lengths[r]), page)):
            table[r, j] = to.get(int(table[r, j]), table[r, j])
    return n


def residual_norm(x, y, post=None, gate=None, scale=1.0, pre=None, eps=1e-6, offset=0.0):
    """(h, slack of h, n, slack of n), n None without pre.

    Slack: a sum of H squares, all of one sign, differs by at most H u
    relative and its root by half of that; ten roundings of the other steps.
    """
    H = x.shape[-1]
    c = (H / 2 + 10) * U
    u = y if post is None else y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * (post + offset)
    u = scale * (u if gate is None else u * gate)
    h = x + u
    dh = c * (np.abs(x) + np.abs(u))
    if pre is None:
        return h, dh, None, None
    root = np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    w = np.abs(pre + offset)
    # a change of h by dh: in the row's root by at most the root of its mean square
    dn = (dh + np.abs(h) * np.sqrt((dh * dh).mean(-1, keepdims=True)) / root) / root * w + c * np.abs(h) / root * w
    return h, dh, h / root * (pre + offset), dn


def token_logprobs(x, tokens, k, scale=1.0):
    """x (T, V) float64: (logprobs, entropy, top logprobs, top ids, slack of the
    log probabilities, slack of the entropy).

    Slack: z = scale (x - max) differs by 3 u |z| of itself, exp(z) by that and
    4 u, a sum of V terms by V u / 64 (at most V / 64 of them in one lane, the
    rest in a tree) + 16 u, its logarithm by 2 u more.
    """
    T, V = x.shape
    lp = np.full((T, V), np.nan)
    entropy, dl, de = np.full(T, np.nan), np.zeros(T), np.zeros(T)
    for t in range(T):
        m = x[t].max()
        if m == -np.inf:
            lp[t], entropy[t] = -np.inf, 0.0
            continue
        if not m < np.inf:
            continue
        z = scale * (x[t] - m)
        p = np.exp(z)
        S = p.sum()
        live = p > 0
        lp[t] = z - np.log(S)
        pz = np.where(live, p * np.where(live, z, 0), 0)
        entropy[t] = np.log(S) - pz.sum() / S
        rel = (V / 64 + 20) * U + 3 * U * np.abs(pz).sum() / S
        dl[t] = rel + 2 * U * (1 + np.log(S))
        de[t] = dl[t] + 4 * rel * np.abs(pz).sum() / S + 4 * U * np.abs(pz * np.where(live, z, 0)).sum() / S
    given = np.full(tokens.shape, np.nan)
    for t in range(T):
        for j, tok in enumerate(tokens[t]):
            if 0 <= tok < V:
                given[t, j] = lp[t, tok]
    order = np.where(np.isnan(x), np.inf, x)
    ids = np.lexsort((np.broadcast_to(np.arange(V), x.shape), -order, ~np.isnan(x)), axis=-1)[:, :k]
    return given, entropy, np.take_along_axis(lp, ids, -1), ids, dl, de


def chunk_attention(q, k, v, table, lengths, starts, scale, softcap=0.0, window=0, sinks=None, split=0.0):
    """q (T, Hq, D): (out, slack, which rows belong to a sequence).  Token i of n
    new ones is the last of a sequence of length - n + i + 1 tokens."""
    out, slack, live = np.zeros(q.shape), np.zeros(q.shape), np.zeros(len(q), bool)
    cap = table.shape[1] * k.shape[2]
    for b, length in enumerate(lengths):
        t = np.arange(starts[b], starts[b + 1])
        ends = min(max(int(length), 0), cap) - (starts[b + 1] - t) + 1
        rows = np.repeat(table[b:b + 1], len(t), 0)
        out[t], slack[t] = attention(q[t], k, v, rows, ends, scale, softcap, window, sinks, split)
        live[t] = True
    return out, slack, live


def rotary(x, positions, inv_freq, interleaved=False, factor=1.0):
    """x (T, H, D): (y, slack).

    Slack: an angle of up to 2^20 turns differs by 2^-30 turns (64 bits, two
    roundings); what is left of it, at most pi / 4, is rounded to 32 bits and its
    sine and cosine come from series of five terms: 4 u; the factor, a product and
    the sum round once each."""
    n = len(inv_freq)
    # exact: 31 and 24 bits of a 64-bit significand, then whole turns off
    angle = positions.astype(np.longdouble)[:, None] * inv_freq.astype(np.longdouble)
    turn = 2 * np.longdouble("3.14159265358979323846264338327950288")
    angle = (angle - turn * np.round(angle / turn)).astype(np.float64)[:, None]
    c, s = factor * np.cos(angle), factor * np.sin(angle)
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., first], x[..., second]
    y, slack = x.copy(), np.zeros(x.shape)
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    slack[..., first] = slack[..., second] = 8 * U * abs(factor) * (np.abs(a) + np.abs(b))
    return y, slack


def adjust_logits(x, history=None, history_lengths=None, prompts=None, repetition=None, presence=None, frequency=None,
                  bias_ids=None, bias=None, mask=None):
    """x (T, V) float64: (y, slack, which logits a step changed).  Slack: a rounding of each step."""
    T, V = x.shape
    y, slack, changed = x.copy(), np.zeros(x.shape), np.zeros(x.shape, bool)
    for t in range(T):
        if history is not None:
            n = history.shape[1] if history_lengths is None else min(max(int(history_lengths[t]), 0), history.shape[1])
            p = 0 if prompts is None else int(prompts[t])
            times = {}
            for i, v in enumerate(history[t, :n].tolist()):
                if 0 <= v < V:
                    times[v] = times.get(v, 0) + (i >= p)
            for v, c in times.items():
                changed[t, v] = True
                if repetition is not None:
                    y[t, v] = y[t, v] / repetition[t] if y[t, v] > 0 else y[t, v] * repetition[t]
                    slack[t, v] += U * abs(y[t, v])
                if c:
                    a, b = (0.0 if w is None else w[t] * k for w, k in ((presence, 1), (frequency, c)))
                    y[t, v] -= a + b
                    slack[t, v] += U * (2 * abs(a) + 2 * abs(b) + abs(y[t, v]))
        if bias is not None:
            last = {v: j for j, v in enumerate(bias_ids[t].tolist()) if 0 <= v < V}
            for v, j in last.items():
                changed[t, v] = True
                y[t, v] += bias[t, j]
                slack[t, v] += U * abs(y[t, v])
        if mask is not None:
            bits = (mask[t].astype(np.int64)[:, None] >> np.arange(32)) & 1
            off = bits.reshape(-1)[:V] == 0
            y[t, off], slack[t, off], changed[t, off] = -np.inf, 0, True
    return y, slack, changed
