"""Plain statements, in numpy and 64 bits, of the serving operators: pages and slots, 4-bit rows, attention over them, beam selection and
reordering.  (Test infrastructure; the reference has no counterpart.)"""
import numpy as np


def pages(have, want, page, table, free, n_free, max_tokens):
    """(table, free, state, starts, slots) behind ``caten_b200_kv_pages``."""
    table, free, have, want = table.copy(), free.copy(), [int(x) for x in have], [int(x) for x in want]
    n, columns = table.shape
    count = lambda t: -(-t // page)   # noqa: E731
    refused = lambda missing, why: (table, free, np.array([n_free, 0, missing, why]), np.zeros(n + 1, np.int64), np.full(max_tokens, -1))   # noqa: E731
    if any(h < 0 or w < 0 or count(h) > columns or count(w) > columns for h, w in zip(have, want)):
        return refused(0, 1)
    more = [max(0, w - h) for h, w in zip(have, want)]
    gives = sum(max(0, count(h) - count(w)) for h, w in zip(have, want))
    takes = sum(max(0, count(w) - count(h)) for h, w in zip(have, want))
    if sum(more) > max_tokens:
        return refused(0, 2)
    if n_free < 0 or n_free + gives > len(free):
        return refused(0, 3)
    if takes > n_free + gives:
        return refused(takes - n_free - gives, 0)
    for r in range(n):
        for j in range(count(want[r]), count(have[r])):
            free[n_free], table[r, j] = table[r, j], -1
            n_free += 1
    slots, starts = [], [0]
    for r in range(n):
        for j in range(count(have[r]), count(want[r])):
            n_free -= 1
            table[r, j] = free[n_free]
        slots += [table[r, t // page] * page + t % page for t in range(have[r], want[r])]
        starts.append(len(slots))
    return table, free, np.array([n_free, len(slots), 0, 0]), np.array(starts), np.array(slots + [-1] * (max_tokens - len(slots)))


def blocks(x, q4_1):
    """x [..., 32] fp32 -> (codes, scale fp16, minimum fp16 or None)."""
    x = x.astype(np.float64)
    with np.errstate(all="ignore"):
        if q4_1:
            low = x.min(-1, keepdims=True)
            d = (x.max(-1, keepdims=True) - low) / 15
            code = np.trunc((x - low) / d + 0.5)
        else:
            low, d = None, np.take_along_axis(x, np.abs(x).argmax(-1, keepdims=True), -1) / -8
            code = np.trunc(x / d + 8.5)
        stored = d.astype(np.float32).astype(np.float16)
        code = np.where(stored == 0, 0 if q4_1 else 8, np.nan_to_num(code, nan=0.0).clip(0, 15)).astype(np.uint8)
        return code, stored, low.astype(np.float32).astype(np.float16) if q4_1 else None


def values(x, q4_1):
    """The fp32 values that rows [..., n * 32] have once they are stored."""
    code, d, m = blocks(x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32), q4_1)
    d = d.astype(np.float32)
    y = d * code.astype(np.float32) + m.astype(np.float32) if q4_1 else d * (code.astype(np.float32) - np.float32(8))
    return y.reshape(x.shape)


def put(pool, page, kv_heads, dim, q4_1, slot, head, k, v):
    """Writes one token's key and value of a head into a pool [pages, bytes], byte by byte as the layout is stated."""
    part = (10 if q4_1 else 9) * dim
    for x, of_k in ((k, True), (v, False)):
        code, d, m = blocks(x.reshape(-1, 32), q4_1)
        t = slot % page % 16
        base = (head * (page // 16) + slot % page // 16) * 2 * part + (0 if of_k else part)
        row = pool[slot // page]
        for b in range(dim // 32):
            for j in range(32):
                lane, word, nibble = ((t % 8 * 4 + j // 8, t // 8 * 2 + b % 2, j % 8) if of_k else
                                      (j // 4 * 4 + t % 8 // 2, t // 8 * 2 + t % 2, b % 2 * 4 + j % 4))
                at = base + b // 2 * 512 + lane * 16 + word * 4 + nibble // 2
                keep = 0x0f if nibble % 2 else 0xf0
                row[at] = row[at] & keep | int(code[b, j]) << nibble % 2 * 4
            place = base + 8 * dim + 2 * ((t % 8 // 2 * (dim // 32) + b) * 4 + t // 8 * 2 + t % 2)
            row[place:place + 2] = np.frombuffer(d[b].tobytes(), np.uint8)
            if q4_1:
                row[place + dim:place + dim + 2] = np.frombuffer(m[b].tobytes(), np.uint8)


def attention(q, k, v, length, scale):
    """q [rows, heads, dim] of the last rows of a sequence, k and v [tokens, kv_heads, dim] -> [rows, heads, dim] in 64 bits."""
    rows, heads, _ = q.shape
    group = heads // k.shape[1]
    out = np.zeros(q.shape)
    for i in range(rows):
        sees = max(0, length - rows + i + 1)
        for h in range(heads if sees else 0):
            s = k[:sees, h // group].astype(np.float64) @ q[i, h].astype(np.float64) * scale
            p = np.exp(s - s.max())
            out[i, h] = p @ v[:sees, h // group].astype(np.float64) / p.sum()
    return out


def select(logits, scores, ended, eos, keep):
    """(scores, parents, tokens, ended) of one request: logits [beams, V], scores [beams], ended [beams]."""
    beams, V = logits.shape
    x = logits.astype(np.float64)
    with np.errstate(all="ignore"):
        top = x.max(1, keepdims=True)
        value = scores.astype(np.float64)[:, None] + ((x - top) - np.log(np.exp(x - top).sum(1, keepdims=True)))   # (top + log would lose the log beside a top of -3e38)
    for b in range(beams):
        if ended[b]:
            value[b] = -np.inf
            value[b, eos] = scores[b]
    value = np.where(np.isnan(value), -np.inf, value).reshape(-1)
    x, order = x.reshape(-1), np.argsort(-value, kind="stable")
    last = value[order[min(keep, len(order)) - 1]]
    order = np.flatnonzero(value >= last)   # where values of a beam coincide in 64 bits, its logits say which is larger
    order = order[np.lexsort((order, -x[order], order // V, -value[order]))][:keep]
    order = [i for i in order if value[i] > -np.inf]
    parents = [i // V for i in order] + [min(i, beams - 1) for i in range(len(order), keep)]
    tokens = [i % V for i in order] + [max(eos, 0)] * (keep - len(order))
    with np.errstate(over="ignore"):
        found = np.array([value[i] for i in order] + [-np.inf] * (keep - len(order))).astype(np.float32)
    return found, np.array(parents), np.array(tokens), np.array([bool(ended[p]) or (eos >= 0 and t == eos) for p, t in zip(parents, tokens)])


def parts(x, q4_1):
    """|d (code - 8)| + |minimum + 8 d| (Q4_1) of the values that rows [.., n * 32] are stored as: what the kernels add up in the place of a value."""
    code, d, m = blocks(x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32), q4_1)
    d = np.abs(d.astype(np.float64)) if not q4_1 else d.astype(np.float64)
    y = d * np.abs(code.astype(np.float64) - 8)
    return (y + np.abs(m.astype(np.float64) + 8 * d) if q4_1 else y).reshape(x.shape)


def attention_bound(q, k, k_parts, v_parts, length, scale):
    """How far the kernels' answers for these rows may be off, [rows, heads, dim], in roundings of u = 2^-23 (sums of tensor cores may be cut off instead of
    rounded: a whole step).

    A score's terms, of magnitude a = scale sum |q| parts(k): q in two halves 2 u, sums of 16 and their halves and blocks 8 + 10 / 2, factors 2: 20 u a
    with room.  A probability is off by that and, relatively, by its power of two (2 u) and up to ten corrections when a larger score is met (2.5 u
    each): 30 u.  It counts twice, in the outputs' sum and in the probabilities'.  Outputs add p times parts(v) in a block of 32 dims: halves of p d
    2 u, sums of 16 and their halves 8 u, groups of 32 tokens at least u / 2 each, in both sums; what is left for joining parts: 20 u."""
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    out = np.zeros(q.shape)
    for i in range(rows):
        sees = max(0, length - rows + i + 1)
        for h in range(heads if sees else 0):
            x = q[i, h].astype(np.float64)
            s = k[:sees, h // group].astype(np.float64) @ x * scale
            a = k_parts[:sees, h // group] @ np.abs(x) * abs(scale)
            p = np.exp(s - s.max())
            p /= p.sum()
            block = (p @ v_parts[:sees, h // group].reshape(sees, dim // 32, 32).max(2))
            # (a token's own a counts as much as its probability; the normalising sum's is the mean)
            mine = (p * (40 * a)) @ v_parts[:sees, h // group].reshape(sees, dim // 32, 32).max(2) / 2 + block * (p @ (40 * a)) / 2
            out[i, h] = np.repeat((mine + (90 + sees / 32) * block) * 2.0 ** -23, 32)
    return out


def few_tokens(rng, length, kv, dim, heads, news, scale):
    """(k, v, q) [tokens, kv, dim] and [news, heads, dim] of a sequence in which a dozen tokens have nearly all of every row's probability, each a share that
    counts: the first, those on both sides of borders of 64 tokens and of halves, and the last ones, of which each row sees one more than the row before.
    Values of q lie next to the middle between two of 16 bits, each block of 32 dims of v has one of the tokens stand out."""
    marks = {0, 15, 16, 63, 64, length // 2 - 1, length // 2, length // 64 * 64 - 1, length // 64 * 64} | set(range(length - news, length))
    marks = np.array(sorted(t for t in marks if 0 <= t < length))
    way, even = rng.choice([-1.0, 1.0], (kv, dim)), np.arange(dim) % 2 == 0
    # rounded to 16 bits, the even dims of q lose twice as much of themselves as the odd ones, and half of the tokens are turned to either
    size = (np.where(even, 1.02, 1.92) * rng.uniform(1.0, 1.01, (news, heads, dim))).astype(np.float16)
    size = size.astype(np.float64) + 0.49 * np.spacing(size).astype(np.float64)
    to_even, to_odd = np.where(even, 1.0, 0.125), np.where(even, 0.125, 0.56)
    turned = np.where((np.arange(len(marks)) % 2 == 0)[:, None, None], to_even, to_odd) * rng.uniform(0.97, 1.0, (len(marks), 1, 1))
    k = rng.standard_normal((length, kv, dim)) * 0.1
    k[marks] = way * turned
    k *= (np.log(length) + 4) / (abs(scale) * dim * 0.63)
    q = np.repeat(way[None], news, 0).repeat(heads // kv, 1) * size
    v = rng.standard_normal((length, kv, dim // 32, 32)) * 0.05
    for h in range(kv):
        for b in range(dim // 32):
            v[marks[-1 - (h * (dim // 32) + b) % len(marks)], h, b] *= 20
    return k.astype(np.float32), v.reshape(length, kv, dim).astype(np.float32), q.astype(np.float32)
