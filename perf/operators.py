"""Operators of a serving loop, as cases to be timed and compared: page tables and slots from request lengths, rows stored into a
4-bit cache and read back, attention over that cache, beam search's selection, and the reordering of states behind it.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what a program has in hand before the
call, ``run`` is one pass (``own`` False: elementary torch operations in 32 bits, 64 where a border or an order hangs on it; True:
the package's entry points), ``exact`` the same from the definitions in 64 bits, ``work`` the bytes and operations of a pass."""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"q4_0": 2, "q4_1": 3}   # ggml ids
_kept = {}


def listed():
    return [
        # a decode step of an ordinary batch: every request grows by a token, few take a page
        {"name": "pages-step-64", "kind": "pages", "requests": 64, "page": 64, "longest": 1000, "what": "step"},
        # a busy server's turn: prompts arrive, requests go on, others end or give tokens back
        {"name": "pages-mixed-1000", "kind": "pages", "requests": 1000, "page": 16, "longest": 1024, "what": "mixed"},
        # the keys and values of such a step, heads of GPT-2 XL
        {"name": "store-q4_0-64x25x64", "kind": "store", "tokens": 64, "heads": 25, "kv_heads": 25, "dim": 64, "type": "q4_0", "page": 64},
        # those of prompts, grouped heads
        {"name": "store-q4_1-8191x4x128", "kind": "store", "tokens": 8191, "heads": 16, "kv_heads": 4, "dim": 128, "type": "q4_1", "page": 32},
        # one interactive user of the largest model: latency is all
        {"name": "attention-q4_0-h25-1x700", "kind": "attention", "batch": 1, "heads": 25, "kv_heads": 25, "dim": 64, "type": "q4_0", "page": 64,
         "longest": 700, "ragged": False, "new": 1},
        # the largest batch
        {"name": "attention-q4_0-h25-256x768", "kind": "attention", "batch": 256, "heads": 25, "kv_heads": 25, "dim": 64, "type": "q4_0", "page": 64,
         "longest": 768, "ragged": False, "new": 1},
        # a few very long documents, grouped heads
        {"name": "attention-q4_1-h32g4-3x100001", "kind": "attention", "batch": 3, "heads": 32, "kv_heads": 8, "dim": 128, "type": "q4_1", "page": 128,
         "longest": 100001, "ragged": True, "new": 1},
        # portions of prompts behind a history
        {"name": "attention-q4_0-h16g4-5x333", "kind": "attention", "batch": 5, "heads": 16, "kv_heads": 4, "dim": 128, "type": "q4_0", "page": 32,
         "longest": 1200, "ragged": True, "new": 333},
        # one user's beams
        {"name": "select-1x4", "kind": "select", "batch": 1, "beams": 4, "vocab": 50257, "keep": 4, "ended": False},
        # a server's, with candidates to spare and hypotheses that have ended
        {"name": "select-64x8", "kind": "select", "batch": 64, "beams": 8, "vocab": 50257, "keep": 16, "ended": True},
        # the caches of GPT-2 medium behind a step of 16 requests' beams
        {"name": "reorder-medium-16x4", "kind": "reorder", "layers": 24, "batch": 16, "beams": 4, "heads": 16, "positions": 333, "capacity": 512},
        # a paged 4-bit cache behind the same
        {"name": "reorder-paged-16x8", "kind": "reorder_paged", "batch": 16, "beams": 8, "kv_heads": 8, "dim": 128, "type": "q4_1", "page": 64, "positions": 1500},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["pages", "store", "attention", "attention", "attention", "select", "select", "reorder", "reorder_paged"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "pages":
        return {"kind": kind, "requests": _log(rng, 1, 1000), "page": page, "longest": _log(rng, 8, 1024), "what": rng.choice(["step", "mixed"])}
    dim, kind_of = rng.choice([64, 64, 128, 128, 192, 256]), rng.choice(["q4_0", "q4_1"])
    if kind == "store":
        kv = _log(rng, 1, 25)
        return {"kind": kind, "tokens": _log(rng, 1, max(1, int(4e6 / (kv * dim)))), "heads": kv * rng.choice([1, 2, 4]), "kv_heads": kv, "dim": dim,
                "type": kind_of, "page": page}
    if kind == "attention":
        kv, group = _log(rng, 1, 25), rng.choice([1, 1, 2, 3, 4, 8])
        new = rng.choice([1, 1, 1, _log(rng, 2, 12), _log(rng, 12, 600)])
        longest = _log(rng, max(8, new), 100000 if new == 1 else max(new, 2000))
        most = 2.4e8 if new == 1 else min(2.4e8, 6e8 / (new * group) * dim / 2, 4e10 / (new * group))   # values of K; scores and products of the plain form
        kv = max(1, min(kv, int(most / (longest * dim))))
        batch = _log(rng, 1, max(1, min(256, int(most / (longest * kv * dim)))))
        return {"kind": kind, "batch": batch, "heads": kv * group, "kv_heads": kv, "dim": dim, "type": kind_of, "page": page,
                "longest": longest, "ragged": rng.random() < 0.7, "new": new}
    beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
    if kind == "select":
        vocab = rng.choice([50257, 32000, _log(rng, 100, 130000)])
        return {"kind": kind, "batch": _log(rng, 1, max(1, min(64, int(2.5e7 / (beams * vocab))))), "beams": beams, "vocab": vocab,
                "keep": rng.choice([beams, 2 * beams]), "ended": rng.random() < 0.5}
    batch = _log(rng, 1, max(1, 64 // beams))
    if kind == "reorder":
        layers, heads = rng.choice([(12, 12), (24, 16), (36, 20)])
        capacity = _log(rng, 32, 512)
        return {"kind": kind, "layers": layers, "batch": batch, "beams": beams, "heads": heads, "positions": rng.randint(1, capacity), "capacity": capacity}
    return {"kind": kind, "batch": batch, "beams": beams, "kv_heads": _log(rng, 1, 16), "dim": dim, "type": kind_of, "page": page, "positions": _log(rng, 1, 1500)}


# ---- inputs ---------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) % (1 << 40))


def _ints(gen, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=gen, device=DEV)


def _pages_of(lengths, page):
    return (lengths + page - 1) // page


def _spread(gen, count, lo, hi):
    """`count` numbers spread evenly over [lo, hi], in an order of the seed's: sums and largest ones are the same for every seed."""
    even = (torch.linspace(lo, hi, count, dtype=torch.float64, device=DEV) + 0.5).long() if count > 1 else torch.full((count,), hi, device=DEV)
    return even[torch.randperm(count, generator=gen, device=DEV)]


def _shortest(case):
    return max(case["new"], case["longest"] // 5)


def _tokens_added(case):
    """Tokens that the requests of a "pages" case grow by."""
    n = case["requests"]
    return n if case["what"] == "step" else int(_spread(_generator(0), n // 3, 1, case["longest"]).sum()) + n // 3


def _new_table(gen, lengths, page):
    """Table [len(lengths), most pages] of pages in no order, -1 behind them; pages in all."""
    count = _pages_of(lengths, page)
    columns = max(1, int(count.max()))
    total, used = int(count.sum()), torch.arange(columns, device=DEV)[None, :] < count[:, None]
    pool = total + total // 8 + 2
    order = torch.randperm(pool, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((len(lengths), columns), -1, dtype=torch.int32, device=DEV)
    table[used] = order[:total]
    return table, pool


def _tile_bytes(case):
    return case["dim"] * 16 + (4 if case["type"] == "q4_1" else 2) * case["dim"]   # 16 tokens: codes of K and V, scales (and minima)


def _random_pool(gen, case, pages):
    """A pool of pages as rows of keys and values (deviation 1) leave it: tile by tile through the plain form of the store, in portions."""
    tiles = pages * case["kv_heads"] * (case["page"] // 16)
    pool = torch.empty(tiles, _tile_bytes(case), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 26) // (16 * case["dim"]))
    for i in range(0, tiles, step):
        n = min(step, tiles - i)
        k, v = (torch.randn(n, 16, case["dim"], generator=gen, device=DEV) for _ in range(2))
        pool[i:i + n] = _to_tiles(case, k, v)
    return pool.view(-1)


def prepare(case, seed):
    gen, kind = _generator(seed), case["kind"]
    s = {"case": dict(case)}
    if kind == "pages":
        n, page, longest = case["requests"], case["page"], case["longest"]
        have = _spread(gen, n, 0, longest)
        if case["what"] == "step":
            want = have + 1
        else:   # a third are new, a third go on, of the rest some give tokens back and most end
            third = n // 3
            have[:third] = 0
            want = torch.cat([_spread(gen, third, 1, longest), have[third:2 * third] + 1, (have[2 * third:] - _ints(gen, 1, 8, n - 2 * third)).clamp(min=0)])
            want[2 * third + (n - 2 * third) // 4:] = 0
            mixed = torch.randperm(n, generator=gen, device=DEV)
            have, want = have[mixed], want[mixed]
        columns, tokens = longest // page + 1, _tokens_added(case)
        pool = n * columns   # what a server of so many requests keeps
        taken = torch.randperm(pool, generator=gen, device=DEV).to(torch.int32)
        held = torch.arange(columns, device=DEV)[None, :] < _pages_of(have, page)[:, None]
        full = torch.full((n, columns), -1, dtype=torch.int32, device=DEV)
        full[held] = taken[:int(held.sum())]
        rest = taken[int(held.sum()):]
        free = torch.full((pool,), -1, dtype=torch.int32, device=DEV)
        free[:len(rest)] = rest
        state = torch.zeros(4, dtype=torch.int32, device=DEV)
        state[0] = len(rest)
        s.update(have=have.to(torch.int32), want=want.to(torch.int32), columns=columns, pool=pool, tokens=tokens + 3,
                 before=torch.cat([full.view(-1), free, state]))
        s["after"] = torch.empty_like(s["before"])
        s["starts"] = torch.empty(n + 1, dtype=torch.int32, device=DEV)
        s["slots"] = torch.empty(s["tokens"], dtype=torch.int32, device=DEV)
    elif kind == "store":
        n, page, cols = case["tokens"], case["page"], case["kv_heads"] * case["dim"]
        s["x"] = torch.randn(n, case["heads"] * case["dim"] + 2 * cols, generator=gen, device=DEV) * torch.exp(torch.randn(n, 1, generator=gen, device=DEV) / 2)
        pages = -(-n // page) + 3
        order = torch.randperm(pages, generator=gen, device=DEV)
        at = torch.arange(n, device=DEV) + int(_ints(gen, 0, page, 1))
        slots = (order[at // page] * page + at % page).to(torch.int32)
        if n > 8:
            slots[-2:] = -1   # rows behind the last request
        pool = torch.zeros(pages * case["kv_heads"] * (page // 16) * _tile_bytes(case), dtype=torch.uint8, device=DEV)
        s.update(pages=pages, slots=slots, pool=pool, k=torch.zeros(n, cols, device=DEV), v=torch.zeros(n, cols, device=DEV))
    elif kind == "attention":
        b, new, longest = case["batch"], case["new"], case["longest"]
        if case["ragged"]:
            none = 1 if b > 3 else 0   # a place of the batch that no request has
            lengths, news = _spread(gen, b - none, _shortest(case), longest), _spread(gen, b - none, (new + 1) // 2, new)
            order = torch.randperm(b, generator=gen, device=DEV)
            lengths, news = (torch.cat([x, x.new_zeros(none)])[order] for x in (lengths, news))
        else:
            lengths, news = torch.full((b,), longest, device=DEV), torch.full((b,), new, device=DEV)
        table, pages = _new_table(gen, lengths, case["page"])
        starts = torch.zeros(b + 1, dtype=torch.int32, device=DEV)
        starts[1:] = news.cumsum(0)
        rows = int(starts[-1])
        q = torch.randn(rows, case["heads"] * case["dim"] + 64, generator=gen, device=DEV) * 2   # part of a wider matrix
        s.update(table=table, pages=pages, lengths=lengths.to(torch.int32), starts=starts, rows=rows, q=q, pool=_random_pool(gen, case, pages),
                 out=torch.zeros(rows, case["heads"] * case["dim"], device=DEV), by_starts=new > 1 or case["ragged"])
    elif kind == "select":
        b, beams, vocab = case["batch"], case["beams"], case["vocab"]
        x = torch.randn(b * beams, vocab, generator=gen, device=DEV) * 2.5
        x[:, :5] = -math.inf   # ids that are never produced
        scores = -(torch.rand(b, beams, generator=gen, device=DEV) * 12).sort(1).values - 20
        ended = _ints(gen, 0, 4, b, beams) == 0 if case["ended"] else torch.zeros(b, beams, dtype=torch.bool, device=DEV)
        s.update(x=x, scores=scores.contiguous(), ended=ended.to(torch.uint8), eos=vocab - 1,
                 out_scores=torch.empty(b, case["keep"], device=DEV), out_parents=torch.empty(b, case["keep"], dtype=torch.int32, device=DEV),
                 out_tokens=torch.empty(b, case["keep"], dtype=torch.int64, device=DEV), out_ended=torch.empty(b, case["keep"], dtype=torch.uint8, device=DEV))
    else:
        b, beams = case["batch"], case["beams"]
        # half of the hypotheses go on where they are, the others are given up for copies of them (a second pass then changes nothing more)
        rank = torch.rand(b, beams, generator=gen, device=DEV).argsort(1)
        lives = -(-beams // 2)
        chosen = rank.gather(1, _ints(gen, 0, lives, b, beams))
        keeps = torch.zeros(b, beams, dtype=torch.bool, device=DEV).scatter_(1, rank[:, :lives], True)
        s["parents"] = torch.where(keeps, torch.arange(beams, device=DEV), chosen).to(torch.int32)
        if kind == "reorder":
            shape = (b * beams, case["heads"], case["capacity"], 64)
            s["states"] = [torch.randn(shape, generator=gen, device=DEV) for _ in range(2 * case["layers"])]
        else:
            lengths = torch.full((b * beams,), case["positions"], device=DEV)
            table, pages = _new_table(gen, lengths, case["page"])
            s.update(table=table, pages=pages, lengths=lengths.to(torch.int32), pool=_random_pool(gen, case, pages))
    torch.cuda.synchronize()
    return s


# ---- plain forms ----------------------------------------------------------------------------------
def _quantise(x, q4_1):
    """x [..., 32] -> codes 0..15, scale (and minimum) in 16 bits: the blocks of the GGUF formats Q4_0 and Q4_1.  Which code is the
    nearest is decided in 64 bits."""
    x = x.double()
    if q4_1:
        low = x.amin(-1, keepdim=True)
        d = (x.amax(-1, keepdim=True) - low) / 15
        code = (x - low) / d + 0.5
    else:
        low, d = None, x.gather(-1, x.abs().argmax(-1, keepdim=True)) / -8
        code = x / d + 8.5
    d = d.float().half()
    code = torch.where(d == 0, 0.0 if q4_1 else 8.0, code.trunc().clamp(0, 15))
    return code.to(torch.uint8), d, low.half() if q4_1 else None


def _to_tiles(case, k, v):
    """Rows of 16 tokens, k and v [tiles, 16, dim], as tiles [tiles, bytes]."""
    n, dim, q4_1, parts = k.shape[0], case["dim"], case["type"] == "q4_1", []
    for x, of_k in ((k, True), (v, False)):
        codes, d, m = _quantise(x.reshape(n, 16, dim // 32, 32), q4_1)
        if of_k:   # token (hi, g), dim (chunk, block, t, byte, nibble) -> chunk, g, t, hi, block, byte, nibble
            codes = codes.reshape(n, 2, 8, dim // 64, 2, 4, 4, 2).permute(0, 3, 2, 5, 1, 4, 6, 7)
        else:      # token (hi, t, lo), dim (chunk, block, g, byte, nibble) -> chunk, g, t, hi, lo, block, byte, nibble
            codes = codes.reshape(n, 2, 4, 2, dim // 64, 2, 8, 2, 2).permute(0, 4, 6, 2, 1, 3, 5, 7, 8)
        parts.append((codes[..., 0] | codes[..., 1] << 4).reshape(n, -1))
        for h in (d, m):
            if h is not None:
                parts.append(h.reshape(n, 2, 4, 2, dim // 32).permute(0, 2, 4, 1, 3).contiguous().view(n, -1).view(torch.uint8).view(n, -1))
    return torch.cat(parts, 1)


def _from_tiles(case, tiles):
    """Tiles [..., bytes] -> k and v [..., 16, dim] in 32 bits."""
    dim, q4_1, lead, found, at = case["dim"], case["type"] == "q4_1", tiles.shape[:-1], [], 0
    tiles = tiles.reshape(-1, tiles.shape[-1])
    n = tiles.shape[0]
    for of_k in (True, False):
        raw, at = tiles[:, at:at + 8 * dim], at + 8 * dim
        codes = torch.stack([raw & 15, raw >> 4], -1)
        if of_k:
            codes = codes.reshape(n, dim // 64, 8, 4, 2, 2, 4, 2).permute(0, 4, 2, 1, 5, 3, 6, 7)
        else:
            codes = codes.reshape(n, dim // 64, 8, 4, 2, 2, 2, 2, 2).permute(0, 4, 3, 5, 1, 6, 2, 7, 8)
        halves = []
        for _ in range(2 if q4_1 else 1):
            h, at = tiles[:, at:at + dim].contiguous().view(torch.float16), at + dim
            halves.append(h.reshape(n, 4, dim // 32, 2, 2).permute(0, 3, 1, 4, 2).reshape(n, 16, dim // 32, 1).float())
        codes = codes.reshape(n, 16, dim // 32, 32).float()
        x = halves[0] * codes + halves[1] if q4_1 else halves[0] * (codes - 8)
        found.append(x.reshape(*lead, 16, dim))
    return found


def _plain_pages(s):
    case, n = s["case"], s["case"]["requests"]
    have, want, page, columns, pool, dev = s["have"].long(), s["want"].long(), s["case"]["page"], s["columns"], s["pool"], s["have"].device
    table = s["before"][:n * columns].view(n, columns)
    free, count = s["before"][n * columns:n * columns + pool], s["before"][n * columns + pool].long()
    held, wanted = _pages_of(have, page), _pages_of(want, page)
    column = torch.arange(columns, device=dev)
    gone = (column >= wanted[:, None]) & (column < held[:, None])
    come = (column >= held[:, None]) & (column < wanted[:, None])
    place = gone.view(-1).cumsum(0) - 1 + count
    back = torch.zeros(pool + 1, dtype=torch.int32, device=dev)
    back[:pool] = free
    back.scatter_(0, torch.where(gone.view(-1), place, pool), table.reshape(-1))
    back = back[:pool]
    top = count + gone.sum()
    pick = (top - come.view(-1).cumsum(0)).clamp(0, pool - 1)
    table = torch.where(come, back[pick].view(n, columns), torch.where(gone, -1, table))
    more = (want - have).clamp(min=0)
    starts = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), more.cumsum(0)])
    token = torch.arange(s["tokens"], device=dev)
    row = torch.searchsorted(starts, token, right=True).sub(1).clamp(max=n - 1)
    position = have[row] + token - starts[row]
    slot = table[row, (position // page).clamp(max=columns - 1)].long() * page + position % page
    slots = torch.where(token < starts[-1], slot, -1)
    state = torch.stack([top - come.sum(), starts[-1], torch.zeros_like(top), torch.zeros_like(top)])
    return {"table": table, "free": back, "state": state.to(torch.int32), "starts": starts.to(torch.int32), "slots": slots.to(torch.int32)}


def _plain_store(s):
    case, n = s["case"], s["case"]["tokens"]
    cols, at = case["kv_heads"] * case["dim"], case["heads"] * case["dim"]
    there = (s["slots"] >= 0)[:, None]
    found = {}
    for name, x in (("k", s["x"][:, at:at + cols]), ("v", s["x"][:, at + cols:])):
        codes, d, m = _quantise(x.reshape(n, -1, 32), case["type"] == "q4_1")
        y = d.float() * codes.float() + m.float() if m is not None else d.float() * (codes.float() - 8)
        found[name] = torch.where(there, y.reshape(n, cols), s[name])
    return found


def _plain_attention(s):
    case, dev = s["case"], s["q"].device
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    group, b, new = case["heads"] // kv, case["batch"], case["new"]
    pool = s["pool"].view(s["pages"], kv, page // 16, -1)
    k, v = _from_tiles(case, pool[s["table"].clamp(min=0)])                    # [b, pages, kv, page / 16, 16, dim]
    k, v = (x.permute(0, 2, 1, 3, 4, 5).reshape(b, kv, -1, dim) for x in (k, v))
    starts = s["starts"].long()
    news = starts[1:] - starts[:-1]
    i = torch.arange(new, device=dev)
    row = (starts[:-1, None] + i).clamp(max=s["rows"] - 1)                    # [b, new]
    q = s["q"][:, :case["heads"] * dim][row].view(b, new, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(b, kv, new * group, dim)
    score = torch.matmul(q, k.transpose(2, 3)) * (1 / math.sqrt(dim))
    last = s["lengths"].long()[:, None] - news[:, None] + i                    # position of row i
    seen = torch.arange(k.shape[2], device=dev) <= last[:, :, None]            # [b, new, t]
    seen = seen[:, None, :, None, :].expand(b, kv, new, group, -1).reshape(score.shape)
    score = torch.where(seen, score, -math.inf)
    top = score.amax(3, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    total = p.sum(3, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    o = o.view(b, kv, new, group, dim).permute(0, 2, 1, 3, 4).reshape(b, new, -1)
    out = s["out"].clone()
    there = i < news[:, None]
    out[row[there]] = o[there]
    return out


def _plain_select(s):
    case, dev = s["case"], s["x"].device
    b, beams, vocab, keep = case["batch"], case["beams"], case["vocab"], case["keep"]
    x, scores, ended = s["x"].view(b, beams, vocab).double(), s["scores"].double()[:, :, None], s["ended"][:, :, None] > 0
    top = x.amax(2, keepdim=True)
    total = torch.exp(x - top).sum(2, keepdim=True)
    value = scores + (x - (top + torch.log(total)))
    at_end = torch.arange(vocab, device=dev) == s["eos"]
    value = torch.where(ended, torch.where(at_end, scores, -math.inf), value).view(b, -1)
    value = torch.where(torch.isnan(value), -math.inf, value)
    among = min(2 * keep, value.shape[1])
    index = value.topk(among, 1).indices.sort(1).values                       # equal ones in the order of their index
    found, order = value.gather(1, index).sort(dim=1, descending=True, stable=True)
    found, index = found[:, :keep], index.gather(1, order)[:, :keep]
    none = found == -math.inf                                                 # places that no candidate is left for
    parents = torch.where(none, torch.arange(keep, device=dev).clamp(max=beams - 1), index // vocab)
    tokens = torch.where(none, s["eos"], index % vocab)
    ended = (ended[:, :, 0].gather(1, parents) | (tokens == s["eos"]))
    return {"scores": found.float(), "parents": parents.to(torch.int32), "tokens": tokens, "ended": ended.to(torch.uint8)}


def _plain_reorder(s):
    case = s["case"]
    b, beams, n = case["batch"], case["beams"], case["positions"]
    source = (s["parents"].long() + torch.arange(b, device=DEV)[:, None] * beams).view(-1)
    for x in s["states"]:
        x[:, :, :n] = x[:, :, :n][source]
    return s["states"]


def _plain_reorder_paged(s):
    case = s["case"]
    b, beams = case["batch"], case["beams"]
    source = (s["parents"].long() + torch.arange(b, device=DEV)[:, None] * beams).view(-1)
    pool = s["pool"].view(s["pages"], -1)
    pool[s["table"].view(-1).long()] = pool[s["table"][source].view(-1).long()]
    return s["pool"]


# ---- the package's entry points -------------------------------------------------------------------
def _runtime():
    if "runtime" not in _kept:
        from caten_b200 import _lib
        from caten_b200.runtime import B200Runtime
        _kept["runtime"] = rt = B200Runtime(0)
        _lib.check(rt.ctx, rt.lib.caten_b200_set_stream(rt.ctx, 1))   # the stream that torch's work is on
    return _kept["runtime"]


def _buffers(s):
    """The state's tensors as the package takes device memory, and its description of the cache: made at the first pass."""
    if "buffers" not in s:
        import numpy as np
        from caten_b200 import _lib
        from caten_b200.runtime import B200Buffer
        rt, case = _runtime(), s["case"]
        kinds = {torch.float32: np.float32, torch.int32: np.int32, torch.int64: np.int64, torch.uint8: np.uint8}
        wrap = lambda t: B200Buffer(rt, t.data_ptr(), t.shape, kinds[t.dtype], owned=False)   # noqa: E731
        u = {k: wrap(t) for k, t in s.items() if isinstance(t, torch.Tensor)}
        if "type" in case:
            u["desc"] = _lib.Kv4Desc(heads=case.get("heads", case["kv_heads"]), kv_heads=case["kv_heads"], dim=case["dim"], type=TYPES[case["type"]],
                                     page=case["page"], pages=s["pages"], scale=1 / math.sqrt(case["dim"]))
        if case["kind"] == "pages":
            n, columns = case["requests"], s["columns"]
            parts = [s["after"][:n * columns].view(n, columns), s["after"][n * columns:n * columns + s["pool"]], s["after"][n * columns + s["pool"]:]]
            u["parts"], u["views"] = parts, [wrap(p) for p in parts]
        elif case["kind"] == "store":
            cols, at = case["kv_heads"] * case["dim"], case["heads"] * case["dim"]
            u["xk"], u["xv"] = u["x"].view(at, (case["tokens"], cols)), u["x"].view(at + cols, (case["tokens"], cols))
        elif case["kind"] == "attention":
            u["work"] = rt.open_buffer(rt.kv4_attention_work(u["desc"], case["batch"], s["rows"], case["new"], case["longest"]), np.uint8)
        elif case["kind"] == "select":
            u["work"] = rt.open_buffer(rt.beam_select_work(case["batch"], case["beams"], case["vocab"], case["keep"]), np.uint8)
        elif case["kind"] == "reorder_paged":
            u["pages_of_pool"] = u["pool"].view(0, (s["pages"], s["pool"].numel() // s["pages"]))   # moved as the bytes that they are
        elif case["kind"] == "reorder":
            u["states"] = [wrap(t) for t in s["states"]]
        s["buffers"] = u
    return s["buffers"]


def _own(s):
    rt, u, case, kind = _runtime(), _buffers(s), s["case"], s["case"]["kind"]
    if kind == "pages":
        s["after"].copy_(s["before"])   # the call changes table, free list and state where they are
        table, free, state = u["views"]
        rt.kv_pages(u["have"], u["want"], case["page"], table, free, state, u["starts"], u["slots"])
        return {"table": u["parts"][0], "free": u["parts"][1], "state": u["parts"][2], "starts": s["starts"], "slots": s["slots"]}
    if kind == "store":
        rt.kv4_store(u["desc"], u["pool"], u["xk"], u["xv"], u["slots"], ld=s["x"].shape[1])
        rt.kv4_load(u["desc"], u["pool"], u["slots"], u["k"], u["v"])
        return {"k": s["k"], "v": s["v"]}
    if kind == "attention":
        rt.kv4_attention(u["desc"], u["q"], u["pool"], u["table"], u["lengths"], starts=u["starts"] if s["by_starts"] else None, max_new=case["new"],
                         max_length=case["longest"], out=u["out"], work=u["work"])
        return s["out"]
    if kind == "select":
        rt.beam_select(u["x"], u["scores"], case["keep"], ended=u["ended"], eos=s["eos"], out=(u["out_scores"], u["out_parents"], u["out_tokens"], u["out_ended"]),
                       work=u["work"])
        return {"scores": s["out_scores"], "parents": s["out_parents"], "tokens": s["out_tokens"], "ended": s["out_ended"]}
    if kind == "reorder":
        rt.beam_reorder(u["states"], u["parents"], case["positions"])
        return s["states"]
    rt.beam_reorder_pages(u["pages_of_pool"], u["table"], u["lengths"], u["parents"], case["page"])
    return s["pool"]


def run(state):
    if own:
        return _own(state)
    return {"pages": _plain_pages, "store": _plain_store, "attention": _plain_attention, "select": _plain_select, "reorder": _plain_reorder,
            "reorder_paged": _plain_reorder_paged}[state["case"]["kind"]](state)


# ---- the definitions in 64 bits -------------------------------------------------------------------
def _values(case, pool, page_ids, head):
    """Keys and values [tokens, dim] of one head in a list of pages, address by address."""
    dim, page, q4_1 = case["dim"], case["page"], case["type"] == "q4_1"
    tile, kv = _tile_bytes(case), case["kv_heads"]
    token = torch.arange(len(page_ids) * page, device=DEV)[:, None]
    j = torch.arange(dim, device=DEV)[None, :]
    base = ((page_ids.long()[token // page] * kv + head) * (page // 16) + token % page // 16) * tile
    t, block, within = token % 16, j // 32, j % 32
    found = []
    for of_k in (True, False):
        if of_k:
            lane, word, nibble = t % 8 * 4 + within // 8, t // 8 * 2 + block % 2, within % 8
        else:
            lane, word, nibble = within // 4 * 4 + t % 8 // 2, t // 8 * 2 + t % 2, block % 2 * 4 + within % 4
        start = base if of_k else base + tile // 2
        code = pool[start + block // 2 * 512 + lane * 16 + word * 4 + nibble // 2].long() >> nibble % 2 * 4 & 15
        place = (t % 8 // 2 * (dim // 32) + block) * 4 + t // 8 * 2 + t % 2
        halves = pool.view(torch.float16)
        d = halves[(start + 8 * dim) // 2 + place].double()
        found.append(d * code + halves[(start + 9 * dim) // 2 + place].double() if q4_1 else d * (code - 8))
    return found


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("pages",):
        return None   # whole numbers
    if kind == "store":
        cols, at, n, found = case["kv_heads"] * case["dim"], case["heads"] * case["dim"], case["tokens"], {}
        for name, x in (("k", s["x"][:, at:at + cols]), ("v", s["x"][:, at + cols:])):
            x = x.double().reshape(n, -1, 32)
            if case["type"] == "q4_1":
                low, high = x.min(2, keepdim=True).values, x.max(2, keepdim=True).values
                d = (high - low) / 15
                y = d.float().half().double() * ((x - low) / d + 0.5).floor().clamp(max=15) + low.half().double()
            else:
                d = torch.take_along_dim(x, x.abs().max(2, keepdim=True).indices, 2) / -8
                y = d.float().half().double() * ((x / d + 8.5).floor().clamp(max=15) - 8)
            found[name] = torch.where(s["slots"][:, None] < 0, 0.0, y.view(n, cols))
        return found
    if kind == "attention":
        dim, group, page = case["dim"], case["heads"] // case["kv_heads"], case["page"]
        out = torch.zeros(s["rows"], case["heads"], dim, dtype=torch.float64, device=DEV)
        q = s["q"][:, :case["heads"] * dim].double().view(s["rows"], case["heads"], dim)
        if 2 * case["batch"] * case["kv_heads"] * case["longest"] * dim > 8e9:
            return None
        starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
        for b, length in enumerate(lengths):
            new = starts[b + 1] - starts[b]
            if not new or not length:
                continue
            ids = s["table"][b, :-(-length // page)]
            ahead = torch.arange(length, device=DEV)[None, :] > torch.arange(length - new, length, device=DEV)[:, None]
            for head in range(case["kv_heads"]):
                k, v = _values(case, s["pool"], ids, head)
                k, v = k[:length], v[:length]
                for h in range(head * group, (head + 1) * group):
                    w = (q[starts[b]:starts[b + 1], h] @ k.T / math.sqrt(dim)).masked_fill(ahead, -math.inf)
                    w = (w - w.max(1, keepdim=True).values).exp()
                    out[starts[b]:starts[b + 1], h] = w @ v / w.sum(1, keepdim=True)
        return out.view(s["rows"], -1)
    if kind == "select":
        b, beams, vocab, found = case["batch"], case["beams"], case["vocab"], []
        for r in range(b):
            x = s["x"][r * beams:(r + 1) * beams].double()
            value = s["scores"][r].double()[:, None] + x - torch.logsumexp(x, 1, keepdim=True)
            for i in range(beams):
                if s["ended"][r, i]:
                    value[i] = -math.inf
                    value[i, s["eos"]] = s["scores"][r, i].double()
            found.append(value.view(-1).topk(case["keep"]).values)
        return {"scores": torch.stack(found), "parents": None, "tokens": None, "ended": None}
    if kind == "reorder":
        n, beams = case["positions"], case["beams"]
        parents = s["parents"].tolist()
        if sum(t.numel() for t in s["states"]) > 2e9:
            return None
        found = []
        for x in s["states"]:
            y = x.double()
            for r, row in enumerate(parents):
                for i, p in enumerate(row):
                    y[r * beams + i, :, :n] = x[r * beams + p, :, :n].double()
            found.append(y)
        return found
    return None   # bytes


def work(case):
    kind = case["kind"]
    if kind == "pages":
        n, tokens = case["requests"], _tokens_added(case)
        return {"bytes": 8 * n + 4 * (n + 1) + 4 * tokens + 16 * tokens / case["page"] + 16, "flops": 0}
    if kind in ("store", "attention", "reorder_paged"):
        packed = 2 * case["dim"] * (0.625 if case["type"] == "q4_1" else 0.5625) * case["kv_heads"]   # a token's keys and values
    if kind == "store":   # rows in, packed out, packed in, rows out
        return {"bytes": case["tokens"] * (2 * packed + 16 * case["kv_heads"] * case["dim"]), "flops": 0}
    if kind == "attention":
        b, new, longest = case["batch"], case["new"], case["longest"]
        there = b - 1 if case["ragged"] and b > 3 else b
        length = longest if not case["ragged"] or there == 1 else (_shortest(case) + longest) / 2
        rows = there * (new if not case["ragged"] or there == 1 else ((new + 1) // 2 + new) / 2)
        return {"bytes": there * length * packed + 8 * rows * case["heads"] * case["dim"],
                "flops": 4.0 * case["dim"] * case["heads"] * rows * (length - (rows / there - 1) / 2)}
    if kind == "select":
        n = case["batch"] * case["beams"]
        return {"bytes": n * (4 * case["vocab"] + 5) + case["batch"] * case["keep"] * 17, "flops": 0}
    moved = case["batch"] * (case["beams"] // 2)
    if kind == "reorder":
        each = 2 * case["layers"] * case["heads"] * case["positions"] * 256
    else:
        each = -(-case["positions"] // case["page"]) * case["page"] * packed
    return {"bytes": 2.0 * moved * each + 4 * case["batch"] * case["beams"] + 1, "flops": 0}
