"""GPU tests of the serving operators (pages and slots, 4-bit rows, attention over them, beam selection, reordering) against the plain
statements in oracle/serving_ref.py, at the sizes and masks where each can go wrong, and of a run of them together.

Tolerances.  Attention: u = 2^-23 a rounding (tensor-core sums may cut instead of round: a whole step).  A score is a sum over blocks of
d (sum q code + 8 sum q) with q in two halves (2^-22): its error is at most scale * sum |q| |d| (code + 8) * (16 + 16 + 16 + 16 + 4 + n blocks)
roundings of that magnitude, 80 u with room for the factors' own; probabilities then err by twice that relatively (numerator and sum), and the
second product, likewise a sum of d (code + 8)-sized terms, by (80 + tokens / 16) u of sum p |d| (code + 8) <= 23 max |d|.  Q4_1 has minima in the place
of 8 d.  Everything else (stores, pages, choices, moves) is exact."""
import ctypes as C

import numpy as np
import pytest

from caten_b200 import _lib as L
from caten_b200 import synthetic as S
from caten_b200._lib import B200Error
from oracle import serving_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"q4_0": L.Q4_0, "q4_1": L.Q4_1}


def rng_of(*seed):
    return np.random.Generator(np.random.PCG64(abs(hash(seed)) % (1 << 32) if any(isinstance(s, str) for s in seed) else list(seed)))


def put(rt, a, kind=None):
    return rt.transfer_from_array(np.ascontiguousarray(a, kind))


# ---- pages and slots ------------------------------------------------------------------------------
def run_pages(rt, have, want, page, table, free, n_free, max_tokens):
    n = len(have)
    b = dict(have=put(rt, have, np.int32), want=put(rt, want, np.int32), table=put(rt, table, np.int32), free=put(rt, free, np.int32),
             state=put(rt, [n_free, 7, 7, 7], np.int32), starts=put(rt, np.full(n + 1, 99), np.int32), slots=put(rt, np.full(max_tokens, 99), np.int32))
    rt.kv_pages(b["have"], b["want"], page, b["table"], b["free"], b["state"], b["starts"], b["slots"])
    return [b[k].numpy() for k in ("table", "free", "state", "starts", "slots")]


def some_pages(rng, n, page, longest, pool=None):
    have = rng.integers(0, longest + 1, n)
    have[rng.random(n) < 0.3] = 0
    want = np.where(rng.random(n) < 0.4, have + 1, rng.integers(0, longest + 2, n))
    want[rng.random(n) < 0.2] = 0
    columns = longest // page + 2
    pool = pool or n * columns + 3
    order = rng.permutation(pool)
    table, at = np.full((n, columns), -1), 0
    for r in range(n):
        c = -(-have[r] // page)
        table[r, :c] = order[at:at + c]
        at += c
    free = np.full(pool, -1)
    free[:pool - at] = order[at:]
    return have, want, columns, table, free, pool - at


@pytest.mark.parametrize("n,page,longest", [(1, 16, 40), (2, 64, 1), (31, 16, 700), (33, 128, 300), (64, 64, 1000), (1024, 16, 90), (2500, 32, 100), (3, 16, 30000)])
def test_pages_against_the_plain_plan(rt, n, page, longest):
    rng = rng_of(n, page, longest)
    have, want, columns, table, free, n_free = some_pages(rng, n, page, longest)
    tokens = int(np.maximum(want - have, 0).sum())
    for spare in (0, 5):
        got = run_pages(rt, have, want, page, table, free, n_free, tokens + spare)
        for g, w in zip(got, ref.pages(have, want, page, table, free, n_free, tokens + spare)):
            np.testing.assert_array_equal(g, w)


def test_pages_that_do_not_suffice_change_nothing(rt):
    rng = rng_of(5)
    have, want, columns, table, free, n_free = some_pages(rng, 40, 16, 200)
    want = np.maximum(want, have) + 40
    want = np.minimum(want, columns * 16)
    tokens = int((want - have).sum())
    takes = int((-(-want // 16) - -(-have // 16)).sum())
    few = takes - 3                      # three pages are missing
    bad = []
    for change, why in ((lambda h, w: w.__setitem__(7, -1), 1), (lambda h, w: h.__setitem__(39, -5), 1), (lambda h, w: w.__setitem__(0, columns * 16 + 1), 1),
                        (lambda h, w: w.__setitem__(0, 2**31 - 1), 1)):
        h, w = have.copy(), want.copy()
        change(h, w)
        bad.append((h, w, n_free, tokens + 500, why, 0))
    bad += [(have, want, few, tokens, 0, 3), (have, want, n_free, tokens - 1, 2, 0), (have, want, -1, tokens, 3, 0), (have, want, len(free) + 1, tokens, 3, 0)]
    for h, w, free_now, room, why, missing in bad:
        got = run_pages(rt, h, w, 16, table, free, free_now, room)
        np.testing.assert_array_equal(got[0], table)
        np.testing.assert_array_equal(got[1], free)
        assert got[2].tolist() == [free_now, 0, missing, why]
        assert (got[3] == 0).all() and (got[4] == -1).all()


def test_pages_of_no_requests(rt):
    got = run_pages(rt, [], [], 16, np.zeros((0, 3)), np.arange(9), 9, 4)
    assert got[2].tolist() == [9, 0, 0, 0] and got[3].tolist() == [0] and (got[4] == -1).all()
    got = run_pages(rt, [3], [3], 16, [[2, -1]], np.arange(9), 5, 0)
    assert got[2].tolist() == [5, 0, 0, 0] and got[3].tolist() == [0, 0]


# ---- rows -----------------------------------------------------------------------------------------
def description(kind, dim, page, pages, heads, kv_heads, scale=None):
    return L.Kv4Desc(heads=heads, kv_heads=kv_heads, dim=dim, type=TYPES[kind], page=page, pages=pages, scale=scale or dim ** -0.5)


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("dim,page,kv,tokens,extra,shift", [(64, 16, 1, 1, 0, 0), (64, 64, 25, 7, 64, 0), (128, 32, 3, 33, 1, 0), (192, 16, 2, 50, 0, 1), (256, 128, 1, 130, 4, 2)])
def test_rows_in_and_out(rt, kind, dim, page, kv, tokens, extra, shift):
    """Values, and the pool's bytes; rows of any stride and alignment, slots in any order, rows that go nowhere."""
    rng = rng_of(dim, page, tokens)
    cols, pages = kv * dim, -(-tokens // page) + 2
    ld = 2 * cols + extra
    x = rng.standard_normal(tokens * ld + shift, dtype=np.float32) * np.exp(rng.standard_normal(tokens * ld + shift, dtype=np.float32))
    x = x.astype(np.float32)
    rows = x[shift:].reshape(tokens, ld)
    rows[0, :32] = 0.0                                     # a block of zeros
    rows[0, 32:64] = 1e-9                                  # whose scale is none in 16 bits
    rows[-1, cols:cols + 32] = np.tile([3.0, -3.0], 16)    # equal magnitudes
    rows[-1, :32] = np.arange(32) / 31 * 15                # codes' own values, and halves of steps
    rows[tokens // 2, :32] = np.arange(32) / 2 - 8
    rows[tokens // 2, 32:64] = 7.25                        # one value only
    slots = rng.permutation(pages * page)[:tokens]
    if tokens > 5:
        slots[3] = slots[tokens - 2] = -1
    d = description(kind, dim, page, pages, kv, kv)
    pool = rt.kv4_pool(d)
    dx = put(rt, x)
    rt.kv4_store(d, pool, dx.view(shift, (tokens, cols)), dx.view(shift + cols, (tokens, cols)), put(rt, slots, np.int32), ld=ld)
    k, v = (put(rt, np.full((tokens, cols), 55.0), np.float32) for _ in range(2))
    rt.kv4_load(d, pool, put(rt, slots, np.int32), k, v)
    want_pool = np.zeros(pool.shape, np.uint8)
    for got, part in ((k.numpy(), rows[:, :cols]), (v.numpy(), rows[:, cols:2 * cols])):
        want = ref.values(part, kind == "q4_1")
        np.testing.assert_array_equal(got[slots >= 0], want[slots >= 0])
        assert (got[slots < 0] == 55.0).all()
    for i, slot in enumerate(slots):
        for h in range(kv if slot >= 0 else 0):
            ref.put(want_pool, page, kv, dim, kind == "q4_1", slot, h, rows[i, h * dim:(h + 1) * dim], rows[i, cols + h * dim:cols + (h + 1) * dim])
    np.testing.assert_array_equal(pool.numpy(), want_pool)   # the rest is as it was
    # out again into rows of a wider matrix that cannot be written by 16 bytes
    step = 2 * cols + 3
    wide = put(rt, np.zeros(tokens * step + 1, np.float32))
    rt.kv4_load(d, pool, put(rt, slots, np.int32), wide.view(1, (tokens, cols)), wide.view(1 + cols, (tokens, cols)), ld=step)
    got = wide.numpy()[1:].reshape(tokens, step)
    np.testing.assert_array_equal(got[slots >= 0][:, :2 * cols], np.concatenate([ref.values(rows[:, i:i + cols], kind == "q4_1") for i in (0, cols)], 1)[slots >= 0])
    assert (got[:, 2 * cols:] == 0).all() and (got[slots < 0] == 0).all()


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
def test_codes_next_to_a_border(rt, kind):
    """Values half a step apart, moved by single roundings: the codes are those that 64 bits give."""
    rng = rng_of(11)
    steps = rng.integers(-8, 8, (4000, 64)) + 0.5
    top = np.float32(2.0) ** rng.integers(-9, 9, (4000, 1)) * rng.choice([1.0, 1.3, 0.7], (4000, 1)).astype(np.float32)
    x = (steps.astype(np.float32) * top).astype(np.float32)
    x[:, 0::32] = -8 * top
    x[:, 1::32] = 7 * top
    x = np.nextafter(x, np.float32(1e30) * rng.integers(-1, 2, x.shape).astype(np.float32), dtype=np.float32)
    x = np.where(rng.random(x.shape) < 0.3, np.nextafter(x, np.float32(-1e30)), x).astype(np.float32)
    d = description(kind, 64, 16, 250, 1, 1)
    pool = rt.kv4_pool(d)
    slots = put(rt, np.arange(4000), np.int32)
    rt.kv4_store(d, pool, put(rt, x), put(rt, -x), slots)
    k, v = rt.kv4_load(d, pool, slots)
    np.testing.assert_array_equal(k.numpy(), ref.values(x, kind == "q4_1"))
    np.testing.assert_array_equal(v.numpy(), ref.values(-x, kind == "q4_1"))


def test_rows_that_are_not_finite_or_too_large_stay_in_their_blocks(rt):
    x = np.ones((4, 128), np.float32)
    x[0, 5], x[1, 40], x[2, 70], x[3, 100] = np.nan, np.inf, -np.inf, 3e38
    for kind in ("q4_0", "q4_1"):
        d = description(kind, 128, 16, 1, 1, 1)
        pool = rt.kv4_pool(d)
        slots = put(rt, np.arange(4), np.int32)
        rt.kv4_store(d, pool, put(rt, x), put(rt, x), slots)
        for y in rt.kv4_load(d, pool, slots):
            y = y.numpy().reshape(4, 4, 32)
            hit = np.eye(4, dtype=bool)
            assert np.isnan(y[hit]).all()                   # each such block is NaN
            assert (y[~hit] == 1.0).all() and not np.isnan(y[~hit]).any()


def test_slots_outside_the_pool_are_skipped_and_reported(rt):
    d = description("q4_0", 64, 16, 3, 1, 1)
    pool = rt.kv4_pool(d)
    x = put(rt, np.ones((5, 64)), np.float32)
    slots = put(rt, [0, 48, 47, -2, -2**31], np.int32)
    rt.kv4_store(d, pool, x, x, slots)
    with pytest.raises(B200Error) as e:
        rt.sync()
    assert e.value.code == L.EDEVICE and "bad index" in str(e.value)
    out = [put(rt, np.zeros((5, 64)), np.float32) for _ in range(2)]
    rt.kv4_load(d, pool, slots, *out)
    with pytest.raises(B200Error):
        rt.sync()
    np.testing.assert_array_equal(out[0].numpy()[:, 0], [1, 0, 1, 0, 0])
    rt.sync()


# ---- attention ------------------------------------------------------------------------------------
class Cache:
    """A pool in which sequences' pages lie in no order, full of NaN where nothing was stored."""

    def __init__(self, rt, rng, kind, dim, page, heads, kv, lengths, spare=2, k_scale=1.0, pages=None, scale=None):
        count = [-(-n // page) for n in lengths]
        columns = max(1, max(count, default=1)) + spare
        pages = pages or sum(count) + 3
        self.desc = description(kind, dim, page, pages, heads, kv, scale)
        self.pool = rt.kv4_pool(self.desc)
        L.check(rt.ctx, rt.lib.caten_b200_memset(rt.ctx, self.pool.ptr, 0xff, self.pool.nbytes))
        order, at = rng.permutation(pages) if pages < 1e6 else np.arange(pages - 1, 0, -1), 0
        self.table = np.full((len(lengths), columns), -1)
        slots = []
        for b, n in enumerate(lengths):
            self.table[b, :count[b]] = order[at:at + count[b]]
            at += count[b]
            slots += [self.table[b, t // page] * page + t % page for t in range(n)]
        total = len(slots)
        k = rng.standard_normal((total, kv * dim), dtype=np.float32) * np.float32(k_scale)
        v = rng.standard_normal((total, kv * dim), dtype=np.float32) * np.exp(rng.standard_normal((total, 1), dtype=np.float32))
        if total:
            rt.kv4_store(self.desc, self.pool, put(rt, k), put(rt, v), put(rt, slots, np.int32))
        q41 = kind == "q4_1"
        self.k, self.v = (ref.values(x, q41).reshape(total, kv, dim) for x in (k, v.astype(np.float32)))
        self.lengths, self.first = list(lengths), np.concatenate([[0], np.cumsum(lengths)]).astype(int)
        self.size = max([1e-3] + [np.abs(x).max() for x in (self.v,) if x.size])


def bound(c, q, tokens):
    """The stated tolerance: blocks' d (code + 8) is at most 3 (Q4_0) times their largest magnitude, minima included."""
    u = 2.0 ** -23
    if not c.k.size:
        return 0.0
    score = c.desc.scale * np.abs(q).reshape(-1, c.desc.dim).sum(1).max() * 3 * np.abs(c.k).max() * 80 * u
    return (2 * score + (80 + tokens / 16) * u * 3) * c.size


def check_attention(rt, c, q, news, extra_cols=0, rows_behind=0, starts=True, tol=None, max_length=0):
    heads, dim = c.desc.heads, c.desc.dim
    at = np.concatenate([[0], np.cumsum(news)]).astype(int)
    rows = at[-1] + rows_behind
    assert q.shape == (rows, heads, dim)
    wide = np.zeros((rows, heads * dim + extra_cols), np.float32)
    wide[:, :heads * dim] = q.reshape(rows, -1)
    out = put(rt, np.full((rows, heads * dim), 77.0), np.float32)
    rt.kv4_attention(c.desc, put(rt, wide), c.pool, put(rt, c.table, np.int32), put(rt, c.lengths, np.int32), put(rt, at, np.int32) if starts else None,
                     max_new=max(1, max(news)), max_length=max_length, out=out)
    got = out.numpy().reshape(rows, heads, dim)
    for b, n in enumerate(c.lengths):
        part = slice(c.first[b], c.first[b + 1])
        want = ref.attention(q[at[b]:at[b + 1]], c.k[part], c.v[part], n, c.desc.scale)
        np.testing.assert_allclose(got[at[b]:at[b + 1]], want, rtol=0, atol=tol or bound(c, q, n), err_msg=f"sequence {b} of {n}")
    assert (got[at[-1]:] == 77.0).all()
    return got


LENGTHS = [1, 15, 16, 17, 0, 63, 64, 65, 130, 257]


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("dim,page,heads,kv", [(64, 64, 25, 25), (64, 16, 4, 1), (128, 32, 6, 2), (128, 128, 16, 2), (192, 16, 3, 3), (256, 64, 10, 1),
                                                (64, 32, 1, 1), (128, 32, 3, 3), (256, 16, 2, 2), (256, 128, 1, 1),
                                                (64, 16, 6, 3), (128, 64, 8, 2), (192, 32, 4, 1), (256, 32, 3, 1), (128, 16, 12, 4)])
def test_single_tokens(rt, kind, dim, page, heads, kv):
    rng = rng_of(dim, page, heads)
    c = Cache(rt, rng, kind, dim, page, heads, kv, LENGTHS)
    q = rng.standard_normal((len(LENGTHS), heads, dim), dtype=np.float32) * 2
    check_attention(rt, c, q, [1] * len(LENGTHS), starts=False)
    check_attention(rt, c, q, [1] * len(LENGTHS), extra_cols=5)


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("dim,page,heads,kv", [(64, 16, 4, 4), (64, 64, 5, 1), (128, 32, 8, 2), (192, 128, 2, 2), (256, 16, 3, 1)])
def test_several_tokens_and_prompts(rt, kind, dim, page, heads, kv):
    """Rows of their own number a sequence, over a history or none; sequences without rows, without tokens, with fewer tokens than rows;
    rows behind the last sequence."""
    rng = rng_of(dim, page, heads, 2)
    lengths, news = [70, 33, 0, 100, 129, 3, 0, 40], [5, 33, 0, 0, 97, 7, 2, 1]
    c = Cache(rt, rng, kind, dim, page, heads, kv, lengths)
    q = rng.standard_normal((sum(news) + 3, heads, dim), dtype=np.float32)
    check_attention(rt, c, q, news, rows_behind=3, extra_cols=64)


@pytest.mark.parametrize("kind,dim,heads,kv,lengths,news", [("q4_0", 64, 2, 2, [5000], [1]), ("q4_1", 128, 8, 1, [4097, 1], [1, 1]), ("q4_0", 64, 2, 1, [3000, 2, 700], [9, 2, 1]),
                                                            ("q4_1", 256, 1, 1, [2500], [1]), ("q4_0", 128, 4, 4, [1, 1, 2100], [1, 0, 3]), ("q4_1", 128, 8, 2, [5000, 3, 0, 700], [1, 1, 0, 1]),
                                                            ("q4_0", 64, 6, 2, [4100], [1]), ("q4_1", 192, 4, 1, [2049], [1]), ("q4_1", 256, 3, 3, [1600, 90], [4, 2])])
def test_long_histories_are_shared_out(rt, kind, dim, heads, kv, lengths, news):
    rng = rng_of(dim, heads, 3)
    c = Cache(rt, rng, kind, dim, 64, heads, kv, lengths, k_scale=0.5)
    q = rng.standard_normal((sum(news), heads, dim), dtype=np.float32) * 2
    check_attention(rt, c, q, news)
    check_attention(rt, c, q, news, max_length=max(lengths))


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("heads,kv,lengths", [(4, 4, [(i * 7) % 41 for i in range(601)]), (8, 4, [(i * 7) % 41 for i in range(601)]),
                                              (8, 4, [5] * 57 + [4200] + [130, 1, 64, 0] * 14), (4, 4, [5] * 57 + [4200] + [130, 1, 64, 0] * 14)])
def test_many_sequences(rt, kind, heads, kv, lengths):
    rng = rng_of(len(lengths), heads, 4)
    c = Cache(rt, rng, kind, 64, 16, heads, kv, lengths)
    q = rng.standard_normal((len(lengths), heads, 64), dtype=np.float32)
    check_attention(rt, c, q, [1] * len(lengths))


def columns_for(rows, heads, dim, page):
    """Spare columns of a table with which the call may be large enough (rows x heads x tokens x dims) for the kernel for prompts."""
    return int(1.1e8 / (rows * heads * dim * page)) + 1


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("dim,page,heads,kv,lengths,news", [
    (64, 16, 50, 50, [130, 257, 300], [130, 257, 40]), (128, 64, 80, 40, [150, 5, 260], [150, 5, 100]), (64, 16, 1, 1, [64], [64]), (128, 64, 2, 1, [65], [33]), (64, 64, 3, 3, [128, 129, 0, 200, 257], [128, 129, 0, 50, 257]), (128, 128, 8, 2, [300, 64, 1], [300, 64, 1]),
    (128, 32, 4, 1, [1000, 20], [40, 60]), (64, 128, 2, 1, [2500], [70]), (128, 16, 2, 2, [2113], [129]), (64, 32, 9, 3, [191, 50, 63], [65, 50, 63])])
def test_long_prompts(rt, kind, dim, page, heads, kv, lengths, news):
    """Many rows a sequence: whole and ragged tiles of rows, histories shared out, sequences without tokens or with fewer tokens than rows; scales far apart."""
    rng = rng_of(dim, page, heads, 5)
    c = Cache(rt, rng, kind, dim, page, heads, kv, lengths, spare=columns_for(sum(news), heads, dim, page))
    q = rng.standard_normal((sum(news) + 2, heads, dim), dtype=np.float32)
    q[::3] *= 1e-3
    one = check_attention(rt, c, q, news, rows_behind=2, extra_cols=3)
    np.testing.assert_array_equal(check_attention(rt, c, q, news, rows_behind=2, extra_cols=3), one)
    check_attention(rt, c, q, news, rows_behind=2, max_length=max(lengths))


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("k_scale,q_scale", [(1e-3, 1e3), (300.0, 1e-3), (30.0, 1.0), (1.0, 1e-30), (1.0, 0.0)])
def test_prompts_with_scales_far_from_one(rt, kind, k_scale, q_scale):
    rng = rng_of(39)
    c = Cache(rt, rng, kind, 128, 64, 2, 1, [200], k_scale=k_scale, spare=columns_for(150, 2, 128, 64))
    check_attention(rt, c, rng.standard_normal((150, 2, 128), dtype=np.float32) * np.float32(q_scale), [150])


def test_a_prompt_whose_pages_or_lengths_are_wrong(rt):
    """Reported by the next synchronising call; other sequences are answered as before."""
    rng = rng_of(40)
    c = Cache(rt, rng, "q4_0", 64, 16, 2, 1, [150, 150, 150], spare=columns_for(240, 2, 64, 16))
    q = rng.standard_normal((240, 2, 64), dtype=np.float32)
    clean = check_attention(rt, c, q, [80, 80, 80])

    def run(table=c.table, lengths=c.lengths, starts=(0, 80, 160, 240)):
        out = rt.kv4_attention(c.desc, put(rt, q.reshape(240, -1)), c.pool, put(rt, table, np.int32), put(rt, lengths, np.int32), put(rt, starts, np.int32), max_new=80)
        with pytest.raises(B200Error) as e:
            rt.sync()
        assert e.value.code == L.EDEVICE
        return out.numpy().reshape(240, 2, 64)
    for wrong in (-1, c.desc.pages, 2**31 - 1, -2**31):
        t = c.table.copy()
        t[1, 4] = wrong
        got = run(table=t)
        np.testing.assert_array_equal(got[:80], clean[:80])
        np.testing.assert_array_equal(got[160:], clean[160:])
    for wrong in (-1, 2**31 - 1):
        got = run(lengths=[150, wrong, 150])
        np.testing.assert_array_equal(got[:80], clean[:80])
        np.testing.assert_array_equal(got[160:], clean[160:])
    got = run(starts=(0, 80, 1000, 240))
    np.testing.assert_array_equal(got[:80], clean[:80])
    rt.sync()


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
def test_one_workspace_for_every_call_up_to_the_largest(rt, kind):
    """Sized by kv4_attention_work for the largest turn; no call writes beyond what kv4_attention_call_work says of it."""
    rng = rng_of(22)
    for heads, kv, dim in ((4, 4, 64), (8, 2, 128), (3, 1, 256)):
        lengths = [2500, 700, 40, 1, 900, 64]
        c = Cache(rt, rng, kind, dim, 64, heads, kv, lengths)
        size = rt.kv4_attention_work(c.desc, 6, 6 * 60, 60, 2560)
        work = rt.open_buffer((size,), np.uint8)
        for batch, new, top in ((6, 60, 2560), (1, 60, 2560), (6, 1, 2560), (1, 1, 2560), (3, 3, 2560), (2, 12, 2500), (1, 2, 2500), (6, 60, 2500)):
            rows = [min(new, n) for n in lengths[:batch]]
            at = np.concatenate([[0], np.cumsum(rows)])
            need = rt.lib.caten_b200_kv4_attention_call_work(C.byref(c.desc), batch, int(at[-1]), new, top)
            assert 16 <= need <= size
            L.check(rt.ctx, rt.lib.caten_b200_memset(rt.ctx, work.ptr, 0x5a, size))
            q = rng.standard_normal((int(at[-1]), heads * dim), dtype=np.float32)
            args = (c.desc, put(rt, q), c.pool, put(rt, c.table[:batch], np.int32), put(rt, lengths[:batch], np.int32), put(rt, at, np.int32))
            out = rt.kv4_attention(*args, max_new=new, max_length=top, work=work).numpy()
            assert (work.numpy()[need if need > 16 else 0:] == 0x5a).all()   # (16: none is used)
            np.testing.assert_array_equal(out, rt.kv4_attention(*args, max_new=new, max_length=top).numpy())


def test_results_are_the_same_every_time(rt):
    rng = rng_of(21)
    c = Cache(rt, rng, "q4_0", 64, 64, 4, 2, [3000, 65, 900])
    q = rng.standard_normal((3, 4, 64), dtype=np.float32)
    one = check_attention(rt, c, q, [1, 1, 1])
    for _ in range(3):
        np.testing.assert_array_equal(check_attention(rt, c, q, [1, 1, 1]), one)


@pytest.mark.parametrize("k_scale,q_scale", [(1e-3, 1e3), (300.0, 1e-3), (30.0, 1.0), (1.0, 1e-30), (1.0, 0.0)])
def test_scales_far_from_one(rt, k_scale, q_scale):
    """Operands are brought into fp16's range by powers of two, whatever the sizes; sharp softmaxes pick single tokens."""
    rng = rng_of(31)
    for kind in ("q4_0", "q4_1"):
        c = Cache(rt, rng, kind, 64, 32, 2, 1, [150], k_scale=k_scale)
        q = rng.standard_normal((4, 2, 64), dtype=np.float32) * np.float32(q_scale)
        check_attention(rt, c, q, [4])


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("heads,kv,dim,news", [(2, 2, 64, 1), (2, 1, 64, 1), (8, 1, 64, 1), (4, 1, 128, 12)])
def test_queries_up_to_the_largest_float(rt, kind, heads, kv, dim, news):
    """Rows of q whose largest value is anywhere up to fp32's end, beside keys that are small: one token has all of the probability, and which one is
    plain from scores that differ in their second digit."""
    rng = rng_of(32, heads, news)
    c = Cache(rt, rng, kind, dim, 16, heads, kv, [70], k_scale=1e-6)
    for top in (1e30, 1e34, 3e35, 1e37, 3e38):
        q = rng.standard_normal((news, heads, dim), dtype=np.float32)
        q *= np.float32(top) / np.abs(q).max(-1, keepdims=True)
        out = rt.kv4_attention(c.desc, put(rt, q.reshape(news, -1)), c.pool, put(rt, c.table, np.int32), put(rt, c.lengths, np.int32), put(rt, [0, news], np.int32),
                               max_new=news).numpy().reshape(news, heads, dim)
        for i in range(news):
            sees = 70 - news + i + 1
            for h in range(heads):
                k, v = c.k[:sees, h // (heads // kv)], c.v[:sees, h // (heads // kv)]
                score = k.astype(np.float64) @ q[i, h].astype(np.float64)
                order = np.argsort(-score)
                # (scores are right to 2^-16 of sum |q k|, by far; the difference is many times that in units of the scale, so p is 1 and 0)
                if score[order[0]] - score[order[1]] > 2.0 ** -16 * (np.abs(k).astype(np.float64) @ np.abs(q[i, h]).astype(np.float64)).max():
                    np.testing.assert_allclose(out[i, h], v[order[0]], rtol=2.0 ** -20, atol=2.0 ** -20 * np.abs(v[order[0]]).max())
                else:
                    assert np.isfinite(out[i, h]).all()


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("q_scale", [3e5, 1e8, 1e20, 1e38])
@pytest.mark.parametrize("scale", [0.125, 0.0873, -3.1, 7e-20])
def test_prompts_whose_scores_are_large(rt, kind, q_scale, scale):
    """Scores beyond the whole numbers that fp32 holds: what has the largest one has all of the probability."""
    rng = rng_of(34)
    c = Cache(rt, rng, kind, 64, 16, 8, 1, [200], k_scale=1e-2, spare=columns_for(130, 8, 64, 16), scale=scale)
    q = rng.uniform(-1, 1, (130, 8, 64)).astype(np.float32) * np.float32(q_scale)
    out = rt.kv4_attention(c.desc, put(rt, q.reshape(130, -1)), c.pool, put(rt, c.table, np.int32), put(rt, c.lengths, np.int32), put(rt, [0, 130], np.int32),
                           max_new=130).numpy().reshape(130, 8, 64)
    assert np.isfinite(out).all()
    sure = 0
    for i in range(130):
        k, v = c.k[:200 - 130 + i + 1, 0].astype(np.float64), c.v[:200 - 130 + i + 1, 0]
        for h in range(8):
            score = scale * (k @ q[i, h].astype(np.float64))
            order = np.argsort(-score)
            # (scores are right to 2^-18 of scale sum |q k|: 22 bits of either operand, and sums that are cut off at the last bit)
            if score[order[0]] - score[order[1]] > 30 + 2.0 ** -17 * abs(scale) * (np.abs(k) @ np.abs(q[i, h]).astype(np.float64)).max():
                np.testing.assert_allclose(out[i, h], v[order[0]], rtol=2.0 ** -20, atol=2.0 ** -20 * np.abs(v[order[0]]).max())
                sure += 1
    assert sure > (500 if abs(scale) * q_scale > 1e5 else -1)


def test_values_of_very_different_sizes(rt):
    """Tokens of large values with small probabilities beside small values with large ones."""
    rng = rng_of(33)
    for kind in ("q4_0", "q4_1"):
        c = Cache(rt, rng, kind, 64, 16, 1, 1, [96])
        k, v = c.k.reshape(96, 64).copy(), c.v.reshape(96, 64) * np.exp(3 * rng.standard_normal((96, 1))).astype(np.float32)
        slots = [c.table[0, t // 16] * 16 + t % 16 for t in range(96)]
        rt.kv4_store(c.desc, c.pool, put(rt, k), put(rt, v), put(rt, slots, np.int32))
        c.k, c.v = (ref.values(x.astype(np.float32), kind == "q4_1").reshape(96, 1, 64) for x in (k, v))
        c.size = np.abs(c.v).max()
        check_attention(rt, c, rng.standard_normal((1, 1, 64), dtype=np.float32) * 2, [1])


def refill(rt, c, kind, k, v):
    """The cache's sequences hold these keys and values [tokens, kv_heads, dim]; what they are stored as, and the parts that they are added up from."""
    page, q41 = c.desc.page, kind == "q4_1"
    slots = [c.table[b, t // page] * page + t % page for b, n in enumerate(c.lengths) for t in range(n)]
    rows = [np.ascontiguousarray(x.reshape(len(slots), -1), np.float32) for x in (k, v)]
    rt.kv4_store(c.desc, c.pool, put(rt, rows[0]), put(rt, rows[1]), put(rt, slots, np.int32))
    c.k, c.v = (ref.values(x, q41).reshape(k.shape) for x in rows)
    c.k_parts, c.v_parts = (ref.parts(x, q41).reshape(k.shape) for x in rows)


def check_closely(rt, c, q, news, max_length=0):
    """Every value of every row against 64 bits, within the bound of its own row and block of 32 dims."""
    heads, dim = c.desc.heads, c.desc.dim
    at = np.concatenate([[0], np.cumsum(news)]).astype(int)
    got = rt.kv4_attention(c.desc, put(rt, q.reshape(len(q), -1)), c.pool, put(rt, c.table, np.int32), put(rt, c.lengths, np.int32), put(rt, at, np.int32),
                           max_new=max(news), max_length=max_length).numpy().reshape(-1, heads, dim)
    for b, n in enumerate(c.lengths):
        part, rows = slice(c.first[b], c.first[b + 1]), q[at[b]:at[b + 1]]
        want = ref.attention(rows, c.k[part], c.v[part], n, c.desc.scale)
        tol = ref.attention_bound(rows, c.k[part], c.k_parts[part], c.v_parts[part], n, c.desc.scale)
        off = np.abs(got[at[b]:at[b + 1]] - want)
        assert (off <= tol).all(), f"sequence {b} of {n}: {(off / np.maximum(tol, 1e-300)).max():.3g} times the bound"
    return got


# heads, key heads, dim, new tokens: the kernels for one row, for two to four, for tiles of eight, and for tiles of 128
ONE_ROW = [(2, 2, 64, 1), (3, 3, 128, 1), (1, 1, 192, 1), (2, 2, 256, 1)]
FEW_ROWS = [(2, 1, 64, 1), (8, 2, 128, 1), (3, 3, 64, 3), (4, 2, 192, 2), (3, 1, 256, 1), (4, 4, 128, 4)]
EIGHT_ROWS = [(8, 1, 64, 1), (12, 2, 128, 1), (2, 2, 64, 13), (8, 1, 128, 5), (6, 1, 192, 3), (2, 1, 256, 9)]
MANY_ROWS = [(8, 1, 64, 40), (4, 2, 128, 60), (3, 3, 64, 140)]


def spare_for(rows, heads, dim, page):
    return columns_for(rows, heads, dim, page) if rows >= 40 else 2


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("heads,kv,dim,news", ONE_ROW + FEW_ROWS + EIGHT_ROWS + MANY_ROWS)
def test_values_a_row_has_no_part_in_do_not_cost_it_bits(rt, kind, heads, kv, dim, news):
    """Tokens and blocks of 32 dims whose values are 1e8 times others': each block of a row is as close as its own sum of p |v| allows, whether the large values
    are behind the row's last token, have probabilities next to none, or are other dims'."""
    rng = rng_of(70, heads, dim, news)
    lengths = [90, 33, 200] if news < 40 else [news + 9, news, 200]
    c = Cache(rt, rng, kind, dim, 16, heads, kv, lengths, spare=spare_for(news, heads, dim, 16))
    total = sum(lengths)
    q = rng.standard_normal((3 * news, heads, dim), dtype=np.float32)
    shape = (total, kv, dim)
    v = rng.standard_normal(shape, dtype=np.float32)
    k = rng.standard_normal(shape, dtype=np.float32)
    far = 10.0 ** rng.uniform(-4, 4, (total, kv, dim // 32, 1)).astype(np.float32)
    refill(rt, c, kind, k, (v.reshape(*shape[:2], -1, 32) * far).reshape(shape))          # tokens and blocks in any order
    check_closely(rt, c, q, [news] * 3)
    of_block = 10.0 ** rng.uniform(-4, 4, (1, 1, dim // 32, 1)).astype(np.float32)
    refill(rt, c, kind, k, (v.reshape(*shape[:2], -1, 32) * of_block).reshape(shape))     # dims that are always large
    check_closely(rt, c, q, [news] * 3)
    late = np.ones((total, 1, 1), np.float32)
    for b in range(3):
        late[c.first[b + 1] - max(1, news // 2):c.first[b + 1]] = 1e6                     # seen by the last rows only
    refill(rt, c, kind, k, v * 1e-2 * late)
    check_closely(rt, c, q, [news] * 3)
    against = np.where(np.arange(total) % 3 == 0, np.float32(1e4), np.float32(1e-4))[:, None, None]
    same = np.repeat(q[:1, :1], len(q), 0).repeat(heads, 1)                               # large values where the probability is e^-30
    away = np.where(against > 1, -30.0, 0.0).astype(np.float32) / (c.desc.scale * (same[0, 0] ** 2).sum())
    refill(rt, c, kind, (k * 0.05 + same[0, 0] * away).astype(np.float32), v * against)
    check_closely(rt, c, same, [news] * 3)


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("heads,kv,dim,news", MANY_ROWS)
def test_small_keys_beside_large_ones_that_are_never_chosen(rt, kind, heads, kv, dim, news):
    """Every third key far against the queries, so that it has no probability, and 1e10 times as large as the others, whose scores decide."""
    rng = rng_of(73, heads, dim)
    c = Cache(rt, rng, kind, dim, 16, heads, kv, [160, 160], spare=spare_for(news, heads, dim, 16))
    k, v = (rng.standard_normal((320, kv, dim), dtype=np.float32) for _ in range(2))
    q = rng.standard_normal((2 * news, heads, dim), dtype=np.float32) * 5e4 + 1.5e5
    large = 4e5 if kind == "q4_0" else 5e4   # (of what the format holds)
    k = np.where(np.arange(320)[:, None, None] % 3 == 1, large * (-1 + 0.05 * k), k * 4e-6).astype(np.float32)
    refill(rt, c, kind, k, v)
    check_closely(rt, c, q, [news] * 2)


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("heads,kv,dim,spread", [(4, 1, 128, 0), (2, 2, 64, 0), (4, 1, 128, 400)])
def test_prompts_over_values_far_apart(rt, kind, heads, kv, dim, spread):
    """A few tokens whose keys or values halves of a common power of two cannot hold beside the others', with a token that is not finite behind them and a page that
    is none: each row is as close as ever, later tokens do not matter, and the page is reported."""
    rng = rng_of(72, heads, dim)
    lengths, news = [300 + spread, 150], [150, 150]
    c = Cache(rt, rng, kind, dim, 16, heads, kv, lengths, spare=0 if spread else columns_for(300, heads, dim, 16))
    shape = (sum(lengths), kv, dim)
    k, v = (rng.standard_normal(shape, dtype=np.float32) for _ in range(2))
    k[20], v[21], v[130], k[295 + spread] = k[20] * 1e-4, v[21] * 1e-6, v[130] * 1e4, k[295 + spread] * 30   # (k of 30: a score of hundreds)
    refill(rt, c, kind, k, v)
    q = rng.standard_normal((300, heads, dim), dtype=np.float32) * 0.3
    q[:, :, :32] = 0                                     # the large keys are elsewhere
    top = max(lengths)
    clean = check_closely(rt, c, q, news, max_length=top if spread else 0)
    np.testing.assert_array_equal(check_closely(rt, c, q, news, max_length=top if spread else 0), clean)

    def run(table=c.table):
        return rt.kv4_attention(c.desc, put(rt, q.reshape(300, -1)), c.pool, put(rt, table, np.int32), put(rt, lengths, np.int32), put(rt, [0, 150, 300], np.int32), max_new=150,
                                max_length=top if spread else 0).numpy().reshape(300, heads, dim)
    token = 240 + spread                                 # row 90
    for which in range(2):
        rows = [np.zeros((1, kv * dim), np.float32) for _ in range(2)]
        rows[which][0, 40::dim] = np.nan
        slot = put(rt, [c.table[0, token // 16] * 16 + token % 16], np.int32)
        kept = rt.kv4_load(c.desc, c.pool, slot)
        rt.kv4_store(c.desc, c.pool, put(rt, rows[0]), put(rt, rows[1]), slot)
        out = run()
        np.testing.assert_array_equal(out[:90], clean[:90])
        np.testing.assert_array_equal(out[150:], clean[150:])
        assert np.isnan(out[90:150, :, 32:64]).all()
        rt.kv4_store(c.desc, c.pool, *kept, slot)
    table = c.table.copy()
    table[0, 2] = -1                                     # tokens 32 to 47 count for nothing
    out = rt.kv4_attention(c.desc, put(rt, q.reshape(300, -1)), c.pool, put(rt, table, np.int32), put(rt, lengths, np.int32), put(rt, [0, 150, 300], np.int32), max_new=150,
                           max_length=top if spread else 0)
    with pytest.raises(B200Error) as e:
        rt.sync()
    assert e.value.code == L.EDEVICE
    out = out.numpy().reshape(300, heads, dim)
    there = (np.arange(lengths[0]) < 32) | (np.arange(lengths[0]) >= 48)
    part = slice(0, lengths[0])
    if kind == "q4_0":                                   # (its own values were stored back as they are)
        want = ref.attention(q[:150], c.k[part][there], c.v[part][there], lengths[0] - 16, c.desc.scale)
        tol = ref.attention_bound(q[:150], c.k[part][there], c.k_parts[part][there], c.v_parts[part][there], lengths[0] - 16, c.desc.scale)
        assert (np.abs(out[:150] - want) <= tol).all()
        np.testing.assert_array_equal(out[150:], clean[150:])


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("heads,kv,dim,news", ONE_ROW + FEW_ROWS + EIGHT_ROWS + MANY_ROWS)
@pytest.mark.parametrize("length", [65, 257, 1200, 5000])
def test_every_token_counts(rt, kind, heads, kv, dim, news, length):
    """Rows whose probability is on a few tokens: the last that they see, the first, and both sides of every border of groups, pages and parts.  The bound is such
    that none of them can be missing, nor one behind the last be seen, nor q or p be held in fewer bits (tests/test_serving.py)."""
    rng = rng_of(71, heads, dim, length)
    news = min(news, length)
    c = Cache(rt, rng, kind, dim, 64, heads, kv, [length], spare=spare_for(news, heads, dim, 64))
    k, v, q = ref.few_tokens(rng, length, kv, dim, heads, news, c.desc.scale)
    refill(rt, c, kind, k, v)
    check_closely(rt, c, q, [news])
    check_closely(rt, c, q, [news], max_length=length)


def test_nan_in_a_row_stays_in_it(rt):
    rng = rng_of(35)
    c = Cache(rt, rng, "q4_0", 64, 16, 2, 1, [40, 40])
    q = rng.standard_normal((6, 2, 64), dtype=np.float32)
    clean = check_attention(rt, c, q, [3, 3])
    bad = q.copy()
    bad[1, 0, 7], bad[5, 1, 0] = np.nan, np.inf
    out = rt.kv4_attention(c.desc, put(rt, bad.reshape(6, -1)), c.pool, put(rt, c.table, np.int32), put(rt, c.lengths, np.int32), put(rt, [0, 3, 6], np.int32),
                           max_new=3).numpy().reshape(6, 2, 64)
    hit = np.zeros((6, 2), bool)
    hit[1, 0] = hit[5, 1] = True
    assert np.isnan(out[hit]).all()
    np.testing.assert_array_equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 1), (16, 1)])
def test_what_later_tokens_hold_does_not_matter_to_earlier_ones(rt, kind, heads, kv):
    """A token whose keys or values are not finite, seen by the rows from its own on: those say so, the rows before it are as they were."""
    rng = rng_of(36, heads)
    c = Cache(rt, rng, kind, 64, 16, heads, kv, [90])
    q = rng.standard_normal((30, heads, 64), dtype=np.float32)
    clean = check_attention(rt, c, q, [30])
    for token in (60, 75, 89):
        for which in range(2):
            for value in (np.nan, np.inf):
                rows = [np.zeros((1, kv * 64), np.float32) for _ in range(2)]
                rows[which][0, 40] = value
                slot = put(rt, [c.table[0, token // 16] * 16 + token % 16], np.int32)
                kept = rt.kv4_load(c.desc, c.pool, slot)
                rt.kv4_store(c.desc, c.pool, put(rt, rows[0]), put(rt, rows[1]), slot)
                out = rt.kv4_attention(c.desc, put(rt, q.reshape(30, -1)), c.pool, put(rt, c.table, np.int32), put(rt, c.lengths, np.int32), put(rt, [0, 30], np.int32),
                                       max_new=30).numpy().reshape(30, heads, 64)
                seen = token - 60   # row i is token 60 + i
                np.testing.assert_array_equal(out[:seen], clean[:seen])
                assert not np.isfinite(out[seen:, :, 32:]).any()
                rt.kv4_store(c.desc, c.pool, *kept, slot)
                if kind == "q4_0":   # (its own values are stored as they are)
                    np.testing.assert_array_equal(rt.kv4_load(c.desc, c.pool, slot)[0].numpy(), kept[0].numpy())


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
@pytest.mark.parametrize("heads,news", [(1, 4), (1, 3), (2, 2), (24, 4), (32, 2), (8, 40)])
def test_what_later_tokens_hold_does_not_matter_to_few_rows(rt, kind, heads, news):
    """The same with two to four rows, and with many: a token of the last few that is not finite, or a row of q that is not."""
    rng = rng_of(38, heads, news)
    c = Cache(rt, rng, kind, 64, 16, heads, 1, [90], spare=columns_for(news, heads, 64, 16))
    q = rng.standard_normal((news, heads, 64), dtype=np.float32)
    clean = check_attention(rt, c, q, [news])

    def run(x):
        return rt.kv4_attention(c.desc, put(rt, x.reshape(news, -1)), c.pool, put(rt, c.table, np.int32), put(rt, c.lengths, np.int32), put(rt, [0, news], np.int32),
                                max_new=news).numpy().reshape(news, heads, 64)
    for token in {90 - news, 90 - news + 1, 90 - news // 2, 89}:
        for which in range(2):
            for value in (np.nan, np.inf):
                rows = [np.zeros((1, 64), np.float32) for _ in range(2)]
                rows[which][0, 40] = value
                slot = put(rt, [c.table[0, token // 16] * 16 + token % 16], np.int32)
                kept = rt.kv4_load(c.desc, c.pool, slot)
                rt.kv4_store(c.desc, c.pool, put(rt, rows[0]), put(rt, rows[1]), slot)
                out, seen = run(q), token - (90 - news)
                np.testing.assert_array_equal(out[:seen], clean[:seen])
                assert not np.isfinite(out[seen:, :, 32:]).any()
                rt.kv4_store(c.desc, c.pool, *kept, slot)
    bad = q.copy()
    bad[1, 0, 7], bad[0, heads - 1, 0] = np.nan, np.inf
    hit = np.zeros((news, heads), bool)
    hit[1, 0] = hit[0, heads - 1] = True
    out = run(bad)
    assert np.isnan(out[hit]).all()
    if kind == "q4_0":   # (its own values were stored back as they are)
        np.testing.assert_array_equal(out[~hit], clean[~hit])
    else:
        assert np.isfinite(out[~hit]).all()


def test_what_the_device_says_is_checked(rt):
    """Page numbers, lengths and starts outside what the call allows: skipped or cut, reported by the next synchronising call; other sequences
    are answered."""
    rng = rng_of(37)
    c = Cache(rt, rng, "q4_0", 64, 16, 2, 1, [40, 50, 20])
    q = rng.standard_normal((3, 2, 64), dtype=np.float32)
    clean = check_attention(rt, c, q, [1, 1, 1])
    pages = c.desc.pages

    def run(table=c.table, lengths=c.lengths, starts=(0, 1, 2, 3)):
        out = put(rt, np.full((3, 128), 77.0), np.float32)
        rt.kv4_attention(c.desc, put(rt, q.reshape(3, -1)), c.pool, put(rt, table, np.int32), put(rt, lengths, np.int32), put(rt, starts, np.int32), max_new=1, out=out)
        with pytest.raises(B200Error) as e:
            rt.sync()
        assert e.value.code == L.EDEVICE
        return out.numpy().reshape(3, 2, 64)
    for wrong in (-1, pages, 2**31 - 1, -2**31):
        t = c.table.copy()
        t[1, 1] = wrong
        got = run(table=t)
        np.testing.assert_array_equal(got[[0, 2]], clean[[0, 2]])
    for wrong in (-1, 2**31 - 1, c.table.shape[1] * 16 + 1):
        got = run(lengths=[40, wrong, 20])
        np.testing.assert_array_equal(got[[0, 2]], clean[[0, 2]])
    for wrong in ([0, 1, 5, 3], [-1, 1, 2, 3], [0, 3, 2, 3], [0, 1, 1, 3]):
        got = run(starts=wrong)
        for b in range(3):
            if wrong[b:b + 2] == [b, b + 1]:
                np.testing.assert_array_equal(got[b], clean[b])
    rt.sync()


def test_pages_beyond_four_gigabytes(rt):
    rng = rng_of(39)
    pages = 5 * 2**30 // (128 * 2 * 64 * 18 // 32 * 4)
    c = Cache(rt, rng, "q4_0", 64, 128, 4, 4, [300, 131], pages=pages)
    c.table[0, :3] = [pages - 1, pages - 2, pages // 2]
    c.table[1, :2] = [0, pages - 3]
    slots = [c.table[b, t // 128] * 128 + t % 128 for b, n in enumerate(c.lengths) for t in range(n)]
    k, v = (rng.standard_normal((431, 256), dtype=np.float32) for _ in range(2))
    rt.kv4_store(c.desc, c.pool, put(rt, k), put(rt, v), put(rt, slots, np.int32))
    got = rt.kv4_load(c.desc, c.pool, put(rt, slots, np.int32))
    c.k, c.v = (ref.values(x, False).reshape(431, 4, 64) for x in (k, v))
    np.testing.assert_array_equal(got[0].numpy(), c.k.reshape(431, 256))
    np.testing.assert_array_equal(got[1].numpy(), c.v.reshape(431, 256))
    check_attention(rt, c, rng.standard_normal((2, 4, 64), dtype=np.float32), [1, 1])
    c.pool.close()


# ---- beam selection -------------------------------------------------------------------------------
def check_select(rt, logits, scores, keep, ended=None, eos=-1, shift=0):
    groups, beams = scores.shape
    V = logits.shape[-1]
    flat = np.concatenate([np.zeros(shift, np.float32), logits.astype(np.float32).ravel()])
    dx = put(rt, flat).view(shift, (groups * beams, V))
    out = rt.beam_select(dx, put(rt, scores, np.float32), keep, ended=put(rt, ended, np.uint8) if ended is not None else None, eos=eos)
    got = [b.numpy() for b in out]
    for r in range(groups):
        want = ref.select(logits.reshape(groups, beams, V)[r].astype(np.float32), scores[r].astype(np.float32), ended[r] if ended is not None else np.zeros(beams), eos, keep)
        # a value is rounded once; its log of the sum is off by the exponentials' 2^-21 at most
        fin = np.isfinite(want[0])
        assert (got[0][r][~fin] == want[0][~fin]).all()
        np.testing.assert_allclose(got[0][r][fin], want[0][fin], rtol=2.0 ** -23, atol=2.0 ** -21)
        for g, w in zip(got[1:], want[1:]):
            np.testing.assert_array_equal(g[r], w)
    return got


@pytest.mark.parametrize("groups,beams,V,keep", [(1, 1, 1, 1), (1, 1, 7, 3), (2, 3, 2, 8), (3, 4, 50257, 4), (2, 5, 32000, 10), (1, 32, 1003, 32), (7, 2, 8192, 31), (1, 16, 8189, 32),
                                                 (1, 8, 130001, 16), (65, 1, 300, 2), (1, 32, 40000, 32), (1, 3, 1040384, 9), (20, 8, 20000, 16)])
def test_selection(rt, groups, beams, V, keep):
    rng = rng_of(groups, beams, V, keep)
    logits = rng.standard_normal((groups, beams, V), dtype=np.float32) * 3
    scores = -rng.random((groups, beams)).astype(np.float32) * 4
    for shift in range(4):
        check_select(rt, logits, scores, keep, shift=shift)
    ended = rng.random((groups, beams)) < 0.4
    check_select(rt, logits, scores, keep, ended=ended, eos=V // 2)
    check_select(rt, logits, scores, keep, ended=np.ones((groups, beams), bool), eos=0)
    first = np.where(np.arange(beams) == 0, 0.0, -np.inf) + np.zeros((groups, 1))
    check_select(rt, logits, first, keep, ended=np.zeros((groups, beams), bool), eos=V - 1)


def test_selection_of_equal_values_takes_the_lowest_index(rt):
    beams, V = 3, 20000
    flat = np.zeros((2, beams, V), np.float32)
    check_select(rt, flat, np.zeros((2, beams)), 32)                       # everything is equal
    check_select(rt, flat, np.array([[0, 1, 1], [-1, -1, 0]]), 20)
    flat[:, :, 1::2] = -0.0                                                # (zeros of both signs)
    check_select(rt, flat, np.zeros((2, beams)), 32)
    rng = rng_of(41)
    few = rng.integers(0, 3, (2, beams, V)).astype(np.float32)             # a few values, many times each
    check_select(rt, few, np.zeros((2, beams)), 32)
    for groups, beams, V in ((60, 2, 9000), (1, 32, 20000)):                # larger chunks; more lists than threads
        check_select(rt, rng.integers(0, 2, (groups, beams, V)).astype(np.float32), np.zeros((groups, beams)), 32)
        check_select(rt, np.zeros((groups, beams, V)), np.zeros((groups, beams)), 32)


@pytest.mark.parametrize("groups,beams,V,keep", [(1, 8, 50257, 32), (4, 8, 50257, 16), (3, 5, 1003, 32), (40, 4, 30011, 8), (1, 32, 20003, 32)])
def test_selection_is_decided_in_64_bits_between_beams(rt, groups, beams, V, keep):
    """Rows that are equal bit for bit, at every alignment that a vocabulary of odd size gives them, and rows whose sums differ by less than fp32 can
    tell: which beam comes first is what 64 bits say, equal ones by their index."""
    rng = rng_of(groups, beams, V)
    row = rng.standard_normal((groups, 1, V), dtype=np.float32) * 3
    same = np.repeat(row, beams, 1)
    scores = np.full((groups, beams), -2.5)
    for shift in range(4):
        check_select(rt, same, scores, keep, shift=shift)
    ended = np.zeros((groups, beams), bool)
    ended[:, 1] = True
    check_select(rt, same, scores, keep, ended=ended, eos=7)
    # a logit of small probability raised in the beams before the last: their sums are larger by 1e-8 to 1e-10 of themselves, their candidates later
    for down in (18.0, 20.0, 23.0):
        x = same.copy()
        low = x.argmin(-1)
        for g in range(groups):
            for b in range(beams):
                x[g, b, low[g, b]] = x[g, b].max() - down - b / 64
        check_select(rt, x, scores, keep, shift=1)
        check_select(rt, x[:, ::-1], scores, keep, shift=2)
    # the last that is taken and the first that is left: equal values of beams in turn, all but the first at a distance from those before
    few = np.full((groups, beams, V), -30.0, np.float32)
    few[:, :, V // 2:V // 2 + 5] = 0.0
    check_select(rt, few, scores, min(keep, 7))
    many = np.where(np.arange(V) < keep - 1, np.float32(1), np.float32(-20)) + np.zeros((groups, beams, 1), np.float32)
    check_select(rt, many, scores - np.where(np.arange(beams) == 0, 0.0, 2.0), keep, shift=3)


@pytest.mark.parametrize("groups,beams,V,keep", [(3, 4, 20000, 32), (30, 3, 9001, 20), (1, 32, 20000, 32)])
def test_selection_among_more_equal_values_than_are_looked_at(rt, groups, beams, V, keep):
    """Beams whose logits are a few values, so that hundreds of candidates are equal, with ended, masked and broken hypotheses between them."""
    rng = rng_of(groups, beams, V, 1)
    x = np.repeat(rng.integers(0, 2, (groups, 1, V)).astype(np.float32) * np.float32(0.7) - np.float32(0.3), beams, 1)
    scores = np.full((groups, beams), -1.5, np.float32)
    for eos, ended in ((-1, None), (5, rng.random((groups, beams)) < 0.4)):
        check_select(rt, x, scores, keep, ended=ended, eos=eos, shift=1)
    y = x.copy()
    y[0, 0] = -np.inf
    y[0, beams // 2, 7] = np.nan
    y[:, beams - 1, :V - 3] = np.finfo(np.float32).min
    scores[-1, 1] = -np.inf
    for eos, ended in ((-1, None), (5, rng.random((groups, beams)) < 0.4)):
        check_select(rt, y, scores, keep, ended=ended, eos=eos)


@pytest.mark.parametrize("score", [-1e30, float(np.finfo(np.float32).min)])
@pytest.mark.parametrize("groups,beams,V,keep", [(2, 3, 5000, 32), (20, 8, 9001, 16), (1, 4, 40, 20)])
def test_selection_from_scores_that_leave_no_room_for_logits(rt, groups, beams, V, keep, score):
    """Hypotheses kept out by a very low score, all of whose candidates have one value in 64 bits: in the order of their beams, and of a beam's
    logits."""
    rng = rng_of(groups, beams, V)
    x = rng.integers(-40, 40, (groups, beams, V)).astype(np.float32) / 4
    check_select(rt, x, np.full((groups, beams), score), keep)
    check_select(rt, x, np.where(np.arange(beams) == 1, 0.0, score) + np.zeros((groups, 1)), keep, ended=np.arange(groups * beams).reshape(groups, beams) % 5 == 0, eos=3)


@pytest.mark.parametrize("order", ["up", "down"])
def test_selection_from_sorted_logits(rt, order):
    """The largest logits lie side by side, in one block's share."""
    V = 30011
    x = np.linspace(-6, 6, V, dtype=np.float32)[None, None].repeat(2, 1)
    check_select(rt, x if order == "up" else x[:, :, ::-1].copy(), np.array([[0.0, -0.25]]), 32)


def test_selection_with_masks(rt):
    rng = rng_of(43)
    V = 9001
    x = rng.standard_normal((6, 4, V), dtype=np.float32)
    x[0, :, 100:] = -np.inf                      # a short list of allowed ids
    x[1, 1] = -np.inf                            # a hypothesis that cannot go on
    x[2, :, :] = -np.inf                         # none can
    x[2, 3, 8999] = 1.0
    x[3] = -np.inf                               # nothing at all
    x[4, 2, 17], x[4, 0, 5], x[4, 1] = np.nan, np.inf, np.finfo(np.float32).min   # rows without a distribution; the lowest value as a mask
    x[5, :, ::2] = np.finfo(np.float32).min
    scores = -rng.random((6, 4)).astype(np.float32)
    scores[5] = [-np.inf, 0, np.nan, -1]
    for keep in (1, 8, 32):
        check_select(rt, x, scores, keep, ended=np.zeros((6, 4), bool), eos=3)
        ended = np.zeros((6, 4), bool)
        ended[2:4, 1] = True
        check_select(rt, x, scores, keep, ended=ended, eos=3)


def test_selection_leaves_the_logits_of_ended_hypotheses_alone_and_needs_no_flags_out(rt):
    rng = rng_of(45)
    x = rng.standard_normal((4, 500), dtype=np.float32)
    x[1] = np.nan
    out = rt.beam_select(put(rt, x), put(rt, [[-1, -2, -3, -4]], np.float32), 4, ended=put(rt, [[0, 1, 0, 0]], np.uint8), eos=7,
                         out=(rt.open_buffer((1, 4)), rt.open_buffer((1, 4), np.int32), rt.open_buffer((1, 4), np.int64), None))
    want = ref.select(x, np.array([-1, -2, -3, -4.0]), np.array([0, 1, 0, 0]), 7, 4)
    np.testing.assert_array_equal(out[1].numpy()[0], want[1])
    np.testing.assert_array_equal(out[2].numpy()[0], want[2])


# ---- reordering -----------------------------------------------------------------------------------
@pytest.mark.parametrize("groups,beams,H,T,X,n,kind", [(1, 2, 1, 1, 64, 1, np.float32), (3, 4, 5, 40, 64, 17, np.float32), (2, 7, 2, 9, 3, 5, np.float32), (1, 16, 2, 33, 64, 33, np.float32),
                                                       (2, 32, 1, 20, 16, 19, np.int32), (5, 1, 2, 4, 4, 4, np.float32), (2, 5, 3, 12, 8, 0, np.float32), (4, 9, 1, 6, 6, 6, np.float16)])
def test_reordering(rt, groups, beams, H, T, X, n, kind):
    rng = rng_of(groups, beams, H, T)
    states = [(rng.standard_normal((groups * beams, H, T, X)) * 100).astype(kind) for _ in range(3)]
    some = [rng.integers(0, beams, (groups, beams)), np.stack([rng.permutation(beams) for _ in range(groups)]), np.tile(np.roll(np.arange(beams), 1), (groups, 1)),
            np.full((groups, beams), beams - 1), np.tile(np.arange(beams), (groups, 1))]
    for parents in some:
        b = [put(rt, x) for x in states]
        rt.beam_reorder(b, put(rt, parents, np.int32), n)
        source = (parents + np.arange(groups)[:, None] * beams).ravel()
        for x, y in zip(states, b):
            want = x.copy()
            want[:, :, :n] = x[source][:, :, :n]
            np.testing.assert_array_equal(y.numpy(), want)


def test_reordering_many_states_in_one_call(rt):
    """More than one launch's worth, at addresses of every alignment."""
    rng = rng_of(51)
    x = rng.standard_normal((301, 2 * 3 * 1 * 4 * 4 + 1), dtype=np.float32)
    buf = put(rt, x)
    states = [buf.view(i * x.shape[1], (6, 1, 4, 4)) for i in range(301)]
    parents = np.array([[1, 2, 0], [2, 2, 2]])
    rt.beam_reorder(states, put(rt, parents, np.int32), 3)
    want = x[:, :-1].reshape(301, 6, 4, 4).copy()
    want[:, :, :3] = x[:, :-1].reshape(301, 6, 4, 4)[:, [1, 2, 0, 5, 5, 5]][:, :, :3]
    got = buf.numpy()
    np.testing.assert_array_equal(got[:, :-1].reshape(301, 6, 4, 4), want)
    np.testing.assert_array_equal(got[:, -1], x[:, -1])
    rt.beam_reorder([], put(rt, parents, np.int32), 3)


def test_parents_out_of_range_leave_rows_and_are_reported(rt):
    x = np.arange(4 * 2 * 3 * 4, dtype=np.float32).reshape(4, 2, 3, 4)
    for wrong in (-1, 4, 2**31 - 1, -2**31):
        b = put(rt, x)
        rt.beam_reorder([b], put(rt, [[1, wrong, 0, 2]], np.int32), 3)
        with pytest.raises(B200Error) as e:
            rt.sync()
        assert e.value.code == L.EDEVICE
        np.testing.assert_array_equal(b.numpy(), x[[1, 1, 0, 2]])
    b = put(rt, x)
    rt.beam_reorder([b], put(rt, [[0], [1], [0], [0]], np.int32), 3)   # one beam has one parent
    with pytest.raises(B200Error):
        rt.sync()
    np.testing.assert_array_equal(b.numpy(), x)


@pytest.mark.parametrize("groups,beams,page,width,longest", [(1, 2, 16, 16, 5), (3, 4, 16, 4624, 100), (2, 8, 64, 48, 300), (1, 32, 32, 160, 64), (2, 13, 16, 32, 40)])
def test_reordering_pages(rt, groups, beams, page, width, longest):
    rng = rng_of(groups, beams, page)
    columns, n = -(-longest // page) + 1, groups * beams
    lengths = np.repeat(rng.integers(0, longest + 1, groups), beams)
    lengths[:beams] = longest
    pages = n * columns
    pool = rng.integers(0, 256, (pages, width)).astype(np.uint8)
    table = np.where(np.arange(columns) * page < lengths[:, None], rng.permutation(pages).reshape(n, columns), -1)
    for parents in (rng.integers(0, beams, (groups, beams)), np.stack([rng.permutation(beams) for _ in range(groups)])):
        b = put(rt, pool)
        rt.beam_reorder_pages(b, put(rt, table, np.int32), put(rt, lengths, np.int32), put(rt, parents, np.int32), page)
        want = pool.copy()
        for i, p in enumerate((parents + np.arange(groups)[:, None] * beams).ravel()):
            for j in range(-(-lengths[i] // page)):
                want[table[i, j]] = pool[table[p, j]]
        np.testing.assert_array_equal(b.numpy(), want)
    # a page number that is none, in the second sequence of a pair
    t, p = table.copy(), np.tile(np.arange(beams), (groups, 1))
    t[1, 0], p[0, 0] = pages, 1
    b = put(rt, pool)
    rt.beam_reorder_pages(b, put(rt, t, np.int32), put(rt, lengths, np.int32), put(rt, p, np.int32), page)
    with pytest.raises(B200Error):
        rt.sync()
    np.testing.assert_array_equal(b.numpy()[table[0, 1:][table[0, 1:] >= 0]], pool[table[1, 1:][table[1, 1:] >= 0]])


# ---- together -------------------------------------------------------------------------------------
def test_a_serving_loop(rt):
    """Requests of their own lengths come, grow and end: every turn plans pages, stores its rows and attends, against caches that are kept
    plainly on the host."""
    rng = rng_of(61)
    R, page, heads, kv, dim, pool_pages, columns = 5, 16, 4, 2, 64, 24, 8
    for kind in ("q4_0", "q4_1"):
        d = description(kind, dim, page, pool_pages, heads, kv)
        pool = rt.kv4_pool(d)
        table, free, state = put(rt, np.full((R, columns), -1), np.int32), put(rt, rng.permutation(pool_pages), np.int32), put(rt, [pool_pages, 0, 0, 0], np.int32)
        starts, slots = rt.open_buffer((R + 1,), np.int32), rt.open_buffer((128,), np.int32)
        kept = [np.zeros((0, 2, kv, dim), np.float32) for _ in range(R)]
        lengths = np.zeros(R, int)
        plan = [[20, 0, 5, 33, 0], [21, 16, 6, 34, 1], [22, 17, 0, 35, 2], [23, 18, 40, 20, 3], [0, 19, 41, 21, 4], [60, 20, 42, 22, 0], [61, 21, 43, 23, 9]]
        for want in plan:
            want = np.array(want)
            before, after = put(rt, lengths, np.int32), put(rt, want, np.int32)
            rt.kv_pages(before, after, page, table, free, state, starts, slots)
            assert state.numpy()[2:].tolist() == [0, 0]
            news = np.maximum(want - lengths, 0)
            T = int(news.sum())
            qkv = rng.standard_normal((128, (heads + 2 * kv) * dim), dtype=np.float32)
            dq = put(rt, qkv)
            rt.kv4_store(d, pool, dq.view(heads * dim, (128, kv * dim)), dq.view((heads + kv) * dim, (128, kv * dim)), slots, ld=qkv.shape[1])
            out = rt.kv4_attention(d, dq, pool, table, after, starts, max_new=int(news.max()), max_length=int(want.max())).numpy().reshape(128, heads, dim)
            at = 0
            for r in range(R):
                rows = qkv[at:at + news[r]]
                new = np.stack([ref.values(rows[:, (heads + i * kv) * dim:(heads + (i + 1) * kv) * dim], kind == "q4_1").reshape(-1, kv, dim) for i in range(2)], 1)
                kept[r] = np.concatenate([kept[r][:min(lengths[r], want[r])], new])
                want_out = ref.attention(rows[:, :heads * dim].reshape(-1, heads, dim), kept[r][:, 0], kept[r][:, 1], want[r], d.scale)
                np.testing.assert_allclose(out[at:at + news[r]], want_out, rtol=0, atol=2e-3)   # (bound() of these sizes: 4e-3)
                at += news[r]
            assert at == T
            lengths = want
        held = sum(-(-n // page) for n in lengths)
        assert state.numpy()[0] == pool_pages - held
        ids = np.concatenate([free.numpy()[:pool_pages - held], table.numpy()[table.numpy() >= 0]])
        assert sorted(ids) == list(range(pool_pages))   # no page lost, none twice


def test_captured_and_replayed_on_a_stream_of_the_caller(rt):
    """Plan, rows, attention and selection in one graph, twice over: two graphs with workspaces of their own are replayed on two streams at once."""
    import torch
    from caten_b200.runtime import B200Runtime
    rng = rng_of(63)
    r = B200Runtime(0)
    try:
        sets = []
        for which in range(2):
            c = Cache(r, rng, "q4_0", 64, 64, 4, 2, [1500, 70])
            slots = [c.table[b, (n - 1) // 64] * 64 + (n - 1) % 64 for b, n in enumerate(c.lengths)]
            x = rng.standard_normal((2, 8 * 64), dtype=np.float32)
            logits = rng.standard_normal((8, 20000), dtype=np.float32)
            s = dict(c=c, x=put(r, x), slots=put(r, slots, np.int32), table=put(r, c.table, np.int32), lengths=put(r, c.lengths, np.int32), out=r.open_buffer((2, 256)),
                     work=r.open_buffer(r.kv4_attention_work(c.desc, 2, 2, 1, 1500), np.uint8), logits=put(r, logits), scores=put(r, np.zeros((2, 4)), np.float32),
                     picked=tuple(r.open_buffer((2, 4), t) for t in (np.float32, np.int32, np.int64, np.uint8)),
                     swork=r.open_buffer(r.beam_select_work(2, 4, 20000, 4), np.uint8), host=(x, logits), stream=torch.cuda.Stream(), graph=torch.cuda.CUDAGraph())

            def step(s=s, c=c):
                r.kv4_store(c.desc, c.pool, s["x"].view(256, (2, 128)), s["x"].view(384, (2, 128)), s["slots"], ld=512)
                r.kv4_attention(c.desc, s["x"], c.pool, s["table"], s["lengths"], max_length=1500, out=s["out"], work=s["work"])
                r.beam_select(s["logits"], s["scores"], 4, out=s["picked"], work=s["swork"])
            step()
            r.sync()
            L.check(r.ctx, r.lib.caten_b200_set_stream(r.ctx, s["stream"].cuda_stream))
            with torch.cuda.graph(s["graph"], stream=s["stream"], capture_error_mode="thread_local"):
                step()
            L.check(r.ctx, r.lib.caten_b200_set_stream(r.ctx, None))
            sets.append(s)
        want = []
        for s in sets:
            for b in (s["out"], s["picked"][0]):
                L.check(r.ctx, r.lib.caten_b200_memset(r.ctx, b.ptr, 0, b.nbytes))
        r.sync()
        for _ in range(5):
            for s in sets:
                with torch.cuda.stream(s["stream"]):
                    s["graph"].replay()
        torch.cuda.synchronize()
        for s in sets:
            c, (x, logits) = s["c"], s["host"]
            for b, n in enumerate(c.lengths):
                part = slice(c.first[b], c.first[b + 1])
                k, v = c.k[part].copy(), c.v[part].copy()
                k[-1], v[-1] = (ref.values(x[b, i:i + 128], False).reshape(2, 64) for i in (256, 384))
                want = ref.attention(x[b, :256].reshape(1, 4, 64), k, v, n, c.desc.scale)
                np.testing.assert_allclose(s["out"].numpy()[b].reshape(1, 4, 64), want, rtol=0, atol=bound(c, x[:, :256], n))
                sel = ref.select(logits[4 * b:4 * b + 4], np.zeros(4), np.zeros(4), -1, 4)
                np.testing.assert_array_equal(s["picked"][2].numpy()[b], sel[2])
            del s["graph"]
    finally:
        r.close()


def test_prompts_on_two_streams_at_once(rt):
    """Graphs of attention over prompts, one cut into parts and one whole, and of few rows, each replayed on a stream of its own."""
    import torch
    from caten_b200.runtime import B200Runtime
    r = B200Runtime(0)
    try:
        sets = []
        for heads, kv, dim, lengths, news in ((4, 1, 128, [900], [200]), (50, 50, 64, [260, 131, 300], [260, 131, 300]), (8, 2, 64, [900, 40], [3, 3])):
            rng = rng_of(64, heads)
            c = Cache(r, rng, "q4_1", dim, 64, heads, kv, lengths, spare=columns_for(sum(news), heads, dim, 64) if heads == 4 else 2)
            at = np.concatenate([[0], np.cumsum(news)])
            q = rng.standard_normal((int(at[-1]), heads, dim), dtype=np.float32)
            top = c.table.shape[1] * 64
            s = dict(c=c, q=put(r, q.reshape(at[-1], -1)), table=put(r, c.table, np.int32), lengths=put(r, lengths, np.int32), starts=put(r, at, np.int32),
                     out=r.open_buffer((int(at[-1]), heads * dim)), work=r.open_buffer(r.kv4_attention_work(c.desc, len(lengths), int(at[-1]), max(news), top), np.uint8),
                     stream=torch.cuda.Stream(), graph=torch.cuda.CUDAGraph())

            def step(s=s, c=c, news=news, top=top):
                r.kv4_attention(c.desc, s["q"], c.pool, s["table"], s["lengths"], starts=s["starts"], max_new=max(news), max_length=top, out=s["out"], work=s["work"])
            step()
            r.sync()
            s["want"] = s["out"].numpy().copy()
            for b, m in enumerate(lengths):
                part = slice(c.first[b], c.first[b + 1])
                want = ref.attention(q[at[b]:at[b + 1]], c.k[part], c.v[part], m, c.desc.scale)
                np.testing.assert_allclose(s["want"][at[b]:at[b + 1]].reshape(want.shape), want, rtol=0, atol=bound(c, q, m))
            L.check(r.ctx, r.lib.caten_b200_set_stream(r.ctx, s["stream"].cuda_stream))
            with torch.cuda.graph(s["graph"], stream=s["stream"], capture_error_mode="thread_local"):
                step()
            L.check(r.ctx, r.lib.caten_b200_set_stream(r.ctx, None))
            L.check(r.ctx, r.lib.caten_b200_memset(r.ctx, s["out"].ptr, 0, s["out"].nbytes))
            sets.append(s)
        r.sync()
        for _ in range(5):
            for s in sets:
                with torch.cuda.stream(s["stream"]):
                    s["graph"].replay()
        torch.cuda.synchronize()
        for s in sets:
            np.testing.assert_array_equal(s["out"].numpy(), s["want"])
            del s["graph"]
    finally:
        r.close()


def plain_beam_search(logits_of, prompt, beams, steps, eos):
    """[(tokens, score)] by beam search on the host, and the smallest gap between the last value taken and the first left."""
    hyps, gap = [(list(prompt), 0.0, False)], np.inf
    for _ in range(steps):
        cand = []
        for i, (t, s, end) in enumerate(hyps):
            if end:
                cand.append((s, i, eos))
                continue
            x = logits_of(t).astype(np.float64)
            lp = x - x.max() - np.log(np.exp(x - x.max()).sum())
            cand += [(s + lp[j], i, int(j)) for j in np.argsort(-lp)[:beams + 1]]
        cand.sort(key=lambda c: -c[0])
        values = [c[0] for c in cand[:beams + 1]]
        gap = min([gap] + [a - b for a, b in zip(values, values[1:])])
        hyps = [(hyps[i][0] + [j], s, hyps[i][2] or j == eos) for s, i, j in cand[:beams]]
    return hyps, gap


@pytest.mark.parametrize("wtype,eos", [("f32", -1), ("q8_0", 5)])
def test_beam_search_of_gpt2(rt, wtype, eos):
    """`beam_search` (caches moved with their hypotheses, everything on the device) against a search on the host that reads every hypothesis anew."""
    from caten_b200.gpt2 import GPT2, gpt2_beam_search, gpt2_generate
    p = S.GPT2Params(n_layers=3, n_heads=2, dim=128, vocab_size=1003)
    sd = S.synth_state_dict(p, wtype, seed=4, max_seq_len=32, trivial_affine=False, weight_std=0.12)
    one = GPT2(rt, p, sd, max_seq_len=32, batch=1)

    def logits_of(tokens):
        one.forward([tokens], len(tokens), 0)
        return one.logits()[0]
    prompts = S.synth_prompts(2, 6, p.vocab_size, seed=3)
    if eos >= 0:   # an id that the search does meet: the likeliest third token of the first prompt
        eos = int(plain_beam_search(logits_of, prompts[0].tolist(), 1, 3, -1)[0][0][0][-1])
    beams, steps = 4, 10
    m = GPT2(rt, p, sd, max_seq_len=32, batch=2 * beams)
    tokens, scores = gpt2_beam_search(m, prompts, beams, steps, eos)
    assert tokens.shape == (2, beams, 16) and (np.diff(scores, axis=1) <= 0).all()
    for g in range(2):
        want, gap = plain_beam_search(logits_of, prompts[g].tolist(), beams, steps, eos)
        assert gap > 1e-5, "the search's choices are too close to compare"
        np.testing.assert_array_equal(tokens[g], np.array([h[0] for h in want]))
        np.testing.assert_allclose(scores[g], [h[1] for h in want], rtol=0, atol=2e-3)
    m.close()
    one.close()
    # one beam is greedy; no step returns the prompt
    m = GPT2(rt, p, sd, max_seq_len=32, batch=2)
    np.testing.assert_array_equal(gpt2_beam_search(m, prompts, 1, 8)[0][:, 0], gpt2_generate(m, prompts, 8))
    t, s = gpt2_beam_search(m, prompts[:1], 2, 0)
    np.testing.assert_array_equal(t, np.repeat(prompts[:1][:, None], 2, 1))
    with pytest.raises(ValueError):
        gpt2_beam_search(m, prompts, 3, 2)
    m.close()
