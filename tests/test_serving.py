"""CPU tests of the serving operators' boundary: what the entry points refuse (arguments are checked before the context is touched, so no
GPU is needed), where the cache's values lie, and the plain statements that the GPU tests compare with."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from oracle import serving_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from caten_b200 import _lib, build
    build.build()
    return _lib.load()


def desc(**kw):
    from caten_b200 import _lib as L
    d = dict(heads=8, kv_heads=4, dim=64, type=L.Q4_0, page=32, scale=0.125, pages=10)
    d.update(kw)
    return L.Kv4Desc(**d)


def refused(lib, rc, *words):
    from caten_b200 import _lib as L
    said = lib.caten_b200_last_error(None).decode()
    assert rc in (L.EINVAL, L.EUNSUPPORTED, -1) and all(w in said for w in words), (rc, said)


A = 1 << 20   # an aligned address that is never followed


def test_descriptions_that_are_refused(lib):
    for kw, word in ((dict(dim=80), "heads of 80"), (dict(dim=32), "heads of 32"), (dict(page=24), "pages of 24"), (dict(page=0), "pages of 0"), (dict(type=8), "type 8"),
                     (dict(heads=6), "6 heads"), (dict(kv_heads=0), "heads"), (dict(pages=0), "0 pages"), (dict(pages=1 << 27), "32-bit")):
        d = desc(**kw)
        refused(lib, lib.caten_b200_kv4_nbytes(C.byref(d)), word)
        refused(lib, lib.caten_b200_kv4_store(None, C.byref(d), A, A, A, 256, A, 1), word)
        refused(lib, lib.caten_b200_kv4_load(None, C.byref(d), A, A, 1, A, A, 256), word)
        refused(lib, lib.caten_b200_kv4_attention(None, C.byref(d), A, 512, A, A, 4, A, None, 1, 1, 1, 64, A, A), word)
    refused(lib, lib.caten_b200_kv4_nbytes(None), "NULL")


def test_pool_sizes(lib):
    assert lib.caten_b200_kv4_nbytes(C.byref(desc())) == 10 * 32 * 4 * 2 * 64 * 18 // 32
    assert lib.caten_b200_kv4_nbytes(C.byref(desc(type=3, dim=192))) == 10 * 32 * 4 * 2 * 192 * 20 // 32


def test_rows_that_are_refused(lib):
    d = desc()
    for bad in ((None, A, A, 256, A, 1), (A, None, A, 256, A, 1), (A, A, None, 256, A, 1), (A, A, A, 256, None, 1)):
        refused(lib, lib.caten_b200_kv4_store(None, C.byref(d), *bad), "NULL")
    refused(lib, lib.caten_b200_kv4_store(None, C.byref(d), A, A, A, 255, A, 1), "ld=255")
    refused(lib, lib.caten_b200_kv4_store(None, C.byref(d), A + 8, A, A, 256, A, 1), "16 bytes")
    refused(lib, lib.caten_b200_kv4_store(None, C.byref(d), A, A + 2, A, 256, A, 1), "misaligned")
    refused(lib, lib.caten_b200_kv4_store(None, C.byref(d), A, A, A, 256, A, -1), "-1 tokens")
    refused(lib, lib.caten_b200_kv4_load(None, C.byref(d), A, A, 1 << 31, A, A, 256), "tokens")
    refused(lib, lib.caten_b200_kv4_store(None, C.byref(d), A, A, A, 256, A, 1), "ctx is NULL")   # all else is in order


def test_attention_calls_that_are_refused(lib):
    d = desc()
    call = lambda **k: lib.caten_b200_kv4_attention(None, C.byref(d), *[dict(q=A, ldq=512, pool=A, table=A, max_pages=4, lengths=A, starts=A, batch=2, rows=5,   # noqa: E731
                                                                             max_new=3, max_length=128, out=A, work=A, **{})[n] if n not in k else k[n]
                                                                        for n in ("q", "ldq", "pool", "table", "max_pages", "lengths", "starts", "batch", "rows", "max_new",
                                                                                  "max_length", "out", "work")])
    refused(lib, call(), "ctx is NULL")
    for n in ("q", "pool", "table", "lengths", "out", "work"):
        refused(lib, call(**{n: None}), "NULL argument")
    refused(lib, call(ldq=511), "ldq=511")
    refused(lib, call(max_length=129), "lengths up to 129")
    refused(lib, call(max_pages=0), "tables of 0")
    refused(lib, call(starts=None), "without starts")
    refused(lib, call(starts=None, rows=2), "without starts")
    refused(lib, call(max_new=0), "bad shape")
    refused(lib, call(rows=-1), "bad shape")
    refused(lib, call(pool=A + 4), "16 bytes")
    refused(lib, call(work=A + 4), "16 bytes")
    refused(lib, call(out=A + 2), "misaligned")
    assert lib.caten_b200_kv4_attention_work(C.byref(d), 2, 5, 3, 128) >= 16
    refused(lib, lib.caten_b200_kv4_attention_work(C.byref(d), 2, 5, 0, 128), "bad shape")


def test_page_plans_that_are_refused(lib):
    call = lambda *k: lib.caten_b200_kv_pages(None, *k)   # noqa: E731
    good = [A, A, 3, 16, A, 4, A, 100, A, A, A, 50]
    refused(lib, call(*good), "ctx is NULL")
    for i in (0, 1, 4, 6, 8, 9, 10):
        bad = list(good)
        bad[i] = None
        refused(lib, call(*bad), "NULL argument")
    for i, v in ((2, -1), (3, 0), (5, 0), (7, 0), (7, 1 << 28), (11, -1), (11, 1 << 31), (5, 1 << 28)):
        bad = list(good)
        bad[i] = v
        refused(lib, call(*bad), "kv_pages")
        assert "ctx" not in lib.caten_b200_last_error(None).decode()


def test_beam_calls_that_are_refused(lib):
    work = lib.caten_b200_beam_select_work
    assert work(2, 4, 50257, 8) > 0 and work(0, 4, 50257, 8) >= 0
    for bad in ((2, 33, 100, 4), (2, 4, 100, 33), (2, 4, 0, 4), (2, 0, 100, 4), (-1, 4, 100, 4), (2, 4, 100, 0), (65536, 1, 100, 1), (1 << 60, 32, 100, 1), (2, 4, 1 << 30, 4)):
        refused(lib, work(*bad), "beam_select")
    call = lambda **k: lib.caten_b200_beam_select(None, *[k.get(n, v) for n, v in dict(x=A, s=A, e=A, batch=2, beams=4, V=100, eos=5, keep=4, os=A, op=A, ot=A, oe=A, w=A).items()])   # noqa: E731
    refused(lib, call(), "ctx is NULL")
    refused(lib, call(e=None, oe=None, eos=-1), "ctx is NULL")
    for n in ("x", "s", "os", "op", "ot", "w"):
        refused(lib, call(**{n: None}), "NULL argument")
    refused(lib, call(eos=100), "eos=100")
    refused(lib, call(eos=-1), "need an eos")
    refused(lib, call(ot=A + 4), "misaligned")
    refused(lib, call(x=A + 2), "misaligned")
    states = lambda *p: (C.c_void_p * len(p))(*p)   # noqa: E731
    move = lambda st, n, *k: lib.caten_b200_beam_reorder(None, st, n, *k)   # noqa: E731
    refused(lib, move(states(A), 1, A, 2, 4, 3, 1024, 256), "ctx is NULL")
    refused(lib, move(states(A), 1, A, 2, 33, 3, 1024, 256), "33 beams")
    refused(lib, move(states(A), 1, A, 2, 4, 3, 1024, 1028), "bad shape")
    refused(lib, move(states(A), 1, A, 2, 4, 3, 1024, 258), "multiples of 4")
    refused(lib, move(states(None), 1, A, 2, 4, 3, 1024, 256), "state 0")
    refused(lib, move(states(A, A + 2), 2, A, 2, 4, 3, 1024, 256), "state 1")
    refused(lib, move(states(A), 1, None, 2, 4, 3, 1024, 256), "NULL")
    refused(lib, move(states(A), 1, A, 65536, 4, 3, 1024, 256), "bad shape")
    refused(lib, move(states(A, A + 8 * 3 * 1024 - 16), 2, A, 2, 4, 3, 1024, 256), "overlap")
    refused(lib, move(states(A, 5 * A, A), 3, A, 2, 4, 3, 1024, 256), "overlap")
    paged = lambda **k: lib.caten_b200_beam_reorder_pages(None, *[k.get(n, v) for n, v in dict(pool=A, pages=9, nb=1024, table=A, mp=4, lens=A, page=16, par=A, groups=2, beams=4).items()])   # noqa: E731
    refused(lib, paged(), "ctx is NULL")
    for n in ("pool", "table", "lens", "par"):
        refused(lib, paged(**{n: None}), "NULL argument")
    refused(lib, paged(nb=1000), "multiple of 16")
    refused(lib, paged(beams=40), "40 beams")
    refused(lib, paged(mp=65536), "bad shape")
    refused(lib, paged(pool=A + 8), "16 bytes")


def test_layout_is_the_stated_one(tmp_path):
    """The index arithmetic that the kernels use (csrc/kv4_layout.h, as plain C++): every value has a place of its own, the stated one, inside its
    page; page numbers outside the pool are told apart."""
    src = tmp_path / "layout.cpp"
    src.write_text('#include <cstdio>\n#include <initializer_list>\n#include "kv4_layout.h"\nusing namespace cb;\nint main() {\n'
                   '  for (int q41 = 0; q41 < 2; ++q41) for (int dim = 64; dim <= 256; dim += 64) {\n'
                   '    Kv4Shape s = {3, dim, q41, 32, 7};\n'
                   '    printf("s %d %d %d %lld %lld\\n", q41, dim, kv4_part_bytes(s), (long long)kv4_page_bytes(s), (long long)kv4_tile_at(s, 5, 2, 17));\n'
                   '    for (int t = 0; t < 16; ++t) for (int j = 0; j < dim; ++j) printf("c %d %d\\n", kv4_k_byte(t, j), kv4_v_byte(t, j));\n'
                   '    for (int t = 0; t < 16; ++t) for (int b = 0; b < dim / 32; ++b) printf("h %d\\n", kv4_scale_index(t, b, dim));\n'
                   '  }\n  Kv4Shape s = {3, 64, 0, 32, 7};\n'
                   '  for (long long p : {-1ll, 0ll, 6ll, 7ll, 1ll << 31, -(1ll << 31)}) printf("p %d\\n", (int)kv4_page_ok(s, p));\n'
                   '  Kv4Shape far = {8, 128, 1, 128, 1 << 20};\n  printf("f %lld\\n", (long long)kv4_tile_at(far, (1 << 20) - 1, 7, 127));\n}\n')
    exe = tmp_path / "layout"
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "caten_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    lines = [x.split() for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()]
    at = 0
    for q41 in (0, 1):
        for dim in (64, 128, 192, 256):
            part = dim * (10 if q41 else 9)
            assert lines[at] == ["s", str(q41), str(dim), str(part), str(3 * 2 * 2 * part), str(5 * 12 * part + (2 * 2 + 1) * 2 * part)]
            codes = np.array([[int(a), int(b)] for _, a, b in lines[at + 1:at + 1 + 16 * dim]]).reshape(16, dim, 2)
            halves = np.array([int(a) for _, a in lines[at + 1 + 16 * dim:at + 1 + 16 * dim + dim // 2]])
            assert (np.bincount(codes[..., 0].ravel(), minlength=8 * dim) == 2).all() and (np.bincount(codes[..., 1].ravel(), minlength=8 * dim) == 2).all()
            assert (codes[:, 0::2] == codes[:, 1::2]).all()   # an odd code beside its even one
            assert sorted(halves) == list(range(dim // 2))
            # one token by the plain statement: its codes and scales lie where the arithmetic says
            pool = np.zeros((7, 3 * 2 * 2 * part), np.uint8)
            k = np.linspace(-1, 1, dim, dtype=np.float32)
            ref.put(pool, 32, 3, dim, bool(q41), 5 * 32 + 16 + 11, 2, k, k[::-1].copy())
            base = (2 * 2 + 1) * 2 * part
            for which, x in ((0, k), (1, k[::-1].copy())):
                code, d, _ = ref.blocks(x.reshape(-1, 32), bool(q41))
                for j in range(dim):
                    assert pool[5, base + which * part + codes[11, j, which]] >> j % 2 * 4 & 15 == code[j // 32, j % 32]
                for b in range(dim // 32):
                    place = base + which * part + 8 * dim + 2 * halves[11 * (dim // 32) + b]
                    assert pool[5, place:place + 2].tobytes() == d[b].tobytes()
            at += 1 + 16 * dim + dim // 2
    assert [x[1] for x in lines[at:at + 6]] == ["0", "1", "1", "0", "0", "0"]
    assert int(lines[at + 6][1]) == ((1 << 20) - 1) * 8 * 8 * 2560 + (7 * 8 + 7) * 2560   # beyond 32 bits


def test_attention_workspace_is_enough_for_every_smaller_call(lib, tmp_path):
    """A host allocates once, for its largest turn.  The plan that a call is cut by (csrc/kv4_plan.h, as plain C++) needs no more than the stated bytes,
    whatever smaller sizes it is made for, and the entry point says what that arithmetic says."""
    src = tmp_path / "plan.cpp"
    src.write_text('''#include <cmath>
#include <cstdio>
#include <random>
#include "kv4_plan.h"
using namespace cb;
int main() {
  std::mt19937_64 rng(7);
  auto of = [&](double lo, double hi) { return (int64_t)std::exp(std::uniform_real_distribution<double>(std::log(lo), std::log(hi + 0.99))(rng)); };
  auto some = [&](int64_t hi) { return hi < 2 || rng() % 4 == 0 ? hi : std::min(hi, of(1, (double)hi)); };
  int64_t parts[4] = {0, 0, 0, 0}, smaller_needs_more = 0;
  for (int i = 0; i < 300000; ++i) {
    const Kv4Heads h = {(int)(64 * (1 + rng() % 4)), (int)of(1, 50), of(1, 16)};
    const int64_t batch = of(1, 3000), max_new = rng() % 2 ? 1 : of(1, 2000), max_length = of(1, 300000), rows = some(batch * max_new);
    Kv4Plan p, q;
    if (!kv4_plan_of(h, batch, rows, max_new, max_length, &p)) continue;
    const int64_t bound = kv4_work_bound(h, batch, max_new, max_length);
    const int64_t b = some(batch), n = some(max_new), l = some(max_length), r = some(std::min(rows, b * n));
    if (!kv4_plan_of(h, b, r, n, l, &q)) { printf("refused\\n"); return 1; }
    for (const Kv4Plan *x : {&p, &q}) {
      if (kv4_plan_bytes(*x, h.dim) > bound) {
        printf("dim %d heads %d x %lld: %lld bytes for batch %lld rows %lld new %lld length %lld (tiles of %d), %lld stated for %lld %lld %lld\\n", h.dim, h.kv_heads, (long long)h.group,
               (long long)kv4_plan_bytes(*x, h.dim), (long long)b, (long long)r, (long long)n, (long long)l, x->tile_rows, (long long)bound, (long long)batch, (long long)max_new, (long long)max_length);
        return 1;
      }
      if (x->parts > 1) ++parts[x->tile_rows == 1 ? 0 : x->tile_rows == K2_ROWS ? 1 : x->tile_rows == K4_ROWS ? 2 : 3];
    }
    smaller_needs_more += kv4_plan_bytes(q, h.dim) > kv4_plan_bytes(p, h.dim);
    if (kv4_work_bound(h, b, n, l) > bound) { printf("not monotonic\\n"); return 1; }
  }
  printf("%lld %lld %lld %lld %lld\\n", (long long)parts[0], (long long)parts[1], (long long)parts[2], (long long)parts[3], (long long)smaller_needs_more);
  for (int64_t batch : {1, 7, 300}) for (int64_t n : {1, 2, 40}) for (int64_t l : {1, 700, 5000}) {
    Kv4Plan p;
    kv4_plan_of({128, 8, 2}, batch, batch * n, n, l, &p);
    printf("%lld\\n%lld\\n", (long long)kv4_work_bound({128, 8, 2}, batch, n, l), (long long)std::max<int64_t>(16, kv4_plan_bytes(p, 128)));
  }
}
''')
    exe = tmp_path / "plan"
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", os.path.join(ROOT, "caten_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
    seen, *said = r.stdout.splitlines()
    assert min(map(int, seen.split())) > 100   # every kernel with parts; smaller calls that need more than the larger one itself
    d = desc(dim=128, heads=16, kv_heads=8)
    for entry, want in ((lib.caten_b200_kv4_attention_work, said[::2]), (lib.caten_b200_kv4_attention_call_work, said[1::2])):
        assert [entry(C.byref(d), b, b * n, n, ln) for b in (1, 7, 300) for n in (1, 2, 40) for ln in (1, 700, 5000)] == [int(x) for x in want]
    refused(lib, lib.caten_b200_kv4_attention_call_work(C.byref(d), 2, 5, 0, 128), "bad shape")


def test_selection_workspace_is_enough_for_every_smaller_call(lib):
    """A host allocates once, for its largest batch, and calls with what is left of it."""
    work = lib.caten_b200_beam_select_work
    for V in (50257, 1003, 130001):
        for beams, keep in ((7, 16), (1, 1), (32, 32)):
            said = [work(batch, beams, V, keep) for batch in range(1, 400)]
            assert said == sorted(said)
            for batch, n in zip(range(1, 400), said):   # in chunks of 2048 logits as long as those of 8192 are fewer than 148, and the request's lists at most 4096
                few = batch * beams * -(-(V + 3) // 8192) < 148 and beams * -(-(V + 3) // 2048) <= 4096
                assert n >= 8 * (keep + 1) * batch * beams * -(-(V + 3) // (2048 if few else 8192))
    rng = np.random.Generator(np.random.PCG64(9))
    for _ in range(3000):
        large = [int(np.exp(rng.uniform(0, np.log(x)))) for x in (500, 32, 1040384, 32)]
        small = [int(rng.integers(1, x + 1)) for x in large]
        assert work(*small) <= work(*large)


def test_the_bound_on_attention_tells_mistakes():
    """The bound that the GPU tests compare attention with, on their inputs: every row is beyond it if a token that it sees is left out, be it the last, the
    first or one at a border, or if it sees one token more; some row of a call is if q, or p, is held in 16 bits."""
    for length in (65, 257, 1200, 5000):
        for heads, kv, dim, news in ((2, 1, 64, 1), (4, 4, 128, 4), (1, 1, 64, 1), (3, 1, 256, 1), (8, 1, 64, 12), (2, 2, 64, 60)):
            rng = np.random.Generator(np.random.PCG64([length, heads, dim]))
            scale, group = dim ** -0.5, heads // kv
            k, v, q = ref.few_tokens(rng, length, kv, dim, heads, news, scale)
            q = q[-4:]   # (the rest is the same)
            for q41 in (False, True):
                ks, vs = (ref.values(x.reshape(length, -1), q41).reshape(k.shape) for x in (k, v))
                kp, vp = (ref.parts(x.reshape(length, -1), q41).reshape(k.shape) for x in (k, v))
                want, tol = ref.attention(q, ks, vs, length, scale), ref.attention_bound(q, ks, kp, vp, length, scale)
                off = lambda x: (np.abs(x - want) > tol).any(2)   # noqa: E731
                assert (tol < 2e-4 * np.abs(vs).max()).all()
                for left_out in (0, 16, 63, 64, length // 2, length // 64 * 64 - 1):
                    there = np.arange(length) != left_out
                    if left_out < length - len(q):
                        assert off(ref.attention(q, ks[there], vs[there], length - 1, scale)).all(), left_out
                shorter = np.concatenate([q, q[-1:]])   # a row fewer behind each: row i sees a token less
                assert off(ref.attention(shorter, ks, vs, length, scale)[:-1]).all()
                if len(q) > 1:                          # and one more
                    assert off(np.concatenate([ref.attention(q[:-1], ks, vs, length, scale), want[-1:]]))[:-1].all()
                assert off(ref.attention(q.astype(np.float16).astype(np.float32), ks, vs, length, scale)).any()
                low = np.empty_like(want)
                for i in range(len(q)):
                    sees = length - len(q) + i + 1
                    for h in range(heads):
                        s = ks[:sees, h // group].astype(np.float64) @ q[i, h].astype(np.float64) * scale
                        p = np.exp(s - s.max())
                        low[i, h] = p.astype(np.float16).astype(np.float64) @ vs[:sees, h // group] / p.sum()
                assert off(low).any() or news > 4   # (with more tokens to share a row's probability, their roundings are lost among them)


def test_copies_of_a_ring_land_before_it_is_given_up(tmp_path):
    """What the attention kernels wait for when a wait ran out (csrc/kv4_ring.h, as plain C++), at every step of rings of every length: the copies that
    are under way then, each once with the parity of its own step, and no others (a wait for one that was never asked for would last to its limit)."""
    src = tmp_path / "ring.cpp"
    src.write_text('#include <cstdio>\n#include "kv4_ring.h"\nint main() {\n  for (int count = 1; count < 9; ++count) {\n    int stage = 0;\n    unsigned phase = 0;\n'
                   '    for (int k = 0; k < count; ++k) {\n      printf("%d %d :", count, k);\n'
                   '      cb::ring_land(stage, phase, k + 1 < count, [](int s, unsigned p) { printf(" %d %u", s, p); });\n      puts("");\n'
                   '      phase ^= stage;\n      stage ^= 1;\n    }\n  }\n}\n')
    exe = tmp_path / "ring"
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "caten_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    said = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    want = []
    for count in range(1, 9):
        for k in range(count):   # steps before k were used, and for each of them the step two further on was asked for
            under_way = [j for j in range(count) if j < 2 or j - 2 < k]
            want.append(f"{count} {k} : " + " ".join(f"{j % 2} {j // 2 % 2}" for j in under_way if j >= k))
    assert said == want


def test_plain_blocks_are_those_of_the_file_format():
    """At values that are not next to a border: the codes of the GGUF package's quantisers, which work in fp32."""
    from gguf import quants
    rng = np.random.Generator(np.random.PCG64(3))
    x = rng.standard_normal((200, 32), dtype=np.float32)
    for q4_1, kind in ((False, quants.Q4_0), (True, quants.Q4_1)):
        np.testing.assert_array_equal(ref.values(x, q4_1), kind.dequantize_blocks(kind.quantize_blocks(x.copy())))


def test_runtime_refuses_buffers_that_do_not_fit(lib):
    """The Python methods' own checks, on buffers without memory."""
    from caten_b200 import _lib as L
    from caten_b200.runtime import B200Buffer, B200Runtime
    rt = B200Runtime.__new__(B200Runtime)
    rt.lib, rt.ctx = lib, None
    buf = lambda kind, *shape: B200Buffer(rt, A, shape, kind, owned=False)   # noqa: E731
    f, i, u = np.float32, np.int32, np.uint8
    out = lambda n, kind=i: (buf(f, 2, n), buf(kind, 2, n), buf(np.int64, 2, n), buf(u, 2, n))   # noqa: E731
    work = buf(u, 1 << 20)
    for bad in (dict(logits=buf(f, 7, 50)), dict(scores=buf(np.float64, 2, 4)), dict(ended=buf(u, 2, 3)), dict(out=out(5)), dict(out=out(4, f)), dict(work=buf(u, 8))):
        a = dict(logits=buf(f, 8, 50), scores=buf(f, 2, 4), keep=4, ended=buf(u, 2, 4), eos=3, out=out(4), work=work)
        a.update(bad)
        with pytest.raises(ValueError):
            rt.beam_select(**a)
    d = desc()
    pool = buf(u, 10, lib.caten_b200_kv4_nbytes(C.byref(d)) // 10)
    with pytest.raises(ValueError):
        rt.kv4_store(d, pool, buf(f, 5, 256), buf(f, 5, 255), buf(i, 5))
    with pytest.raises(ValueError):
        rt.kv4_store(d, buf(u, 100), buf(f, 5, 256), buf(f, 5, 256), buf(i, 5))
    for bad in (dict(q=buf(f, 2, 511)), dict(lengths=buf(np.int64, 2)), dict(table=buf(i, 3, 4)), dict(starts=buf(i, 2)), dict(out=buf(f, 2, 511)), dict(pool=buf(u, 10, 10))):
        a = dict(desc=d, q=buf(f, 2, 512), pool=pool, table=buf(i, 2, 4), lengths=buf(i, 2), out=buf(f, 2, 512), work=work)
        a.update(bad)
        with pytest.raises(ValueError):
            rt.kv4_attention(**a)
    with pytest.raises(ValueError):
        rt.beam_reorder([buf(f, 8, 3, 10, 64)], buf(i, 2, 4), 11)
    with pytest.raises(ValueError):
        rt.beam_reorder([buf(f, 8, 3, 10, 64), buf(f, 8, 3, 11, 64)], buf(i, 2, 4), 5)
    with pytest.raises(ValueError):
        rt.kv_pages(buf(i, 3), buf(i, 4), 16, buf(i, 3, 4), buf(i, 9), buf(i, 4), buf(i, 4), buf(i, 8))
    with pytest.raises(L.B200Error):
        rt.kv4_attention_work(desc(dim=48), 1, 1, 1, 10)


def test_command_refuses_beams_it_cannot_have():
    from caten_b200.generate import main
    for bad in (["--beams", "33"], ["--beams", "-1"], ["--beams", "4", "--temperature", "1"]):
        with pytest.raises(SystemExit):
            main(["--model", "none", "--ids", "1"] + bad)


class HostRuntime:
    """The runtime calls of ``beam_search`` on host arrays, which are counted."""

    class Buffer:
        def __init__(self, rt, a):
            self.rt, self.a = rt, a
            rt.open.append(self)

        def view(self, at, shape):
            v = object.__new__(type(self))
            v.rt, v.a = self.rt, self.a.reshape(-1)[at:at + int(np.prod(shape))].reshape(shape)
            return v

        def numpy(self):
            return self.a

        def close(self):
            self.rt.open.remove(self)

    def __init__(self):
        self.open, self.selects = [], 0

    def open_buffer(self, shape, kind=np.float32):
        return self.Buffer(self, np.zeros(shape, kind))

    def transfer_from_array(self, a):
        return self.Buffer(self, a.copy())

    def beam_select_work(self, *sizes):
        return 8

    def beam_select(self, logits, scores, keep, ended=None, eos=-1, out=None, work=None):
        self.selects += 1
        for r, s in enumerate(scores.a):
            x = logits.reshape(len(scores.a), -1, logits.shape[-1])[r]
            for o, w in zip(out, ref.select(x, s, ended.a[r] if ended else np.zeros(len(s)), eos, keep)):
                o.a[r] = w

    def beam_reorder(self, states, parents, positions):
        for x in states:
            x[:] = x.reshape(len(parents.a), -1, x.shape[-1])[np.arange(len(parents.a))[:, None], parents.a].reshape(x.shape)


def host_model(batch, vocab=20, length=16, fails_at=None):
    """A model whose "cache" is the tokens that it has read, with logits that are a function of them."""
    from caten_b200.model import Model

    class Host(Model):
        def __init__(self):
            self.rt, self.batch, self.vocab_size, self.max_seq_len, self.read, self.steps = HostRuntime(), batch, vocab, length, np.zeros((batch, length), np.int64), 0

        def _step(self, tokens, n):
            self.steps += 1
            if self.steps == fails_at:
                raise RuntimeError("a step that fails")
            self.read[:, n:n + tokens.shape[1]] = tokens
            self.logits_now = np.stack([np.random.Generator(np.random.PCG64(list(r[:n + tokens.shape[1]]))).standard_normal(vocab).astype(np.float32) * 3 for r in self.read])
            return self.logits_now.argmax(1)

        def _step_device(self, ids, s, n, out):
            out.a[:] = self._step(ids.a.reshape(batch, s), n)

        def _logits_buffer(self):
            return self.logits_now

        def _caches(self):
            return [self.read]
    return Host()


def test_beam_search_takes_a_prompt_a_group():
    """On a model of host arrays: each prompt's hypotheses are its own, and prompts that are not one a group are refused, not cut anew."""
    from caten_b200.model import beam_search
    prompts = np.array([[1, 2, 3], [4, 5, 6]])
    both = beam_search(host_model(6), prompts, 3, 5)
    for g in range(2):
        one = beam_search(host_model(3), prompts[g], 3, 5)
        np.testing.assert_array_equal(both[0][g], one[0][0])
        np.testing.assert_array_equal(both[1][g], one[1][0])
    assert (both[0][:, :, :3] == prompts[:, None]).all()
    for bad in (np.arange(8).reshape(4, 2), np.arange(6).reshape(1, 6), np.arange(6), np.arange(12).reshape(2, 3, 2)):
        m = host_model(6)
        with pytest.raises(ValueError):
            beam_search(m, bad, 3, 5)
        assert m.steps == 0


def test_beam_search_closes_what_it_opened():
    """Whether it ends, is refused (before the prompt is read), or a step or a selection fails on the way."""
    from caten_b200 import _lib as L
    from caten_b200.model import beam_search
    prompts = np.array([[1, 2, 3], [4, 5, 6]])
    m = host_model(6)
    beam_search(m, prompts, 3, 5, eos=7)
    assert not m.rt.open and m.steps == 5
    for steps in (1, 2, 4):
        m = host_model(6, fails_at=steps)
        with pytest.raises(RuntimeError):
            beam_search(m, prompts, 3, 5)
        assert not m.rt.open and m.steps == steps
    m = host_model(6)
    m.rt.beam_select = lambda *a, **k: (_ for _ in ()).throw(L.B200Error(L.EUNSUPPORTED, "no"))
    with pytest.raises(L.B200Error):
        beam_search(m, prompts, 3, 5)
    assert not m.rt.open
    for bad in (dict(eos=20), dict(max_length=15)):          # 20 ids; 3 + 14 positions of 16
        m = host_model(6)
        with pytest.raises(ValueError):
            beam_search(m, prompts, 3, **{"max_length": 5, **bad})
        assert m.steps == 0 and not m.rt.open
    m = host_model(6)
    beam_search(m, prompts, 3, 14)                           # the last one's logits need no position
    m = host_model(40)
    m.rt.beam_select_work = lambda *a: (_ for _ in ()).throw(L.B200Error(L.EUNSUPPORTED, "40 beams"))
    with pytest.raises(L.B200Error):
        beam_search(m, prompts[:1], 40, 3)
    assert m.steps == 0


def test_beam_search_moves_states_by_the_models_own_call():
    """``Model.reorder`` is what a subclass with other states overrides."""
    from caten_b200.model import beam_search
    m, moved = host_model(3), []
    own = m.reorder
    m.reorder = lambda parents, positions: (moved.append(positions), own(parents, positions))
    out = beam_search(m, [1, 2, 3], 3, 5)
    assert moved == [3, 4, 5, 6]
    np.testing.assert_array_equal(out[0], beam_search(host_model(3), [1, 2, 3], 3, 5)[0])


def test_command_refuses_beams_over_models_whose_states_do_not_move(tmp_path, capsys):
    """Said by the command before anything is loaded."""
    from caten_b200.generate import main
    for name in ("Binusun", "Goselix"):
        (tmp_path / "config.json").write_text('{"architecture": "%s"}' % name)
        with pytest.raises(SystemExit) as e:
            main(["--model", str(tmp_path), "--ids", "1,2", "--beams", "2"])
        assert e.value.code == 2 and name in capsys.readouterr().err
