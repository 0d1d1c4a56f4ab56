"""K/V pages held in 8 bits (cj_kv8_append, cj_kv8_read, cj_kv8_attend) on the MI355X against the definition in 64 bits:
codes and scales exactly, attention within what f32 arithmetic allows (kv8_reference.attention says how that follows)."""
import ctypes
import math

import numpy as np
import pytest

from kv8_reference import BLOCK, PAGE, Cache, attention, normed, turned

pytestmark = pytest.mark.gpu

EPS = 1e-5
MARK = np.float32(-7.5)          # what untouched output rows hold


def say(*a):
    print(*a, flush=True)


def rope_table(hd, ctx):
    ang = np.arange(ctx)[:, None] * 10000.0 ** (-np.arange(0, hd, 2) / hd)
    return np.stack((np.cos(ang), np.sin(ang)), -1).astype(np.float32)


class Pages:
    """Two planes, a page table and the calls on them, with the 64-bit cache beside."""

    def __init__(self, gpu, heads, kv, hd, slots, slot_pages, pool=None, seed=0, ctx=None, garbage=True):
        self.gpu, self.L = gpu, gpu.native.lib()
        self.heads, self.kv, self.hd, self.slots, self.slot_pages = heads, kv, hd, slots, slot_pages
        self.pool = pool or slots * slot_pages + 3
        rng = np.random.default_rng(seed + 99)
        self.nbytes = self.L.cj_kv8_plane_bytes(self.pool, kv, hd)
        codes = self.pool * kv * PAGE * hd
        assert self.nbytes == codes + self.pool * kv * 16
        self.planes = []
        for _ in range(2):
            b = gpu.Buffer(self.nbytes)
            if garbage:   # codes at random and scales that are none: what no append wrote must not be seen
                img = rng.integers(0, 256, self.nbytes, dtype=np.uint8)
                img[codes:].view(np.float32)[:] = np.nan
                b.upload(img)
            self.planes.append(b)
        self.table = rng.permutation(self.pool)[:slots * slot_pages].reshape(slots, slot_pages).astype(np.int32)
        self.tab = gpu.Buffer.of(self.table)
        self.ctx = ctx or slot_pages * PAGE
        self.rope = rope_table(hd, self.ctx)
        self.rope_b = gpu.Buffer.of(self.rope)
        self.ref = Cache(kv, hd)
        self.status = gpu.Buffer.of(np.zeros(4, np.int32))

    def segs(self, segs):
        return self.gpu.Buffer.of(np.asarray(segs, np.int32).reshape(-1, 4))

    def stat(self):
        v = int(self.status.download(np.int32, 1)[0])
        self.status.zero()
        return v

    def append(self, segs, q, k, v, qw=None, kw=None, form=0, max_rows=None, in_place=False, model=True):
        """One call on a fused q|k|v row buffer; q's rotated rows, and the reference kept up with it."""
        H, KV, D = self.heads, self.kv, self.hd
        n = len(k)
        wide = (H + 2 * KV) * D + 4                       # rows apart by more than their width
        rows = np.full((n, wide), 3.0, np.float32)
        rows[:, :H * D], rows[:, H * D:(H + KV) * D] = q.reshape(n, -1), k.reshape(n, -1)
        rows[:, (H + KV) * D:(H + 2 * KV) * D] = v.reshape(n, -1)
        b = self.gpu.Buffer.of(rows)
        out = b if in_place else self.gpu.Buffer.of(np.full((n, H * D), MARK))
        stride = wide if in_place else H * D
        sb = self.segs(segs)
        w = [self.gpu.Buffer.of(x) if x is not None else None for x in (qw, kw)]
        self.gpu.native.check(self.L.cj_kv8_append(
            out.h, b.h, b.h + 4 * H * D, b.h + 4 * (H + KV) * D, self.planes[0].h, self.planes[1].h, w[0].h if w[0] else 0,
            w[1].h if w[1] else 0, self.rope_b.h, self.tab.h, sb.h, len(segs), max_rows or max(1, max(s[3] for s in segs)), n,
            self.ctx, self.pool, self.slots, self.slot_pages, H, KV, D, stride, wide, wide, int(kw is not None),
            ctypes.c_float(EPS), form, self.status.h), "append")
        got = out.download(np.float32, n * stride).reshape(n, stride)[:, :H * D].reshape(n, H, D)
        want = np.full((n, H, D), q if in_place else MARK, np.float64)
        if model:
            q64, k64, v64 = (x.astype(np.float64) for x in (q, k, v))
            if kw is not None:
                q64, k64 = normed(q64, qw.astype(np.float64), np.float64(np.float32(EPS)), form), \
                    normed(k64, kw.astype(np.float64), np.float64(np.float32(EPS)), form)
            for slot, pos, row, cnt in segs:
                want[row:row + cnt] = turned(q64[row:row + cnt], self.rope, pos)
                self.ref.append(slot, pos, turned(k64[row:row + cnt], self.rope, pos), v64[row:row + cnt])
        return got, want

    def read(self, segs, max_rows=None, n=None):
        n = n or max(s[2] + s[3] for s in segs)
        w = self.kv * self.hd
        outs = [self.gpu.Buffer.of(np.full((n, w + 8), MARK)) for _ in range(2)]
        sb = self.segs(segs)
        self.gpu.native.check(self.L.cj_kv8_read(
            outs[0].h, outs[1].h, self.planes[0].h, self.planes[1].h, self.tab.h, sb.h, len(segs),
            max_rows or max(1, max(s[3] for s in segs)), n, self.pool, self.slots, self.slot_pages, self.kv, self.hd, w + 8,
            self.status.h), "read")
        k, v = (o.download(np.float32, n * (w + 8)).reshape(n, w + 8) for o in outs)
        assert (k[:, w:] == MARK).all() and (v[:, w:] == MARK).all()
        return k[:, :w].reshape(n, self.kv, self.hd), v[:, :w].reshape(n, self.kv, self.hd)

    def attend(self, segs, q, window=0, scale=None, max_rows=None, max_count=None, bufs=None):
        H, D, n = self.heads, self.hd, len(q)
        scale = np.float32(1 / math.sqrt(D) if scale is None else scale)
        max_rows = max_rows or max(1, max(s[3] for s in segs))
        max_count = max_count or max(1, max(s[1] + s[3] for s in segs))
        need = self.L.cj_kv8_attend_bytes(len(segs), max_rows, max_count, H, self.kv, D, window)
        assert need >= 0, self.gpu.native.last_error()
        part = self.gpu.Buffer(max(16, need))
        out = self.gpu.Buffer.of(np.full((n, H * D + 4), MARK))
        qb, sb = self.gpu.Buffer.of(q.reshape(n, -1)), self.segs(segs)
        self.gpu.native.check(self.L.cj_kv8_attend(
            out.h, qb.h, self.planes[0].h, self.planes[1].h, self.tab.h, sb.h, part.h if need else 0, len(segs), max_rows, n,
            max_count, self.pool, self.slots, self.slot_pages, H, self.kv, D, H * D, H * D + 4, window, ctypes.c_float(scale),
            self.status.h), "attend")
        got = out.download(np.float32, n * (H * D + 4)).reshape(n, -1)
        assert (got[:, H * D:] == MARK).all()
        return got[:, :H * D].reshape(n, H, D), np.float64(scale)

    def check_attend(self, segs, q, window=0, **kw):
        got, scale = self.attend(segs, q, window, **kw)
        seen = np.zeros(len(q), bool)
        for slot, pos, row, cnt in segs:
            if not cnt:
                continue
            seen[row:row + cnt] = True
            want, tol = attention(q[row:row + cnt].astype(np.float64), self.ref.values(slot, "k", 0, pos + cnt),
                                  self.ref.values(slot, "v", 0, pos + cnt), pos, scale, window,
                                  self.ref.steps(slot, "v").repeat(BLOCK, 0))
            off = np.abs(got[row:row + cnt] - want)
            assert np.isfinite(got[row:row + cnt]).all(), (slot, pos, cnt)
            assert (off <= tol).all(), (slot, pos, cnt, float((off / tol).max()))
        assert (got[~seen] == MARK).all()
        return got

    def check_read(self):
        for slot, s in self.ref.slots.items():
            if not s["n"]:
                continue
            got = self.read([(slot, 0, 0, s["n"])])
            for name, x in zip("kv", got):
                want = self.ref.values(slot, name, 0, s["n"]).astype(np.float32)
                assert np.array_equal(x, want, equal_nan=True), (slot, name)


def rows_of(rng, n, heads, kv, hd, loud=1.0):
    q = rng.standard_normal((n, heads, hd)).astype(np.float32)
    k = (rng.standard_normal((n, kv, hd)) * loud).astype(np.float32)
    v = (rng.standard_normal((n, kv, hd)) * loud).astype(np.float32)
    return q, k, v


def near(got, want):
    """Rotated rows: one rounding to f32 of a value whose 64-bit form is off by far less."""
    return (np.abs(got - want) <= 2.0 ** -24 * 1.01 * np.abs(want) + 1e-37).all()


SHAPES = [(8, 2, 64), (32, 8, 128), (6, 6, 128), (40, 2, 64)]


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("norm,form", [(False, 0), (True, 0), (True, 1)])
def test_append_stores_the_codes_of_the_exact_values(gpu, heads, kv, hd, norm, form):
    say("kv8 append", heads, kv, hd, norm, form)
    rng = np.random.default_rng(heads * 7 + hd + 2 * norm + form)
    P = Pages(gpu, heads, kv, hd, 5, 4, seed=heads)
    w = [(1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) if norm else None for _ in range(2)]
    # first rows: whole blocks, odd ends, pages' ends, one row, none; rows 3 and 4 of the buffers are nobody's
    first = [(0, 0, 0, 3), (3, 0, 5, 64), (1, 0, 69, 0), (4, 0, 69, 130), (2, 0, 199, 17)]
    got, want = P.append(first, *rows_of(rng, 216, heads, kv, hd), *w, form)
    assert near(got, want) and (got[3:5] == MARK).all()
    # then rows from inside blocks and pages, decode rows and chunks together, in another order
    then = [(2, 17, 0, 1), (0, 3, 1, 61), (1, 0, 62, 1), (3, 64, 63, 1), (4, 130, 64, 126)]
    got, want = P.append(then, *rows_of(rng, 190, heads, kv, hd), *w, form)
    assert near(got, want)
    P.check_read()
    # rewinding drops what stood from there on
    P.append([(4, 100, 0, 2), (0, 16, 2, 5)], *rows_of(rng, 7, heads, kv, hd), *w, form, in_place=True)
    P.check_read()
    assert P.stat() == 0


@pytest.mark.parametrize("hd", [64, 128])
def test_blocks_that_fill_token_by_token_rescale_and_stay_within_a_step(gpu, hd):
    rng = np.random.default_rng(hd)
    P = Pages(gpu, 4, 2, hd, 2, 2, seed=3)
    given, grew, was = {0: [], 1: []}, 0, {}
    for t in range(70):
        q, k, v = rows_of(rng, 2, 4, 2, hd)
        loud = np.exp2(rng.uniform(-3, 6) if t % 5 == 0 else -3).astype(np.float32)
        v *= loud
        if t == 37:
            v[:] = 0
        for s in (0, 1):
            given[s].append(v[s].astype(np.float64))
        P.append([(1, t, 1, 1), (0, t, 0, 1)], q, k, v)
        for s in (0, 1):
            now = P.ref.steps(s, "v")[-1]
            grew += int((now > was[s]).sum()) if t % BLOCK else 0
            was[s] = now
    assert grew >= 16      # older codes were rescaled
    P.check_read()
    for s in (0, 1):
        x = np.stack(given[s])
        step = np.repeat(P.ref.steps(s, "v"), BLOCK, 0)[:70]
        assert (np.abs(P.ref.values(s, "v", 0, 70) - x) < step[..., None]).all()
    assert P.stat() == 0


def test_values_that_eight_bits_cannot_hold_poison_their_block_alone(gpu):
    rng = np.random.default_rng(5)
    P = Pages(gpu, 4, 2, 64, 4, 2)
    q, k, v = rows_of(rng, 160, 4, 2, 64)
    k[20, 1, 3] = np.nan               # slot 0, position 20, head 1
    v[40 + 33, 0, 63] = np.inf         # slot 1, position 33, head 0
    v[80 + 5, 1] = 3.0e38              # slot 2, position 5: beyond 127 x 2^63
    k[120:160] *= np.float32(1e-30)    # slot 3: nothing but values below the least step
    v[120:160] *= np.float32(2.0 ** 60)
    P.append([(s, 0, 40 * s, 40) for s in range(4)], q, k, v)
    assert P.stat() == 1
    kk, vv = P.read([(s, 0, 40 * s, 40) for s in range(4)])
    bad_k, bad_v = np.zeros((160, 2), bool), np.zeros((160, 2), bool)
    bad_k[16:32, 1] = bad_v[40 + 32:80, 0] = bad_v[80:96, 1] = True
    assert np.array_equal(np.isnan(kk).any(-1), bad_k) and np.array_equal(np.isnan(vv).any(-1), bad_v)
    assert (kk[120:] == 0).all() and np.isfinite(vv[120:]).all()
    # a poisoned block stays one when more is appended to it
    P.append([(1, 40, 0, 3)], *rows_of(rng, 3, 4, 2, 64), model=False)
    assert P.stat() == 1
    assert np.isnan(P.read([(1, 0, 0, 43)])[1][32:, 0]).all()
    # rows that attend it come out NaN, others do not
    got, _ = P.attend([(0, 10, 0, 30), (1, 0, 30, 40), (2, 39, 70, 1), (3, 0, 71, 40)], rows_of(rng, 111, 4, 2, 64)[0])
    nan = np.isnan(got).all(-1)
    assert np.array_equal(np.isnan(got).any(-1), nan)
    want = np.zeros((111, 4), bool)
    want[30 - 24:30, 2:] = True        # slot 0 from position 16 on
    want[30 + 32:70, :2] = True        # slot 1 from position 32 on
    want[70, 2:] = True                # slot 2
    assert np.array_equal(nan, want)


def test_a_row_that_is_not_finite_stays_alone(gpu):
    rng = np.random.default_rng(15)
    for rows in (1, 3, 40):
        P = Pages(gpu, 8, 2, 64, 2, 4)
        P.append([(0, 0, 0, 150), (1, 0, 150, 150)], *rows_of(rng, 300, 8, 2, 64))
        q = rows_of(rng, 2 * rows, 8, 2, 64)[0]
        clean = P.check_attend([(0, 150 - rows, 0, rows), (1, 150 - rows, rows, rows)], q)
        q[rows, 3, 5], q[rows - 1, 6, 0] = np.nan, np.inf
        got, _ = P.attend([(0, 150 - rows, 0, rows), (1, 150 - rows, rows, rows)], q)
        bad = np.zeros((2 * rows, 8), bool)
        bad[rows, 3] = bad[rows - 1, 6] = True
        assert np.isnan(got[bad]).all()
        assert np.array_equal(got[~bad], clean[~bad])


def test_refused_segments_are_skipped_and_reported(gpu):
    rng = np.random.default_rng(8)
    heads, kv, hd = 8, 2, 64
    P = Pages(gpu, heads, kv, hd, 4, 2)
    P.append([(s, 0, 30 * s, 30) for s in range(4)], *rows_of(rng, 120, heads, kv, hd))
    assert P.stat() == 0
    q, k, v = rows_of(rng, 16, heads, kv, hd)
    good = (2, 30, 0, 3)
    for bad in [(-1, 0, 4, 2), (4, 0, 4, 2), (1, -1, 4, 2), (1, 127, 4, 2), (1, 30, -1, 2), (1, 30, 15, 2), (1, 30, 4, 5),
                (1, 30, 4, -1), (1, 2 ** 31 - 1, 4, 2), (1, 30, 2 ** 31 - 1, 2), (1, 30, 4, 2 ** 31 - 1),
                (-2 ** 31, -2 ** 31, -2 ** 31, -2 ** 31)]:
        got, _ = P.append([good, bad], q, k, v, max_rows=4, model=False)
        assert P.stat() == 1 and (got[3:] == MARK).all(), bad
        got, _ = P.attend([good, bad], q, max_rows=4, max_count=128)
        assert P.stat() == 1 and (got[3:] == MARK).all(), bad
        kk, vv = P.read([good, bad], max_rows=4, n=16)
        assert P.stat() == 1 and (kk[3:] == MARK).all() and (vv[3:] == MARK).all(), bad
    # past max_count, which only the attention has
    got, _ = P.attend([good, (1, 25, 4, 4)], q, max_rows=4, max_count=28)
    assert P.stat() == 1 and (got == MARK).all()
    P.ref.append(2, 30, turned(k[:3].astype(np.float64), P.rope, 30), v[:3].astype(np.float64))
    P.check_read()
    P.check_attend([good], q)
    # a slot given twice: neither is appended, the others are
    P.append([(1, 30, 0, 2), (3, 30, 2, 2), (1, 40, 4, 2)], q, k, v, model=False)
    assert P.stat() == 1
    P.ref.append(3, 30, turned(k[2:4].astype(np.float64), P.rope, 30), v[2:4].astype(np.float64))
    P.check_read()
    # without rows it may stand there twice, and a segment without rows may say anything
    P.append([(1, 30, 0, 2), (1, 30, 2, 0), (-1, -2 ** 31, 2 ** 31 - 1, 0)], q, k, v, model=False)
    assert (P.read([(7, 2 ** 31 - 1, -5, 0)], n=3)[0] == MARK).all()
    assert (P.attend([(-1, 2 ** 31 - 16, -5, 0), (9, 0, 0, 0)], q, max_count=100)[0] == MARK).all()
    assert P.stat() == 0
    P.ref.append(1, 30, turned(k[:2].astype(np.float64), P.rope, 30), v[:2].astype(np.float64))
    P.check_read()


@pytest.mark.parametrize("page", [-1, 11, 2 ** 31 - 1, -2 ** 31])
def test_pages_outside_the_pool_are_not_touched(gpu, page):
    rng = np.random.default_rng(9)
    P = Pages(gpu, 8, 2, 64, 2, 4, pool=11)
    P.append([(0, 0, 0, 200), (1, 0, 200, 200)], *rows_of(rng, 400, 8, 2, 64))
    before = [b.download(np.uint8, P.nbytes) for b in P.planes]
    P.table[0, 2] = page
    P.tab.upload(P.table)
    assert P.stat() == 0
    P.append([(0, 140, 0, 30)], *rows_of(rng, 30, 8, 2, 64), model=False)
    assert P.stat() == 1
    assert all(np.array_equal(b.download(np.uint8, P.nbytes), x) for b, x in zip(P.planes, before))
    kk, vv = P.read([(0, 100, 0, 60), (1, 100, 60, 60)])
    assert P.stat() == 1
    assert np.isnan(kk[28:60]).all() and np.isnan(vv[28:60]).all()
    assert np.isfinite(kk[:28]).all() and np.isfinite(vv[60:]).all()
    q = rows_of(rng, 200, 8, 2, 64)[0]
    for rows in (1, 100):
        segs = [(0, 180, 0, rows)] if rows == 1 else [(0, 50, 0, rows)]
        got, _ = P.attend(segs + [(1, 200 - rows, rows, rows)], q)
        assert P.stat() == 1
        assert np.isnan(got[:1] if rows == 1 else got[78:100]).all() and np.isfinite(got[rows:2 * rows]).all()
        assert rows == 1 or np.isfinite(got[:78]).all()
    # a page that no row attends may be none
    P.check_attend([(0, 90, 0, 38), (1, 190, 38, 10)], q[:48])
    P.check_attend([(0, 195, 0, 1)], q[:1], window=3)
    assert P.stat() == 0


COUNTS = [1, 2, 15, 16, 17, 63, 64, 65, 127, 200, 449, 1030]


@pytest.mark.parametrize("rows,heads,kv,count,names", [
    (1, 32, 8, 64, ["c16"]), (1, 32, 8, 512, ["c16"]), (1, 32, 8, 2049, ["c16", "join"]), (1, 40, 2, 64, ["c32"]),
    (6, 32, 8, 2049, ["c32", "join"]), (300, 32, 8, 300, ["c32"])])
def test_which_kernels_run(gpu, launched, rows, heads, kv, count, names):
    """Few and many columns, with and without a split, alone and in both head sizes (128 columns: below)."""
    rng = np.random.default_rng(rows + count)
    for hd in (64, 128):
        P = Pages(gpu, heads, kv, hd, 1, 33, seed=rows)
        P.append([(0, 0, 0, count)], *rows_of(rng, count, heads, kv, hd))
        q = rows_of(rng, rows, heads, kv, hd)[0]
        got, seen = launched(lambda: P.check_attend([(0, count - rows, 0, rows)], q))
        assert seen == ["cj_kv8_%s_h%d" % ("join" if n == "join" else "attend_" + n, hd) for n in names]
        assert np.array_equal(got, P.check_attend([(0, count - rows, 0, rows)], q))


@pytest.mark.parametrize("window", [0, 1, 40])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 64), (32, 8, 128), (2, 2, 128), (16, 1, 64), (24, 1, 128), (64, 1, 64)])
def test_attention_of_one_row(gpu, heads, kv, hd, window):
    say("kv8 decode", heads, kv, hd, window)
    rng = np.random.default_rng(heads + hd + window)
    n = len(COUNTS)
    P = Pages(gpu, heads, kv, hd, n, 17, seed=hd)
    total = sum(COUNTS)
    at = np.cumsum([0] + COUNTS)
    P.append([(s, 0, int(at[s]), c) for s, c in enumerate(COUNTS)], *rows_of(rng, total, heads, kv, hd))
    q = rows_of(rng, n + 2, heads, kv, hd)[0] * np.float32(2)
    P.check_attend([(s, c - 1, n - s, 1) for s, c in enumerate(COUNTS)], q, window)
    for s in (0, 4, n - 1):   # alone, the positions are split over more workgroups
        P.check_attend([(s, COUNTS[s] - 1, 0, 1)], q[:1], window)
    assert P.stat() == 0


@pytest.mark.parametrize("rows", [2, 3, 4, 7, 16, 33])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 64), (32, 8, 128), (3, 3, 64), (10, 2, 128)])
def test_attention_of_a_few_rows(gpu, heads, kv, hd, rows):
    say("kv8 rows", heads, kv, hd, rows)
    rng = np.random.default_rng(heads + hd + rows)
    counts = [rows, rows + 1, 64 + rows, 300]
    P = Pages(gpu, heads, kv, hd, len(counts), 6, seed=rows)
    at = np.cumsum([0] + counts)
    P.append([(s, 0, int(at[s]), c) for s, c in enumerate(counts)], *rows_of(rng, int(at[-1]), heads, kv, hd))
    q = rows_of(rng, 4 * rows, heads, kv, hd)[0] * np.float32(2)
    for window in (0, 1, 20):
        P.check_attend([(s, c - rows, s * rows, rows) for s, c in enumerate(counts)], q, window)
    # ragged: fewer rows than the most, and none
    P.check_attend([(0, 0, 0, rows), (1, rows, rows, 1), (2, 5, rows + 1, 0), (3, 290 - rows, rows + 1, rows)], q)
    assert P.stat() == 0


@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 64), (4, 1, 128), (3, 1, 128), (1, 1, 64), (40, 1, 64)])
def test_attention_of_chunks(gpu, heads, kv, hd, window):
    say("kv8 chunk", heads, kv, hd, window)
    rng = np.random.default_rng(heads + hd + window)
    P = Pages(gpu, heads, kv, hd, 4, 9, seed=window)
    P.append([(0, 0, 0, 211), (1, 0, 211, 512), (2, 0, 723, 64), (3, 0, 787, 129)], *rows_of(rng, 916, heads, kv, hd))
    q = rows_of(rng, 500, heads, kv, hd)[0] * np.float32(2)
    P.check_attend([(0, 0, 0, 211), (1, 450, 211, 62), (2, 0, 273, 64), (3, 1, 337, 128)], q, window)
    P.check_attend([(1, 385, 0, 127)], q[:127], window)
    assert P.stat() == 0


@pytest.mark.parametrize("window", [0, 37])
@pytest.mark.parametrize("heads,kv,hd,n", [(32, 8, 128, 44), (8, 8, 64, 44), (30, 6, 128, 56)])
def test_attention_of_chunks_that_fill_the_chip(gpu, launched, heads, kv, hd, n, window):
    """Enough segments of enough rows for the 128-column workgroups; ragged, from inside pages, some of one row or none."""
    say("kv8 many", heads, kv, hd, window)
    rng = np.random.default_rng(heads + hd + window)
    rows = rng.integers(17, 34, n) * (4 if heads == kv else 1)
    rows[3], rows[5], rows[7] = 0, 1, rows.max()
    before = rng.integers(0, 90, n)
    before[:8] = (0, 64, 63, 5, 1, 100, 47, 48)
    slots = rng.permutation(n)
    P = Pages(gpu, heads, kv, hd, n, 4, seed=window)
    at = np.cumsum(np.concatenate(([0], before + rows)))
    P.append([(int(s), 0, int(a), int(b + r)) for s, a, b, r in zip(slots, at, before, rows)],
             *rows_of(rng, int(at[-1]), heads, kv, hd))
    at = np.cumsum(np.concatenate(([2], rows)))
    q = rows_of(rng, int(at[-1]) + 2, heads, kv, hd)[0] * np.float32(2)
    segs = [(int(s), int(b), int(a), int(r)) for s, a, b, r in zip(slots, at, before, rows)]
    got, names = launched(lambda: P.check_attend(segs, q, window))
    assert names == ["cj_kv8_attend_c128_h%d" % hd]
    assert np.array_equal(got, P.check_attend(segs, q, window))      # and the same again
    q[at[5], 0, 3] = np.nan
    bad, _ = P.attend(segs, q, window)
    same = np.isnan(bad[at[5], 0]).all() and np.array_equal(bad[at[5], 1:], got[at[5], 1:])
    assert same and np.array_equal(np.delete(bad, at[5], 0), np.delete(got, at[5], 0))
    assert P.stat() == 0
    # a page outside the pool: its rows are NaN, the others stay
    k = 7
    P.table[slots[k], 0] = P.pool
    P.tab.upload(P.table)
    q[at[5], 0, 3] = 1.0
    bad, _ = P.attend(segs, q, window)
    assert P.stat() == 1
    mine = slice(int(at[k]), int(at[k] + rows[k]))
    last = before[k] + np.arange(rows[k])
    first = np.maximum(0, last + 1 - window) if window else np.zeros_like(last)
    assert np.array_equal(np.isnan(bad[mine]).all((1, 2)), first < PAGE)
    assert np.isfinite(np.delete(bad, np.r_[mine], 0)).all()


def test_loud_and_quiet_blocks_and_far_scores(gpu):
    """Blocks whose scales differ by up to 2^20, and scores of some hundreds."""
    rng = np.random.default_rng(77)
    for heads, kv, hd, rows in ((8, 2, 64, 1), (4, 1, 128, 40)):
        P = Pages(gpu, heads, kv, hd, 1, 8)
        q, k, v = rows_of(rng, 400, heads, kv, hd)
        v *= np.exp2(rng.integers(-10, 11, 25)).repeat(16).astype(np.float32)[:, None, None]
        k *= np.exp2(rng.integers(-2, 3, 25)).repeat(16).astype(np.float32)[:, None, None]
        P.append([(0, 0, 0, 400)], q, k, v)
        q = rows_of(rng, rows, heads, kv, hd)[0]
        for loud in (0.0, 1e-30, 1.0, 30.0, 1e4):
            P.check_attend([(0, 400 - rows, 0, rows)], (q * np.float32(loud)).astype(np.float32))
        P.check_attend([(0, 400 - rows, 0, rows)], q, scale=-0.3)
        P.check_attend([(0, 400 - rows, 0, rows)], q, scale=0.0)


def test_a_pool_past_four_gigabytes(gpu):
    """Pages whose bytes lie past 2^32, and rows of q and out past 2^31 bytes apart."""
    rng = np.random.default_rng(4)
    heads, kv, hd = 16, 8, 128
    P = Pages(gpu, heads, kv, hd, 2, 4, pool=70000, garbage=False)
    P.table[:] = 70000 - 1 - np.arange(8).reshape(2, 4) * 3
    P.tab.upload(P.table)
    P.append([(0, 0, 0, 190), (1, 0, 190, 201)], *rows_of(rng, 391, heads, kv, hd))
    P.check_read()
    q = rows_of(rng, 80, heads, kv, hd)[0]
    P.check_attend([(0, 189, 0, 1), (1, 200, 1, 1)], q[:2])
    P.check_attend([(0, 150, 0, 40), (1, 161, 40, 40)], q)
    assert P.stat() == 0


def test_positions_near_two_to_the_31(gpu):
    """A slot of 2^25 pages, of which the last few exist, and a bound on the rows that would wrap a position."""
    rng = np.random.default_rng(6)
    heads, kv, hd, L = 4, 1, 64, gpu.native.lib()
    P = Pages(gpu, heads, kv, hd, 1, 4, pool=9)
    P.append([(0, 0, 0, 200)], *rows_of(rng, 200, heads, kv, hd))
    want = P.read([(0, 0, 0, 200)])
    pages = (2 ** 31 - 1) // 64
    table = np.full((1, pages), -1, np.int32)
    table[0, -4:] = P.table[0]
    base = (pages - 4) * 64
    P.tab, P.slot_pages = gpu.Buffer.of(table), pages
    got = P.read([(0, base, 0, 200)], max_rows=2 ** 27)
    assert all(np.array_equal(x, y) for x, y in zip(got, want))
    for rows in (1, 7, 40):      # the rows that a window lets see the four pages alone
        q = rows_of(rng, rows, heads, kv, hd)[0]
        got, scale = P.attend([(0, base + 200 - rows, 0, rows)], q, window=100)
        ref, tol = attention(q.astype(np.float64), P.ref.values(0, "k", 0, 200), P.ref.values(0, "v", 0, 200), 200 - rows, scale,
                             100, P.ref.steps(0, "v").repeat(BLOCK, 0))
        assert (np.abs(got - ref) <= tol).all()
    assert P.stat() == 0


def serve(P, rng, steps, lens, attend=True):
    """Prompts in chunks of uneven sizes, then decode steps, as a serving loop runs them."""
    heads, kv, hd = P.heads, P.kv, P.hd
    done = [0] * len(lens)
    while any(d < n for d, n in zip(done, lens)):
        segs, row = [], 0
        for s, n in enumerate(lens):
            c = min(n - done[s], int(rng.integers(1, 50)))
            if c:
                segs.append((s, done[s], row, c))
                done[s], row = done[s] + c, row + c
        q, k, v = rows_of(rng, row, heads, kv, hd)
        q, _ = P.append(segs, q, k, v)
        P.check_attend(segs, q)
    for _ in range(steps):
        segs = [(s, done[s], i, 1) for i, s in enumerate(rng.permutation(len(lens)).tolist())]
        q, _ = P.append(segs, *rows_of(rng, len(lens), heads, kv, hd))
        for s in range(len(lens)):
            done[s] += 1
        P.check_attend(segs, q)
    return done


@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 64), (8, 2, 128)])
def test_prompts_in_chunks_then_decode_steps(gpu, heads, kv, hd):
    P = Pages(gpu, heads, kv, hd, 3, 4)
    serve(P, np.random.default_rng(hd), 20, [130, 7, 63])
    P.check_read()
    assert P.stat() == 0


def test_a_captured_step_follows_its_segments_and_tables(gpu):
    """Append and attend captured once, replayed with other segments, pages and rows; each replay against eager calls."""
    rng = np.random.default_rng(21)
    heads, kv, hd, n = 8, 2, 128, 3
    check, L = gpu.native.check, gpu.native.lib()
    P = Pages(gpu, heads, kv, hd, 4, 8)
    lens = [70, 5, 250, 31]
    at = np.cumsum([0] + lens)
    P.append([(s, 0, int(at[s]), c) for s, c in enumerate(lens)], *rows_of(rng, int(at[-1]), heads, kv, hd))
    wide, B = (heads + 2 * kv) * hd, gpu.Buffer
    qkv, q, out, segs = B(n * wide * 4), B(n * heads * hd * 4), B(n * heads * hd * 4), B(n * 16)
    need = L.cj_kv8_attend_bytes(n, 1, 512, heads, kv, hd, 0)
    parts = [B(max(16, need)) for _ in range(2)]

    def step(part):
        check(L.cj_kv8_append(q.h, qkv.h, qkv.h + 4 * heads * hd, qkv.h + 4 * (heads + kv) * hd, P.planes[0].h, P.planes[1].h,
                              0, 0, P.rope_b.h, P.tab.h, segs.h, n, 1, n, P.ctx, P.pool, 4, 8, heads, kv, hd, heads * hd, wide,
                              wide, 0, ctypes.c_float(EPS), 0, P.status.h), "append")
        check(L.cj_kv8_attend(out.h, q.h, P.planes[0].h, P.planes[1].h, P.tab.h, segs.h, part.h, n, 1, n, 512, P.pool, 4, 8,
                              heads, kv, hd, heads * hd, heads * hd, 0, ctypes.c_float(1 / math.sqrt(hd)), P.status.h), "attend")

    graphs = []
    for _ in range(2):   # two graphs that share the workspace, and an eager call with its own
        check(L.cj_graph_begin(), "begin")
        step(parts[0])
        graphs.append(gpu.native.handle(L.cj_graph_end(), "end"))
    for t in range(6):
        chosen = rng.permutation(4)[:n].tolist()
        rows = rng.standard_normal((n, wide)).astype(np.float32)
        segs.upload(np.array([(s, lens[s], i, 1) for i, s in enumerate(chosen)], np.int32))
        qkv.upload(rows)
        check(L.cj_graph_launch(graphs[t % 2]), "launch")
        gpu.native.sync()
        got = out.download(np.float32, n * heads * hd).copy()
        step(parts[1])            # the same once more: the rows are stored as they are already
        gpu.native.sync()
        assert np.array_equal(got, out.download(np.float32, n * heads * hd))
        for i, s in enumerate(chosen):
            x = rows[i].astype(np.float64).reshape(1, -1, hd)
            P.ref.append(s, lens[s], turned(x[:, heads:heads + kv], P.rope, lens[s]), x[:, heads + kv:])
            qq = turned(x[:, :heads], P.rope, lens[s]).astype(np.float32).astype(np.float64)
            want, tol = attention(qq, P.ref.values(s, "k", 0, lens[s] + 1), P.ref.values(s, "v", 0, lens[s] + 1), lens[s],
                                  np.float64(np.float32(1 / math.sqrt(hd))), 0, P.ref.steps(s, "v").repeat(BLOCK, 0))
            # q's own rounding to f32 may fall the other way: 2^-23 of each value moves a score by that share of sum|q k|
            assert (np.abs(got.reshape(n, heads, hd)[i] - want[0]) <= 2 * tol[0]).all()
            lens[s] += 1
    for g in graphs:
        check(L.cj_graph_free(g), "free")
    P.check_read()
    assert P.stat() == 0


def test_beside_the_fp16_planes(gpu):
    """The same token through cj_qk_prep and cj_attend over fp16 planes: q by the same table, and an attention that differs
    by what eight bits lose of K and V."""
    L, check, f = gpu.native.lib(), gpu.native.check, ctypes.c_float
    rng = np.random.default_rng(12)
    heads, kv, hd, count = 32, 8, 128, 150
    P = Pages(gpu, heads, kv, hd, 1, 3, pool=3)
    check(L.cj_rope_table(P.rope_b.h, hd, f(10000.0), P.ctx), "rope table")
    P.rope = P.rope_b.download(np.float32, P.ctx * hd).reshape(P.ctx, hd // 2, 2)
    q, k, v = rows_of(rng, count, heads, kv, hd)
    got, want = P.append([(0, 0, 0, count)], q, k, v)
    assert near(got, want)
    kc, vc = gpu.Buffer(3 * kv * 64 * hd * 2), gpu.Buffer(3 * kv * 64 * hd * 2)
    part, cnt, out = gpu.Buffer(heads * 64 * (hd + 2) * 4), gpu.Buffer(kv * 4), gpu.Buffer(heads * hd * 4)
    cnt.zero()
    for t in range(count):
        qb, kb, vb = gpu.Buffer.of(q[t]), gpu.Buffer.of(k[t]), gpu.Buffer.of(v[t])
        check(L.cj_qk_prep(qb.h, kb.h, vb.h, kc.h, vc.h, 0, 0, P.rope_b.h, P.tab.h, 0, heads, kv, hd, 0, f(EPS), 0, t), "qk prep")
    turned_q = qb.download(np.float32, heads * hd).reshape(heads, hd)
    # two products and a sum in f32 there, each rounded: 2^-23 of |a| + |b| at most
    size = np.abs(q[-1]).astype(np.float64)
    size = size + np.roll(size, hd // 2, -1)
    assert (np.abs(turned_q - got[-1]) <= 2.0 ** -23 * size).all()
    check(L.cj_attend(part.h, out.h, qb.h, kc.h, vc.h, P.tab.h, 0, cnt.h, heads, kv, hd, count, 0, 512, f(1 / math.sqrt(hd))), "attend")
    ours, scale = P.attend([(0, count - 1, 0, 1)], turned_q[None])
    # the codes' errors lie evenly within half a step, one apart from the other: a score is off by step x |q| x scale / sqrt(12)
    # in the root mean square, and a channel by the root of the sum of p^2 x ((that x |v|)^2 + step_v^2 / 12), where the sum of
    # p^2 is the largest p at most; seven times that, and fp16's 2^-11 of a value, over 4096 values
    there = out.download(np.float32, heads * hd).reshape(heads, hd)
    ks, vs = (P.ref.steps(0, n).max(0) for n in ("k", "v"))
    kk, vv = P.ref.values(0, "k", 0, count), P.ref.values(0, "v", 0, count)
    for h in range(heads):
        g, x = h * kv // heads, turned_q[h].astype(np.float64)
        s = scale * kk[:, g] @ x
        p = np.exp(s - s.max())
        p /= p.sum()
        big = np.abs(vv[:, g]).max()
        sd = math.sqrt(p.max()) * math.hypot(ks[g] * np.linalg.norm(x) * scale / math.sqrt(12) * big, vs[g] / math.sqrt(12))
        half = 2.0 ** -11 * (1 + scale * np.abs(x).sum() * np.abs(kk[:, g]).max()) * big
        assert (np.abs(ours[0, h] - there[h]) <= 7 * sd + half).all(), h


@pytest.mark.parametrize("rows,count", [(1, 100), (1, 2049), (12, 2049), (200, 300)])
def test_out_may_be_q(gpu, rows, count):
    rng = np.random.default_rng(rows)
    heads, kv, hd, L = 32, 8, 128, gpu.native.lib()
    P = Pages(gpu, heads, kv, hd, 1, 33)
    P.append([(0, 0, 0, count)], *rows_of(rng, count, heads, kv, hd))
    q = rows_of(rng, rows, heads, kv, hd)[0]
    want, scale = P.attend([(0, count - rows, 0, rows)], q)
    b, sb = gpu.Buffer.of(q), P.segs([(0, count - rows, 0, rows)])
    need = L.cj_kv8_attend_bytes(1, rows, count, heads, kv, hd, 0)
    part = gpu.Buffer(max(16, need))
    gpu.native.check(L.cj_kv8_attend(
        b.h, b.h, P.planes[0].h, P.planes[1].h, P.tab.h, sb.h, part.h, 1, rows, rows, count, P.pool, P.slots, P.slot_pages, heads,
        kv, hd, heads * hd, heads * hd, 0, ctypes.c_float(scale), P.status.h), "attend")
    assert np.array_equal(b.download(np.float32, q.size).reshape(q.shape), want)
    # a workspace that is too small is refused before anything runs
    if need:
        small = gpu.Buffer(need - 16)
        assert L.cj_kv8_attend(
            b.h, b.h, P.planes[0].h, P.planes[1].h, P.tab.h, sb.h, small.h, 1, rows, rows, count, P.pool, P.slots, P.slot_pages,
            heads, kv, hd, heads * hd, heads * hd, 0, ctypes.c_float(scale), P.status.h) == gpu.native.CJ_ERR_ARG
        assert "part" in gpu.native.last_error()


def test_two_threads_with_a_workspace_each(gpu):
    """Calls of two threads land on the one stream in any order; each thread's results are those of its calls alone."""
    import threading
    heads, kv, hd, L = 32, 8, 128, gpu.native.lib()
    work = []
    for seed in (1, 2):
        rng = np.random.default_rng(seed)
        P = Pages(gpu, heads, kv, hd, 2, 33, seed=seed)
        P.append([(0, 0, 0, 2049), (1, 0, 2049, 700)], *rows_of(rng, 2749, heads, kv, hd))
        q = rows_of(rng, 8, heads, kv, hd)[0]
        segs = [(0, 2045, 0, 4), (1, 696, 4, 4)]
        need = L.cj_kv8_attend_bytes(2, 4, 2049, heads, kv, hd, 0)
        assert need > 0
        work.append((P, P.attend(segs, q, max_count=2049)[0], P.segs(segs), gpu.Buffer.of(q), gpu.Buffer(need),
                     gpu.Buffer(q.nbytes)))
    wrong = []

    def run(P, want, sb, qb, part, out):
        for _ in range(30):
            rc = L.cj_kv8_attend(out.h, qb.h, P.planes[0].h, P.planes[1].h, P.tab.h, sb.h, part.h, 2, 4, 8, 2049, P.pool, 2, 33,
                                 heads, kv, hd, heads * hd, heads * hd, 0, ctypes.c_float(1 / math.sqrt(hd)), 0)
            if rc or not np.array_equal(out.download(np.float32, want.size).reshape(want.shape), want):
                wrong.append(rc)

    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_refusals(gpu):
    """Arguments that the host refuses before anything is launched."""
    L, ARG = gpu.native.lib(), gpu.native.CJ_ERR_ARG
    heads, kv, hd = 8, 2, 64
    P = Pages(gpu, heads, kv, hd, 2, 2)
    n = 4
    q, k, o, w = gpu.Buffer(n * heads * hd * 4), gpu.Buffer(n * kv * hd * 4), gpu.Buffer(n * heads * hd * 4), gpu.Buffer(hd * 4)
    segs = P.segs([(0, 0, 0, 1), (1, 0, 1, 1)])
    f = ctypes.c_float

    def good(call):
        if call == "append":
            return dict(q_out=o.h, q=q.h, k=k.h, v=k.h, kplane=P.planes[0].h, vplane=P.planes[1].h, qw=w.h, kw=w.h,
                        rope=P.rope_b.h, pgtab=P.tab.h, segs=segs.h, n_segs=2, max_rows=1, n_rows=n, rope_ctx=P.ctx,
                        n_pages=P.pool, n_slots=2, slot_pages=2, n_q=heads, n_kv=kv, head_dim=hd, q_out_stride=heads * hd,
                        q_stride=heads * hd, kv_stride=kv * hd, norm=1, eps=f(EPS), form=0, status=P.status.h)
        if call == "read":
            return dict(k_out=k.h, v_out=k.h, kplane=P.planes[0].h, vplane=P.planes[1].h, pgtab=P.tab.h, segs=segs.h, n_segs=2,
                        max_rows=1, n_rows=n, n_pages=P.pool, n_slots=2, slot_pages=2, n_kv=kv, head_dim=hd,
                        out_stride=kv * hd, status=P.status.h)
        return dict(out=o.h, q=q.h, kplane=P.planes[0].h, vplane=P.planes[1].h, pgtab=P.tab.h, segs=segs.h, part=0, n_segs=2,
                    max_rows=1, n_rows=n, max_count=64, n_pages=P.pool, n_slots=2, slot_pages=2, n_q=heads, n_kv=kv,
                    head_dim=hd, q_stride=heads * hd, out_stride=heads * hd, window=0, scale=f(0.1), status=P.status.h)

    def call(name, **changes):
        a = good(name)
        assert set(changes) <= set(a)
        return getattr(L, "cj_kv8_" + name)(*{**a, **changes}.values())

    both = [dict(n_segs=0), dict(n_segs=3), dict(max_rows=0), dict(n_rows=0), dict(n_rows=n + 1), dict(n_pages=0),
            dict(n_pages=P.pool + 1), dict(n_slots=0), dict(n_slots=3), dict(slot_pages=0), dict(slot_pages=3),
            dict(slot_pages=2 ** 31 - 1), dict(n_kv=0), dict(head_dim=32), dict(head_dim=96), dict(head_dim=0),
            dict(kplane=0), dict(vplane=P.planes[1].h + 16), dict(kplane=P.planes[0].h + 4), dict(pgtab=0), dict(segs=0),
            dict(segs=segs.h + 4), dict(status=12), dict(status=P.status.h + 2)]
    extra = {
        "append": [dict(q=0), dict(q_out=0), dict(q=q.h + 4), dict(k=0), dict(v=k.h + 16), dict(k=k.h + 4), dict(rope=0),
                   dict(rope_ctx=0), dict(rope_ctx=P.ctx + 1), dict(qw=0), dict(kw=0), dict(q_stride=heads * hd - 4),
                   dict(q_stride=heads * hd + 1), dict(kv_stride=kv * hd - 4), dict(kv_stride=-kv * hd),
                   dict(q_out_stride=2 ** 62), dict(n_q=7), dict(n_q=0), dict(n_q=65 * kv)],
        "read": [dict(k_out=0, v_out=0), dict(max_rows=2 ** 28), dict(k_out=k.h + 4), dict(out_stride=kv * hd + 4), dict(out_stride=2)],
        "attend": [dict(out=0), dict(q=0), dict(q=q.h + 8), dict(max_count=0), dict(window=-1), dict(n_q=7), dict(n_q=65 * kv),
                   dict(out_stride=heads * hd + 4), dict(q_stride=heads * hd - 64), dict(max_rows=2 ** 31 - 1)],
    }
    for name in ("append", "read", "attend"):
        assert call(name) == 0, (name, gpu.native.last_error())
        for change in both + extra[name]:
            assert call(name, **change) == ARG, (name, change)
            assert ("cj_kv8_" + name) in gpu.native.last_error(), (name, change)
    # the queries, the norm and one of the outputs may be left out
    assert call("append", q=0, q_out=0, qw=0) == 0 and call("append", norm=0, qw=0, kw=0, status=0) == 0
    assert call("read", k_out=0, status=0) == 0 and call("read", v_out=0) == 0
    gpu.native.sync()
