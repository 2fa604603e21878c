"""The 4-bit KV cache on the device: its bytes, and attention over it against 64 bits."""
import ctypes as C

import numpy as np
import pytest

from atlas_amd._lib import Kv4BatchC, Kv4CacheC, check
from tests import kv4_parts, mx_ref
from tests.gpu_util import Dev, lib, sync
from tests.stream_util import Stream, on_thread

pytestmark = pytest.mark.gpu


class Case:
    """A cache of random tokens, a batch over it, and what both hold on the host."""

    def __init__(self, seed, lens, rows=None, n_kv=2, hd=128, page=32, spare=2, junk=True, width=None, tail_rows=0):
        rng = np.random.default_rng(seed)
        self.rng, self.n_kv, self.hd, self.page = rng, n_kv, hd, page
        self.lens, self.rows = list(lens), list(rows) if rows is not None else [1] * len(lens)
        need = [-(-n // page) for n in lens]
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages)
        self.width = max(max(need), 1) if width is None else width
        self.table = np.full((len(lens), self.width), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n][:self.width]
            at += n
        total = self.n_pages * page
        self.k = (rng.standard_normal((total, n_kv, hd)) * np.exp(0.5 * rng.standard_normal((n_kv, hd)))).astype(np.float32)
        self.v = rng.standard_normal((total, n_kv, hd)).astype(np.float32)
        self.bytes = mx_ref.pages(self.k, self.v, page)
        if junk:                       # what lies behind a sequence's end is anything, NaN scales among it
            self._junk(need)
        self.starts = np.concatenate([[0], np.cumsum(self.rows)]).astype(np.int32)
        self.n_rows = int(self.starts[-1]) + tail_rows
        self.packed = rows is not None

    def _junk(self, need):
        kb, hd, page = self.hd // 32, self.hd, self.page
        d, sc = page * hd // 2, page * kb
        for s, n in enumerate(self.lens):
            if n % page == 0 or need[s] > self.width:
                continue
            p, first = self.table[s, need[s] - 1], n % page
            for part in (d, 2 * d + sc):
                x = self.bytes[p, :, part:part + sc].reshape(self.n_kv, page // 8, kb, 8)
                for t in range(first, page):
                    x[:, t // 8, :, t % 8] = self.rng.integers(250, 256, (self.n_kv, kb))

    def slot(self, s, t):
        """Row of k and v of token t of sequence s, or None."""
        if t < 0 or t // self.page >= self.width:
            return None
        p = self.table[s, t // self.page]
        return p * self.page + t % self.page if 0 <= p < self.n_pages else None

    def upload(self):
        self.d = dict(cache=Dev(self.bytes), lens=Dev(np.asarray(self.lens, np.int32)), starts=Dev(self.starts),
                      table=Dev(self.table))
        self.c = Kv4CacheC(self.d["cache"].ptr, self.n_pages, self.page, self.n_kv, self.hd)
        self.b = Kv4BatchC(self.d["starts"].ptr if self.packed else None, self.d["lens"].ptr, self.d["table"].ptr,
                           self.width, len(self.lens), self.n_rows, 0)
        return C.byref(self.c), C.byref(self.b)

    def each_row(self):
        """(row, sequence, position) of the batch's rows."""
        for s, n in enumerate(self.lens):
            for i in range(self.rows[s]):
                yield int(self.starts[s]) + i, s, n - self.rows[s] + i


def _check_attention(c, heads, window=0, scale=None, max_len=0, pad_q=0, pad_o=0, args=None):
    rng, hd = c.rng, c.hd
    scale = scale if scale is not None else hd ** -0.5
    wide = heads * hd
    q = rng.standard_normal((c.n_rows, wide + pad_q)).astype(np.float32)
    out = Dev(np.full((c.n_rows, wide + pad_o), 7, np.float32))
    qd = Dev(q)
    cache, batch = args or c.upload()
    c.b.max_len = max_len
    check(lib().atlas_kv4_attention_f32(cache, batch, qd.ptr, wide + pad_q, heads, scale, window, out.ptr, wide + pad_o))
    sync()
    got = out.get()
    assert (got[:, wide:] == 7).all()
    assert (got[int(c.starts[-1]):] == 7).all()        # rows behind the last sequence
    kd, vd = mx_ref.rounded(c.k), mx_ref.rounded(c.v)
    worst = 0.0
    for row, s, pos in c.each_row():
        keys = np.array([t for t in range(pos + 1) if c.slot(s, t) is not None], np.int64)
        at = np.array([c.slot(s, t) for t in keys], np.int64)
        x = q[row, :wide].reshape(heads, hd)
        want = mx_ref.attend(x, keys, kd[at], vd[at], pos, scale, window)
        bound = _bound(x, keys, kd[at], vd[at], pos, scale, window)
        err = np.abs(got[row, :wide].reshape(heads, hd) - want)
        assert (err <= bound).all(), (row, s, pos, float((err / np.maximum(bound, 1e-30)).max()))
        worst = max(worst, float(err.max()))
    return got, worst


def _bound(q, keys, k, v, pos, scale, window):
    """What the formula's roundings can do to a row: q as the cache's products use it is off by 2^-20 of the
    row's largest value in each element; a score's sums by a last place (2^-23) at each of the 128 + 10 steps
    and 4 roundings around them; a weight by 2^-16 (two 8-bit parts) and 2^-21 (exp2, its argument's rounding
    is counted with the score); the sums over n tokens by 2^-23 at each of 32 + n / 32 + 64 steps."""
    see = (keys <= pos) & (keys > pos - window if window else keys >= 0)
    bound = np.zeros(q.shape)
    if not see.any():
        return bound
    heads, n_kv = q.shape[0], k.shape[1]
    for h in range(heads):
        kk, vv = k[see, h * n_kv // heads], v[see, h * n_kv // heads]
        s = kk @ q[h].astype(np.float64) * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        size = np.abs(kk) @ np.abs(q[h].astype(np.float64)) * abs(scale)
        ds = abs(scale) * 2.0 ** -20 * np.abs(q[h]).max() * np.abs(kk).sum(1) + 142 * 2.0 ** -23 * size
        rel = 2 * ds.max() + 2 * (2.0 ** -16 + 2.0 ** -21) + (96 + see.sum() / 32) * 2.0 ** -23
        bound[h] = rel * (p @ np.abs(vv))
    return bound


# ---- writing and reading ------------------------------------------------------------


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("lens,rows,n_kv,page", [([1], None, 1, 32), ([40, 33, 64], None, 3, 32), ([70, 5, 130], [70, 2, 31], 2, 64),
                                                 ([9, 0, 12, 33], [9, 0, 1, 8], 5, 32), ([300], [300], 8, 256)])
def test_write_and_read(hd, lens, rows, n_kv, page):
    """The new tokens' bytes are the layout's, every other byte stays; reading gives their values."""
    c = Case(hd + len(lens), lens, rows, n_kv, hd, page, tail_rows=2 if rows is not None else 0)
    wide = n_kv * hd
    k = c.rng.standard_normal((c.n_rows, wide + 4)).astype(np.float32)
    v = c.rng.standard_normal((c.n_rows, wide + 4)).astype(np.float32)
    before = c.rng.integers(0, 256, c.bytes.shape, dtype=np.uint8)
    c.bytes = before.copy()
    cache, batch = c.upload()
    kd, vd = Dev(k), Dev(v)
    check(lib().atlas_kv4_write_f32(cache, batch, kd.ptr, vd.ptr, wide + 4))
    sync()
    # pages with the new rows in their places, and which of their bytes those are
    for row, s, pos in c.each_row():
        c.k[c.slot(s, pos)] = k[row, :wide].reshape(n_kv, hd)
        c.v[c.slot(s, pos)] = v[row, :wide].reshape(n_kv, hd)
    full = mx_ref.pages(c.k, c.v, page)
    mark = np.zeros_like(c.k)
    for row, s, pos in c.each_row():
        mark[c.slot(s, pos)] = 6.0               # code 7 in every nibble, scale byte 127 (0: codes 0, 127)
    touched = mx_ref.pages(mark, mark, page)
    d, sc = page * hd // 2, page * hd // 32
    sel = np.zeros(full.shape, bool)
    for a in (0, d + sc):
        sel[..., a:a + d] = touched[..., a:a + d] != 0
        sel[..., a + d:a + d + sc] = touched[..., a + d:a + d + sc] != 127
    # (6 has scale byte 127 as well: mark the scales by a value of another one)
    mark2 = np.where(mark != 0, 12.0, 0.0).astype(np.float32)
    touched = mx_ref.pages(mark2, mark2, page)
    for a in (0, d + sc):
        sel[..., a + d:a + d + sc] = touched[..., a + d:a + d + sc] != 127
    got = c.d["cache"].get()
    np.testing.assert_array_equal(got, np.where(sel, full, before))
    ko, vo = Dev(np.full(k.shape, 7, np.float32)), Dev(np.full(v.shape, 7, np.float32))
    check(lib().atlas_kv4_read_f32(cache, batch, ko.ptr, vo.ptr, wide + 4))
    sync()
    live = int(c.starts[-1])
    for x, y in ((k, ko.get()), (v, vo.get())):
        want = np.full(x.shape, 7, np.float32)
        want[:live, :wide] = mx_ref.rounded(x[:live, :wide].reshape(live, n_kv, hd)).reshape(live, wide)
        np.testing.assert_array_equal(y, want)


def test_write_special_values():
    """Infinities and NaN make their block read as NaN, nothing else; tiny and huge values keep theirs."""
    c = Case(5, [20], [20], 1, 64, 32)
    x = c.rng.standard_normal((20, 64)).astype(np.float32)
    x[3, 5], x[4, 40], x[5, 63] = np.nan, np.inf, -np.inf
    x[6] *= np.float32(2.0) ** -140
    x[7] *= np.float32(2.0) ** 125
    x[8] = 0
    cache, batch = c.upload()
    kd, ko, vo = Dev(x), Dev(np.empty_like(x)), Dev(np.empty_like(x))
    check(lib().atlas_kv4_write_f32(cache, batch, kd.ptr, kd.ptr, 64))
    check(lib().atlas_kv4_read_f32(cache, batch, ko.ptr, vo.ptr, 64))
    sync()
    want = mx_ref.rounded(x).astype(np.float32)
    np.testing.assert_array_equal(ko.get(), want)
    np.testing.assert_array_equal(vo.get(), want)


def test_tokens_without_a_page():
    """Entries that are no page, and tokens past the table: not written, read as zeros, not attended to."""
    c = Case(6, [90, 200, 40], [90, 3, 2], 2, 64, 32, width=3)
    c.table[0, 1] = -1
    c.table[1] = [c.n_pages, 1 << 30, -(1 << 31)]      # none of them a page
    wide = 128
    cache, batch = c.upload()
    k = c.rng.standard_normal((c.n_rows, wide)).astype(np.float32)
    before = c.d["cache"].get()
    kd, ko, vo = Dev(k), Dev(np.full(k.shape, 7, np.float32)), Dev(np.full(k.shape, 7, np.float32))
    check(lib().atlas_kv4_write_f32(cache, batch, kd.ptr, kd.ptr, wide))
    check(lib().atlas_kv4_read_f32(cache, batch, ko.ptr, vo.ptr, wide))
    sync()
    want = np.zeros_like(k)
    for row, s, pos in c.each_row():
        if c.slot(s, pos) is not None:
            c.k[c.slot(s, pos)] = c.v[c.slot(s, pos)] = k[row].reshape(2, 64)
            want[row] = mx_ref.rounded(k[row].reshape(2, 64)).reshape(-1)
    np.testing.assert_array_equal(ko.get(), want)
    np.testing.assert_array_equal(vo.get(), want)
    got, _ = _check_attention(c, 4, args=(cache, batch))
    assert (got[90:93] == 0).all()                     # sequence 1 has no page at all
    pages = [p for p in range(c.n_pages) if p not in c.table]
    np.testing.assert_array_equal(c.d["cache"].get()[pages], before[pages])


def test_sequences_that_share_pages():
    """A page in the tables of several sequences, and twice in one's: read by all of them."""
    c = Case(7, [100, 77, 128], None, 2, 128, 32, junk=False)
    c.table[1, :2] = c.table[0, :2]
    c.table[2] = c.table[0, 0]
    _check_attention(c, 4)


# ---- attention ----------------------------------------------------------------------


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 7, 8, 11, 16])
def test_decode_groups(hd, group):
    c = Case(group * hd, [1, 31, 32, 33, 70], None, 2, hd, 32)
    _check_attention(c, 2 * group)


@pytest.mark.parametrize("lens", [[1], [2], [19], [64], [500], [1025], [3001], [7, 900, 1, 2000, 64], [0, 5, 0]])
@pytest.mark.parametrize("page", [32, 64, 512])
def test_decode_lengths(lens, page):
    c = Case(sum(lens) + page, lens, None, 3, 64, page)
    _check_attention(c, 9)
    _check_attention(c, 9, max_len=max(lens))
    _check_attention(c, 9, max_len=1)                  # lengths that the caller did not know of


@pytest.mark.parametrize("window", [1, 7, 32, 33, 100, 1 << 30, (1 << 31) - 1])
@pytest.mark.parametrize("hd", [64, 128])
def test_window(window, hd):
    c = Case(window % 1000 + hd, [130, 40, 257, 3], [70, 1, 5, 3], 2, hd, 64)
    _check_attention(c, 4, window=window)
    c = Case(window % 1000 + hd, [130, 700], None, 2, hd, 64)
    _check_attention(c, 4, window=window)


@pytest.mark.parametrize("window", [2046, 2047, 2048, 2049])
@pytest.mark.parametrize("n_kv,hd,length,rows", [(96, 64, 2500, 1), (64, 128, 2500, 1), (96, 64, 2511, 3), (32, 128, 2060, 1)])
def test_window_in_runs(n_kv, hd, length, rows, window):
    """As many runs as the window's chunks have room for; its first and last chunks are parts."""
    c = Case(window + length, [length], None if rows == 1 else [rows], n_kv, hd, 64)
    for _ in range(2):                                 # the second call finds what the first left
        _check_attention(c, n_kv, window=window)


@pytest.mark.parametrize("hd,group,n_kv", [(64, 4, 2), (64, 3, 3), (128, 1, 4), (128, 8, 1), (128, 5, 2), (256, 2, 2), (256, 16, 1)])
@pytest.mark.parametrize("lens,rows", [([1], [1]), ([33], [33]), ([100, 65, 200], [100, 1, 37]), ([5, 0, 64, 70], [5, 0, 0, 70]),
                                       ([300], [17]), ([130, 129], [128, 129])])
def test_prompts(hd, group, n_kv, lens, rows):
    c = Case(sum(lens) + group, lens, rows, n_kv, hd, 64, tail_rows=3)
    _check_attention(c, group * n_kv, pad_q=8, pad_o=4)


@pytest.mark.parametrize("hd,group,n_kv", [(64, 4, 1), (128, 1, 2), (128, 7, 1), (256, 2, 1)])
@pytest.mark.parametrize("rows", [[140, 70], [9, 40]])
def test_prompts_in_runs(hd, group, n_kv, rows):
    """Tiles of 16 and of 32 columns over caches that several blocks share."""
    c = Case(rows[0] + group, [2500, 1300], rows, n_kv, hd, 64, tail_rows=2)
    for _ in range(2):
        _check_attention(c, group * n_kv)


def test_many_sequences():
    """More sequences than lanes, empty ones among them, in one packed batch."""
    rng = np.random.default_rng(1)
    lens = rng.integers(0, 80, 150)
    rows = np.minimum(lens, rng.integers(0, 4, 150))
    c = Case(8, lens.tolist(), rows.tolist(), 1, 64, 32)
    _check_attention(c, 4)


def test_large_scores():
    """Scores far apart, growing and falling along the cache: the running maximum moves often."""
    c = Case(9, [700, 300], None, 2, 128, 64)
    ramp = np.linspace(0.1, 6, c.k.shape[0])[:, None, None].astype(np.float32)
    for up in (ramp, ramp[::-1]):
        c.k = c.k / np.abs(c.k).max() * up * 4
        c.bytes = mx_ref.pages(c.k, c.v, c.page)
        _check_attention(c, 2, scale=1.0)
        _check_attention(c, 2, scale=-0.7)


def test_scores_at_the_documented_limit():
    """A score whose products sum to 0.98 2^127: a row that has seen only such has seen its tokens."""
    c = Case(11, [1, 40], None, 1, 64, 32)
    c.k[:] = 1.0
    c.bytes = mx_ref.pages(c.k, c.v, 32)
    scale = 0.98 * 2.0 ** 127 / 64
    for sign in (-1, 1):
        q, out = Dev(np.full((2, 64), sign, np.float32)), Dev(np.zeros((2, 64), np.float32))
        check(lib().atlas_kv4_attention_f32(*c.upload(), q.ptr, 64, 1, scale, 0, out.ptr, 64))
        sync()
        vd = mx_ref.rounded(c.v)
        want = np.stack([vd[[c.slot(s, t) for t in range(n)], 0].mean(0) for s, n in enumerate(c.lens)])
        # equal scores: weights of exactly 1, sums of up to 40 of them
        assert (np.abs(out.get() - want) <= 64 * 2.0 ** -23 * np.abs(vd).max()).all()


def test_scale_zero_and_equal_scores():
    """Every weight the same: the mean of V."""
    c = Case(10, [333], None, 2, 64, 32)
    _check_attention(c, 6, scale=0.0)


def test_nan_tokens():
    """A token that reads as NaN: rows that see it get NaN (V: in its block's elements), others their values."""
    for hd in (64, 128, 256):
        for part in ("k", "v"):
            c = Case(11 + hd, [90], [60], 2, hd, 32, junk=False)
            t, head, blk = 70, 1, hd // 32 - 1
            x = c.k if part == "k" else c.v
            x[c.slot(0, t), head, 32 * blk + 3] = np.nan
            c.bytes = mx_ref.pages(c.k, c.v, c.page)
            clean = x.copy()
            clean[c.slot(0, t), head, 32 * blk:32 * blk + 32] = 0
            wide, heads = 4 * hd, 4
            for window in (0, 9):
                q = c.rng.standard_normal((c.n_rows, heads, hd)).astype(np.float32)
                out, qd = Dev.empty((c.n_rows, wide)), Dev(q)
                cache, batch = c.upload()
                check(lib().atlas_kv4_attention_f32(cache, batch, qd.ptr, wide, heads, hd ** -0.5, window, out.ptr, wide))
                sync()
                got = out.get().reshape(c.n_rows, heads, hd)
                want = np.zeros(got.shape, bool)
                for row, s, pos in c.each_row():
                    if t <= pos and (not window or t > pos - window):
                        want[row, 2:, slice(None) if part == "k" else slice(32 * blk, 32 * blk + 32)] = True
                np.testing.assert_array_equal(np.isnan(got), want)
                kd = mx_ref.rounded(clean if part == "k" else c.k)
                vd = mx_ref.rounded(clean if part == "v" else c.v)
                for row, s, pos in c.each_row():
                    keys = np.arange(pos + 1)
                    at = np.array([c.slot(0, i) for i in keys])
                    ref = mx_ref.attend(q[row], keys, kd[at], vd[at], pos, hd ** -0.5, window)
                    bound = _bound(q[row], keys, kd[at], vd[at], pos, hd ** -0.5, window)
                    ok = ~want[row]
                    assert (np.abs(got[row] - ref)[ok] <= bound[ok]).all()


def test_query_not_finite():
    """A row with NaN or an infinity in q is NaN; its neighbours are not touched."""
    c = Case(12, [50], [8], 1, 128, 32)
    cache, batch = c.upload()
    q = c.rng.standard_normal((8, 2, 128)).astype(np.float32)
    q[2, 1, 7], q[5, 0, 100], q[6, 0, 0] = np.nan, np.inf, -np.inf
    out, qd = Dev.empty((8, 256)), Dev(q)
    check(lib().atlas_kv4_attention_f32(cache, batch, qd.ptr, 256, 2, 0.1, 0, out.ptr, 256))
    sync()
    want = np.zeros((8, 2, 128), bool)
    want[2, 1], want[5, 0], want[6, 0] = True, True, True
    np.testing.assert_array_equal(np.isnan(out.get().reshape(8, 2, 128)), want)


def test_same_bits_again():
    c = Case(13, [700, 90, 1500], None, 2, 128, 64)
    args = c.upload()
    q = Dev(c.rng.standard_normal((3, 4 * 128)).astype(np.float32))
    outs = []
    for _ in range(4):
        out = Dev.empty((3, 512))
        check(lib().atlas_kv4_attention_f32(*args, q.ptr, 512, 4, 0.09, 0, out.ptr, 512))
        sync()
        outs.append(out.get())
    for x in outs[1:]:
        np.testing.assert_array_equal(x, outs[0])


def test_cache_past_4_gib():
    """Pages whose bytes lie past 32-bit offsets."""
    n_kv, hd, page = 32, 128, 64
    c = Case(14, [150], [150], n_kv, hd, page, spare=0, junk=False)
    per = c.bytes[0].size
    n_pages = (5 << 30) // per
    big = Dev(np.zeros(1, np.uint8))
    from atlas_amd.tensor import _DevMem
    big.mem = _DevMem(n_pages * per, sync_alloc=True)
    c.d = None
    cache, batch = c.upload()
    c.table = np.array([[n_pages - 1, 3, n_pages - 2]], np.int32)
    c.d["table"] = Dev(c.table)
    c.c = Kv4CacheC(big.mem.ptr, n_pages, page, n_kv, hd)
    c.b.block_table = c.d["table"].ptr
    args = C.byref(c.c), C.byref(c.b)
    wide = n_kv * hd
    k, v = (c.rng.standard_normal((150, n_kv, hd)).astype(np.float32) for _ in range(2))
    kd, vd, ko, vo = Dev(k), Dev(v), Dev.empty(k.shape), Dev.empty(v.shape)
    check(lib().atlas_kv4_write_f32(*args, kd.ptr, vd.ptr, wide))
    check(lib().atlas_kv4_read_f32(*args, ko.ptr, vo.ptr, wide))
    sync()
    kr, vr = mx_ref.rounded(k), mx_ref.rounded(v)
    np.testing.assert_array_equal(ko.get(), kr.astype(np.float32))
    np.testing.assert_array_equal(vo.get(), vr.astype(np.float32))
    q, out = c.rng.standard_normal((150, n_kv, hd)).astype(np.float32), Dev.empty((150, wide))
    qd = Dev(q)
    check(lib().atlas_kv4_attention_f32(*args, qd.ptr, wide, n_kv, hd ** -0.5, 0, out.ptr, wide))
    sync()
    got = out.get().reshape(150, n_kv, hd)
    for pos in (0, 63, 64, 149):
        keys = np.arange(pos + 1)
        ref = mx_ref.attend(q[pos], keys, kr[keys], vr[keys], pos, hd ** -0.5, 0)
        assert (np.abs(got[pos] - ref) <= _bound(q[pos], keys, kr[keys], vr[keys], pos, hd ** -0.5, 0)).all()


def test_classes():
    """GpuKv4Cache and Kv4Batch: a prompt, then decode steps of two sequences, as a program uses them."""
    from atlas_amd.tensor import AtlasError, GpuKv4Cache, GpuVec, Kv4Batch
    n_kv, hd, heads, page = 2, 64, 6, 32
    cache = GpuKv4Cache.new(8, page, n_kv, hd)
    rng = np.random.default_rng(4)
    table = [[5, 1, 7], [0, 3, -1]]
    have = [np.zeros((0, 2, n_kv, hd)), np.zeros((0, 2, n_kv, hd))]
    lens = [0, 0]
    for rows in ([40, 7], [1, 1], [1, 20], [1, 1], [0, 1], [25, 0]):
        lens = [a + b for a, b in zip(lens, rows)]
        batch = Kv4Batch(lens, table, None if rows == [1, 1] else rows)
        n = sum(rows)
        k, v = (rng.standard_normal((n, n_kv, hd)).astype(np.float32) for _ in range(2))
        q = rng.standard_normal((n, heads, hd)).astype(np.float32)
        cache.write(batch, GpuVec.from_slice(k), GpuVec.from_slice(v))
        kr, vr = cache.read(batch)
        np.testing.assert_array_equal(kr.download().reshape(k.shape), mx_ref.rounded(k).astype(np.float32))
        np.testing.assert_array_equal(vr.download().reshape(v.shape), mx_ref.rounded(v).astype(np.float32))
        got = cache.attention(batch, GpuVec.from_slice(q), heads, hd ** -0.5, 30).download().reshape(q.shape)
        at = 0
        for s in range(2):
            new = np.stack([mx_ref.rounded(k[at:at + rows[s]]), mx_ref.rounded(v[at:at + rows[s]])], 1)
            have[s] = np.concatenate([have[s], new])
            for i in range(rows[s]):
                pos = lens[s] - rows[s] + i
                keys = np.arange(lens[s])
                args = q[at + i], keys, have[s][:, 0], have[s][:, 1], pos, hd ** -0.5, 30
                assert (np.abs(got[at + i] - mx_ref.attend(*args)) <= _bound(*args)).all()
            at += rows[s]
    with pytest.raises(AtlasError):
        cache.write(Kv4Batch([3], [[0]]), GpuVec.zeros(8), GpuVec.zeros(8))
    with pytest.raises(AtlasError):
        cache.attention(Kv4Batch([3], [[0]]), GpuVec.zeros(7 * hd), 7, 1.0)


def _step(c, args, bufs, heads):
    """Write the new rows, attend: the calls of a layer's step."""
    wide, hd = c.n_kv * c.hd, c.hd
    check(lib().atlas_kv4_write_f32(*args, bufs["k"].ptr, bufs["v"].ptr, wide))
    return lib().atlas_kv4_attention_f32(*args, bufs["q"].ptr, heads * hd, heads, hd ** -0.5, 0, bufs["out"].ptr, heads * hd)


def _bufs(c, heads):
    wide = c.n_kv * c.hd
    return dict(k=Dev.empty((c.n_rows, wide)), v=Dev.empty((c.n_rows, wide)), q=Dev.empty((c.n_rows, heads * c.hd)),
                out=Dev.empty((c.n_rows, heads * c.hd)))


def _put(dev, x):
    x = np.ascontiguousarray(x)
    check(lib().atlas_memcpy_h2d(dev.ptr, x.ctypes.data_as(C.c_void_p), x.nbytes))


def _check_step(c, bufs, heads, rng, run):
    """New rows for the batch as its lengths are now; run() the step; compare."""
    k, v = (rng.standard_normal((c.n_rows, c.n_kv, c.hd)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((c.n_rows, heads, c.hd)).astype(np.float32)
    for name, x in (("k", k), ("v", v), ("q", q)):
        _put(bufs[name], x)
    _put(bufs["out"], np.full(q.shape, 7, np.float32))
    run()
    got = bufs["out"].get().reshape(q.shape)
    for row, s, pos in c.each_row():
        c.k[c.slot(s, pos)], c.v[c.slot(s, pos)] = k[row], v[row]
    kd, vd = mx_ref.rounded(c.k), mx_ref.rounded(c.v)
    for row, s, pos in c.each_row():
        keys = np.arange(pos + 1)
        at = np.array([c.slot(s, t) for t in keys])
        args = q[row], keys, kd[at], vd[at], pos, c.hd ** -0.5, 0
        assert (np.abs(got[row] - mx_ref.attend(*args)) <= _bound(*args)).all(), (row, s, pos)


@pytest.mark.parametrize("lens", [[30, 900, 5], [2400]])
def test_decode_steps_in_a_graph(lens):
    """A captured step replayed while the lengths on the device grow, with eager steps in between."""
    def work(hip):
        heads = 4
        c = Case(20, [n + 8 for n in lens], None, 2, 64, 32, junk=False)
        c.lens = list(lens)
        args = c.upload()
        bufs = _bufs(c, heads)
        with Stream(hip) as st:
            def run():
                assert _step(c, args, bufs, heads) == 0

            rng = np.random.default_rng(3)
            _check_step(c, bufs, heads, rng, run)
            exe, _ = st.capture(run)
            for i in range(7):
                c.lens = [n + 1 for n in c.lens]
                _put(c.d["lens"], np.asarray(c.lens, np.int32))
                _check_step(c, bufs, heads, rng, run if i == 3 else lambda: st.launch(exe))

    on_thread(work)


def test_two_graphs_and_two_streams():
    """Graphs of two batches replayed in turn, and eager calls of both on two streams at once: each has its own results."""
    def work(hip):
        heads = 6
        cs = [Case(30, [700, 20], None, 2, 128, 32), Case(31, [64, 1300, 9], None, 2, 128, 64)]
        qs = [c.rng.standard_normal((c.n_rows, heads * 128)).astype(np.float32) for c in cs]
        args, q = [c.upload() for c in cs], [Dev(x) for x in qs]
        outs = [Dev.empty(x.shape) for x in qs]

        def call(i):
            assert lib().atlas_kv4_attention_f32(*args[i], q[i].ptr, heads * 128, heads, 0.09, 0, outs[i].ptr, heads * 128) == 0

        with Stream(hip) as a, Stream(hip) as b:
            want = []
            for i, st in enumerate((a, b)):
                st.use()
                call(i)
                st.sync()
                want.append(outs[i].get())
            graphs = []
            for i in (0, 1):
                a.use()
                call(i)
                a.sync()
                graphs.append(a.capture(lambda: call(i))[0])
            for turn in range(4):
                for o in outs:
                    check(lib().atlas_memset_zero(o.ptr, o.a.nbytes))
                for i in (turn % 2, 1 - turn % 2):
                    a.launch(graphs[i])
                a.sync()
                for i in (0, 1):
                    np.testing.assert_array_equal(outs[i].get(), want[i])
            for _ in range(10):
                for i, st in enumerate((a, b)):
                    st.use()
                    call(i)
            a.sync(), b.sync()
            for i in (0, 1):
                np.testing.assert_array_equal(outs[i].get(), want[i])
        for i, c in enumerate(cs):
            kd, vd = mx_ref.rounded(c.k), mx_ref.rounded(c.v)
            for row, s, pos in c.each_row():
                keys = np.arange(pos + 1)
                at = np.array([c.slot(s, t) for t in keys])
                w = qs[i][row].reshape(heads, 128), keys, kd[at], vd[at], pos, 0.09, 0
                assert (np.abs(want[i][row].reshape(heads, 128) - mx_ref.attend(*w)) <= _bound(*w)).all()

    on_thread(work)


def test_capture_that_has_to_grow():
    """A captured call that needs more scratch than the thread has is refused; after an eager one it is recorded."""
    def work(hip):
        heads, hd = 4, 64
        c = Case(40, [3000], None, 2, hd, 64)
        args = c.upload()
        q = c.rng.standard_normal((1, heads * hd)).astype(np.float32)
        qd, out = Dev(q), Dev(np.full(q.shape, 7, np.float32))

        def call():
            return lib().atlas_kv4_attention_f32(*args, qd.ptr, heads * hd, heads, 0.1, 0, out.ptr, heads * hd)

        with Stream(hip) as st:
            def refused():
                rc = call()
                # (a kernel for the graph to hold)
                assert lib().atlas_kv4_write_f32(*args, out.ptr, out.ptr, 2 * hd) == 0
                return rc

            _, rc = st.capture(refused)
            assert rc == -4 and b"scratch" in lib().atlas_last_error()
            lib().atlas_clear_error()
            st.sync()
            assert (out.get() == 7).all()
            assert call() == 0
            st.sync()
            want = out.get()
            exe, rc = st.capture(call)
            assert rc == 0
            for _ in range(3):
                check(lib().atlas_memset_zero(out.ptr, out.a.nbytes))
                st.launch(exe)
                st.sync()
                np.testing.assert_array_equal(out.get(), want)

    on_thread(work)


def test_two_threads():
    """Calls of two threads on streams of their own at once: each thread has its own scratch."""
    import threading
    heads, hd = 8, 128
    cs = [Case(50 + i, [1500 + 700 * i, 40], None, 2, hd, 64) for i in range(2)]
    args = [c.upload() for c in cs]
    q = [Dev(c.rng.standard_normal((2, heads * hd)).astype(np.float32)) for c in cs]
    outs = [[Dev(np.zeros((2, heads * hd), np.float32)) for _ in range(12)] for _ in cs]

    def call(i, out):
        assert lib().atlas_kv4_attention_f32(*args[i], q[i].ptr, heads * hd, heads, 0.1, 0, out.ptr, heads * hd) == 0

    for i in range(2):
        call(i, outs[i][0])
    sync()
    want, gate = [outs[i][0].get() for i in range(2)], threading.Barrier(2)

    def work(i):
        def run(hip):
            with Stream(hip) as st:
                gate.wait(60)
                for out in outs[i][1:]:
                    call(i, out)
                st.sync()
        return run

    threads = [threading.Thread(target=on_thread, args=(work(i),)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        for out in outs[i][1:]:
            np.testing.assert_array_equal(out.get(), want[i])


def test_nothing_and_no_memory():
    """Batches without sequences or rows; allocations that fail."""
    from atlas_amd.quant import MxFp4Tensor
    from atlas_amd.tensor import GpuKv4Cache, GpuMatrix, GpuVec, Kv4Batch
    cache = GpuKv4Cache.new(2, 32, 1, 64)
    for batch in (Kv4Batch([], []), Kv4Batch([5, 0], [[0], [1]], [0, 0])):
        none = GpuVec.zeros(0)
        cache.write(batch, none, none)
        assert cache.read(batch)[0].len == 0
        assert cache.attention(batch, none, 2, 1.0).len == 0
    g = GpuMatrix.upload_mxfp4(MxFp4Tensor.quantize(np.ones((64, 64), np.float32)))
    x, out = np.ones((64, 1), np.float32), np.zeros((64, 1), np.float32)

    def work(hip):
        c = Case(60, [3000], None, 2, 64, 64)
        args = c.upload()
        q = Dev(np.ones((1, 256), np.float32))
        try:
            for skip in (0, 1):                            # the counters, the partial sums
                lib().atlas_debug_fail_allocations(skip, 1)
                assert lib().atlas_kv4_attention_f32(*args, q.ptr, 256, 4, 0.1, 0, q.ptr, 256) == -3
                lib().atlas_clear_error()
            lib().atlas_debug_fail_allocations(0, 1)
            assert GpuKv4Cache.new(2, 32, 1, 64) is None
            lib().atlas_debug_fail_allocations(2, 1)       # the activations' codes, after x and out
            assert not g.sgemm(x, 64, 1, out)
        finally:
            lib().atlas_debug_fail_allocations(0, 0)
            lib().atlas_clear_error()
        _check_attention(c, 4, args=args)
        assert g.sgemm(x, 64, 1, out) and (out == 64).all()

    on_thread(work)


def test_rows_without_memory():
    """Results of the cache's class that find no memory are reported; the cache is as it was."""
    from atlas_amd.tensor import AtlasError, GpuKv4Cache, GpuVec, Kv4Batch
    cache, batch = GpuKv4Cache.new(2, 32, 1, 64), Kv4Batch([3], [[1]], [3])
    x = np.random.default_rng(8).standard_normal((3, 64)).astype(np.float32)
    k = GpuVec.from_slice(x)
    cache.write(batch, k, k)
    try:
        for skip, call in [(0, lambda: cache.read(batch)), (1, lambda: cache.read(batch)),
                           (0, lambda: cache.attention(batch, k, 1, 0.1))]:
            lib().atlas_debug_fail_allocations(skip, 1)
            with pytest.raises(AtlasError) as bad:
                call()
            assert bad.value.code == -3
    finally:
        lib().atlas_debug_fail_allocations(0, 0)
    np.testing.assert_array_equal(cache.read(batch)[1].download().reshape(3, 64), mx_ref.rounded(x).astype(np.float32))


@pytest.mark.parametrize("have", [45, 50, 61, 64])
@pytest.mark.parametrize("heads", [2, 16])
def test_fewer_rows_than_the_starts_count(have, heads):
    """Buffers that end inside a sequence's rows: each row that is there is the token that row_starts make it."""
    c = Case(70 + have, [70, 40], [40, 25], 2, 64, 32)
    wide = 2 * 64
    k, v = (c.rng.standard_normal((have, 2, 64)).astype(np.float32) for _ in range(2))
    q = c.rng.standard_normal((have, heads, 64)).astype(np.float32)
    args = c.upload()
    c.b.n_rows = have
    kd, vd, qd = Dev(k), Dev(v), Dev(q)
    ko, vo, out = Dev(np.zeros_like(k)), Dev(np.zeros_like(v)), Dev(np.zeros_like(q))
    check(lib().atlas_kv4_write_f32(*args, kd.ptr, vd.ptr, wide))
    check(lib().atlas_kv4_read_f32(*args, ko.ptr, vo.ptr, wide))
    check(lib().atlas_kv4_attention_f32(*args, qd.ptr, heads * 64, heads, 0.125, 0, out.ptr, heads * 64))
    sync()
    np.testing.assert_array_equal(ko.get(), mx_ref.rounded(k).astype(np.float32))
    rows = [(row, s, pos) for row, s, pos in c.each_row() if row < have]
    for row, s, pos in rows:
        c.k[c.slot(s, pos)], c.v[c.slot(s, pos)] = k[row], v[row]
    kr, vr, got = mx_ref.rounded(c.k), mx_ref.rounded(c.v), out.get()
    for row, s, pos in rows:
        keys = np.arange(pos + 1)
        at = np.array([c.slot(s, t) for t in keys])
        x = q[row], keys, kr[at], vr[at], pos, 0.125, 0
        assert (np.abs(got[row] - mx_ref.attend(*x)) <= _bound(*x)).all(), (row, s, pos)


def _left(case, scale, *terms):
    """Error and limit of the outputs of a case of tests/kv4_parts.py."""
    c, heads, q = case
    at, want, size, parts = kv4_parts.outputs(c, heads, q, scale, kv4_parts.Q_PARTS, 3)
    qd, out, wide = Dev(q), Dev.empty(q.shape), heads * c.hd
    check(lib().atlas_kv4_attention_f32(*c.upload(), qd.ptr, wide, heads, scale, 0, out.ptr, wide))
    sync()
    left, limit = kv4_parts.error(out.get()[at], want, size), kv4_parts.limit(parts, want, size, *terms)
    print(f"{left:.2e}, the parts {kv4_parts.error(parts, want, size):.2e}, limit {limit:.2e}", flush=True)
    return left, limit


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("form", kv4_parts.FORMS)
def test_parts_of_q_and_of_the_weights(hd, form):
    """As exact as the documented parts are: within a bound that two parts of q less, or one of the weights', pass
    (tests/test_kv4_parts.py)."""
    left, limit = _left(kv4_parts.case(Case, hd, form), hd ** -0.5)
    assert left <= limit


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("form", kv4_parts.SHORT_FORMS)
def test_every_part_of_q(hd, form):
    """Few tokens and scores far apart, and a bound that one part of q less passes."""
    case = kv4_parts.short_case(Case, hd, form)
    left, limit = _left(case, kv4_parts.SHORT_SCALE * hd ** -0.5, kv4_parts.SHORT_STEPS, 2)
    assert left <= limit


def _check_bad_tokens(c, heads, bad, window, q=None, blind=()):
    """NaN where a row sees one of the tokens `bad` ((sequence, token, head, block of V or None for K)) or its q is not
    finite (unless it sees nothing: rows `blind`), values elsewhere; twice, for what the first call leaves."""
    hd, n_kv = c.hd, c.n_kv
    k, v = c.k.copy(), c.v.copy()
    for s, t, head, blk in bad:
        at = c.slot(s, t)
        if blk is None:
            c.k[at, head, 5], k[at, head, :32] = np.nan, 0
        else:
            c.v[at, head, 32 * blk + 3], v[at, head, 32 * blk:32 * blk + 32] = np.nan, 0
    c.bytes = mx_ref.pages(c.k, c.v, c.page)
    k, v = mx_ref.rounded(k), mx_ref.rounded(v)
    if q is None:
        q = c.rng.standard_normal((c.n_rows, heads, hd)).astype(np.float32)
    want, per = np.zeros(q.shape, bool), heads // n_kv
    for row, s, pos in c.each_row():
        for seq, t, head, blk in bad:
            if seq == s and t <= pos and (not window or t > pos - window):
                want[row, head * per:(head + 1) * per, slice(None) if blk is None else slice(32 * blk, 32 * blk + 32)] = True
        if row not in blind:
            want[row, ~np.isfinite(q[row]).all(-1)] = True
    args, qd = c.upload(), Dev(q)
    for _ in range(2):
        out = Dev(np.full(q.shape, 7, np.float32))
        check(lib().atlas_kv4_attention_f32(*args, qd.ptr, heads * hd, heads, hd ** -0.5, window, out.ptr, heads * hd))
        sync()
        got = out.get()
        np.testing.assert_array_equal(np.isnan(got), want)
    clean = np.where(np.isfinite(q).all(-1, keepdims=True), q, 0)
    for row, s, pos in list(c.each_row())[::1 if c.n_rows < 16 else 9]:
        keys = np.array([t for t in range(pos + 1) if c.slot(s, t) is not None], np.int64)
        at = np.array([c.slot(s, t) for t in keys], np.int64)
        x = clean[row], keys, k[at], v[at], pos, hd ** -0.5, window
        ok = ~want[row]
        assert (np.abs(got[row] - mx_ref.attend(*x))[ok] <= _bound(*x)[ok]).all(), (row, s, pos)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("part", ["k", "v"])
@pytest.mark.parametrize("rows,group", [(1, 2), (5, 1), (70, 4)])
def test_nan_tokens_in_runs(hd, part, rows, group):
    """Several blocks to a sequence, 16 and 32 columns: NaN in a first, a middle and the last run, in each block of V."""
    for bad, window in [([1200], 0), ([2499], 0), ([2455], 0), ([1100, 2410], 1400), ([10, 900], 1400)]:
        c = Case(hd + rows + len(bad), [2500, 1500], None if rows == 1 else [rows, 1], 2, hd, 64, junk=False)
        tokens = [(0, t, i % 2, None if part == "k" else t % (hd // 32)) for i, t in enumerate(bad)]
        _check_bad_tokens(c, 2 * group, tokens, window)


@pytest.mark.parametrize("hd,group", [(64, 2), (128, 1), (128, 2), (256, 2)])
def test_query_not_finite_in_runs(hd, group):
    c = Case(90 + hd, [2500], [90], 2, hd, 64)
    q = c.rng.standard_normal((90, 2 * group, hd)).astype(np.float32)
    q[3, 0, 1], q[40, 1, hd - 1], q[89, 0, 40] = np.nan, np.inf, -np.inf
    _check_bad_tokens(c, 2 * group, [], 0, q)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_query_not_finite_and_nothing_to_see(hd):
    """A row that sees no token is zero, whatever its q: before the sequence's start, or without a page."""
    c = Case(95 + hd, [2, 40, 2000], [5, 1, 3], 2, hd, 32, junk=False)
    c.table[1:] = -1
    q = c.rng.standard_normal((9, 4, hd)).astype(np.float32)
    q[1, 0, 1], q[4, 1, 2], q[5, 2, 3], q[7] = np.nan, np.inf, np.nan, np.inf
    _check_bad_tokens(c, 4, [], 0, q, blind=(0, 1, 2, 5, 6, 7, 8))


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_scale_bytes_past_the_encoders(hd):
    """V's scale bytes 253 and 254, from elsewhere: NaN to the rows that see their token, nothing to the others;
    252, the largest that is encoded, is a scale as any."""
    c = Case(97 + hd, [90], [60], 1, hd, 32, junk=False)
    d, kb = 16 * hd, hd // 32
    seen = {253: 45, 254: 62, 255: 80}
    c.v[c.slot(0, 33), 0, hd - 32:] = 0                    # codes of 0, whose scale changes nothing
    c.bytes = mx_ref.pages(c.k, c.v, 32)
    for byte, t in [(252, 33)] + list(seen.items()):
        at = c.slot(0, t)
        c.bytes[at // 32, 0, 2 * d + kb * 32:].reshape(4, kb, 8)[at % 32 // 8, kb - 1, at % 8] = byte
    q = c.rng.standard_normal((60, 1, hd)).astype(np.float32)
    for window in (0, 10):
        args, qd, out = c.upload(), Dev(q), Dev.empty(q.shape)
        check(lib().atlas_kv4_attention_f32(*args, qd.ptr, hd, 1, hd ** -0.5, window, out.ptr, hd))
        sync()
        want = np.zeros((60, 1, hd), bool)
        for row, s, pos in c.each_row():
            want[row, 0, hd - 32:] = any(t <= pos and (not window or t > pos - window) for t in seen.values())
        np.testing.assert_array_equal(np.isnan(out.get()), want)
        assert np.isfinite(out.get()[~want]).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_values_at_the_documented_limit(hd):
    """Elements of V that sum to 0.94 2^119 over 160 tokens, under weights that grow to 2^7.9 without a new maximum
    (chunks of 32 tokens; the fifth follows the first in its wave)."""
    c = Case(98 + hd, [160], None, 1, hd, 32)
    at = np.array([c.slot(0, t) for t in range(160)])
    c.k[:] = 0
    c.k[at[128:], 0, 0] = 1
    c.v[:] = 1.5 * 2.0 ** 111 * np.where(c.rng.random(c.v.shape) < 0.02, -1, 1)
    c.bytes = mx_ref.pages(c.k, c.v, 32)
    q = np.zeros((1, 1, hd), np.float32)
    q[0, 0, 0] = 7.9 * np.log(2)
    args, qd, out = c.upload(), Dev(q), Dev.empty(q.shape)
    check(lib().atlas_kv4_attention_f32(*args, qd.ptr, hd, 1, 1.0, 0, out.ptr, hd))
    sync()
    x = q[0], np.arange(160), mx_ref.rounded(c.k)[at], mx_ref.rounded(c.v)[at], 159, 1.0, 0
    assert (np.abs(out.get()[0] - mx_ref.attend(*x)) <= _bound(*x)).all()


@pytest.mark.parametrize("hd", [64, 256])
def test_caches_and_tables_without_pages(hd):
    """A cache of no pages, a table of no columns, lengths below zero: nothing is there, and nothing is touched."""
    rows = Dev(np.ones((4, 2 * hd), np.float32))
    lens, starts, table = Dev(np.array([70, -3], np.int32)), Dev(np.array([0, 3, 4], np.int32)), Dev(np.zeros((2, 3), np.int32))
    page = Dev(np.full((2, 32 * hd * 17 // 16), 0xA5, np.uint8))
    past = Dev(np.ones((2, 3), np.int32))
    for cache, table_ptr, stride in [(Kv4CacheC(None, 0, 32, 2, hd), table.ptr, 3), (Kv4CacheC(page.ptr, 1, 32, 2, hd), None, 0),
                                     (Kv4CacheC(page.ptr, 1, 32, 2, hd), past.ptr, 3)]:
        for starts_ptr, n_rows in ((starts.ptr, 4), (None, 2)):
            batch = Kv4BatchC(starts_ptr, lens.ptr, table_ptr, stride, 2, n_rows, 0)
            args = C.byref(cache), C.byref(batch)
            ko, vo, out = (Dev(np.full((4, 2 * hd), 7, np.float32)) for _ in range(3))
            check(lib().atlas_kv4_write_f32(*args, rows.ptr, rows.ptr, 2 * hd))
            check(lib().atlas_kv4_read_f32(*args, ko.ptr, vo.ptr, 2 * hd))
            check(lib().atlas_kv4_attention_f32(*args, rows.ptr, 2 * hd, 2, 1.0, 0, out.ptr, 2 * hd))
            sync()
            want = np.zeros((4, 2 * hd), np.float32)
            want[n_rows:] = 7
            for x in (ko, vo, out):
                np.testing.assert_array_equal(x.get(), want)
    assert (page.get() == 0xA5).all()


def test_lengths_below_zero_beside_others():
    """A sequence of length -1 or the least int32 sees nothing; its neighbour is not touched."""
    c = Case(99, [40, 64, 33], None, 2, 64, 32)
    args = c.upload()
    _put(c.d["lens"], np.array([-1, 64, -(1 << 31)], np.int32))
    q = c.rng.standard_normal((3, 4, 64)).astype(np.float32)
    qd, out = Dev(q), Dev.empty(q.shape)
    check(lib().atlas_kv4_attention_f32(*args, qd.ptr, 256, 4, 0.125, 0, out.ptr, 256))
    sync()
    got, keys = out.get(), np.arange(64)
    assert (got[[0, 2]] == 0).all()
    at = np.array([c.slot(1, t) for t in keys])
    x = q[1], keys, mx_ref.rounded(c.k)[at], mx_ref.rounded(c.v)[at], 63, 0.125, 0
    assert (np.abs(got[1] - mx_ref.attend(*x)) <= _bound(*x)).all()


@pytest.mark.parametrize("lens,rows,heads", [([300, 40], None, 4), ([3000], None, 4), ([150, 40], [150, 9], 8), ([2500], [90], 4)])
def test_attention_into_its_query(lens, rows, heads):
    """out may be q: a tile's rows and heads are read by its own blocks, all of them before the results are stored."""
    for hd in (64, 128, 256):
        c = Case(sum(lens) + hd, lens, rows, 2, hd, 32)
        args = c.upload()
        q = c.rng.standard_normal((c.n_rows, heads, hd)).astype(np.float32)
        qd, both, out = Dev(q), Dev(q), Dev.empty(q.shape)
        for to, src in ((out, qd), (both, both)):
            check(lib().atlas_kv4_attention_f32(*args, src.ptr, heads * hd, heads, hd ** -0.5, 0, to.ptr, heads * hd))
        sync()
        np.testing.assert_array_equal(both.get(), out.get())
