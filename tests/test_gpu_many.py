"""Attention over shared prefixes, beam selection, reordering of states and low-rank adapters on the
device, against 64 bits."""
import ctypes as C
import threading

import numpy as np
import pytest

from atlas_amd import tensor as T
from atlas_amd._lib import AtlasError, LoraC, PrefixBatchC, SlotCacheC, check
from tests import many_ref
from tests.gpu_util import Dev, lib, sync
from tests.stream_util import Stream, on_thread

pytestmark = pytest.mark.gpu


# ---- attention over shared prefixes ------------------------------------------------


class Batch:
    """Random slots and a batch over them, on the host and on the device.  Groups of `sizes` rows with
    prefixes of `prefix` tokens; `own` tokens of each row.  table: a slot for each token, drawn anew."""

    def __init__(self, seed, sizes, prefix, own, n_kv=2, group=2, hd=64, table=True, stride=None, extra_rows=0, slack=3,
                 junk=True, pad_q=0):
        rng = self.rng = np.random.default_rng(seed)
        n = int(np.sum(sizes))
        self.n, self.hd, self.n_kv, self.heads = n, hd, n_kv, n_kv * group
        self.starts = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
        self.prefix = np.asarray(prefix, np.int32)
        which = np.repeat(np.arange(len(sizes)), sizes)
        self.lens = np.concatenate([self.prefix[which] + np.asarray(own), np.full(extra_rows, 5)]).astype(np.int32)
        self.max_seq = int(max([1, *self.lens])) + slack
        self.n_slots = max(n, 1) + len(sizes)
        self.prefix_slots = (max(n, 1) + rng.permutation(len(sizes))).astype(np.int32)
        most = max([1, *own])
        if table:
            self.slots = rng.integers(0, max(n, 1), (n + extra_rows, most if stride is None else stride)).astype(np.int32)
        else:
            self.slots = rng.permutation(n + extra_rows).astype(np.int32) % max(n, 1)
        shape = (self.n_slots, self.max_seq, n_kv, hd)
        self.k = (rng.standard_normal(shape) * np.exp(0.5 * rng.standard_normal((n_kv, hd)))).astype(np.float32)
        self.v = rng.standard_normal(shape).astype(np.float32)
        if junk:                       # what no row sees is anything
            seen = np.zeros(shape[:2], bool)
            for g in range(len(sizes)):
                seen[self.prefix_slots[g], :self.prefix[g]] = True
                for r in range(self.starts[g], self.starts[g + 1]):
                    for t in range(self.prefix[g], self.lens[r]):
                        i = t - self.prefix[g]
                        s = self.slots[r] if not table else self.slots[r, i] if i < self.slots.shape[1] else -1
                        if s >= 0:
                            seen[s, t] = True
            self.k[~seen] = np.nan
            self.v[~seen] = np.inf
        self.q = rng.standard_normal((n + extra_rows, self.heads * hd + pad_q)).astype(np.float32)

    def upload(self, one_group=False, hints=True):
        self.d = {x: Dev(getattr(self, x)) for x in ("k", "v", "q", "starts", "prefix", "prefix_slots", "lens", "slots")}
        self.c = SlotCacheC(self.d["k"].ptr, self.d["v"].ptr, self.n_slots, self.max_seq, self.n_kv, self.hd)
        stride = self.slots.shape[1] if self.slots.ndim == 2 else 0
        own = int(max(0, (self.lens[:self.n] - np.repeat(self.prefix, np.diff(self.starts))).max(initial=0)))
        self.b = PrefixBatchC(None if one_group else self.d["starts"].ptr, self.d["prefix_slots"].ptr, self.d["prefix"].ptr,
                              self.d["lens"].ptr, self.d["slots"].ptr, stride, len(self.prefix), len(self.lens),
                              int(self.prefix.max()) if hints else 0, own if hints else 0)
        return self

    def call(self, out, window=0, scale=None):
        check(lib().atlas_prefix_attention_f32(C.byref(self.c), C.byref(self.b), self.d["q"].ptr, self.q.shape[1], self.heads,
                                               self.hd ** -0.5 if scale is None else scale, window, out.ptr, out.a.shape[1]))

    def want(self, window=0, scale=None, out=None):
        q = self.q[:, :self.heads * self.hd].reshape(-1, self.heads, self.hd)
        return many_ref.attention(self.k, self.v, q, self.lens, self.starts, self.prefix_slots, self.prefix, self.slots,
                                  self.hd ** -0.5 if scale is None else scale, window, out)

    def check(self, window=0, scale=None, pad_out=0, out=None):
        wide = self.heads * self.hd
        out = Dev(np.full((len(self.lens), wide + pad_out), 7, np.float32)) if out is None else out
        self.call(out, window, scale)
        got = out.get()
        want, off = self.want(window, scale, np.full((len(self.lens), self.heads, self.hd), 7.0))
        _near(got[:, :wide].reshape(want.shape), want, off[..., None])
        assert (got[:, wide:] == 7).all()
        return got


def _near(got, want, off):
    with np.errstate(invalid="ignore"):
        bad = int((~((np.abs(got - want) <= off) | (got == want) | (np.isnan(got) & np.isnan(want)))).sum())
        worst = np.nanmax(np.abs(got - want) / np.maximum(off, 1e-30), initial=0)
    assert bad == 0, f"{bad} of {got.size} values, off by up to {worst} of what they may be"


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n_kv,group", [(1, 1), (3, 3), (8, 4), (2, 16), (2, 5)])
def test_prefix_attention_shapes(hd, n_kv, group):
    Batch(1, [5], [37], [9, 0, 3, 21, 1], n_kv=n_kv, group=group, hd=hd).upload().check()


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 17, 63, 64, 257])
@pytest.mark.parametrize("table", [False, True])
def test_prefix_attention_lengths(prefix, table):
    # rows without a token of their own, and, with prefix 0, without any
    Batch(2, [6], [prefix], [0, 1, 2, 0, 33, 16], hd=64, table=table).upload().check()


@pytest.mark.parametrize("rows,group", [(1, 1), (16, 1), (17, 1), (33, 1), (64, 1), (65, 1), (130, 1), (9, 4), (40, 4), (14, 5), (23, 3)])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prefix_attention_many_rows(rows, group, hd):
    own = np.random.default_rng(3).integers(0, 25, rows)
    Batch(3, [rows], [70], own, n_kv=2, group=group, hd=hd).upload().check()


@pytest.mark.parametrize("hd,group", [(64, 4), (128, 1), (256, 2)])
@pytest.mark.parametrize("window", [0, 1, 16, 40, 300])
def test_prefix_attention_groups_and_windows(hd, group, window):
    # groups of different sizes, one of them empty, rows behind the last group left as they were
    sizes, prefix = [3, 0, 1, 12], [90, 5, 1, 333]
    own = [0, 50, 7, 1, 3, 0, 100, 2, 64, 17, 5, 5, 5, 31, 1, 8]
    Batch(4, sizes, prefix, own, group=group, hd=hd, extra_rows=3).upload().check(window=window)


@pytest.mark.parametrize("hints", [False, True])
@pytest.mark.parametrize("hd,n_kv,group", [(128, 8, 1), (64, 1, 4), (128, 32, 1), (256, 1, 2)])
def test_prefix_attention_long(hd, n_kv, group, hints):
    # several blocks to a tile, which the last one joins
    b = Batch(5, [7], [3001], [97, 0, 97, 300, 97, 1, 97], n_kv=n_kv, group=group, hd=hd)
    if not hints:
        b.slots = b.slots[:, :150]     # a table that ends before a row's tokens do
        b.v[~np.isfinite(b.v)] = 1
        b.k[~np.isfinite(b.k)] = 1
    b.upload(hints=hints).check()


@pytest.mark.parametrize("rows,group", [(65, 1), (100, 1), (17, 4), (33, 4), (40, 2), (14, 5), (23, 3), (5, 16)])
@pytest.mark.parametrize("window", [0, 2060])
def test_prefix_attention_wide_groups_of_long_caches(rows, group, window):
    # two tiles of columns to a block, by what the cache can hold; then by the prefix
    own = np.random.default_rng(3).integers(0, 25, rows)
    Batch(3, [rows], [70], own, n_kv=1, group=group, hd=128, slack=2100, table=rows % 2 == 0).upload(hints=False).check(window=window)


def test_prefix_attention_wide_groups_over_long_prefixes():
    own = np.random.default_rng(5).integers(0, 60, 40)
    b = Batch(15, [23, 0, 17], [2100, 30, 700], own, n_kv=1, group=6, hd=128, extra_rows=2).upload()
    b.check()
    b.check(window=2080)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prefix_attention_infinities_in_the_last_of_several_runs(hd):
    b = Batch(17, [4], [1300], [9, 9, 0, 9], n_kv=1, group=3, hd=hd, table=False, junk=False)
    b.v[b.slots[3], 1308] = np.inf
    b.v[b.slots[1], 1300, 0, 2] = -np.inf
    got = b.upload().check().reshape(4, 3, hd)
    assert (got[3] == np.inf).all() and (got[1, :, 2] == -np.inf).all() and np.isfinite(got[[0, 2]]).all()


@pytest.mark.parametrize("window", [0, 2080])
def test_prefix_attention_wide_groups_with_infinities_and_nan(window):
    b = Batch(16, [20, 12], [2090, 18], [12, 3, 12, 0] * 8, n_kv=2, group=5, hd=128, table=False, junk=False)
    own = b.slots
    b.v[own[0], 2091, :, 3] = np.nan
    b.v[own[2], 2100, 1, :] = np.inf
    b.k[own[4], 2094, 0, 5] = np.nan
    b.v[b.prefix_slots[0], 4, 0, 7] = -np.inf       # the rows whose window begins after it do not see it
    b.v[b.prefix_slots[1], 2, 1, 0] = np.nan
    b.q[3] = np.nan
    b.upload().check(window=window)


def test_prefix_attention_short_lengths():
    # rows whose length ends inside the prefix, is zero or below
    b = Batch(6, [7], [60], [0] * 7, hd=128, junk=False)
    b.lens = np.array([60, 31, 1, 0, -5, 59, 16], np.int32)
    got = b.upload().check()
    assert (got[3] == 0).all() and (got[4] == 0).all()


def test_prefix_attention_slots_that_are_none():
    b = Batch(7, [4, 3, 2], [40, 20, 33], [12] * 9, hd=64, junk=False)
    b.slots[0, 3] = -1
    b.slots[1, :] = b.n_slots
    b.slots[5, 11] = 1 << 30
    b.prefix_slots[1] = -3
    b.prefix_slots[2] = b.n_slots
    b.upload().check()
    # positions past the slots' end: 40 of 45 tokens
    b.lens[:4] = 60
    b.prefix[0] = 45
    b.max_seq = 40
    b.k, b.v = b.k[:, :40].copy(), b.v[:, :40].copy()
    b.upload().check()


@pytest.mark.parametrize("window", [0, 10])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prefix_attention_infinities_and_nan(hd, window):
    # in K, V and q: nothing to the rows that do not see them
    b = Batch(8, [5, 2], [40, 18], [12, 3, 12, 0, 8, 5, 5], hd=hd, table=False, junk=False)
    own = b.slots
    b.v[own[0], 41, :, 3] = np.nan
    b.v[own[2], 50, 1, :] = np.inf
    b.k[own[4], 44, 0, 5] = np.nan
    b.v[b.prefix_slots[0], 39, 0, 7] = -np.inf      # the rows whose window ends before it do not see it
    b.v[b.prefix_slots[1], 2, 1, 0] = np.nan
    b.q[3] = np.nan
    b.upload().check(window=window)


def test_prefix_attention_query_of_row_without_tokens():
    b = Batch(9, [3], [0], [0, 4, 0], hd=64)
    b.q[0], b.q[2] = np.nan, np.inf
    assert (b.upload().check()[[0, 2]] == 0).all()


def test_prefix_attention_strides_one_group_and_in_place():
    b = Batch(10, [6], [45], [3, 8, 8, 0, 1, 30], hd=128, pad_q=12).upload(one_group=True)
    b.check(pad_out=8)
    b.q = b.q[:, :b.heads * b.hd].copy()
    b.upload(one_group=True).check(out=b.d["q"])


@pytest.mark.parametrize("one_row", [False, True])
def test_prefix_attention_rows_of_q_and_out_between_each_other(one_row):
    # both are columns of one matrix, with something behind them; a single row may be written in place at any stride
    rows, wide = 1 if one_row else 6, 4 * 64
    b = Batch(20, [rows], [45], [3, 8, 8, 0, 1, 30][:rows], pad_q=wide + 12)
    b.q[:, wide:] = 7
    b.upload()
    at = 0 if one_row else 4 * wide
    check(lib().atlas_prefix_attention_f32(C.byref(b.c), C.byref(b.b), b.d["q"].ptr, b.q.shape[1], 4, b.hd ** -0.5, 0, b.d["q"].ptr + at,
                                           wide if one_row else b.q.shape[1]))
    got, (want, off) = b.d["q"].get(), b.want()
    _near(got[:, at // 4:at // 4 + wide].reshape(want.shape), want, off[..., None])
    assert (got[:, 2 * wide:] == 7).all() and (got[:, wide:2 * wide] == 7).all() == one_row
    assert one_row or (got[:, :wide] == b.q[:, :wide]).all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_prefix_attention_scales(scale):
    Batch(11, [5], [100], [9, 2, 0, 1, 40], hd=64).upload().check(scale=scale)


def test_prefix_attention_far_slots():
    # cells past 4 GB
    n_kv, hd, max_seq, n_slots = 8, 128, 32768, 34
    total = n_slots * max_seq * n_kv * hd
    k, v = (T._DevMem(4 * total, sync_alloc=True) for _ in range(2))
    rng = np.random.default_rng(12)
    host = rng.standard_normal((2, n_slots, 6, n_kv, hd)).astype(np.float32)
    at = [0, 1, 32764, 32765, 32766, 32767]
    for s in range(n_slots):
        for x, m in enumerate((k, v)):
            for i, t in enumerate(at):
                row = np.ascontiguousarray(host[x, s, i])
                check(lib().atlas_memcpy_h2d(m.ptr + 4 * n_kv * hd * (s * max_seq + t), row.ctypes.data_as(C.c_void_p), row.nbytes))
    rows, heads, window = 3, 8, 4
    q = rng.standard_normal((rows, heads, hd)).astype(np.float32)
    slots = np.array([33, 31, 2], np.int32)
    d = [Dev(x) for x in (np.array([32], np.int32), np.array([32766], np.int32), np.array([32768, 32768, 32767], np.int32), slots)]
    dq, out = Dev(q), Dev.empty((rows, heads * hd))
    c = SlotCacheC(k.ptr, v.ptr, n_slots, max_seq, n_kv, hd)
    b = PrefixBatchC(None, d[0].ptr, d[1].ptr, d[2].ptr, d[3].ptr, 0, 1, rows, 0, 0)
    check(lib().atlas_prefix_attention_f32(C.byref(c), C.byref(b), dq.ptr, heads * hd, heads, 0.09, window, out.ptr, heads * hd))
    got = out.get().reshape(rows, heads, hd)
    for r in range(rows):
        last = [32764, 32765, 32766, 32767] if r < 2 else [32764, 32765, 32766]
        first = 0 if r < 2 else -1     # the third row's window begins at 32763, of which the cache holds anything
        if first < 0:
            continue
        cells = [(32 if t < 32766 else slots[r], at.index(t)) for t in last]
        for h in range(heads):
            kk, vv = (np.stack([host[x, s, i, h] for s, i in cells]).astype(np.float64) for x in (0, 1))
            s = kk @ q[r, h].astype(np.float64) * 0.09
            p = np.exp(s - s.max())
            off = np.abs(vv).max() * (2 * 136 * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[r, h])).max() * 0.09 + 136 * 2.0 ** -24)
            assert np.abs(got[r, h] - (p / p.sum()) @ vv).max() <= off


def test_prefix_attention_far_slots_of_rows_that_differ():
    # cells past 4 GB, rows whose windows begin in the prefix and behind it, one of them a token before the others'
    n_kv, hd, max_seq, n_slots, first = 8, 128, 32768, 34, 32763
    total = n_slots * max_seq * n_kv * hd
    mem = [T._DevMem(4 * total, sync_alloc=True) for _ in range(2)]
    rng = np.random.default_rng(23)
    host = rng.standard_normal((2, n_slots, max_seq - first, n_kv, hd)).astype(np.float32)
    for s in range(n_slots):
        for x, m in enumerate(mem):
            row = np.ascontiguousarray(host[x, s])
            check(lib().atlas_memcpy_h2d(m.ptr + 4 * n_kv * hd * (s * max_seq + first), row.ctypes.data_as(C.c_void_p), row.nbytes))
    heads, window = 8, 4
    lens, slots = np.array([32768, 32768, 32767, 32768], np.int32), np.array([33, 31, 2, 0], np.int32)
    q = rng.standard_normal((4, heads, hd)).astype(np.float32)
    d = [Dev(x) for x in (np.array([32], np.int32), np.array([32766], np.int32), lens, slots)]
    dq, out = Dev(q), Dev(np.full((4, heads * hd), 7, np.float32))
    c = SlotCacheC(mem[0].ptr, mem[1].ptr, n_slots, max_seq, n_kv, hd)
    b = PrefixBatchC(None, d[0].ptr, d[1].ptr, d[2].ptr, d[3].ptr, 0, 1, 4, 0, 0)
    check(lib().atlas_prefix_attention_f32(C.byref(c), C.byref(b), dq.ptr, heads * hd, heads, 0.09, window, out.ptr, heads * hd))
    # (the cells from `first` on, as a cache of their own)
    want, off = many_ref.attention(host[0], host[1], q, lens - first, [0, 4], [32], [32766 - first], slots, 0.09, window)
    _near(out.get().reshape(want.shape), want, off[..., None])


def test_prefix_attention_captured():
    # a captured call follows the batch's contents; eager calls between the replays
    def work(hip):
        b = Batch(13, [4, 4], [700, 90], [30] * 8, hd=128, junk=False).upload()
        out = Dev(np.zeros((8, b.heads * b.hd), np.float32))
        with Stream(hip) as s:
            b.call(out)
            s.sync()
            exe, _ = s.capture(lambda: b.call(out))
            for turn in range(4):
                b.lens = (np.repeat(b.prefix, 4) + b.rng.integers(0, 31, 8)).astype(np.int32)
                b.slots = b.rng.integers(0, b.n_slots, b.slots.shape).astype(np.int32)
                for name in ("lens", "slots"):
                    x = np.ascontiguousarray(getattr(b, name))
                    check(lib().atlas_memcpy_h2d(b.d[name].ptr, x.ctypes.data_as(C.c_void_p), x.nbytes))
                s.launch(exe)
                s.sync()
                want, off = b.want()
                _near(out.get().reshape(want.shape), want, off[..., None])
                b.call(out)
                s.sync()
    on_thread(work)


def test_prefix_attention_needs_scratch_before_a_capture():
    def work(hip):
        b = Batch(14, [4], [3000], [30] * 4, hd=128, junk=False).upload()
        out = Dev(np.zeros((4, b.heads * b.hd), np.float32))
        with Stream(hip) as s:
            def call():
                with pytest.raises(AtlasError) as e:
                    b.call(out)
                assert e.value.code == -4
            s.capture(call)
            b.call(out)
            s.sync()
    on_thread(work)


# ---- selection ---------------------------------------------------------------------


def _select(logits, scores, n_out, pad=0, shift=0):
    groups, width, vocab = logits.shape
    flat = np.full((groups * width, vocab + pad), 1e9, np.float32)
    flat[:, :vocab] = logits.reshape(-1, vocab)
    flat = np.concatenate([np.zeros(shift, np.float32), flat.reshape(-1)])
    z, s = Dev(flat), Dev(np.asarray(scores, np.float64))
    out = [Dev(np.full((groups, n_out), 99, t)) for t in (np.uint32, np.int32, np.float64)]
    check(lib().atlas_beam_select_f32(z.ptr + 4 * shift, vocab + pad, vocab, s.ptr, groups, width, n_out, *(x.ptr for x in out)))
    return [x.get() for x in out]


def _check_select(logits, scores, n_out, **kw):
    got, want = _select(logits, scores, n_out, **kw), many_ref.select(logits, np.asarray(scores, np.float64), n_out)
    assert (got[1] == want[1]).all(), (got[1], want[1])
    assert (got[0] == want[0]).all(), (got[0], want[0])
    some = want[1] >= 0
    assert (got[2][~some] == -np.inf).all()
    # 64-bit sums of up to 1e5 positive terms, exp and log: 1e-12 of a score
    assert (np.abs(got[2][some] - want[2][some]) <= 1e-12 * (1 + np.abs(want[2][some]))).all()


@pytest.mark.parametrize("vocab", [1, 3, 64, 255, 4095, 4096, 4097, 20001])
@pytest.mark.parametrize("groups,width,n_out", [(1, 1, 1), (1, 4, 8), (3, 5, 10), (2, 16, 32), (1, 64, 64), (2, 1, 64)])
def test_select(vocab, groups, width, n_out):
    rng = np.random.default_rng(vocab + width)
    logits = (3 * rng.standard_normal((groups, width, vocab))).astype(np.float32)
    _check_select(logits, -100 * rng.random((groups, width)), n_out, pad=vocab % 3)


@pytest.mark.parametrize("shift,pad", [(0, 0), (1, 0), (0, 1), (2, 2), (0, 4)])
def test_select_alignment(shift, pad):
    rng = np.random.default_rng(5)
    _check_select(rng.standard_normal((2, 3, 5000)).astype(np.float32), rng.random((2, 3)), 6, shift=shift, pad=pad)


def test_select_7b_vocabulary():
    rng = np.random.default_rng(6)
    _check_select((4 * rng.standard_normal((2, 8, 100278))).astype(np.float32), -800 * rng.random((2, 8)) ** 6, 16)


@pytest.mark.parametrize("kind", ["equal", "up", "down", "two values", "steps", "zeros of both signs"])
@pytest.mark.parametrize("width,n_out", [(1, 7), (4, 8), (16, 64)])
def test_select_ties_and_orders(kind, width, n_out):
    # equal candidates go to the lower beam, then to the lower token; sorted logits put the largest side by side
    n = 9000
    z = {"equal": np.zeros(n), "up": np.arange(n) / 1000, "down": -np.arange(n) / 1000, "two values": np.arange(n) % 2,
         "steps": np.arange(n) // 100 % 7, "zeros of both signs": np.where(np.arange(n) % 3, 0.0, -0.0)}[kind].astype(np.float32)
    _check_select(np.broadcast_to(z, (2, width, n)), np.zeros((2, width)), n_out)


def test_select_dead_beams_and_masks():
    rng = np.random.default_rng(8)
    z = rng.standard_normal((3, 6, 6000)).astype(np.float32)
    scores = -rng.random((3, 6))
    scores[0, 1:] = -np.inf                          # the first step: one beam
    scores[1, 0], scores[1, 3] = np.nan, np.inf
    z[1, 1, 77] = np.nan
    z[1, 2, 5999] = np.inf
    z[1, 4] = -np.inf
    z[2, :, 1000:] = -np.inf                         # masked tokens
    z[2, 3, :] = -np.inf
    z[2, 3, [5, 5000]] = 1.0, 2.0
    z[2, 4] = -3.4e38                                # the type's lowest value is a logit like any other
    z[2, 5] = 3.4e38
    _check_select(z, scores, 12)
    # fewer candidates than asked for, and none
    z[:] = -np.inf
    z[0, 0, [3, 4100]] = -7.0
    _check_select(z, scores, 5)


def test_select_dead_beams_rows_are_not_read_into_the_result():
    z = np.full((1, 3, 500), np.nan, np.float32)
    z[0, 2] = np.arange(500)
    _check_select(z, [[-np.inf, -np.inf, -4.0]], 4)


def test_select_close_candidates():
    # candidates of two beams that 32 bits of a sum near -500 do not tell apart
    z = np.zeros((1, 2, 100), np.float32)
    z[0, :, 7] = 9.0
    z[0, 1, 8] = 9.0 - 1e-6
    z[0, 0, 8] = 9.0 - 2e-6
    scores = np.array([[-500.0, -500.0 - 1e-7]])
    _check_select(z, scores, 4)


def test_select_captured():
    def work(hip):
        rng = np.random.default_rng(9)
        z, s = Dev(np.zeros((2, 4, 5000), np.float32)), Dev(np.zeros((2, 4)))
        out = [Dev(np.zeros((2, 8), t)) for t in (np.uint32, np.int32, np.float64)]

        def call():
            check(lib().atlas_beam_select_f32(z.ptr, 5000, 5000, s.ptr, 2, 4, 8, *(x.ptr for x in out)))
        with Stream(hip) as st:
            call()
            exe, _ = st.capture(call)
            for turn in range(3):
                logits, scores = rng.standard_normal(z.a.shape).astype(np.float32), rng.random((2, 4))
                for d, x in ((z, logits), (s, scores)):
                    check(lib().atlas_memcpy_h2d(d.ptr, x.ctypes.data_as(C.c_void_p), x.nbytes))
                st.launch(exe)
                st.sync()
                want = many_ref.select(logits, scores, 8)
                assert (out[0].get() == want[0]).all() and (out[1].get() == want[1]).all()
                call()
                st.sync()
    on_thread(work)


# ---- reordering --------------------------------------------------------------------


@pytest.mark.parametrize("row,stride", [(1, 1), (3, 5), (16, 16), (37, 64), (1332, 2048), (4096, 4096), (5000, 5004)])
@pytest.mark.parametrize("groups,width", [(1, 1), (1, 2), (3, 5), (2, 8), (1, 13), (2, 33), (1, 64)])
@pytest.mark.parametrize("in_place", [False, True])
def test_reorder(row, stride, groups, width, in_place):
    rng = np.random.default_rng(row + width)
    n = groups * width
    src = rng.integers(0, 256, (3, n, stride)).astype(np.uint8)
    old = rng.integers(0, 256, (3, n, stride)).astype(np.uint8)
    parents = rng.integers(-1, width + 1, (groups, width)).astype(np.int32)      # -1 and width are none
    want = src.copy() if in_place else old.copy()
    for g in range(groups):
        for b in range(width):
            if 0 <= parents[g, b] < width:
                want[:, g * width + b, :row] = src[:, g * width + parents[g, b], :row]
    a = [Dev(x) for x in src]
    to = a if in_place else [Dev(x) for x in old]
    p = Dev(parents)
    check(lib().atlas_beam_reorder((C.c_void_p * 3)(*(x.ptr for x in to)), (C.c_void_p * 3)(*(x.ptr for x in a)), 3, row, stride,
                                   p.ptr, groups, width))
    got = np.stack([x.get() for x in to])
    assert (got == want).all()


@pytest.mark.parametrize("off", [0, 1, 4, 8])
def test_reorder_part_of_a_row_and_many_states(off):
    rng = np.random.default_rng(3)
    states = [rng.integers(0, 256, (6, 400)).astype(np.uint8) for _ in range(70)]
    parents = np.array([5, 5, 0, 3, 3, 1], np.int32)
    d, p = [Dev(x) for x in states], Dev(parents)
    ptrs = (C.c_void_p * 70)(*(x.ptr + off for x in d))
    check(lib().atlas_beam_reorder(ptrs, ptrs, 70, 101, 400, p.ptr, 1, 6))
    for x, y in zip(states, d):
        want = x.copy()
        want[:, off:off + 101] = x[parents, off:off + 101]
        assert (y.get() == want).all()


def test_reorder_states_whose_rows_lie_between_each_other():
    rng = np.random.default_rng(4)
    x = rng.integers(0, 256, (6, 400)).astype(np.uint8)
    parents = np.array([5, 5, 0, 3, 3, 1], np.int32)
    d, p = Dev(x), Dev(parents)
    ptrs = (C.c_void_p * 3)(d.ptr + 296, d.ptr, d.ptr + 96)
    check(lib().atlas_beam_reorder(ptrs, ptrs, 3, 96, 400, p.ptr, 1, 6))
    want = x.copy()
    for at in (0, 96, 296):
        want[:, at:at + 96] = x[parents, at:at + 96]
    assert (d.get() == want).all()


def test_reorder_many_states_whose_rows_lie_between_each_other():
    # 150 columns of one matrix, each a state, moved in place, then into another matrix
    rng = np.random.default_rng(5)
    x = rng.integers(0, 1 << 30, (6, 150, 12)).astype(np.int32)
    parents = np.array([4, 0, 2, 2, -1, 5], np.int32)
    d, p = Dev(x), Dev(parents)
    ptrs = (C.c_void_p * 150)(*(d.ptr + 48 * i for i in range(150)))
    check(lib().atlas_beam_reorder(ptrs, ptrs, 150, 48, 7200, p.ptr, 1, 6))
    want = x.copy()
    for b in (0, 1, 3):
        want[b] = x[parents[b]]
    assert (d.get() == want).all()
    e = Dev(x)
    check(lib().atlas_beam_reorder((C.c_void_p * 150)(*(e.ptr + 48 * i for i in range(150))), ptrs, 150, 48, 7200, p.ptr, 1, 6))
    moved = x.copy()
    for b in (0, 1, 2, 3, 5):
        moved[b] = want[parents[b]]
    assert (e.get() == moved).all()


# ---- adapters ----------------------------------------------------------------------


def _bf16(x):
    """bf16 bits by truncation, and their values."""
    bits = (np.ascontiguousarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)
    return bits, (bits.astype(np.uint32) << 16).view(np.float32)


class Adapters:
    def __init__(self, seed, n, rank, m, k, rows, fmt="bf16", scales=True, pads=(0, 0, 0), shift=0):
        rng = np.random.default_rng(seed)
        a = rng.standard_normal((n, rank, k)).astype(np.float32) / np.float32(np.sqrt(k))
        b = 0.1 * rng.standard_normal((n, m, rank)).astype(np.float32)
        self.fmt, self.raw = fmt, (a, b)
        if fmt == "bf16":
            (ra, a), (rb, b) = _bf16(a), _bf16(b)
            self.raw = ra, rb
        self.a, self.b = a, b
        self.scales = rng.uniform(0.5, 2, n).astype(np.float32) if scales else None
        self.pick = rng.integers(-1, n + 1, rows).astype(np.int32)              # n is none
        self.x = rng.standard_normal((rows, k + pads[0])).astype(np.float32)
        self.base = rng.standard_normal((rows, m + pads[1])).astype(np.float32)
        self.m, self.k, self.rank, self.n, self.pads, self.shift = m, k, rank, n, pads, shift

    def check(self, in_place=False):
        m, k, s = self.m, self.k, self.shift

        def moved(x):                  # not on 16 bytes
            return Dev(np.concatenate([np.zeros(s, x.dtype), x.reshape(-1)]))
        da, db, dx, dbase = (moved(x) for x in (*self.raw, self.x, self.base))
        y = np.full((len(self.pick), m + self.pads[2]), 7, np.float32)
        dy = dbase if in_place else moved(y)
        dp, ds = Dev(self.pick), None if self.scales is None else Dev(self.scales)
        size = 2 if self.fmt == "bf16" else 4
        c = LoraC(1 if size == 2 else 0, da.ptr + size * s, db.ptr + size * s, ds.ptr if ds else None, self.n, self.rank, m, k)
        ld_y = self.base.shape[1] if in_place else y.shape[1]
        check(lib().atlas_lora_add_f32(C.byref(c), dp.ptr, dx.ptr + 4 * s, self.x.shape[1], dbase.ptr + 4 * s, self.base.shape[1],
                                       dy.ptr + 4 * s, ld_y, len(self.pick)))
        got = dy.get()[s:].reshape(-1, ld_y)
        want, off = many_ref.lora(self.base[:, :m], self.x[:, :k], self.a, self.b, self.scales, self.pick)
        _near(got[:, :m], want, off)
        none = (self.pick < 0) | (self.pick >= self.n)
        assert (got[none, :m] == self.base[none, :m]).all()
        assert (got[:, m:] == (self.base[:, m:] if in_place else 7)).all()


@pytest.mark.parametrize("fmt", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 2, 13, 16, 17, 100])
@pytest.mark.parametrize("rank,m,k", [(1, 1, 1), (8, 64, 64), (16, 300, 520), (5, 77, 131), (64, 128, 96), (20, 1000, 33), (256, 40, 64)])
def test_lora(fmt, rows, rank, m, k):
    Adapters(rank + m, 3, rank, m, k, rows, fmt).check()


@pytest.mark.parametrize("fmt", ["bf16", "f32"])
@pytest.mark.parametrize("pads,shift", [((4, 4, 8), 0), ((1, 2, 3), 0), ((0, 0, 0), 1), ((8, 8, 8), 2)])
def test_lora_strides_and_alignment(fmt, pads, shift):
    Adapters(3, 4, 16, 200, 256, 21, fmt, pads=pads, shift=shift).check()


def test_lora_sixteen_adapters_in_a_tile_and_no_scales():
    a = Adapters(4, 40, 16, 512, 2048, 48, scales=False)
    a.pick = np.arange(48).astype(np.int32) % 43
    a.check()
    a.check(in_place=True)


@pytest.mark.parametrize("m,k", [(40, 64), (70, 2100)])
@pytest.mark.parametrize("rows,n", [(63, 1), (64, 2), (65, 2), (65, 70), (300, 1), (513, 300), (4096, 3), (4099, 4095), (8200, 17)])
def test_lora_rows_of_an_adapter_in_any_order(rows, n, m, k):
    """Rows are gathered by adapter: in one wave's registers up to 64, in spans of 4096."""
    Adapters(rows, n, 3, m, k, rows, "f32").check(in_place=rows % 2 == 0)


def test_lora_one_adapter_for_all_rows_and_rows_without():
    a = Adapters(9, 3, 16, 64, 2000, 500)
    a.pick[:] = 1
    a.check()
    a.pick[:] = -5
    a.check()


def test_lora_no_adapters():
    Adapters(5, 0, 8, 64, 64, 200).check()
    Adapters(5, 0, 8, 64, 64, 5).check()


def test_lora_same_adapter_far_apart():
    a = Adapters(6, 3, 8, 200, 4096, 20)
    a.pick = np.array([2, 0, 2, 2, 1, 0, -1, 2, 0, 0, 0, 1, 2, 5, 0, 2, 2, 2, 1, 1], np.int32)
    a.check()


@pytest.mark.parametrize("rank", [16, 6])
def test_lora_infinities_and_nan_stay_with_their_rows(rank):
    a = Adapters(7, 4, rank, 100, 128, 16, "f32")
    a.pick = np.array([0, 1, 2, 3] * 4, np.int32)
    a.a[1, 2, 5] = np.nan
    a.b[2, 7, 0] = np.inf
    a.x[3, 9] = np.inf
    a.base[4, 4] = np.nan
    a.a[3, rank - 1] = 3e38            # rank's last row, which the tiles' padding repeats
    a.x[[7, 11, 15]] *= 1e-30
    want = many_ref.lora(a.base, a.x, a.a, a.b, a.scales, a.pick)[0]
    y, c = Dev(a.base), None
    d = [Dev(v) for v in (a.a, a.b, a.x, a.pick, a.scales)]
    c = LoraC(0, d[0].ptr, d[1].ptr, d[4].ptr, 4, rank, 100, 128)
    check(lib().atlas_lora_add_f32(C.byref(c), d[3].ptr, d[2].ptr, 128, y.ptr, 100, y.ptr, 100, 16))
    got = y.get()
    for r in (0, 4, 8, 12, 7, 11, 15):               # adapters 0 and 3, finite rows
        assert (np.isfinite(got[r]) == np.isfinite(want[r])).all()
    assert np.isnan(got[1]).all() and np.isnan(got[5]).all()
    assert np.isfinite(got[2]).sum() == 99 and not np.isfinite(got[2, 7])


def test_lora_rows_between_each_other():
    # x, base and y are columns of one matrix
    a = Adapters(10, 3, 16, 100, 60, 40, "f32")
    a.pick = (np.arange(40) % 5 - 1).astype(np.int32)
    d = Dev(np.concatenate([a.x, a.base, np.full((40, 104), 7, np.float32)], 1))
    w = [Dev(v) for v in (a.a, a.b, a.pick, a.scales)]
    c = LoraC(0, w[0].ptr, w[1].ptr, w[3].ptr, 3, 16, 100, 60)
    check(lib().atlas_lora_add_f32(C.byref(c), w[2].ptr, d.ptr, 264, d.ptr + 4 * 60, 264, d.ptr + 4 * 160, 264, 40))
    got = d.get()
    want, off = many_ref.lora(a.base, a.x, a.a, a.b, a.scales, a.pick)
    _near(got[:, 160:260], want, off)
    assert (got[:, 260:] == 7).all() and (got[:, :60] == a.x).all() and (got[:, 60:160] == a.base).all()


def test_scratch_refused_in_a_capture_or_short_of_memory_then_there():
    def work(hip):
        a = Adapters(11, 3, 16, 64, 2000, 9)
        d = [Dev(v) for v in (*a.raw, a.x, a.base, a.pick, a.scales)]
        y = Dev(np.zeros((9, 64), np.float32))
        c = LoraC(1, d[0].ptr, d[1].ptr, d[5].ptr, 3, 16, 64, 2000)
        z, s = Dev(np.tile(np.arange(10, dtype=np.float32), 2)), Dev(np.zeros(2))
        out = [Dev(np.zeros(2, t)) for t in (np.uint32, np.int32, np.float64)]
        b = Batch(12, [4], [3000], [30] * 4, hd=128, junk=False).upload()
        to = Dev(np.zeros((4, b.heads * b.hd), np.float32))
        calls = [lambda: check(lib().atlas_lora_add_f32(C.byref(c), d[4].ptr, d[2].ptr, 2000, d[3].ptr, 64, y.ptr, 64, 9)),
                 lambda: check(lib().atlas_beam_select_f32(z.ptr, 10, 10, s.ptr, 1, 2, 2, *(x.ptr for x in out))),
                 lambda: b.call(to)]

        def refused(call, code):
            with pytest.raises(AtlasError) as e:
                call()
            assert e.value.code == code
        with Stream(hip) as st:
            for call in calls:
                st.capture(lambda: refused(call, -4))
                check(lib().atlas_debug_fail_allocations(0, 1))
                refused(call, -3)
                check(lib().atlas_debug_fail_allocations(0, 0))
                call()
                st.sync()
            exe, _ = st.capture(lambda: [call() for call in calls])
            for _ in range(3):
                st.launch(exe)
                st.sync()
        _near(y.get(), *many_ref.lora(a.base, a.x, a.a, a.b, a.scales, a.pick))
        assert out[0].get().tolist() == [9, 9] and out[1].get().tolist() == [0, 1]
        want, off = b.want()
        _near(to.get().reshape(want.shape), want, off[..., None])
    on_thread(work)


def test_one_graph_of_all_kinds_of_calls_writes_its_results():
    """Replays over results that were cleared and inputs that were changed: adapters, selection and attention."""
    def work(hip):
        a = Adapters(21, 3, 16, 64, 2000, 9)
        d = [Dev(v) for v in (*a.raw, a.x, a.base, a.pick, a.scales)]
        c = LoraC(1, d[0].ptr, d[1].ptr, d[5].ptr, 3, 16, 64, 2000)
        b = Batch(22, [4], [3000], [30] * 4, hd=128, junk=False).upload()
        z, s = Dev(np.zeros((2, 500), np.float32)), Dev(np.zeros(2))
        shapes = ((9, 64), np.float32), (2, np.uint32), (2, np.int32), (2, np.float64), (b.q.shape, np.float32)
        y, tokens, parents, best, out = outs = [Dev(np.full(n, 77, t)) for n, t in shapes]

        def put(dev, x):
            x = np.ascontiguousarray(x)
            check(lib().atlas_memcpy_h2d(dev.ptr, x.ctypes.data_as(C.c_void_p), x.nbytes))

        def calls():
            check(lib().atlas_lora_add_f32(C.byref(c), d[4].ptr, d[2].ptr, 2000, d[3].ptr, 64, y.ptr, 64, 9))
            check(lib().atlas_beam_select_f32(z.ptr, 500, 500, s.ptr, 1, 2, 2, tokens.ptr, parents.ptr, best.ptr))
            b.call(out)
        with Stream(hip) as st:
            calls()
            exe, _ = st.capture(calls)
            for turn in range(4):
                a.x, b.q = (b.rng.standard_normal(v.shape).astype(np.float32) for v in (a.x, b.q))
                logits, scores = b.rng.standard_normal((1, 2, 500)).astype(np.float32), -b.rng.random((1, 2))
                for dev, v in ((d[2], a.x), (b.d["q"], b.q), (z, logits), (s, scores), *((o, o.a) for o in outs)):
                    put(dev, v)
                st.launch(exe)
                st.sync()
                _near(y.get(), *many_ref.lora(a.base, a.x, a.a, a.b, a.scales, a.pick))
                want = many_ref.select(logits, scores, 2)
                assert (tokens.get() == want[0][0]).all() and (parents.get() == want[1][0]).all()
                assert np.abs(best.get() - want[2][0]).max() <= 1e-12 * (1 + np.abs(want[2]).max())
                want, off = b.want()
                _near(out.get().reshape(want.shape), want, off[..., None])
                calls()
                st.sync()
    on_thread(work)


def test_lora_captured():
    def work(hip):
        a = Adapters(8, 5, 16, 256, 1024, 9)
        d = [Dev(v) for v in (*a.raw, a.x, a.base, a.pick, a.scales)]
        y = Dev(np.zeros((9, 256), np.float32))
        c = LoraC(1, d[0].ptr, d[1].ptr, d[5].ptr, 5, 16, 256, 1024)

        def call():
            check(lib().atlas_lora_add_f32(C.byref(c), d[4].ptr, d[2].ptr, 1024, d[3].ptr, 256, y.ptr, 256, 9))
        with Stream(hip) as s:
            call()
            exe, _ = s.capture(call)
            for turn in range(3):
                a.pick = a.pick[::-1].copy() if turn else a.pick
                check(lib().atlas_memcpy_h2d(d[4].ptr, a.pick.ctypes.data_as(C.c_void_p), a.pick.nbytes))
                s.launch(exe)
                s.sync()
                want, off = many_ref.lora(a.base, a.x, a.a, a.b, a.scales, a.pick)
                _near(y.get(), want, off)
                call()
                s.sync()
    on_thread(work)


# ---- the host side, and a run of them together --------------------------------------


def test_slot_cache_steps_of_a_beam_search():
    """A toy decoder of one layer whose logits are its attention's output: six steps of beams in slots, chosen by
    beam_select_gpu, once with a table of slots and once with the caches reordered, against numpy."""
    rng = np.random.default_rng(1)
    n_kv, group, hd, width, prompt, vocab, steps = 2, 2, 64, 4, 21, 300, 6
    heads, wide = n_kv * group, n_kv * hd
    emb = [rng.standard_normal((vocab, w)).astype(np.float32) for w in (heads * hd, wide, wide)]       # q, k, v of a token
    head = rng.standard_normal((vocab, heads * hd)).astype(np.float32)
    tokens = rng.integers(0, vocab, prompt)
    w = T.GpuMatrix.upload_bf16(_bf16(head)[0], vocab, heads * hd)
    head = _bf16(head)[1].astype(np.float64)

    def pos(x, t):                     # tokens at different places differ
        return (x * np.cos(0.3 * np.asarray(t))[..., None]).astype(np.float32)

    table_cache, moved_cache = (T.GpuSlotCache.new(width, 64, n_kv, hd) for _ in range(2))
    at = np.arange(prompt)
    for s in range(width):
        for cache in (table_cache, moved_cache):
            if s == 0 or cache is moved_cache:
                cache.write(s, 0, T.GpuVec.from_slice(pos(emb[1][tokens], at)), T.GpuVec.from_slice(pos(emb[2][tokens], at)))
    beams, scores = [[int(rng.integers(vocab))] for _ in range(width)], np.array([0.0] + [-np.inf] * (width - 1))
    table = np.zeros((width, steps), np.int32)
    for i in range(steps):
        t = prompt + i
        last = np.array([b[-1] for b in beams])
        for b in range(width):
            kv = [T.GpuVec.from_slice(pos(e[last[b]], t)) for e in emb[1:]]
            table_cache.write(b, t, *kv)
            moved_cache.write(b, t, *kv)
        table[:, i] = np.arange(width)
        q = T.GpuVec.from_slice(pos(emb[0][last], np.full(width, t)))
        outs = []
        for cache, slots, first, prefix in ((table_cache, table[:, :i + 1], 0, prompt), (moved_cache, np.arange(width), 0, 0)):
            batch = T.PrefixBatch([t + 1] * width, [first], [prefix], slots)
            outs.append(cache.attention(batch, q, heads, hd ** -0.5))
        a, b_ = (o.download().reshape(width, -1) for o in outs)
        # many_ref's bound with 64 elements, 27 tokens, values up to 4.5 and products' magnitudes up to 64
        assert np.abs(a - b_).max() <= 8e-4
        want = np.zeros((width, heads * hd))
        for b in range(width):
            toks = np.concatenate([tokens, np.array(beams[b])])
            kk, vv = (pos(e[toks], np.arange(t + 1)).astype(np.float64).reshape(t + 1, n_kv, hd) for e in emb[1:])
            qq = pos(emb[0][last[b]], t).astype(np.float64).reshape(heads, hd)
            for h in range(heads):
                s = kk[:, h // group] @ qq[h] * hd ** -0.5
                p = np.exp(s - s.max())
                want[b, h * hd:(h + 1) * hd] = (p / p.sum()) @ vv[:, h // group]
        assert np.abs(a - want).max() <= 4e-4
        logits = w.sgemm_rows(outs[0], width)
        toks, parents, best = T.beam_select_gpu(logits, scores, width)
        z = (logits.download().reshape(1, width, vocab))
        wt, wp, ws = many_ref.select(z, scores[None], width)
        assert (toks == wt).all() and (parents == wp).all()
        assert np.abs(z[0] - want @ head.T).max() <= 1e-3 * np.abs(z).max()
        moved_cache.reorder(parents, prompt, t + 1)
        table = table[parents[0]]
        beams = [beams[p] + [int(x)] for p, x in zip(parents[0], toks[0])]
        scores = best[0]
    assert len({tuple(b) for b in beams}) == width


def test_slot_cache_after_an_op_on_its_vectors():
    # add_inplace gives keys and values buffers of their own: attention, write and reorder use those
    rng = np.random.default_rng(3)
    k, v, dk, dv = (rng.standard_normal((3, 16, 2, 64)).astype(np.float32) for _ in range(4))
    cache = T.GpuSlotCache(T.GpuVec.from_slice(k), T.GpuVec.from_slice(v), 3, 16, 2, 64)
    cache.keys.add_inplace(T.GpuVec.from_slice(dk))
    cache.values.add_inplace(T.GpuVec.from_slice(dv))
    k, v = k + dk, v + dv
    new = rng.standard_normal((2, 2, 64)).astype(np.float32)
    cache.write(1, 9, T.GpuVec.from_slice(new[0]), T.GpuVec.from_slice(new[1]))
    k[1, 9], v[1, 9] = new
    cache.reorder([0, 1, 1], 9, 10)
    k[2, 9], v[2, 9] = k[1, 9], v[1, 9]
    q = rng.standard_normal((2, 4, 64)).astype(np.float32)
    lens, slots = [10, 10], np.array([1, 2])
    got = cache.attention(T.PrefixBatch(lens, [0], [9], slots), T.GpuVec.from_slice(q), 4, 0.125).download().reshape(q.shape)
    want, off = many_ref.attention(k, v, q, lens, [0, 2], [0], [9], slots, 0.125)
    _near(got, want, off[..., None])


def test_sgemm_rows_with_adapters():
    rng = np.random.default_rng(2)
    m, k, rows = 192, 256, 7
    a = Adapters(9, 3, 8, m, k, rows)
    w = rng.standard_normal((m, k)).astype(np.float32)
    wb, w = _bf16(w)
    mat = T.GpuMatrix.upload_bf16(wb, m, k)
    x = T.GpuVec.from_slice(a.x)
    lora = T.GpuLora(*a.raw, a.scales)
    plain = mat.sgemm_rows(x, rows).download().reshape(rows, m)
    got = mat.sgemm_rows(x, rows, lora, a.pick).download().reshape(rows, m)
    want, off = many_ref.lora(plain, a.x, a.a, a.b, a.scales, a.pick)
    _near(got, want, off)
    with pytest.raises(AtlasError):
        mat.sgemm_rows(x, rows, lora, a.pick[:3])
    with pytest.raises(AtlasError):
        T.GpuMatrix.upload_bf16(wb, m // 2, k * 2).sgemm_rows(x, rows, lora, a.pick)


def test_beam_reorder_gpu():
    rng = np.random.default_rng(4)
    x = [rng.standard_normal((2, 3, n)).astype(np.float32) for n in (5, 64, 5)]
    d = [T.GpuVec.from_slice(v) for v in x]
    p = np.array([[2, 2, 0], [1, 0, -1]])
    T.beam_reorder_gpu(d, p)
    for v, g in zip(x, d):
        want = v.copy()
        for i in range(2):
            for b in range(3):
                if p[i, b] >= 0:
                    want[i, b] = v[i, p[i, b]]
        assert (g.download().reshape(v.shape) == want).all()


def test_two_threads_on_streams_of_their_own_at_once():
    """Scratch is each thread's: both run all kinds of calls with other sizes, together."""
    failed = []

    def worker(seed, ready):
        def work(hip):
            b = Batch(seed, [8, 5], [700 + 300 * seed, 40], [20] * 13, group=4, hd=128, n_kv=2).upload()
            out = Dev(np.full((13, b.heads * b.hd), 7, np.float32))
            want, want_off = b.want()
            a = Adapters(seed, 5, 16, 256 + seed, 2100, 70 * seed)
            d = [Dev(v) for v in (*a.raw, a.x, a.base, a.pick, a.scales)]
            y = Dev(np.zeros((70 * seed, 256 + seed), np.float32))
            c = LoraC(1, d[0].ptr, d[1].ptr, d[5].ptr, 5, 16, 256 + seed, 2100)
            sum_want, off = many_ref.lora(a.base, a.x, a.a, a.b, a.scales, a.pick)
            rng = np.random.default_rng(seed)
            logits, scores = rng.standard_normal((2, 4, 5000 * seed)).astype(np.float32), np.zeros((2, 4))
            with Stream(hip) as s:
                ready.wait(60)
                for _ in range(10):
                    b.call(out)
                    check(lib().atlas_lora_add_f32(C.byref(c), d[4].ptr, d[2].ptr, 2100, d[3].ptr, 256 + seed, y.ptr, 256 + seed,
                                                   70 * seed))
                    _check_select(logits, scores, 6)
                    s.sync()
                    _near(out.get().reshape(want.shape), want, want_off[..., None])
                    _near(y.get(), sum_want, off)
        try:
            on_thread(work)
        except BaseException as e:     # (of a thread)
            failed.append(e)

    ready = threading.Barrier(2)
    threads = [threading.Thread(target=worker, args=(seed, ready)) for seed in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
