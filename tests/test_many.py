"""Refusals of attention over shared prefixes, beam selection, reordering of states and low-rank adapters:
made on the host, before any device is needed."""
import ctypes as C

import numpy as np
import pytest

from atlas_amd import tensor as T
from atlas_amd._lib import AtlasError, LoraC, PrefixBatchC, SlotCacheC, check, load

X = 1 << 12                            # a pointer that no refused call follows


def _refused(rc):
    with pytest.raises(AtlasError) as e:
        check(rc)
    assert e.value.code == -1
    return str(e.value)


CACHE = dict(k=X, v=X, n_slots=4, max_seq=64, n_kv=2, head_dim=64)
BATCH = dict(group_starts=X, prefix_slots=X, prefix_lens=X, kv_lens=X, slots=X, slot_stride=8, n_groups=2, n_rows=4,
             max_prefix=0, max_own=0)


def _attention(cache=(), batch=(), q=X, ld_q=256, heads=4, window=0, out=X, ld_out=256):
    c, b = SlotCacheC(**{**CACHE, **dict(cache)}), PrefixBatchC(**{**BATCH, **dict(batch)})
    return load().atlas_prefix_attention_f32(C.byref(c), C.byref(b), q, ld_q, heads, 1.0, window, out, ld_out)


@pytest.mark.parametrize("kw", [
    dict(cache=dict(head_dim=96)), dict(cache=dict(n_kv=0)), dict(cache=dict(n_slots=-1)), dict(cache=dict(max_seq=-1)),
    dict(cache=dict(max_seq=(1 << 24) + 1)), dict(cache=dict(k=0)), dict(cache=dict(v=X + 4)), dict(batch=dict(n_rows=-1)),
    dict(batch=dict(n_groups=-1)), dict(batch=dict(slot_stride=-1)), dict(batch=dict(max_own=-1)), dict(batch=dict(max_prefix=-1)),
    dict(batch=dict(group_starts=0)), dict(batch=dict(prefix_slots=0)), dict(batch=dict(prefix_lens=0)), dict(batch=dict(kv_lens=0)),
    dict(batch=dict(slots=0)), dict(batch=dict(slots=X + 2)), dict(batch=dict(n_rows=(1 << 20) + 1)),
    dict(batch=dict(n_groups=(1 << 20) + 1)), dict(heads=3), dict(heads=0), dict(heads=34, ld_q=4096, ld_out=4096), dict(window=-1),
    dict(q=0), dict(out=0), dict(q=X + 4), dict(out=X + 8), dict(ld_q=252), dict(ld_out=255), dict(ld_q=258),
    dict(cache=dict(n_kv=4096, n_slots=1), heads=4096, ld_q=1 << 20, ld_out=1 << 20, batch=dict(n_rows=1 << 20)),
    dict(cache=dict(n_slots=1 << 10, max_seq=1 << 21)), dict(cache=dict(n_kv=1, head_dim=256), heads=16, ld_q=4096, ld_out=4096,
                                                             batch=dict(n_rows=1 << 20, n_groups=1, group_starts=0)),
], ids=str)
def test_prefix_attention_refusals(kw):
    assert "prefix_attention" in _refused(_attention(**kw))


def test_prefix_attention_null_and_nothing_to_do():
    lib = load()
    c, b = SlotCacheC(**CACHE), PrefixBatchC(**BATCH)
    _refused(lib.atlas_prefix_attention_f32(None, C.byref(b), X, 256, 4, 1.0, 0, X, 256))
    _refused(lib.atlas_prefix_attention_f32(C.byref(c), None, X, 256, 4, 1.0, 0, X, 256))
    check(_attention(batch=dict(n_rows=0), q=0, out=0))
    check(_attention(batch=dict(n_groups=0, group_starts=0)))


def _select(logits=X, ld=100, vocab=100, scores=X, groups=2, width=4, n_out=8, tokens=X, parents=X, out=1 << 20):
    return load().atlas_beam_select_f32(logits, ld, vocab, scores, groups, width, n_out, tokens, parents, out)


@pytest.mark.parametrize("kw", [
    dict(logits=0), dict(scores=0), dict(tokens=0), dict(parents=0), dict(out=0), dict(vocab=0), dict(ld=99), dict(vocab=(1 << 30) + 1, ld=1 << 31), dict(groups=-1),
    dict(width=0), dict(width=65), dict(n_out=0), dict(n_out=65), dict(groups=65536, width=1), dict(groups=20000, width=4),
    dict(out=X), dict(out=X + 56), dict(out=X - 120),
    dict(scores=X + 4), dict(out=X + 4), dict(logits=X + 2), dict(tokens=X + 1), dict(parents=X + 1)], ids=str)
def test_beam_select_refusals(kw):
    assert "beam_select" in _refused(_select(**kw))


def test_beam_select_nothing_to_do():
    check(_select(groups=0))


def _reorder(dst=(X, 2 * X), src=(X, 2 * X), n=2, row=64, stride=128, parents=X, groups=1, width=4):
    d, s = ((C.c_void_p * 2)(*x) if x is not None else None for x in (dst, src))
    return load().atlas_beam_reorder(d, s, n, row, stride, parents, groups, width)


@pytest.mark.parametrize("kw", [
    dict(dst=None), dict(src=None), dict(dst=(X, 0)), dict(src=(0, X)), dict(n=-1), dict(row=-1), dict(row=129), dict(parents=0),
    dict(parents=X + 1), dict(groups=-1), dict(groups=65536), dict(width=0), dict(width=65),
    dict(dst=(X + 64, 2 * X)), dict(dst=(X, 2 * X - 3 * 128 - 63)), dict(stride=1 << 40),
    # a state twice, and states whose rows meet, in place or not
    dict(dst=(X, X), src=(X, X)), dict(dst=(X, X + 65), src=(X, X + 65)), dict(dst=(X, X + 3 * 128 + 63), src=(X, X + 3 * 128 + 63)),
    dict(dst=(X, 2 * X), src=(3 * X, X)), dict(dst=(X, X + 32), src=(3 * X, 3 * X))], ids=str)
def test_beam_reorder_refusals(kw):
    assert "beam_reorder" in _refused(_reorder(**kw))


def test_beam_reorder_nothing_to_do():
    for kw in (dict(n=0), dict(row=0), dict(groups=0)):
        check(_reorder(**kw))


LORA = dict(fmt=1, a=X, b=X, scales=X, n_adapters=3, rank=8, m=64, k=32)


Y = 1 << 20


def _lora(lora=(), adapters=X, x=X, ld_x=32, base=Y, ld_base=64, y=Y, ld_y=64, n=4):
    return load().atlas_lora_add_f32(C.byref(LoraC(**{**LORA, **dict(lora)})), adapters, x, ld_x, base, ld_base, y, ld_y, n)


@pytest.mark.parametrize("kw", [
    dict(lora=dict(fmt=2)), dict(lora=dict(a=0)), dict(lora=dict(b=0)), dict(lora=dict(n_adapters=-1)), dict(lora=dict(n_adapters=4096)), dict(lora=dict(rank=0)),
    dict(lora=dict(rank=257)), dict(lora=dict(m=0)), dict(lora=dict(k=0)), dict(lora=dict(m=(1 << 24) + 1), ld_base=1 << 25, ld_y=1 << 25),
    dict(lora=dict(a=X + 1)), dict(lora=dict(fmt=0, b=X + 2)), dict(lora=dict(scales=X + 2)), dict(adapters=0), dict(x=0), dict(base=0),
    dict(y=0), dict(ld_x=31), dict(ld_base=63), dict(ld_y=63), dict(n=-1), dict(n=(1 << 20) + 1), dict(x=X + 2), dict(y=X + 1),
    dict(ld_x=1 << 40), dict(x=Y + 4 * 255), dict(x=Y - 4 * 127), dict(base=Y + 4), dict(base=Y, ld_base=65), dict(x=Y + 4 * 63, ld_x=64),
    dict(x=Y + 4 * 64, ld_x=96, ld_y=95)], ids=str)
def test_lora_refusals(kw):
    assert "lora_add" in _refused(_lora(**kw))


def test_lora_null_and_nothing_to_do():
    _refused(load().atlas_lora_add_f32(None, X, X, 32, X, 64, X, 64, 4))
    check(_lora(n=0))


@pytest.mark.parametrize("args", [
    ([5, 5], [0], [3], [0, 1], [1]), ([5, 5], [0, 1], [3], [0, 1]), ([5, 5], [0], [3, 3], [0, 1]), ([5, 5], [0], [3], [0, 1, 2]),
    ([5, -1], [0], [3], [0, 1]), ([5, 5], [0], [-3], [0, 1]), ([5, 5], [0], [3], [[0, 1], [1]]), ([5, 5], [0], [3], [[[0]], [[1]]]),
    ([5, 1 << 31], [0], [3], [0, 1]), ([5, 5], [0, 0], [3, 3], [0, 1], [3, -1])], ids=str)
def test_prefix_batch_refusals(args):
    with pytest.raises(AtlasError) as e:
        T.PrefixBatch(*args)
    assert e.value.code == -1


def test_host_side_refusals():
    v = T.GpuVec(None, np.zeros(8, np.float32), 8)
    for call in (lambda: T.beam_select_gpu(v, [0.0, 0.0], 2), lambda: T.beam_reorder_gpu([v], [0, 1]),
                 lambda: T.beam_reorder_gpu([], []), lambda: T.GpuSlotCache.new(-1, 4, 2, 64),
                 lambda: T.GpuLora(np.zeros((2, 4, 8), np.float32), np.zeros((2, 8, 3), np.float32)),
                 lambda: T.GpuLora(np.zeros((2, 4, 8)), np.zeros((2, 8, 4))),
                 lambda: T.GpuLora(np.zeros((2, 4, 8), np.float32), np.zeros((2, 8, 4), np.float32), [1.0])):
        with pytest.raises(AtlasError) as e:
            call()
        assert e.value.code == -1


@pytest.mark.parametrize("n", ["0", "17", "x"])
def test_beams_argument(n):
    from atlas_amd import cli
    assert cli.parse_args(["--weights", "/x"]).beams == 1 and cli.parse_args(["--weights", "/x", "--beams", "16"]).beams == 16
    with pytest.raises(SystemExit):
        cli.parse_args(["--weights", "/x", "--beams", n])


@pytest.mark.parametrize("kw", [
    # each result where another group's scores are read: from the first to the last, and up to their ends
    dict(tokens=X), dict(tokens=X + 60), dict(tokens=X - 60), dict(parents=X), dict(parents=X + 60), dict(parents=X - 60)], ids=str)
def test_beam_select_results_apart_from_scores(kw):
    """Scores [2 x 4] f64 at X; results [2 x 8], 64 bytes of tokens and of parents."""
    assert "overlap" in _refused(_select(**{**dict(logits=1 << 21, tokens=2 * X, parents=3 * X), **kw}))


def _reorder_many(dst, src, n=None, row=64, stride=128, groups=1, width=4):
    d, s = ((C.c_void_p * len(x))(*x) for x in (dst, src))
    return load().atlas_beam_reorder(d, s, len(dst) if n is None else n, row, stride, X, groups, width)


@pytest.mark.parametrize("first,second", [(3, 70), (0, 199), (63, 64), (130, 131)])
@pytest.mark.parametrize("off", [0, 65, 3 * 128 + 63, -63])
def test_beam_reorder_states_that_meet_among_many(first, second, off):
    """States of one call are apart, however many they are: rows of 64 bytes, 128 apart, 4 to a state."""
    at = [(1 << 20) + 4096 * i for i in range(200)]
    at[second] = at[first] + off
    assert "overlap" in _refused(_reorder_many(at, at))
    # what one state reads is not what another writes
    src = [(1 << 30) + 4096 * i for i in range(200)]
    src[first] = at[second]
    assert "overlap" in _refused(_reorder_many(at, src))


def test_beam_reorder_states_that_meet_between_others():
    # 150 states whose rows lie between each other's, one of them a byte into the next one's
    at = [(1 << 20) + 64 * i for i in range(150)]
    at[97] += 1
    assert "overlap" in _refused(_reorder_many(at, at, row=64, stride=64 * 150))
    # the row before that of the first state, as far on as the stride is
    at = [(1 << 20) + 64 * i for i in range(149)] + [(1 << 20) + 64 * 150 * 3 - 63]
    assert "overlap" in _refused(_reorder_many(at, at, row=64, stride=64 * 150))


@pytest.mark.parametrize("off", [0, 60, 128, 3 * 128 + 60, -12])
@pytest.mark.parametrize("state", [0, 70])
def test_beam_reorder_parents_in_a_state(off, state):
    """Blocks read the parents while others write: they are in no row that is written (4 of them, 16 bytes)."""
    at = [(1 << 20) + 4096 * i for i in range(80)]
    d = (C.c_void_p * 80)(*at)
    assert "parents" in _refused(load().atlas_beam_reorder(d, d, 80, 64, 128, at[state] + off, 1, 4))


# K and V of 4 x 64 tokens of 2 heads of 64 (128 KB each), a batch of 4 rows in 2 groups, a table of 8 slots for each, rows of
# 4 heads of 64 (1 KB)
K, V, Q, OUT, TABLE = (i << 24 for i in range(1, 6))
FAR = dict(cache=dict(k=K, v=V), q=Q, out=OUT,
           batch=dict(group_starts=TABLE, prefix_slots=TABLE + 64, prefix_lens=TABLE + 128, kv_lens=TABLE + 192, slots=TABLE + 256))


@pytest.mark.parametrize("kw", [
    # a part of q's rows, from before and behind, and q with rows further apart or closer than its own
    dict(out=Q + 16), dict(out=Q - 16), dict(out=Q + 4 * 1024 - 16), dict(out=Q - 4 * 1024 + 16), dict(out=Q, ld_out=260),
    dict(out=Q, ld_q=260), dict(out=Q + 1024, ld_q=512, ld_out=260), dict(out=Q + 1008, ld_q=512, ld_out=512),
    dict(out=Q - 2048 + 16, ld_q=512, ld_out=512), dict(out=Q + 3 * 2048 - 16, ld_q=512, ld_out=256),
    # K, V and what describes the batch
    dict(out=K), dict(out=K - 4096 + 16), dict(out=K + (1 << 17) - 16), dict(out=V), dict(out=V + (1 << 17) - 16), dict(out=V - 16),
    dict(out=TABLE - 4096 + 16), dict(out=TABLE + 64 + 16 - 1024), dict(out=TABLE + 256 + 112), dict(out=TABLE + 192, ld_out=1024),
    dict(out=TABLE + 112, batch=dict(group_starts=0, n_groups=1))],
    ids=str)
def test_prefix_attention_out_apart_from_what_is_read(kw):
    args = {**FAR, **kw}
    args["batch"] = {**FAR["batch"], **kw.get("batch", {})}
    assert "overlaps" in _refused(_attention(**args))


class _Mem:
    """An allocation that nothing follows."""

    def __init__(self, ptr):
        self.ptr = ptr

    free = staticmethod(lambda: None)


def _vec(n, ptr=X):
    return T.GpuVec(T.GpuBuf(_Mem(ptr), n), np.zeros(0, np.float32), n)


@pytest.mark.parametrize("keys,values", [(4, 4), (8191, 8192), (8192, 8191), (0, 8192)])
def test_slot_cache_of_vectors_that_are_too_short(keys, values):
    with pytest.raises(AtlasError) as e:
        T.GpuSlotCache(_vec(keys), _vec(values), 2, 32, 2, 64)
    assert e.value.code == -1
    T.GpuSlotCache(_vec(8192), _vec(8193), 2, 32, 2, 64)


def test_slot_cache_of_vectors_that_are_not_there():
    off = T.GpuVec(None, np.zeros(8192, np.float32), 8192)
    for args in ((off, _vec(8192), 2, 32, 2, 64), (_vec(8192), off, 2, 32, 2, 64), (_vec(8192), _vec(8192), -2, -32, 2, 64)):
        with pytest.raises(AtlasError) as e:
            T.GpuSlotCache(*args)
        assert e.value.code == -1


def test_slot_cache_follows_its_vectors(monkeypatch):
    # an op that swaps a vector's buffer (add_inplace) leaves the cache with the new one, a shorter one is refused
    cache, at = T.GpuSlotCache(_vec(8192, X), _vec(8192, 2 * X), 2, 32, 2, 64), []
    batch = T.PrefixBatch.__new__(T.PrefixBatch)
    batch.n_rows, batch.n_groups, batch.c = 1, 1, PrefixBatchC()

    class Lib:
        @staticmethod
        def atlas_prefix_attention_f32(c, *_):
            at.append((c._obj.k, c._obj.v))
            return 0

        @staticmethod
        def atlas_memcpy_d2d(to, *_):
            at.append(to)
            return 0
    monkeypatch.setattr(T, "load", lambda: Lib)
    monkeypatch.setattr(T.GpuBuf, "alloc", staticmethod(lambda n: _vec(n).buf))
    cache.attention(batch, _vec(256), 4, 1.0)
    cache.keys.buf, cache.values = _vec(8192, 3 * X).buf, _vec(8192, 4 * X)
    cache.attention(batch, _vec(256), 4, 1.0)
    cache.write(0, 0, _vec(128), _vec(128))
    assert at == [(X, 2 * X), (3 * X, 4 * X), 3 * X, 4 * X] and (cache.c.k, cache.c.v) == (3 * X, 4 * X)
    cache.values = _vec(8191)
    for call in (lambda: cache.attention(batch, _vec(256), 4, 1.0), lambda: cache.write(0, 0, _vec(128), _vec(128)),
                 lambda: cache.reorder([0, 1])):
        with pytest.raises(AtlasError) as e:
            call()
        assert e.value.code == -1


def _lora_of(n, rank, rows, cols):
    lora = T.GpuLora.__new__(T.GpuLora)
    lora.n, lora.rank, lora.rows, lora.cols, lora.c = n, rank, rows, cols, LoraC()
    return lora


@pytest.mark.parametrize("n,kw", [
    (1, dict(lora=True)), (3, dict(lora=True)), (1, dict(adapters=[0])), (3, dict(adapters=[0, 1, -1])), (1, dict(lora=True, adapters=[])),
    (3, dict(lora=True, adapters=[0, 1])), (1, dict(lora=True, adapters=[1 << 31])), (1, dict(lora=True, adapters=[-(1 << 31) - 1]))], ids=str)
def test_sgemm_rows_adapters_that_do_not_belong(monkeypatch, n, kw):
    """Adapters without their matrices, or the other way round, are refused before the shared product runs."""
    mat, ran = T.GpuMatrix(T.GpuBufKind.BF16, object(), 8, 16), []
    monkeypatch.setattr(T.GpuMatrix, "_sgemm_rows", lambda *a: ran.append(a))
    monkeypatch.setattr(T.GpuLora, "add", lambda *a: ran.append(a))
    with pytest.raises(AtlasError) as e:
        mat.sgemm_rows(_vec(16 * n), n, **{**kw, **(dict(lora=_lora_of(2, 4, 8, 16)) if "lora" in kw else {})})
    assert e.value.code == -1 and not ran
    mat.sgemm_rows(_vec(16 * n), n)
    mat.sgemm_rows(_vec(16 * n), n, _lora_of(2, 4, 8, 16), [0] * n)
    assert len(ran) == 3


@pytest.mark.parametrize("with_lora", [False, True])
def test_sgemm_rows_of_a_vector_that_is_too_short(monkeypatch, with_lora):
    """Nothing runs that would read past the rows there are."""
    mat, ran = T.GpuMatrix(T.GpuBufKind.BF16, _vec(128).buf, 8, 16), []
    monkeypatch.setattr(T.GpuBuf, "alloc", staticmethod(lambda n: ran.append(n) or _vec(n).buf))
    monkeypatch.setattr(T, "load", lambda: ran.append("load"))
    with pytest.raises(AtlasError) as e:
        mat.sgemm_rows(_vec(47), 3, *((_lora_of(2, 4, 8, 16), [0, 1, 0]) if with_lora else ()))
    assert e.value.code == -1 and not ran


def test_beam_reorder_of_states_that_come_once(monkeypatch):
    """States may be any iterable, also one that can be gone through once."""
    done = []
    monkeypatch.setattr(T, "_reorder", lambda ptrs, row, stride, p: done.append((ptrs, row)))
    T.beam_reorder_gpu((_vec(n, X * n) for n in (6, 12, 6)), [1, 0])
    assert done == [([6 * X, 6 * X], 12), ([12 * X], 24)]


@pytest.mark.parametrize("kw", [
    # y: 4 rows of 256 bytes.  16 bytes of adapters, 12 of scales, A 3 x 8 x 32 and B 3 x 64 x 8 bf16
    dict(adapters=Y), dict(adapters=Y + 1020), dict(adapters=Y - 12), dict(lora=dict(scales=Y + 1020)), dict(lora=dict(scales=Y - 8)),
    dict(lora=dict(a=Y + 1022)), dict(lora=dict(a=Y - 1534)), dict(lora=dict(b=Y + 512)), dict(lora=dict(b=Y - 3070)),
    dict(lora=dict(fmt=0, b=Y - 6140)), dict(adapters=Y + 1524, ld_y=128, ld_base=128)], ids=str)
def test_lora_result_apart_from_adapters(kw):
    assert "overlaps" in _refused(_lora(**{**dict(x=1 << 22, base=1 << 23, adapters=1 << 24), **kw}))


@pytest.mark.parametrize("beams", ["1", "3"])
def test_infer_without_tokens(monkeypatch, tmp_path, beams):
    """--max-tokens 0 prints the prompt's logits, with beams too: a search of no tokens is nothing to ask the model for."""
    from atlas_amd import cli

    class Model:
        weight_bytes = reset = close = prefill = staticmethod(lambda *_: 0)
        forward_one = staticmethod(lambda t: np.arange(50, dtype=np.float32))
        generate = staticmethod(lambda prompt, n, temperature: [])

        @staticmethod
        def generate_beam(prompt, n, width):
            raise AtlasError(-1, "generate_beam: 0 new tokens")
    monkeypatch.setattr(cli.loader, "load_model_from_dir", lambda *a, **kw: Model())
    args = cli.parse_args(["--weights", str(tmp_path), "--model", "olmo3-1b", "--max-tokens", "0", "--beams", beams])
    assert cli.run_infer(args, out=lambda x: None)["tokens"] == []


@pytest.mark.parametrize("kw", [dict(parents=2 * X), dict(parents=2 * X + 60), dict(out=2 * X - 120), dict(out=3 * X + 56)], ids=str)
def test_beam_select_results_apart_from_each_other(kw):
    assert "each other" in _refused(_select(**{**dict(logits=1 << 21, scores=X, tokens=2 * X, parents=3 * X), **kw}))
