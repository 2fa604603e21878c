"""MXFP4 and the 4-bit KV cache without a device: the host encoder, and the calls that are refused."""
import ctypes as C

import numpy as np
import pytest

from tests import mx_ref


@pytest.fixture(scope="module")
def lib():
    import os

    import atlas_amd
    from atlas_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from atlas_amd import build
        build.build()
    return atlas_amd.load()


def special():
    """Blocks with ties, the format's limits, zeros of both signs, tiny and huge values, infinities and NaN."""
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, 7.99, 4, 0, 0.2499, 0.2501, 4.99, 5.01], np.float32)
    b = np.concatenate([ties, -ties])
    tiny = np.float32(2.0) ** -149
    rows = [b, b * np.float32(2.0) ** 100, b * np.float32(2.0) ** -100, np.zeros(32, np.float32), -np.zeros(32, np.float32),
            b * np.float32(2.0) ** -128, np.full(32, tiny), b * np.float32(2.0) ** -146, np.full(32, 3.4e38, np.float32)]
    for bad in (np.inf, -np.inf, np.nan):
        x = b.copy()
        x[17] = bad
        rows.append(x)
    one = np.zeros(32, np.float32)
    one[31] = 1
    rows.append(one)
    return np.stack(rows).astype(np.float32)


def test_host_encoder(lib):
    from atlas_amd.quant import MxFp4Tensor
    rng = np.random.default_rng(3)
    cases = [special()]
    for shape in [(1, 1), (3, 31), (5, 32), (7, 33), (4, 576), (2, 1000)]:
        cases.append((rng.standard_normal(shape) * np.exp(3 * rng.standard_normal(shape))).astype(np.float32))
    for x in cases:
        t = MxFp4Tensor.quantize(x)
        data, scales = mx_ref.matrix(x)
        np.testing.assert_array_equal(t.data, data.reshape(-1))
        np.testing.assert_array_equal(t.scales, scales.reshape(-1))
        # every value of the format is an f32 (2^-128 the smallest), or reads as NaN
        np.testing.assert_array_equal(t.dequantize(), mx_ref.rounded(x).astype(np.float32))
        assert t.memory_bytes() == 17 * t.scales.size


def test_encoding_is_nearest(lib):
    """Against the definition by distance: no other magnitude of the block's scale lies nearer."""
    from atlas_amd.quant import MxFp4Tensor
    x = np.random.default_rng(5).standard_normal((64, 96)).astype(np.float32)
    t = MxFp4Tensor.quantize(x)
    got = t.dequantize().astype(np.float64).reshape(-1, 32)
    scale = np.exp2(t.scales.astype(np.float64) - 127)[:, None, None]
    all_of = scale * mx_ref.VALUES[None, None, :]
    best = np.abs(all_of - x.astype(np.float64).reshape(-1, 32, 1)).min(-1)
    np.testing.assert_array_equal(np.abs(got - x.reshape(-1, 32)), best)
    # a step is at most 2 of a largest magnitude of 4 or more, and 8 becomes 6: 1/4 of it at most
    top = np.abs(x.reshape(-1, 32)).max(-1, keepdims=True)
    assert (np.abs(got - x.reshape(-1, 32)) <= top / 4).all()


def _refused(lib, rc):
    assert rc == -1
    assert lib.atlas_last_error()
    lib.atlas_clear_error()


def test_matrix_refusals(lib):
    a = 4096                      # an aligned address that no refused call looks at
    _refused(lib, lib.atlas_quantize_mxfp4_dev(a, 0, -1, 32, 32, a, a))
    _refused(lib, lib.atlas_quantize_mxfp4_dev(a, 0, 2, 32, 31, a, a))       # rows that overlap
    _refused(lib, lib.atlas_quantize_mxfp4_dev(None, 0, 2, 32, 32, a, a))
    _refused(lib, lib.atlas_quantize_mxfp4_dev(a + 2, 0, 2, 32, 32, a, a))   # f32 off its alignment
    _refused(lib, lib.atlas_quantize_mxfp4_dev(a + 1, 1, 2, 32, 32, a, a))
    _refused(lib, lib.atlas_quantize_mxfp4_dev(a, 0, 2, 32, 32, a + 2, a))
    _refused(lib, lib.atlas_quantize_mxfp4_dev(a, 0, 1 << 40, 1 << 20, 1 << 20, a, a))
    _refused(lib, lib.atlas_quantize_mxfp4_dev(a, 0, 1, 1 << 40, 1 << 40, a, a))
    _refused(lib, lib.atlas_dequantize_mxfp4_dev(a, a, 2, 32, None, 32))
    _refused(lib, lib.atlas_dequantize_mxfp4_dev(a, a, 2, 33, a, 32))
    _refused(lib, lib.atlas_dequantize_mxfp4_dev(a, a, 2, 32, a + 2, 32))
    _refused(lib, lib.atlas_quantize_mxfp4_host(None, 2, 32, a, a))
    _refused(lib, lib.atlas_gemm_mxfp4_f32(a, a, a, a, a, -1, 1, 32, 4))
    _refused(lib, lib.atlas_gemm_mxfp4_f32(a, a, a, a, a, 5, 1, 32, 4))      # rows of y that overlap
    _refused(lib, lib.atlas_gemm_mxfp4_f32(a + 8, a, a, a, a, 4, 1, 32, 4))
    _refused(lib, lib.atlas_gemm_mxfp4_f32(a, a, a + 4, a, a, 4, 1, 32, 4))
    _refused(lib, lib.atlas_gemm_mxfp4_f32(a, a, a, a, a + 2, 4, 1, 32, 4))
    _refused(lib, lib.atlas_gemm_mxfp4_f32(a, a, a, None, a, 4, 1, 32, 4))
    _refused(lib, lib.atlas_gemm_mxfp4_f32(a, a, a, a, None, 4, 1, 32, 4))
    # nothing to do is done without a device
    assert lib.atlas_quantize_mxfp4_dev(None, 0, 0, 32, 32, None, None) == 0
    assert lib.atlas_dequantize_mxfp4_dev(None, None, 3, 0, None, 0) == 0
    assert lib.atlas_gemm_mxfp4_f32(None, None, None, None, None, 0, 3, 32, 0) == 0


def test_cache_refusals(lib):
    from atlas_amd._lib import Kv4BatchC, Kv4CacheC
    a = 4096

    def cache(**kw):
        d = dict(data=a, n_pages=4, page_len=64, n_kv=2, head_dim=128)
        d.update(kw)
        return C.byref(Kv4CacheC(*[d[n] for n, _ in Kv4CacheC._fields_]))

    def batch(**kw):
        d = dict(row_starts=a, kv_lens=a, block_table=a, table_stride=2, n_seqs=2, n_rows=3, max_len=0)
        d.update(kw)
        return C.byref(Kv4BatchC(*[d[n] for n, _ in Kv4BatchC._fields_]))

    assert lib.atlas_kv4_cache_bytes(cache()) == 4 * 2 * 64 * (128 + 8)
    bad = [dict(head_dim=96), dict(head_dim=0), dict(page_len=16), dict(page_len=48), dict(page_len=1 << 23),
           dict(n_pages=-1), dict(n_kv=0), dict(n_kv=5000)]
    for kw in bad:
        _refused(lib, lib.atlas_kv4_cache_bytes(cache(**kw)))
        _refused(lib, lib.atlas_kv4_write_f32(cache(**kw), batch(), a, a, 256))
        _refused(lib, lib.atlas_kv4_read_f32(cache(**kw), batch(), a, a, 256))
        _refused(lib, lib.atlas_kv4_attention_f32(cache(**kw), batch(), a, 512, 4, 1.0, 0, a, 512))
    _refused(lib, lib.atlas_kv4_cache_bytes(None))
    wrong = [dict(n_seqs=-1), dict(n_rows=-1), dict(table_stride=-1), dict(max_len=-1), dict(kv_lens=None),
             dict(block_table=None), dict(row_starts=None), dict(kv_lens=a + 2), dict(n_rows=1 << 23)]
    for kw in wrong:
        _refused(lib, lib.atlas_kv4_write_f32(cache(), batch(**kw), a, a, 256))
        _refused(lib, lib.atlas_kv4_read_f32(cache(), batch(**kw), a, a, 256))
        _refused(lib, lib.atlas_kv4_attention_f32(cache(), batch(**kw), a, 512, 4, 1.0, 0, a, 512))
    for fn in (lib.atlas_kv4_write_f32, lib.atlas_kv4_read_f32):
        _refused(lib, fn(cache(), batch(), None, a, 256))
        _refused(lib, fn(cache(), batch(), a + 4, a, 256))
        _refused(lib, fn(cache(), batch(), a, a, 255))
        _refused(lib, fn(cache(), batch(), a, a, 258))
        _refused(lib, fn(cache(data=None), batch(), a, a, 256))
        _refused(lib, fn(cache(data=a + 8), batch(), a, a, 256))
        _refused(lib, fn(cache(), None, a, a, 256))
        assert fn(cache(), batch(n_rows=0), None, None, 0) == 0
        assert fn(cache(), batch(n_seqs=0), None, None, 0) == 0
    fn = lib.atlas_kv4_attention_f32
    _refused(lib, fn(cache(), batch(), a, 512, 3, 1.0, 0, a, 512))             # heads that do not divide
    _refused(lib, fn(cache(), batch(), a, 512 * 17, 34, 1.0, 0, a, 512 * 17))  # 17 to a KV head
    _refused(lib, fn(cache(), batch(), a, 512, 4, 1.0, -1, a, 512))
    _refused(lib, fn(cache(), batch(), a, 508, 4, 1.0, 0, a, 512))
    _refused(lib, fn(cache(), batch(), a, 512, 4, 1.0, 0, a, 510))
    _refused(lib, fn(cache(), batch(), a, 512, 4, 1.0, 0, None, 512))
    _refused(lib, fn(cache(), batch(), a + 4, 512, 4, 1.0, 0, a, 512))
    _refused(lib, fn(None, batch(), a, 512, 4, 1.0, 0, a, 512))
    assert fn(cache(), batch(n_rows=0), None, 0, 4, 1.0, 0, None, 0) == 0


def test_batches_that_are_refused(lib):
    from atlas_amd import AtlasError
    from atlas_amd.tensor import GpuKv4Cache, Kv4Batch, cuda_available
    for lens, table, rows in [([3], [[0]], [4]), ([3, -1], [[0], [1]], None), ([3, 4], [[0], [1]], [1]),
                              ([3], [[0]], [-1])]:
        with pytest.raises(AtlasError):
            Kv4Batch(lens, table, rows)
    with pytest.raises(AtlasError):
        GpuKv4Cache.new(4, 48, 2, 128)
    if not cuda_available():
        assert GpuKv4Cache.new(4, 64, 2, 128) is None


def test_sizes_past_the_limits(lib):
    """More bytes than an address has, more blocks than a launch has, lengths that an int32 does not hold."""
    from atlas_amd import AtlasError
    from atlas_amd._lib import Kv4BatchC, Kv4CacheC
    from atlas_amd.tensor import Kv4Batch
    a = 4096
    huge = Kv4CacheC(a, (1 << 31) - 1, 1 << 22, 4096, 256)
    one = Kv4BatchC(None, a, a, 1, 1, 1, 0)
    _refused(lib, lib.atlas_kv4_cache_bytes(C.byref(huge)))
    _refused(lib, lib.atlas_kv4_write_f32(C.byref(huge), C.byref(one), a, a, 4096 * 256))
    assert lib.atlas_kv4_cache_bytes(C.byref(Kv4CacheC(a, 1 << 20, 1 << 22, 1, 256))) == (272 << 42)
    _refused(lib, lib.atlas_gemm_mxfp4_f32(a, a, a, a, a, (1 << 28) + 1, 1, 32, 1 << 29))
    _refused(lib, lib.atlas_gemm_mxfp4_f32(a, a, a, a, a, 4, (1 << 20) + 1, 32, 4))
    for lens, table, rows in [([1 << 31], [[0]], [1]), ([1 << 32], [[0]], [0])]:
        with pytest.raises(AtlasError):
            Kv4Batch(lens, table, rows)


def test_matrix_of_another_size_is_refused(lib):
    """Codes and scales that are not those of rows x cols."""
    from atlas_amd import AtlasError
    from atlas_amd.quant import MxFp4Tensor
    from atlas_amd.tensor import GpuMatrix
    t = MxFp4Tensor.quantize(np.ones((3, 40), np.float32))
    for kw in (dict(rows=4), dict(cols=65), dict(data=t.data[:-1]), dict(scales=t.scales[:-1])):
        with pytest.raises(AtlasError):
            GpuMatrix.upload_mxfp4(MxFp4Tensor(**{**t.__dict__, **kw}))


def test_tables_of_another_number_of_sequences_are_refused(lib):
    """A table is a row of pages for each sequence; its entries are never dealt out anew."""
    from atlas_amd import AtlasError
    from atlas_amd.tensor import Kv4Batch
    four = np.arange(12).reshape(4, 3)
    for lens, table in [([3, 4], four), ([3, 4], four.T), ([3], four[:2]), ([3, 4], four[:1]), ([3, 4], [1, 2]), ([3], [0, 1]),
                        ([3, 4], 7), ([], four), ([3, 4], [[0, 1], [2]]), ([3, 4], four.reshape(2, 2, 3))]:
        with pytest.raises(AtlasError):
            Kv4Batch(lens, table)


def test_more_rows_than_row_starts_can_count(lib):
    """Rows whose number an int32 does not hold, or holds as another one (2^32: 0), are refused."""
    from atlas_amd import AtlasError
    from atlas_amd.tensor import Kv4Batch
    for n in (2, 3, 4, 5):
        with pytest.raises(AtlasError):
            Kv4Batch([1 << 30] * n, [[0]] * n, [1 << 30] * n)


def test_empty_matrices(lib):
    """No rows, or rows of no columns: decoded to their shape."""
    from atlas_amd.quant import MxFp4Tensor
    for shape in [(0, 64), (0, 33), (3, 0), (0, 0)]:
        t = MxFp4Tensor.quantize(np.zeros(shape, np.float32))
        assert t.dequantize().shape == shape and t.memory_bytes() == 0


class _Gone:
    """Device memory that there is none of (a stand-in for it that holds nothing, and one that fails)."""
    def __init__(self, nbytes, sync_alloc):
        raise MemoryError(f"{nbytes} bytes")


class _Held:
    def __init__(self, ptr=4096):
        self.ptr = self.scales_ptr = ptr


def test_rows_without_memory(lib, monkeypatch):
    """sgemm_rows reports a failed allocation as every caller of it expects: AtlasError with ATLAS_ENOMEM."""
    import atlas_amd.tensor as tensor
    from atlas_amd import AtlasError
    x = tensor.GpuVec(_Held(), np.ones(96, np.float32), 96)
    monkeypatch.setattr(tensor, "_DevMem", _Gone)
    for kind in (tensor.GpuBufKind.MXFP4, tensor.GpuBufKind.BF16):
        g = tensor.GpuMatrix(kind, _Held(), 4, 32)
        with pytest.raises(AtlasError) as bad:
            g.sgemm_rows(x, 3)
        assert bad.value.code == -3
    monkeypatch.setattr(tensor.GpuBuf, "alloc", staticmethod(lambda n: _Held()))
    with pytest.raises(AtlasError) as bad:                 # the encoded activations
        tensor.GpuMatrix(tensor.GpuBufKind.MXFP4, _Held(), 4, 32).sgemm_rows(x, 3)
    assert bad.value.code == -3


def test_cache_rows_without_memory(lib, monkeypatch):
    """The same of a 4-bit cache's read and attention, which allocate their results."""
    import atlas_amd.tensor as tensor
    from atlas_amd import AtlasError
    from atlas_amd._lib import Kv4BatchC, Kv4CacheC
    cache = tensor.GpuKv4Cache(_Held(), Kv4CacheC(4096, 4, 64, 2, 64))
    batch = object.__new__(tensor.Kv4Batch)
    batch.n_rows, batch.c = 1, Kv4BatchC(None, 4096, 4096, 1, 1, 1, 3)
    q = tensor.GpuVec(_Held(), np.ones(256, np.float32), 256)
    monkeypatch.setattr(tensor, "cuda_available", lambda: True)
    monkeypatch.setattr(tensor, "_DevMem", _Gone)
    for call in (lambda: cache.read(batch), lambda: cache.attention(batch, q, 4, 1.0)):
        with pytest.raises(AtlasError) as bad:
            call()
        assert bad.value.code == -3


def test_batches_at_the_documented_limits(lib):
    """One past each limit of the header is refused (what is within it would be launched)."""
    from atlas_amd._lib import Kv4BatchC, Kv4CacheC
    a, top = 4096, 1 << 20
    one = C.byref(Kv4CacheC(a, 4, 64, 1, 64))
    for n_seqs, n_rows in [(top + 1, 5), (5, top + 1)]:
        b = C.byref(Kv4BatchC(a, a, a, 1, n_seqs, n_rows, 0))
        for fn in (lib.atlas_kv4_write_f32, lib.atlas_kv4_read_f32):
            _refused(lib, fn(one, b, a, a, 64))
        _refused(lib, lib.atlas_kv4_attention_f32(one, b, a, 64, 1, 1.0, 0, a, 64))
    # n_kv, n_heads, head_dim, sequences, rows (None: no row_starts): n_kv times the tiles is 2^23 + 1 at least
    for n_kv, heads, hd, seqs, rows in [(9, 9, 64, 932068, None), (1025, 1025, 64, 8185, None), (8, 128, 256, 1, top),
                                        (128, 128, 256, 1, top), (256, 256, 128, 1, top), (4096, 4096, 64, 2047, 32)]:
        cache = C.byref(Kv4CacheC(a, 4, 64, n_kv, hd))
        b = C.byref(Kv4BatchC(a if rows else None, a, a, 1, seqs, rows or seqs, 0))
        per = 1 if rows is None else (32 if hd < 256 and rows * heads // n_kv > 128 * seqs else 16) * n_kv // heads
        assert n_kv * (seqs if rows is None else seqs + rows // per) > 1 << 23
        _refused(lib, lib.atlas_kv4_attention_f32(cache, b, a, heads * hd, heads, 1.0, 0, a, heads * hd))
