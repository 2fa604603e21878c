"""MXFP4 matrices on the device: encoding and decoding bit for bit, products against 64 bits."""
import ctypes as C

import numpy as np
import pytest

from atlas_amd._lib import check
from tests import mx_ref
from tests.gpu_util import Dev, lib, sync
from tests.stream_util import Stream, on_thread
from tests.test_mxfp4 import special

pytestmark = pytest.mark.gpu


def _bf16(x):
    """x as bf16 bits (truncated) and the values they stand for."""
    bits = (np.ascontiguousarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)
    return bits, (bits.astype(np.uint32) << 16).view(np.float32)


def _encode_dev(x, src, ld=None, shift=0):
    """data, scales of x by the device, from rows ld apart that start `shift` elements into a buffer."""
    rows, cols = x.shape
    ld = ld or cols
    kb = -(-cols // 32)
    bits, vals = _bf16(x) if src == "bf16" else (x, x)
    buf = np.full(shift + rows * ld + 8, 7, bits.dtype)
    for r in range(rows):
        buf[shift + r * ld:shift + r * ld + cols] = bits[r]
    s = Dev(buf)
    d, sc = Dev(np.full(rows * kb * 16 + 16, 0xA5, np.uint8)), Dev(np.full(rows * kb + 16, 0xA5, np.uint8))
    check(lib().atlas_quantize_mxfp4_dev(s.ptr + shift * bits.itemsize, int(src == "bf16"), rows, cols, ld, d.ptr, sc.ptr))
    sync()
    d, sc = d.get(), sc.get()
    assert (d[rows * kb * 16:] == 0xA5).all() and (sc[rows * kb:] == 0xA5).all()
    return d[:rows * kb * 16], sc[:rows * kb], vals


@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols,ld,shift", [(1, 1, 1, 0), (1, 32, 32, 0), (3, 31, 31, 0), (5, 33, 40, 3), (7, 96, 96, 1),
                                                (4, 576, 576, 0), (2, 1000, 1001, 1), (129, 65, 65, 0), (17, 2080, 4096, 0),
                                                (300, 32, 32, 0)])
def test_encode(src, rows, cols, ld, shift):
    rng = np.random.default_rng(rows * 1000 + cols)
    x = (rng.standard_normal((rows, cols)) * np.exp(2 * rng.standard_normal((rows, 1)))).astype(np.float32)
    d, sc, vals = _encode_dev(x, src, ld, shift)
    data, scales = mx_ref.matrix(vals)
    np.testing.assert_array_equal(d, data.reshape(-1))
    np.testing.assert_array_equal(sc, scales.reshape(-1))


def test_encode_special():
    x = special()
    d, sc, vals = _encode_dev(x, "f32")
    data, scales = mx_ref.matrix(vals)
    np.testing.assert_array_equal(sc, scales.reshape(-1))
    np.testing.assert_array_equal(d, data.reshape(-1))


@pytest.mark.parametrize("rows,cols,ld,shift", [(1, 1, 1, 0), (2, 32, 32, 0), (3, 31, 35, 1), (9, 1000, 1000, 0), (5, 64, 64, 1)])
def test_decode(rows, cols, ld, shift):
    """Every code under every scale byte, the smallest and NaN among them; the gaps between rows stay as they were."""
    kb = -(-cols // 32)
    rng = np.random.default_rng(cols)
    data = rng.integers(0, 256, (rows, kb * 16), dtype=np.uint8)
    scales = rng.integers(0, 253, (rows, kb), dtype=np.uint8)
    scales[0, 0], scales[-1, -1] = 0, 255
    out = Dev(np.full(shift + rows * ld + 8, 7, np.float32))
    d, s = Dev(data), Dev(scales)
    check(lib().atlas_dequantize_mxfp4_dev(d.ptr, s.ptr, rows, cols, out.ptr + 4 * shift, ld))
    sync()
    got = out.get()
    code = np.stack([data & 15, data >> 4], -1).reshape(rows, -1)
    want = np.full(got.shape, 7, np.float32)
    for r in range(rows):
        want[shift + r * ld:shift + r * ld + cols] = mx_ref.decode(code[r], scales[r])[:cols]
    np.testing.assert_array_equal(got, want)


def _operand(rng, rows, k, spread):
    x = (rng.standard_normal((rows, k)) * np.exp(spread * rng.standard_normal((rows, k)))).astype(np.float32)
    data, scales = mx_ref.matrix(x) if k else (np.zeros((rows, 0), np.uint8),) * 2
    return Dev(data), Dev(scales), mx_ref.rounded(x) if k else np.zeros((rows, 0))


def _gemm(m, n, k, ld=None, spread=0.7):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    ld = ld or m
    w, ws, wv = _operand(rng, m, k, spread)
    x, xs, xv = _operand(rng, n, k, spread)
    y = Dev(np.full((n, ld), 7, np.float32))
    check(lib().atlas_gemm_mxfp4_f32(w.ptr, ws.ptr, x.ptr, xs.ptr, y.ptr, m, n, k, ld))
    sync()
    got = y.get()
    assert (got[:, m:] == 7).all()
    want = xv @ wv.T
    # products of two codes and scales are exact in f32.  Each step of a sum is off by at most a whole last
    # place of the partial sum (2^-23; the matrix units round down): 128 in an instruction, k / 128
    # instructions one after the other, up to 64 partial sums joined.
    bound = (128 + k / 128 + 64) * 2.0 ** -23 * (np.abs(xv) @ np.abs(wv).T)
    assert (np.abs(got[:, :m] - want) <= bound + 1e-37).all(), float(np.max(np.abs(got[:, :m] - want) / (bound + 1e-37)))


@pytest.mark.parametrize("k", [1, 31, 32, 33, 96, 128, 160, 576, 1000, 2080, 4096])
@pytest.mark.parametrize("m,n", [(1, 1), (16, 1), (67, 3), (129, 16), (65, 17)])
def test_gemm_inner(m, n, k):
    _gemm(m, n, k)


@pytest.mark.parametrize("n", [1, 2, 8, 15, 16, 17, 31, 32, 33, 48, 64, 65, 100, 127, 128, 129, 200, 256, 257, 300, 511, 513])
@pytest.mark.parametrize("m,k", [(100, 288), (576, 576), (1031, 1024)])
def test_gemm_rows(m, n, k):
    _gemm(m, n, k)


@pytest.mark.parametrize("m,n,k,ld", [(4096, 1, 4096, 0), (11008, 5, 4096, 0), (2048, 13, 8192, 0), (4096, 1, 11008, 0),
                                      (1000, 300, 500, 1003), (33, 7, 64, 40), (2304, 700, 1152, 0), (1, 1000, 4096, 0),
                                      (40000, 2, 64, 0), (5, 3, 0, 7), (256, 256, 12288, 0)])
def test_gemm_shapes(m, n, k, ld):
    _gemm(m, n, k, ld)


@pytest.mark.parametrize("k", [32, 100, 288, 1056])
@pytest.mark.parametrize("m,n", [(20001, 16), (2050, 63), (2050, 129), (1500, 600), (4100, 1030), (22001, 501), (11000, 1030)])
def test_gemm_tiles(m, n, k):
    """Products of every size of tile, with ragged ends of each."""
    _gemm(m, n, k, ld=m + 3)


def test_gemm_scales_apart():
    """Scales that leave nothing of some blocks beside others, up to the ends of f32."""
    for spread in (4.0, 12.0):
        _gemm(64, 20, 512, spread=spread)


def test_gemm_nan_rows():
    """A NaN block reaches its row's products and no others."""
    rng = np.random.default_rng(9)
    m, n, k = 80, 37, 288
    w, ws, wv = _operand(rng, m, k, 0.5)
    x, xs, xv = _operand(rng, n, k, 0.5)
    s = xs.get().copy()
    s[5, 3] = 255
    xs = Dev(s)
    s = ws.get().copy()
    s[70, 0] = 255
    ws = Dev(s)
    y = Dev.empty((n, m))
    check(lib().atlas_gemm_mxfp4_f32(w.ptr, ws.ptr, x.ptr, xs.ptr, y.ptr, m, n, k, m))
    sync()
    want = np.zeros((n, m), bool)
    want[5], want[:, 70] = True, True
    np.testing.assert_array_equal(np.isnan(y.get()), want)


def test_matrix_products():
    """GpuMatrix: the activations are encoded, then multiplied."""
    from atlas_amd.quant import MxFp4Tensor
    from atlas_amd.tensor import AtlasError, GpuBufKind, GpuMatrix, GpuVec
    rng = np.random.default_rng(11)
    m, k = 200, 100
    w, x = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((5, k)).astype(np.float32)
    t = MxFp4Tensor.quantize(w)
    g = GpuMatrix.upload_mxfp4(t)
    assert g.kind is GpuBufKind.MXFP4 and g.is_on_gpu() and not g.is_bf16()
    wv, xv = mx_ref.rounded(w), mx_ref.rounded(x)
    bound = 256 * 2.0 ** -23 * (np.abs(xv) @ np.abs(wv).T)
    got = g.sgemm_rows(GpuVec.from_slice(x), 5).download().reshape(5, m)
    assert (np.abs(got - xv @ wv.T) <= bound).all()
    one = g.sgemm_vec(GpuVec.from_slice(x[0])).download()
    assert (np.abs(one - (xv @ wv.T)[0]) <= bound[0]).all()
    out = np.empty((m, 1), np.float32)
    assert g.sgemm(x[1][:, None], k, 1, out)
    assert (np.abs(out[:, 0] - (xv @ wv.T)[1]) <= bound[1]).all()
    with pytest.raises(AtlasError):
        g.sgemm_rows(GpuVec.from_slice(x[0]), 2)
    with pytest.raises(AtlasError):
        g.sgemm_vec(GpuVec.from_slice(x), 5)


def test_chain_on_a_stream_and_in_a_graph():
    """Encode, multiply and decode in order on a stream of the caller's, eagerly and replayed."""
    L = lib()
    m, n, k = 300, 21, 416
    kb = -(-k // 32)

    def work(hip):
        rng = np.random.default_rng(2)
        w, ws, wv = _operand(rng, m, k, 0.5)
        x, d, s = Dev.empty((n, k)), Dev.empty((n, kb * 16), np.uint8), Dev.empty((n, kb), np.uint8)
        back, y = Dev.empty((n, k)), Dev.empty((n, m))

        def step():
            check(L.atlas_quantize_mxfp4_dev(x.ptr, 0, n, k, k, d.ptr, s.ptr))
            check(L.atlas_gemm_mxfp4_f32(w.ptr, ws.ptr, d.ptr, s.ptr, y.ptr, m, n, k, m))
            check(L.atlas_dequantize_mxfp4_dev(d.ptr, s.ptr, n, k, back.ptr, k))

        with Stream(hip) as st:
            step()
            st.sync()
            exe, _ = st.capture(step)
            for seed in range(5):
                xv = np.random.default_rng(seed).standard_normal((n, k)).astype(np.float32)
                check(L.atlas_memcpy_h2d(x.ptr, xv.ctypes.data_as(C.c_void_p), xv.nbytes))
                check(L.atlas_memset_zero(y.ptr, y.a.nbytes))
                if seed == 1:
                    step()
                else:
                    st.launch(exe)
                r = mx_ref.rounded(xv)
                np.testing.assert_array_equal(back.get(), r.astype(np.float32))
                bound = 256 * 2.0 ** -23 * (np.abs(r) @ np.abs(wv).T)
                assert (np.abs(y.get() - r @ wv.T) <= bound).all()

    on_thread(work)


@pytest.mark.parametrize("m,n,kb", [(300, 1, (1 << 20) + 3), (520, 400, 1 << 20), (1024, 416, (1 << 20) - 1)])
def test_gemm_rows_of_16_megabytes(m, n, kb):
    """Operands past 4 GB, zero but for the first, a middle and the last block of some rows."""
    from atlas_amd.tensor import _DevMem
    rng = np.random.default_rng(kb + m)
    blocks = [0, kb // 2 + 1, kb - 1]
    rows, values, held = [], [], []
    for count in (m, n):
        data, scales = _DevMem(count * kb * 16, sync_alloc=True), _DevMem((count * kb + 3) // 4 * 4, sync_alloc=True)
        held += [data, scales]
        check(lib().atlas_memset_zero(data.ptr, data.nbytes))
        check(lib().atlas_memset_zero(scales.ptr, scales.nbytes))
        pick = sorted({0, count // 2, count - 1})
        x = rng.standard_normal((len(pick), 3 * 32)).astype(np.float32)
        codes, sc = mx_ref.matrix(x)
        codes, sc = codes.reshape(len(pick), 3, 16), sc.reshape(len(pick), 3)
        for r, row in enumerate(pick):
            for b, at in enumerate(blocks):
                for mem, src, width in ((data, codes[r, b], 16), (scales, sc[r, b:b + 1], 1)):
                    src = np.ascontiguousarray(src)
                    check(lib().atlas_memcpy_h2d(mem.ptr + (row * kb + at) * width, src.ctypes.data, src.nbytes))
        rows.append(pick)
        values.append(mx_ref.rounded(x))
    y = Dev(np.full((n, m), 7, np.float32))
    check(lib().atlas_gemm_mxfp4_f32(held[0].ptr, held[1].ptr, held[2].ptr, held[3].ptr, y.ptr, m, n, kb * 32, m))
    sync()
    want = np.zeros((n, m))
    want[np.ix_(rows[1], rows[0])] = values[1] @ values[0].T
    size = np.zeros((n, m))
    size[np.ix_(rows[1], rows[0])] = np.abs(values[1]) @ np.abs(values[0]).T
    # 96 products in three instructions, and at most 8 partial sums of which the others are zero
    assert (np.abs(y.get() - want) <= 110 * 2.0 ** -23 * size).all()
    for mem in held:
        mem.free()


def test_activations_that_are_too_few():
    from atlas_amd._lib import AtlasError
    from atlas_amd.quant import MxFp4Tensor
    from atlas_amd.tensor import GpuMatrix, GpuVec
    g = GpuMatrix.upload_mxfp4(MxFp4Tensor.quantize(np.ones((4, 96), np.float32)))
    with pytest.raises(AtlasError):
        g.sgemm_vec(GpuVec.from_slice(np.ones(95, np.float32)))
    with pytest.raises(AtlasError):
        g.sgemm(np.ones(95, np.float32), 96, 1, np.zeros(4, np.float32))
    assert (g.sgemm_vec(GpuVec.from_slice(np.ones(96, np.float32))).download() == 96).all()


def test_rows_without_memory():
    """sgemm_rows says so when the results, or the encoded activations, find no memory, and works again after."""
    from atlas_amd._lib import AtlasError
    from atlas_amd.quant import MxFp4Tensor
    from atlas_amd.tensor import GpuMatrix, GpuVec
    g = GpuMatrix.upload_mxfp4(MxFp4Tensor.quantize(np.ones((4, 96), np.float32)))
    x = GpuVec.from_slice(np.ones((3, 96), np.float32))
    try:
        for skip in range(3):                              # the results, the codes, the scales
            lib().atlas_debug_fail_allocations(skip, 1)
            with pytest.raises(AtlasError) as bad:
                g.sgemm_rows(x, 3)
            assert bad.value.code == -3
    finally:
        lib().atlas_debug_fail_allocations(0, 0)
    assert (g.sgemm_rows(x, 3).download() == 96).all()


@pytest.mark.parametrize("m,n", [(40, 3), (3000, 16), (2050, 63), (4100, 129), (1500, 600), (4100, 1030), (11000, 1030)])
def test_gemm_without_inner_elements(m, n):
    """k = 0: zeros, and operands that are not there, in every kernel."""
    y = Dev(np.full((n, m + 1), 7, np.float32))
    check(lib().atlas_gemm_mxfp4_f32(None, None, None, None, y.ptr, m, n, 0, m + 1))
    sync()
    got = y.get()
    assert (got[:, :m] == 0).all() and (got[:, m] == 7).all()


@pytest.mark.parametrize("shift", [1, 3, 15])
@pytest.mark.parametrize("m,n,k", [(300, 5, 1000), (2050, 129, 1056), (1500, 600, 100)])
def test_gemm_scales_on_any_byte(m, n, k, shift):
    rng = np.random.default_rng(m + shift)
    held = [_operand(rng, rows, k, 0.5) for rows in (m, n)]
    moved = []
    for _, scales, _ in held:
        s = scales.get().reshape(-1)
        moved.append(Dev(np.concatenate([np.full(shift, 255, np.uint8), s, np.full(16, 255, np.uint8)])))
    ys = [Dev.empty((n, m)) for _ in range(2)]
    for y, ptrs in zip(ys, ([h[1].ptr for h in held], [d.ptr + shift for d in moved])):
        check(lib().atlas_gemm_mxfp4_f32(held[0][0].ptr, ptrs[0], held[1][0].ptr, ptrs[1], y.ptr, m, n, k, m))
    sync()
    np.testing.assert_array_equal(ys[1].get(), ys[0].get())
