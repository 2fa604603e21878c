"""Host mirror of the reference's `atlas-tensor` GPU surface.

Same names and argument meaning as crates/atlas-tensor/src/lib.rs:
``GpuBuf`` (178-237), ``GpuBufBf16`` (242-280), ``GpuBufKind`` (284-292),
``GpuMatrix`` (309-436), ``GpuVec`` (460-556), ``GpuRopeTables`` (662-693),
``GpuKvCache`` (701-785) and the free functions (97-142, 570-654), over the
C ABI of include/atlas_kernels.h.  Extensions: ``GpuBufKind.INT8`` /
``GpuBufKind.INT4`` and ``GpuMatrix.upload_int8`` / ``upload_int4`` for the
dequant-fused GEMVs, ``GpuBufKind.MXFP4`` / ``upload_mxfp4`` for products of
4-bit matrices, ``GpuKv4Cache``, a paged KV cache in 4 bits, and what decodes many
continuations together: ``GpuSlotCache`` with attention over shared prefixes,
``beam_select_gpu`` and ``beam_reorder_gpu``, ``GpuLora``.

Error behaviour follows the reference's Option/bool contract where it has
one (allocation -> None, ``sgemm`` -> False when no device is present), but
there is no CPU compute fallback: an op called on a vector that is not on the
GPU raises ``AtlasError`` instead of silently computing on the host.
"""
from __future__ import annotations

import ctypes as C
from enum import Enum
from typing import Optional

import numpy as np

from ._lib import (AtlasError, Kv4BatchC, Kv4CacheC, LoraC, PrefixBatchC, SlotCacheC, check, check_void,
                   load)


def _p(a: np.ndarray):
    return a.ctypes.data_as(C.c_void_p)


def cuda_available() -> bool:
    """lib.rs:129-135 -- a HIP device is reachable."""
    return load().atlas_cuda_available() != 0


def cuda_device_count() -> int:
    """lib.rs:137-142."""
    return load().atlas_cuda_device_count()


def device_sync() -> None:
    """lib.rs:97-100 -- drain the device."""
    load().atlas_sync()
    check_void()


class _DevMem:
    """Owns one device allocation (RAII like GpuBuf's Drop, lib.rs:226-237)."""

    def __init__(self, nbytes: int, sync_alloc: bool):
        self.ptr = None
        self.nbytes = nbytes
        self._sync = sync_alloc
        p = C.c_void_p()
        fn = load().atlas_dev_malloc_sync if sync_alloc else load().atlas_dev_malloc
        rc = fn(C.byref(p), nbytes)
        if rc < 0:
            # delivered here (GpuBuf.alloc turns it into None): not left
            # recorded for the next call's check
            msg = load().atlas_last_error().decode()
            load().atlas_clear_error()
            raise MemoryError(msg)
        self.ptr = p.value or 0

    def free(self):
        if self.ptr:
            lib = load()
            (lib.atlas_dev_free_sync if self._sync else lib.atlas_dev_free)(self.ptr)
            self.ptr = 0

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class GpuBuf:
    """f32 device buffer (lib.rs:178-237): alloc / upload / download."""

    def __init__(self, mem: _DevMem, length: int):
        self._mem = mem
        self.len = length

    @property
    def ptr(self) -> int:
        return self._mem.ptr

    @staticmethod
    def alloc(length: int) -> Optional["GpuBuf"]:
        try:
            return GpuBuf(_DevMem(max(length, 1) * 4, sync_alloc=False), length)
        except MemoryError:
            return None

    @staticmethod
    def upload(data) -> Optional["GpuBuf"]:
        a = np.ascontiguousarray(data, np.float32)
        b = GpuBuf.alloc(a.size)
        if b is None:
            return None
        if check(load().atlas_memcpy_h2d(b.ptr, _p(a), a.nbytes)) < 0:
            return None
        return b

    def download(self) -> np.ndarray:
        out = np.empty(self.len, np.float32)
        check(load().atlas_memcpy_d2h(_p(out), self.ptr, out.nbytes))
        return out


class GpuBufBf16:
    """bf16-bits device buffer for weights (lib.rs:242-280)."""

    def __init__(self, mem: _DevMem, length: int):
        self._mem = mem
        self.len = length

    @property
    def ptr(self) -> int:
        return self._mem.ptr

    @staticmethod
    def alloc(length: int) -> Optional["GpuBufBf16"]:
        try:
            return GpuBufBf16(_DevMem(max(length, 1) * 2, sync_alloc=True), length)
        except MemoryError:
            return None

    @staticmethod
    def upload(data) -> Optional["GpuBufBf16"]:
        a = np.ascontiguousarray(data, np.uint16)
        b = GpuBufBf16.alloc(a.size)
        if b is None:
            return None
        check(load().atlas_memcpy_h2d(b.ptr, _p(a), a.nbytes))
        return b


class _QuantBuf:
    """int8 / int4 weight buffer: packed data + f32 scales (extension)."""

    def __init__(self, data: np.ndarray, scales: np.ndarray, block: int):
        self.block = block
        self._d = _DevMem(max(data.nbytes, 1), sync_alloc=True)
        self._s = _DevMem(max(scales.nbytes, 4), sync_alloc=True)
        check(load().atlas_memcpy_h2d(self._d.ptr, _p(data), data.nbytes))
        check(load().atlas_memcpy_h2d(self._s.ptr, _p(scales), scales.nbytes))

    @property
    def ptr(self) -> int:
        return self._d.ptr

    @property
    def scales_ptr(self) -> int:
        return self._s.ptr


class GpuBufKind(Enum):
    """lib.rs:284-292 (F32, BF16) plus the INT8 / INT4 / MXFP4 extensions."""
    F32 = 0
    BF16 = 1
    INT8 = 2
    INT4 = 3
    MXFP4 = 4

    def is_bf16(self) -> bool:
        return self is GpuBufKind.BF16


class GpuMatrix:
    """Weight matrix resident in HBM (lib.rs:309-436)."""

    def __init__(self, kind: Optional[GpuBufKind], buf, rows: int, cols: int):
        self.kind = kind
        self.buf = buf
        self.rows = rows
        self.cols = cols

    @staticmethod
    def upload(data, rows: int, cols: int) -> "GpuMatrix":
        buf = GpuBuf.upload(data) if cuda_available() else None
        return GpuMatrix(GpuBufKind.F32 if buf else None, buf, rows, cols)

    @staticmethod
    def upload_bf16(data, rows: int, cols: int) -> "GpuMatrix":
        buf = GpuBufBf16.upload(data) if cuda_available() else None
        return GpuMatrix(GpuBufKind.BF16 if buf else None, buf, rows, cols)

    @staticmethod
    def upload_int8(t) -> "GpuMatrix":
        """From an ``atlas_amd.quant.Int8Tensor`` (extension)."""
        buf = _QuantBuf(np.ascontiguousarray(t.data, np.int8), np.ascontiguousarray(t.scales, np.float32), 0) \
            if cuda_available() else None
        return GpuMatrix(GpuBufKind.INT8 if buf else None, buf, t.rows, t.cols)

    @staticmethod
    def upload_int4(t) -> "GpuMatrix":
        """From an ``atlas_amd.quant.Int4Tensor`` (extension)."""
        buf = _QuantBuf(np.ascontiguousarray(t.data, np.uint8), np.ascontiguousarray(t.scales, np.float32),
                        t.block_size) if cuda_available() else None
        return GpuMatrix(GpuBufKind.INT4 if buf else None, buf, t.rows, t.cols)

    @staticmethod
    def upload_mxfp4(t) -> "GpuMatrix":
        """From an ``atlas_amd.quant.MxFp4Tensor`` (extension).  Products encode
        their activations as MXFP4 too: both operands have 4 bits."""
        blocks = t.rows * -(-t.cols // 32)
        if np.size(t.data) != 16 * blocks or np.size(t.scales) != blocks:
            raise AtlasError(-1, f"upload_mxfp4: {t.rows} x {t.cols} has {blocks} blocks of 16 bytes and a scale")
        buf = _QuantBuf(np.ascontiguousarray(t.data, np.uint8), np.ascontiguousarray(t.scales, np.uint8), 0) \
            if cuda_available() else None
        return GpuMatrix(GpuBufKind.MXFP4 if buf else None, buf, t.rows, t.cols)

    def is_on_gpu(self) -> bool:
        return self.buf is not None

    def is_bf16(self) -> bool:
        return self.kind is GpuBufKind.BF16

    def _launch(self, x_ptr: int, y_ptr: int, n: int) -> None:
        lib = load()
        m, k = self.rows, self.cols
        if self.kind is GpuBufKind.F32:
            lib.atlas_matmul_f32(self.buf.ptr, x_ptr, y_ptr, m, n, k)
            check_void()
        elif self.kind is GpuBufKind.BF16:
            lib.atlas_sgemm_bf16_f32(self.buf.ptr, x_ptr, y_ptr, m, n, k)
            check_void()
        elif self.kind is GpuBufKind.MXFP4 and n == 1:
            self._launch_mxfp4(x_ptr, y_ptr, 1)
        else:
            fmt = 2 if self.kind is GpuBufKind.INT8 else 3
            if n == 1:
                check(lib.atlas_gemv_f32(fmt, self.buf.ptr, self.buf.scales_ptr, self.buf.block,
                                         x_ptr, y_ptr, m, k))
            else:
                raise AtlasError(-4, "quantised GpuMatrix: use sgemm_rows for n > 1")

    def _launch_mxfp4(self, x_ptr: int, y_ptr: int, n: int) -> None:
        lib = load()
        blocks = n * -(-self.cols // 32)
        data, scales = _DevMem(max(16 * blocks, 16), sync_alloc=False), _DevMem(max(blocks, 4), sync_alloc=False)
        check(lib.atlas_quantize_mxfp4_dev(x_ptr, 0, n, self.cols, self.cols, data.ptr, scales.ptr))
        check(lib.atlas_gemm_mxfp4_f32(self.buf.ptr, self.buf.scales_ptr, data.ptr, scales.ptr, y_ptr,
                                       self.rows, n, self.cols, self.rows))

    def sgemm(self, rhs, k: int, n: int, out: np.ndarray) -> bool:
        """out[m x n] = self[m x k] rhs[k x n]; H2D rhs, D2H out (lib.rs:371-400)."""
        if self.buf is None:
            return False
        assert self.cols == k
        if self.kind is GpuBufKind.MXFP4 and np.size(rhs) != k * n:
            raise AtlasError(-1, f"sgemm: a right operand of {k} x {n} expected")
        b = GpuBuf.upload(np.ascontiguousarray(rhs, np.float32).reshape(-1))
        c = GpuBuf.alloc(self.rows * n)
        if b is None or c is None:
            return False
        try:
            self._launch(b.ptr, c.ptr, n)
        except MemoryError:                  # the encoded activations of an MXFP4 product
            return False
        out[...] = c.download().reshape(out.shape)
        return True

    def sgemm_vec(self, x: "GpuVec", n: int = 1) -> Optional["GpuVec"]:
        """Device-to-device GEMV; returns a new GpuVec (lib.rs:409-435)."""
        if self.buf is None or x.buf is None:
            return None
        if self.kind is GpuBufKind.MXFP4 and x.len < self.cols * n:
            raise AtlasError(-1, f"sgemm_vec: {n} x {self.cols} elements expected")
        out = GpuBuf.alloc(self.rows * n)
        if out is None:
            return None
        try:
            self._launch(x.buf.ptr, out.ptr, n)
        except MemoryError:
            return None
        return GpuVec(out, np.zeros(self.rows * n, np.float32), self.rows * n)

    def sgemm_rows(self, x: "GpuVec", n: int, lora: Optional["GpuLora"] = None, adapters=None) -> "GpuVec":
        """Ragged micro-batch: x holds n activation rows [n x cols]; returns
        [n x rows] (extension, skinny MFMA GEMM).  With ``lora`` each row r gets the product
        of its adapter ``adapters[r]`` (-1: none) on top."""
        if (lora is None) != (adapters is None):
            raise AtlasError(-1, "sgemm_rows: lora and adapters go together")
        if lora is not None and (lora.rows, lora.cols) != (self.rows, self.cols):
            raise AtlasError(-1, f"sgemm_rows: adapters of {lora.rows}x{lora.cols} beside {self.rows}x{self.cols}")
        if lora is not None and np.size(adapters) != n:
            raise AtlasError(-1, f"sgemm_rows: {np.size(adapters)} adapters for {n} rows")
        pick = None if lora is None else _ints("sgemm_rows", adapters)
        out = self._sgemm_rows(x, n)
        if lora is not None:
            lora.add(out, x, pick)
        return out

    def _sgemm_rows(self, x: "GpuVec", n: int) -> "GpuVec":
        if self.buf is None or x.buf is None:
            raise AtlasError(-1, "sgemm_rows: operands are not on the GPU")
        if x.len < n * self.cols:
            raise AtlasError(-1, f"sgemm_rows: {n} rows of {self.cols} elements expected")
        out = GpuBuf.alloc(self.rows * n)
        if out is None:
            raise AtlasError(-3, f"sgemm_rows: no device memory for {n} rows of {self.rows} results")
        if self.kind is GpuBufKind.MXFP4:
            try:
                self._launch_mxfp4(x.buf.ptr, out.ptr, n)
            except MemoryError as e:         # the encoded activations
                raise AtlasError(-3, f"sgemm_rows: {e}") from None
            return GpuVec(out, np.zeros(self.rows * n, np.float32), self.rows * n)
        fmt = {GpuBufKind.BF16: 1, GpuBufKind.INT8: 2, GpuBufKind.INT4: 3}[self.kind]
        scales = getattr(self.buf, "scales_ptr", None)
        block = getattr(self.buf, "block", 0)
        check(load().atlas_gemm_skinny_f32(fmt, self.buf.ptr, scales, block, x.buf.ptr, out.ptr,
                                           self.rows, n, self.cols))
        return GpuVec(out, np.zeros(self.rows * n, np.float32), self.rows * n)

    def __repr__(self):
        kind = "cpu" if self.kind is None else self.kind.name.lower()
        return f"GpuMatrix({self.rows}x{self.cols}, {kind})"


class GpuVec:
    """Activation vector in HBM (lib.rs:460-556); ``cpu`` mirrors the field."""

    def __init__(self, buf: Optional[GpuBuf], cpu: np.ndarray, length: int):
        self.buf = buf
        self.cpu = cpu
        self.len = length

    @staticmethod
    def zeros(length: int) -> "GpuVec":
        buf = GpuBuf.alloc(length) if cuda_available() else None
        if buf is not None:
            check(load().atlas_memset_zero(buf.ptr, max(length, 1) * 4))
        return GpuVec(buf, np.zeros(length, np.float32), length)

    @staticmethod
    def from_slice(data) -> "GpuVec":
        a = np.ascontiguousarray(data, np.float32).reshape(-1)
        buf = GpuBuf.upload(a) if cuda_available() else None
        return GpuVec(buf, a.copy(), a.size)

    def download(self) -> np.ndarray:
        if self.buf is not None:
            return self.buf.download()
        return self.cpu.copy()

    def is_on_gpu(self) -> bool:
        return self.buf is not None

    def gpu_ptr(self) -> Optional[int]:
        return self.buf.ptr if self.buf is not None else None

    def gpu_ptr_mut(self) -> Optional[int]:
        return self.gpu_ptr()

    def _need(self, *others: "GpuVec") -> None:
        if self.buf is None or any(o.buf is None for o in others):
            raise AtlasError(-1, "GpuVec op on a vector that is not on the GPU (no CPU fallback)")

    def add_inplace(self, other: "GpuVec") -> None:
        """lib.rs:506-519: self += other (device, new buffer swapped in)."""
        self._need(other)
        out = GpuBuf.alloc(self.len)
        load().atlas_vec_add_f32(self.buf.ptr, other.buf.ptr, out.ptr, self.len)
        check_void()
        self.buf = out

    def rmsnorm_inplace(self, w: "GpuVec", eps: float) -> None:
        """lib.rs:522-543: self = rmsnorm(self) * w."""
        self._need(w)
        out = GpuBuf.alloc(self.len)
        load().atlas_rmsnorm_f32(self.buf.ptr, w.buf.ptr, out.ptr, self.len, eps)
        check_void()
        self.buf = out

    def residual_rmsnorm_inplace(self, y: "GpuVec", w: "GpuVec", eps: float) -> None:
        """self += rmsnorm(y) * w in one launch (post-norm block, extension)."""
        self._need(y, w)
        check(load().atlas_residual_rmsnorm_f32(self.buf.ptr, y.buf.ptr, w.buf.ptr, self.len, 1, eps))

    def __repr__(self):
        return f"GpuVec(len={self.len}, gpu={self.is_on_gpu()})"


def gpu_argmax(x: GpuVec) -> Optional[int]:
    """lib.rs:107-126: index of the maximum (last one on ties)."""
    if x.buf is None:
        raise AtlasError(-1, "gpu_argmax: vector is not on the GPU (no CPU fallback)")
    out = GpuBuf.alloc(1)
    load().atlas_gpu_argmax(x.buf.ptr, out.ptr, x.len)
    check_void()
    return int(out.download()[0])


def rope_apply_gpu(x: GpuVec, pos: int, head_dim: int, theta_base: float) -> None:
    """lib.rs:570-587."""
    x._need()
    load().atlas_rope_apply_f32(x.buf.ptr, pos, head_dim, theta_base)
    check_void()


def silu_mul_gpu(gate: GpuVec, up: GpuVec) -> GpuVec:
    """lib.rs:590-609: silu(gate) * up into a new GpuVec."""
    gate._need(up)
    out = GpuBuf.alloc(gate.len)
    load().atlas_silu_mul_f32(gate.buf.ptr, up.buf.ptr, out.ptr, gate.len)
    check_void()
    return GpuVec(out, np.zeros(gate.len, np.float32), gate.len)


def adamw_step_gpu(param: int, m: int, v: int, grad: int, lr: float, beta1: float, beta2: float,
                   eps: float, wd: float, bc1: float, bc2: float, n: int) -> bool:
    """lib.rs:612-628 (training kernel, kept for ABI completeness)."""
    if not cuda_available():
        return False
    load().atlas_adamw_step(param, m, v, grad, lr, beta1, beta2, eps, wd, bc1, bc2, n)
    check_void()
    return True


def qk_norm_inplace_gpu(x: GpuVec, w: GpuVec, n_heads: int, head_dim: int, eps: float) -> None:
    """lib.rs:633-654."""
    x._need(w)
    load().atlas_qk_norm_inplace(x.buf.ptr, w.buf.ptr, n_heads, head_dim, eps)
    check_void()


class GpuRopeTables:
    """lib.rs:662-693: cos/sin [max_seq x half_dim] in HBM."""

    def __init__(self, cos: GpuVec, sin: GpuVec, max_seq: int, half_dim: int):
        self.cos, self.sin, self.max_seq, self.half_dim = cos, sin, max_seq, half_dim

    @staticmethod
    def upload(cos_flat, sin_flat, max_seq: int, half_dim: int) -> Optional["GpuRopeTables"]:
        if not cuda_available():
            return None
        return GpuRopeTables(GpuVec.from_slice(cos_flat), GpuVec.from_slice(sin_flat), max_seq, half_dim)

    def apply_to(self, x: GpuVec, n_heads: int, head_dim: int, pos: int) -> None:
        x._need(self.cos, self.sin)
        load().atlas_rope_precomputed(x.buf.ptr, self.cos.buf.ptr, self.sin.buf.ptr, n_heads,
                                      head_dim, pos, self.max_seq)
        check_void()


class GpuKvCache:
    """lib.rs:701-785: keys/values [max_seq x n_kv_heads x head_dim] f32."""

    def __init__(self, keys: GpuVec, values: GpuVec, max_seq: int, n_kv_heads: int, head_dim: int):
        self.keys, self.values = keys, values
        self.max_seq, self.n_kv_heads, self.head_dim = max_seq, n_kv_heads, head_dim

    @staticmethod
    def new(max_seq: int, n_kv_heads: int, head_dim: int) -> Optional["GpuKvCache"]:
        if not cuda_available():
            return None
        total = max_seq * n_kv_heads * head_dim
        return GpuKvCache(GpuVec.zeros(total), GpuVec.zeros(total), max_seq, n_kv_heads, head_dim)

    def write(self, pos: int, new_k: GpuVec, new_v: GpuVec) -> None:
        if not 0 <= pos < self.max_seq:
            raise AtlasError(-1, f"GpuKvCache.write: pos {pos} outside [0, {self.max_seq})")
        self.keys._need(self.values, new_k, new_v)
        load().atlas_kv_cache_write(self.keys.buf.ptr, self.values.buf.ptr, new_k.buf.ptr,
                                    new_v.buf.ptr, pos, self.n_kv_heads, self.head_dim)
        check_void()

    def decode_attention(self, q: GpuVec, n_heads: int, pos: int, scale: float,
                         window_size: int) -> Optional[GpuVec]:
        if q.buf is None:
            return None
        if not 0 <= pos < self.max_seq:
            raise AtlasError(-1, f"decode_attention: pos {pos} outside [0, {self.max_seq})")
        n = n_heads * self.head_dim
        out = GpuBuf.alloc(n)
        load().atlas_decode_attention(q.buf.ptr, self.keys.buf.ptr, self.values.buf.ptr, out.ptr,
                                      n_heads, self.n_kv_heads, self.head_dim, pos, scale, window_size)
        check_void()
        return GpuVec(out, np.zeros(n, np.float32), n)

    def reset(self) -> None:
        """No-op by design (lib.rs:772-784): positions beyond pos are never read."""


class Kv4Batch:
    """The sequences of one step over a ``GpuKv4Cache`` (extension): lengths with
    the new tokens included, a row of page ids for each sequence (-1: no page),
    and how many of its last tokens are the step's rows (default one)."""

    def __init__(self, kv_lens, block_table, row_lens=None):
        lens = np.asarray(kv_lens, np.int64).reshape(-1)
        rows = np.ones(lens.size, np.int64) if row_lens is None else np.asarray(row_lens, np.int64).reshape(-1)
        if rows.size != lens.size or (rows < 0).any() or (rows > lens).any() or (lens >= 1 << 31).any():
            raise AtlasError(-1, "Kv4Batch: each sequence has 0 <= new rows <= length < 2^31")
        if rows.sum() >= 1 << 31:            # (row_starts are int32)
            raise AtlasError(-1, f"Kv4Batch: {rows.sum()} rows")
        lens = lens.astype(np.int32)
        try:
            table = np.asarray(block_table, np.int64)
        except ValueError:
            raise AtlasError(-1, "Kv4Batch: the block table's rows have one length") from None
        if lens.size == 0 and table.size == 0:
            table = table.reshape(0, 0)
        if table.ndim != 2 or table.shape[0] != lens.size:
            raise AtlasError(-1, f"Kv4Batch: a block table of shape {table.shape} for {lens.size} sequences")
        table = np.where((table < 0) | (table >= 1 << 31), -1, table).astype(np.int32)
        starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.kv_lens, self.block_table, self.row_starts = lens, table, starts
        self.n_seqs, self.n_rows = lens.size, int(starts[-1])
        # (each in its own piece of one allocation)
        flat = np.concatenate([lens, starts, table.reshape(-1)])
        self._mem = _DevMem(max(flat.nbytes, 4), sync_alloc=False)
        check(load().atlas_memcpy_h2d(self._mem.ptr, _p(flat), flat.nbytes))
        p = self._mem.ptr
        self.c = Kv4BatchC(None if row_lens is None else p + 4 * lens.size, p,
                           p + 4 * (lens.size + starts.size), table.shape[1], self.n_seqs, self.n_rows,
                           int(lens.max(initial=0)))


class GpuKv4Cache:
    """One layer's K and V in MXFP4 pages (extension; ``GpuKvCache`` holds f32)."""

    def __init__(self, mem: _DevMem, c: Kv4CacheC):
        self._mem, self.c = mem, c

    @staticmethod
    def new(n_pages: int, page_len: int, n_kv_heads: int, head_dim: int) -> Optional["GpuKv4Cache"]:
        c = Kv4CacheC(None, n_pages, page_len, n_kv_heads, head_dim)
        nbytes = check(load().atlas_kv4_cache_bytes(C.byref(c)))
        if not cuda_available():
            return None
        try:
            mem = _DevMem(max(nbytes, 16), sync_alloc=True)
        except MemoryError:
            return None
        check(load().atlas_memset_zero(mem.ptr, mem.nbytes))
        c.data = mem.ptr
        return GpuKv4Cache(mem, c)

    def _need(self, batch: Kv4Batch, *rows) -> None:
        for x, wide in rows:
            if x.buf is None or x.len < batch.n_rows * wide:
                raise AtlasError(-1, f"GpuKv4Cache: {batch.n_rows} rows of {wide} elements expected on the GPU")

    @staticmethod
    def _rows(batch: Kv4Batch, wide: int) -> GpuVec:
        """The result's rows, cleared."""
        out = GpuVec.zeros(batch.n_rows * wide)
        if out.buf is None:
            raise AtlasError(-3, f"GpuKv4Cache: no device memory for {batch.n_rows} rows of {wide} elements")
        return out

    def write(self, batch: Kv4Batch, k: GpuVec, v: GpuVec) -> None:
        wide = self.c.n_kv * self.c.head_dim
        self._need(batch, (k, wide), (v, wide))
        check(load().atlas_kv4_write_f32(C.byref(self.c), C.byref(batch.c), k.buf.ptr, v.buf.ptr, wide))

    def read(self, batch: Kv4Batch):
        wide = self.c.n_kv * self.c.head_dim
        k, v = self._rows(batch, wide), self._rows(batch, wide)
        check(load().atlas_kv4_read_f32(C.byref(self.c), C.byref(batch.c), k.buf.ptr, v.buf.ptr, wide))
        return k, v

    def attention(self, batch: Kv4Batch, q: GpuVec, n_heads: int, scale: float, window_size: int = 0) -> GpuVec:
        wide = n_heads * self.c.head_dim
        self._need(batch, (q, wide))
        out = self._rows(batch, wide)
        check(load().atlas_kv4_attention_f32(C.byref(self.c), C.byref(batch.c), q.buf.ptr, wide, n_heads, scale,
                                             window_size, out.buf.ptr, wide))
        return out


def _scratch(nbytes: int) -> _DevMem:
    try:
        return _DevMem(max(nbytes, 4), sync_alloc=False)
    except MemoryError as e:
        raise AtlasError(-3, str(e)) from None


def _upload(a: np.ndarray) -> _DevMem:
    """A device copy of a host array."""
    a = np.ascontiguousarray(a)
    mem = _scratch(a.nbytes)
    check(load().atlas_memcpy_h2d(mem.ptr, _p(a), a.nbytes))
    return mem


def _ints(who: str, x, lo: int = -(1 << 31)) -> np.ndarray:
    a = np.asarray(x, np.int64)
    if (a < lo).any() or (a >= 1 << 31).any():
        raise AtlasError(-1, f"{who}: values from {lo} to 2^31 - 1 expected")
    return a.astype(np.int32)


class PrefixBatch:
    """The rows of one step over a ``GpuSlotCache`` (extension).  Groups of
    ``group_sizes`` rows (default: all rows are one) share their first ``prefix_lens[g]``
    tokens, in slot ``prefix_slots[g]``; row r has ``kv_lens[r]`` tokens, its newest
    included, of which those of its own lie in slot ``slots[r]``, or token i of
    them in slot ``slots[r][i]`` where ``slots`` is a table."""

    def __init__(self, kv_lens, prefix_slots, prefix_lens, slots, group_sizes=None):
        who = "PrefixBatch"
        lens, at, pre = (_ints(who, x, 0 if i != 1 else -(1 << 31)).reshape(-1)
                         for i, x in enumerate((kv_lens, prefix_slots, prefix_lens)))
        try:
            slots = _ints(who, slots)
        except ValueError:
            raise AtlasError(-1, f"{who}: the table's rows have one length") from None
        sizes = _ints(who, [lens.size] if group_sizes is None else group_sizes, 0).reshape(-1)
        if sizes.size != at.size or sizes.size != pre.size or int(sizes.astype(np.int64).sum()) != lens.size:
            raise AtlasError(-1, f"{who}: {sizes.size} groups of {sizes.sum()} rows, {at.size} slots and {pre.size} lengths of "
                                 f"prefixes, {lens.size} rows")
        if slots.ndim not in (1, 2) or slots.shape[0] != lens.size:
            raise AtlasError(-1, f"{who}: slots of shape {slots.shape} for {lens.size} rows")
        if slots.ndim == 2 and slots.shape[1] == 0:
            slots = np.full((lens.size, 1), -1, np.int32)
        self.n_rows, self.n_groups = lens.size, sizes.size
        starts = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
        own = lens - np.repeat(pre, sizes)
        parts = [starts, at, pre, lens, slots.reshape(-1)]
        self._mem = _upload(np.concatenate(parts))
        p = self._mem.ptr + 4 * np.concatenate([[0], np.cumsum([x.size for x in parts])])
        self.c = PrefixBatchC(int(p[0]), int(p[1]), int(p[2]), int(p[3]), int(p[4]),
                              slots.shape[1] if slots.ndim == 2 else 0, self.n_groups, self.n_rows,
                              max(int(pre.max(initial=0)), 1), max(int(own.max(initial=0)), 1))


class GpuSlotCache:
    """f32 KV caches of several sequences side by side (extension): keys and values
    [n_slots x max_seq x n_kv_heads x head_dim], ``GpuKvCache``'s layout slot after slot."""

    def __init__(self, keys: GpuVec, values: GpuVec, n_slots: int, max_seq: int, n_kv_heads: int, head_dim: int):
        self.keys, self.values = keys, values
        self.n_slots, self.max_seq, self.n_kv_heads, self.head_dim = n_slots, max_seq, n_kv_heads, head_dim
        self.c                         # (refuses what does not fit)

    @staticmethod
    def _total(n_slots: int, max_seq: int, n_kv_heads: int, head_dim: int) -> int:
        if min(n_slots, max_seq, n_kv_heads, head_dim) < 0:
            raise AtlasError(-1, f"GpuSlotCache: {n_slots} slots of {max_seq} tokens, {n_kv_heads} heads of {head_dim}")
        return n_slots * max_seq * n_kv_heads * head_dim

    @property
    def c(self) -> SlotCacheC:
        """The cache as its vectors are now: an op may have given them other buffers."""
        shape = self.n_slots, self.max_seq, self.n_kv_heads, self.head_dim
        total = self._total(*shape)
        for x in (self.keys, self.values):
            x._need()
            if min(x.len, x.buf.len) < total:
                raise AtlasError(-1, f"GpuSlotCache: {min(x.len, x.buf.len)} elements, {total} expected")
        return SlotCacheC(self.keys.buf.ptr, self.values.buf.ptr, *shape)

    @staticmethod
    def new(n_slots: int, max_seq: int, n_kv_heads: int, head_dim: int) -> Optional["GpuSlotCache"]:
        total = GpuSlotCache._total(n_slots, max_seq, n_kv_heads, head_dim)
        if not cuda_available():
            return None
        keys, values = GpuVec.zeros(total), GpuVec.zeros(total)
        if keys.buf is None or values.buf is None:
            return None
        return GpuSlotCache(keys, values, n_slots, max_seq, n_kv_heads, head_dim)

    def write(self, slot: int, pos: int, new_k: GpuVec, new_v: GpuVec) -> None:
        """K and V rows of one or more tokens from position ``pos`` on."""
        wide = self.n_kv_heads * self.head_dim
        n = new_k.len // max(wide, 1)
        if new_k.len != n * wide or new_v.len != new_k.len or not 0 <= slot < self.n_slots or not 0 <= pos <= self.max_seq - n:
            raise AtlasError(-1, f"GpuSlotCache.write: {new_k.len} and {new_v.len} elements at slot {slot}, position {pos}")
        new_k._need(new_v)
        c = self.c
        for at, new in ((c.k, new_k), (c.v, new_v)):
            check(load().atlas_memcpy_d2d(at + 4 * wide * (slot * self.max_seq + pos), new.buf.ptr, 4 * new.len))

    def attention(self, batch: PrefixBatch, q: GpuVec, n_heads: int, scale: float, window_size: int = 0) -> GpuVec:
        """Attention of the batch's query rows [n_rows x n_heads x head_dim]."""
        c, wide = self.c, n_heads * self.head_dim
        if q.buf is None or q.len < batch.n_rows * wide:
            raise AtlasError(-1, f"GpuSlotCache: {batch.n_rows} rows of {wide} elements expected on the GPU")
        out = GpuBuf.alloc(batch.n_rows * wide)
        if out is None:
            raise AtlasError(-3, f"GpuSlotCache: no device memory for {batch.n_rows} rows of {wide} elements")
        check(load().atlas_prefix_attention_f32(C.byref(c), C.byref(batch.c), q.buf.ptr, wide, n_heads, scale,
                                                window_size, out.ptr, wide))
        return GpuVec(out, np.zeros(out.len, np.float32), out.len)

    def reorder(self, parents, begin: int = 0, end: Optional[int] = None) -> None:
        """Slot g * width + b takes over positions [begin, end) of slot g * width + parents[g][b],
        for the first slots ([n_groups x width] parents, or [width] of one group)."""
        end = self.max_seq if end is None else end
        p = np.atleast_2d(_ints("GpuSlotCache.reorder", parents))
        wide = 4 * self.n_kv_heads * self.head_dim
        if p.ndim != 2 or p.size > self.n_slots or not 0 <= begin <= end <= self.max_seq:
            raise AtlasError(-1, f"GpuSlotCache.reorder: parents of shape {p.shape}, positions {begin} to {end}")
        c = self.c
        _reorder([c.k + wide * begin, c.v + wide * begin], wide * (end - begin), wide * self.max_seq, p)


def _reorder(ptrs, row_bytes: int, stride: int, parents: np.ndarray) -> None:
    mem = _upload(parents)
    states = (C.c_void_p * max(len(ptrs), 1))(*ptrs)
    check(load().atlas_beam_reorder(states, states, len(ptrs), row_bytes, stride, mem.ptr, parents.shape[0], parents.shape[1]))


def beam_reorder_gpu(states, parents) -> None:
    """Beams take over the states of the beams that they continue, in place (extension):
    row g * width + b of each ``GpuVec`` becomes row g * width + parents[g][b]
    ([n_groups x width], or [width] of one group; another number: the row stays)."""
    p = np.atleast_2d(_ints("beam_reorder_gpu", parents))
    if p.ndim != 2 or p.size == 0:
        raise AtlasError(-1, f"beam_reorder_gpu: parents of shape {p.shape}")
    states = list(states)
    for x in states:
        x._need()
        if x.len % p.size:
            raise AtlasError(-1, f"beam_reorder_gpu: {x.len} elements in {p.size} rows")
    for wide in sorted({x.len // p.size for x in states}):
        _reorder([x.buf.ptr for x in states if x.len // p.size == wide], 4 * wide, 4 * wide, p)


def beam_select_gpu(logits: GpuVec, scores, n_out: int):
    """Beam search's choice (extension): the ``n_out`` best continuations of each group, from
    logits [n_groups x width x vocab] and the beams' sums of log probabilities
    [n_groups x width] (or [width]; not finite: no such beam).  Returns tokens, parents and scores,
    each [n_groups x n_out] in descending order; parent -1: there are no more."""
    s = np.atleast_2d(np.asarray(scores, np.float64))
    if s.ndim != 2 or s.size == 0 or logits.buf is None or logits.len == 0 or logits.len % s.size:
        raise AtlasError(-1, f"beam_select_gpu: {logits.len} logits on the GPU for scores of shape {s.shape}")
    vocab = logits.len // s.size
    if not 1 <= n_out <= 64:
        raise AtlasError(-1, f"beam_select_gpu: {n_out} continuations (1 to 64)")
    n = s.shape[0] * n_out
    mem, out = _upload(s), _scratch(16 * n)      # scores, tokens, parents
    check(load().atlas_beam_select_f32(logits.buf.ptr, vocab, vocab, mem.ptr, s.shape[0], s.shape[1], n_out, out.ptr + 8 * n,
                                       out.ptr + 12 * n, out.ptr))
    got = np.empty(16 * n, np.uint8)
    check(load().atlas_memcpy_d2h(_p(got), out.ptr, got.nbytes))
    shape = (s.shape[0], n_out)
    return (got[8 * n:12 * n].view(np.uint32).reshape(shape), got[12 * n:].view(np.int32).reshape(shape),
            got[:8 * n].view(np.float64).reshape(shape))


class GpuLora:
    """Low-rank adapters of one rows x cols projection (extension): ``a`` [n x rank x cols] and
    ``b`` [n x rows x rank], f32, or uint16 bf16 bits, and a scale for each (default 1)."""

    def __init__(self, a, b, scales=None):
        a, b = np.asarray(a), np.asarray(b)
        fmt = {np.dtype(np.uint16): 1, np.dtype(np.float32): 0}.get(a.dtype)
        if fmt is None or a.dtype != b.dtype or a.ndim != 3 or b.ndim != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise AtlasError(-1, f"GpuLora: a {a.shape} {a.dtype}, b {b.shape} {b.dtype}")
        self.n, self.rank, self.cols, self.rows = a.shape[0], a.shape[1], a.shape[2], b.shape[1]
        if scales is not None and np.size(scales) != self.n:
            raise AtlasError(-1, f"GpuLora: {np.size(scales)} scales for {self.n} adapters")
        self._a, self._b = _upload(a), _upload(b)
        self._s = None if scales is None else _upload(np.asarray(scales, np.float32))
        self.c = LoraC(fmt, self._a.ptr, self._b.ptr, self._s.ptr if self._s else None, self.n, self.rank, self.rows, self.cols)

    def add(self, y: GpuVec, x: GpuVec, adapters) -> None:
        """y [n x rows] += the product of each row's adapter with x [n x cols]; -1: none."""
        pick = _ints("GpuLora.add", adapters).reshape(-1)
        y._need(x)
        if x.len < pick.size * self.cols or y.len < pick.size * self.rows:
            raise AtlasError(-1, f"GpuLora.add: {pick.size} rows of {self.cols} and {self.rows} elements expected")
        mem = _upload(pick)
        check(load().atlas_lora_add_f32(C.byref(self.c), mem.ptr, x.buf.ptr, self.cols, y.buf.ptr, self.rows, y.buf.ptr, self.rows,
                                        pick.size))
