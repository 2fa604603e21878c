// mxfp4.hip -- MXFP4 matrices: encoding, decoding and their product.
#include "mxfp4.hpp"

namespace atlas {

// ---- encoding and decoding --------------------------------------------------------
//
// Both move bytes: 4 (f32) or 2 (bf16) in and 17/32 out for each element, or the
// reverse.  A thread has 8 elements, so four lanes a block: one or two 16-byte
// loads, a dword of codes, the block's largest magnitude by two DPP steps.

typedef u32x4 __attribute__((aligned(4))) u32x4_dw;    // a row of f32 starts on any dword,
typedef u32x4 __attribute__((aligned(2))) u32x4_hw;    // one of bf16 on any halfword

template <bool BF>
__device__ __forceinline__ void mx_load8(const void* src, long at, int left, float (&v)[8]) {
    if (left >= 8) {
        if constexpr (BF) {
            const u32x4 w = *reinterpret_cast<const u32x4_hw*>(static_cast<const uint16_t*>(src) + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = bf16_lo(w[i]); v[2 * i + 1] = bf16_hi(w[i]); }
        } else {
            const u32x4_dw* p = reinterpret_cast<const u32x4_dw*>(static_cast<const float*>(src) + at);
            const u32x4 a = p[0], b = p[1];
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[i] = __uint_as_float(a[i]); v[4 + i] = __uint_as_float(b[i]); }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = 0.f;
        if (i < left)
            v[i] = BF ? bf16_lo(static_cast<const uint16_t*>(src)[at + i]) : static_cast<const float*>(src)[at + i];
    }
}

// Row and first column of thread t's 8 elements, eights of them to a row: the
// block's first by one uniform 64-bit division, the threads' from there.
__device__ __forceinline__ void mx_place(uint32_t eights, long& row, uint32_t& eight) {
    const long first = blockIdx.x * 256L;
    const long r0 = first / eights;
    const uint32_t e = (uint32_t)(first - r0 * eights) + threadIdx.x;
    row = r0 + e / eights;
    eight = e % eights;
}

// FLAT: rows follow each other without gaps and are whole blocks, one long row
template <bool BF, bool FLAT>
__global__ __launch_bounds__(256) void mxfp4_quant_kernel(const void* __restrict__ src, long rows, long cols,
                                                          long ld, uint8_t* __restrict__ data,
                                                          uint8_t* __restrict__ scales) {
    long t, at;
    int left;
    bool live;
    if constexpr (FLAT) {
        t = blockIdx.x * 256L + threadIdx.x;
        at = t * 8;
        live = at < cols;                        // a quad is live or not as a whole
        left = live ? 8 : 0;
    } else {
        const uint32_t eights = (uint32_t)((cols + kMxBlock - 1) / kMxBlock * 4);
        long row;
        uint32_t eight;
        mx_place(eights, row, eight);
        live = row < rows;
        t = row * eights + eight;
        at = row * ld + eight * 8L;
        const long l = cols - eight * 8L;
        left = !live || l < 0 ? 0 : l < 8 ? (int)l : 8;
    }
    float v[8];
    mx_load8<BF>(src, at, left, v);
    float mx = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = fmaxf(mx, mx_mag(v[i]));
    const int byte = mx_byte(quad_max(mx));
    if (!live) return;
    reinterpret_cast<uint32_t*>(data)[t] = mx_encode8(v, byte);
    if ((t & 3) == 0) scales[t >> 2] = (uint8_t)byte;
}

template <bool FLAT>
__global__ __launch_bounds__(256) void mxfp4_dequant_kernel(const uint8_t* __restrict__ data,
                                                            const uint8_t* __restrict__ scales, long rows,
                                                            long cols, float* __restrict__ out, long ld) {
    long t, at;
    int left;
    if constexpr (FLAT) {
        t = blockIdx.x * 256L + threadIdx.x;
        at = t * 8;
        if (at >= cols) return;
        left = 8;
    } else {
        const uint32_t eights = (uint32_t)((cols + kMxBlock - 1) / kMxBlock * 4);
        long row;
        uint32_t eight;
        mx_place(eights, row, eight);
        if (row >= rows) return;
        t = row * eights + eight;
        at = row * ld + eight * 8L;
        const long l = cols - eight * 8L;
        if (l <= 0) return;
        left = l < 8 ? (int)l : 8;
    }
    float v[8];
    mx_decode8(reinterpret_cast<const uint32_t*>(data)[t], mx_scale(scales[t >> 2]), v);
    if (left == 8) {
        u32x4 a, b;
#pragma unroll
        for (int i = 0; i < 4; ++i) { a[i] = __float_as_uint(v[i]); b[i] = __float_as_uint(v[4 + i]); }
        u32x4_dw* p = reinterpret_cast<u32x4_dw*>(out + at);
        p[0] = a;
        p[1] = b;
    } else {
        for (int i = 0; i < left; ++i) out[at + i] = v[i];
    }
}

static int mx_grid(const char* who, long rows, long cols, long ld, bool& flat, long& threads, dim3& grid) {
    ATLAS_REQUIRE(rows >= 0 && cols >= 0 && ld >= cols, "%s: bad shape %ld x %ld, row stride %ld", who, rows, cols, ld);
    ATLAS_REQUIRE(cols <= (1L << 31) - 64, "%s: %ld columns", who, cols);
    flat = ld == cols && cols % kMxBlock == 0;
    const long eights = (cols + kMxBlock - 1) / kMxBlock * 4;
    // (a launch has fewer than 2^32 threads)
    ATLAS_REQUIRE(rows == 0 || eights == 0 || rows <= 0xFFFFF000L / eights, "%s: %ld x %ld is too large", who, rows, cols);
    threads = rows * eights;
    grid = dim3((unsigned)((threads + 255) / 256));
    return ATLAS_OK;
}

int mxfp4_quant_launch(const void* src, int src_bf16, long rows, long cols, long ld, uint8_t* data,
                       uint8_t* scales, hipStream_t st) {
    bool flat;
    long threads;
    dim3 grid;
    const int rc = mx_grid("quantize_mxfp4", rows, cols, ld, flat, threads, grid);
    if (rc) return rc;
    if (threads == 0) return ATLAS_OK;
    ATLAS_REQUIRE(src && data && scales, "quantize_mxfp4: null argument");
    ATLAS_REQUIRE(((uintptr_t)src & (src_bf16 ? 1 : 3)) == 0 && ((uintptr_t)data & 3) == 0,
                  "quantize_mxfp4: misaligned argument");
    if (flat) { cols *= rows; rows = 1; }
    if (src_bf16 && flat)
        hipLaunchKernelGGL((mxfp4_quant_kernel<true, true>), grid, dim3(256), 0, st, src, rows, cols, ld, data, scales);
    else if (src_bf16)
        hipLaunchKernelGGL((mxfp4_quant_kernel<true, false>), grid, dim3(256), 0, st, src, rows, cols, ld, data, scales);
    else if (flat)
        hipLaunchKernelGGL((mxfp4_quant_kernel<false, true>), grid, dim3(256), 0, st, src, rows, cols, ld, data, scales);
    else
        hipLaunchKernelGGL((mxfp4_quant_kernel<false, false>), grid, dim3(256), 0, st, src, rows, cols, ld, data, scales);
    ATLAS_LAUNCH_CHECK("quantize_mxfp4");
    return ATLAS_OK;
}

int mxfp4_dequant_launch(const uint8_t* data, const uint8_t* scales, long rows, long cols, float* out,
                         long ld, hipStream_t st) {
    bool flat;
    long threads;
    dim3 grid;
    const int rc = mx_grid("dequantize_mxfp4", rows, cols, ld, flat, threads, grid);
    if (rc) return rc;
    if (threads == 0) return ATLAS_OK;
    ATLAS_REQUIRE(data && scales && out, "dequantize_mxfp4: null argument");
    ATLAS_REQUIRE(((uintptr_t)out & 3) == 0 && ((uintptr_t)data & 3) == 0, "dequantize_mxfp4: misaligned argument");
    if (flat) {
        cols *= rows;
        rows = 1;
        hipLaunchKernelGGL(mxfp4_dequant_kernel<true>, grid, dim3(256), 0, st, data, scales, rows, cols, out, ld);
    } else {
        hipLaunchKernelGGL(mxfp4_dequant_kernel<false>, grid, dim3(256), 0, st, data, scales, rows, cols, out, ld);
    }
    ATLAS_LAUNCH_CHECK("dequantize_mxfp4");
    return ATLAS_OK;
}

// ---- product ------------------------------------------------------------------------
//
// Y[n, m] = sum_k X[n, k] W[m, k].  v_mfma_scale_f32_16x16x128_f8f6f4 multiplies
// blocks as they are stored: lane (g, i) = 16 g + i gives block g of the 128 (16
// bytes and their scale byte) of row i of A = X and of B = W, and has rows
// 4g .. 4g+3 of column i of the product.  Codes and scales are exact, the sums
// are f32.

typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ i32x8 mx_frag(u32x4 v) {
    return i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
}

constexpr int kFp4 = 4;               // format code of both operands

// One 16 x 16 tile to a wave, straight from global memory.
__global__ __launch_bounds__(256) void mxfp4_tile_kernel(const u32x4* __restrict__ w, const uint8_t* __restrict__ ws,
                                                         const u32x4* __restrict__ x, const uint8_t* __restrict__ xs,
                                                         float* __restrict__ y, int m, int n, int kb, long ldy) {
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int m0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 16, n0 = blockIdx.y * 16;
    if (m0 >= m) return;
    // rows past the last one repeat it; their results are not stored
    const long wr = (long)min(m0 + i, m - 1) * kb, xr = (long)min(n0 + i, n - 1) * kb;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int b0 = 0; b0 < kb; b0 += 4) {
        u32x4 a = {0u, 0u, 0u, 0u}, b = a;
        int sa = 127, sb = 127;
        if (b0 + g < kb) {
            a = x[xr + b0 + g];
            b = w[wr + b0 + g];
            sa = xs[xr + b0 + g];
            sb = ws[wr + b0 + g];
        }
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_frag(a), mx_frag(b), acc, kFp4, kFp4, 0, sa, 0, sb);
    }
    if (m0 + i >= m) return;
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (n0 + 4 * g + r < n) y[(n0 + 4 * g + r) * ldy + m0 + i] = acc[r];
}

int mxfp4_gemm_launch(const uint8_t* w, const uint8_t* ws, const uint8_t* x, const uint8_t* xs, float* y,
                      int m, int n, int k, long ldy, hipStream_t st) {
    ATLAS_REQUIRE(m >= 0 && n >= 0 && k >= 0 && ldy >= m, "gemm_mxfp4: bad shape m %d n %d k %d, row stride %ld", m, n, k, ldy);
    if (m == 0 || n == 0) return ATLAS_OK;
    ATLAS_REQUIRE(y && (k == 0 || (w && ws && x && xs)), "gemm_mxfp4: null argument");
    ATLAS_REQUIRE(((uintptr_t)w & 15) == 0 && ((uintptr_t)x & 15) == 0 && ((uintptr_t)y & 3) == 0,
                  "gemm_mxfp4: w and x start on 16 bytes, y on 4");
    const int kb = (int)(((long)k + kMxBlock - 1) / kMxBlock);
    const dim3 grid((m + 63L) / 64, (n + 15L) / 16);
    ATLAS_REQUIRE(grid.y <= 65535, "gemm_mxfp4: %d rows", n);
    hipLaunchKernelGGL(mxfp4_tile_kernel, grid, dim3(256), 0, st, reinterpret_cast<const u32x4*>(w), ws,
                       reinterpret_cast<const u32x4*>(x), xs, y, m, n, kb, ldy);
    ATLAS_LAUNCH_CHECK("gemm_mxfp4");
    return ATLAS_OK;
}

}  // namespace atlas
