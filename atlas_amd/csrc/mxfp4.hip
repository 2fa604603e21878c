// mxfp4.hip -- MXFP4 matrices: encoding, decoding and their product.
#include <algorithm>
#include <type_traits>
#include "mxfp4.hpp"

namespace atlas {

// ---- encoding and decoding --------------------------------------------------------
//
// Both move bytes: 4 (f32) or 2 (bf16) in and 17/32 out for each element, or the
// reverse.  A thread has 8 elements, so four lanes a block: one or two 16-byte
// loads, a dword of codes, the block's largest magnitude by two DPP steps.
// 11008 x 4096 from bf16 and back to f32 (318 MB): 57 us, 5.6 TB/s, a large copy's rate.

typedef u32x4 __attribute__((aligned(4))) u32x4_dw;    // a row of f32 starts on any dword,
typedef u32x4 __attribute__((aligned(2))) u32x4_hw;    // one of bf16 on any halfword,
typedef u32x4 __attribute__((aligned(1))) u32x4_b;     // and one of scale bytes on any byte
typedef uint64_t __attribute__((aligned(1))) u64_b;
typedef float f32x16 __attribute__((ext_vector_type(16)));

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

// 16 blocks (512 elements) of 16 rows: lane (g, i) has blocks 4s + g of row i for
// s = 0 .. 3, and the row's scale bytes, four to a dword.
struct MxUnit {
    u32x4 d[4], s;

    // row: its first block; blocks from kb on give zeros
    __device__ __forceinline__ void load(const u32x4* data, const uint8_t* scales, long row, int u, int kb, int g) {
        const int b0 = u * 16;
        const u32x4* p = data + row + b0 + g;
        const uint8_t* q = scales + row + b0;
        if (b0 + 16 <= kb) {
#pragma unroll
            for (int t = 0; t < 4; ++t) d[t] = p[4 * t];
            s = *reinterpret_cast<const u32x4_b*>(q);
        } else {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const bool in = b0 + 4 * t + g < kb;
                d[t] = in ? p[4 * t] : u32x4{0u, 0u, 0u, 0u};
                s[t] = (in ? (uint32_t)q[4 * t + g] : 127u) << (8 * g);
            }
        }
    }
};

// Few rows: the weights' stream.  A block has MT x 16 weight rows and NT x 16 rows
// of x, its waves every WAVES-th unit of 512 elements, straight from global memory
// into the matrix instructions' registers; their sums meet in LDS.  Bound by the
// weights' bytes: 22016 x 1 x 4096 (48 MB) in 10.4 us, 4.6 TB/s, 128000 x 1 x 2048 in 23.6,
// 5.9; small ones by a launch's latency, 4 us.  (A unit on its way while the one before
// is multiplied changes nothing: there are several waves to a SIMD.)
template <int MT, int NT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void mxfp4_rows_kernel(const u32x4* __restrict__ w, const uint8_t* __restrict__ ws,
                                                                const u32x4* __restrict__ x, const uint8_t* __restrict__ xs,
                                                                float* __restrict__ y, int m, int n, int kb, long ldy) {
    __shared__ f32x4 part[WAVES][MT * NT * 64];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
    const int m0 = blockIdx.x * (MT * 16), n0 = blockIdx.y * (NT * 16);
    // rows past the last one repeat it; their results are not stored
    long wr[MT], xr[NT];
#pragma unroll
    for (int t = 0; t < MT; ++t) wr[t] = (long)min(m0 + 16 * t + i, m - 1) * kb;
#pragma unroll
    for (int t = 0; t < NT; ++t) xr[t] = (long)min(n0 + 16 * t + i, n - 1) * kb;
    f32x4 acc[MT][NT];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int units = (kb + 15) / 16;
    for (int u = wave; u < units; u += WAVES) {
        MxUnit wu[MT], xu[NT];
#pragma unroll
        for (int t = 0; t < MT; ++t) wu[t].load(w, ws, wr[t], u, kb, g);
#pragma unroll
        for (int t = 0; t < NT; ++t) xu[t].load(x, xs, xr[t], u, kb, g);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int b = 0; b < NT; ++b)
                    acc[a][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        mx_frag(xu[b].d[s]), mx_frag(wu[a].d[s]), acc[a][b], kFp4, kFp4, 0, xu[b].s[s] >> (8 * g), 0,
                        wu[a].s[s] >> (8 * g));
    }
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) part[wave][(a * NT + b) * 64 + lane] = acc[a][b];
    __syncthreads();
    for (int e = threadIdx.x; e < MT * NT * 64; e += WAVES * 64) {
        f32x4 sum = part[0][e];
#pragma unroll
        for (int v = 1; v < WAVES; ++v) sum += part[v][e];
        const int tile = e >> 6, col = m0 + tile / NT * 16 + (e & 15), row = n0 + tile % NT * 16 + (e >> 4 & 3) * 4;
        if (col < m)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (row + r < n) y[(row + r) * ldy + col] = sum[r];
    }
}

// Many rows: tiles of BM weight rows x BN rows of x through LDS, 256 elements (a
// 128-byte line of each row) at a time, two such steps deep: one loads while the
// other is multiplied.
//  * Codes reach LDS by direct loads, 16-byte chunk c of row r into slot
//    c ^ (r >> 1 & 7), so that the fragment reads (32 rows, one chunk) hit the 64 banks
//    alike (no conflicts; with r & 7 there are 3.3 cycles to a read).  Scale
//    bytes, whose rows start on any byte, go through registers, 8 to a thread.
//  * v_mfma_scale_f32_32x32x64_f8f6f4, A = x, B = weights: lane (h, i) = 32 h + i gives
//    block h of the 64 of row i, and has rows 8q + 4h + 0..3 (q = 0 .. 3) of column i,
//    so that a store writes 128 bytes of a row of y.
//  * Past the end of a row lies the next one: codes there are numbers whatever they
//    are, and their scale bytes are set to 0, 2^-254 for a product, which is zero in
//    an f32.  Rows past the last one are multiplied and not stored.
//  * What it reaches: 8192 x 4096 x 8192 in 166 us, 3.3 PFLOP/s, 11008 x 2047 x 4096 in 69,
//    2.7, where a bare loop of these instructions makes 6.3 on such data (and the library's
//    bf16 product of that size 1.3).  Of the 69 us the products are 29, y's 90 MB to
//    memory 17, which a CU's one tile does not overlap, and a step's loads and barrier
//    the rest.  Rows of y that are not whole 128-byte lines cost much more, since these stores
//    put no line together: 9001 x 3000 x 1024 takes 100 us and writes 138 MB for 108, where
//    9024 takes 36 and writes 108.  No faster: steps of 128 elements in a ring of four (89 us: half
//    a line to a request), 256 x 128 with three steps in LDS (78), the block's meeting
//    before a step's last quarter (69; 5 % less with the small tiles, and 256 x 256 out of
//    registers).
constexpr int kMxStep = 8;            // blocks of a step

// 16 bytes per lane from global memory to lds + 16 lane (lds wave-uniform); zeros
// past the buffer's end.  All of the offset is in the register that is checked.
__device__ __forceinline__ void mx_load_lds(__amdgpu_buffer_rsrc_t src, uint32_t at, void* lds) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void*)lds, 16, at, 0, 0, 0);
}

// the wave's loads and LDS writes have landed; then the block meets
__device__ __forceinline__ void mx_meet() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// rows of `pitch` bytes as a buffer
__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_rows(const u32x4* p, int rows, uint32_t pitch) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<u32x4*>(p), 0, rows * pitch, 0x00020000);
}

// Scale bytes of step `step` of a row of kb >= kMxStep blocks, from the eight that are loaded at
// mx_bytes_at: a row's last step is its last eight bytes, those of the step before shifted out.
constexpr int mx_bytes_at(int step, int kb) { return step * kMxStep < kb - kMxStep ? step * kMxStep : kb - kMxStep; }
constexpr uint64_t mx_bytes(uint64_t v, int step, int kb) { return v >> (8 * (step * kMxStep - mx_bytes_at(step, kb))); }
// The step whose bytes are loaded during step t: after the last one there is none to come,
// and its own come again.  (With the load under a condition, as the codes' are, the kernels
// take 16 to 55 registers more and the largest spills: 8192 x 4096 x 8192 207 us, 165 so.)
constexpr int mx_ahead(int t, int steps) { return t + 1 < steps ? t + 1 : steps - 1; }

// every byte of a row in its place, whatever the row's length
constexpr bool mx_bytes_hold() {
    for (int kb = kMxStep; kb <= 4 * kMxStep; ++kb) {
        const int steps = (kb + kMxStep - 1) / kMxStep;
        for (int t = -1; t < steps; ++t) {
            const int step = mx_ahead(t, steps);
            uint64_t v = 0, want = 0;
            for (int j = 0; j < kMxStep; ++j) v |= (uint64_t)(mx_bytes_at(step, kb) + j + 1) << (8 * j);
            for (int j = 0; j < kMxStep; ++j) want |= (uint64_t)(step * kMxStep + j < kb ? step * kMxStep + j + 1 : 0) << (8 * j);
            if (mx_bytes(v, step, kb) != want) return false;
        }
    }
    return true;
}
static_assert(mx_bytes_hold(), "scale bytes of a row's steps");

template <int WM, int WN, int MT, int NT>
struct MxTile {
    static constexpr int WAVES = WM * WN, BM = WM * MT * 32, BN = WN * NT * 32, ROWS = BM + BN;
    static constexpr int LOADS = ROWS / 8 / WAVES;       // of 8 rows each, for a wave and step
    static constexpr int BYTES = 2 * ROWS * (128 + 8);
    static_assert(ROWS % (8 * WAVES) == 0 && BM % 8 == 0 && ROWS <= WAVES * 64, "loads in whole waves");
};

template <int WM, int WN, int MT, int NT>
__global__ __launch_bounds__(WM * WN * 64) void mxfp4_tile_kernel(const u32x4* __restrict__ w, const uint8_t* __restrict__ ws,
                                                                  const u32x4* __restrict__ x, const uint8_t* __restrict__ xs,
                                                                  float* __restrict__ y, int m, int n, int kb, long ldy,
                                                                  int tiles_m, int tiles_n) {
    typedef MxTile<WM, WN, MT, NT> T;
    // [2][ROWS * 8] chunks of codes, the weights' rows, then x's; [2][ROWS] eights of scale bytes
    extern __shared__ __align__(1024) uint8_t lds[];
    u32x4* const codes = reinterpret_cast<u32x4*>(lds);
    uint64_t* const bytes = reinterpret_cast<uint64_t*>(lds + 2 * T::ROWS * 128);
    // consecutive blocks run on different XCDs: each takes a run of the tiles, so
    // that its L2 serves the weights of a tile to all but the first
    const int per = (tiles_m * tiles_n + 7) / 8, tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (tile >= tiles_m * tiles_n) return;
    const int m0 = tile / tiles_n * T::BM, n0 = tile % tiles_n * T::BN;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 31, h = lane >> 5, wm = wave / WN, wn = wave % WN;
    const uint32_t pitch = (uint32_t)kb * 16;
    const auto wbuf = mx_rows(w + (long)m0 * kb, min(m - m0, T::BM), pitch), xbuf = mx_rows(x + (long)n0 * kb, min(n - n0, T::BN), pitch);
    // of a load's eight rows, for those whose number has bit 3 clear and set
    const uint32_t voff[2] = {(lane >> 3) * pitch + ((lane & 7) ^ (lane >> 4)) * 16, (lane >> 3) * pitch + ((lane & 7) ^ (lane >> 4) ^ 4) * 16};
    const auto load_codes = [&](int step, int buf) {
#pragma unroll
        for (int l = 0; l < T::LOADS; ++l) {
            const int r8 = (wave * T::LOADS + l) * 8;    // first of the load's rows
            const uint32_t off = r8 & 8 ? voff[1] : voff[0];
            if (r8 < T::BM) mx_load_lds(wbuf, off + r8 * pitch + step * 128, codes + (buf * T::ROWS + r8) * 8);
            else mx_load_lds(xbuf, off + (r8 - T::BM) * pitch + step * 128, codes + (buf * T::ROWS + r8) * 8);
        }
    };
    const int sr = min((int)threadIdx.x, T::ROWS - 1);
    const uint8_t* const sp = sr < T::BM ? ws + (long)min(m0 + sr, m - 1) * kb : xs + (long)min(n0 + sr - T::BM, n - 1) * kb;
    // (shifted out by trim, once the bytes have come)
    const auto load_bytes = [&](int step) {
        if (kb >= kMxStep) return *reinterpret_cast<const u64_b*>(sp + mx_bytes_at(step, kb));
        uint64_t v = 0;
        for (int j = 0; j < kb; ++j) v |= (uint64_t)sp[j] << (8 * j);
        return v;
    };
    const auto trim = [&](uint64_t v, int step) { return kb >= kMxStep ? mx_bytes(v, step, kb) : v; };
    f32x16 acc[MT][NT];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[a][b][e] = 0.f;

    const int steps = (kb + kMxStep - 1) / kMxStep;
    load_codes(0, 0);
    bytes[sr] = trim(load_bytes(0), 0);
    mx_meet();
    for (int t = 0; t < steps; ++t) {
        const int buf = t & 1;
        const int ahead = mx_ahead(t, steps);
        if (t + 1 < steps) load_codes(ahead, buf ^ 1);
        const uint64_t next = load_bytes(ahead);
        // h's byte of each pair in bytes 0 and 2
        u32x2 sa[MT], sb[NT];
#pragma unroll
        for (int a = 0; a < MT; ++a) sa[a] = __builtin_bit_cast(u32x2, bytes[buf * T::ROWS + (wm * MT + a) * 32 + i]) >> (8 * h);
#pragma unroll
        for (int b = 0; b < NT; ++b) sb[b] = __builtin_bit_cast(u32x2, bytes[buf * T::ROWS + T::BM + (wn * NT + b) * 32 + i]) >> (8 * h);
        // fragments one quarter of a step ahead
        u32x4 fa[2][MT], fb[2][NT];
        const auto read = [&](int s) {
            const int slot = (2 * s + h) ^ (i >> 1 & 7);
#pragma unroll
            for (int a = 0; a < MT; ++a) fa[s & 1][a] = codes[(buf * T::ROWS + (wm * MT + a) * 32 + i) * 8 + slot];
#pragma unroll
            for (int b = 0; b < NT; ++b) fb[s & 1][b] = codes[(buf * T::ROWS + T::BM + (wn * NT + b) * 32 + i) * 8 + slot];
        };
        const auto multiply = [&](auto sub) {
            constexpr int s = decltype(sub)::value, pick = 2 * (s & 1);
            if (s < 3) read(s + 1);
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
                for (int b = 0; b < NT; ++b)
                    acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                        mx_frag(fb[s & 1][b]), mx_frag(fa[s & 1][a]), acc[a][b], kFp4, kFp4, pick, sb[b][s >> 1], pick, sa[a][s >> 1]);
            __builtin_amdgcn_sched_barrier(0);
        };
        read(0);
        multiply(std::integral_constant<int, 0>{});
        multiply(std::integral_constant<int, 1>{});
        multiply(std::integral_constant<int, 2>{});
        multiply(std::integral_constant<int, 3>{});
        bytes[(buf ^ 1) * T::ROWS + sr] = trim(next, ahead);
        mx_meet();
    }
#pragma unroll
    for (int a = 0; a < MT; ++a) {
        const int col = m0 + (wm * MT + a) * 32 + i;
        if (col >= m) continue;
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            const int row = n0 + (wn * NT + b) * 32 + 4 * h;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int r = row + 8 * (e >> 2) + (e & 3);
                // (past the L2, which the operands are to have)
                if (r < n) __builtin_nontemporal_store(acc[a][b][e], &y[r * ldy + col]);
            }
        }
    }
}

int mxfp4_gemm_launch(const uint8_t* w, const uint8_t* ws, const uint8_t* x, const uint8_t* xs, float* y,
                      int m, int n, int k, long ldy, hipStream_t st) {
    ATLAS_REQUIRE(m >= 0 && n >= 0 && k >= 0 && ldy >= m, "gemm_mxfp4: bad shape m %d n %d k %d, row stride %ld", m, n, k, ldy);
    if (m == 0 || n == 0) return ATLAS_OK;
    ATLAS_REQUIRE(y && (k == 0 || (w && ws && x && xs)), "gemm_mxfp4: null argument");
    ATLAS_REQUIRE(((uintptr_t)w & 15) == 0 && ((uintptr_t)x & 15) == 0 && ((uintptr_t)y & 3) == 0,
                  "gemm_mxfp4: w and x start on 16 bytes, y on 4");
    const int kb = (int)(((long)k + kMxBlock - 1) / kMxBlock);
    // (a launch has fewer than 2^32 threads)
    ATLAS_REQUIRE(m <= 1 << 28 && n <= 1 << 20, "gemm_mxfp4: %d rows of weights, %d of x", m, n);
    const u32x4 *wv = reinterpret_cast<const u32x4*>(w), *xv = reinterpret_cast<const u32x4*>(x);
#define MX_ROWS(MT, NT, WAVES)                                                                                        \
    hipLaunchKernelGGL((mxfp4_rows_kernel<MT, NT, WAVES>), dim3((m + 16L * MT - 1) / (16 * MT), (n + 16L * NT - 1) / (16 * NT)), \
                       dim3(WAVES * 64), 0, st, wv, ws, xv, xs, y, m, n, kb, ldy)
#define MX_TILE(WM, WN, MT, NT)                                                                                       \
    do {                                                                                                              \
        typedef MxTile<WM, WN, MT, NT> T;                                                                             \
        const int tm = (m + T::BM - 1) / T::BM, tn = (n + T::BN - 1) / T::BN;                                         \
        hipLaunchKernelGGL((mxfp4_tile_kernel<WM, WN, MT, NT>), dim3((tm * tn + 7) / 8 * 8), dim3(T::WAVES * 64), T::BYTES, st, wv, \
                           ws, xv, xs, y, m, n, kb, ldy, tm, tn);                                                     \
    } while (0)
    // Times in us, m x n x k.  While the blocks are no more than the CUs, the one with
    // fewer rows: it has the shorter way through k (4096 x 32 x 4096: 5.7 with 32 x 16,
    // 6.8 with 32 x 32).  For up to 16 rows of x 16 of the weights as long as they
    // are no more than four blocks to a CU (4096 x 13 x 4096: 4.4, 5.5 with 32; 8192:
    // alike), then 32 (22016: 14.5 and 11.8).  32 x 32 gives way to the tiles, which read
    // the weights for 64 rows of x or more, at 1.5 blocks to a CU (4096 x 64 x 4096: 7.1,
    // 11.3 in tiles; 4096 x 129 x 4096: 15.5 and 11.6).
    const long cus = device_cu_count(), m16 = (m + 15L) / 16, n16 = (n + 15L) / 16, m32 = (m + 31L) / 32, n32 = (n + 31L) / 32;
    // more than a tile's buffers address, or none, where operands need not be there (a tile loads its first step whatever k is)
    const bool long_rows = kb >= 1 << 20 || kb == 0;
    if (m16 * n16 <= cus || (n16 == 1 && m16 <= 4 * cus)) MX_ROWS(1, 1, 8);
    else if (n16 == 1 || m32 * n16 <= cus) MX_ROWS(2, 1, 4);
    else if (long_rows || 2 * m32 * n32 <= 3 * cus) MX_ROWS(2, 2, 8);
    else {
        // The tile that takes least by the time of its rounds, in us for 4096 elements: a
        // CU does its 64 x 64 tiles at one per 6 us, and the first in 11; 128 x 128 at 14 and
        // 16; it has one at a time of 192 x 256, 35 us, and of 256 x 256, 43.
        // Measured in this order: 4096 x 256 x 4096 12.5 18.0 29.6 34.8; 11008 x 2047 x 4096
        // 119 77 69 78; 4096 x 4096 x 4096 100 56 64 46; 8192 x 4096 x 8192 366 203 182 166.
        // (Both sides are known at these k alone, and for rows of y that are whole lines; the
        // rule has no k, and a short k's epilogue weighs more than it says: 11008 x 2047 x 512 takes
        // 26 us, 18 of bytes.)
        const auto rounds = [&](long bm, long bn) { return ((m + bm - 1) / bm * ((n + bn - 1) / bn) + cus - 1) / cus; };
        const long t64 = std::max(6 * rounds(64, 64), 11L), t128 = std::max(14 * rounds(128, 128), 16L);
        const long t192 = 35 * rounds(192, 256), t256 = 43 * rounds(256, 256);
        if (t64 <= std::min({t128, t192, t256})) MX_TILE(2, 2, 1, 1);
        else if (t128 <= std::min(t192, t256)) MX_TILE(2, 2, 2, 2);
        else if (t192 <= t256) MX_TILE(2, 4, 3, 2);
        else MX_TILE(4, 2, 2, 4);
    }
#undef MX_ROWS
#undef MX_TILE
    ATLAS_LAUNCH_CHECK("gemm_mxfp4");
    return ATLAS_OK;
}

}  // namespace atlas
