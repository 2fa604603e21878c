// lora.hip -- low-rank adapters beside a shared projection: each row has its own.
//
// y_r = base_r + s_a B_a (A_a x_r), a the row's adapter.  Two launches, because every
// element of y needs the whole of A_a x_r:
//   1  v_r = A_a x_r: a block takes 16 rows, one of the adapters that they name and a
//      piece of k;
//   2  y = base + s B v: a block takes 16 rows and a piece of m, and of v the sum over
//      the pieces of k.
// Both are f32 matrix products of 16 x 16 x 4, exact products of bf16 or f32 weights
// and f32 activations.  A tile's columns are its 16 rows; an adapter's product is
// computed for all of them and kept by those that name it.
#include <algorithm>

#include "many.hpp"

namespace atlas {

struct LoraArgs {
    const void *a, *b;
    const float* scales;               // or null: 1
    int n_adapters, rank, m, k;
    const int* pick;
    const float* x;
    long ld_x;
    const float* base;
    long ld_base;
    float* y;
    long ld_y;
    int n;
    float* v;                          // [splits][n][vr] partial products
    int vr;                            // rank in whole tiles of 16
    int splits, k_piece;               // k's pieces, multiples of 64
};

// N elements of T of a row of n from `at` on, as f32.  Rows may start anywhere: the loads
// need no alignment beyond the elements'.
template <typename T, int N>
__device__ __forceinline__ void lora_load(const T* row, int at, float (&to)[N]) {
    if constexpr (sizeof(T) == 2) {
        uint32_t w[N / 2];
        __builtin_memcpy(w, row + at, N * 2);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            to[2 * i] = bf16_lo(w[i]);
            to[2 * i + 1] = bf16_hi(w[i]);
        }
    } else {
        __builtin_memcpy(to, row + at, N * 4);
    }
}

// ... at the row's end: those past it are zero.  (One by one, without conditions, so that
// no load waits for another.)
template <typename T, int N>
__device__ __forceinline__ void lora_load_end(const T* row, int at, int n, float (&to)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const T v = row[min(at + i, n - 1)];
        float x;
        if constexpr (sizeof(T) == 2) x = __uint_as_float((uint32_t)v << 16);
        else x = v;
        to[i] = at + i < n ? x : 0.f;
    }
}

// The adapters that a tile's 16 rows name, one bit for the first row of each.  A
// lane's row is lane % 16; -1: none.
struct LoraTile {
    int mine, lead;                    // the lane's adapter, and the first row that names it
    uint32_t firsts;

    __device__ __forceinline__ void set(const LoraArgs& a, int row0, int lane) {
        const int row = row0 + (lane & 15), p = row < a.n ? a.pick[row] : -1;
        mine = p >= 0 && p < a.n_adapters ? p : -1;
        lead = lane & 15;
#pragma unroll
        for (int j = 14; j >= 0; --j) {
            const int before = __builtin_amdgcn_readlane(mine, j);
            lead = (j < (lane & 15)) & (before == mine) ? j : lead;
        }
        firsts = (uint32_t)__ballot(mine >= 0 && lead == (lane & 15)) & 0xFFFFu;
    }
    // the adapter of the lowest bit of `left`
    __device__ __forceinline__ int adapter(uint32_t left) const {
        return __builtin_amdgcn_readlane(mine, __builtin_ctz(left));
    }
    // every n-th of them from the z-th on
    __device__ __forceinline__ uint32_t share(int z, int n) const {
        if (n == 1) return firsts;
        uint32_t got = 0;
        int d = 0;
        for (uint32_t left = firsts; left; left &= left - 1, ++d)
            if (d % n == z) got |= left & -left;
        return got;
    }
};

constexpr int kLoraWaves = 4;
constexpr long kLoraWhole = 16384;     // elements of an adapter's A, up to which a launch is saved
constexpr int kLoraMaxTiles = 16;      // tiles of rank

// Ranks t .. t + 15 of A_ad x over elements [k0, k1) of k, every `turns`-th 128 of them from the
// turn-th on: ranks 4g .. of row i.  A step of 32 elements is eight to a lane; the loads of four
// are on their way before the first product.
template <typename T>
__device__ __forceinline__ f32x4 lora_down(const LoraArgs& a, int ad, int t, const float* x, int k0, int k1, int turn, int turns,
                                           int lane) {
    constexpr int STEPS = 4;
    const int i = lane & 15, g = lane >> 4;
    const T* const w = static_cast<const T*>(a.a) + ((long)ad * a.rank + min(t + i, a.rank - 1)) * a.k;
    f32x4 acc[2] = {};
    for (int k = k0 + turn * (32 * STEPS); k < k1; k += turns * 32 * STEPS) {
        float wv[STEPS][8], xv[STEPS][8];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int at = k + 32 * s + 8 * g;
            if (k + 32 * s + 32 <= k1) {                 // (the same in every lane)
                lora_load<T, 8>(w, at, wv[s]);
                lora_load<float, 8>(x, at, xv[s]);
            } else if (k + 32 * s < k1) {
                lora_load_end<T, 8>(w, at, k1, wv[s]);
                lora_load_end<float, 8>(x, at, k1, xv[s]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) wv[s][e] = xv[s][e] = 0.f;
            }
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(wv[s][e], xv[s][e], acc[e & 1], 0, 0, 0);
    }
    return acc[0] + acc[1];
}

// Blocks: 16 rows, a piece of k, and of the tile's adapters (x their tiles of rank) every
// so many.
template <typename T>
__global__ __launch_bounds__(kLoraWaves * 64) void lora_down_kernel(LoraArgs a) {
    __shared__ f32x4 part[kLoraWaves][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const int row0 = blockIdx.x * 16, split = blockIdx.y, ranks = a.vr / 16;
    const int rank_blocks = gridDim.z > 1 ? ranks : 1, rb = blockIdx.z % rank_blocks;
    LoraTile tile;
    tile.set(a, row0, lane);
    const int k0 = split * a.k_piece, k1 = min(k0 + a.k_piece, a.k);
    const float* const x = a.x + min(row0 + i, a.n - 1) * a.ld_x;
    for (uint32_t left = tile.share(blockIdx.z / rank_blocks, gridDim.z / rank_blocks); left; left &= left - 1) {
        const int ad = tile.adapter(left);
        for (int t = rb * 16; t < a.vr; t += rank_blocks * 16) {
            const f32x4 acc = lora_down<T>(a, ad, t, x, k0, k1, wave, kLoraWaves, lane);
            __syncthreads();
            part[wave][lane] = acc;
            __syncthreads();
            // lane (row i, ranks 4g ..)
            if (wave == 0 && tile.mine == ad) {
                f32x4 sum = part[0][lane];
#pragma unroll
                for (int o = 1; o < kLoraWaves; ++o) sum += part[o][lane];
                *reinterpret_cast<f32x4*>(a.v + ((long)split * a.n + row0 + i) * a.vr + t + 4 * g) = sum;
            }
        }
    }
}

// A wave: 16 rows, and 64 elements of m.  Blocks of z take every so many of the tile's
// adapters and write these adapters' rows; block 0 also the rows without one.
// WHOLE: a block forms A x itself, a tile of rank (or, of few, a part of k) to a wave.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(kLoraWaves * 64) void lora_up_kernel(LoraArgs a) {
    constexpr int MT = 4;
    __shared__ f32x4 part[WHOLE ? kLoraMaxTiles : 1][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const int row0 = blockIdx.y * 16, row = row0 + i, here = min(row, a.n - 1), m0 = (blockIdx.x * kLoraWaves + wave) * (16 * MT);
    if (!WHOLE && m0 >= a.m) return;
    // (on their way before the adapters are known)
    f32x4 y[MT];
    const float* const base = a.base + here * a.ld_base;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        float b[4] = {0.f, 0.f, 0.f, 0.f};
        if (m0 + 16 * t + 16 <= a.m) lora_load<float, 4>(base, m0 + 16 * t + 4 * g, b);
        else if (m0 + 16 * t < a.m) lora_load_end<float, 4>(base, m0 + 16 * t + 4 * g, a.m, b);
        y[t] = f32x4{b[0], b[1], b[2], b[3]};
    }
    LoraTile tile;
    tile.set(a, row0, lane);
    const uint32_t todo = tile.share(blockIdx.z, gridDim.z);
    if (todo == 0 && blockIdx.z) return;
    const bool write = row < a.n && (tile.mine < 0 ? blockIdx.z == 0 : (todo >> tile.lead & 1) != 0);
    const float* const x = a.x + here * a.ld_x;
    const int ranks = a.vr / 16, parts = WHOLE && ranks < kLoraWaves ? kLoraWaves / ranks : 1;
    for (uint32_t left = todo; left; left &= left - 1) {
        const int ad = tile.adapter(left);
        const float scale = a.scales ? a.scales[ad] : 1.f;
        const bool mine = tile.mine == ad;
        if constexpr (WHOLE) {
            __syncthreads();                             // (the adapter before has been read)
            for (int item = wave; item < ranks * parts; item += kLoraWaves)
                part[item][lane] = lora_down<T>(a, ad, item / parts * 16, x, 0, a.k, item % parts, parts, lane);
            __syncthreads();
        }
        f32x4 acc[MT] = {};
        for (int t = 0; t < a.vr; t += 16) {
            float w[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const T* const b = static_cast<const T*>(a.b) + ((long)ad * a.m + min(m0 + 16 * mt + i, a.m - 1)) * a.rank;
                if (t + 16 <= a.rank) lora_load<T, 4>(b, t + 4 * g, w[mt]);
                else lora_load_end<T, 4>(b, t + 4 * g, a.rank, w[mt]);
            }
            // B operand: ranks t + 4g + e of row i at step e; past the last zero
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if constexpr (WHOLE) {
                for (int p = 0; p < parts; ++p) v += part[t / 16 * parts + p][lane];
            } else {
                const float* p = a.v + (long)here * a.vr + t + 4 * g;
#pragma unroll 4
                for (int s = 0; s < a.splits; ++s) v += *reinterpret_cast<const f32x4*>(p + (long)s * a.n * a.vr);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = t + 4 * g + e < a.rank ? v[e] : 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[mt] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[mt][e], v[e], acc[mt], 0, 0, 0);
        }
        // (other rows' columns hold what their x gives with this adapter: not theirs)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[mt][e] = mine ? y[mt][e] + scale * acc[mt][e] : y[mt][e];
    }
    if (!write) return;
    float* const to = a.y + row * a.ld_y;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = m0 + 16 * t + 4 * g;
        if (m + 4 <= a.m) __builtin_memcpy(to + m, &y[t], 16);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (m + e < a.m) to[m + e] = y[t][e];
    }
}

int lora_add_launch(const atlas_lora& l, const int* adapters, const float* x, long ld_x, const float* base, long ld_base,
                    float* y, long ld_y, int n, hipStream_t st) {
    const char* who = "lora_add";
    ATLAS_REQUIRE(l.fmt == ATLAS_W_F32 || l.fmt == ATLAS_W_BF16, "%s: format %d (f32 or bf16)", who, l.fmt);
    ATLAS_REQUIRE(l.n_adapters >= 0 && l.rank >= 1 && l.rank <= 256 && l.m >= 1 && l.k >= 1, "%s: %d adapters of rank %d (1 to 256), %d x %d",
                  who, l.n_adapters, l.rank, l.m, l.k);
    ATLAS_REQUIRE(l.m <= 1 << 24 && l.k <= 1 << 24 && n >= 0 && n <= 1 << 20, "%s: %d rows, %d x %d", who, n, l.m, l.k);
    ATLAS_REQUIRE(ld_x >= l.k && ld_base >= l.m && ld_y >= l.m, "%s: rows of %d and %d elements, %ld, %ld and %ld apart", who, l.k,
                  l.m, ld_x, ld_base, ld_y);
    if (n == 0) return ATLAS_OK;
    ATLAS_REQUIRE(adapters && x && base && y && (l.n_adapters == 0 || (l.a && l.b)), "%s: null argument", who);
    const int size = l.fmt == ATLAS_W_F32 ? 4 : 2;
    const uintptr_t floats = (uintptr_t)x | (uintptr_t)base | (uintptr_t)y | (uintptr_t)adapters | (uintptr_t)l.scales;
    const uintptr_t weights = (uintptr_t)l.a | (uintptr_t)l.b;
    ATLAS_REQUIRE((floats & 3) == 0 && weights % size == 0, "%s: misaligned argument", who);
    LoraArgs a{};
    a.a = l.a; a.b = l.b; a.scales = l.scales;
    a.n_adapters = l.n_adapters; a.rank = l.rank; a.m = l.m; a.k = l.k;
    a.pick = adapters;
    a.x = x; a.ld_x = ld_x; a.base = base; a.ld_base = ld_base; a.y = y; a.ld_y = ld_y;
    a.n = n;
    a.vr = (l.rank + 15) / 16 * 16;
    const int cus = device_cu_count(), tiles = (n + 15) / 16, named = std::min({16, n, std::max(l.n_adapters, 1)});
    ATLAS_REQUIRE(tiles <= 65535, "%s: %d rows", who, n);
    // blocks of their own for the adapters of a tile, where the tiles alone leave CUs idle
    const int wide = (l.m + 64 * kLoraWaves - 1) / (64 * kLoraWaves);
    const dim3 up(wide, tiles, (long)wide * tiles < 2 * cus ? named : 1);
#define LORA_RUN(KERNEL, GRID, ...) hipLaunchKernelGGL((KERNEL<__VA_ARGS__>), GRID, dim3(kLoraWaves * 64), 0, st, a)
    if (l.n_adapters > 0 && (long)l.k * a.vr <= kLoraWhole) {
        if (size == 2) LORA_RUN(lora_up_kernel, up, uint16_t, true);
        else LORA_RUN(lora_up_kernel, up, float, true);
        ATLAS_LAUNCH_CHECK("lora_up");
        return ATLAS_OK;
    }
    if (l.n_adapters > 0) {
        // pieces of k, of a turn of the waves at least, while the blocks do not fill the chip
        const bool apart = tiles < cus / 4;
        const int each = apart ? named * (a.vr / 16) : 1;
        const int most = (l.k + 511) / 512, want = std::max(1, 4 * cus / (tiles * each));
        a.splits = std::min(most, want);
        a.k_piece = ((l.k + a.splits - 1) / a.splits + 127) / 128 * 128;
        a.splits = (l.k + a.k_piece - 1) / a.k_piece;
        void* p = nullptr;
        const int rc = thread_scratch(SCR_LORA, (size_t)a.splits * n * a.vr * sizeof(float), &p);
        if (rc) return rc;
        a.v = static_cast<float*>(p);
        const dim3 down(tiles, a.splits, each);
        if (size == 2) LORA_RUN(lora_down_kernel, down, uint16_t);
        else LORA_RUN(lora_down_kernel, down, float);
        ATLAS_LAUNCH_CHECK("lora_down");
    }
    if (size == 2) LORA_RUN(lora_up_kernel, up, uint16_t, false);
    else LORA_RUN(lora_up_kernel, up, float, false);
#undef LORA_RUN
    ATLAS_LAUNCH_CHECK("lora_up");
    return ATLAS_OK;
}

}  // namespace atlas
