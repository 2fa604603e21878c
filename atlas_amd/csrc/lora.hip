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

// elements of T at p, p + 1, .. as f32; those from n on are zero
template <typename T, int N, bool VEC>
__device__ __forceinline__ void lora_load(const T* p, int n, float (&to)[N]) {
    if (VEC && n >= N) {
        if constexpr (sizeof(T) == 2) {
            uint32_t w[N / 2];
            __builtin_memcpy(w, __builtin_assume_aligned(p, N * 2), N * 2);
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                to[2 * i] = bf16_lo(w[i]);
                to[2 * i + 1] = bf16_hi(w[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) {
                const f32x4 w = reinterpret_cast<const f32x4*>(p)[i];
                to[4 * i] = w.x; to[4 * i + 1] = w.y; to[4 * i + 2] = w.z; to[4 * i + 3] = w.w;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (i < n) {
                if constexpr (sizeof(T) == 2) to[i] = __uint_as_float((uint32_t)p[i] << 16);
                else to[i] = p[i];
            } else {
                to[i] = 0.f;
            }
        }
    }
}

// The adapters that a tile's 16 rows name, one bit for the first row of each.  A
// lane's row is lane % 16; -1: none.
struct LoraTile {
    int mine;
    uint32_t firsts;

    __device__ __forceinline__ void set(const LoraArgs& a, int row0, int lane) {
        const int row = row0 + (lane & 15), p = row < a.n ? a.pick[row] : -1;
        mine = p >= 0 && p < a.n_adapters ? p : -1;
        bool first = mine >= 0;
#pragma unroll
        for (int j = 0; j < 15; ++j) {
            const int before = __builtin_amdgcn_readlane(mine, j);
            first = first & !((j < (lane & 15)) & (before == mine));
        }
        firsts = (uint32_t)__ballot(first) & 0xFFFFu;
    }
    // the adapter of the lowest bit of `left`
    __device__ __forceinline__ int adapter(uint32_t left) const {
        return __builtin_amdgcn_readlane(mine, __builtin_ctz(left));
    }
};

constexpr int kLoraWaves = 4;

template <typename T, bool VEC>
__global__ __launch_bounds__(kLoraWaves * 64) void lora_down_kernel(LoraArgs a) {
    __shared__ f32x4 part[kLoraWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int row0 = blockIdx.x * 16, split = blockIdx.y;
    LoraTile tile;
    tile.set(a, row0, lane);
    const int k0 = split * a.k_piece, k1 = min(k0 + a.k_piece, a.k);
    const float* const x = a.x + min(row0 + i, a.n - 1) * a.ld_x;
    int d = 0;
    for (uint32_t left = tile.firsts; left; left &= left - 1, ++d) {
        if (d % gridDim.z != blockIdx.z) continue;
        const int ad = tile.adapter(left);
        for (int t = 0; t < a.vr; t += 16) {
            const T* const w = static_cast<const T*>(a.a) + ((long)ad * a.rank + min(t + i, a.rank - 1)) * a.k;
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
            // 32 elements of k a step, eight to a lane
#pragma unroll 2
            for (int k = k0 + wave * 32 + 8 * g; k - 8 * g < k1; k += kLoraWaves * 32) {
                float wv[8], xv[8];
                lora_load<T, 8, VEC>(w + k, k1 - k, wv);
                lora_load<float, 8, VEC>(x + k, k1 - k, xv);
#pragma unroll
                for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(wv[e], xv[e], acc, 0, 0, 0);
            }
            __syncthreads();
            part[wave][lane] = acc;
            __syncthreads();
            // lane (row i, ranks 4g ..)
            if (wave == 0 && tile.mine == ad && row0 + i < a.n) {
                f32x4 sum = part[0][lane];
#pragma unroll
                for (int o = 1; o < kLoraWaves; ++o) sum += part[o][lane];
                *reinterpret_cast<f32x4*>(a.v + ((long)split * a.n + row0 + i) * a.vr + t + 4 * g) = sum;
            }
        }
    }
}

// a wave: 16 rows, and 64 elements of m in four tiles
template <typename T, bool VEC>
__global__ __launch_bounds__(kLoraWaves * 64) void lora_up_kernel(LoraArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int row0 = blockIdx.y * 16, m0 = (blockIdx.x * kLoraWaves + wave) * 64;
    if (m0 >= a.m) return;
    LoraTile tile;
    tile.set(a, row0, lane);
    const int row = row0 + i;
    f32x4 y[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int m = m0 + 16 * t + 4 * g;
        float b[4];
        if (row < a.n && m < a.m) lora_load<float, 4, VEC>(a.base + row * a.ld_base + m, a.m - m, b);
        else b[0] = b[1] = b[2] = b[3] = 0.f;
        y[t] = f32x4{b[0], b[1], b[2], b[3]};
    }
    for (uint32_t left = tile.firsts; left; left &= left - 1) {
        const int ad = tile.adapter(left);
        const float scale = a.scales ? a.scales[ad] : 1.f;
        const bool mine = tile.mine == ad;
        f32x4 acc[4] = {};
        for (int t = 0; t < a.vr; t += 16) {
            // B operand: ranks t + 4g + e of row i at step e
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if (mine)
                for (int s = 0; s < a.splits; ++s)
                    v += *reinterpret_cast<const f32x4*>(a.v + ((long)s * a.n + row) * a.vr + t + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (t + 4 * g + e >= a.rank) v[e] = 0.f;
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                const int m = min(m0 + 16 * mt + i, a.m - 1);
                float w[4];
                lora_load<T, 4, VEC>(static_cast<const T*>(a.b) + ((long)ad * a.m + m) * a.rank + t + 4 * g, a.rank - t - 4 * g, w);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[mt] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[e], v[e], acc[mt], 0, 0, 0);
            }
        }
        if (mine)
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) y[mt] += scale * acc[mt];
    }
    if (row >= a.n) return;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int m = m0 + 16 * t + 4 * g;
        float* to = a.y + row * a.ld_y + m;
        if (VEC && m + 4 <= a.m) *reinterpret_cast<f32x4*>(to) = y[t];
        else
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (m + e < a.m) to[e] = y[t][e];
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
    const uintptr_t floats = (uintptr_t)x | (uintptr_t)base | (uintptr_t)y | (uintptr_t)adapters | (uintptr_t)l.scales;
    const uintptr_t weights = (uintptr_t)l.a | (uintptr_t)l.b;
    const int size = l.fmt == ATLAS_W_F32 ? 4 : 2;
    ATLAS_REQUIRE((floats & 3) == 0 && weights % size == 0, "%s: misaligned argument", who);
    LoraArgs a{};
    a.a = l.a; a.b = l.b; a.scales = l.scales;
    a.n_adapters = l.n_adapters; a.rank = l.rank; a.m = l.m; a.k = l.k;
    a.pick = adapters;
    a.x = x; a.ld_x = ld_x; a.base = base; a.ld_base = ld_base; a.y = y; a.ld_y = ld_y;
    a.n = n;
    a.vr = (l.rank + 15) / 16 * 16;
    const int tiles = (n + 15) / 16, named = std::min({16, n, std::max(l.n_adapters, 1)});
    // pieces of k, of 512 elements at least, while the blocks do not fill the chip
    const int most = std::max(1, (l.k + 511) / 512), want = std::max(1, 2 * device_cu_count() / (tiles * named));
    a.splits = std::min(most, want);
    a.k_piece = ((l.k + a.splits - 1) / a.splits + 63) / 64 * 64;
    a.splits = (l.k + a.k_piece - 1) / a.k_piece;
    void* p = nullptr;
    const int rc = thread_scratch(SCR_LORA, (size_t)a.splits * n * a.vr * sizeof(float), &p);
    if (rc) return rc;
    a.v = static_cast<float*>(p);
    // whole vectors of every operand on their boundaries
    const bool vx = (((uintptr_t)x | weights) & 15) == 0 && ld_x % 4 == 0 && l.k % 8 == 0;
    const bool vy = (((uintptr_t)base | (uintptr_t)y | weights) & 15) == 0 && ld_base % 4 == 0 && ld_y % 4 == 0 && l.rank % 4 == 0;
    const dim3 down(tiles, a.splits, named), up((l.m + 64 * kLoraWaves - 1) / (64 * kLoraWaves), tiles);
    ATLAS_REQUIRE(tiles <= 65535, "%s: %d rows", who, n);
#define LORA_RUN(KERNEL, GRID, T, VEC) hipLaunchKernelGGL((KERNEL<T, VEC>), GRID, dim3(kLoraWaves * 64), 0, st, a)
    if (l.n_adapters > 0) {
        if (size == 2 && vx) LORA_RUN(lora_down_kernel, down, uint16_t, true);
        else if (size == 2) LORA_RUN(lora_down_kernel, down, uint16_t, false);
        else if (vx) LORA_RUN(lora_down_kernel, down, float, true);
        else LORA_RUN(lora_down_kernel, down, float, false);
        ATLAS_LAUNCH_CHECK("lora_down");
    }
    if (size == 2 && vy) LORA_RUN(lora_up_kernel, up, uint16_t, true);
    else if (size == 2) LORA_RUN(lora_up_kernel, up, uint16_t, false);
    else if (vy) LORA_RUN(lora_up_kernel, up, float, true);
    else LORA_RUN(lora_up_kernel, up, float, false);
#undef LORA_RUN
    ATLAS_LAUNCH_CHECK("lora_up");
    return ATLAS_OK;
}

}  // namespace atlas
