// lora.hip -- low-rank adapters beside a shared projection: each row has its own.
//
// y_r = base_r + s_a B_a (A_a x_r), a the row's adapter.  A tile is up to 16 rows of one
// adapter, wherever they are in the batch, so that no product is computed for rows of
// others.  Two launches, because every element of y needs the whole of A_a x_r:
//   1  v_r = A_a x_r: a block takes a tile and a piece of k, and leaves the tile's rows;
//   2  y = base + s B v: a block takes a tile and pieces of m, and of v the sum over
//      the pieces of k.
// Both are f32 matrix products of 16 x 16 x 4, exact products of bf16 or f32 weights
// and f32 activations; v stays f32.
//
// Few rows are bound by latency: 6.6 us for a row of 576 x 576 rank 8 (one launch), 9.2 for
// 13 rows of 4096 x 4096 rank 16 over 32 bf16 adapters (6.4 and 6.0 of kernel with cold
// caches), 15.8 for 70 rows of 8192 x 2048 rank 64 over 9 f32 adapters (23 MB of them:
// 5.6 us of bytes).  Many are bound by the stream of base and y: 64 us for 2047 rows of
// 11008 x 4096, 215 MB, 42 us at a copy's rate.  With tiles of 16 consecutive rows, each
// multiplied by every adapter that they name, the last two took 20.8 and 66, and 13 rows 9.9.
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
    int* lists;                        // [spans][tiles][17]: the adapter, 16 rows
    int tiles;                         // of a span of the rows, some of them empty
    int vr;                            // rank in whole tiles of 16
    int splits, k_piece;               // k's pieces, multiples of 512
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

constexpr int kLoraWaves = 4;
constexpr int kLoraSpan = 4096;        // rows that are sorted together
constexpr int kLoraMaxAdapters = 4095;
// Adapters up to which a wave counts its rows before it adds them in LDS, where adds to one
// word wait for each other (2047 rows of 5 adapters: 19.4 us of lora_down, 23.6 without).
constexpr int kLoraFewBins = 16;
constexpr int kLoraNone = -1, kLoraEmpty = -2;   // adapters of a tile

// A tile of a span of the rows: up to 16 rows of one adapter (or of none), in order.
// Every block finds its own, from the rows' adapters alone: rows of an adapter are counted
// in the order of the batch, so that all blocks agree.
struct LoraTile {
    int adapter, row, count;           // row of column lane % 16 (the first where there are fewer)

    __device__ __forceinline__ static int pick(const LoraArgs& a, int row) {
        const int p = a.pick[row];
        return p >= 0 && p < a.n_adapters ? p : kLoraNone;
    }
    __device__ __forceinline__ void keep(int* list, int lane) const {
        if (lane < 16) list[1 + lane] = lane < count ? row : -1;
        if (lane == 0) list[0] = adapter;
    }
    __device__ __forceinline__ void recall(const int* list, int lane) {
        adapter = __builtin_amdgcn_readfirstlane(list[0]);
        const int r = list[1 + (lane & 15)], first = __builtin_amdgcn_readfirstlane(r);
        count = __popcll(__ballot(r >= 0)) / 4;
        row = r >= 0 ? r : first;
    }

    // Up to 64 rows from row0 on: in a wave's registers.
    __device__ __forceinline__ void few(const LoraArgs& a, int row0, int n, int t, int lane) {
        const int mine = pick(a, row0 + min(lane, n - 1)), p = lane < n ? mine : kLoraEmpty;
        int before = 0;                                  // rows before it of its adapter
        for (int j = 0; j < n; ++j) {
            const int o = __builtin_amdgcn_readlane(p, j);
            before += (j < lane) & (o == p);
        }
        uint64_t heads = __ballot((lane < n) & ((before & 15) == 0));
        for (int s = 0; s < t; ++s) heads &= heads - 1;
        if (heads == 0) {
            adapter = kLoraEmpty;
            return;
        }
        const int head = __builtin_ctzll(heads);
        adapter = __builtin_amdgcn_readlane(p, head);
        const int nth = __builtin_amdgcn_readlane(before, head) >> 4;
        uint64_t rows = __ballot((p == adapter) & (before >> 4 == nth));
        count = __popcll(rows);
#pragma unroll
        for (int s = 0; s < 15; ++s) rows = s < (lane & 15) ? rows & (rows - 1) : rows;
        row = row0 + (rows ? __builtin_ctzll(rows) : head);
    }

    // Up to kLoraSpan: a count of each adapter's rows in LDS (the last: of none), a sum over
    // the tiles of the adapters before, and the rows of the adapter found.
    struct Counts {
        int rows[kLoraMaxAdapters + 1], waves[kLoraSpan / 64], total[kLoraWaves], found[3], tile[16];
    };
    __device__ __forceinline__ void many(Counts& c, const LoraArgs& a, int row0, int n, int t, int lane, int wave) {
        constexpr int THREADS = kLoraWaves * 64, STEPS = kLoraSpan / THREADS;
        const int tid = wave * 64 + lane, bins = a.n_adapters + 1;
        int p[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (s * THREADS >= n) break;
            p[s] = a.pick[row0 + min(s * THREADS + tid, n - 1)];
        }
        for (int b = tid; b < bins; b += THREADS) c.rows[b] = 0;
        if (tid < kLoraSpan / 64) c.waves[tid] = 0;
        if (tid == 0) c.found[0] = -1;
        __syncthreads();
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (s * THREADS >= n) break;
            const int r = s * THREADS + tid;
            p[s] = p[s] >= 0 && p[s] < a.n_adapters ? p[s] : a.n_adapters;
            p[s] = r < n ? p[s] : -1;
            if (bins > kLoraFewBins && r < n) atomicAdd(&c.rows[p[s]], 1);
        }
        if (bins <= kLoraFewBins) {
            int of = 0;                                  // lane b: rows of adapter b
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                if (s * THREADS >= n) break;
                for (int b = 0; b < bins; ++b) {
                    const int rows = __popcll(__ballot(p[s] == b));
                    of += lane == b ? rows : 0;
                }
            }
            if (lane < bins) atomicAdd(&c.rows[lane], of);
        }
        __syncthreads();
        const int each = (bins + THREADS - 1) / THREADS, b0 = min(tid * each, bins), b1 = min(b0 + each, bins);
        int own = 0;
        for (int b = b0; b < b1; ++b) own += (c.rows[b] + 15) / 16;
        int upto = own;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int o = __shfl_up(upto, s, 64);
            upto += lane >= s ? o : 0;
        }
        if (lane == 63) c.total[wave] = upto;
        __syncthreads();
        int at = upto - own;
#pragma unroll
        for (int w = 0; w < kLoraWaves; ++w) at += w < wave ? c.total[w] : 0;
        if (t >= at && t < at + own)                     // (one thread)
            for (int b = b0; b < b1; ++b) {
                const int tiles = (c.rows[b] + 15) / 16;
                if (t >= at && t < at + tiles) {
                    c.found[0] = b;
                    c.found[1] = t - at;
                    c.found[2] = c.rows[b];
                }
                at += tiles;
            }
        __syncthreads();
        const int bin = __builtin_amdgcn_readfirstlane(c.found[0]);
        if (bin < 0) {
            adapter = kLoraEmpty;
            return;
        }
        adapter = bin == a.n_adapters ? kLoraNone : bin;
        const int lo = c.found[1] * 16;
        count = __builtin_amdgcn_readfirstlane(min(16, c.found[2] - lo));
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (s * THREADS >= n) break;
            const int of = __popcll(__ballot(p[s] == bin));
            if (lane == 0) c.waves[s * kLoraWaves + wave] = of;
        }
        __syncthreads();
        const int mine = c.waves[lane];
        int before = mine;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int o = __shfl_up(before, s, 64);
            before += lane >= s ? o : 0;
        }
        before -= mine;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (s * THREADS >= n) break;
            const uint64_t m = __ballot(p[s] == bin);
            const int pos = __builtin_amdgcn_readlane(before, s * kLoraWaves + wave) + __popcll(m & ((1ull << lane) - 1)) - lo;
            if (p[s] == bin && pos >= 0 && pos < 16) c.tile[pos] = row0 + s * THREADS + tid;
        }
        __syncthreads();
        row = c.tile[(lane & 15) < count ? lane & 15 : 0];
    }
};

// Elements of an adapter's A up to which every block forms A x itself, which saves a launch
// (rank 16, 13 rows of 1024 x 1024: 7.4 us, 8.9 in two; 2048 x 2048: 9.8 and 8.9; 4096 x
// 4096: 14.5 and 9.2; 70 rows of 4096 x 1024 9.7 and 10.6).  Blocks of one tile form it anew
// each, and count its rows, which many rows make longer than a launch: 500 rows of 1024 x 1024
// 11.3 and 12.0, but of 4096 x 1024 16.1 and 14.6, 2000 rows 45 and 32.
constexpr long kLoraWhole = 16384;
constexpr int kLoraUp = 4;             // blocks of a CU (2047 rows: 65 us, 71 with a block to each 256 of m)
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

// A block's tile: t of the span's.
template <bool MANY>
__device__ __forceinline__ void lora_tile(LoraTile& tile, const LoraArgs& a, int span, int t, int lane, int wave) {
    const int row0 = span * kLoraSpan, n = min(a.n - row0, kLoraSpan);
    if constexpr (MANY) {
        __shared__ LoraTile::Counts counts;
        tile.many(counts, a, row0, n, t, lane, wave);
    } else {
        tile.few(a, row0, n, t, lane);
    }
}

// Blocks: a tile, a piece of k, and a span of the rows (x a tile of rank).
template <typename T, bool MANY>
__global__ __launch_bounds__(kLoraWaves * 64) void lora_down_kernel(LoraArgs a, int rank_blocks) {
    __shared__ f32x4 part[kLoraWaves][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    const int t0 = blockIdx.x, split = blockIdx.y, span = blockIdx.z / rank_blocks, rb = blockIdx.z % rank_blocks;
    LoraTile tile;
    lora_tile<MANY>(tile, a, span, t0, lane, wave);
    if (split == 0 && rb == 0 && wave == 0) tile.keep(a.lists + ((long)span * a.tiles + t0) * 17, lane);
    if (tile.adapter < 0) return;
    const int k0 = split * a.k_piece, k1 = min(k0 + a.k_piece, a.k);
    const float* const x = a.x + tile.row * a.ld_x;
    for (int t = rb * 16; t < a.vr; t += rank_blocks * 16) {
        const f32x4 acc = lora_down<T>(a, tile.adapter, t, x, k0, k1, wave, kLoraWaves, lane);
        __syncthreads();
        part[wave][lane] = acc;
        __syncthreads();
        // lane (row i, ranks 4g ..)
        if (wave == 0 && (lane & 15) < tile.count) {
            f32x4 sum = part[0][lane];
#pragma unroll
            for (int o = 1; o < kLoraWaves; ++o) sum += part[o][lane];
            *reinterpret_cast<f32x4*>(a.v + ((long)split * a.n + tile.row) * a.vr + t + 4 * g) = sum;
        }
    }
}

// A wave: a tile, and of m every so many 64 elements.
// WHOLE: a block finds its tile and forms A x itself, a tile of rank (or, of few, a part of
// k) to a wave.
template <typename T, bool WHOLE, bool MANY>
__global__ __launch_bounds__(kLoraWaves * 64) void lora_up_kernel(LoraArgs a) {
    constexpr int MT = 4, WIDE = 16 * MT * kLoraWaves;
    __shared__ f32x4 part[kLoraMaxTiles][64];
    __shared__ float turn[kLoraWaves][16][16 * MT + 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    LoraTile tile;
    if constexpr (WHOLE) lora_tile<MANY>(tile, a, blockIdx.z, blockIdx.y, lane, wave);
    else tile.recall(a.lists + ((long)blockIdx.z * a.tiles + blockIdx.y) * 17, lane);
    if (tile.adapter == kLoraEmpty) return;
    // y by rows: four a step, 64 elements of each in 16 lanes
    long base_at[MT], y_at[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = __shfl(tile.row, 4 * t + g, 64);
        base_at[t] = row * a.ld_base;
        y_at[t] = row * a.ld_y;
    }
    float y[MT][4] = {};
    const auto load = [&](int m0) {
        if (m0 + 16 * MT <= a.m) {
#pragma unroll
            for (int t = 0; t < MT; ++t) lora_load<float, 4>(a.base + base_at[t], m0 + 4 * i, y[t]);
        } else if (m0 < a.m) {
#pragma unroll
            for (int t = 0; t < MT; ++t) lora_load_end<float, 4>(a.base + base_at[t], m0 + 4 * i, a.m, y[t]);
        }
    };
    // A operand: ranks t + 4g .. of B's rows
    const int ad = tile.adapter;
    const T* const bs = static_cast<const T*>(a.b) + (long)max(ad, 0) * a.m * a.rank;
    float w[MT][4] = {};
    const auto weights = [&](int m0, int t) {
        const T* b[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) b[mt] = bs + (long)min(m0 + 16 * mt + i, a.m - 1) * a.rank;
        if (t + 16 <= a.rank) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) lora_load<T, 4>(b[mt], t + 4 * g, w[mt]);
        } else {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) lora_load_end<T, 4>(b[mt], t + 4 * g, a.rank, w[mt]);
        }
    };
    int m0 = blockIdx.x * WIDE + wave * (16 * MT);
    load(m0);
    if (ad >= 0) weights(m0, 0);
    float scale = 1.f;
    if (ad >= 0) {
        if (a.scales) scale = a.scales[ad];
        // v in LDS, a part of it to a wave: ranks t + 4g .. of row i, as the products want them
        const int ranks = a.vr / 16, parts = ranks < kLoraWaves ? kLoraWaves / ranks : 1;
        for (int item = wave; item < ranks * parts; item += kLoraWaves) {
            const int t = item / parts * 16, p = item % parts;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if constexpr (WHOLE) {
                v = lora_down<T>(a, ad, t, a.x + tile.row * a.ld_x, 0, a.k, p, parts, lane);
            } else {
                const float* const from = a.v + (long)tile.row * a.vr + t + 4 * g;
#pragma unroll 4
                for (int s = p; s < a.splits; s += parts) v += *reinterpret_cast<const f32x4*>(from + (long)s * a.n * a.vr);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = t + 4 * g + e < a.rank ? v[e] : 0.f;   // (past the rank: what the last gives)
            part[item][lane] = v;
        }
        __syncthreads();
    }
    for (; m0 < a.m; m0 += gridDim.x * WIDE) {
        float now[MT][4];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) now[t][e] = y[t][e];
        if (ad >= 0) {
            const int parts = a.vr < 16 * kLoraWaves ? kLoraWaves / (a.vr / 16) : 1;
            f32x4 acc[MT] = {};
            for (int t = 0; t < a.vr; t += 16) {
                f32x4 v = part[t / 16 * parts][lane];
                for (int p = 1; p < parts; ++p) v += part[t / 16 * parts + p][lane];
                float this_w[MT][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) this_w[mt][e] = w[mt][e];
                const bool more = t + 16 < a.vr;         // (the next are on their way)
                weights(more ? m0 : m0 + (int)gridDim.x * WIDE, more ? t + 16 : 0);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[mt] = __builtin_amdgcn_mfma_f32_16x16x4f32(this_w[mt][e], v[e], acc[mt], 0, 0, 0);
            }
            load(m0 + gridDim.x * WIDE);
            // from columns to rows, in the wave's own part of LDS
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) *reinterpret_cast<f32x4*>(&turn[wave][i][16 * mt + 4 * g]) = scale * acc[mt];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const f32x4 add = *reinterpret_cast<const f32x4*>(&turn[wave][4 * t + g][4 * i]);
#pragma unroll
                for (int e = 0; e < 4; ++e) now[t][e] += add[e];
            }
            __builtin_amdgcn_wave_barrier();
        } else {
            load(m0 + gridDim.x * WIDE);
        }
        const int m = m0 + 4 * i;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if (4 * t + g >= tile.count) continue;
            float* const to = a.y + y_at[t] + m;
            if (m + 4 <= a.m) __builtin_memcpy(to, now[t], 16);
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (m + e < a.m) to[e] = now[t][e];
        }
    }
}

int lora_add_launch(const atlas_lora& l, const int* adapters, const float* x, long ld_x, const float* base, long ld_base,
                    float* y, long ld_y, int n, hipStream_t st) {
    const char* who = "lora_add";
    ATLAS_REQUIRE(l.fmt == ATLAS_W_F32 || l.fmt == ATLAS_W_BF16, "%s: format %d (f32 or bf16)", who, l.fmt);
    ATLAS_REQUIRE(l.n_adapters >= 0 && l.n_adapters <= kLoraMaxAdapters && l.rank >= 1 && l.rank <= 256 && l.m >= 1 && l.k >= 1,
                  "%s: %d adapters (up to 4095) of rank %d (1 to 256), %d x %d",
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
    ATLAS_REQUIRE(std::max({ld_x, ld_base, ld_y}) < 1L << 40, "%s: rows %ld, %ld and %ld elements apart", who, ld_x, ld_base, ld_y);
    // y's rows and p's of w elements (which may lie between them) have nothing in common
    const auto apart = [&](const float* p, long w, long ld) {
        const uintptr_t y0 = (uintptr_t)y, p0 = (uintptr_t)p;
        if (y0 + ((n - 1) * ld_y + l.m) * 4 <= p0 || p0 + ((n - 1) * ld + w) * 4 <= y0) return true;
        const long at = ((((long)p0 - (long)y0) / 4) % ld_y + ld_y) % ld_y;
        return ld == ld_y && at >= l.m && at + w <= ld_y;
    };
    ATLAS_REQUIRE(apart(x, l.k, ld_x) && ((base == y && ld_base == ld_y) || apart(base, l.m, ld_base)), "%s: y overlaps x or base", who);
    const ByteRows to(y, n, l.m * 4L, ld_y * 4);
    const long each = (long)l.n_adapters * l.rank * size;
    ATLAS_REQUIRE(rows_apart(ByteRows(adapters, n * 4L), to) && (!l.scales || rows_apart(ByteRows(l.scales, l.n_adapters * 4L), to)) &&
                      rows_apart(ByteRows(l.a, each * l.k), to) && rows_apart(ByteRows(l.b, each * l.m), to),
                  "%s: y overlaps adapters", who);
    LoraArgs a{};
    a.a = l.a; a.b = l.b; a.scales = l.scales;
    a.n_adapters = l.n_adapters; a.rank = l.rank; a.m = l.m; a.k = l.k;
    a.pick = adapters;
    a.x = x; a.ld_x = ld_x; a.base = base; a.ld_base = ld_base; a.y = y; a.ld_y = ld_y;
    a.n = n;
    a.vr = (l.rank + 15) / 16 * 16;
    // tiles of a span: each adapter's last may be short
    const int cus = device_cu_count(), spans = (n + kLoraSpan - 1) / kLoraSpan, span = std::min(n, kLoraSpan);
    const int tiles = span / 16 + std::min(span, l.n_adapters + 1), wide = (l.m + 64 * kLoraWaves - 1) / (64 * kLoraWaves);
    a.tiles = tiles;
    // (a block goes on along m where there are enough without)
    const dim3 up(std::max(1, std::min(wide, kLoraUp * cus / (tiles * spans))), tiles, spans);
    const bool many = n > 64;
#define LORA_RUN(KERNEL, GRID, ...) hipLaunchKernelGGL(KERNEL, GRID, dim3(kLoraWaves * 64), 0, st, __VA_ARGS__)
    if (l.n_adapters == 0 || (long)l.k * a.vr <= kLoraWhole) {
        if (size == 2 && many) LORA_RUN((lora_up_kernel<uint16_t, true, true>), up, a);
        else if (size == 2) LORA_RUN((lora_up_kernel<uint16_t, true, false>), up, a);
        else if (many) LORA_RUN((lora_up_kernel<float, true, true>), up, a);
        else LORA_RUN((lora_up_kernel<float, true, false>), up, a);
        ATLAS_LAUNCH_CHECK("lora_up");
        return ATLAS_OK;
    }
    // pieces of k, of a turn of the waves at least, while the blocks do not fill the chip
    const int rank_blocks = tiles * spans < cus ? a.vr / 16 : 1;
    const int most = (l.k + 511) / 512, blocks = tiles * spans * rank_blocks, want = (4 * cus + blocks - 1) / blocks;
    a.splits = std::min(most, want);
    a.k_piece = ((l.k + a.splits - 1) / a.splits + 511) / 512 * 512;
    a.splits = (l.k + a.k_piece - 1) / a.k_piece;
    const size_t sums = (size_t)a.splits * n * a.vr;
    void* p = nullptr;
    const int rc = thread_scratch(SCR_LORA, (sums + (size_t)spans * tiles * 17) * sizeof(float), &p);
    if (rc) return rc;
    a.v = static_cast<float*>(p);
    a.lists = reinterpret_cast<int*>(a.v + sums);
    const dim3 down(tiles, a.splits, spans * rank_blocks);
    if (size == 2 && many) LORA_RUN((lora_down_kernel<uint16_t, true>), down, a, rank_blocks);
    else if (size == 2) LORA_RUN((lora_down_kernel<uint16_t, false>), down, a, rank_blocks);
    else if (many) LORA_RUN((lora_down_kernel<float, true>), down, a, rank_blocks);
    else LORA_RUN((lora_down_kernel<float, false>), down, a, rank_blocks);
    ATLAS_LAUNCH_CHECK("lora_down");
    if (size == 2) LORA_RUN((lora_up_kernel<uint16_t, false, false>), up, a);
    else LORA_RUN((lora_up_kernel<float, false, false>), up, a);
#undef LORA_RUN
    ATLAS_LAUNCH_CHECK("lora_up");
    return ATLAS_OK;
}

}  // namespace atlas
