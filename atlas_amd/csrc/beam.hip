// beam.hip -- beam search: the choice of a group's best continuations over its beams
// and the vocabulary, and the reordering of the beams' states.
#include <algorithm>
#include <memory>
#include <new>

#include "many.hpp"

namespace atlas {

// ---- selection --------------------------------------------------------------------
//
// A candidate is a beam r and a token t, its score s_r + (z_rt - lse_r) with
// lse_r = log sum_t exp z_rt, in 64 bits: sums of log probabilities over a long text
// have steps of 1e-5 in 32 bits, where candidates lie closer.  Within a row the order
// is that of the logits, so that only a row's n_out largest can be chosen.
//   1  a block takes a piece of a row: its largest logit, sum of exponentials, and
//      n_out largest (in one pass, from registers);
//   2  a block joins a group's pieces: lse of each row, then the largest scores.
// The n_out largest of many: each lane's largest first; the n_out-th largest of a wave's
// 64 is a bound that at least n_out elements reach, so that what lies below it goes, and
// the few that are left are ranked by counting.  Where many reach the bound (equal
// logits), the largest is taken n_out times.
//
// Bound by what is not the stream of logits: 64 rows of 100278 of them, 25.7 MB and 5 us of
// bytes, take 24 us: the loads and 64-bit exponentials (5 us of the VALU) of 448 pieces, then
// their bounds and ranks, each pass over a block's registers a chain of LDS and barriers,
// and the join (7).  4 rows of 49152, less than a block to a CU, take 11: a block's chain (6) and
// the join's (5).

constexpr int kBeamMaxOut = 64;
constexpr int kBeamThreads = 512;
constexpr int kBeamWaves = kBeamThreads / 64;
constexpr int kBeamList = 1024;

// order-preserving: larger logits have larger keys; 0 for what is no candidate
__device__ __forceinline__ uint32_t beam_order(float z) {
    const uint32_t u = __float_as_uint(z);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float beam_logit(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

constexpr uint32_t kBeamLowest = 0x00800000u;            // of the lowest finite logit

// larger first; of equal logits the lower token
__device__ __forceinline__ uint64_t beam_key(float z, uint32_t token) {
    return z > -__builtin_inff() ? (uint64_t)beam_order(z + 0.f) << 32 | (uint32_t)~token : 0;   // (-0 is 0)
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int mask) {
    const uint32_t lo = __shfl_xor((int)(uint32_t)v, mask, 64), hi = __shfl_xor((int)(uint32_t)(v >> 32), mask, 64);
    return (uint64_t)hi << 32 | lo;
}

// One step of a reduction over the wave's lanes (DPP: quads, rows of 16, then rows to the
// next); after all six, lane 63 has the result.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp32(uint32_t v) {
    return __builtin_amdgcn_update_dpp(v, v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
    return (uint64_t)dpp32<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | dpp32<CTRL, ROWS>((uint32_t)v);
}
template <typename T, int CTRL, int ROWS>
__device__ __forceinline__ T dpp_of(T v) {
    if constexpr (sizeof(T) == 8) return dpp64<CTRL, ROWS>(v);
    else return dpp32<CTRL, ROWS>(v);
}
__device__ __forceinline__ uint32_t last_lane(uint32_t v) { return __builtin_amdgcn_readlane(v, 63); }
__device__ __forceinline__ uint64_t last_lane(uint64_t v) {
    return (uint64_t)last_lane((uint32_t)(v >> 32)) << 32 | last_lane((uint32_t)v);
}
template <typename T>
__device__ __forceinline__ T wave_most(T v) {
    const auto step = [&](T w) { v = w > v ? w : v; };
    step(dpp_of<T, 0xB1, 0xF>(v));
    step(dpp_of<T, 0x4E, 0xF>(v));
    step(dpp_of<T, 0x141, 0xF>(v));
    step(dpp_of<T, 0x140, 0xF>(v));
    step(dpp_of<T, 0x142, 0xA>(v));
    step(dpp_of<T, 0x143, 0xC>(v));
    return last_lane(v);
}

// A bound that n or a few more of the wave's 64 keys reach (0: fewer than n are not 0), found
// between 0 and the largest key `most`.
template <typename T>
__device__ __forceinline__ T wave_bound(T key, T most, int n) {
    if (__popcll(__ballot(key != 0)) < n) return 0;
    T lo = ~wave_most((T)~(key ? key : most)), hi = most;    // (the smallest key) n keys reach lo
    if (__popcll(__ballot(key == most)) >= n) return most;
    while (hi - lo > 1) {
        const T mid = lo + (hi - lo) / 2;
        const int reach = __popcll(__ballot(key >= mid));
        if (reach >= n) {
            lo = mid;
            if (reach <= n + n / 4) break;
        } else {
            hi = mid;
        }
    }
    return lo;
}

__device__ __forceinline__ uint64_t beam_order(double s) {
    const uint64_t u = (uint64_t)__double_as_longlong(s);
    return u >> 63 ? ~u : u | 1ull << 63;
}

// the wave's sum, in every lane (DPP, as wave_sum)
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add64(double v) {
    const int2 w = __builtin_bit_cast(int2, v);
    const int2 m = {__builtin_amdgcn_update_dpp(0, w.x, CTRL, ROWS, 0xF, false),
                    __builtin_amdgcn_update_dpp(0, w.y, CTRL, ROWS, 0xF, false)};
    return v + __builtin_bit_cast(double, m);
}
__device__ __forceinline__ double wave_sum64(double v) {
    v = dpp_add64<0xB1, 0xF>(v);
    v = dpp_add64<0x4E, 0xF>(v);
    v = dpp_add64<0x141, 0xF>(v);
    v = dpp_add64<0x140, 0xF>(v);
    v = dpp_add64<0x142, 0xA>(v);
    v = dpp_add64<0x143, 0xC>(v);
    const int2 w = __builtin_bit_cast(int2, v);
    const int2 r = {__builtin_amdgcn_readlane(w.x, 63), __builtin_amdgcn_readlane(w.y, 63)};
    return __builtin_bit_cast(double, r);
}

// exp(x) of N values side by side, -708 <= x <= 0: x = n ln 2 + r with |r| <= ln 2 / 2 (ln 2 in
// two parts, as Cody and Waite have it; n by adding a number whose last place is 1), and
// exp r by its series, of which the first term left out is 2e-16.
template <int N>
__device__ __forceinline__ void beam_exp(double (&x)[N]) {
    constexpr double ROUND = 0x1.8p52;
    constexpr double C[13] = {1.0 / 479001600.0, 1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0,
                              1.0 / 5040.0, 1.0 / 720.0, 1.0 / 120.0, 1.0 / 24.0, 1.0 / 6.0, 0.5, 1.0, 1.0};
    double r[N], p[N];
    int k[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const double t = __builtin_fma(x[i], 1.4426950408889634, ROUND), n = t - ROUND;
        k[i] = (int)__builtin_bit_cast(uint64_t, t);
        r[i] = __builtin_fma(n, -0x1.62e42fee00000p-1, x[i]);      // the first 32 bits of ln 2
        r[i] = __builtin_fma(n, -0x1.a39ef35793c76p-33, r[i]);     // and the rest
        p[i] = C[0];
    }
#pragma unroll
    for (int c = 1; c < 13; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = __builtin_fma(p[i], r[i], C[c]);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __builtin_ldexp(p[i], k[i]);
}

// what a piece of a row leaves
struct BeamPiece {
    double sum;                        // of exp(z - top); NaN: the row has a NaN or +inf
    float top;
    int pad;
};

__device__ __forceinline__ bool beam_dead(double score) { return !(fabs(score) < __builtin_inf()); }

// PER: logits of a thread
template <int PER>
__global__ __launch_bounds__(kBeamThreads, PER > 16 ? 4 : 8) void beam_rows_kernel(const float* __restrict__ logits, long ld, int vocab,
                                                                 const double* __restrict__ scores, int n_out,
                                                                 BeamPiece* __restrict__ pieces, uint64_t* __restrict__ keys) {
    constexpr int W = kBeamWaves;
    __shared__ uint64_t list[kBeamList];
    __shared__ uint64_t largest[W];
    __shared__ uint32_t bound[W];
    __shared__ float tops[W];
    __shared__ double sums[W];
    __shared__ int count;
    const int row = blockIdx.y, piece = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* z = logits + (long)row * ld;
    const int first = piece * (PER * kBeamThreads);
    const bool dead = beam_dead(scores[row]);
    // Vectors on their boundaries, wherever the row starts; lanes at its ends load a vector
    // of its middle and then what they have one by one, so that no load waits for another.
    const int shift = (int)((uintptr_t)z >> 2 & 3);
    const auto token = [&](int j) { return first + (j / 4 * kBeamThreads + tid) * 4 + j % 4 - shift; };
    float x[PER];
    bool edge = vocab < 8;
    if (!edge) {
#pragma unroll
        for (int j = 0; j < PER; j += 4) {
            const int t = token(j);
            const bool inside = (t >= 0) & (t + 4 <= vocab);
            const f32x4 v = *reinterpret_cast<const f32x4*>(z + (inside ? t : 4 - shift));
#pragma unroll
            for (int i = 0; i < 4; ++i) x[j + i] = v[i];
            edge = edge | !inside;
        }
    }
    if (edge)
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int t = token(j);
            const float v = z[min(max(t, 0), vocab - 1)];
            x[j] = t >= 0 && t < vocab ? v : -__builtin_inff();
        }
    if (dead) return;                                    // (the join does not look at its rows' pieces either)
    if (tid == 0) count = 0;
    float mine = -__builtin_inff();
    bool nan = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        mine = fmaxf(mine, x[j]);
        nan = nan | (x[j] != x[j]);
    }
    const uint32_t order = mine > -__builtin_inff() ? beam_order(mine + 0.f) : 0, most_order = wave_most(order);
    const float top = most_order ? beam_logit(most_order) : -__builtin_inff();
    // relative to the wave's largest; terms below e^-708 are as good as none
    double sum = 0.0;
    if (top > -__builtin_inff())
#pragma unroll
        for (int j = 0; j < PER; j += 4) {
            double d[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) d[i] = __builtin_fmax((double)x[j + i] - (double)top, -708.0);
            beam_exp(d);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += d[i];
        }
    sum = wave_sum64(nan || top == __builtin_inff() ? __builtin_nan("") : sum);
    const uint32_t nth = wave_bound(order, most_order, n_out);
    if (lane == 0) {
        bound[wave] = nth;
        tops[wave] = top;
        sums[wave] = sum;
    }
    __syncthreads();
    uint32_t least = kBeamLowest;
#pragma unroll
    for (int w = 0; w < W; ++w) least = max(least, bound[w]);
    if (order >= least) {
        const float reach = beam_logit(least);
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (x[j] >= reach) {
                const int at = atomicAdd(&count, 1);
                if (at < kBeamList) list[at] = beam_key(x[j], token(j));
            }
    }
    __syncthreads();
    const long at = (long)row * gridDim.x + piece;
    if (wave == W - 1) {                                 // (a lane to a wave)
        const float most = wave_max(tops[min(lane, W - 1)]);
        double f[1] = {__builtin_fmax((double)tops[min(lane, W - 1)] - (double)most, -708.0)};
        beam_exp(f);
        const double part = lane < W ? sums[lane] : 0.0, all = wave_sum64(part == 0.0 ? 0.0 : part * f[0]);
        if (lane == 0) pieces[at] = {all, most, 0};
    }
    uint64_t* to = keys + at * n_out;
    const int n = count;
    if (n > kBeamList) {
        uint64_t last = ~0ull;
        for (int k = 0; k < n_out; ++k) {
            uint64_t best = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const uint64_t key = beam_key(x[j], token(j));
                best = key < last && key > best ? key : best;
            }
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) {
                const uint64_t other = shfl_xor64(best, d);
                best = other > best ? other : best;
            }
            __syncthreads();
            if (lane == 0) largest[wave] = best;
            __syncthreads();
            last = 0;
            for (int w = 0; w < W; ++w) last = largest[w] > last ? largest[w] : last;
            if (tid == 0) to[k] = last;
        }
        return;
    }
    for (int e = tid; e < n; e += kBeamThreads) {
        const uint64_t key = list[e];
        int rank = 0;
#pragma unroll 8
        for (int i = 0; i < n; ++i) rank += list[i] > key;
        if (rank < n_out) to[rank] = key;
    }
    for (int e = n + tid; e < n_out; e += kBeamThreads) to[e] = 0;
}

// a candidate: larger scores first, of equal ones the lower beam, then its order there
struct BeamCand {
    double score;
    uint64_t key;
    int beam;
};

__device__ __forceinline__ bool beam_before(const BeamCand& a, const BeamCand& b) {
    return a.score > b.score || (a.score == b.score && (a.beam < b.beam || (a.beam == b.beam && a.key > b.key)));
}

constexpr double kBeamNone = -__builtin_huge_val();
constexpr BeamCand kBeamNobody = {kBeamNone, 0, 64};

__device__ __forceinline__ BeamCand wave_first(BeamCand v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const BeamCand w = {__shfl_xor(v.score, d, 64), shfl_xor64(v.key, d), __shfl_xor(v.beam, d, 64)};
        if (beam_before(w, v)) v = w;
    }
    return v;
}

__global__ __launch_bounds__(kBeamThreads) void beam_join_kernel(const double* __restrict__ scores, int vocab, int width,
                                                                 int n_out, int n_pieces, const BeamPiece* __restrict__ pieces,
                                                                 const uint64_t* __restrict__ keys, uint32_t* __restrict__ tokens,
                                                                 int* __restrict__ parents, double* __restrict__ out_scores) {
    constexpr int W = kBeamWaves, HELD = 4;              // candidates of a thread in registers
    __shared__ double less[64], given[64];               // a row's lse (NaN: no candidates) and score
    __shared__ uint64_t bound[W];
    __shared__ BeamCand first[W];
    __shared__ double list_score[kBeamList];
    __shared__ uint64_t list_key[kBeamList];
    __shared__ int list_beam[kBeamList];
    __shared__ int count;
    const int group = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long row0 = (long)group * width;
    const uint32_t per_row = n_pieces * n_out, all = width * per_row;
    // (on their way before the rows' sums are known)
    const uint64_t* const from = keys + row0 * per_row;
    uint64_t held[HELD];
#pragma unroll
    for (int j = 0; j < HELD; ++j) held[j] = from[min((uint32_t)(tid + j * kBeamThreads), all - 1)];   // (of dead beams: anything)
    if (tid == 0) count = 0;
    for (int r = wave; r < width; r += W) {
        const double score = scores[row0 + r];
        const BeamPiece* p = pieces + (row0 + r) * n_pieces;
        const BeamPiece mine = p[min(lane, n_pieces - 1)];
        double z = __builtin_nan("");
        if (!beam_dead(score)) {
            float top = mine.top;
            for (int i = lane + 64; i < n_pieces; i += 64) top = fmaxf(top, p[i].top);
            top = wave_max(top);
            // (a piece of -inf only has sum 0, or NaN)
            const auto part = [&](const BeamPiece& x) {
                return x.sum == 0.0 ? 0.0 : x.sum * exp((double)x.top - (double)top);
            };
            double sum = lane < n_pieces ? part(mine) : 0.0;
            for (int i = lane + 64; i < n_pieces; i += 64) sum += part(p[i]);
            z = (double)top + log(wave_sum64(sum));
            if (!(fabs(z) < __builtin_inf())) z = __builtin_nan("");
        }
        if (lane == 0) {
            less[r] = z;
            given[r] = score;
        }
    }
    __syncthreads();
    const auto candidate = [&](uint32_t e, uint64_t key) {
        const int r = (int)(e / per_row);
        const double z = less[r];
        if (z != z || !key) return kBeamNobody;
        return BeamCand{given[r] + ((double)beam_logit((uint32_t)(key >> 32)) - z), key, r};
    };
    const auto each = [&](auto f) {
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
            const uint32_t e = tid + j * kBeamThreads;
            if (e < all) f(candidate(e, held[j]));
        }
        for (uint32_t e = tid + HELD * kBeamThreads; e < all; e += kBeamThreads) f(candidate(e, from[e]));
    };
    uint64_t best = 0;
    each([&](const BeamCand& c) {
        const uint64_t order = c.score > kBeamNone ? beam_order(c.score) : 0;
        best = order > best ? order : best;
    });
    const uint64_t nth = wave_bound(best, wave_most(best), n_out);
    if (lane == 0) bound[wave] = nth;
    __syncthreads();
    uint64_t least = 1;
#pragma unroll
    for (int w = 0; w < W; ++w) least = bound[w] > least ? bound[w] : least;
    each([&](const BeamCand& c) {
        if (c.score > kBeamNone && beam_order(c.score) >= least) {
            const int at = atomicAdd(&count, 1);
            if (at < kBeamList) {
                list_score[at] = c.score;
                list_key[at] = c.key;
                list_beam[at] = c.beam;
            }
        }
    });
    __syncthreads();
    int n = count;
    if (n > kBeamList) {
        BeamCand last = kBeamNobody;
        for (n = 0; n < n_out; ++n) {
            BeamCand b = kBeamNobody;
            each([&](const BeamCand& c) {
                if (beam_before(c, b) && (n == 0 || beam_before(last, c))) b = c;
            });
            b = wave_first(b);
            __syncthreads();
            if (lane == 0) first[wave] = b;
            __syncthreads();
            last = first[0];
            for (int w = 1; w < W; ++w)
                if (beam_before(first[w], last)) last = first[w];
            if (tid == 0) {
                list_score[n] = last.score;
                list_key[n] = last.key;
                list_beam[n] = last.beam;
            }
        }
        __syncthreads();
    }
    const long to = (long)group * n_out;
    const auto store = [&](int rank, const BeamCand& c) {
        const bool some = c.score > kBeamNone;
        tokens[to + rank] = some ? ~(uint32_t)c.key : 0u;
        parents[to + rank] = some ? c.beam : -1;
        out_scores[to + rank] = some ? c.score : kBeamNone;
    };
    for (int e = tid; e < n; e += kBeamThreads) {
        const BeamCand c = {list_score[e], list_key[e], list_beam[e]};
        int rank = 0, same = 0;
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
            const double s = list_score[i];
            rank += s > c.score;
            same += s == c.score;
        }
        if (same > 1)
            for (int i = 0; i < n; ++i)
                rank += list_score[i] == c.score && beam_before({list_score[i], list_key[i], list_beam[i]}, c);
        if (rank < n_out) store(rank, c);
    }
    for (int e = n + tid; e < n_out; e += kBeamThreads) store(e, kBeamNobody);
}

// Logits of a thread: what a block does once (bounds, ranks) is as much work as eight
// exponentials of a thread, and what a piece leaves is the join's work; few blocks leave
// CUs idle.  8, 16 and 32 of them: 4 beams over 49152 tokens 11.1, 12.0 and 13.6 us; 8 over
// 100278 18.7, 17.1, 18.2; 4 x 8 of them 23.3, 19.4, 20.2; 8 x 8 29.8, 25.2, 23.8.
static int beam_per(int vocab, long rows) {
    const long all = (long)vocab * rows, chip = (long)device_cu_count() * kBeamThreads;
    return all >= 32 * chip ? 32 : all >= 4 * chip ? 16 : 8;
}

// (a row may start up to three logits into its first vector)
static long beam_pieces(int vocab, int per) { return (vocab + 3L + per * kBeamThreads - 1) / (per * kBeamThreads); }

size_t beam_select_workspace(int vocab, int n_groups, int width, int n_out) {
    const long rows = (long)n_groups * width;
    return rows * beam_pieces(vocab, beam_per(vocab, rows)) * (sizeof(BeamPiece) + (size_t)n_out * sizeof(uint64_t));
}

int beam_select_launch(const float* logits, long ld, int vocab, const double* scores, int n_groups, int width, int n_out,
                       uint32_t* tokens, int* parents, double* out_scores, const Workspace& ws, hipStream_t st) {
    const char* who = "beam_select";
    ATLAS_REQUIRE(vocab > 0 && vocab <= 1 << 30 && ld >= vocab, "%s: rows of %d logits, %ld apart", who, vocab, ld);
    ATLAS_REQUIRE(width >= 1 && width <= 64 && n_out >= 1 && n_out <= kBeamMaxOut, "%s: %d beams, %d continuations (1 to 64)", who,
                  width, n_out);
    ATLAS_REQUIRE(n_groups >= 0 && (long)n_groups * width <= 65535, "%s: %d groups of %d beams (65535 beams at most)", who,
                  n_groups, width);
    if (n_groups == 0) return ATLAS_OK;
    ATLAS_REQUIRE(logits && scores && tokens && parents && out_scores, "%s: null argument", who);
    ATLAS_REQUIRE((((uintptr_t)logits | (uintptr_t)tokens | (uintptr_t)parents) & 3) == 0 &&
                      (((uintptr_t)scores | (uintptr_t)out_scores) & 7) == 0, "%s: misaligned argument", who);
    // a group's results are written while others' scores are read
    const long n_best = (long)n_groups * n_out;
    const ByteRows given(scores, (long)n_groups * width * 8), best(out_scores, n_best * 8), toks(tokens, n_best * 4),
        beams(parents, n_best * 4);
    ATLAS_REQUIRE(rows_apart(given, best) && rows_apart(given, toks) && rows_apart(given, beams), "%s: a result overlaps scores", who);
    ATLAS_REQUIRE(rows_apart(toks, beams) && rows_apart(toks, best) && rows_apart(beams, best), "%s: results overlap each other", who);
    const size_t bytes = beam_select_workspace(vocab, n_groups, width, n_out);
    void* p = ws.p;
    if (p) {
        ATLAS_REQUIRE(ws.bytes >= bytes, "%s: workspace of %zu bytes, %zu needed", who, ws.bytes, bytes);
    } else {
        const int rc = thread_scratch(SCR_BEAM, bytes, &p);
        if (rc) return rc;
    }
    const int per = beam_per(vocab, (long)n_groups * width), n_pieces = (int)beam_pieces(vocab, per);
    BeamPiece* pieces = static_cast<BeamPiece*>(p);
    uint64_t* keys = reinterpret_cast<uint64_t*>(pieces + (size_t)n_groups * width * n_pieces);
#define BEAM_ROWS(PER) \
    hipLaunchKernelGGL(beam_rows_kernel<PER>, dim3(n_pieces, n_groups * width), dim3(kBeamThreads), 0, st, logits, ld, vocab, \
                       scores, n_out, pieces, keys)
    if (per == 32) BEAM_ROWS(32);
    else if (per == 16) BEAM_ROWS(16);
    else BEAM_ROWS(8);
#undef BEAM_ROWS
    ATLAS_LAUNCH_CHECK("beam_rows");
    hipLaunchKernelGGL(beam_join_kernel, dim3(n_groups), dim3(kBeamThreads), 0, st, scores, vocab, width, n_out, n_pieces, pieces,
                       keys, tokens, parents, out_scores);
    ATLAS_LAUNCH_CHECK("beam_join");
    return ATLAS_OK;
}

// ---- reordering -------------------------------------------------------------------
//
// A thread has columns of a group's rows: it reads what any of them takes over and then
// writes, so that a state is reordered in place.  Bound by the bytes: 60 caches of 6 beams
// of 777 x 3 x 64 f32 40 to 45 us, 215 MB, 42 at a copy's rate; as many bytes of 12 beams 45,
// of 32 and 64, whose rows leave a wave to a SIMD, 54.  A launch has up to 64 states and a
// thread up to four columns, W rows of each in registers, so that all its loads are under way
// at once (a column to a thread, and fewer states to a launch: 85 us).

constexpr int kBeamStates = 64;

struct BeamStates {
    char* dst[kBeamStates];
    const char* src[kBeamStates];
};

// a state's rows, read or written
struct BeamSpan {
    uintptr_t at;
    long phase;                        // in the stride
    bool write;
};

// No rows that are written meet others, which may lie between them: m states of the same rows.
// Of those whose spans hang together only neighbours within the stride are looked at, so
// that the time is a sort's.
static bool beam_apart(BeamSpan* all, long m, long span, long row_bytes, long stride) {
    const auto same = [](const BeamSpan& a, const BeamSpan& b) { return a.at == b.at && !a.write && !b.write; };
    std::sort(all, all + m, [](const BeamSpan& a, const BeamSpan& b) { return a.at != b.at ? a.at < b.at : a.write > b.write; });
    m = std::unique(all, all + m, same) - all;           // (many may read one)
    for (long lo = 0, hi; lo < m; lo = hi) {
        for (hi = lo + 1; hi < m && all[hi].at - all[hi - 1].at < (uintptr_t)span;) ++hi;
        BeamSpan* const c = all + lo;
        const long n = hi - lo;
        std::sort(c, c + n, [](const BeamSpan& a, const BeamSpan& b) { return a.phase < b.phase; });
        for (long j = 0; j < n; ++j)
            for (long k = 1; k < n; ++k) {
                const BeamSpan& o = c[(j + k) % n];
                if (o.phase - c[j].phase + (j + k >= n ? stride : 0) >= row_bytes) break;
                const uintptr_t apart = o.at > c[j].at ? o.at - c[j].at : c[j].at - o.at;
                if ((o.write || c[j].write) && apart < (uintptr_t)span) return false;
            }
    }
    return true;
}

// One column to a thread in each of U places `apart` columns from each other, as far as
// there are `columns`; parents are the same in every lane.
template <typename T, int W, int U>
__device__ __forceinline__ void beam_move(char* dst, const char* src, long column, long columns, long apart, long stride,
                                          const int* parents, int width) {
    const bool in_place = dst == src;
    T v[U][W];
    int parent[W];
#pragma unroll
    for (int b = 0; b < W; ++b) {
        const int p = parents[min(b, width - 1)];
        parent[b] = b < width && (unsigned)p < (unsigned)width && !(in_place && p == b) ? p : -1;
    }
#pragma unroll
    for (int b = 0; b < W; ++b)
        if (parent[b] >= 0)
#pragma unroll
            for (int u = 0; u < U; ++u)
                v[u][b] = reinterpret_cast<const T*>(src + parent[b] * stride)[min(column + u * apart, columns - 1)];
#pragma unroll
    for (int b = 0; b < W; ++b)
        if (parent[b] >= 0)
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (column + u * apart < columns) reinterpret_cast<T*>(dst + b * stride)[column + u * apart] = v[u][b];
}

// full: units of T in a row; the bytes after them follow one by one, in the last block
template <typename T, int W, int U>
__global__ __launch_bounds__(256) void beam_reorder_kernel(BeamStates s, long full, int tail, long stride,
                                                           const int* __restrict__ parents, int width) {
    const long base = (long)blockIdx.y * width * stride;
    char* const dst = s.dst[blockIdx.z] + base;
    const char* const src = s.src[blockIdx.z] + base;
    parents += blockIdx.y * width;
    const long first = (long)blockIdx.x * (256 * U);
    if (first < full) {
        beam_move<T, W, U>(dst, src, first + threadIdx.x, full, 256, stride, parents, width);
    } else if (threadIdx.x < tail) {
        beam_move<char, W, 1>(dst + full * sizeof(T), src + full * sizeof(T), threadIdx.x, tail, 0, stride, parents, width);
    }
}

int beam_reorder_launch(void* const* dst, const void* const* src, int n_states, long row_bytes, long row_stride,
                        const int* parents, int n_groups, int width, hipStream_t st) {
    const char* who = "beam_reorder";
    ATLAS_REQUIRE(n_states >= 0 && row_bytes >= 0 && row_stride >= row_bytes, "%s: %d states, rows of %ld bytes %ld apart", who,
                  n_states, row_bytes, row_stride);
    ATLAS_REQUIRE(width >= 1 && width <= 64 && n_groups >= 0 && n_groups <= 65535, "%s: %d groups of %d beams (65535 of 64 at most)",
                  who, n_groups, width);
    if (n_states == 0 || row_bytes == 0 || n_groups == 0) return ATLAS_OK;
    ATLAS_REQUIRE(dst && src && parents, "%s: null argument", who);
    ATLAS_REQUIRE(((uintptr_t)parents & 3) == 0, "%s: misaligned parents", who);
    ATLAS_REQUIRE(row_stride < 1L << 40, "%s: rows %ld bytes apart", who, row_stride);
    const long n_rows = (long)n_groups * width, span = (n_rows - 1) * row_stride + row_bytes;
    const ByteRows given(parents, n_rows * 4);
    uintptr_t bits = (uintptr_t)row_stride;
    for (int i = 0; i < n_states; ++i) {
        ATLAS_REQUIRE(dst[i] && src[i], "%s: null state %d", who, i);
        const char *d = static_cast<const char*>(dst[i]), *s = static_cast<const char*>(src[i]);
        ATLAS_REQUIRE(d == s || d + span <= s || s + span <= d, "%s: state %d overlaps its new place", who, i);
        ATLAS_REQUIRE(rows_apart(given, ByteRows(d, n_rows, row_bytes, row_stride)), "%s: state %d overlaps parents", who, i);
        bits |= (uintptr_t)d | (uintptr_t)s;
    }
    const int unit = (bits & 15) == 0 ? 16 : (bits & 3) == 0 ? 4 : 1;
    const long full = row_bytes / unit, per = 256L * (width <= 8 ? 4 : width <= 16 ? 2 : 1);
    const long blocks = (full + per - 1) / per + (row_bytes % unit != 0);
    ATLAS_REQUIRE(blocks < 1 << 24, "%s: rows of %ld bytes", who, row_bytes);
    // states are moved side by side: none may be written that another reads or writes
    {
        BeamSpan few[2 * kBeamStates];
        std::unique_ptr<BeamSpan[]> many;
        if (n_states > kBeamStates) {
            many.reset(new (std::nothrow) BeamSpan[2 * (size_t)n_states]);
            if (!many) {
                set_error(ATLAS_ENOMEM, "%s: no host memory for %d states", who, n_states);
                return ATLAS_ENOMEM;
            }
        }
        BeamSpan* const all = many ? many.get() : few;
        long m = 0;
        const auto add = [&](const void* p, bool write) { all[m++] = {(uintptr_t)p, (long)((uintptr_t)p % (uintptr_t)row_stride), write}; };
        for (int i = 0; i < n_states; ++i) {
            add(dst[i], true);
            if (src[i] != dst[i]) add(src[i], false);
        }
        ATLAS_REQUIRE(beam_apart(all, m, span, row_bytes, row_stride), "%s: states overlap", who);
    }
    for (int i = 0; i < n_states; i += kBeamStates) {
        BeamStates s{};
        const int n = std::min(kBeamStates, n_states - i);
        for (int j = 0; j < n; ++j) {
            s.dst[j] = static_cast<char*>(dst[i + j]);
            s.src[j] = static_cast<const char*>(src[i + j]);
        }
        const dim3 grid((unsigned)blocks, n_groups, n);
#define BEAM_RUN(T, W, U) \
    hipLaunchKernelGGL((beam_reorder_kernel<T, W, U>), grid, dim3(256), 0, st, s, full, (int)(row_bytes % unit), row_stride, parents, width)
#define BEAM_WIDTH(T) if (width <= 8) BEAM_RUN(T, 8, 4); else if (width <= 16) BEAM_RUN(T, 16, 2); else BEAM_RUN(T, 64, 1)
        if (unit == 16) { BEAM_WIDTH(u32x4); }
        else if (unit == 4) { BEAM_WIDTH(uint32_t); }
        else { BEAM_WIDTH(char); }
#undef BEAM_WIDTH
#undef BEAM_RUN
        ATLAS_LAUNCH_CHECK("beam_reorder");
    }
    return ATLAS_OK;
}

}  // namespace atlas
