// beam.hip -- beam search: the choice of a group's best continuations over its beams
// and the vocabulary, and the reordering of the beams' states.
#include <algorithm>

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
// the few that are left are ranked by counting.

constexpr int kBeamMaxOut = 64;
constexpr int kBeamPer = 16, kBeamThreads = 256, kBeamPiece = kBeamPer * kBeamThreads;

// order-preserving: larger logits have larger keys; 0 for what is no candidate
__device__ __forceinline__ uint32_t beam_order(float z) {
    const uint32_t u = __float_as_uint(z);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float beam_logit(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// larger first; of equal logits the lower token
__device__ __forceinline__ uint64_t beam_key(float z, uint32_t token) {
    return z > -__builtin_inff() ? (uint64_t)beam_order(z + 0.f) << 32 | (uint32_t)~token : 0;   // (-0 is 0)
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int mask) {
    const uint32_t lo = __shfl_xor((int)(uint32_t)v, mask, 64), hi = __shfl_xor((int)(uint32_t)(v >> 32), mask, 64);
    return (uint64_t)hi << 32 | lo;
}

// the wave's values in descending order of the lanes
__device__ __forceinline__ uint64_t wave_sort(uint64_t v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
        for (int step = size >> 1; step > 0; step >>= 1) {
            const uint64_t w = shfl_xor64(v, step);
            const bool large = ((lane & size) == 0) == ((lane & step) == 0);   // the lane keeps the larger
            v = (v > w) == large ? v : w;
        }
    return v;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// what a piece of a row leaves
struct BeamPiece {
    double sum;                        // of exp(z - top); NaN: the row has a NaN or +inf
    float top;
    int pad;
};

__device__ __forceinline__ bool beam_dead(double score) { return !(fabs(score) < __builtin_inf()); }

__global__ __launch_bounds__(kBeamThreads) void beam_rows_kernel(const float* __restrict__ logits, long ld, int vocab,
                                                                 const double* __restrict__ scores, int n_out, int vec,
                                                                 BeamPiece* __restrict__ pieces, uint64_t* __restrict__ keys) {
    constexpr int W = kBeamThreads / 64;
    __shared__ uint64_t list[kBeamPiece];
    __shared__ uint64_t bound[W];
    __shared__ float tops[W];
    __shared__ double sums[W];
    __shared__ int count;
    const int row = blockIdx.y, piece = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (beam_dead(scores[row])) return;                  // (the join does not look at its rows' pieces either)
    const float* z = logits + (long)row * ld;
    const int first = piece * kBeamPiece;
    float x[kBeamPer];
#pragma unroll
    for (int j = 0; j < kBeamPer / 4; ++j) {
        const int e = first + (j * kBeamThreads + tid) * 4;
        if (vec && e + 4 <= vocab) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(z + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[4 * j + i] = v[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[4 * j + i] = e + i < vocab ? z[e + i] : -__builtin_inff();
        }
    }
    if (tid == 0) count = 0;
    float top = -__builtin_inff();
    bool nan = false;
    uint64_t best = 0;
#pragma unroll
    for (int j = 0; j < kBeamPer; ++j) {
        top = fmaxf(top, x[j]);
        nan = nan || x[j] != x[j];
        const uint64_t key = beam_key(x[j], first + (j / 4 * kBeamThreads + tid) * 4 + j % 4);
        best = key > best ? key : best;
    }
    top = wave_max(top);
    const uint64_t sorted = wave_sort(best);
    if (lane == n_out - 1) bound[wave] = sorted;
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    uint64_t least = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        top = fmaxf(top, tops[w]);
        least = bound[w] > least ? bound[w] : least;
    }
    double sum = nan ? __builtin_nan("") : 0.0;
    if (top > -__builtin_inff())
#pragma unroll
        for (int j = 0; j < kBeamPer; ++j) sum += exp((double)x[j] - (double)top);
    sum = wave_sum64(sum);
    if (lane == 0) sums[wave] = sum;
#pragma unroll
    for (int j = 0; j < kBeamPer; ++j) {
        const uint64_t key = beam_key(x[j], first + (j / 4 * kBeamThreads + tid) * 4 + j % 4);
        if (key && key >= least) list[atomicAdd(&count, 1)] = key;
    }
    __syncthreads();
    const long at = (long)row * gridDim.x + piece;
    if (tid == 0) {
        double all = 0.0;
#pragma unroll
        for (int w = 0; w < W; ++w) all += sums[w];
        pieces[at] = {all, top, 0};
    }
    const int n = count;
    uint64_t* to = keys + at * n_out;
    for (int e = tid; e < n; e += kBeamThreads) {
        const uint64_t key = list[e];
        int rank = 0;
        for (int i = 0; i < n; ++i) rank += list[i] > key;
        if (rank < n_out) to[rank] = key;
    }
    for (int e = n + tid; e < n_out; e += kBeamThreads) to[e] = 0;
}

constexpr int kBeamJoin = 1024, kBeamList = 2048;

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

__device__ __forceinline__ BeamCand wave_sort(BeamCand v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
        for (int step = size >> 1; step > 0; step >>= 1) {
            const BeamCand w = {__shfl_xor(v.score, step, 64), shfl_xor64(v.key, step), __shfl_xor(v.beam, step, 64)};
            const bool first = ((lane & size) == 0) == ((lane & step) == 0);
            if (beam_before(w, v) == first) v = w;
        }
    return v;
}

__global__ __launch_bounds__(kBeamJoin) void beam_join_kernel(const double* __restrict__ scores, int vocab, int width,
                                                              int n_out, int n_pieces, const BeamPiece* __restrict__ pieces,
                                                              const uint64_t* __restrict__ keys, uint32_t* __restrict__ tokens,
                                                              int* __restrict__ parents, double* __restrict__ out_scores) {
    constexpr int W = kBeamJoin / 64;
    __shared__ double lse[64];                           // NaN: the row has no candidates
    __shared__ BeamCand bound[W];
    __shared__ BeamCand list[kBeamList];
    __shared__ int count;
    const int group = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    scores += (long)group * width;
    const long row0 = (long)group * width;
    if (tid == 0) count = 0;
    for (int r = wave; r < width; r += W) {
        double z = __builtin_nan("");
        if (!beam_dead(scores[r])) {
            const BeamPiece* p = pieces + (row0 + r) * n_pieces;
            float top = -__builtin_inff();
            for (int i = lane; i < n_pieces; i += 64) top = fmaxf(top, p[i].top);
            top = wave_max(top);
            double sum = 0.0;
            for (int i = lane; i < n_pieces; i += 64) {
                const double s = p[i].sum;               // (a piece of -inf only has sum 0, or NaN)
                sum += s == 0.0 ? 0.0 : s * exp((double)p[i].top - (double)top);
            }
            sum = wave_sum64(sum);
            z = (double)top + log(sum);
        }
        if (lane == 0) lse[r] = z;
    }
    __syncthreads();
    const int per_row = n_pieces * n_out;
    const long all = (long)width * per_row;
    const auto candidate = [&](long e) {
        const int r = (int)(e / per_row);
        BeamCand c = kBeamNobody;
        const double z = lse[r];
        if (!(fabs(z) < __builtin_inf())) return c;
        const uint64_t key = keys[(row0 + r) * per_row + (e - (long)r * per_row)];
        if (!key) return c;
        c.score = scores[r] + ((double)beam_logit((uint32_t)(key >> 32)) - z);
        c.key = key;
        c.beam = r;
        return c;
    };
    BeamCand best = kBeamNobody;
    for (long e = tid; e < all; e += kBeamJoin) {
        const BeamCand c = candidate(e);
        if (beam_before(c, best)) best = c;
    }
    const BeamCand sorted = wave_sort(best);
    if (lane == n_out - 1) bound[wave] = sorted;
    __syncthreads();
    BeamCand least = bound[0];
    for (int w = 1; w < W; ++w)
        if (beam_before(bound[w], least)) least = bound[w];
    for (long e = tid; e < all; e += kBeamJoin) {
        const BeamCand c = candidate(e);
        if (c.score > kBeamNone && !beam_before(least, c)) {
            const int at = atomicAdd(&count, 1);
            if (at < kBeamList) list[at] = c;
        }
    }
    __syncthreads();
    int n = count;
    if (n > kBeamList) {
        // too many reach the bound: the largest one after the other
        BeamCand last = kBeamNobody;
        for (n = 0; n < n_out; ++n) {
            __syncthreads();
            best = kBeamNobody;
            for (long e = tid; e < all; e += kBeamJoin) {
                const BeamCand c = candidate(e);
                if (beam_before(c, best) && (n == 0 || beam_before(last, c))) best = c;
            }
            const BeamCand s = wave_sort(best);
            if (lane == 0) bound[wave] = s;
            __syncthreads();
            last = bound[0];
            for (int w = 1; w < W; ++w)
                if (beam_before(bound[w], last)) last = bound[w];
            if (tid == 0) list[n] = last;
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
    for (int e = tid; e < n; e += kBeamJoin) {
        const BeamCand c = list[e];
        int rank = 0;
        for (int i = 0; i < n; ++i) rank += beam_before(list[i], c);
        if (rank < n_out) store(rank, c);
    }
    for (int e = n + tid; e < n_out; e += kBeamJoin) store(e, kBeamNobody);
}

static long beam_pieces(int vocab) { return (vocab + kBeamPiece - 1) / kBeamPiece; }

size_t beam_select_workspace(int vocab, int n_groups, int width, int n_out) {
    return (size_t)n_groups * width * beam_pieces(vocab) * (sizeof(BeamPiece) + (size_t)n_out * sizeof(uint64_t));
}

int beam_select_launch(const float* logits, long ld, int vocab, const double* scores, int n_groups, int width, int n_out,
                       uint32_t* tokens, int* parents, double* out_scores, const Workspace& ws, hipStream_t st) {
    const char* who = "beam_select";
    ATLAS_REQUIRE(vocab > 0 && ld >= vocab, "%s: rows of %d logits, %ld apart", who, vocab, ld);
    ATLAS_REQUIRE(width >= 1 && width <= 64 && n_out >= 1 && n_out <= kBeamMaxOut, "%s: %d beams, %d continuations (1 to 64)", who,
                  width, n_out);
    ATLAS_REQUIRE(n_groups >= 0 && (long)n_groups * width <= 65535, "%s: %d groups of %d beams (65535 beams at most)", who,
                  n_groups, width);
    if (n_groups == 0) return ATLAS_OK;
    ATLAS_REQUIRE(logits && scores && tokens && parents && out_scores, "%s: null argument", who);
    ATLAS_REQUIRE((((uintptr_t)logits | (uintptr_t)tokens | (uintptr_t)parents) & 3) == 0 &&
                      (((uintptr_t)scores | (uintptr_t)out_scores) & 7) == 0, "%s: misaligned argument", who);
    const size_t bytes = beam_select_workspace(vocab, n_groups, width, n_out);
    void* p = ws.p;
    if (p) {
        ATLAS_REQUIRE(ws.bytes >= bytes, "%s: workspace of %zu bytes, %zu needed", who, ws.bytes, bytes);
    } else {
        const int rc = thread_scratch(SCR_BEAM, bytes, &p);
        if (rc) return rc;
    }
    const int n_pieces = (int)beam_pieces(vocab);
    BeamPiece* pieces = static_cast<BeamPiece*>(p);
    uint64_t* keys = reinterpret_cast<uint64_t*>(pieces + (size_t)n_groups * width * n_pieces);
    const int vec = ((uintptr_t)logits & 15) == 0 && ld % 4 == 0;
    hipLaunchKernelGGL(beam_rows_kernel, dim3(n_pieces, n_groups * width), dim3(kBeamThreads), 0, st, logits, ld, vocab, scores,
                       n_out, vec, pieces, keys);
    ATLAS_LAUNCH_CHECK("beam_rows");
    hipLaunchKernelGGL(beam_join_kernel, dim3(n_groups), dim3(kBeamJoin), 0, st, scores, vocab, width, n_out, n_pieces, pieces,
                       keys, tokens, parents, out_scores);
    ATLAS_LAUNCH_CHECK("beam_join");
    return ATLAS_OK;
}

// ---- reordering -------------------------------------------------------------------
//
// A thread has a column of a group's rows: it reads what any of them takes over and
// then writes, so that a state is reordered in place.

constexpr int kBeamStates = 32;

struct BeamStates {
    char* dst[kBeamStates];
    const char* src[kBeamStates];
};

template <typename T, int W>
__device__ __forceinline__ void beam_move(const BeamStates& s, int state, long at, long stride, const int* parent, int width) {
    char* const dst = s.dst[state] + at;
    const char* const src = s.src[state] + at;
    const bool in_place = dst == src;
    T v[W];
#pragma unroll
    for (int b = 0; b < W; ++b)
        if (b < width && parent[b] >= 0 && !(in_place && parent[b] == b)) v[b] = *reinterpret_cast<const T*>(src + parent[b] * stride);
#pragma unroll
    for (int b = 0; b < W; ++b)
        if (b < width && parent[b] >= 0 && !(in_place && parent[b] == b)) *reinterpret_cast<T*>(dst + b * stride) = v[b];
}

// full: units of T in a row; the bytes after them follow one by one
template <typename T, int W>
__global__ __launch_bounds__(256) void beam_reorder_kernel(BeamStates s, long full, int tail, long stride,
                                                           const int* __restrict__ parents, int width) {
    __shared__ int parent[W];
    const int group = blockIdx.y;
    if (threadIdx.x < width) {
        const int p = parents[group * width + threadIdx.x];
        parent[threadIdx.x] = p >= 0 && p < width ? p : -1;
    }
    __syncthreads();
    const long e = (long)blockIdx.x * 256 + threadIdx.x, base = (long)group * width * stride;
    if (e < full) beam_move<T, W>(s, blockIdx.z, base + e * sizeof(T), stride, parent, width);
    else if (e < full + tail) beam_move<char, W>(s, blockIdx.z, base + full * sizeof(T) + (e - full), stride, parent, width);
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
    const long span = (((long)n_groups * width) - 1) * row_stride + row_bytes;
    uintptr_t bits = (uintptr_t)row_stride;
    for (int i = 0; i < n_states; ++i) {
        ATLAS_REQUIRE(dst[i] && src[i], "%s: null state %d", who, i);
        const char *d = static_cast<const char*>(dst[i]), *s = static_cast<const char*>(src[i]);
        ATLAS_REQUIRE(d == s || d + span <= s || s + span <= d, "%s: state %d overlaps its new place", who, i);
        bits |= (uintptr_t)d | (uintptr_t)s;
    }
    const int unit = (bits & 15) == 0 ? 16 : (bits & 3) == 0 ? 4 : 1;
    const long full = row_bytes / unit, blocks = (full + row_bytes % unit + 255) / 256;
    ATLAS_REQUIRE(blocks <= 0x7FFFFFFF, "%s: rows of %ld bytes", who, row_bytes);
    for (int i = 0; i < n_states; i += kBeamStates) {
        BeamStates s{};
        const int n = std::min(kBeamStates, n_states - i);
        for (int j = 0; j < n; ++j) {
            s.dst[j] = static_cast<char*>(dst[i + j]);
            s.src[j] = static_cast<const char*>(src[i + j]);
        }
        const dim3 grid((unsigned)blocks, n_groups, n);
#define BEAM_RUN(T, W) \
    hipLaunchKernelGGL((beam_reorder_kernel<T, W>), grid, dim3(256), 0, st, s, full, (int)(row_bytes % unit), row_stride, parents, width)
#define BEAM_WIDTH(T) if (width <= 8) BEAM_RUN(T, 8); else if (width <= 16) BEAM_RUN(T, 16); else BEAM_RUN(T, 64)
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
