// prefix.hip -- decode attention of rows that share their first tokens, over an f32
// cache of slots.
//
// The rows of a group (a prompt's beams, requests over one system prompt) see the
// same first tokens, which lie in one slot; their own follow, each in a slot that a
// table names.  A tile is up to 16 CT columns of (row, head of the KV head's group):
// the shared tokens are read once for all of them, and their products are matrix
// instructions.  A row's own tokens go through the same instructions, seen by its
// columns only.
//
// With scores in powers of two (s = q.k scale log2 e), a wave keeps for each column
//   m >= max s - 8,  l = sum 2^(s - m),  O = sum 2^(s - m) v
// over its chunks of 16 tokens; waves and then blocks are joined by their maxima.
// S = K Q^T and O^T += V^T P are f32 products of 16 x 16 x 4, in which a lane's scores are
// just what its next product's B operand wants: P stays in registers, K and V pass from
// memory to registers in whole 64-byte pieces and through no LDS.
//
// Bound by the cache's stream where a group has few columns: 8 beams of 32 heads of 128
// over 4001 shared tokens and up to 97 of each 32 us, 135 MB, 26 at a copy's rate; and
// by the f32 products where groups are wide (64 requests of 32 heads over 8 of 128, 8191 tokens
// and up to 1023 of each: 69 of 124 us; shared tokens alone go at 114 TFLOP/s of 155), with
// masks and exponentials between them that a SIMD's two waves do not quite cover.  Heads
// of 256 leave a wave to a SIMD: 8 rows of 16 heads over 8, 4001 shared tokens and up to 97
// of each, 27 to 29 us, 68 MB, 13 at a copy's rate; the first shape with a window of 1024
// tokens 17 us, 35 MB, 7 at that rate.  The smallest, 4 beams of 9 heads over 3 of 64, are a
// launch and the chain of its loads: 4.9 us.
#include <algorithm>
#include <type_traits>

#include "many.hpp"

namespace atlas {

constexpr float kPfFloor = -3.0e38f;   // running maximum of a column that has seen nothing
constexpr float kPfLazy = 8.0f;
constexpr float kPfLog2e = 1.4426950408889634f;
constexpr int kPfChunk = 16;           // tokens that a wave takes at a time
constexpr int kPfMaxSplits = 64;
// Chunks of a block, where a tile has several: a wave of eight then has one.  A chunk's
// chain of loads, products and exponentials is as long as what a block costs by itself.
// (4 beams of 9 heads over 700 tokens: 9.7 us, 10.6 with 16.)
constexpr int kPfLeast = 8;

// What a tile and KV head leave for the join.
struct PfUnit {
    int runs, cols, row0, pad;         // runs 0 and 1: nothing to join
};

// Waves of a block, and blocks of a CU by their registers.  (Head dimension 128, 8 beams of 32
// heads and 64 requests of 32 over 8: four waves 33.3 and 152 us, eight 32.4 and 124, twelve 35.7
// and, with what does not fit the registers in memory, 151.  256, four waves of 314
// registers and eight of 250: 4 rows over 300 tokens 15.2 and 16.1, 8 over 4001 28.7 and 35.1, 40
// of five groups 35.0 and 39.4; 64 rows of 32 heads over 8 149 and 144.)
constexpr int pf_waves(int hd) { return hd == 256 ? 4 : 8; }
constexpr int pf_at_once(int hd, int ct) { return hd * ct <= 64 ? 2 : 1; }

struct PfArgs {
    const float *k, *v;
    int n_slots, max_seq, n_kv;
    const int *starts, *prefix_slots, *prefix_lens, *lens, *slots;
    int slot_stride, n_groups, n_rows;
    const float* q;
    long ld_q;
    float* out;
    long ld_out;
    int group;                         // heads of a KV head
    int rows;                          // of a tile, at most
    int tiles;                         // of the batch, some of them empty
    float scale;
    int window;
    int splits, cols;                  // blocks of a tile and KV head at most; [tiles][n_kv][splits][cols] partial sums
    float *part_o, *part_ml;
    PfUnit* unit;                      // [tiles][n_kv]
};

// The group of the batch's tile u.  Tiles of group g begin at starts[g] / rows + g,
// which leaves each group as many as it needs, whatever the sizes.
__device__ __forceinline__ int pf_group(const PfArgs& a, int u) {
    int lo = 0, hi = a.n_groups;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.starts[mid] / a.rows + mid <= u) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <int HD, int CT>
struct PfShared {
    static constexpr int W = pf_waves(HD);
    union {
        f32x4 q[CT][HD / 16][64];      // [column tile][step of 16 elements][lane]
        float o[W][16][HD + 4]; // the waves' sums of a column tile
    };
    float m[W][16 * CT], l[W][16 * CT];

};

__device__ __forceinline__ bool pf_infinite(float x) { return (__float_as_uint(x) & 0x7F800000u) == 0x7F800000u; }

// all lanes' largest value, and the sum of the lanes up to this one (DPP: rows of 16, then
// the last lane of one row, and of two, to the next)
__device__ __forceinline__ int wave_max_int(int v) {
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x142, 0xA, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x143, 0xC, 0xF, false));
    return __builtin_amdgcn_readlane(v, 63);
}

__device__ __forceinline__ int wave_scan_int(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

// A tile's tokens: the shared ones that any of its rows sees, [first, last), then the
// rows' own ones one row after the other, each part in whole chunks.  Lane r has what
// concerns row r.
struct PfTokens {
    int n_rows, row0;
    int from, to;                      // the row sees tokens [from, to)
    int own_from, own_begin, own_end;  // its first own one that is seen; its places among the own ones
    int shared_len, shared_cell;       // the shared slot's first cell
    int first, last, own;
    int shared_chunks, chunks;
    int lo_all, hi_all;                // tokens [lo_all, hi_all) are seen by all rows

    __device__ __forceinline__ void set(const PfArgs& a, int group, int row0_, int n_rows_, int lane) {
        row0 = row0_;
        n_rows = n_rows_;
        const bool mine = lane < n_rows;
        const int r = row0 + (mine ? lane : 0), raw = a.lens[r];
        shared_len = __builtin_amdgcn_readfirstlane(max(a.prefix_lens[group], 0));
        const int shared_slot = __builtin_amdgcn_readfirstlane(a.prefix_slots[group]);
        const bool cells = a.n_slots > 0 && a.max_seq > 0, there = cells && shared_slot >= 0 && shared_slot < a.n_slots;
        const int own_cap = cells ? min(a.slot_stride ? a.slot_stride : a.max_seq, max(a.max_seq - shared_len, 0)) : 0;
        to = mine ? max(raw, 0) : 0;
        from = a.window > 0 && to > a.window ? to - a.window : 0;
        own_from = max(from - shared_len, 0);
        const int n = max(min(to - shared_len, own_cap) - own_from, 0);
        own_end = wave_scan_int(n);
        own_begin = own_end - n;
        own = __builtin_amdgcn_readlane(own_end, 63);
        const int hi = wave_max_int(to), lo = -wave_max_int(to > from ? -from : -0x7FFFFFFF);
        lo_all = wave_max_int(mine ? from : 0);
        hi_all = -wave_max_int(mine ? -to : -0x7FFFFFFF);
        last = there ? min(min(shared_len, a.max_seq), hi) : 0;
        first = min(lo, last);
        shared_cell = there ? shared_slot * a.max_seq : 0;
        shared_chunks = (last - first + kPfChunk - 1) / kPfChunk;
        chunks = shared_chunks + (own + kPfChunk - 1) / kPfChunk;
    }
};

// A chunk's tokens, token i in the lanes of i.
struct PfChunk {
    int row, t;                        // its row (-1: shared) and position (-1: not there)
    int slot, x;                       // of an own one: its slot, on its way, and place in the row
    int row_first, row_last;           // of the chunk
    bool own, live;
    bool plain;                        // every column sees every token

    // which tokens; the table's entries are asked for
    __device__ __forceinline__ void find(const PfArgs& a, const PfTokens& k, int chunk, int i) {
        own = chunk >= k.shared_chunks;
        plain = false;
        if (!own) {
            const int c0 = k.first + chunk * kPfChunk;
            t = c0 + i;
            live = t < k.last;
            row = -1;
            plain = c0 >= k.lo_all && c0 + kPfChunk <= min(k.hi_all, k.last);
        } else {
            const int e0 = (chunk - k.shared_chunks) * kPfChunk, e = e0 + i;
            row_first = __popcll(__ballot(k.own_end <= e0));
            row_last = __popcll(__ballot(k.own_end <= min(e0 + kPfChunk, k.own) - 1));
            row = row_first;
            for (int r = row_first; r < row_last; ++r) row += e >= __builtin_amdgcn_readlane(k.own_end, r) ? 1 : 0;
            live = e < k.own;
            const int begin = __shfl(k.own_begin, row, 64), from = __shfl(k.own_from, row, 64);   // (of every lane)
            x = live ? e - begin + from : 0;
            slot = a.slots[(long)(k.row0 + row) * max(a.slot_stride, 1) + (a.slot_stride ? x : 0)];
        }
    }
    // the token's cell; of one that is not there some cell that is
    __device__ __forceinline__ int cell(const PfArgs& a, const PfTokens& k) {
        int c;
        if (!own) {
            c = k.shared_cell + min(t, k.last - 1);
        } else {
            live = live & (slot >= 0) & (slot < a.n_slots);
            t = k.shared_len + x;
            c = live ? slot * a.max_seq + t : 0;
        }
        t = live ? t : -1;
        return c;
    }
};

template <int HD, int CT>
__global__ __launch_bounds__(pf_waves(HD) * 64, pf_at_once(HD, CT) * pf_waves(HD) / 4) void pf_attention_kernel(PfArgs a) {
    constexpr int S = HD / 16, H = HD / 64, W = pf_waves(HD);
    __shared__ PfShared<HD, CT> sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    // block -> (tile, KV head, split): consecutive blocks run on different XCDs; the
    // tiles of a KV head and split, which read the same tokens if their group is the
    // same, come one after the other on one
    const int xcd = blockIdx.x & 7, at = blockIdx.x >> 3, pair = at / a.tiles * 8 + xcd, u = at % a.tiles;
    if (pair >= a.n_kv * a.splits) return;
    const int split = pair / a.n_kv, kvh = pair - split * a.n_kv;
    int grp = 0, row0 = u * a.rows, end = a.n_rows;
    if (a.starts) {
        grp = __builtin_amdgcn_readfirstlane(pf_group(a, u));
        const int begin = min(max(a.starts[grp], 0), a.n_rows), skip = (u - (a.starts[grp] / a.rows + grp)) * a.rows;
        end = min(a.starts[grp + 1], a.n_rows);
        if (skip < 0 || skip >= end - begin) {
            if (split == 0 && threadIdx.x == 0 && a.splits > 1) a.unit[u * a.n_kv + kvh] = {0, 0, 0, 0};
            return;
        }
        row0 = begin + skip;
    }
    row0 = __builtin_amdgcn_readfirstlane(row0);
    const int n_rows = __builtin_amdgcn_readfirstlane(min(a.rows, end - row0)), cols = n_rows * a.group;
    // the query, scaled for exp2; columns past the last repeat it
    constexpr int ITEMS = CT * S * 64, PER = (ITEMS + W * 64 - 1) / (W * 64);
    f32x4 query[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = threadIdx.x + j * W * 64;
        if (e >= ITEMS) break;
        const int l = e & 63, s = e / 64 % S, c = min(e / (64 * S) * 16 + (l & 15), cols - 1), row = c / a.group;
        query[j] = *reinterpret_cast<const f32x4*>(a.q + (row0 + row) * a.ld_q + ((long)kvh * a.group + c - row * a.group) * HD +
                                                   s * 16 + (l >> 4) * 4);
    }
    PfTokens tokens;
    tokens.set(a, grp, row0, n_rows, lane);
    // Every wave of the tile's blocks takes every so many chunks: shared tokens are more
    // work than own ones, and each has its share of both.
    const int runs = min(max((tokens.chunks + kPfLeast - 1) / kPfLeast, 1), a.splits);
    if (split >= runs) return;
    if (split == 0 && threadIdx.x == 0 && a.splits > 1) a.unit[u * a.n_kv + kvh] = {runs, cols, row0, 0};
    const int stride = runs * W;

    int col_row[CT], from[CT], to[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int col = 16 * c + i, row = col < cols ? col / a.group : 63;
        from[c] = __shfl(tokens.from, row, 64);
        to[c] = __shfl(tokens.to, row, 64);
        col_row[c] = col < cols ? row : -2;
    }
    f32x4 o[CT][H][4];
    float m[CT], l[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        m[c] = kPfFloor;
        l[c] = 0.f;
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[c][h][e] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    const long pitch = (long)a.n_kv * HD;            // (times a cell, both as 32 bits: one instruction)
    const float *const kb = a.k + (long)kvh * HD + 4 * g, *const vb = a.v + (long)kvh * HD + 4 * i;
    const int w0 = split * W + wave, n = w0 < tokens.chunks ? (tokens.chunks - w0 + stride - 1) / stride : 0;
    // (half of a SIMD's waves from the end, so that shared and own tokens, the ones bound by
    // products and the others by memory, are under way together)
    const bool back = wave >= W / 2 && (tokens.chunks - tokens.shared_chunks) * 4 > tokens.chunks;
    const auto chunk_of = [&](int t) { return w0 + (back ? n - 1 - t : t) * stride; };
    f32x4 kf[S], vf[4][H];
    PfChunk cur, next;
    int next_cell = 0;
    bool infinite = false;
    const auto fetch_k = [&](int c) {
        const float* p = kb + (uint64_t)(uint32_t)c * (uint32_t)pitch;
#pragma unroll
        for (int s = 0; s < S; ++s) kf[s] = *reinterpret_cast<const f32x4*>(p + 16 * s);
    };
    const auto fetch_v = [&](int r, int c) {             // of token 4g + r
        const float* p = vb + (uint64_t)(uint32_t)c * (uint32_t)pitch;
#pragma unroll
        for (int h = 0; h < H; ++h) vf[r][h] = *reinterpret_cast<const f32x4*>(p + 64 * h);
    };
    if (n > 0) {
        cur.find(a, tokens, chunk_of(0), i);
        next.find(a, tokens, chunk_of(min(1, n - 1)), i);
        const int cell = cur.cell(a, tokens);
        fetch_k(cell);
#pragma unroll
        for (int r = 0; r < 4; ++r) fetch_v(r, __shfl(cell, 4 * g + r, 64));
        next_cell = next.cell(a, tokens);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (threadIdx.x + j * W * 64 < ITEMS) sh.q[0][0][threadIdx.x + j * W * 64] = query[j] * (a.scale * kPfLog2e);
    __syncthreads();

    // Loads return in order, and what is copied from one step to the next is waited for: the
    // table's entry for the chunk after the next is asked for before the next one's K and V,
    // and used before its own are.
    const auto round = [&](int t, auto more) {
        PfChunk after;
        int after_cell = 0;
        if constexpr (decltype(more)::value) after.find(a, tokens, chunk_of(min(t + 2, n - 1)), i);
        // the column tiles that see any of the chunk
        const int c_first = cur.own ? cur.row_first * a.group >> 4 : 0;
        const int c_last = cur.own ? ((cur.row_last + 1) * a.group - 1) >> 4 : CT - 1;
        const auto needs = [&](int c) { return CT == 1 || (c >= c_first && c <= c_last); };
        // S: tokens 4g + r of column i
        // Each piece of K and V makes room for the next chunk's as soon as it is used.  (The
        // barriers keep the loads where they stand.)
        f32x4 d[CT][2] = {};
        const float* const next_k = kb + (uint64_t)(uint32_t)next_cell * (uint32_t)pitch;
        f32x4 qf[2][CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) qf[0][c] = sh.q[c][0][lane];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            if (s + 1 < S)
#pragma unroll
                for (int c = 0; c < CT; ++c) qf[(s + 1) & 1][c] = sh.q[c][s + 1][lane];
#pragma unroll
            for (int c = 0; c < CT; ++c)
                if (needs(c))
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        d[c][e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[s][e], qf[s & 1][c][e], d[c][e & 1], 0, 0, 0);
            if constexpr (decltype(more)::value) kf[s] = *reinterpret_cast<const f32x4*>(next_k + 16 * s);
            __builtin_amdgcn_sched_barrier(0);
        }
        float sc[CT][4];
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[c][r] = d[c][0][r] + d[c][1][r];
        if (!cur.plain) {
            // (without short circuits, which would be branches)
            int tok_row[4], tok[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                tok_row[r] = __shfl(cur.row, 4 * g + r, 64);
                tok[r] = __shfl(cur.t, 4 * g + r, 64);
            }
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t ok = (uint32_t)(tok[r] >= from[c]) & (uint32_t)(tok[r] < to[c]) &
                                        ((uint32_t)(tok_row[r] < 0) | (uint32_t)(tok_row[r] == col_row[c]));
                    sc[c][r] = ok ? sc[c][r] : -__builtin_inff();
                }
        }
        // weights; the maximum is raised only when a score passes it by more than 2^8
        f32x4 p[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            float top = fmaxf(fmaxf(sc[c][0], sc[c][1]), fmaxf(sc[c][2], sc[c][3]));
            if (__any(top > m[c] + kPfLazy)) {
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                const float up = fmaxf(m[c], top), down = __builtin_amdgcn_exp2f(m[c] - up);
                m[c] = up;
                l[c] *= down;
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[c][h][e] *= down;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[c][r] = __builtin_amdgcn_exp2f(sc[c][r] - m[c]);
                l[c] += p[c][r];
            }
        }
        if (!cur.plain) {
            // Infinities and NaN of V are nothing to the columns that do not see their
            // token: they leave the matrix product, and are seen to at the end.
            float none = 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) none = fmaf(vf[r][h][e], 0.f, none);
            if (__any(none != 0.f)) {
                infinite = true;
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int h = 0; h < H; ++h)
#pragma unroll
                        for (int e = 0; e < 4; ++e) vf[r][h][e] = pf_infinite(vf[r][h][e]) ? 0.f : vf[r][h][e];
            }
        }
        if constexpr (decltype(more)::value) after_cell = after.cell(a, tokens);
        // (where products are the bound, a SIMD's two waves are kept from going through the same
        // parts of a chunk together: 64 requests 123.8 us, 125.9 without; 8 beams 32.9, 32.4)
        if constexpr (CT == 2) __builtin_amdgcn_s_setprio(1);
        // O^T += V^T P: elements 64 h + 4 (4g + r) + e of column i
        int v_cell[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v_cell[r] = __shfl(next_cell, 4 * g + r, 64);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
            for (int c = 0; c < CT; ++c)
                if (needs(c))
#pragma unroll
                    for (int h = 0; h < H; ++h)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            o[c][h][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[r][h][e], p[c][r], o[c][h][e], 0, 0, 0);
            if constexpr (decltype(more)::value) fetch_v(r, v_cell[r]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (CT == 2) __builtin_amdgcn_s_setprio(0);
        if constexpr (decltype(more)::value) {
            cur = next;
            next = after;
            next_cell = after_cell;
        }
    };
    int t = 0;
#pragma unroll 1
    for (; t + 1 < n; ++t) round(t, std::true_type{});
    if (t < n) round(t, std::false_type{});
    // (Rare: the tokens are gone through again.)
    if (infinite) {
#pragma unroll 1
        for (t = 0; t < n; ++t) {
            cur.find(a, tokens, chunk_of(t), i);
            const int cell = cur.cell(a, tokens);
            if (cur.plain) continue;
#pragma unroll 1
            for (int j = 0; j < kPfChunk; ++j) {
                const int tok = __builtin_amdgcn_readlane(cur.t, j), row = __builtin_amdgcn_readlane(cur.row, j);
                if (tok < 0) continue;
                const float* p = vb - 4 * i + __builtin_amdgcn_readlane(cell, j) * pitch + 16 * g;
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const f32x4 y = *reinterpret_cast<const f32x4*>(p + 64 * h + 4 * x);
#pragma unroll
                        for (int c = 0; c < CT; ++c) {
                            const bool ok = (tok >= from[c]) & (tok < to[c]) & ((row < 0) | (row == col_row[c]));
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[c][h][e][x] += ok & pf_infinite(y[e]) ? y[e] : 0.f;
                        }
                    }
            }
        }
    }

    // ---- the waves' sums, a column tile at a time
    const auto store = [&](int c, int d, f32x4 x, float sum) {
        const int r = c / a.group;
        float* p = a.out + (row0 + r) * a.ld_out + ((long)kvh * a.group + c - r * a.group) * HD + d;
        *reinterpret_cast<f32x4*>(p) = x * (sum == 0.f ? 0.f : 1.f / sum);   // a row that has seen nothing is zero
    };
    const long part = (((long)u * a.n_kv + kvh) * a.splits) * a.cols;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        l[c] += __shfl_xor(l[c], 16, 64);
        l[c] += __shfl_xor(l[c], 32, 64);
        if (g == 0) {
            sh.m[wave][16 * c + i] = m[c];
            sh.l[wave][16 * c + i] = l[c];
        }
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        __syncthreads();
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                *reinterpret_cast<f32x4*>(&sh.o[wave][i][64 * h + 16 * g + 4 * x]) =
                    f32x4{o[ct][h][0][x], o[ct][h][1][x], o[ct][h][2][x], o[ct][h][3][x]};
        __syncthreads();
        const int here = min(max(cols - 16 * ct, 0), 16);
        for (int e = threadIdx.x; e < here * (HD / 4); e += W * 64) {
            const int c = e / (HD / 4), d = e % (HD / 4) * 4, col = 16 * ct + c;
            float top = kPfFloor, sum = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) top = fmaxf(top, sh.m[w][col]);
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float f = __builtin_amdgcn_exp2f(sh.m[w][col] - top);
                sum += f * sh.l[w][col];
                x += f * *reinterpret_cast<const f32x4*>(&sh.o[w][c][d]);
            }
            if (runs == 1) {
                store(col, d, x, sum);
            } else {
                const long at = part + (long)split * a.cols + col;
                *reinterpret_cast<f32x4*>(a.part_o + at * HD + d) = x;
                if (d == 0) {
                    a.part_ml[2 * at] = top;
                    a.part_ml[2 * at + 1] = sum;
                }
            }
        }
    }
}

// The runs' sums of a column: a wave, each of whose lanes has four elements of every so
// many runs.
template <int HD>
__global__ __launch_bounds__(256) void pf_join_kernel(PfArgs a) {
    constexpr int LANES = HD / 4, RG = 64 / LANES;
    const int lane = threadIdx.x & 63, unit = blockIdx.x, c = blockIdx.y * 4 + (threadIdx.x >> 6);
    const PfUnit x = a.unit[unit];
    if (x.runs <= 1 || c >= x.cols) return;
    const long part = (long)unit * a.splits * a.cols + c;
    float top = kPfFloor, sum = 0.f;
    if (lane < x.runs) {
        top = a.part_ml[2 * (part + (long)lane * a.cols)];
        sum = a.part_ml[2 * (part + (long)lane * a.cols) + 1];
    }
    const float f = __builtin_amdgcn_exp2f(top - wave_max(top));
    sum = wave_sum(lane < x.runs ? f * sum : 0.f);
    const int rg = lane / LANES, d = lane % LANES * 4;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    // eight loads at a time, without conditions (past the last run it again, for nothing)
    for (int r0 = 0; r0 < x.runs; r0 += 8 * RG) {
        f32x4 y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            y[j] = *reinterpret_cast<const f32x4*>(a.part_o + (part + (long)min(r0 + j * RG + rg, x.runs - 1) * a.cols) * HD + d);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = r0 + j * RG + rg;
            const float fr = __shfl(f, min(r, 63), 64);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += r < x.runs ? fr * y[j][e] : 0.f;   // (not 0 times an infinity)
        }
    }
#pragma unroll
    for (int s = LANES; s < 64; s <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], s, 64);
    if (rg) return;
    const int row = c / a.group, kvh = unit % a.n_kv;
    float* p = a.out + (x.row0 + row) * a.ld_out + ((long)kvh * a.group + c - row * a.group) * HD + d;
    *reinterpret_cast<f32x4*>(p) = o * (sum == 0.f ? 0.f : 1.f / sum);
}

// ---- launches ---------------------------------------------------------------------

// The shape of a launch: tile, splits, scratch.
struct PfShape {
    int ct, rows, tiles, splits, cols;
    size_t parts() const { return (size_t)tiles * splits * cols; }
};

static PfShape pf_shape(const atlas_slot_cache& c, const atlas_prefix_batch& b, int n_heads, int window) {
    PfShape s{};
    const int group = n_heads / c.n_kv;
    // the caller's hints
    int64_t prefix = std::min(b.max_prefix > 0 ? b.max_prefix : c.max_seq, c.max_seq);
    int64_t own = std::min(b.max_own > 0 ? b.max_own : c.max_seq, c.max_seq);
    if (b.slot_stride > 0) own = std::min<int64_t>(own, b.slot_stride);
    if (window > 0) {
        prefix = std::min<int64_t>(prefix, window);
        own = std::min<int64_t>(own, window);
    }
    // A second tile of columns halves the loads of K and V and the masks and exponentials' share,
    // where an average group is wide and its prefix long, and halves the blocks elsewhere.  With one
    // tile and two, 8 KV heads of 128: 64 columns over 8191 tokens 35.0 and 34.3 us, 96 columns 49.6
    // and 46.8, 128 columns 61.5 and 54.6, 256 columns over 4095 66.6 and 60.9; 128 columns over
    // 2047 28.0 and 28.3, eight such groups 120 and 141; 512 columns over 511 48 and 53.  Heads
    // of 64, 256 columns over 4095 tokens: 36.0 and 37.8; of 256 have no registers for it.
    const long wide = (long)b.n_rows * group / std::max(b.n_groups, 1);
    s.ct = c.head_dim == 128 && wide > 64 && prefix > 2048 ? 2 : 1;
    s.rows = 16 * s.ct / group;
    s.cols = s.rows * group;
    s.tiles = b.group_starts ? b.n_rows / s.rows + b.n_groups : (b.n_rows + s.rows - 1) / s.rows;
    if (b.n_groups == 1) s.tiles = (b.n_rows + s.rows - 1) / s.rows;
    // chunks of a tile
    const int64_t chunks = (prefix + kPfChunk - 1) / kPfChunk + (own * s.rows + kPfChunk - 1) / kPfChunk;
    // A block to every place of the chip; four to a tile where groups of different lengths
    // would leave a part of the places empty (16 groups of 1 to 15 rows of 16 heads over 4 of
    // 128, 700 shared and up to 700 own tokens: 58 us, 96 with one).
    const long units = std::max(1L, (long)s.tiles * c.n_kv), chip = (long)device_cu_count() * pf_at_once(c.head_dim, s.ct);
    const long want = chip / units < 2 && units < 2 * chip && b.n_groups > 1 ? 4 : chip / units;
    const long most = chunks <= 2 * kPfLeast ? 1 : (chunks + kPfLeast - 1) / kPfLeast;
    const long fit = (long)((256u << 20) / ((size_t)units * s.cols * (c.head_dim + 2) * sizeof(float)));
    s.splits = (int)std::max(1L, std::min({want, most, fit, (long)kPfMaxSplits}));
    return s;
}

static size_t pf_bytes(const PfShape& s, const atlas_slot_cache& c) {
    return s.splits > 1 ? s.parts() * c.n_kv * (c.head_dim + 2) * sizeof(float) + (size_t)s.tiles * c.n_kv * sizeof(PfUnit) : 0;
}

size_t prefix_attention_workspace(const atlas_slot_cache& c, const atlas_prefix_batch& b, int n_heads, int window) {
    return pf_bytes(pf_shape(c, b, n_heads, window), c);
}

int prefix_attention_launch(const atlas_slot_cache& c, const atlas_prefix_batch& b, const float* q, long ld_q, int n_heads,
                            float scale, int window, float* out, long ld_out, const Workspace& ws, hipStream_t st) {
    const char* who = "prefix_attention";
    ATLAS_REQUIRE(c.head_dim == 64 || c.head_dim == 128 || c.head_dim == 256, "%s: head_dim %d (64, 128 or 256)", who,
                  c.head_dim);
    ATLAS_REQUIRE(c.n_slots >= 0 && c.max_seq >= 0 && c.max_seq <= 1 << 24 && c.n_kv > 0 && c.n_kv <= 4096, "%s: %d slots of %d tokens, %d KV heads",
                  who, c.n_slots, c.max_seq, c.n_kv);
    ATLAS_REQUIRE((long)c.n_slots * c.max_seq < 1L << 31, "%s: %d slots of %d tokens", who, c.n_slots, c.max_seq);
    ATLAS_REQUIRE(b.n_groups >= 0 && b.n_rows >= 0 && b.slot_stride >= 0 && b.max_prefix >= 0 && b.max_own >= 0,
                  "%s: %d groups, %d rows, slot stride %d, max_prefix %d, max_own %d", who, b.n_groups, b.n_rows,
                  b.slot_stride, b.max_prefix, b.max_own);
    ATLAS_REQUIRE(b.group_starts || b.n_groups <= 1, "%s: %d groups need group_starts", who, b.n_groups);
    ATLAS_REQUIRE(b.n_groups <= 1 << 20 && b.n_rows <= 1 << 20, "%s: %d rows of %d groups", who, b.n_rows, b.n_groups);
    ATLAS_REQUIRE(n_heads > 0 && n_heads % c.n_kv == 0 && n_heads / c.n_kv <= 16, "%s: %d heads over %d KV heads (up to 16 to each)",
                  who, n_heads, c.n_kv);
    ATLAS_REQUIRE(window >= 0, "%s: window %d", who, window);
    if (b.n_rows == 0 || b.n_groups == 0) return ATLAS_OK;
    ATLAS_REQUIRE(b.prefix_slots && b.prefix_lens && b.kv_lens && b.slots && ((long)c.n_slots * c.max_seq == 0 || (c.k && c.v)) && q && out,
                  "%s: null argument", who);
    ATLAS_REQUIRE((((uintptr_t)b.group_starts | (uintptr_t)b.prefix_slots | (uintptr_t)b.prefix_lens | (uintptr_t)b.kv_lens |
                    (uintptr_t)b.slots) & 3) == 0, "%s: misaligned batch", who);
    const long wide = (long)n_heads * c.head_dim;
    ATLAS_REQUIRE((((uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)q | (uintptr_t)out) & 15) == 0 && ld_q % 4 == 0 &&
                      ld_out % 4 == 0 && ld_q >= wide && ld_out >= wide,
                  "%s: the cache and rows start on 16 bytes, rows at least %ld elements apart (strides %ld and %ld)", who, wide,
                  ld_q, ld_out);
    // a block writes its rows while others read
    const ByteRows to(out, b.n_rows, wide * 4, ld_out * 4);
    const long cells = (long)c.n_slots * c.max_seq * c.n_kv * c.head_dim * 4, ints = sizeof(int);
    ATLAS_REQUIRE((out == q && (ld_out == ld_q || b.n_rows == 1)) || rows_apart(to, ByteRows(q, b.n_rows, wide * 4, ld_q * 4)),
                  "%s: out overlaps q", who);
    ATLAS_REQUIRE(rows_apart(ByteRows(c.k, cells), to) && rows_apart(ByteRows(c.v, cells), to), "%s: out overlaps the cache", who);
    ATLAS_REQUIRE((!b.group_starts || rows_apart(ByteRows(b.group_starts, (b.n_groups + 1) * ints), to)) &&
                      rows_apart(ByteRows(b.prefix_slots, b.n_groups * ints), to) &&
                      rows_apart(ByteRows(b.prefix_lens, b.n_groups * ints), to) && rows_apart(ByteRows(b.kv_lens, b.n_rows * ints), to) &&
                      rows_apart(ByteRows(b.slots, (long)b.n_rows * std::max(b.slot_stride, 1) * ints), to),
                  "%s: out overlaps the batch", who);
    const PfShape s = pf_shape(c, b, n_heads, window);
    const long units = (long)s.tiles * c.n_kv;
    const long blocks = ((long)c.n_kv * s.splits + 7) / 8 * 8 * s.tiles;
    ATLAS_REQUIRE(blocks < 1 << 23, "%s: %d tiles of rows and %d KV heads", who, s.tiles, c.n_kv);   // 2^32 threads
    PfArgs a{};
    a.k = c.k; a.v = c.v;
    a.n_slots = c.n_slots; a.max_seq = c.max_seq; a.n_kv = c.n_kv;
    a.starts = b.group_starts;
    a.prefix_slots = b.prefix_slots; a.prefix_lens = b.prefix_lens; a.lens = b.kv_lens; a.slots = b.slots;
    a.slot_stride = b.slot_stride; a.n_groups = b.n_groups; a.n_rows = b.n_rows;
    a.q = q; a.ld_q = ld_q; a.out = out; a.ld_out = ld_out;
    a.group = n_heads / c.n_kv;
    a.rows = s.rows; a.tiles = s.tiles; a.cols = s.cols; a.splits = s.splits;
    a.scale = scale; a.window = window;
    if (s.splits > 1) {
        const size_t bytes = pf_bytes(s, c);
        void* p = ws.p;
        if (p) {
            ATLAS_REQUIRE(ws.bytes >= bytes, "%s: workspace of %zu bytes, %zu needed", who, ws.bytes, bytes);
        } else {
            const int rc = thread_scratch(SCR_PREFIX, bytes, &p);
            if (rc) return rc;
        }
        a.unit = static_cast<PfUnit*>(p);
        a.part_o = reinterpret_cast<float*>(a.unit + units);
        a.part_ml = a.part_o + s.parts() * c.n_kv * c.head_dim;
    }
    const dim3 grid((unsigned)blocks);
#define PF_RUN(HD, CT) hipLaunchKernelGGL((pf_attention_kernel<HD, CT>), grid, dim3(pf_waves(HD) * 64), 0, st, a)
    if (c.head_dim == 64) PF_RUN(64, 1);
    else if (c.head_dim == 128 && s.ct == 1) PF_RUN(128, 1);
    else if (c.head_dim == 128) PF_RUN(128, 2);
    else PF_RUN(256, 1);
#undef PF_RUN
    ATLAS_LAUNCH_CHECK("prefix_attention");
    if (s.splits > 1) {
        const dim3 join((unsigned)units, (s.cols + 3) / 4);
        if (c.head_dim == 64) hipLaunchKernelGGL(pf_join_kernel<64>, join, dim3(256), 0, st, a);
        else if (c.head_dim == 128) hipLaunchKernelGGL(pf_join_kernel<128>, join, dim3(256), 0, st, a);
        else hipLaunchKernelGGL(pf_join_kernel<256>, join, dim3(256), 0, st, a);
        ATLAS_LAUNCH_CHECK("prefix_join");
    }
    return ATLAS_OK;
}

}  // namespace atlas
