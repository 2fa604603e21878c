// kv4.hip -- the 4-bit KV cache: writing and reading tokens, and attention over it.
//
// K and V rows are MXFP4 along the head dimension (mxfp4.hpp), in pages of
// page_len tokens that a block table strings together for each sequence.  A page
// holds for each KV head, one after the other,
//   K codes   [page_len][hd/2 bytes]          a token's elements in order
//   K scales  [page_len/8][hd/32][8 tokens]
//   V codes   [page_len/8][16][8 tokens][hd/32 bytes]
//   V scales  [page_len/8][hd/32][8 tokens]
// V's elements are cut into 16 groups of hd/16, a group of eight tokens side by
// side, because the product P V contracts over tokens: a lane of the matrix
// instruction has eight tokens of the same elements, and so finds them in one
// piece.  A token still fills whole bytes, so that writing one touches no other.
#include <algorithm>
#include <type_traits>

#include "mfma.hpp"
#include "mxfp4.hpp"

namespace atlas {

// what the kernels take of a cache and a batch
struct Kv4Args {
    uint8_t* cache;
    int n_pages, n_kv, page_shift;      // page_len = 1 << page_shift
    const int* starts;                  // [n_seqs + 1] or null: one row to a sequence
    const int* lens;
    const int* table;
    int table_stride, n_seqs, n_rows;
    int cap;                            // tokens that the table can hold
};

template <int HD>
struct Kv4Layout {
    static constexpr int KB = HD / 32;                  // blocks of a token
    // offsets of the parts within a (page, head)'s bytes
    __device__ static long k_scales(int page_len) { return (long)page_len * (HD / 2); }
    __device__ static long v_codes(int page_len) { return (long)page_len * (HD / 2 + KB); }
    __device__ static long v_scales(int page_len) { return (long)page_len * (HD + KB); }
    __device__ static long bytes(int page_len) { return (long)page_len * (HD + 2 * KB); }
};

// Sequence and position of a batch's row; false: behind the last sequence.
// The starts are the caller's: whatever they hold, s stays within [0, n_seqs).
__device__ __forceinline__ bool kv4_row(const Kv4Args& a, int row, int& s, int& pos) {
    if (!a.starts) {
        s = row;
        pos = max(a.lens[row], 0) - 1;
        return row < a.n_seqs;
    }
    int lo = 0, hi = a.n_seqs;          // the last s with starts[s] <= row
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.starts[mid] <= row) lo = mid;
        else hi = mid;
    }
    s = lo;
    const int end = a.starts[lo + 1];
    pos = max(a.lens[lo], 0) - (end - row);
    return row < end && row >= a.starts[lo];
}

// the page of a position, or -1: outside the table, or an entry that is no page
__device__ __forceinline__ int kv4_page(const Kv4Args& a, int s, int pos) {
    if (pos < 0 || pos >= a.cap) return -1;
    const int page = a.table[(long)s * a.table_stride + (pos >> a.page_shift)];
    return page >= 0 && page < a.n_pages ? page : -1;
}

// ---- writing and reading ----------------------------------------------------------

// Both move bytes.  A wave has 64 elements of eight rows of K and of V, a lane eight
// of each: on the side of the rows lane = 8 row + eighth, so that a row gives 256
// bytes in one piece.  Eight tokens of V lie side by side in the cache; there
// lane = 8 eighth + row, 256 bytes in one piece again, and V's codes change lanes on
// the way.  Blocks of eight rows write whole lines where the positions of the tokens
// allow.  2047 tokens of 32 heads of 128, written (67 MB in, 9 out) and read: 41 us, where
// bytes at a large copy's rate are 29; 45 with a row to a block, whose lines are
// put together from several XCDs' caches.

// lane 8 i + j's value from lane 8 j + i
__device__ __forceinline__ int kv4_turn(int x) {
    const int lane = threadIdx.x & 63;
    return __builtin_amdgcn_ds_bpermute(((lane & 7) * 8 + (lane >> 3)) * 4, x);
}

// The lane's row and element on the side of the rows; where its eight elements' codes
// and scale bytes are in the cache, V's those of the lane that it turns to.
template <int HD>
struct Kv4Place {
    typedef Kv4Layout<HD> L;
    int row, e, page, v_page;                            // pages -1: none
    bool mine;                                           // a row of a sequence
    uint8_t *k, *k_scale, *v, *v_scale;
    bool k_first, v_first;                               // of a block of 32

    __device__ __forceinline__ Kv4Place() {
        const int lane = threadIdx.x & 63;
        row = blockIdx.x * 8 + (lane >> 3);
        e = blockIdx.y * 256 + (threadIdx.x >> 6) * 64 + (lane & 7) * 8;
    }
    __device__ __forceinline__ bool inside(const Kv4Args& a) const { return row < a.n_rows && e < a.n_kv * HD; }
    __device__ __forceinline__ void find(const Kv4Args& a) {
        int s = 0, pos = 0;
        mine = inside(a) && kv4_row(a, row, s, pos);
        page = mine ? kv4_page(a, s, pos) : -1;
        const int plen = 1 << a.page_shift, at = pos & (plen - 1);
        uint8_t* p = part(a, page, e) + at * (long)(HD / 2);
        k = p + e % HD / 2;
        k_scale = p - at * (long)(HD / 2) + L::k_scales(plen) + scale_at(at, e);
        k_first = e % 32 == 0;
        v_page = kv4_turn(page);
        const int v_at = kv4_turn(at), lane = threadIdx.x & 63, ve = e - (lane & 7) * 8 + (lane >> 3) * 8;
        p = part(a, v_page, ve);
        // group of HD / 16 elements, [token % 8][KB bytes]
        v = p + L::v_codes(plen) + (long)(v_at >> 3) * (HD * 4) + ve % HD / (HD / 16) * (8 * L::KB) + (v_at & 7) * L::KB +
            (HD == 256 ? ve % 16 / 2 : 0);
        v_scale = p + L::v_scales(plen) + scale_at(v_at, ve);
        v_first = ve % 32 == 0;
    }

private:
    __device__ __forceinline__ uint8_t* part(const Kv4Args& a, int page, int e) {
        return a.cache + ((long)max(page, 0) * a.n_kv + e / HD) * L::bytes(1 << a.page_shift);
    }
    __device__ __forceinline__ long scale_at(int at, int e) {
        return (long)(at >> 3) * (L::KB * 8) + e % HD / 32 * 8 + (at & 7);
    }
};

template <int HD>
__global__ __launch_bounds__(256) void kv4_write_kernel(Kv4Args a, const float* __restrict__ k,
                                                        const float* __restrict__ v, long ld) {
    Kv4Place<HD> to;
    f32x4 in[2][2] = {};
    // (on their way before the row's place is known; rows behind the last sequence may not be there)
    if (to.inside(a) && (!a.starts || to.row < a.starts[a.n_seqs])) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            in[0][i] = reinterpret_cast<const f32x4*>(k + to.row * ld + to.e)[i];
            in[1][i] = reinterpret_cast<const f32x4*>(v + to.row * ld + to.e)[i];
        }
    }
    to.find(a);
    uint32_t code[2];
    int byte[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        float x[8], mx = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = in[t][i / 4][i % 4];
            mx = fmaxf(mx, mx_mag(x[i]));
        }
        byte[t] = mx_byte(quad_max(mx));
        code[t] = mx_encode8(x, byte[t]);
    }
    code[1] = kv4_turn(code[1]);
    byte[1] = kv4_turn(byte[1]);
    if (to.page >= 0) {
        *reinterpret_cast<uint32_t*>(to.k) = code[0];
        if (to.k_first) *to.k_scale = (uint8_t)byte[0];
    }
    if (to.v_page >= 0) {
        if constexpr (HD == 64) {                        // two groups
            *reinterpret_cast<uint16_t*>(to.v) = (uint16_t)code[1];
            *reinterpret_cast<uint16_t*>(to.v + 16) = (uint16_t)(code[1] >> 16);
        } else {
            *reinterpret_cast<uint32_t*>(to.v) = code[1];
        }
        if (to.v_first) *to.v_scale = (uint8_t)byte[1];
    }
}

template <int HD>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4Args a, float* __restrict__ k, float* __restrict__ v,
                                                       long ld) {
    Kv4Place<HD> from;
    from.find(a);
    uint32_t code[2] = {0u, 0u};
    int byte[2] = {127, 127};
    if (from.page >= 0) {
        code[0] = *reinterpret_cast<const uint32_t*>(from.k);
        byte[0] = *from.k_scale;
    }
    if (from.v_page >= 0) {
        code[1] = HD == 64 ? *reinterpret_cast<const uint16_t*>(from.v) |
                                 (uint32_t) * reinterpret_cast<const uint16_t*>(from.v + 16) << 16
                           : *reinterpret_cast<const uint32_t*>(from.v);
        byte[1] = *from.v_scale;
    }
    code[1] = kv4_turn(code[1]);
    byte[1] = kv4_turn(byte[1]);
    if (!from.mine) return;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        float x[8];
        mx_decode8(code[t], mx_scale(byte[t]), x);
        f32x4* to = reinterpret_cast<f32x4*>((t ? v : k) + from.row * ld + from.e);
        to[0] = f32x4{x[0], x[1], x[2], x[3]};
        to[1] = f32x4{x[4], x[5], x[6], x[7]};
    }
}

// ---- attention --------------------------------------------------------------------
//
// A tile is up to 16 columns of (query row, head of the KV head's group), which
// walk the cache in chunks of 32 tokens with a running maximum and sum.  Of a
// chunk, with lane = 16 g + i and the token of a matrix row r of part t (0, 1)
// being 2 r + t:
//   S_t = K_t q       v_mfma_scale_f32_16x16x128_f8f6f4: K as it is stored (lane
//                     (g, i): block g of token 2i + t), q as a sum of E2M1 parts
//                     with falling scales.  Lane (g, i) gets tokens 8g .. 8g+7
//                     of column i.
//   O  += V^T P       v_mfma_f32_16x16x32_bf16: lane (g, i) gives tokens 8g ..
//                     8g+7 of elements of group i of V, made bf16 exactly, and of
//                     column i of P = exp2(S - m), which it has already, in three
//                     bf16 parts.  It gets elements of groups 4g .. 4g+3 of
//                     column i of O.
// q in parts, for each block of 32: the first is q / 2^e rounded to E2M1 with the
// block's largest value in [2, 4) 2^e, so at most 2^e / 2 off; each next one is the
// remainder in units 8 times smaller.  8 parts leave 2^-23 of the block's largest
// value.  Products of two E2M1 numbers and their sums of 128 are exact in this
// instruction.  (With E4M3 parts, 5 for 20 bits, it drops the low bits of
// products far below the largest one: 4e-6 of a sum for normal q, against none.  7 parts
// take 1 to 3 % less time and leave 2.3e-7 of an output at 20 to 60 tokens, where f32
// sums, and these 8, leave 5e-8.)
// P in three parts: its 24 bits.  (Two, rounded to nearest, leave 2^-18 of each p, 2.4e-6
// of an output where f32 sums leave 1e-6, and take a third of the P V instructions less:
// three prompts in 61 us, 67 with three parts.  These figures, and the comparisons of shapes below, are with
// seven parts of q on both sides.)
// The maximum is raised only when a score passes it by more than 2^8 (p then
// stays below 2^8, far from any overflow); most chunks need no rescaling.
//
// What bounds it.  Decode reads 17/16 bytes an element pair: 16001 tokens of 32 heads
// of 128 (70 MB) in 20.2 us, 3.5 TB/s; 10.7 of them pass between the first load and
// the last, the others are the start, the last chunk's products and the join.  24
// sequences of up to 8191 tokens, heads 32/8 of 64 (57 MB): 23.0 us.  A short context is
// latency, a chain of kernel arguments, lengths and table, K and V, LDS, the store:
// 4.9 us at 19 tokens.  Prompts are bound by the matrix instructions (of a chunk and 32
// columns at head dim 128, 32 of 16 cycles for the scores and 48 of 16 for P V, the
// latter's three parts) and the VALU beside them: 2048 rows of 32 heads of 128 in 87 us,
// 390 TFLOP/s of the products asked for.
// Why this shape.  16 columns, the least that the instructions have, and as few
// registers as that leaves, so that three or four blocks of a CU have their loads on
// their way (three or four chunks side by side in the 16 columns, where heads are
// few, take fewer instructions a chunk but registers for as many buffers: 24
// sequences of 32 heads of 128 took 70 us with them, 53 without).  32 columns for
// prompts: a chunk's V is made bf16 once for both (three prompts of 36 to 1023 rows of 32
// heads of 128: 67 us, 72 with 16).

constexpr float kKv4Floor = -3.0e38f;  // running maximum of a row that has seen nothing
constexpr float kKv4Lazy = 8.0f;
constexpr float kLog2e = 1.4426950408889634f;

struct Kv4AttnArgs {
    Kv4Args c;
    const float* q;
    long ld_q;
    float* out;
    long ld_out;
    int group;                          // heads of a KV head
    int tokens;                         // rows of a tile, at most 16 / group
    int tiles;                          // of the batch, some of them empty
    float scale;
    int window;
    // a split tile: most blocks, columns, and [tiles][n_kv][splits][cols] partial
    // sums (each HD elements, and maximum and sum of the weights)
    int splits, cols, blocks;
    int min_run;                        // chunks of a run, where there are several; up to twice as many are one
    float *part_o, *part_ml;
    int* counters;                      // [tiles][n_kv] blocks that are done, zero between calls
};

// E2M1 parts of q: the operands of N matrix instructions and their scale bytes.
// HD 64: an instruction's 128 is two parts of the 64 (K's blocks given twice).
// HD 256: part p's two halves are instructions 2p and 2p + 1.
// A block's threads take the tile's columns apart together, eight elements to a
// thread, and share the parts through LDS.
template <int HD, int COLS>
struct Kv4Query {
    static constexpr int PARTS = 8, N = PARTS * HD / 128;
    static constexpr int EIGHTS = HD / 8, ITEMS = COLS * EIGHTS;
    struct Shared {
        uint32_t part[PARTS][COLS][EIGHTS];
        int top[COLS][HD / 32];                            // scale byte of the first part, kMxNan: not finite
    };
    u32x4 q[N];
    int byte[N];

    // what a thread of THREADS takes apart: items of eight elements of a column
    template <int THREADS>
    struct Mine {
        static constexpr int PER = (ITEMS + THREADS - 1) / THREADS;
        f32x4 x[PER][2];

        __device__ __forceinline__ void fetch(const Kv4AttnArgs& a, int row0, int cols, int kvh) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int t = threadIdx.x + j * THREADS, c = t / EIGHTS, row = c / a.group;
                if (c >= cols) continue;
                const float* p = a.q + (row0 + row) * a.ld_q + ((long)kvh * a.group + c - row * a.group) * HD + t % EIGHTS * 8;
                x[j][0] = reinterpret_cast<const f32x4*>(p)[0];
                x[j][1] = reinterpret_cast<const f32x4*>(p)[1];
            }
        }

        __device__ __forceinline__ void split(float scale, int cols, Shared& to) const {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int t = threadIdx.x + j * THREADS;
                if (t < cols * EIGHTS) Kv4Query::split(x[j], scale, t, to);
            }
        }
    };

    __device__ __forceinline__ static void split(const f32x4 (&v)[2], float scale, int t, Shared& to) {
        const int c = t / EIGHTS, e = t % EIGHTS;
        float x[8], mx = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = v[i >> 2][i & 3] * scale;
            mx = fmaxf(mx, mx_mag(x[i]));
        }
        mx = quad_max(mx);                               // of the block's four threads
        const int field = (int)(__float_as_uint(mx) >> 23), top = max(field - 1, 0);
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            const float s = mx_scale(max(top - 3 * p, 0));
            const uint32_t w = mx_round8(x, s);
            float y[8];
            mx_decode8(w, s, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] -= y[i];
            to.part[p][c][e] = w;
        }
        if ((e & 3) == 0) to.top[c][e >> 2] = field == 255 ? kMxNan : top;
    }

    // the lane's column c, lane group g
    __device__ __forceinline__ void load(const Shared& from, int c, int g) {
#pragma unroll
        for (int f = 0; f < N; ++f) {
            const int part = HD == 64 ? 2 * f + (g >> 1) : HD == 128 ? f : f >> 1;
            const int blk = HD == 64 ? g & 1 : HD == 128 ? g : 4 * (f & 1) + g;
            q[f] = *reinterpret_cast<const u32x4*>(&from.part[part][c][4 * blk]);
            const int top = from.top[c][blk];
            byte[f] = top == kMxNan ? kMxNan : max(top - 3 * part, 0);
        }
    }
};

// K of a chunk in the registers of a wave
template <int HD>
struct Kv4K {
    static constexpr int KB = HD / 32, H = HD == 256 ? 2 : 1;   // steps of 128 elements
    u32x4 k[H][2];                                       // [step][part t]
    uint16_t s[H];                                       // scale bytes of parts 0 and 1

    // at: the chunk's first token in the page
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t page, int at, int plen, int lane) {
        const int i = lane & 15, g = lane >> 4, blk = HD == 64 ? g & 1 : g;
        const uint32_t codes = at * (HD / 2), bytes = (uint32_t)Kv4Layout<HD>::k_scales(plen) + at * KB;
#pragma unroll
        for (int h = 0; h < H; ++h) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
                k[h][t] = __builtin_amdgcn_raw_buffer_load_b128(page, (2 * i + t) * (HD / 2) + h * 64 + blk * 16, codes, 0);
            s[h] = __builtin_amdgcn_raw_buffer_load_b16(page, (i >> 2) * (8 * KB) + (4 * h + blk) * 8 + 2 * (i & 3), bytes, 0);
        }
    }

    // scores of tokens 8g + j of the chunk in the lane's column of each tile; the
    // 2 CT sums take turns, so that no instruction waits for the one before
    template <typename Q, int CT>
    __device__ __forceinline__ void scores(const Q (&q)[CT], float (&to)[CT][8]) const {
        f32x4 d[CT][2];
#pragma unroll
        for (int c = 0; c < CT; ++c) d[c][0] = d[c][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int f = Q::N - 1; f >= 0; --f) {
            const int h = HD == 256 ? f & 1 : 0;
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                // (the argument before a scale picks its byte)
                d[c][0] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_frag(k[h][0]), mx_frag(q[c].q[f]), d[c][0], kFp4, kFp4,
                                                                           0, s[h], 0, q[c].byte[f]);
                d[c][1] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_frag(k[h][1]), mx_frag(q[c].q[f]), d[c][1], kFp4, kFp4,
                                                                           1, s[h], 0, q[c].byte[f]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) to[c][j] = d[c][j & 1][j >> 1];
    }
};

// V of a chunk
template <int HD>
struct Kv4V {
    static constexpr int KB = HD / 32, W = HD / 16;      // dwords of a lane
    uint32_t v[W];
    u32x2 s;

    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t page, int at, int plen, int lane) {
        const int i = lane & 15, g = lane >> 4;
        const uint32_t codes = (uint32_t)Kv4Layout<HD>::v_codes(plen) + at * (HD / 2);
        const uint32_t bytes = (uint32_t)Kv4Layout<HD>::v_scales(plen) + at * KB;
#pragma unroll
        for (int w = 0; w < W / 4; ++w) {
            const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(page, (g * 16 + i) * (8 * KB) + 16 * w, codes, 0);
            v[4 * w] = x.x; v[4 * w + 1] = x.y; v[4 * w + 2] = x.z; v[4 * w + 3] = x.w;
        }
        s = __builtin_amdgcn_raw_buffer_load_b64(page, (g * KB + i * (HD / 16) / 32) * 8, bytes, 0);
    }
};

// The bytes of a (page, head) as a buffer.  No page: an empty one (at the cache's
// start), whose loads come back at once with zeros.  Every load of the scan is made
// whether its chunk is there or not: a load under a condition would have the
// compiler wait for all of them wherever it needs one.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t kv4_buffer(const uint8_t* p, bool there) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, there ? 0xFFFFFFFFu : 0u, 0x00020000);
}

// scale bytes past kMxMaxByte, whose blocks read as NaN: their high bits
__device__ __forceinline__ uint32_t kv4_nan_bytes(uint32_t w) {
    return w & ((w & 0x7F7F7F7Fu) + 0x03030303u) & 0x80808080u;
}

typedef bf16x8 Kv4Weights[3];

template <int HD>
struct Kv4State {
    static constexpr int J = HD / 16;                    // elements of a group, and tiles of O
    f32x4 o[J];
    float m, l;

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < J; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        m = kKv4Floor;
        l = 0.f;
    }

    // the weights of 8 scores, in three bf16 parts; maximum and sum move on
    __device__ __forceinline__ void weigh(const float (&s)[8], Kv4Weights& p) {
        u32x4 part[3];
        float top = s[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) top = fmaxf(top, s[j]);
        if (__any(top > m + kKv4Lazy)) {
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float to_m = fmaxf(m, top), down = __builtin_amdgcn_exp2f(m - to_m);
            m = to_m;
            l *= down;
#pragma unroll
            for (int j = 0; j < J; ++j) o[j] *= down;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a = __builtin_amdgcn_exp2f(s[2 * j] - m), b = __builtin_amdgcn_exp2f(s[2 * j + 1] - m);
            l += a + b;
            // two truncations and the rest: 8 + 8 + 8 bits, each p exactly
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                part[e][j] = bf16_hi2(a, b);
                a -= __uint_as_float(__float_as_uint(a) & 0xFFFF0000u);
                b -= __uint_as_float(__float_as_uint(b) & 0xFFFF0000u);
            }
            part[2][j] = bf16_hi2(a, b);
        }
#pragma unroll
        for (int e = 0; e < 3; ++e) p[e] = __builtin_bit_cast(bf16x8, part[e]);
    }
};

// V of a chunk as the matrix instructions take it
template <int HD>
struct Kv4Values {
    const Kv4V<HD>& c;
    float s[8];                                          // the tokens' scales
    bool nans;                                           // there were blocks that read as NaN

    // Tokens that are not there (the chunk has `live`) get the smallest scale:
    // their p is zero, and so, whatever their bytes are, is the product.  Blocks
    // that read as NaN are left out the same way, and seen to at the end.
    __device__ __forceinline__ Kv4Values(const Kv4V<HD>& v, int live, int g) : c(v), nans(false) {
        uint32_t sc[2] = {v.s.x, v.s.y};
        if (live < 32) {
            const int n = min(max(live - 8 * g, 0), 8);
            sc[0] &= n >= 4 ? ~0u : (1u << (8 * n)) - 1u;
            sc[1] &= n >= 8 ? ~0u : n <= 4 ? 0u : (1u << (8 * (n - 4))) - 1u;
        }
        const uint32_t bad[2] = {kv4_nan_bytes(sc[0]), kv4_nan_bytes(sc[1])};
        if (__any((bad[0] | bad[1]) != 0)) {
            nans = true;
#pragma unroll
            for (int w = 0; w < 2; ++w) sc[w] &= ~((bad[w] >> 7) * 255u);
        }
        // (the conversion takes the exponent field of its scale and nothing else)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = __uint_as_float((j & 3) == 3 ? sc[j >> 2] >> 1 : sc[j >> 2] << (23 - 8 * (j & 3)));
    }

    // elements 2e, 2e+1 of token j as bf16
    template <int J8, int E>
    __device__ __forceinline__ uint32_t at() const {
        constexpr int byte = J8 * (HD / 32) + E;
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c.v[byte / 4], s[J8], byte % 4));
    }

    // O += V^T P in elements 2e, 2e + 1 of the groups, for each column tile
    template <int E, int CT>
    __device__ __forceinline__ void pair(const Kv4Weights (&p)[CT], Kv4State<HD> (&st)[CT]) const {
        const uint32_t w[8] = {at<0, E>(), at<1, E>(), at<2, E>(), at<3, E>(), at<4, E>(), at<5, E>(), at<6, E>(), at<7, E>()};
        u32x4 even, odd;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            even[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x05040100u);
            odd[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x07060302u);
        }
        const bf16x8 a = __builtin_bit_cast(bf16x8, even), b = __builtin_bit_cast(bf16x8, odd);
#pragma unroll
        for (int j = 2; j >= 0; --j)
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                st[t].o[2 * E] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, p[t][j], st[t].o[2 * E], 0, 0, 0);
                st[t].o[2 * E + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, p[t][j], st[t].o[2 * E + 1], 0, 0, 0);
            }
    }

    template <int CT>
    __device__ __forceinline__ void add(const Kv4Weights (&p)[CT], Kv4State<HD> (&st)[CT]) const {
        pair<0, CT>(p, st);
        pair<1, CT>(p, st);
        if constexpr (HD >= 128) {
            pair<2, CT>(p, st);
            pair<3, CT>(p, st);
        }
        if constexpr (HD >= 256) {
            pair<4, CT>(p, st);
            pair<5, CT>(p, st);
            pair<6, CT>(p, st);
            pair<7, CT>(p, st);
        }
    }
};

// The sequence of a batch's tile u.  Tiles of sequence s begin at starts[s] / tokens
// + s, which leaves each sequence as many as it needs, whatever the lengths.
__device__ __forceinline__ int kv4_sequence(const Kv4AttnArgs& a, int u) {
    int lo = 0, hi = a.c.n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.c.starts[mid] / a.tokens + mid <= u) lo = mid;
        else hi = mid;
    }
    return lo;
}

// A tile's work: its rows and columns (16 CT at most), the chunks that any column
// sees, and the first pages of its sequence, one to a lane.
struct Kv4Tile {
    int s, row0, rows, cols, pos0;
    int first, last;                    // chunks [first, last)
    int tokens_end;                     // tokens from here on are seen by no column
    int pages;

    __device__ __forceinline__ bool set(const Kv4AttnArgs& a, int u, int lane) {
        s = a.c.starts ? __builtin_amdgcn_readfirstlane(kv4_sequence(a, u)) : u;
        // (the table's entries on their way before the lengths are here)
        pages = lane < a.c.table_stride ? a.c.table[(long)s * a.c.table_stride + lane] : -1;
        const int len = max(a.c.lens[s], 0);
        int end = u + 1, there = end;                    // of the sequence's rows, and of those that q and out have
        row0 = u;
        if (a.c.starts) {
            const int begin = max(a.c.starts[s], 0), skip = (u - (begin / a.tokens + s)) * a.tokens;
            end = a.c.starts[s + 1];
            there = min(end, a.c.n_rows);
            if (skip < 0 || skip >= there - begin) return false;
            row0 = begin + skip;
        }
        // (all of it is the same in every lane; said here, the loops stay in scalar registers)
        row0 = __builtin_amdgcn_readfirstlane(row0);
        rows = __builtin_amdgcn_readfirstlane(min(a.tokens, there - row0));
        pos0 = __builtin_amdgcn_readfirstlane(len - (end - row0));
        cols = rows * a.group;
        tokens_end = min(pos0 + rows, a.c.cap);
        first = seen_from(a, pos0) >> 5;
        last = tokens_end > 0 ? (tokens_end + 31) >> 5 : 0;
        return true;
    }

    __device__ __forceinline__ static int seen_from(const Kv4AttnArgs& a, int pos) {
        return a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0;
    }

    // a chunk of which not every column sees every token
    __device__ __forceinline__ bool masked(const Kv4AttnArgs& a, int chunk) const {
        return chunk * 32 + 31 > pos0 || chunk * 32 < seen_from(a, pos0 + rows - 1);
    }
};

// a lane's column of column tile ct
struct Kv4Column {
    bool mine;                          // it is one (others repeat the last)
    int col;
    int from, to;                       // it sees tokens [from, to]

    __device__ __forceinline__ void set(const Kv4AttnArgs& a, const Kv4Tile& tile, int ct, int lane) {
        const int i = 16 * ct + (lane & 15);
        col = min(i, tile.cols - 1);
        mine = i < tile.cols;
        to = tile.pos0 + col / a.group;
        from = Kv4Tile::seen_from(a, to);
    }
};

// Chunks begin, begin + step, .. below end into st.  K and V of a chunk are loaded
// BUF chunks ahead, page numbers 64 at a time.
// Every thread of a block of THREADS comes here, for the query.
template <int HD, int CT, int BUF, int THREADS>
__device__ __forceinline__ void kv4_scan(const Kv4AttnArgs& a, const Kv4Tile& tile, const Kv4Column (&col)[CT], int kvh,
                                         int begin, int end, int step,
                                         const typename Kv4Query<HD, 16 * CT>::template Mine<THREADS>& mine,
                                         typename Kv4Query<HD, 16 * CT>::Shared& shared, Kv4State<HD> (&st)[CT], int lane) {
    typedef Kv4Query<HD, 16 * CT> Q;
    const int g = lane >> 4, plen = 1 << a.c.page_shift, n = end > begin && a.c.n_pages > 0 ? (end - begin + step - 1) / step : 0;
    const int* const table = a.c.table + (long)tile.s * a.c.table_stride;
    const long head = (long)kvh * Kv4Layout<HD>::bytes(plen), page_bytes = a.c.n_kv * Kv4Layout<HD>::bytes(plen);
    // pages window .. window + 63 of the sequence
    int pages = tile.pages, window = 0;
    const auto page = [&](int chunk) {
        const int at = chunk * 32 >> a.c.page_shift;
        if ((unsigned)(at - window) >= 64u) {
            window = at;
            pages = at + lane < a.c.table_stride ? table[at + lane] : -1;
        }
        const int p = __builtin_amdgcn_readlane(pages, at - window);
        return p < a.c.n_pages ? p : -1;
    };
    Kv4K<HD> k[BUF];
    Kv4V<HD> v[BUF];
    // where a buffer's chunk is: K's, and V's from when K's next one is on its way
    bool k_there[BUF], v_there[BUF];
    __amdgpu_buffer_rsrc_t from[BUF];
    int at[BUF];
    const auto fetch_k = [&](int t, int b) {
        const int p = t < n ? page(begin + t * step) : -1;
        k_there[b] = p >= 0;
        at[b] = p >= 0 ? (begin + t * step) * 32 & (plen - 1) : 0;
        from[b] = kv4_buffer(a.c.cache + (p >= 0 ? p * page_bytes + head : 0), p >= 0);
        k[b].load(from[b], at[b], plen, lane);
    };
    const auto fetch_v = [&](int b) {                    // of the chunk that K's buffer has
        v_there[b] = k_there[b];
        v[b].load(from[b], at[b], plen, lane);
    };
    if (n > 0) {
#pragma unroll
        for (int b = 0; b < BUF; ++b) fetch_k(b, b);
#pragma unroll
        for (int b = 0; b < BUF; ++b) fetch_v(b);
    }
    mine.split(a.scale * kLog2e, tile.cols, shared);
    __syncthreads();
    Q q[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        q[c].load(shared, col[c].col, g);
        st[c].clear();
    }
    bool nans = false;
    // (without loads ahead in the last round)
    const auto round = [&](int t0, auto more) {
#pragma unroll
        for (int b = 0; b < BUF; ++b) {
            const int chunk = begin + (t0 + b) * step;
            float s[CT][8];
            if (k_there[b]) {
                k[b].scores(q, s);
            } else {
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int j = 0; j < 8; ++j) s[c][j] = -__builtin_inff();
            }
            if constexpr (decltype(more)::value) fetch_k(t0 + b + BUF, b);
            if (t0 + b < n && tile.masked(a, chunk))
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int key = chunk * 32 + 8 * g + j;
                        if (key < col[c].from || key > col[c].to) s[c][j] = -__builtin_inff();
                    }
            Kv4Weights p[CT];
#pragma unroll
            for (int c = 0; c < CT; ++c) st[c].weigh(s[c], p[c]);
            if (v_there[b]) {
                const Kv4Values<HD> values(v[b], tile.tokens_end - chunk * 32, g);
                values.template add<CT>(p, st);
                nans = nans || values.nans;
            }
            if constexpr (decltype(more)::value) fetch_v(b);
        }
    };
    int t0 = 0;
#pragma unroll 1
    for (; t0 + BUF < n; t0 += BUF) round(t0, std::true_type{});
    if (t0 < n) round(t0, std::false_type{});
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        st[c].l += __shfl_xor(st[c].l, 16, 64);
        st[c].l += __shfl_xor(st[c].l, 32, 64);
    }
    // Blocks of V that read as NaN: the columns that see their token get NaN in the
    // block's elements.  (Rare: the scale bytes are read again.)
    if (nans) {
        uint32_t rows[CT] = {};                          // rows 4g + r of O^T in the lane's column
#pragma unroll 1
        for (int t = 0; t < n; ++t) {
            const int first = (begin + t * step) * 32, p = table[first >> a.c.page_shift];
            if (p < 0 || p >= a.c.n_pages) continue;
            const uint8_t* sp = a.c.cache + p * page_bytes + head + Kv4Layout<HD>::v_scales(plen) + (first & (plen - 1)) * (HD / 32);
#pragma unroll 1
            for (int e = 0; e < HD; ++e) {               // byte e: token e / (HD / 4) * 8 + e % 8, block e / 8 % (HD / 32)
                const int key = first + e / (HD / 4) * 8 + e % 8, blk = e / 8 % (HD / 32);
                if (key >= tile.tokens_end || sp[e] <= kMxMaxByte) continue;
#pragma unroll
                for (int c = 0; c < CT; ++c)
                    if (key >= col[c].from && key <= col[c].to)
                        for (int x = 0; x < 4; ++x)
                            if ((4 * g + x) * (HD / 16) / 32 == blk) rows[c] |= 1u << x;
            }
        }
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (rows[c] >> x & 1u)
#pragma unroll
                    for (int j = 0; j < Kv4State<HD>::J; ++j) st[c].o[j][x] = __builtin_nanf("");
    }
}

// block -> (tile, KV head): consecutive blocks run on different XCDs, so each takes
// a run of the heads and its L2 their tokens; of its heads, a tile's one after the
// other, so that the tiles come in the order of their lengths.
__device__ __forceinline__ bool kv4_place(int block, int tiles, int n_kv, int& u, int& kvh) {
    const int xcd = block & 7, at = block >> 3;
    if (n_kv % 8 == 0) {
        const int heads = n_kv / 8;
        u = at / heads;
        kvh = xcd * heads + at - u * heads;
        return u < tiles;
    }
    const int per = (tiles * n_kv + 7) / 8, all = xcd * per + at;
    if (at >= per || all >= tiles * n_kv) return false;
    kvh = all / tiles;
    u = all - kvh * tiles;
    return true;
}

// A tile and KV head to up to a.splits blocks, in runs of the same length for every
// tile.  A block's waves take every fourth chunk of its run and join their sums in
// LDS; the blocks' are joined by the one that ends last.
constexpr int kKv4Waves = 4;

// all lanes' sum or largest value, of integers
template <bool MAX>
__device__ __forceinline__ int wave_int(int v) {
    const auto step = [&](int x) { v = MAX ? max(v, x) : v + x; };
    step(__builtin_amdgcn_update_dpp(MAX ? v : 0, v, 0xB1, 0xF, 0xF, false));
    step(__builtin_amdgcn_update_dpp(MAX ? v : 0, v, 0x4E, 0xF, 0xF, false));
    step(__builtin_amdgcn_update_dpp(MAX ? v : 0, v, 0x141, 0xF, 0xF, false));
    step(__builtin_amdgcn_update_dpp(MAX ? v : 0, v, 0x140, 0xF, 0xF, false));
    step(__builtin_amdgcn_update_dpp(MAX ? v : 0, v, 0x142, 0xA, 0xF, false));
    step(__builtin_amdgcn_update_dpp(MAX ? v : 0, v, 0x143, 0xC, 0xF, false));
    return __builtin_amdgcn_readlane(v, 63);
}

// The run's length: the batch's chunks, as its lengths are now, over a.blocks blocks,
// raised until the runs are no more than that (a last run is part of one, and a
// block too many would double the time); no tile has more than a.splits runs.
// (Every lane of a wave takes part.)
// tokens and rows of sequence s, as the caller wrote them
struct Kv4Seq {
    int tokens, begin, end;

    __device__ __forceinline__ void load(const Kv4AttnArgs& a, int s) {
        tokens = a.c.lens[s];
        begin = a.c.starts ? a.c.starts[s] : s;
        end = a.c.starts ? a.c.starts[s + 1] : s + 1;
    }
};

// first: sequence `lane`
__device__ __forceinline__ int kv4_run(const Kv4AttnArgs& a, const Kv4Seq& first, int lane) {
    if (a.splits == 1) return 1 << 26;
    // tiles and chunks of a sequence
    const float per_tile = 1.f / a.tokens;
    const auto size = [&](int s, int& tiles, int& chunks) {
        Kv4Seq seq = first;
        if (s >= 64) seq.load(a, s);
        int tokens = min(max(seq.tokens, 0), a.c.cap);
        tiles = min((int)ceilf(max((float)seq.end - (float)seq.begin, 0.f) * per_tile), a.tiles);
        // (a window's first and last chunk are parts)
        if (a.window > 0 && tokens - a.tokens - 31 > a.window) tokens = a.window + a.tokens + 31;
        chunks = tiles ? (tokens + 31) >> 5 : 0;
    };
    // (sums capped, so that 64 lanes' fit, and roughly rounded: any run is right)
    int all = 0, most = 0, count = 0, tiles, chunks;
    for (int s = lane; s < a.c.n_seqs; s += 64) {
        size(s, tiles, chunks);
        all = (int)min(all + (long)tiles * chunks, 1L << 24);
        count = min(count + tiles, 1 << 24);
        most = max(most, chunks);
    }
    const int units = wave_int<false>(count), long_run = wave_int<true>(most);
    const float per = (float)a.c.n_kv / a.blocks;
    if (long_run <= 2 * a.min_run) return 2 * a.min_run;
    const int least = max(a.min_run, (long_run + a.splits - 1) / a.splits);
    int run = max(least, (int)ceilf(wave_int<false>(all) * per));
    for (int turn = 0; turn < 3 && units * per <= 1.f; ++turn) {
        count = 0;
        const float in_run = __builtin_amdgcn_rcpf((float)run);
        for (int s = lane; s < a.c.n_seqs; s += 64) {
            size(s, tiles, chunks);
            count = min(count + tiles * (int)ceilf(chunks * in_run), 1 << 24);
        }
        const float over = wave_int<false>(count) * per;
        if (over <= 1.f) break;
        run = (int)ceilf(run * over);
    }
    return __builtin_amdgcn_readfirstlane(run);
}

// partial sums past this XCD's L2 and back (agent scope)
__device__ __forceinline__ void kv4_put(float* p, float a, float b) {
    const uint64_t v = (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ void kv4_get(const float* p, float& a, float& b) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    a = __uint_as_float((uint32_t)v);
    b = __uint_as_float((uint32_t)(v >> 32));
}

template <int HD, int COLS>
struct Kv4Shared {
    union {
        typename Kv4Query<HD, COLS>::Shared q;
        float o[kKv4Waves][COLS][HD + 4];                // the waves' sums
        float f[64][COLS];                               // the runs' factors
    };
    f32x4 red[kKv4Waves * 64];
    float m[kKv4Waves][COLS], l[kKv4Waves][COLS];
    float sum[COLS];                                     // the columns' sums of weights
    int last;
};

// waves of a SIMD for the registers of HD and CT, and so blocks of a CU
constexpr int kv4_at_once(int hd, int ct) { return ct > 1 || hd == 256 ? 2 : hd == 128 ? 3 : 4; }

template <int HD, int CT>
__global__ __launch_bounds__(kKv4Waves * 64, kv4_at_once(HD, CT)) void kv4_attention_kernel(Kv4AttnArgs a) {
    __shared__ Kv4Shared<HD, 16 * CT> sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4, split = blockIdx.y;
    int u, kvh;
    if (!kv4_place(blockIdx.x, a.tiles, a.c.n_kv, u, kvh)) return;
    u = a.tiles - 1 - u;                                 // a prompt's last tiles, the longest, first
    Kv4Seq first = {0, 0, 0};                            // (on its way before the tile's own loads are waited for)
    if (lane < a.c.n_seqs) first.load(a, lane);
    Kv4Tile tile;
    if (!tile.set(a, u, lane)) return;
    typename Kv4Query<HD, 16 * CT>::template Mine<kKv4Waves * 64> mine;
    mine.fetch(a, tile.row0, tile.cols, kvh);
    // (never more runs than the grid has blocks for, whatever the starts hold)
    const int run = max(kv4_run(a, first, lane), (tile.last - tile.first + a.splits - 1) / a.splits);
    const int begin = tile.first + split * run;
    if (split > 0 && begin >= tile.last) return;
    const int runs = max((tile.last - tile.first + run - 1) / run, 1);
    Kv4Column col[CT];
    Kv4State<HD> st[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) col[c].set(a, tile, c, lane);
    // (two column tiles, or 256 elements, leave registers for one chunk ahead)
    constexpr int BUF = CT > 1 || HD == 256 ? 1 : 2;
    kv4_scan<HD, CT, BUF, kKv4Waves * 64>(a, tile, col, kvh, begin + wave, min(begin + run, tile.last), kKv4Waves,
                                                             mine, sh.q, st, lane);
    __syncthreads();                                     // the query has been read
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        if (!col[c].mine) continue;
        if (g == 0) {
            sh.m[wave][16 * c + i] = st[c].m;
            sh.l[wave][16 * c + i] = st[c].l;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < Kv4State<HD>::J; j += 4)
                *reinterpret_cast<f32x4*>(&sh.o[wave][16 * c + i][(4 * g + r) * (HD / 16) + j]) =
                    f32x4{st[c].o[j][r], st[c].o[j + 1][r], st[c].o[j + 2][r], st[c].o[j + 3][r]};
    }
    __syncthreads();
    // four elements of a column to a thread
    const int cols = tile.cols;
    const long part = (((long)u * a.c.n_kv + kvh) * a.splits) * a.cols;
    const auto store = [&](int c, int d, f32x4 o, float l) {
        const int t = c / a.group;
        float* to = a.out + (tile.row0 + t) * a.ld_out + ((long)kvh * a.group + c - t * a.group) * HD + d;
        *reinterpret_cast<f32x4*>(to) = o * (l == 0.f ? 0.f : 1.f / l);   // a row that has seen nothing is zero
    };
    for (int e = threadIdx.x; e < cols * (HD / 4); e += kKv4Waves * 64) {
        const int c = e / (HD / 4), d = e % (HD / 4) * 4;
        float m = kKv4Floor, l = 0.f;
#pragma unroll
        for (int w = 0; w < kKv4Waves; ++w) m = fmaxf(m, sh.m[w][c]);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kKv4Waves; ++w) {
            const float f = __builtin_amdgcn_exp2f(sh.m[w][c] - m);
            l += f * sh.l[w][c];
            o += f * *reinterpret_cast<const f32x4*>(&sh.o[w][c][d]);
        }
        if (runs == 1) {
            store(c, d, o, l);
        } else {
            const long at = part + (long)split * a.cols + c;
            kv4_put(a.part_o + at * HD + d, o.x, o.y);
            kv4_put(a.part_o + at * HD + d + 2, o.z, o.w);
            if (d == 0) kv4_put(a.part_ml + 2 * at, m, l);
        }
    }
    if (runs == 1) return;
    // The block that ends last joins the runs.  Every thread's partial sums have
    // arrived before its block is counted, so they are there for the last one.
    __builtin_amdgcn_s_waitcnt(0x0F70);                  // vmcnt(0)
    __syncthreads();
    int* const counter = a.counters + (long)u * a.c.n_kv + kvh;
    if (threadIdx.x == 0)
        sh.last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == runs - 1;
    __syncthreads();
    if (!sh.last) return;
    // a run to a lane (at most 64 of them), a column to a wave
    for (int c = wave; c < cols; c += kKv4Waves) {
        float m = kKv4Floor, l = 0.f;
        if (lane < runs) kv4_get(a.part_ml + 2 * (part + (long)lane * a.cols + c), m, l);
        const float f = __builtin_amdgcn_exp2f(m - wave_max(m));
        l = wave_sum(f * l);
        if (lane < runs) sh.f[lane][c] = f;
        if (lane == 0) sh.sum[c] = l;
    }
    __syncthreads();
    // four elements to a thread; threads beyond the columns' take other runs
    constexpr int T = kKv4Waves * 64;
    const int items = cols * (HD / 4), groups = max(T / items, 1), group = groups > 1 ? threadIdx.x / items : 0;
    for (int e = threadIdx.x - group * items; e < items && group < groups; e += T) {
        const int c = e / (HD / 4), d = e % (HD / 4) * 4;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int r = group; r < runs; r += groups) {
            const float* p = a.part_o + (part + (long)r * a.cols + c) * HD + d;
            float x[4];
            kv4_get(p, x[0], x[1]);
            kv4_get(p + 2, x[2], x[3]);
            o += sh.f[r][c] * f32x4{x[0], x[1], x[2], x[3]};
        }
        if (groups == 1) store(c, d, o, sh.sum[c]);
        else sh.red[threadIdx.x] = o;
    }
    if (groups > 1) {
        __syncthreads();
        if (threadIdx.x < items) {
            f32x4 o = sh.red[threadIdx.x];
            for (int x = 1; x < groups; ++x) o += sh.red[x * items + threadIdx.x];
            store(threadIdx.x / (HD / 4), threadIdx.x % (HD / 4) * 4, o, sh.sum[threadIdx.x / (HD / 4)]);
        }
    }
    if (threadIdx.x == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---- launches ---------------------------------------------------------------------

static int kv4_check(const char* who, const atlas_kv4_cache& c) {
    ATLAS_REQUIRE(c.head_dim == 64 || c.head_dim == 128 || c.head_dim == 256, "%s: head_dim %d (64, 128 or 256)", who,
                  c.head_dim);
    ATLAS_REQUIRE(c.page_len >= 32 && c.page_len <= 1 << 22 && (c.page_len & (c.page_len - 1)) == 0,
                  "%s: page_len %d (a power of two from 32 to 2^22)", who, c.page_len);
    ATLAS_REQUIRE(c.n_pages >= 0 && c.n_kv > 0 && c.n_kv <= 4096, "%s: %d pages, %d KV heads", who, c.n_pages, c.n_kv);
    const int64_t page = (int64_t)c.n_kv * c.page_len * (c.head_dim + c.head_dim / 16);
    ATLAS_REQUIRE(c.n_pages <= INT64_MAX / page, "%s: %d pages of %lld bytes", who, c.n_pages, (long long)page);
    return ATLAS_OK;
}

int64_t kv4_cache_bytes(const atlas_kv4_cache& c) {
    const int rc = kv4_check("kv4_cache_bytes", c);
    if (rc) return rc;
    return (int64_t)c.n_pages * c.n_kv * ((int64_t)c.page_len * (c.head_dim + c.head_dim / 16));
}

// fills the kernels' arguments; *n_rows 0: nothing to do
static int kv4_args(const char* who, const atlas_kv4_cache& c, const atlas_kv4_batch& b, Kv4Args& a) {
    const int rc = kv4_check(who, c);
    if (rc) return rc;
    ATLAS_REQUIRE(b.n_seqs >= 0 && b.n_rows >= 0 && b.table_stride >= 0 && b.max_len >= 0,
                  "%s: %d sequences, %d rows, table stride %d, max_len %d", who, b.n_seqs, b.n_rows, b.table_stride,
                  b.max_len);
    ATLAS_REQUIRE(b.row_starts || b.n_rows == b.n_seqs, "%s: %d rows of %d sequences need row_starts", who, b.n_rows,
                  b.n_seqs);
    ATLAS_REQUIRE(b.n_seqs <= 1 << 20 && b.n_rows <= 1 << 20, "%s: %d rows of %d sequences", who, b.n_rows, b.n_seqs);
    a = Kv4Args{};
    a.n_rows = b.n_seqs == 0 ? 0 : b.n_rows;
    if (a.n_rows == 0) return ATLAS_OK;
    ATLAS_REQUIRE(b.kv_lens && (b.table_stride == 0 || b.block_table) && (c.n_pages == 0 || c.data), "%s: null argument", who);
    ATLAS_REQUIRE(((uintptr_t)c.data & 15) == 0, "%s: the cache starts on 16 bytes", who);
    ATLAS_REQUIRE((((uintptr_t)b.kv_lens | (uintptr_t)b.block_table | (uintptr_t)b.row_starts) & 3) == 0,
                  "%s: misaligned batch", who);
    a.cache = static_cast<uint8_t*>(c.data);
    a.n_pages = c.n_pages;
    a.n_kv = c.n_kv;
    while ((1 << a.page_shift) < c.page_len) ++a.page_shift;
    a.starts = b.row_starts;
    a.lens = b.kv_lens;
    a.table = b.block_table;
    a.table_stride = b.table_stride;
    a.n_seqs = b.n_seqs;
    // (positions are 32-bit and a chunk reaches 31 past one)
    a.cap = (int)std::min<int64_t>((int64_t)b.table_stride * c.page_len, 0x7FFFFFC0);
    return ATLAS_OK;
}

static int kv4_rows_check(const char* who, const void* p, const void* q, long ld, long wide) {
    ATLAS_REQUIRE(p && q, "%s: null argument", who);
    ATLAS_REQUIRE((((uintptr_t)p | (uintptr_t)q) & 15) == 0 && ld % 4 == 0 && ld >= wide,
                  "%s: rows start on 16 bytes, at least %ld elements apart (stride %ld)", who, wide, ld);
    return ATLAS_OK;
}

int kv4_write_launch(const atlas_kv4_cache& c, const atlas_kv4_batch& b, const float* k, const float* v, long ld,
                     hipStream_t st) {
    Kv4Args a;
    int rc = kv4_args("kv4_write", c, b, a);
    if (rc || a.n_rows == 0) return rc;
    const long wide = (long)c.n_kv * c.head_dim;
    if ((rc = kv4_rows_check("kv4_write", k, v, ld, wide))) return rc;
    const dim3 grid((a.n_rows + 7) / 8, (unsigned)((wide + 255) / 256));
    if (c.head_dim == 64) hipLaunchKernelGGL(kv4_write_kernel<64>, grid, dim3(256), 0, st, a, k, v, ld);
    else if (c.head_dim == 128) hipLaunchKernelGGL(kv4_write_kernel<128>, grid, dim3(256), 0, st, a, k, v, ld);
    else hipLaunchKernelGGL(kv4_write_kernel<256>, grid, dim3(256), 0, st, a, k, v, ld);
    ATLAS_LAUNCH_CHECK("kv4_write");
    return ATLAS_OK;
}

int kv4_read_launch(const atlas_kv4_cache& c, const atlas_kv4_batch& b, float* k, float* v, long ld, hipStream_t st) {
    Kv4Args a;
    int rc = kv4_args("kv4_read", c, b, a);
    if (rc || a.n_rows == 0) return rc;
    const long wide = (long)c.n_kv * c.head_dim;
    if ((rc = kv4_rows_check("kv4_read", k, v, ld, wide))) return rc;
    const dim3 grid((a.n_rows + 7) / 8, (unsigned)((wide + 255) / 256));
    if (c.head_dim == 64) hipLaunchKernelGGL(kv4_read_kernel<64>, grid, dim3(256), 0, st, a, k, v, ld);
    else if (c.head_dim == 128) hipLaunchKernelGGL(kv4_read_kernel<128>, grid, dim3(256), 0, st, a, k, v, ld);
    else hipLaunchKernelGGL(kv4_read_kernel<256>, grid, dim3(256), 0, st, a, k, v, ld);
    ATLAS_LAUNCH_CHECK("kv4_read");
    return ATLAS_OK;
}

int kv4_attention_launch(const atlas_kv4_cache& c, const atlas_kv4_batch& b, const float* q, long ld_q, int n_heads,
                         float scale, int window, float* out, long ld_out, hipStream_t st) {
    Kv4AttnArgs a{};
    int rc = kv4_args("kv4_attention", c, b, a.c);
    if (rc) return rc;
    ATLAS_REQUIRE(n_heads > 0 && n_heads % c.n_kv == 0 && n_heads / c.n_kv <= 16,
                  "kv4_attention: %d heads over %d KV heads (up to 16 to each)", n_heads, c.n_kv);
    ATLAS_REQUIRE(window >= 0, "kv4_attention: window %d", window);
    if (a.c.n_rows == 0) return ATLAS_OK;
    const long row = (long)n_heads * c.head_dim;
    if ((rc = kv4_rows_check("kv4_attention", q, q, ld_q, row))) return rc;
    if ((rc = kv4_rows_check("kv4_attention", out, out, ld_out, row))) return rc;
    a.q = q;
    a.ld_q = ld_q;
    a.out = out;
    a.ld_out = ld_out;
    a.group = n_heads / c.n_kv;
    // 32 columns where a sequence fills several such tiles (2048 rows of 32 heads of 128:
    // 87 us, 92 with 16; 8 rows of 32 over 8 heads, 2000 tokens: 24 and 20); head dim 256
    // has no registers for them
    const bool wide = c.head_dim < 256 && (long)b.n_rows * a.group > 128L * b.n_seqs;
    a.tokens = b.row_starts ? (wide ? 32 : 16) / a.group : 1;
    a.tiles = b.row_starts ? a.c.n_rows / a.tokens + a.c.n_seqs : a.c.n_rows;
    a.scale = scale;
    a.window = window;
    a.cols = a.tokens * a.group;
    // chunks of the longest row
    // (of a window, the first and the last are parts)
    int64_t chunks = b.max_len > 0 ? std::min(b.max_len, a.c.cap) : a.c.cap;
    if (window > 0) chunks = std::min<int64_t>(chunks, (int64_t)window + a.tokens + 31);
    chunks = (chunks + 31) / 32;
    const long units = (long)a.tiles * c.n_kv;
    ATLAS_REQUIRE(units <= 1 << 23, "kv4_attention: %d tiles of rows and %d KV heads", a.tiles, c.n_kv);
    // Working blocks: two to a CU for a single sequence.  Of sequences of different
    // lengths the longest get up to twice an even share of runs; the blocks beyond the
    // others' runs come and go between the working ones, and these then fill about 5/8
    // of the places before some of them have to wait.  (24 sequences of up to 8191 tokens,
    // heads 32/8 of 64: 23.8 us with 9/4 to a CU, 25.9 with 2, 28.9 with 11/4; of 128: 36 with
    // 15/8, 41 with 3/2, 36.5 with 21/8; up to 4000 tokens, heads 16/8 of 256: 33 with 3/2, 38 with
    // 1, 40 with 2.  Of 64 for 64 sequences of up to 8000 tokens 50 with 3 and 67 with
    // 9/4, which cut only the longest ones.)  A tile has up to 32 runs, or as
    // many as keep a run to 128 chunks, 64 at most (262144 tokens, and from there longer runs);
    // 256 MB of partial sums.  So one sequence of 1, 2 or 4 KV heads works with 32, 64 or 128 blocks
    // whatever its length: 32768 tokens of 128 take 18.5, 18.6 and 17.3 us, and of 32 heads 30.
    // Runs are joined in 3 to 8 us, by the columns: up to 32 chunks are one run and
    // longer ones have 16 at least (900 tokens, 9 heads of 64 over 3: 9.3 us, 10.3 in runs
    // of 16; 8 rows of 32 over 8 of 128: 16.7 and 20.4; 2000 tokens of the former: 12.4 in
    // runs of 32, 10.1 of 16, 9.7 of 8; 300 tokens: 6.8 and, in runs of 8, 9.4); half of
    // both at head dim 256, where a chunk takes twice as long.
    const int cus = device_cu_count();
    const int eighths = b.n_seqs == 1 ? 16 : wide || c.head_dim == 256 ? 12 : c.head_dim == 128 ? 15 : units > cus ? 24 : 18;
    a.blocks = cus * eighths / 8;
    a.min_run = c.head_dim == 256 ? 8 : 16;
    const size_t each = (size_t)units * a.cols * (c.head_dim + 2) * sizeof(float);
    const long want = std::max<long>(a.blocks * (b.n_seqs > 1 ? 2L : 1L) / units, (chunks + 127) / 128);
    const long most = std::min<long>({std::max<long>(32L, (chunks + 127) / 128), 64L, (long)((chunks + a.min_run - 1) / a.min_run),
                                      (long)((256u << 20) / each)});
    a.splits = chunks <= 2 * a.min_run ? 1 : (int)std::max(1L, std::min(want, most));
    if (a.splits > 1) {
        const size_t n = (size_t)units * a.splits * a.cols;
        void *p = nullptr, *cnt = nullptr;
        if ((rc = thread_scratch(SCR_KV4_CNT, (size_t)units * sizeof(int), &cnt, true))) return rc;
        if ((rc = thread_scratch(SCR_KV4, each * a.splits, &p))) return rc;
        a.counters = static_cast<int*>(cnt);
        a.part_o = static_cast<float*>(p);
        a.part_ml = a.part_o + n * c.head_dim;
    }
    const dim3 grid((unsigned)((units + 7) / 8 * 8), a.splits);
#define KV4_RUN(HD, CT) hipLaunchKernelGGL((kv4_attention_kernel<HD, CT>), grid, dim3(kKv4Waves * 64), 0, st, a)
    if (c.head_dim == 64 && wide) KV4_RUN(64, 2);
    else if (c.head_dim == 64) KV4_RUN(64, 1);
    else if (c.head_dim == 128 && wide) KV4_RUN(128, 2);
    else if (c.head_dim == 128) KV4_RUN(128, 1);
    else KV4_RUN(256, 1);
#undef KV4_RUN
    ATLAS_LAUNCH_CHECK("kv4_attention");
    return ATLAS_OK;
}

}  // namespace atlas
