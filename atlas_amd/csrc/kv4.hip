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

// A thread has 8 elements of a row of K (blockIdx.z 0) or V; four lanes a block.
template <int HD>
__global__ __launch_bounds__(256) void kv4_write_kernel(Kv4Args a, const float* __restrict__ k,
                                                        const float* __restrict__ v, long ld) {
    typedef Kv4Layout<HD> L;
    const int row = blockIdx.x, e = (blockIdx.y * 256 + threadIdx.x) * 8;
    if (e >= a.n_kv * HD) return;                        // whole quads: n_kv * HD is a multiple of 32
    int s, pos;
    if (!kv4_row(a, row, s, pos)) return;
    const int page = kv4_page(a, s, pos);
    if (page < 0) return;
    const f32x4* src = reinterpret_cast<const f32x4*>((blockIdx.z ? v : k) + row * ld + e);
    const f32x4 p = src[0], q = src[1];
    const float x[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
    float mx = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = fmaxf(mx, mx_mag(x[i]));
    const int byte = mx_byte(quad_max(mx));
    const uint32_t code = mx_encode8(x, byte);
    const int plen = 1 << a.page_shift, head = e / HD, d = e % HD, at = pos & (plen - 1);
    uint8_t* base = a.cache + ((long)page * a.n_kv + head) * L::bytes(plen);
    const long sc = (long)(at >> 3) * (L::KB * 8) + (d / 32) * 8 + (at & 7);
    if (blockIdx.z == 0) {
        *reinterpret_cast<uint32_t*>(base + (long)at * (HD / 2) + d / 2) = code;
        if (d % 32 == 0) base[L::k_scales(plen) + sc] = (uint8_t)byte;
    } else {
        // group of HD / 16 elements, [token % 8][KB bytes]
        uint8_t* to = base + L::v_codes(plen) + (long)(at >> 3) * (HD * 4) + (d / (HD / 16)) * (8 * L::KB) + (at & 7) * L::KB;
        if constexpr (HD == 64) {
            *reinterpret_cast<uint16_t*>(to) = (uint16_t)code;
            *reinterpret_cast<uint16_t*>(to + 8 * L::KB) = (uint16_t)(code >> 16);
        } else {
            *reinterpret_cast<uint32_t*>(to + (d % (HD / 16)) / 2) = code;
        }
        if (d % 32 == 0) base[L::v_scales(plen) + sc] = (uint8_t)byte;
    }
}

template <int HD>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4Args a, float* __restrict__ k, float* __restrict__ v,
                                                       long ld) {
    typedef Kv4Layout<HD> L;
    const int row = blockIdx.x, e = (blockIdx.y * 256 + threadIdx.x) * 8;
    if (e >= a.n_kv * HD) return;
    int s, pos;
    if (!kv4_row(a, row, s, pos)) return;
    const int page = kv4_page(a, s, pos);
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (page >= 0) {
        const int plen = 1 << a.page_shift, head = e / HD, d = e % HD, at = pos & (plen - 1);
        const uint8_t* base = a.cache + ((long)page * a.n_kv + head) * L::bytes(plen);
        const long sc = (long)(at >> 3) * (L::KB * 8) + (d / 32) * 8 + (at & 7);
        uint32_t code;
        int byte;
        if (blockIdx.z == 0) {
            code = *reinterpret_cast<const uint32_t*>(base + (long)at * (HD / 2) + d / 2);
            byte = base[L::k_scales(plen) + sc];
        } else {
            const uint8_t* from = base + L::v_codes(plen) + (long)(at >> 3) * (HD * 4) + (d / (HD / 16)) * (8 * L::KB) + (at & 7) * L::KB;
            if constexpr (HD == 64)
                code = *reinterpret_cast<const uint16_t*>(from) |
                       (uint32_t) * reinterpret_cast<const uint16_t*>(from + 8 * L::KB) << 16;
            else
                code = *reinterpret_cast<const uint32_t*>(from + (d % (HD / 16)) / 2);
            byte = base[L::v_scales(plen) + sc];
        }
        mx_decode8(code, mx_scale(byte), x);
    }
    f32x4* to = reinterpret_cast<f32x4*>((blockIdx.z ? v : k) + row * ld + e);
    to[0] = f32x4{x[0], x[1], x[2], x[3]};
    to[1] = f32x4{x[4], x[5], x[6], x[7]};
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
// remainder in units 8 times smaller.  7 parts leave 2^-20 of the block's largest
// value.  Products of two E2M1 numbers and their sums of 128 are exact in this
// instruction.  (With E4M3 parts, 5 for the same 20 bits, it drops the low bits of
// products far below the largest one: 4e-6 of a sum for normal q, against none.)
// P in three parts: its 24 bits.  (Two leave 2^-16 of each p, 2.6e-6 of an output
// where f32 sums leave 1e-6, and take a third of the P V instructions less.)
// The maximum is raised only when a score passes it by more than 2^8 (p then
// stays below 2^8, far from any overflow); most chunks need no rescaling.

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
    float *part_o, *part_ml;
};

// E2M1 parts of q: the operands of N matrix instructions and their scale bytes.
// HD 64: an instruction's 128 is two parts of the 64 (K's blocks given twice).
// HD 256: part p's two halves are instructions 2p and 2p + 1.
template <int HD>
struct Kv4Query {
    static constexpr int PARTS = HD == 64 ? 8 : 7;
    static constexpr int N = HD == 64 ? 4 : HD == 128 ? 7 : 14;
    u32x4 q[N];
    int byte[N];

    // the column's row of q times scale; lane group g has block g
    // of an instruction's four
    __device__ __forceinline__ void load(const float* row, float scale, int g) {
        constexpr int H = HD == 256 ? 2 : 1;
        const int blk = HD == 64 ? g & 1 : g;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            float x[32], mx = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(row + h * 128 + blk * 32 + j * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[4 * j + i] = v[i] * scale;
                    mx = fmaxf(mx, mx_mag(x[4 * j + i]));
                }
            }
            const int e = (int)(__float_as_uint(mx) >> 23), top = max(e - 1, 0);
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                const int b = max(top - 3 * p, 0);
                const u32x4 w = part(x, mx_scale(b));
                const int f = HD == 64 ? p / 2 : HD == 128 ? p : 2 * p + h;
                if (HD != 64 || (p & 1) == 0) {
                    q[f] = w;
                    byte[f] = b;
                } else if (g >= 2) {
                    q[f] = w;
                    byte[f] = b;
                }
            }
            if (e == 255) byte[HD == 256 ? h : 0] = kMxNan;    // an infinity or NaN: so is every score
        }
    }

    // x rounded to E2M1; x keeps the rest
    __device__ __forceinline__ static u32x4 part(float (&x)[32], float scale) {
        u32x4 to;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            uint32_t w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[8 * d], x[8 * d + 1], scale, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[8 * d + 2], x[8 * d + 3], scale, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[8 * d + 4], x[8 * d + 5], scale, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[8 * d + 6], x[8 * d + 7], scale, 3);
            float y[8];
            mx_decode8(w, scale, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[8 * d + i] -= y[i];
            to[d] = w;
        }
        return to;
    }
};

// a chunk's bytes in the registers of a wave
template <int HD>
struct Kv4Chunk {
    typedef Kv4Layout<HD> L;
    static constexpr int H = HD == 256 ? 2 : 1;          // K steps of 128 elements
    static constexpr int VW = HD / 64 * 4;               // dwords of V
    u32x4 k[H][2];                                       // [step][part t]
    uint16_t ks[H];                                      // scale bytes of parts 0 and 1
    uint32_t v[VW];
    u32x2 vs;

    // base: the (page, head)'s bytes; at: the chunk's first token in the page
    __device__ __forceinline__ void load(const uint8_t* base, int at, int plen, int lane) {
        const int i = lane & 15, g = lane >> 4;
        const uint8_t* kp = base + (long)at * (HD / 2);
        const uint8_t* ksp = base + L::k_scales(plen) + at * L::KB;
        const uint8_t* vp = base + L::v_codes(plen) + (long)at * (HD / 2);
        const uint8_t* vsp = base + L::v_scales(plen) + at * L::KB;
        const int blk = HD == 64 ? g & 1 : g;
#pragma unroll
        for (int h = 0; h < H; ++h) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
                k[h][t] = *reinterpret_cast<const u32x4*>(kp + (2 * i + t) * (HD / 2) + h * 64 + blk * 16);
            ks[h] = *reinterpret_cast<const uint16_t*>(ksp + (i >> 2) * (8 * L::KB) + (4 * h + blk) * 8 + 2 * (i & 3));
        }
#pragma unroll
        for (int w = 0; w < VW / 4; ++w) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(vp + (g * 16 + i) * (8 * L::KB) + 16 * w);
            v[4 * w] = x.x; v[4 * w + 1] = x.y; v[4 * w + 2] = x.z; v[4 * w + 3] = x.w;
        }
        vs = *reinterpret_cast<const u32x2*>(vsp + (g * L::KB + i * (HD / 16) / 32) * 8);
    }
};

// Blocks of V that read as NaN (scale bytes past kMxMaxByte), found in sc, the
// scale bytes of the lane's eight tokens: returns sc without those bytes, so that
// the product leaves the columns that do not see their tokens as they were, and
// in z the rows 4g + r of O^T (bit r) that have to be NaN in the lane's column,
// which sees [from, to].  Rare, so its loops stay rolled.
template <int HD>
__device__ __forceinline__ u32x4 kv4_nan_blocks(uint32_t s0, uint32_t s1, int first, int from, int to) {
    constexpr int KB = HD / 32;
    const int g = (threadIdx.x & 63) >> 4;
    uint32_t rows = 0;
#pragma unroll 1
    for (int b = 0; b < KB; ++b)
#pragma unroll 1
        for (int j = 0; j < 32; ++j) {
            // lane (j / 8, first group of block b) has token j's byte
            const int lane = (j >> 3) * 16 + b * (16 / KB);
            const uint32_t w0 = __shfl(s0, lane, 64), w1 = __shfl(s1, lane, 64);
            const uint32_t byte = ((j & 4 ? w1 : w0) >> (8 * (j & 3))) & 255u;
            const int key = first + j;
            if ((int)byte <= kMxMaxByte || key < from || key > to) continue;
            for (int r = 0; r < 4; ++r)
                if ((4 * g + r) * (HD / 16) / 32 == b) rows |= 1u << r;
        }
    for (int j = 0; j < 4; ++j) {
        if ((int)((s0 >> (8 * j)) & 255u) > kMxMaxByte) s0 &= ~(255u << (8 * j));
        if ((int)((s1 >> (8 * j)) & 255u) > kMxMaxByte) s1 &= ~(255u << (8 * j));
    }
    return u32x4{s0, s1, rows, 0u};
}

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

    // V's code dword and byte of elements 2e, 2e+1 of token j
    template <int J8, int E>
    __device__ __forceinline__ static uint32_t v_pair(const Kv4Chunk<HD>& c, float s) {
        constexpr int at = J8 * (HD / 32) + E;
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c.v[at / 4], s, at % 4));
    }

    template <int E>
    __device__ __forceinline__ void pv(const Kv4Chunk<HD>& c, const float (&s)[8], const bf16x8 (&p)[3]) {
        const uint32_t w[8] = {v_pair<0, E>(c, s[0]), v_pair<1, E>(c, s[1]), v_pair<2, E>(c, s[2]), v_pair<3, E>(c, s[3]),
                               v_pair<4, E>(c, s[4]), v_pair<5, E>(c, s[5]), v_pair<6, E>(c, s[6]), v_pair<7, E>(c, s[7])};
        u32x4 even, odd;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            even[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x05040100u);
            odd[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x07060302u);
        }
        const bf16x8 a = __builtin_bit_cast(bf16x8, even), b = __builtin_bit_cast(bf16x8, odd);
#pragma unroll
        for (int j = 2; j >= 0; --j) {
            o[2 * E] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, p[j], o[2 * E], 0, 0, 0);
            o[2 * E + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, p[j], o[2 * E + 1], 0, 0, 0);
        }
    }

    // A chunk's tokens first .. first + 31.  masked: not every column sees all of
    // them; the lane's column sees [from, to].  live: tokens of the chunk that
    // the sequence has (the bytes of others are not looked at).
    __device__ __forceinline__ void add(Kv4Chunk<HD>& c, const Kv4Query<HD>& q, int first, bool masked, int from,
                                        int to, int live, int lane) {
        const int g = lane >> 4;
        f32x4 d[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int f = Kv4Query<HD>::N - 1; f >= 0; --f) {
            const int h = HD == 256 ? f & 1 : 0;
            // (the argument before a scale picks its byte)
            d[0] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_frag(c.k[h][0]), mx_frag(q.q[f]), d[0], kFp4, kFp4, 0,
                                                                    c.ks[h], 0, q.byte[f]);
            d[1] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_frag(c.k[h][1]), mx_frag(q.q[f]), d[1], kFp4, kFp4, 1,
                                                                    c.ks[h], 0, q.byte[f]);
        }
        float s[8];                                      // token first + 8 g + j
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = d[j & 1][j >> 1];
        if (masked) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = first + 8 * g + j;
                if (key < from || key > to) s[j] = -__builtin_inff();
            }
        }
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
        u32x4 part[3];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a = __builtin_amdgcn_exp2f(s[2 * j] - m), b = __builtin_amdgcn_exp2f(s[2 * j + 1] - m);
            l += a + b;
            part[0][j] = bf16_rne2(a, b);
            a -= bf16_lo(part[0][j]);
            b -= bf16_hi(part[0][j]);
            part[1][j] = bf16_rne2(a, b);
            part[2][j] = bf16_rne2(a - bf16_lo(part[1][j]), b - bf16_hi(part[1][j]));
        }
        // tokens that are not there get the smallest scale: their p is zero, and
        // whatever their bytes are the product is too
        uint32_t sc[2] = {c.vs.x, c.vs.y};
        if (live < 32) {
            const int n = min(max(live - 8 * g, 0), 8);
            sc[0] &= n >= 4 ? ~0u : (1u << (8 * n)) - 1u;
            sc[1] &= n >= 8 ? ~0u : n <= 4 ? 0u : (1u << (8 * (n - 4))) - 1u;
        }
        const uint32_t bad = (((~sc[0] - 0x03030303u) & sc[0]) | ((~sc[1] - 0x03030303u) & sc[1])) & 0x80808080u;
        if (__any(bad != 0)) {
            const u32x4 x = kv4_nan_blocks<HD>(sc[0], sc[1], first, from, to);
            sc[0] = x.x;
            sc[1] = x.y;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (x.z >> r & 1u)
#pragma unroll
                    for (int j = 0; j < J; ++j) o[j][r] = __builtin_nanf("");
        }
        float vsc[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) vsc[j] = mx_scale((sc[j >> 2] >> (8 * (j & 3))) & 255u);
        const bf16x8 p[3] = {__builtin_bit_cast(bf16x8, part[0]), __builtin_bit_cast(bf16x8, part[1]),
                             __builtin_bit_cast(bf16x8, part[2])};
        pv<0>(c, vsc, p);
        pv<1>(c, vsc, p);
        if constexpr (HD >= 128) {
            pv<2>(c, vsc, p);
            pv<3>(c, vsc, p);
        }
        if constexpr (HD >= 256) {
            pv<4>(c, vsc, p);
            pv<5>(c, vsc, p);
            pv<6>(c, vsc, p);
            pv<7>(c, vsc, p);
        }
    }
};

// The tile u of a batch: its sequence, first row and rows; false: none.  Tiles
// of sequence s begin at starts[s] / tokens + s, which leaves each sequence as
// many as it needs, whatever the lengths.
__device__ __forceinline__ bool kv4_tile(const Kv4AttnArgs& a, int u, int& s, int& row, int& rows, int& pos) {
    if (!a.c.starts) {
        s = row = u;
        rows = 1;
        pos = max(a.c.lens[u], 0) - 1;
        return true;
    }
    int lo = 0, hi = a.c.n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.c.starts[mid] / a.tokens + mid <= u) lo = mid;
        else hi = mid;
    }
    s = lo;
    const int begin = max(a.c.starts[lo], 0), end = min(a.c.starts[lo + 1], a.c.n_rows);
    const int skip = (u - (begin / a.tokens + lo)) * a.tokens;
    if (skip < 0 || skip >= end - begin) return false;
    row = begin + skip;
    rows = min(a.tokens, end - row);
    pos = max(a.c.lens[lo], 0) - (end - row);
    return true;
}

// A tile's work: its rows, the lane's column, the chunks that any column sees.
template <int HD>
struct Kv4Tile {
    int s, row0, rows, pos0;
    int first, last;                    // chunks [first, last)
    int tokens_end;                     // tokens from here on are seen by no column
    bool mine;                          // the lane's column is one (others repeat the last row)
    int t, from, to;                    // its row of the tile; it sees tokens [from, to]
    long head;

    __device__ __forceinline__ bool set(const Kv4AttnArgs& a, int u, int kvh, int lane) {
        if (!kv4_tile(a, u, s, row0, rows, pos0)) return false;
        const int i = lane & 15;
        t = i / a.group;
        head = (long)kvh * a.group + (i - t * a.group);
        mine = t < rows;
        t = min(t, rows - 1);
        to = pos0 + t;
        from = seen_from(a, to);
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

    // The bytes of a chunk's page and head, or null: no page.  (Uniform.)
    __device__ __forceinline__ const uint8_t* base(const Kv4AttnArgs& a, int chunk, int kvh) const {
        const int page = a.c.table[(long)s * a.c.table_stride + (chunk * 32 >> a.c.page_shift)];
        if (page < 0 || page >= a.c.n_pages) return nullptr;
        return a.c.cache + ((long)page * a.c.n_kv + kvh) * Kv4Layout<HD>::bytes(1 << a.c.page_shift);
    }
};

// Chunks begin, begin + step, .. below end into st, each one's bytes loaded while
// the one before is worked on.
template <int HD>
__device__ __forceinline__ void kv4_scan(const Kv4AttnArgs& a, const Kv4Tile<HD>& tile, int kvh, int begin, int end, int step,
                                         const float* row, Kv4State<HD>& st, int lane) {
    const int plen = 1 << a.c.page_shift;
    Kv4Chunk<HD> c[2];
    bool there[2] = {false, false};
    const auto fetch = [&](int chunk, int b) {
        there[b] = false;
        if (chunk >= end) return;
        const uint8_t* base = tile.base(a, chunk, kvh);
        there[b] = base != nullptr;
        if (base) c[b].load(base, chunk * 32 & (plen - 1), plen, lane);
    };
    fetch(begin, 0);
    Kv4Query<HD> q;
    q.load(row, a.scale * kLog2e, lane >> 4);
    st.clear();
    for (int chunk = begin; chunk < end; chunk += 2 * step)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int at = chunk + b * step;
            fetch(at + step, b ^ 1);
            if (there[b])
                st.add(c[b], q, at * 32, tile.masked(a, at), tile.from, tile.to, tile.tokens_end - at * 32, lane);
        }
    st.l += __shfl_xor(st.l, 16, 64);
    st.l += __shfl_xor(st.l, 32, 64);
}

// block -> (tile, KV head): consecutive blocks run on different XCDs, so each takes
// a run of the heads' tiles and its L2 the heads' tokens
__device__ __forceinline__ bool kv4_place(int block, int tiles, int n_kv, int& u, int& kvh) {
    const int per = (tiles * n_kv + 7) / 8, at = (block & 7) * per + (block >> 3);
    if ((block >> 3) >= per || at >= tiles * n_kv) return false;
    kvh = at / tiles;
    u = at - kvh * tiles;
    return true;
}

// Prompts: a tile and KV head to a wave, the last tiles (the longest) first.
template <int HD>
__global__ __launch_bounds__(64) void kv4_attention_kernel(Kv4AttnArgs a) {
    const int lane = threadIdx.x, g = lane >> 4;
    int u, kvh;
    if (!kv4_place(blockIdx.x, a.tiles, a.c.n_kv, u, kvh)) return;
    Kv4Tile<HD> tile;
    if (!tile.set(a, a.tiles - 1 - u, kvh, lane)) return;
    Kv4State<HD> st;
    const float* row = a.q + (tile.row0 + tile.t) * a.ld_q + tile.head * HD;
    kv4_scan<HD>(a, tile, kvh, tile.first, tile.last, 1, row, st, lane);
    if (!tile.mine) return;
    const float inv = st.l == 0.f ? 0.f : 1.f / st.l;    // a row that has seen nothing is zero
    float* o = a.out + (tile.row0 + tile.t) * a.ld_out + tile.head * HD;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < Kv4State<HD>::J; j += 4)
            *reinterpret_cast<f32x4*>(o + (4 * g + r) * (HD / 16) + j) =
                f32x4{st.o[j][r] * inv, st.o[j + 1][r] * inv, st.o[j + 2][r] * inv, st.o[j + 3][r] * inv};
}

// Few tiles: a tile's chunks are split over up to a.splits blocks of WAVES waves, in
// runs of the same length for every tile.  A block's waves take every WAVES-th chunk
// of its run and join their sums in LDS; the blocks' meet in kv4_join_kernel.
constexpr int kKv4Waves = 4;
constexpr int kKv4MinRun = 2 * kKv4Waves;               // chunks of a block, where a tile has more

// The run's length: what the batch's chunks, as its lengths are now, come to over
// a.blocks blocks; no tile has more than a.splits runs.  (Every lane of a wave
// takes part.)
__device__ __forceinline__ int kv4_run(const Kv4AttnArgs& a, int lane) {
    int all = 0, most = 0;
    for (int s = lane; s < a.c.n_seqs; s += 64) {
        const int n = min(max(a.c.lens[s], 0), a.c.cap);
        int tiles = 1, tokens = n;
        if (a.c.starts) {
            const int rows = a.c.starts[s + 1] - a.c.starts[s];
            tiles = rows <= 0 ? 0 : min((rows + a.tokens - 1) / a.tokens, a.tiles);
        }
        if (a.window > 0 && tokens - a.tokens > a.window) tokens = a.window + a.tokens;
        const int chunks = tiles ? (tokens + 62) >> 5 : 0;
        all += min(tiles * (long)chunks, 1L << 24);
        most = max(most, chunks);
    }
    // (sums of up to 2^20 sequences stay below 2^31 as far as it matters: a longer run is still right)
    for (int o = 32; o >= 1; o >>= 1) {
        all = min(all, 1 << 29) + min(__shfl_xor(all, o, 64), 1 << 29);
        most = max(most, __shfl_xor(most, o, 64));
    }
    const long run = ((long)all * a.c.n_kv + a.blocks - 1) / a.blocks;
    const int n = max(max((int)min(run, 1L << 26), kKv4MinRun), (most + a.splits - 1) / a.splits);
    return __builtin_amdgcn_readfirstlane(n);
}

template <int HD>
__global__ __launch_bounds__(kKv4Waves * 64) void kv4_attention_split_kernel(Kv4AttnArgs a) {
    __shared__ float part_o[kKv4Waves][16][HD + 4];
    __shared__ float part_m[kKv4Waves][16], part_l[kKv4Waves][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4, u = blockIdx.x, kvh = blockIdx.y, split = blockIdx.z;
    Kv4Tile<HD> tile;
    if (!tile.set(a, u, kvh, lane)) return;
    const int run = kv4_run(a, lane), begin = tile.first + split * run;
    if (split > 0 && begin >= tile.last) return;
    const bool alone = tile.first + run >= tile.last;
    Kv4State<HD> st;
    const float* row = a.q + (tile.row0 + tile.t) * a.ld_q + tile.head * HD;
    kv4_scan<HD>(a, tile, kvh, begin + wave, min(begin + run, tile.last), kKv4Waves, row, st, lane);
    if (tile.mine) {
        if (g == 0) {
            part_m[wave][i] = st.m;
            part_l[wave][i] = st.l;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < Kv4State<HD>::J; j += 4)
                *reinterpret_cast<f32x4*>(&part_o[wave][i][(4 * g + r) * (HD / 16) + j]) =
                    f32x4{st.o[j][r], st.o[j + 1][r], st.o[j + 2][r], st.o[j + 3][r]};
    }
    __syncthreads();
    // four elements of a column to a thread
    const int cols = tile.rows * a.group;
    for (int e = threadIdx.x; e < cols * (HD / 4); e += kKv4Waves * 64) {
        const int c = e / (HD / 4), d = e % (HD / 4) * 4;
        float m = part_m[0][c];
#pragma unroll
        for (int w = 1; w < kKv4Waves; ++w) m = fmaxf(m, part_m[w][c]);
        float l = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kKv4Waves; ++w) {
            const float f = __builtin_amdgcn_exp2f(part_m[w][c] - m);
            l += f * part_l[w][c];
            o += f * *reinterpret_cast<const f32x4*>(&part_o[w][c][d]);
        }
        if (alone) {
            const int t = c / a.group;
            float* to = a.out + (tile.row0 + t) * a.ld_out + ((long)kvh * a.group + c - t * a.group) * HD + d;
            *reinterpret_cast<f32x4*>(to) = o * (l == 0.f ? 0.f : 1.f / l);
        } else {
            const long at = (((long)u * a.c.n_kv + kvh) * a.splits + split) * a.cols + c;
            *reinterpret_cast<f32x4*>(a.part_o + at * HD + d) = o;
            if (d == 0) {
                a.part_ml[2 * at] = m;
                a.part_ml[2 * at + 1] = l;
            }
        }
    }
}

// Joins a tile's runs: a wave to a column, four of its elements to a lane; the
// lanes beyond take other runs (HD 64: every fourth, 128: every second).
template <int HD>
__global__ __launch_bounds__(64) void kv4_join_kernel(Kv4AttnArgs a) {
    constexpr int E = HD / 4, G = 64 / E;
    const int lane = threadIdx.x, u = blockIdx.x / a.cols, c = blockIdx.x % a.cols, kvh = blockIdx.y, d = lane % E * 4;
    Kv4Tile<HD> tile;
    if (!tile.set(a, u, kvh, 0)) return;
    const int run = kv4_run(a, lane), n = (tile.last - tile.first + run - 1) / run;
    if (n <= 1 || c >= tile.rows * a.group) return;
    const long at = (((long)u * a.c.n_kv + kvh) * a.splits) * a.cols + c;
    // lane s has run s (at most 64 of them)
    float m = kKv4Floor, l = 0.f;
    if (lane < n) {
        m = a.part_ml[2 * (at + (long)lane * a.cols)];
        l = a.part_ml[2 * (at + (long)lane * a.cols) + 1];
    }
    const float f = __builtin_amdgcn_exp2f(m - wave_max(m));
    l = wave_sum(f * l);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = 0; s < n; s += G) {
        const int r = s + lane / E;
        const float w = __shfl(f, r, 64);
        if (r < n) o += w * *reinterpret_cast<const f32x4*>(a.part_o + (at + (long)r * a.cols) * HD + d);
    }
    for (int x = E; x < 64; x <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], x, 64);
    if (lane >= E) return;
    const int t = c / a.group;
    float* to = a.out + (tile.row0 + t) * a.ld_out + ((long)kvh * a.group + c - t * a.group) * HD + d;
    *reinterpret_cast<f32x4*>(to) = o * (l == 0.f ? 0.f : 1.f / l);
}

// ---- launches ---------------------------------------------------------------------

static int kv4_check(const char* who, const atlas_kv4_cache& c) {
    ATLAS_REQUIRE(c.head_dim == 64 || c.head_dim == 128 || c.head_dim == 256, "%s: head_dim %d (64, 128 or 256)", who,
                  c.head_dim);
    ATLAS_REQUIRE(c.page_len >= 32 && c.page_len <= 1 << 24 && (c.page_len & (c.page_len - 1)) == 0,
                  "%s: page_len %d (a power of two from 32 to 2^24)", who, c.page_len);
    ATLAS_REQUIRE(c.n_pages >= 0 && c.n_kv > 0 && c.n_kv <= 4096, "%s: %d pages, %d KV heads", who, c.n_pages, c.n_kv);
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
    const dim3 grid(a.n_rows, (unsigned)((wide + 2047) / 2048), 2);
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
    const dim3 grid(a.n_rows, (unsigned)((wide + 2047) / 2048), 2);
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
    const long wide = (long)n_heads * c.head_dim;
    if ((rc = kv4_rows_check("kv4_attention", q, q, ld_q, wide))) return rc;
    if ((rc = kv4_rows_check("kv4_attention", out, out, ld_out, wide))) return rc;
    a.q = q;
    a.ld_q = ld_q;
    a.out = out;
    a.ld_out = ld_out;
    a.group = n_heads / c.n_kv;
    a.tokens = b.row_starts ? 16 / a.group : 1;
    a.tiles = b.row_starts ? a.c.n_rows / a.tokens + a.c.n_seqs : a.c.n_rows;
    a.scale = scale;
    a.window = window;
    a.cols = a.tokens * a.group;
    // chunks of the longest row
    int64_t chunks = b.max_len > 0 ? std::min(b.max_len, a.c.cap) : a.c.cap;
    if (window > 0) chunks = std::min<int64_t>(chunks, (int64_t)window + a.tokens);
    chunks = (chunks + 62) / 32;
    const long units = (long)a.tiles * c.n_kv;
    ATLAS_REQUIRE(units <= 1 << 25, "kv4_attention: %d tiles of rows and %d KV heads", a.tiles, c.n_kv);
    const int cus = device_cu_count();
    // Eight waves to a CU without splitting: only few rows to a sequence, whose
    // lengths may differ, are split further, where one may be long.
    if (units >= 8L * cus && (chunks <= 128 || b.n_rows >= 2 * b.n_seqs)) {
        const dim3 grid((unsigned)((units + 7) / 8 * 8));
        if (c.head_dim == 64) hipLaunchKernelGGL(kv4_attention_kernel<64>, grid, dim3(64), 0, st, a);
        else if (c.head_dim == 128) hipLaunchKernelGGL(kv4_attention_kernel<128>, grid, dim3(64), 0, st, a);
        else hipLaunchKernelGGL(kv4_attention_kernel<256>, grid, dim3(64), 0, st, a);
        ATLAS_LAUNCH_CHECK("kv4_attention");
        return ATLAS_OK;
    }
    // As many blocks as run at once (their registers leave 3, 2 or 1 to a CU).  Of
    // sequences of different lengths the longest get up to twice an even share of
    // runs.  At most 128 chunks to a run, 64 runs to a tile, 256 MB of partial sums.
    a.blocks = cus * (c.head_dim == 64 ? 3 : c.head_dim == 128 ? 2 : 1);
    const size_t each = (size_t)units * a.cols * (c.head_dim + 2) * sizeof(float);
    const long want = std::max<long>(a.blocks * (b.n_seqs > 1 ? 2L : 1L) / units, (chunks + 127) / 128);
    const long most = std::min<long>({64L, (long)((chunks + kKv4MinRun - 1) / kKv4MinRun), (long)((256u << 20) / each)});
    a.splits = (int)std::max(1L, std::min(want, most));
    if (a.splits > 1) {
        const size_t n = (size_t)units * a.splits * a.cols;
        void* p = nullptr;
        if ((rc = thread_scratch(SCR_KV4, each * a.splits, &p))) return rc;
        a.part_o = static_cast<float*>(p);
        a.part_ml = a.part_o + n * c.head_dim;
    }
    const dim3 grid(a.tiles, c.n_kv, a.splits), join((unsigned)((long)a.tiles * a.cols), c.n_kv);
#define KV4_SPLIT(HD)                                                                                                 \
    do {                                                                                                              \
        hipLaunchKernelGGL(kv4_attention_split_kernel<HD>, grid, dim3(kKv4Waves * 64), 0, st, a);                     \
        if (a.splits > 1) hipLaunchKernelGGL(kv4_join_kernel<HD>, join, dim3(64), 0, st, a);                          \
    } while (0)
    if (c.head_dim == 64) KV4_SPLIT(64);
    else if (c.head_dim == 128) KV4_SPLIT(128);
    else KV4_SPLIT(256);
#undef KV4_SPLIT
    ATLAS_LAUNCH_CHECK("kv4_attention");
    return ATLAS_OK;
}

}  // namespace atlas
