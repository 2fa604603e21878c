// mxfp4.hpp -- MXFP4 (E2M1 elements in blocks of 32 with an E8M0 scale byte)
// on gfx950, and the launch interfaces of its matrix and cache kernels.
//
// A block of values v with largest magnitude a is stored as a byte b and 32
// codes: b = max(e(a) - 2, 0), e the exponent field of a as an f32, so that
// a 2^(127 - b) lies in [4, 8) (below 4 for a < 2^-124); code = v 2^(127 - b)
// rounded to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 (ties to the even code),
// at most 6, with the sign in bit 3.  A block of zeros has b = 127; one with an
// infinity or NaN has b = 255 and codes 0, and reads as NaN throughout.  The scaling is by a
// power of two and so exact: host, device and any other implementation of the
// rule agree bit for bit.  Two codes to a byte, the first in the low nibble.
//
// gfx950 converts between f32 and scaled E2M1 in one instruction, with this
// rounding and saturation, for every scale byte; it takes the scale as an f32
// whose exponent field is b.
#pragma once
#include "common.hpp"

namespace atlas {

constexpr int kMxBlock = 32;
constexpr int kMxNan = 255;           // scale byte of a block that reads as NaN
constexpr int kMxMaxByte = 252;       // largest scale byte of a finite block

__device__ __forceinline__ float mx_scale(int byte) { return __uint_as_float((uint32_t)byte << 23); }

// scale byte of a block with largest magnitude amax (NaN: fmaxf drops it, so
// the caller passes infinity for a block that holds one)
__device__ __forceinline__ int mx_byte(float amax) {
    const int e = (int)(__float_as_uint(amax) >> 23);
    if (e == 255) return kMxNan;
    if (amax == 0.f) return 127;
    return e > 2 ? e - 2 : 0;
}

// magnitude for the block maximum: NaN and infinity alike count as infinity
__device__ __forceinline__ float mx_mag(float v) {
    const float a = fabsf(v);
    return a < __builtin_inff() ? a : __builtin_inff();
}

// codes of 8 values at this scale (the first in the low nibble)
__device__ __forceinline__ uint32_t mx_round8(const float (&v)[8], float scale) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
    return w;
}

// ... of a block with this scale byte
__device__ __forceinline__ uint32_t mx_encode8(const float (&v)[8], int byte) {
    const uint32_t w = mx_round8(v, mx_scale(byte));
    return byte == kMxNan ? 0u : w;
}

// values of 8 codes
__device__ __forceinline__ void mx_decode8(uint32_t w, float scale, float (&v)[8]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}

// the largest value of the four lanes of a DPP quad (a block of 32 is 8
// elements in each of them), for non-negative v
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, false)));
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, false)));
    return v;
}

// the operand of a matrix instruction with scales: 32 codes of a lane, in the
// lower half of the registers that its widest format takes
typedef int i32x8 __attribute__((ext_vector_type(8)));
constexpr int kFp4 = 4;               // the instruction's format code of E2M1

__device__ __forceinline__ i32x8 mx_frag(u32x4 v) {
    return i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
}

int mxfp4_quant_launch(const void* src, int src_bf16, long rows, long cols, long ld, uint8_t* data,
                       uint8_t* scales, hipStream_t st);
int mxfp4_dequant_launch(const uint8_t* data, const uint8_t* scales, long rows, long cols, float* out,
                         long ld, hipStream_t st);
int mxfp4_gemm_launch(const uint8_t* w, const uint8_t* ws, const uint8_t* x, const uint8_t* xs, float* y,
                      int m, int n, int k, long ldy, hipStream_t st);

int64_t kv4_cache_bytes(const atlas_kv4_cache& c);
int kv4_write_launch(const atlas_kv4_cache& c, const atlas_kv4_batch& b, const float* k, const float* v,
                     long ld, hipStream_t st);
int kv4_read_launch(const atlas_kv4_cache& c, const atlas_kv4_batch& b, float* k, float* v, long ld,
                    hipStream_t st);
int kv4_attention_launch(const atlas_kv4_cache& c, const atlas_kv4_batch& b, const float* q, long ld_q,
                         int n_heads, float scale, int window, float* out, long ld_out, hipStream_t st);

}  // namespace atlas
