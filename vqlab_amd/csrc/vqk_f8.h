// 8-bit floating point (e4m3, finite: up to 448) with fp32 scales: shared
// declarations of the vqk_f8* sources. Activations have a scale for each block
// of 128 along the row, weights one for each 128 x 128:
//     x[n, k] = x8[n, k] * sx[n, k / 128],   W[o, k] = w8[o, k] * sw[o / 128, k / 128]
//
//   * A block of 128 k is one step of every product here: the codes' sum over
//     the block comes from the matrix cores alone (8 bits by 8 bits as they are,
//     or the codes converted to 16 bits, which is exact), and enters the fp32
//     accumulators by one multiply-add with the block's scales.
//   * The 8-bit matrix instructions align eight neighbouring products to the largest
//     and drop what is below 2^-13 of its power of two (measured; the 16-bit ones keep
//     fp32 sums). N(0, 1) operands come out 1.5e-5 of the result off, operands of one
//     sign 7.7e-5, towards zero. Of the smallest half step of the output's rounding
//     (bf16 2^-9 of the value, fp16 2^-12) the first is 0.8 % and 6 %, the second 4 % and
//     32 %. An fp32 output is computed by the 16-bit instructions, at half the rate.
//   * The sum over k inside a block may be taken in any order, so lane i of an
//     operand owns 32 neighbouring k of a row: 32 bytes.
//   * Weights are laid out once so that every load of a wave is one contiguous KB:
//       codes [RT][NC][2][64][16]  RT = ceil(OUT / 16) row tiles, NC = ceil(IN / 128)
//              unit (lane) i of half h: row 16 rt + i % 16, k = 128 c + 32 (i / 16) + 16 h
//     with codes 0 past the row's and the weight's end.
//   * bf16 products take the codes times 2^-16 and the result times 2^16: a block's
//     sum, at most 2^128 * 448 * 128 / 2^16, then stays finite whatever finite x is.
#pragma once

#include "vqk_gemv.h"
#include "vqk_internal.h"
#include "vqk_mx.h"

namespace vqk {

typedef int f8_i8 __attribute__((ext_vector_type(8)));
typedef float f8_f2 __attribute__((ext_vector_type(2)));

constexpr int kF8Block = 128;
constexpr float kF8Max = 448.f;
constexpr float kF8MinScale = 0x1p-126f;
constexpr float kF8Down = 0x1p-16f, kF8Up = 0x1p16f;      // bf16 products

struct F8Geom { int64_t OUT, IN, RT, NC; };
__host__ __device__ constexpr int64_t f8_code_bytes(int64_t RT, int64_t NC) { return RT * NC * 2048; }
int make_f8_geom(const vqk_f8_weights *w, F8Geom *g, const char *what);

// A block's scale from the bits of its largest magnitude (NaN where that is not
// finite), and the factor its values are multiplied by.
__device__ __forceinline__ float f8_scale(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    return fmaxf(__uint_as_float(amax_bits) / kF8Max, kF8MinScale);
}

// Eight values times inv as codes (ok: the block is finite; otherwise zeros).
__device__ __forceinline__ u32x2 f8_encode8(const float (&v)[8], float inv, bool ok) {
    u32x2 r{};
    if (!ok) return r;
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, hi, true);
    r.x = uint32_t(lo);
    r.y = uint32_t(hi);
    return r;
}

// Eight codes as numbers.
__device__ __forceinline__ void f8_decode8(u32x2 c, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f8_f2 a = __builtin_amdgcn_cvt_pk_f32_fp8(int(c[i]), false), b = __builtin_amdgcn_cvt_pk_f32_fp8(int(c[i]), true);
        v[4 * i] = a.x; v[4 * i + 1] = a.y;
        v[4 * i + 2] = b.x; v[4 * i + 3] = b.y;
    }
}

// Eight codes (two words) as the operand of a 16-bit product.
template <int OP>
__device__ __forceinline__ u32x4 f8_operand(uint32_t a, uint32_t b) {
    u32x4 r;
    if constexpr (OP == kOpBF16) {
        r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, kF8Down, false));
        r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, kF8Down, true));
        r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, kF8Down, false));
        r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, kF8Down, true));
    } else {
        r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, false));
        r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, true));
        r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, false));
        r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, true));
    }
    return r;
}

__device__ __forceinline__ f8_i8 f8_pair(u32x4 a, u32x4 b) {
    f8_i8 r;
    r[0] = int(a.x); r[1] = int(a.y); r[2] = int(a.z); r[3] = int(a.w);
    r[4] = int(b.x); r[5] = int(b.y); r[6] = int(b.z); r[7] = int(b.w);
    return r;
}

// 16 weight rows by 16 x rows, a whole block of 128 k of 8-bit codes.
__device__ __forceinline__ f32x4 f8_mma16(f8_i8 w, f8_i8 x) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, f32x4{}, 0, 0, 0, 0, 0, 0);
}

// Largest value over each aligned group of 16 lanes, in every lane of it.
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
    v = quad_max(v);
    v = max(v, dpp_u<kDppRowHalfMirror>(v));
    return max(v, dpp_u<kDppRowMirror>(v));
}

// Rows x [N, C] (ldx apart) -> codes [N][ldc] and scales at n * sn + b * sk, of
// ceil(C / 128) blocks; columns from C up to `cover` are codes 0.
struct F8Quant {
    const void *x;
    int64_t N, C, ldx;
    uint8_t *codes;
    int64_t ldc, cover;
    float *scales;
    int64_t sn, sk;
};
int launch_f8_quant(const F8Quant &q, int32_t type, hipStream_t st);

// x of a product with 8-bit rows: whole blocks of codes, ld apart (a multiple
// of 16), 16-byte aligned; the scale of row n, block b at n * sn + b * sk.
struct F8X {
    const uint8_t *codes;
    int64_t ld;
    const float *scales;
    int64_t sn, sk;
};

// One product y [N, OUT] = x . W^T. swo / swk: floats between the scales of
// neighbouring blocks of OUT / of IN.
struct F8Call {
    const uint8_t *codes;
    const float *scales;
    int64_t swo, swk;
    F8Geom g;
    int64_t N;
    bool a8;                                  // 8-bit x on the 8-bit instructions
    F8X x8;                                   // a8: all; otherwise scales (NULL: none) of x's rows
    MxX x;                                    // otherwise: op, planes (kOpF16, scales: one); f8_tiles: whole blocks
    void *y;
    int32_t y_type;
};

// Few rows (vqk_f8s.h): whether it takes a call, and its launch.
// part: room for the sums of ranges of k, f8_rows_part bytes.
bool f8_rows_ok(const F8Call &c);
size_t f8_rows_part(const F8Call &c);
int f8_rows(const F8Call &c, float *part, size_t part_bytes, hipStream_t st);
// Many rows (vqk_f8t.h). part: room for the K slices of the last tiles, f8_tiles_part
// bytes (scaled: 16-bit x with scales).
size_t f8_tiles_part(int64_t N, const F8Geom &g, bool a8, bool scaled, int P);
int f8_tiles(const F8Call &c, float *part, size_t part_bytes, hipStream_t st);

}  // namespace vqk
