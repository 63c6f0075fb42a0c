// MXFP4 (microscaled 4-bit) weights: shared declarations of the vqk_mx*
// sources. A row of C values is NB = ceil(C / 32) blocks; block b holds 32
// codes of 4 bits in 16 bytes (the earlier element in the low half of a byte,
// codes past C zero) and one scale byte s: element = e2m1(code) * 2^(s - 127),
// s = 255 a block of NaN.
//
// Three facts carry every kernel here:
//   * e2m1 * 2^(s - 127) has at most two significant bits and an exponent
//     inside bf16's, so a bf16 weight is the exact weight
//     (v_cvt_scalef32_pk_bf16_fp4 makes two of them, scale included). Only s = 253
//     from code 4 and s = 254 from code 2 up give 2^128 and more: infinite, in bf16 as
//     in fp32. The 4-bit products alone multiply those as they are;
//   * the sum over k may be taken in any order, so a lane of a matrix
//     instruction can own whole blocks (16 bytes, one scale): in a chunk of 128 k
//     the lane groups take the chunk's four blocks, and step h multiplies
//     elements 8h..8h+7 of each group's block. Weights then go from global
//     memory to registers, no LDS, and the x operand is a 16-byte piece of a row;
//   * the L1 serves one 128-byte line per cycle, and 16 lanes a cycle. Read
//     row by row, a lane's 16 bytes lie in a line of their own: 64 cycles for the
//     1 KB of a wave's load instead of 16 (47 MB of weights at 4.1 TB/s instead of 5.5,
//     and the many-row kernels bound by it). So weights are laid out once in
//     operand order:
//       codes  [E][RT][NC][64][16]   RT = ceil(OUT / 16) row tiles, NC = ceil(IN / 128)
//              unit (lane) i of a tile: row i % 16, block 4 chunk + i / 16
//       scales [E][RT][ceil(NC / 4)][64][4]   byte j of unit i: the scale of its block in
//              chunk 4 group + j (the block-scaled matrix instruction picks a byte itself)
//     with codes 0 and scales 127 past the row's and the weight's end.
#pragma once

#include "vqk_gemv.h"
#include "vqk_internal.h"

namespace vqk {

typedef __bf16 mx_b2 __attribute__((ext_vector_type(2)));
typedef __bf16 mx_b8 __attribute__((ext_vector_type(8)));

constexpr int kMxBlock = 32;
constexpr int kMxChunk = 128;                 // k of one weight load: 4 lane groups x 32

struct MxGeom { int64_t E, OUT, IN, NB, RT, NC; };
__host__ __device__ constexpr int64_t mx_expert_codes(int64_t RT, int64_t NC) { return RT * NC * 1024; }
__host__ __device__ constexpr int64_t mx_expert_scales(int64_t RT, int64_t NC) { return RT * ((NC + 3) / 4) * 256; }
// Validates `w` and fills `g`; returns a VQK_* status and sets the message.
int make_mx_geom(const vqk_mx_weights *w, MxGeom *g, const char *what);

// Whether rows of x [., IN] enter as they lie.
inline bool mx_x_in_place(const vqk_mx_weights *w, const void *x, int32_t type) {
    return (type == VQK_BF16 || (type == VQK_F16 && w->f16_exact)) && w->IN % kMxBlock == 0 &&
           (reinterpret_cast<uintptr_t>(x) & 15) == 0;
}

// 2^(s - 127) as fp32 (s = 0 is the subnormal 2^-127; s = 255 NaN).
__device__ __forceinline__ float mx_scale(uint32_t s) {
    return __uint_as_float(s == 0u ? 0x00400000u : (s == 255u ? 0x7fc00000u : s << 23));
}

// Eight codes (one word) as bf16 weights, scale included.
__device__ __forceinline__ u32x4 mx_decode8(uint32_t w, float sc) {
    u32x4 r;
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3));
    return r;
}

// The same for fp16 operands, exact for weights that are fp16 numbers (f16_exact).
template <int OP>
__device__ __forceinline__ u32x4 mx_decode8_op(uint32_t w, float sc) {
    if constexpr (OP == kOpBF16) return mx_decode8(w, sc);
    u32x4 r;
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 0));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 1));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 2));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 3));
    return r;
}

// Scale bytes under which every code but 0 is an fp16 number: 0.5 * 2^-23 is the
// smallest subnormal, 6 * 2^13 below the largest number.
constexpr uint32_t kMxF16ScaleMin = 104, kMxF16ScaleMax = 140;

// fp16 x enters as it is where the weights are fp16 numbers. Otherwise
// activations enter the matrix cores as bf16 planes whose sum is exact: one
// for bf16, two for fp16 (11 significant bits = 8 + 3), three for fp32 (24).
constexpr int mx_planes(int32_t type) { return type == VQK_BF16 ? 1 : (type == VQK_F16 ? 2 : 3); }

// The next plane of a value: bf16 of what the planes before it leave. A value that
// is not finite stands in plane 0 alone; a finite one that would round past the
// largest bf16 (2^128 (1 - 2^-9) and up) starts with that number instead, and the
// next two planes hold the 16 bits under it.
__device__ __forceinline__ uint16_t mx_plane_next(float &rest) {
    const bool fin = (__float_as_uint(rest) & 0x7f800000u) != 0x7f800000u;
    uint16_t h = f32_to_bf16(rest);
    h -= uint16_t(fin && (h & 0x7fffu) == 0x7f80u);
    rest = fin ? rest - bf16_to_f32(h) : 0.f;
    return h;
}

// Largest magnitude bits of a block -> its scale byte: floor(log2) - 2 in the
// biased exponents, at least 0 (2^-127); 255 where a value is not finite.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
    const int e = int(amax_bits >> 23);
    return e == 255 ? 255u : uint32_t(max(e - 2, 0));
}

// Eight values as codes under the scale byte s (255: zeros).
__device__ __forceinline__ uint32_t mx_encode8(const float (&v)[8], uint32_t s) {
    if (s == 255u) return 0u;
    const float sc = mx_scale(s);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], sc, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], sc, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], sc, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], sc, 3);
    return w;
}

// Eight activations k0..k0+7 of a row (vec: 16-byte aligned and whole), zero
// at and past `cols`.
__device__ __forceinline__ void mx_load8(const void *x, int32_t type, int64_t base, int64_t k0,
                                         int64_t cols, bool vec, float (&v)[8]) {
    if (vec && k0 + 8 <= cols) {
        if (type == VQK_F32) {
            const u32x4 a = *reinterpret_cast<const u32x4 *>(static_cast<const float *>(x) + base + k0);
            const u32x4 b = *reinterpret_cast<const u32x4 *>(static_cast<const float *>(x) + base + k0 + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = __uint_as_float(a[i]);
                v[4 + i] = __uint_as_float(b[i]);
            }
        } else {
            const u32x4 a = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(x) + base + k0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint16_t lo = uint16_t(a[i] & 0xffffu), hi = uint16_t(a[i] >> 16);
                v[2 * i] = type == VQK_BF16 ? bf16_to_f32(lo) : h_to_f32(lo);
                v[2 * i + 1] = type == VQK_BF16 ? bf16_to_f32(hi) : h_to_f32(hi);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k0 + i < cols ? load_act(x, type, base + k0 + i) : 0.f;
}

// Largest value over each aligned group of four lanes, in every lane of it.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, dpp_u<kDppQuadXor1>(v));
    return max(v, dpp_u<kDppQuadXor2>(v));
}

// n (up to 4) neighbouring outputs at element i; al: whole fours are aligned
// wherever i is a multiple of 4.
__device__ __forceinline__ void mx_store4(void *y, int32_t type, int64_t i, const float (&v)[4], int n,
                                          bool al) {
    if (al && n == 4 && (i & 3) == 0) {
        if (type == VQK_F32) {
            *reinterpret_cast<float4 *>(static_cast<float *>(y) + i) = float4{v[0], v[1], v[2], v[3]};
            return;
        }
        if (type == VQK_BF16 || type == VQK_F16) {
            uint32_t q[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) q[u] = type == VQK_BF16 ? f32_to_bf16(v[u]) : f32_to_h(v[u]);
            u32x2 o;
            o.x = q[0] | (q[1] << 16);
            o.y = q[2] | (q[3] << 16);
            *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(y) + i) = o;
            return;
        }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (u < n) store_act(y, type, i + u, v[u]);
}

// x [N, IN] (rows ldx apart) -> bf16 planes [P][N][NB * 32], zero past IN; or
// (quant) the values of its MXFP4 form, one plane.
int launch_mx_planes(const void *x, int32_t type, int64_t N, int64_t IN, int64_t ldx, bool quant,
                     uint16_t *out, hipStream_t st);
// The quantiser without argument checks, into rows of NB >= ceil(cols / 32)
// blocks (those past the row: zeros); permute: scales placed by mxf_scale_at.
int launch_mx_quant(const void *x, int32_t type, int64_t rows, int64_t cols, int64_t ldx, int64_t NB,
                    bool permute, uint8_t *codes, uint8_t *scales, hipStream_t st);

// Rows of x as the product kernels read them: bf16 planes (or fp16 rows) ld apart.
struct MxX {
    const uint16_t *x;
    int64_t ld, plane;                        // elements between rows / planes
    int P;
    int op;                                   // kOpBF16, or kOpF16 (P = 1): fp16 rows
};

// One product, over dense rows, single pairs, or tiles of a sorted routing.
struct MxCall {
    const uint8_t *codes[2], *scales[2];      // [1]: the second projection of a SwiGLU pair
    MxGeom g;
    MxX x;
    int64_t N;                                // rows or pairs
    // routing: none (dense) | ids (tile = pair) | order, meta, ntiles (sorted tiles)
    const int32_t *ids, *order, *meta, *ntiles;
    int64_t xkrep;                            // x row = pair / xkrep; 0: x rows are sorted positions (or pairs)
    void *y;                                  // [row][OUT] in y_type; a SwiGLU pair: rows like x's
    int32_t y_type;
    int64_t ldy, yplane;                      // elements between rows / planes of y
    int yp;                                   // bf16 planes of a SwiGLU pair's output
    bool ysorted;                             // y rows by sorted position
};

// The many-row products (vqk_mxg.h): x tiles of tile_rows (32, 64, 128); part:
// room for fp32 K slices of a dense product, or NULL.
int mx_gemm(const MxCall &c, int tile_rows, float *part, size_t part_bytes, hipStream_t st);
// x rows per tile of a dense product of N rows.
int mxg_dense_rows(int64_t N);
// Bytes of the K slices that a dense product of N rows makes use of.
size_t mxg_part_bytes(int64_t N, const MxGeom &g);

// K slices of a dense product, four outputs a thread, and how many pay.
int mx_splits(int64_t T, int64_t NC, int64_t n, float t1, float t2);
int launch_mx_reduce(const float *part, int splits, int64_t n, void *y, int32_t y_type, hipStream_t st);

// Products of 4-bit rows with 4-bit weights (vqk_mxf.h): x as codes in rows of
// xNB blocks, a multiple of 16, and scales in the order of mxf_scale_at.
struct MxfCall {
    const uint8_t *codes, *scales;
    MxGeom g;
    int64_t N, xNB;
    const uint8_t *xcodes, *xscales;
    void *y;
    int32_t y_type;
};
// Place of block b's scale in a row of x scales: the four chunks' bytes of a
// block position side by side, as in the weights' scales.
__host__ __device__ constexpr int64_t mxf_scale_at(int64_t b) {
    return b / 16 * 16 + b % 4 * 4 + b / 4 % 4;
}
int mxf_gemm(const MxfCall &c, float *part, size_t part_bytes, hipStream_t st);
size_t mxf_part_bytes(int64_t N, const MxGeom &g);

}  // namespace vqk
