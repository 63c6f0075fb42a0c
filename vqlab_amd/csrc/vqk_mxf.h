// Products of 4-bit rows with 4-bit weights on the block-scaled matrix
// instruction (v_mfma_scale_f32_32x32x64_f8f6f4, both operands e2m1): 64 k of
// 32 x 32 outputs in the time that bf16 takes for 16.
//
// A workgroup of four waves takes 256 weight rows and 32 * BT x rows, a wave 64
// weight rows and all of the x rows. k runs in chunks of 256 = 8 blocks; lane
// group g = lane / 32 holds blocks 4g .. 4g+3 of its row, so that a step
// multiplies one whole block per lane (16 bytes), the chunk's four scales are
// one 32-bit load and the instruction picks the step's byte itself. Weights go
// straight to registers; x pieces go global -> LDS without registers, piece p of
// row n at p ^ (n / 2 % 8): the 16 rows of a read phase, two to 256 bytes, then
// fall on 16 different bank groups.
// Bound by the traffic from L2: a chunk of 256 x 32 BT outputs reads
// 32 KB + 4 KB * BT for 256 * BT clocks of matrix work per SIMD.
#pragma once

#include <type_traits>

#include "vqk_mx.h"

namespace vqk {

typedef float f32x16f __attribute__((ext_vector_type(16)));
typedef int mxf_i8 __attribute__((ext_vector_type(8)));

struct MxfArgs {
    const uint8_t *codes, *scales, *xcodes, *xscales;
    int64_t OUT, NB, N, xNB;
    void *y;
    int32_t y_type;
    int32_t nob, nt, NC, splits, per;
    float *part;
};

__device__ __forceinline__ mxf_i8 mxf_operand(u32x4 v) {
    mxf_i8 r{};
    r[0] = int(v.x); r[1] = int(v.y); r[2] = int(v.z); r[3] = int(v.w);
    return r;
}

template <int BT, int WPE>
__global__ void __launch_bounds__(256, WPE) k_mxf_gemm(const MxfArgs p) {
    constexpr int ROWS = 32 * BT;
    constexpr int STAGE = ROWS * 128;
    constexpr int CPW = STAGE / 1024 / 4;
    static_assert(CPW * 4096 == STAGE, "whole copies per wave");
    extern __shared__ __align__(16) uint8_t xs[];       // [2][STAGE]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 31, g = lane >> 5;
    const int total = int(gridDim.x);
    int t = int(blockIdx.x);
    {
        const int x = t % 8, q = total / 8, rest = total % 8;       // contiguous bands per XCD
        t = x * q + min(x, rest) + t / 8;
    }
    const int slice = t % p.splits;
    t /= p.splits;
    const int64_t row0 = int64_t(t % p.nt) * ROWS;
    const int nrows = int(min(int64_t(ROWS), p.N - row0));
    const int ow = t / p.nt * 256 + wave * 64;
    const int c_lo = slice * p.per, c_hi = min(p.NC, c_lo + p.per);

    f32x16f acc[2][BT];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < BT; ++b) acc[a][b] = f32x16f{};

    const uint8_t *wp[2], *sp[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        const int64_t row = min(int64_t(ow + 32 * a + r), p.OUT - 1);
        wp[a] = p.codes + row * p.NB * 16;
        sp[a] = p.scales + row * p.NB;
    }
    const uint8_t *src[CPW], *xsp[BT];
#pragma unroll
    for (int j = 0; j < CPW; ++j) {
        const int n = (wave * CPW + j) * 8 + (lane >> 3);
        src[j] = p.xcodes + (row0 + min(n, nrows - 1)) * p.xNB * 16 + ((lane & 7) ^ ((n >> 1) & 7)) * 16;
    }
#pragma unroll
    for (int b = 0; b < BT; ++b) xsp[b] = p.xscales + (row0 + min(32 * b + r, nrows - 1)) * p.xNB + 4 * g;

    u32x4 w[2][4], wn[2][4];
    int ws[2], wsn[2], xsc[BT], xscn[BT];
    auto issue = [&](int c, int buf) {
#pragma unroll
        for (int j = 0; j < CPW; ++j)
            __builtin_amdgcn_global_load_lds((global_void *)(src[j] + int64_t(c) * 128),
                                             (lds_void *)(xs + buf * STAGE + (wave * CPW + j) * 1024), 16, 0, 0);
        const int64_t blk = 8 * int64_t(c) + 4 * g;       // NB % 4 == 0: a lane's four blocks are in or out together
        const bool in = blk < p.NB;
#pragma unroll
        for (int a = 0; a < 2; ++a) {
#pragma unroll
            for (int s = 0; s < 4; ++s)
                wn[a][s] = in ? *reinterpret_cast<const u32x4 *>(wp[a] + (blk + s) * 16) : u32x4{};
            wsn[a] = in ? *reinterpret_cast<const int *>(sp[a] + blk) : 0;
        }
#pragma unroll
        for (int b = 0; b < BT; ++b) xscn[b] = *reinterpret_cast<const int *>(xsp[b] + 8 * int64_t(c));
    };
    const int at0 = r * 128, sw = (r >> 1) & 7;
    auto step = [&](int buf, auto s_c) {
        constexpr int S = decltype(s_c)::value;
        const int at = at0 + ((4 * g + S) ^ sw) * 16;
#pragma unroll
        for (int b = 0; b < BT; ++b) {
            const mxf_i8 xf = mxf_operand(*reinterpret_cast<const u32x4 *>(xs + buf * STAGE + b * 4096 + at));
#pragma unroll
            for (int a = 0; a < 2; ++a)
                acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mxf_operand(w[a][S]), xf, acc[a][b], 4, 4,
                                                                            S, ws[a], S, xsc[b]);
        }
    };
    if (c_lo < c_hi) issue(c_lo, 0);
#pragma unroll 1
    for (int c = c_lo; c < c_hi; ++c) {
        const int buf = (c - c_lo) & 1;
        wait_vmem();
        __syncthreads();                      // copies of chunk c are in; the other buffer is free
#pragma unroll
        for (int a = 0; a < 2; ++a) {
#pragma unroll
            for (int s = 0; s < 4; ++s) w[a][s] = wn[a][s];
            ws[a] = wsn[a];
        }
#pragma unroll
        for (int b = 0; b < BT; ++b) xsc[b] = xscn[b];
        if (c + 1 < c_hi) issue(c + 1, buf ^ 1);
        step(buf, std::integral_constant<int, 0>{});
        step(buf, std::integral_constant<int, 1>{});
        step(buf, std::integral_constant<int, 2>{});
        step(buf, std::integral_constant<int, 3>{});
    }

    void *y = p.splits > 1 ? static_cast<void *>(p.part + int64_t(slice) * p.N * p.OUT) : p.y;
    const int32_t yt = p.splits > 1 ? VQK_F32 : p.y_type;
    const bool al = (p.OUT & 3) == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0;
#pragma unroll
    for (int b = 0; b < BT; ++b) {
        const int n = 32 * b + r;
        if (n >= nrows) continue;
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int o = ow + 32 * a + 8 * j + 4 * g;
                if (o >= p.OUT) continue;
                const float v[4] = {acc[a][b][4 * j], acc[a][b][4 * j + 1], acc[a][b][4 * j + 2],
                                    acc[a][b][4 * j + 3]};
                mx_store4(y, yt, (row0 + n) * p.OUT + o, v, int(min(int64_t(4), p.OUT - o)), al);
            }
    }
}

}  // namespace vqk
