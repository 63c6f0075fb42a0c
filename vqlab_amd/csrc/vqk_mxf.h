// Products of 4-bit rows with 4-bit weights on the block-scaled matrix
// instruction (v_mfma_scale_f32_32x32x64_f8f6f4, both operands e2m1): 64 k of
// 32 x 32 outputs in the time that bf16 takes for 16.
//
// A workgroup of four waves takes 256 weight rows and 32 * BT x rows, a wave 64
// weight rows and all of the x rows. k runs in groups of four chunks of 128; lane
// group g = lane / 32 holds blocks 2g and 2g + 1 of each chunk, and a step
// multiplies one block per lane (16 bytes). The four chunks' scales of a block
// position are one 32-bit load, and the instruction picks the chunk's byte itself.
// Weights go straight to registers in operand order; x pieces go global -> LDS
// without registers, two chunks (128 bytes of a row) a stage, piece p of row n at
// p ^ (n / 2 % 8): the 16 rows of a read phase, two to 256 bytes, then fall on 16
// different bank groups.
#pragma once

#include <type_traits>

#include "vqk_mx.h"

namespace vqk {

typedef float f32x16f __attribute__((ext_vector_type(16)));
typedef int mxf_i8 __attribute__((ext_vector_type(8)));

struct MxfArgs {
    const uint8_t *codes, *scales, *xcodes, *xscales;
    int64_t OUT, N, xNB;
    void *y;
    int32_t y_type;
    int32_t RT, NC, nob, nt, splits, per;     // per: groups of four chunks in a K slice
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
    const int NC4 = (p.NC + 3) / 4;
    const int h_lo = 2 * slice * p.per, h_hi = min((p.NC + 1) / 2, h_lo + 2 * p.per);   // halves of a group

    f32x16f acc[2][BT];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < BT; ++b) acc[a][b] = f32x16f{};

    uint32_t wo[2], so[2];                    // block 2g of this lane's row tile
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        const uint32_t rt = uint32_t(min((ow + 32 * a) / 16 + (r >> 4), p.RT - 1));
        const uint32_t unit = uint32_t(2 * g * 16 + (r & 15));
        wo[a] = (rt * uint32_t(p.NC) * 64 + unit) * 16;
        so[a] = (rt * uint32_t(NC4) * 64 + unit) * 4;
    }
    // x by 32-bit offsets from the tile's first row
    const uint8_t *xc0 = p.xcodes + row0 * p.xNB * 16, *xs0 = p.xscales + row0 * p.xNB;
    uint32_t src[CPW], xso[BT];
#pragma unroll
    for (int j = 0; j < CPW; ++j) {
        const int n = (wave * CPW + j) * 8 + (lane >> 3);
        src[j] = uint32_t(min(n, nrows - 1)) * uint32_t(p.xNB) * 16 + ((lane & 7) ^ ((n >> 1) & 7)) * 16;
    }
#pragma unroll
    for (int b = 0; b < BT; ++b) xso[b] = uint32_t(min(32 * b + r, nrows - 1)) * uint32_t(p.xNB) + 8 * g;

    u32x4 w[2][4], wn[2][4];                  // [tile][2 * chunk of the half + block]
    int ws[2][2], wsn[2][2], xsc[BT][2], xscn[BT][2];   // [..][block]: a group's scales
    // half h: chunks 2h and 2h + 1. x is padded to whole groups; a weight chunk past the end is none
    auto issue = [&](int h, int buf) {
#pragma unroll
        for (int j = 0; j < CPW; ++j)
            __builtin_amdgcn_global_load_lds((global_void *)(xc0 + (src[j] + uint32_t(h) * 128u)),
                                             (lds_void *)(xs + buf * STAGE + (wave * CPW + j) * 1024), 16, 0, 0);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint32_t ch = uint32_t(min(2 * h + c, p.NC - 1));
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    wn[a][2 * c + q] = *reinterpret_cast<const u32x4 *>(p.codes + (wo[a] + ch * 1024u + q * 256u));
        }
    };
    auto scales = [&](int grp) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
            for (int a = 0; a < 2; ++a)
                wsn[a][q] = *reinterpret_cast<const int *>(p.scales + (so[a] + uint32_t(grp) * 256u + q * 64u));
#pragma unroll
            for (int b = 0; b < BT; ++b)
                xscn[b][q] = *reinterpret_cast<const int *>(xs0 + (xso[b] + uint32_t(grp) * 16u + q * 4u));
        }
    };
    const int at0 = r * 128, sw = (r >> 1) & 7;
    auto half = [&](int h, auto odd) {
        constexpr int ODD = decltype(odd)::value;
        const int buf = h & 1;
        wait_vmem();
        __syncthreads();                      // copies of the half are in; the other buffer is free
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int s = 0; s < 4; ++s) w[a][s] = wn[a][s];
        if (!ODD) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
#pragma unroll
                for (int a = 0; a < 2; ++a) ws[a][q] = wsn[a][q];
#pragma unroll
                for (int b = 0; b < BT; ++b) xsc[b][q] = xscn[b][q];
            }
        }
        if (h + 1 < h_hi) {
            issue(h + 1, buf ^ 1);
            if (ODD) scales(h / 2 + 1);
        }
        auto step = [&](auto c_c, auto q_c) {
            constexpr int C = decltype(c_c)::value, Q = decltype(q_c)::value;
            const int at = at0 + ((4 * C + 2 * g + Q) ^ sw) * 16;
#pragma unroll
            for (int b = 0; b < BT; ++b) {
                const mxf_i8 xf = mxf_operand(*reinterpret_cast<const u32x4 *>(xs + buf * STAGE + b * 4096 + at));
#pragma unroll
                for (int a = 0; a < 2; ++a)
                    acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                        mxf_operand(w[a][2 * C + Q]), xf, acc[a][b], 4, 4, 2 * ODD + C, ws[a][Q], 2 * ODD + C, xsc[b][Q]);
            }
        };
        using c0 = std::integral_constant<int, 0>;
        using c1 = std::integral_constant<int, 1>;
        step(c0{}, c0{});
        step(c0{}, c1{});
        if (2 * h + 1 < p.NC) {
            step(c1{}, c0{});
            step(c1{}, c1{});
        }
    };
    if (h_lo < h_hi) {                        // h_lo is even
        issue(h_lo, 0);
        scales(h_lo / 2);
    }
#pragma unroll 1
    for (int h = h_lo; h < h_hi; h += 2) {
        half(h, std::integral_constant<int, 0>{});
        if (h + 1 < h_hi) half(h + 1, std::integral_constant<int, 1>{});
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
