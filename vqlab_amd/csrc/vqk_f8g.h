// Products of 8-bit weights with many rows of 16-bit x: codes converted in
// registers, multiplied on 32x32x16 matrix instructions.
//
// A workgroup of four waves takes 256 weight rows and a tile of 32 * BT x rows; a
// wave owns 64 weight rows and all of the tile's x rows, so every weight is
// converted by one wave only and its scale is one number a block and wave. Per
// block of 128 k:
//   * weights: 64 bytes per lane and 32-row tile straight from global memory, in
//     operand order. Lane group g = lane / 32 holds 32-byte units 2g and 2g + 1 of
//     its row; step (q, h) multiplies elements 8h..8h+7 of unit 2g + q.
//   * x: the tile's 256-byte row pieces, copied global -> LDS without registers
//     (16 bytes a lane); piece p of row n is stored at p ^ (n & 15), so the 16 rows
//     of a read phase fall on 16 different bank groups.
//   * the sums of a unit pair start from zero and enter the accumulators by a
//     multiply-add with the block's scale, in the shadow of the next tile's matrix
//     instructions: accumulators (32 * BT registers) and sums (32) bound BT to 3.
// The loads of the next block are in flight while one multiplies; two workgroups
// share a CU and fill each other's waits. x in planes (fp32) takes one plane a step,
// the weights again from L2.
#pragma once

#include <type_traits>

#include "vqk_mxg.h"
#include "vqk_f8.h"

namespace vqk {

constexpr int kF8gWaves = 4;
constexpr int kF8gRows = 256;                 // weight rows per workgroup

struct F8gArgs {
    const uint8_t *codes;
    const float *scales;
    int64_t swo, swk;
    int64_t OUT, IN, N;
    int32_t RT, NC, P;
    const uint16_t *x;
    int64_t xld, xplane;
    const float *sx;                          // SX: scales of x's rows
    int64_t sn, sk;
    void *y;
    int32_t y_type;
    int32_t nt, splits, per;                  // x tiles, K slices and blocks in each
    float *part;                              // [splits][N][OUT] when splits > 1
};

// SX: x holds the values of 8-bit codes (one plane), the rows' scales beside them.
template <int OP, int BT, bool SX>
__global__ void __launch_bounds__(64 * kF8gWaves, 2) k_f8_gemm(const F8gArgs p) {
    constexpr int ROWS = 32 * BT;
    constexpr int STAGE = ROWS * 256;
    constexpr int COPIES = ROWS / 16;         // 16-byte copies a lane: 4 rows a wave's instruction
    extern __shared__ __align__(16) uint8_t xs[];       // [2][STAGE]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
    const int ow = t / p.nt * kF8gRows + wave * 64;
    const int c_lo = slice * p.per, c_hi = min(p.NC, c_lo + p.per);

    f32x16g acc[2][BT];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < BT; ++b) acc[a][b] = f32x16g{};

    const uint32_t NC = uint32_t(p.NC);
    uint32_t wo[2];                           // unit 2g of this lane's row
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        const uint32_t rt = uint32_t(min((ow + 32 * a) / 16 + (r >> 4), p.RT - 1));
        wo[a] = rt * NC * 2048u + uint32_t(2 * g * 16 + (r & 15)) * 16u;
    }
    const float *sw = p.scales + int64_t(min(ow, int(p.OUT) - 1) / 128) * p.swo;
    const uint16_t *src[COPIES];
    int piece[COPIES];
#pragma unroll
    for (int j = 0; j < COPIES; ++j) {
        const int n = (j * kF8gWaves + wave) * 4 + (lane >> 4);
        piece[j] = (lane & 15) ^ (n & 15);
        src[j] = p.x + (row0 + min(n, nrows - 1)) * p.xld + piece[j] * 8;
    }
    struct Weights {
        u32x4 w[2][2][2];                     // [tile][unit][half]
        float s, sx[SX ? BT : 1];
    };
    Weights wb[2];
    int64_t sxo[BT];
#pragma unroll
    for (int b = 0; b < BT; ++b) sxo[b] = (row0 + min(32 * b + r, nrows - 1)) * p.sn;
    const int P = p.P, steps = (c_hi - c_lo) * P;
    auto issue = [&](int step, auto slot) {
        constexpr int S = decltype(slot)::value;
        const int c = c_lo + step / P;
#pragma unroll
        for (int j = 0; j < COPIES; ++j) {
            const uint16_t *from = src[j] + (step % P) * p.xplane + int64_t(c) * kF8Block;
            from = int64_t(c) * kF8Block + piece[j] * 8 < p.IN ? from : reinterpret_cast<const uint16_t *>(mxg_zeros);
            __builtin_amdgcn_global_load_lds((global_void *)from,
                                             (lds_void *)(xs + S * STAGE + (j * kF8gWaves + wave) * 1024), 16, 0, 0);
        }
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    wb[S].w[a][q][h] = *reinterpret_cast<const u32x4 *>(p.codes + (wo[a] + uint32_t(c) * 2048u + q * 256u + h * 1024u));
        wb[S].s = load_global(sw, int64_t(c) * p.swk);
        if constexpr (SX) {
#pragma unroll
            for (int b = 0; b < BT; ++b) wb[S].sx[b] = load_global(p.sx, sxo[b] + int64_t(c) * p.sk);
        }
    };
    auto mul = [&](auto slot) {
        constexpr int S = decltype(slot)::value;
        const Weights &d = wb[S];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            u32x4 wf[2][4];
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int h = 0; h < 4; ++h) wf[a][h] = f8_operand<OP>(d.w[a][q][h / 2][h % 2 * 2], d.w[a][q][h / 2][h % 2 * 2 + 1]);
#pragma unroll
            for (int b = 0; b < BT; ++b) {
                f32x16g s[2] = {f32x16g{}, f32x16g{}};
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const int at = ((8 * g + 4 * q + h) ^ (lane & 15)) * 16 + r * 256;
                    const u32x4 xv = *reinterpret_cast<const u32x4 *>(xs + S * STAGE + b * 8192 + at);
#pragma unroll
                    for (int a = 0; a < 2; ++a) s[a] = mx_mma32<OP>(wf[a][h], xv, s[a]);
                }
                const float f = SX ? d.s * d.sx[SX ? b : 0] : d.s;
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[a][b][i] = __builtin_fmaf(f, s[a][i], acc[a][b][i]);
            }
        }
    };
    using s0 = std::integral_constant<int, 0>;
    using s1 = std::integral_constant<int, 1>;
    // past the last step it is loaded again, into a slot that no step reads
    auto one = [&](int step, auto slot) {
        constexpr int S = decltype(slot)::value;
        mxg_keep_order();
        wait_vmcnt<0>();                                // this wave's loads of the step
        __builtin_amdgcn_s_waitcnt(0xC07F);             // lgkmcnt(0): its reads of the other slot
        __builtin_amdgcn_s_barrier();                   // every wave's
        mxg_keep_order();
        issue(min(step + 1, steps - 1), std::integral_constant<int, S ^ 1>{});
        mxg_keep_order();
        if (step < steps) mul(slot);
    };
    if (steps > 0) {
        issue(0, s0{});
#pragma unroll 1
        for (int step = 0; step < steps; step += 2) {
            one(step, s0{});
            one(step + 1, s1{});
        }
        wait_vmem();
    }

    // register i of lane l: weight row 8 * (i / 4) + 4 * (l / 32) + i % 4, x row l % 32
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
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = OP == kOpBF16 ? acc[a][b][4 * j + i] * kF8Up : acc[a][b][4 * j + i];
                mx_store4(y, yt, (row0 + n) * p.OUT + o, v, int(min(int64_t(4), p.OUT - o)), al);
            }
    }
}

}  // namespace vqk
