// Products of 8-bit weights with many 8-bit rows on 32x32x64 matrix instructions.
//
// A workgroup of eight waves takes 256 weight rows and BN x rows; a wave 64 by
// BN / 2. k runs in half blocks of 64: a stage holds 64 bytes of every row of both
// sides and the block's scales of the x rows, copied global -> LDS without
// registers, NST stages in a ring. Weights lie in operand order (a row tile's half
// block is two runs of 512 bytes: reads are contiguous); slot s of x row n is stored
// at s ^ (n / 4 % 4), so the 16 rows of a read phase fall on 16 different bank groups.
// The waves run in two groups of four, one of each on every SIMD. A group reads
// all fragments of a stage (LOAD), then multiplies them (MMA), one phase behind the
// other group, so that one wave of a SIMD multiplies while the other loads. Each
// product starts from zero and enters the accumulators by a multiply-add with its
// scales, sw (a number a wave) times sx (a number a lane), while the next multiplies:
// 64 cycles of 16 multiply-adds beside 64 of a matrix instruction.
#pragma once

#include "vqk_f8.h"

namespace vqk {

constexpr int kF8tRows = 256;                 // weight rows per workgroup

struct F8tArgs {
    const uint8_t *codes;
    const float *scales;
    int64_t swo, swk;
    int64_t OUT, N;
    int32_t RT, NC;
    const uint8_t *x;
    int64_t xld;
    const float *sx;
    int64_t sn, sk;
    void *y;
    int32_t y_type;
    int32_t nt, splits, per;                  // x tiles, K slices and blocks in each
    float *part;
};

template <int BN, int NST>
__global__ void __launch_bounds__(512) k_f8_tiles(const F8tArgs p) {
    constexpr int TM = 2, TN = BN / 64;       // 32 x 32 tiles of a wave
    constexpr int A_INS = kF8tRows / 16, B_INS = BN / 16;   // 1 KB copies of a stage
    constexpr int CPW = (A_INS + B_INS + 7) / 8;
    constexpr int OPS = CPW + 1;              // and one of scales
    constexpr int A_BYTES = A_INS * 1024, STAGE = (A_INS + B_INS) * 1024 + BN * 4;
    extern __shared__ __align__(16) uint8_t smem[];     // [NST][STAGE]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = wave >> 2, wm = wave & 3, wn = grp;
    const int r = lane & 31, lk = lane >> 5;

    const int total = int(gridDim.x);
    int t = int(blockIdx.x);
    {
        const int x = t % 8, q = total / 8, rest = total % 8;       // contiguous bands per XCD
        t = x * q + min(x, rest) + t / 8;
    }
    const int slice = t % p.splits;
    t /= p.splits;
    const int64_t row0 = int64_t(t % p.nt) * BN;
    const int nrows = int(min(int64_t(BN), p.N - row0));
    const int o0 = t / p.nt * kF8tRows, ow = o0 + wm * 64;
    const int c_lo = slice * p.per, KT = 2 * (min(p.NC, c_lo + p.per) - c_lo);   // half blocks

    // this wave's copies: a row tile's half block of weights, 64 bytes of 16 x rows, 64 scales
    // (a wave's base and a lane's 32-bit offset)
    const uint8_t *base[CPW];
    uint32_t off[CPW];
    int dst[CPW];
    bool isw[CPW];
#pragma unroll
    for (int j = 0; j < CPW; ++j) {
        const int c = min(wave * CPW + j, A_INS + B_INS - 1);
        isw[j] = c < A_INS;
        dst[j] = c * 1024;
        if (isw[j]) {
            base[j] = p.codes + (int64_t(min(o0 / 16 + c, p.RT - 1)) * p.NC + c_lo) * 2048;
            off[j] = uint32_t((lane >> 5) * 1024 + (lane & 31) * 16);
        } else {
            const int n = (c - A_INS) * 16 + (lane >> 2);
            base[j] = p.x + row0 * p.xld + int64_t(c_lo) * 128;
            off[j] = uint32_t(min(n, nrows - 1)) * uint32_t(p.xld) + 16 * ((lane & 3) ^ ((n >> 2) & 3));
        }
    }
    const int su = wave % (BN / 64);
    const float *ssrc = p.sx + (row0 + min(su * 64 + lane, nrows - 1)) * p.sn + int64_t(c_lo) * p.sk;
    auto issue = [&](int kt, int buf) {
        uint8_t *to = smem + buf * STAGE;
        kt = min(kt, KT - 1);                 // past the end: a copy nobody reads
        const int64_t c = kt >> 1;
        const int hs = kt & 1;
#pragma unroll
        for (int j = 0; j < CPW; ++j)
            __builtin_amdgcn_global_load_lds((global_void *)(base[j] + (isw[j] ? c * 2048 + hs * 512 : c * 128 + hs * 64) + off[j]),
                                             (lds_void *)(to + dst[j]), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((global_void *)(ssrc + c * p.sk),
                                         (lds_void *)(to + (A_INS + B_INS) * 1024 + su * 256), 4, 0, 0);
    };
    const float *sw = p.scales + int64_t(min(ow, int(p.OUT) - 1) / 128) * p.swo + int64_t(c_lo) * p.swk;

    f32x16g acc[TM][TN];
#pragma unroll
    for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int b = 0; b < TN; ++b) acc[a][b] = f32x16g{};
    f8_i8 fa[TM], fb[TN];
    float f[TN];
    auto load_phase = [&](int kt) {
        const uint8_t *ab = smem + (kt % NST) * STAGE, *bb = ab + A_BYTES;
        const float *sb = reinterpret_cast<const float *>(ab + (A_INS + B_INS) * 1024);
        const float w = sw[int64_t(kt >> 1) * p.swk];
#pragma unroll
        for (int a = 0; a < TM; ++a) {
            const uint8_t *at = ab + (wm * 4 + a * 2 + (r >> 4)) * 1024 + (lk * 16 + (r & 15)) * 16;
            fa[a] = f8_pair(*reinterpret_cast<const u32x4 *>(at), *reinterpret_cast<const u32x4 *>(at + 512));
        }
#pragma unroll
        for (int b = 0; b < TN; ++b) {
            const int n = wn * (BN / 2) + b * 32 + r, z = (n >> 2) & 3;
            fb[b] = f8_pair(*reinterpret_cast<const u32x4 *>(bb + n * 64 + ((2 * lk) ^ z) * 16),
                            *reinterpret_cast<const u32x4 *>(bb + n * 64 + ((2 * lk + 1) ^ z) * 16));
            f[b] = sb[n] * w;
        }
        issue(kt + NST - 1, (kt + NST - 1) % NST);
    };
    // a product a time, the multiply-adds of the one before it in its shadow. The empty asm holds the
    // compiler to that order (two sums alive): a product's operand passes it after the sums two before
    // are used up
    auto mma_phase = [&]() {
        f32x16g s[2];
#pragma unroll
        for (int i = 0; i <= TM * TN; ++i) {
            if (i < TM * TN)
                s[i & 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fa[i % TM], fb[i / TM], f32x16g{}, 0, 0, 0, 0, 0, 0);
            if (i > 0) {
                const int a = (i - 1) % TM, b = (i - 1) / TM;
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[a][b][j] = __builtin_fmaf(f[b], s[(i - 1) & 1][j], acc[a][b][j]);
                if (i + 1 < TM * TN) asm volatile("" : "+v"(acc[a][b]), "+v"(fb[(i + 1) / TM]));
            }
        }
    };

#pragma unroll
    for (int s = 0; s < NST - 1; ++s) issue(s, s);
    wait_vmcnt<(NST - 2) * OPS>();            // this wave's part of stage 0
    __builtin_amdgcn_s_barrier();
    if (grp) __builtin_amdgcn_s_barrier();    // group 1 runs one phase behind
    for (int kt = 0; kt < KT; ++kt) {
        load_phase(kt);
        if (grp) wait_vmcnt<(NST - 2) * OPS>();   // group 1: its part of stage kt + 1
        __builtin_amdgcn_s_waitcnt(0xC07F);       // lgkmcnt(0): fragments in registers
        __builtin_amdgcn_s_barrier();
        mma_phase();
        if (!grp) wait_vmcnt<(NST - 2) * OPS>();  // group 0: its part of stage kt + 1
        __builtin_amdgcn_s_barrier();
    }
    if (!grp) __builtin_amdgcn_s_barrier();   // pairs group 1's last barrier
    wait_vmem();

    // register i of lane l: weight row 8 * (i / 4) + 4 * (l / 32) + i % 4, x row l % 32
    void *y = p.splits > 1 ? static_cast<void *>(p.part + int64_t(slice) * p.N * p.OUT) : p.y;
    const int32_t yt = p.splits > 1 ? VQK_F32 : p.y_type;
    const bool al = (p.OUT & 3) == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0;
#pragma unroll
    for (int b = 0; b < TN; ++b) {
        const int n = wn * (BN / 2) + 32 * b + r;
        if (n >= nrows) continue;
#pragma unroll
        for (int a = 0; a < TM; ++a)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int o = ow + 32 * a + 8 * j + 4 * lk;
                if (o >= p.OUT) continue;
                const float v[4] = {acc[a][b][4 * j], acc[a][b][4 * j + 1], acc[a][b][4 * j + 2], acc[a][b][4 * j + 3]};
                mx_store4(y, yt, (row0 + n) * p.OUT + o, v, int(min(int64_t(4), p.OUT - o)), al);
            }
    }
}

}  // namespace vqk
