// Products of 8-bit weights with many rows of x: 8-bit rows on 16x16x128 matrix
// instructions, one of them a whole block of k, or 16-bit rows on 16x16x32 ones, four
// to a block, the codes converted in registers.
//
// A workgroup of eight waves takes 256 weight rows and BN x rows; a wave 64 by
// BN / 2. A block of 128 k of both sides (and the x rows' scales) is copied global ->
// LDS without registers, into a ring of NST buffers. Weights lie there as they do in
// memory, in operand order (reads of a wave are one contiguous KB); the 16-byte slots of
// an x row are permuted (f8t_swz) so that a read phase falls on 16 different bank groups.
// A wave keeps its weights of the block (32 registers, 64 converted) and walks over its
// x rows, 16 at a time: four products from zero, while the four before them enter the
// accumulators by multiply-adds with their scales, sw (a number a wave) times sx (a
// number a lane): 64 cycles of VALU beside 128 (8 bits) or 256 of the matrix cores. The
// conversions run beside the first x tile's products.
// What bounds the tile: accumulators are VALU operands, so they, the weights and two
// tiles of sums share 256 registers (two waves a SIMD): BN up to 256 with 8-bit x, 192
// with 16-bit x, whose two buffers fill LDS, too.
// Measured (us, slices' sum included): 2048 rows of 5120 to 17408, 8-bit x 203 (1.8 PF; the
// same loop without its copies and barriers 2.4 PF, so the matrix cores and the
// multiply-adds behind them are what it waits for); 2048 rows of 17408 to 5120, bf16 x
// 415 (0.88 PF; 320 tiles are 1.25 rounds), its gradient 374 (0.98 PF) after the
// transposition; 333 rows of 17408 to 5120, fp16 x 87 (384 rows' work at 0.78 PF, 7.4 us of
// them the slices' sum). The long ones are 5 to 10 % shorter on a cool chip.
// Whole rounds of tiles run as they are; the tiles of the last, partial round are cut
// along k, so that every CU has a part, into fp32 partials summed in a fixed order.
#pragma once

#include "vqk_mxs.h"
#include "vqk_f8.h"

namespace vqk {

typedef __attribute__((address_space(4))) float uniform_f32;

constexpr int kF8tRows = 256;                 // weight rows per workgroup
constexpr int kOpF8 = 2;                      // beside kOpF16 and kOpBF16: 8-bit x

struct F8tArgs {
    const uint8_t *codes;
    const float *scales;
    int64_t swo, swk;
    int64_t OUT, N;
    int32_t RT, NC, P;                        // P: planes of x, one a step
    const uint8_t *x;                         // whole blocks
    int64_t xld, xplane;                      // bytes
    const float *sx;
    int64_t sn, sk;
    void *y;
    int32_t y_type;
    int32_t nt, tiles;                        // x tiles, and tiles in all
    int32_t full, splits, per;                // tiles run whole; K slices of the others, steps in each
    float *part;                              // [(tiles - full) * splits][BN * 256], in register order
};

// Bytes of a buffer.
constexpr int f8t_stage(int op, int bn, bool sx) {
    return kF8tRows * 128 + bn * (op == kOpF8 ? 128 : 256) + (sx ? bn * 4 : 0);
}

// 16-byte slot s of x row n is stored at s ^ f8t_swz(n). A read phase of 16 lanes is, of
// 32, lanes 0-3, 12-15 and 20-27 (or the other 16): rows whose bits 3 and 2 are equal of one
// lane group, and rows where they differ of the next, whose slots are 4 (8-bit rows: 2) further.
// They fall on 16 different bank groups where bits 3 and 2 of the row do not meet that bit of
// the slot (rows of 128 bytes: two to 256, bit 0 chooses between them).
template <bool A8>
__device__ __forceinline__ int f8t_swz(int n) {
    if constexpr (A8) return ((n >> 3) & 1) * 4 + ((n >> 1) & 1) * 2 + ((n >> 2) & 1);
    return ((n >> 3) & 1) * 8 + (n & 1) * 4 + ((n >> 1) & 1) * 2 + ((n >> 2) & 1);
}

template <int OP, int BN, bool SX, int NST>
__global__ void __launch_bounds__(512) k_f8_tiles(const F8tArgs p) {
    constexpr bool A8 = OP == kOpF8;
    constexpr int XB = A8 ? 128 : 256;        // bytes of a block of an x row
    constexpr int RPC = 1024 / XB;            // x rows of a 1 KB copy
    constexpr int KS = A8 ? 1 : 4;            // matrix instructions of a block
    constexpr int XR = A8 ? 2 : 4;            // LDS reads of an x tile
    constexpr int TN = BN / 32;               // 16-row tiles of x of a wave
    constexpr int A_INS = kF8tRows / 8, B_INS = BN / RPC;   // 1 KB copies of a block
    constexpr int CPW = (A_INS + B_INS) / 8, OPS = CPW + (SX ? 1 : 0);
    static_assert((A_INS + B_INS) % 8 == 0 && TN >= 1, "whole copies a wave");
    constexpr int PER = (CPW + (TN + 1) / 2 - 1) / ((TN + 1) / 2);      // copies beside each of the first x tiles
    constexpr int A_BYTES = A_INS * 1024, STAGE = f8t_stage(OP, BN, SX);
    extern __shared__ __align__(16) uint8_t smem[];     // [NST][STAGE]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave & 3, wn = wave >> 2;
    const int r = lane & 15, g = lane >> 4;

    // whole tiles in contiguous bands per XCD (workgroup b runs on XCD b % 8), then the K slices
    int t = int(blockIdx.x), unit = -1, s_lo = 0, steps = p.NC * p.P;
    if (t < p.full) {
        const int x = t % 8, q = p.full / 8, rest = p.full % 8;
        t = x * q + min(x, rest) + t / 8;
    } else {
        unit = t - p.full;
        t = __builtin_amdgcn_readfirstlane(p.full + unit / p.splits);       // (divisions leave the scalar registers)
        s_lo = (unit - (t - p.full) * p.splits) * p.per;
        steps = min(steps, s_lo + p.per) - s_lo;
    }
    const int64_t row0 = int64_t(__builtin_amdgcn_readfirstlane(t % p.nt)) * BN;
    const int nrows = int(min(int64_t(BN), p.N - row0));
    const int o0 = __builtin_amdgcn_readfirstlane(t / p.nt) * kF8tRows, ow = o0 + wm * 64;

    // this wave's copies: half a row tile of weights, or a KB of x rows; and 64 scales. A lane's place is a
    // 32-bit offset that stays, a block's a scalar one: a copy costs no VALU instruction
    const int wsize = int(uint32_t(f8_code_bytes(p.RT, p.NC)));
    const uint8_t *xtile = p.x + row0 * p.xld;
    const int xsize = int(uint32_t((nrows - 1) * p.xld) + uint32_t(p.NC) * XB);
    uint32_t off[CPW];
#pragma unroll
    for (int j = 0; j < CPW; ++j) {
        const int c = wave * CPW + j;
        if (c < A_INS) {
            off[j] = uint32_t(min(o0 / 16 + c / 2, p.RT - 1)) * uint32_t(p.NC) * 2048u + uint32_t((c & 1) * 1024 + lane * 16);
        } else {
            const int n = (c - A_INS) * RPC + lane / (64 / RPC);
            const int piece = A8 ? (lane & 7) ^ f8t_swz<true>(n) : (lane & 15) ^ f8t_swz<false>(n);
            off[j] = uint32_t(min(n, nrows - 1)) * uint32_t(p.xld) + 16 * piece;
        }
    }
    const int su = SX ? wave % (BN / 64) : 0;
    const float *ssrc = SX ? p.sx + (row0 + min(su * 64 + lane, nrows - 1)) * p.sn : nullptr;
    // copy j of a step into the buffer at `to`; past the last step: one that nobody reads
    struct Step { const uint8_t *x; int c; };
    auto step_of = [&](int step) {
        step = s_lo + min(step, steps - 1);
        const int c = p.P == 1 ? step : __builtin_amdgcn_readfirstlane(step / p.P);
        const int64_t plane = p.P == 1 ? 0 : int64_t(step - c * p.P) * p.xplane;
        return Step{xtile + plane, c};
    };
    auto copy = [&](const Step &st, uint8_t *to, int j) {
        const bool isw = wave * CPW + j < A_INS;
        const __amdgpu_buffer_rsrc_t buf = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t *>(isw ? p.codes : st.x), 0, isw ? wsize : xsize, 0x00027000);
        lds_void *dst = (lds_void *)(to + (wave * CPW + j) * 1024);
        const int lane_at = int(off[j]), block_at = isw ? st.c * 2048 : st.c * XB;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, dst, 16, lane_at, block_at, 0, 0);
    };
    auto copy_scales = [&](const Step &st, uint8_t *to) {
        if constexpr (SX)
            __builtin_amdgcn_global_load_lds((global_void *)(ssrc + int64_t(st.c) * p.sk),
                                             (lds_void *)(to + (A_INS + B_INS) * 1024 + su * 256), 4, 0, 0);
    };
    // read through the scalar cache: a vector load here would make its wait one for all copies in flight
    const uniform_f32 *sw = (const uniform_f32 *)(uintptr_t)(p.scales + int64_t(min(ow, int(p.OUT) - 1) / 128) * p.swo);
    auto scale_of = [&](int step) {
        step = s_lo + min(step, steps - 1);
        return sw[int64_t(p.P == 1 ? step : __builtin_amdgcn_readfirstlane(step / p.P)) * p.swk];
    };

    f32x4 acc[4][TN];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < TN; ++b) acc[a][b] = f32x4{};

#pragma unroll
    for (int i = 0; i < NST - 1; ++i) {
        const Step st = step_of(i);
        copy_scales(st, smem + i * STAGE);
#pragma unroll
        for (int j = 0; j < CPW; ++j) copy(st, smem + i * STAGE, j);
    }
    const int n0 = wn * (BN / 2) + r;
    int wat, xat[XR];                         // this lane's places in a buffer
    wat = wm * 8192 + lane * 16;
#pragma unroll
    for (int h = 0; h < XR; ++h) xat[h] = A_BYTES + n0 * XB + (A8 ? (2 * g + h) ^ f8t_swz<true>(r) : (4 * g + h) ^ f8t_swz<false>(r)) * 16;
    constexpr int AHEAD = A8 ? 4 : 1;         // row tiles of weights that a block begins with
    u32x4 wr[4][2], x0[XR];                   // codes of the weights, the first x tile: read before their block begins
    float sx[SX ? TN : 1];
    auto begin = [&](const uint8_t *from) {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
#pragma unroll
            for (int h = 0; h < 2; ++h) wr[a][h] = *reinterpret_cast<const u32x4 *>(from + wat + a * 2048 + h * 1024);
#pragma unroll
        for (int h = 0; h < XR; ++h) x0[h] = *reinterpret_cast<const u32x4 *>(from + xat[h]);
        if constexpr (SX) {
#pragma unroll
            for (int b = 0; b < TN; ++b) sx[b] = *reinterpret_cast<const float *>(from + (A_INS + B_INS) * 1024 + (n0 + b * 16) * 4);
        }
    };
    float fw = scale_of(0), fl = 0.f;
    f32x4 sl[4] = {};                         // the last tile's sums, of the block before
    int buf = 0;
    wait_vmcnt<(NST - 2) * OPS>();            // this wave's copies of the first block
    __builtin_amdgcn_s_barrier();
    begin(smem);
    for (int c = 0; c < steps; ++c) {
        const Step next = step_of(c + NST - 1);
        const uint8_t *from = smem + buf * STAGE;
        uint8_t *to = smem + (buf == 0 ? NST - 1 : buf - 1) * STAGE;
        buf = buf + 1 == NST ? 0 : buf + 1;
        copy_scales(next, to);
        const float f0 = fw;
        fw = scale_of(c + 1);
        u32x4 w[4][2], xr[TN][XR];
        u32x4 wf[A8 ? 1 : 4][4];              // the weights converted
        f32x4 s[TN][4];
        float f[TN];
#pragma unroll
        for (int b = 0; b < TN; ++b) f[b] = SX ? sx[SX ? b : 0] * f0 : f0;
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
#pragma unroll
            for (int h = 0; h < 2; ++h) w[a][h] = wr[a][h];
#pragma unroll
        for (int h = 0; h < XR; ++h) xr[0][h] = x0[h];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int b = 0; b < TN; ++b) {
            if (b + 1 < TN) {
#pragma unroll
                for (int h = 0; h < XR; ++h) xr[b + 1][h] = *reinterpret_cast<const u32x4 *>(from + xat[h] + (b + 1) * 16 * XB);
            } else {
                // the block is read: before its last tile's products the next one's copies are waited for, its
                // first reads run beside them, and this buffer is free
                wait_vmcnt<(NST - 2) * OPS>();
                __builtin_amdgcn_s_waitcnt(0xC07F);         // lgkmcnt(0)
                __builtin_amdgcn_s_barrier();
                begin(smem + buf * STAGE);
            }
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                if constexpr (A8) {
                    s[b][a] = f8_mma16(f8_pair(w[a][0], w[a][1]), f8_pair(xr[b][0], xr[b][1]));
                } else {
                    if (b == 0) {
                        if (a + 1 < 4) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) w[a + 1][h] = *reinterpret_cast<const u32x4 *>(from + wat + (a + 1) * 2048 + h * 1024);
                        }
#pragma unroll
                        for (int h = 0; h < 4; ++h) wf[a][h] = f8_operand<A8 ? kOpBF16 : OP>(w[a][h / 2][h % 2 * 2], w[a][h / 2][h % 2 * 2 + 1]);
                    }
                    s[b][a] = f32x4{};
                    if (b == 0 || a % 2 == 0) continue;
                    // two chains of four at a time: a product waits for the one before it
#pragma unroll
                    for (int h = 0; h < 4; ++h)
#pragma unroll
                        for (int i = a - 1; i <= a; ++i) s[b][i] = mx_mma16<A8 ? kOpBF16 : OP>(wf[i][h], xr[b][h], s[b][i]);
                }
            }
            if constexpr (!A8) {
                if (b == 0) {
#pragma unroll
                    for (int a = 0; a < 4; ++a)
#pragma unroll
                        for (int h = 0; h < 4; ++h) s[0][a] = mx_mma16<A8 ? kOpBF16 : OP>(wf[a][h], xr[0][h], s[0][a]);
                }
            }
#pragma unroll
            for (int j = b * PER; j < (b + 1) * PER && j < CPW; ++j) copy(next, to, j);
            // the sums of the tile before enter the accumulators
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (b > 0) acc[a][b - 1][i] = __builtin_fmaf(f[b > 0 ? b - 1 : 0], s[b > 0 ? b - 1 : 0][a][i], acc[a][b - 1][i]);
                    else acc[a][TN - 1][i] = __builtin_fmaf(fl, sl[a][i], acc[a][TN - 1][i]);
                }
            // the compiler is held to: beside a tile's products the reads of the next, some copies (all at once they
            // would keep every wave of the CU from its products) and the multiply-adds of the last tile (the
            // first tile's: the weights' conversions), in a region of their own for each tile
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                if (!A8 && b == 0) {
                    if (a + 1 < 4) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 20, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
                    if (TN > 1) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    if (a < PER) __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
                } else if (!A8) {
                    if (a % 2) continue;
                    __builtin_amdgcn_sched_group_barrier(0x008, 8, 0);
                    if (b + 1 < TN) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                    else __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
                    if (b * PER < CPW) __builtin_amdgcn_sched_group_barrier(0x010, (PER + 1) / 2, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);
                } else {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    if (b + 1 == TN) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                    else if (a < 2) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    if (b * PER + a < CPW && a < PER) __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
                }
            }
#pragma unroll
            for (int a = 0; a < 4; ++a) asm volatile("" : "+v"(acc[a][b > 0 ? b - 1 : TN - 1]));
            __builtin_amdgcn_sched_barrier(0);
        }
        fl = f[TN - 1];
#pragma unroll
        for (int a = 0; a < 4; ++a) sl[a] = s[TN - 1][a];
    }
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[a][TN - 1][i] = __builtin_fmaf(fl, sl[a][i], acc[a][TN - 1][i]);
    wait_vmem();

    if constexpr (OP == kOpBF16) {
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b = 0; b < TN; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[a][b][i] *= kF8Up;
    }
    if (unit >= 0 && p.splits > 1) {
        float *dst = p.part + int64_t(unit) * (BN * kF8tRows) + (wave * 4 * TN * 64 + lane) * 4;
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b = 0; b < TN; ++b) *reinterpret_cast<f32x4 *>(dst + (a * TN + b) * 256) = acc[a][b];
        return;
    }
    // register i of lane l: weight row 4 * (l / 16) + i, x row l % 16
    const bool al = (p.OUT & 3) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
#pragma unroll
    for (int b = 0; b < TN; ++b) {
        const int n = wn * (BN / 2) + 16 * b + r;
        if (n >= nrows) continue;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const int o = ow + 16 * a + 4 * g;
            if (o >= p.OUT) continue;
            const float v[4] = {acc[a][b][0], acc[a][b][1], acc[a][b][2], acc[a][b][3]};
            mx_store4(p.y, p.y_type, (row0 + n) * p.OUT + o, v, int(min(int64_t(4), p.OUT - o)), al);
        }
    }
}

// Sum of the K slices of tile full + blockIdx.y in slice order, four outputs a thread.
template <int BN>
__global__ void __launch_bounds__(256) k_f8_reduce(const F8tArgs p) {
    constexpr int TN = BN / 32;
    const int e = int(blockIdx.x) * 256 + int(threadIdx.x);             // (wave, a, b, lane)
    const int t = p.full + int(blockIdx.y);
    const float *src = p.part + int64_t(blockIdx.y) * p.splits * (BN * kF8tRows) + e * 4;
    f32x4 v = *reinterpret_cast<const f32x4 *>(src);
    for (int s = 1; s < p.splits; ++s) {
        const f32x4 w = *reinterpret_cast<const f32x4 *>(src + int64_t(s) * (BN * kF8tRows));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += w[i];
    }
    const int lane = e & 63, b = (e >> 6) % TN, a = (e >> 6) / TN % 4, wave = (e >> 6) / (TN * 4);
    const int64_t n = int64_t(t % p.nt) * BN + (wave >> 2) * (BN / 2) + 16 * b + (lane & 15);
    const int o = t / p.nt * kF8tRows + (wave & 3) * 64 + 16 * a + 4 * (lane >> 4);
    if (n >= p.N || o >= p.OUT) return;
    const float q[4] = {v[0], v[1], v[2], v[3]};
    const bool al = (p.OUT & 3) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
    mx_store4(p.y, p.y_type, n * p.OUT + o, q, int(min(int64_t(4), p.OUT - o)), al);
}

}  // namespace vqk
