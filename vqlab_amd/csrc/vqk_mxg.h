// Products of MXFP4 weights with many rows: decoded in registers, multiplied
// on 32x32x16 bf16 matrix instructions.
//
// A workgroup of four waves takes 256 weight rows (128 of each projection of a
// SwiGLU pair) and a tile of 32 * BT x rows; a wave owns 64 weight rows and all
// of the tile's x rows, so every weight is decoded by one wave only. Per chunk
// of 128 k:
//   * weights: 32 bytes per lane and 32-row tile straight from global memory,
//     in operand order. Lane group g = lane / 32 holds blocks 2g and 2g + 1 of
//     the chunk and step (q, h) multiplies elements 8h..8h+7 of block 2g + q: a
//     lane decodes with one scale per block.
//   * x: the tile's 256-byte row pieces, copied global -> LDS without registers
//     (16 bytes a lane); piece p of row n is stored at p ^ (n & 15), so the 16
//     rows of a read phase fall on 16 different bank groups.
// The loads of the next chunk are in flight while one multiplies; two
// workgroups share a CU and fill each other's waits. The four conversions of a
// fragment (v_cvt_scalef32_pk_bf16_fp4) issue in the shadow of the matrix
// instructions: one conversion for each of them at BT = 4.
// The loop exists for every number of 32-row groups that a tile may hold: a
// routed expert's last rows cost what they are. x in planes (fp16 beyond exact
// weights, fp32): the chunk's planes one after the other, weights loaded once.
#pragma once

#include <type_traits>

#include "vqk_mxs.h"

namespace vqk {

typedef float f32x16v __attribute__((ext_vector_type(16)));

constexpr int kMxgWaves = 4;
constexpr int kMxgRows = 256;                 // weight rows per workgroup

struct MxgArgs {
    MxsArgs a;
    int32_t ntiles_host;                      // x tiles when they are not counted on the device
    int32_t planes;                           // bf16 planes of x
    int32_t splits, per;                      // K slices and chunks in each (splits = 1: none)
    float *part;                              // [splits][N][OUT] when splits > 1
};

template <int OP>
__device__ __forceinline__ f32x16v mx_mma32(u32x4 w, u32x4 x, f32x16v c) {
    if constexpr (OP == kOpBF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(mx_b8, w), __builtin_bit_cast(mx_b8, x), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, w), __builtin_bit_cast(h8, x), c, 0, 0, 0);
}

// PL: x in more planes than one.
template <int OP, int BT, bool GLU, bool PL>
__global__ void __launch_bounds__(64 * kMxgWaves, 2) k_mx_gemm(const MxgArgs ga) {
    const MxsArgs &p = ga.a;
    constexpr int ROWS = 32 * BT;
    constexpr int STAGE = ROWS * 256;         // bytes of x per chunk
    constexpr int CPW = STAGE / 1024 / kMxgWaves;
    static_assert(CPW * kMxgWaves * 1024 == STAGE, "whole copies per wave");
    extern __shared__ __align__(16) uint8_t xs[];       // [2][STAGE]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 31, g = lane >> 5;

    // tiles in contiguous bands per XCD (workgroup b runs on XCD b % 8)
    const int nt = p.meta ? p.ntiles[0] : ga.ntiles_host;
    const int total = nt * p.nob * ga.splits;
    int t = int(blockIdx.x);
    if (t >= total) return;
    {
        const int x = t % 8, q = total / 8, rest = total % 8;
        t = x * q + min(x, rest) + t / 8;
    }
    const int slice = t % ga.splits;
    t /= ga.splits;
    const int tt = p.meta ? t / p.nob : t % nt, ob = p.meta ? t % p.nob : t / nt;
    MxTile tile;
    if (!mx_tile<ROWS>(p, tt, &tile)) return;
    const int o0 = ob * (GLU ? kMxgRows / 2 : kMxgRows);
    const int ow = o0 + wave * (GLU ? 32 : 64);         // this wave's first output
    const int c_lo = slice * ga.per, c_hi = min(p.NC, c_lo + ga.per);

    f32x16v acc[2][BT];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < BT; ++b) acc[a][b] = f32x16v{};
    bool nan[2] = {};

    if (tile.expert >= 0) {
        // unit of block 2g in this lane's row tile; the second block's is 16 further
        const uint32_t NC = uint32_t(p.NC), NC4 = (NC + 3) / 4;
        const uint8_t *cb[2], *sb[2];
        uint32_t wo[2], so[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const int m = GLU ? a : 0;
            cb[a] = p.codes[m] + int64_t(tile.expert) * mx_expert_codes(p.RT, p.NC);
            sb[a] = p.scales[m] + int64_t(tile.expert) * mx_expert_scales(p.RT, p.NC);
            const uint32_t rt = uint32_t(min((ow + (GLU ? 0 : 32 * a)) / 16 + (r >> 4), p.RT - 1));
            const uint32_t unit = uint32_t(2 * g * 16 + (r & 15));
            wo[a] = (rt * NC * 64 + unit) * 16;
            so[a] = (rt * NC4 * 64 + unit) * 4;
        }
        // the x copies of this lane: 16 bytes of one row each
        const uint16_t *src[CPW];
        int piece[CPW];
#pragma unroll
        for (int j = 0; j < CPW; ++j) {
            const int n = (j * kMxgWaves + wave) * 4 + (lane >> 4);
            piece[j] = (lane & 15) ^ (n & 15);
            src[j] = p.x + int64_t(mx_x_row(p, tile.row0 + min(n, tile.nrows - 1))) * p.xld + piece[j] * 8;
        }
        // NA: groups of 32 rows that the tile holds
        auto issue = [&](int c, int pl, int buf, auto na) {
#pragma unroll
            for (int j = 0; j < 2 * decltype(na)::value; ++j) {
                // past the row's last block: the row's start again (multiplied by no weight, masked below)
                const bool in = 4 * c + piece[j] / 4 < p.NB;
                const uint16_t *s = src[j] + pl * p.xplane + (in ? int64_t(c) * kMxChunk : -int64_t(piece[j] * 8));
                __builtin_amdgcn_global_load_lds((global_void *)s,
                                                 (lds_void *)(xs + buf * STAGE + (j * kMxgWaves + wave) * 1024), 16, 0, 0);
            }
        };
        u32x4 w[2][2], wn[2][2];
        uint32_t s[2][2], sn[2][2];
        auto load_w = [&](int c, u32x4 (&ww)[2][2], uint32_t (&ss)[2][2]) {
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    ww[a][q] = *reinterpret_cast<const u32x4 *>(cb[a] + (wo[a] + uint32_t(c) * 1024u + q * 256u));
                    ss[a][q] = sb[a][so[a] + uint32_t(c / 4) * 256u + q * 64u + uint32_t(c % 4)];
                }
        };
        auto mul = [&](int c, int buf, auto na) {
            const bool tail = 4 * c + 4 > p.NB;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float sc[2];
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    nan[a] = nan[a] || s[a][q] == 255u;
                    sc[a] = mx_scale(s[a][q] == 255u ? 127u : s[a][q]);
                }
                const bool in = !tail || 4 * c + 2 * g + q < p.NB;
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    u32x4 wf[2];
#pragma unroll
                    for (int a = 0; a < 2; ++a) wf[a] = mx_decode8_op<OP>(w[a][q][h], sc[a]);
                    const int at = ((8 * g + 4 * q + h) ^ (lane & 15)) * 16 + r * 256;
#pragma unroll
                    for (int b = 0; b < decltype(na)::value; ++b) {
                        u32x4 xv = *reinterpret_cast<const u32x4 *>(xs + buf * STAGE + b * 8192 + at);
                        if (tail && !in) xv = u32x4{};
#pragma unroll
                        for (int a = 0; a < 2; ++a) acc[a][b] = mx_mma32<OP>(wf[a], xv, acc[a][b]);
                    }
                }
            }
        };
        // steps: chunk c_lo + step / P, plane step % P
        auto walk = [&](auto na) {
            const int P = PL ? ga.planes : 1, steps = (c_hi - c_lo) * P;
            if (steps > 0) {
                issue(c_lo, 0, 0, na);
                load_w(c_lo, wn, sn);
            }
            int c = c_lo, pl = 0;
#pragma unroll 1
            for (int step = 0; step < steps; ++step) {
                wait_vmem();                  // this wave's copies of the step, and its weights
                __syncthreads();              // every wave's copies; every wave is done with the other buffer
                if (!PL || pl == 0) {
#pragma unroll
                    for (int a = 0; a < 2; ++a)
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            w[a][q] = wn[a][q];
                            s[a][q] = sn[a][q];
                        }
                }
                const int cc = c;
                if (!PL || ++pl == P) {
                    pl = 0;
                    ++c;
                }
                if (step + 1 < steps) {
                    issue(c, pl, (step + 1) & 1, na);
                    if (!PL || pl == 0) load_w(c, wn, sn);
                }
                mul(cc, step & 1, na);
            }
        };
        const int groups = (tile.nrows + 31) / 32;
        if (BT > 1 && groups <= 1) walk(std::integral_constant<int, 1>{});
        else if (BT > 2 && groups == 2) walk(std::integral_constant<int, (BT > 2 ? 2 : BT)>{});
        else if (BT > 3 && groups == 3) walk(std::integral_constant<int, (BT > 3 ? 3 : BT)>{});
        else walk(std::integral_constant<int, BT>{});
    }

    // register i of lane l: weight row 8 * (i / 4) + 4 * (l / 32) + i % 4, x row l % 32. A NaN block
    // makes its output NaN: the flag of weight row r is in lanes r and r + 32
    uint64_t nm[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        const uint64_t m = __ballot(nan[a]);
        nm[a] = (m | (m >> 32)) & 0xffffffffu;
    }
    auto value = [&](int a, int b, int i) {
        const int o = 8 * (i / 4) + 4 * g + i % 4;
        return (nm[a] >> o) & 1 ? __uint_as_float(0x7fc00000u) : acc[a][b][i];
    };
#pragma unroll
    for (int b = 0; b < BT; ++b) {
        const int n = 32 * b + r;
        if (n >= tile.nrows) continue;
        const int64_t yr = mx_y_row(p, tile.row0 + n);
        if constexpr (GLU) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int o = ow + 8 * j + 4 * g;
                if (o >= p.ocover) continue;  // ocover is whole blocks of 32
                float h[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float v = value(0, b, 4 * j + i), u = value(1, b, 4 * j + i);
                    h[i] = o + i < p.OUT ? mx_swiglu(v, u) : 0.f;
                }
                for (int pl = 0; pl < (OP == kOpF16 ? 1 : p.yp); ++pl) {
                    uint16_t q[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) q[i] = OP == kOpF16 ? f32_to_h(h[i]) : mx_plane_next(h[i]);
                    u32x2 v2;
                    v2.x = q[0] | (uint32_t(q[1]) << 16);
                    v2.y = q[2] | (uint32_t(q[3]) << 16);
                    *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(p.y) + pl * p.yplane + yr * p.ldy + o) = v2;
                }
            }
        } else {
            void *y = ga.splits > 1 ? static_cast<void *>(ga.part + int64_t(slice) * p.N * p.OUT) : p.y;
            const int32_t yt = ga.splits > 1 ? VQK_F32 : p.y_type;
            const bool al = (p.ldy & 3) == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0;
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int o = ow + 32 * a + 8 * j + 4 * g;
                    if (o >= p.OUT) continue;
                    float v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = value(a, b, 4 * j + i);
                    mx_store4(y, yt, yr * p.ldy + o, v, int(min(int64_t(4), p.OUT - o)), al);
                }
        }
    }
}

}  // namespace vqk
