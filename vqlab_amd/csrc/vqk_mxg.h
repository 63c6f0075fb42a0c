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
// The loads of the next chunk (or two) are in flight while one multiplies; two
// workgroups share a CU and fill each other's waits. The four conversions of a
// fragment (v_cvt_scalef32_pk_bf16_fp4) issue in the shadow of the matrix
// instructions: one conversion for each of them at BT = 4.
// The loop exists for every number of 32-row groups that a tile may hold: a
// routed expert's last rows cost what they are. x in planes (SwiGLU rows, fp16
// beyond exact weights, fp32): where a tile's rows leave room for all planes in its
// LDS stage, the planes stand there as more rows, their sums meet, and the weights
// are loaded and decoded once; otherwise one plane a step, the weights again from
// L2. (Blocks of experts whose SwiGLU rows stand in two planes: 64 tokens through
// 512 experts, one or two rows a tile, 466 us folded, 555 in turn; 2048 through 256,
// about 60 rows, 270 both ways.)
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

// How a tile of up to 32 * G rows (G = 0: 16) in P planes stands in a stage of 32 * BT
// rows: `planes` of them, `rows` apart, `groups` of 32 rows each; copies of 16 rows.
template <int BT, int P, int G>
struct MxgSpan {
    static constexpr bool half = G == 0;                  // two planes in one group
    static constexpr int groups = half ? 1 : G;
    static constexpr int planes = half ? 2 : (G * P <= BT ? P : 1);
    static constexpr int rows = half ? 16 : 32 * G;
    static constexpr int copies = rows * planes / 16;
};

// What x is past its rows' ends.
static __device__ __align__(16) uint8_t mxg_zeros[16];

// The counted waits need the loads of a stage where the source has them: none may
// move across this.
__device__ __forceinline__ void mxg_keep_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// ST: stages of x in LDS and of weights in registers (ST - 1 chunks in flight).
// P: planes of x.
template <int OP, int BT, int ST, bool GLU, int P>
__global__ void __launch_bounds__(64 * kMxgWaves, 2) k_mx_gemm(const MxgArgs ga) {
    const MxsArgs &p = ga.a;
    constexpr int ROWS = 32 * BT;
    constexpr int STAGE = ROWS * 256;         // bytes of x per chunk
    extern __shared__ __align__(16) uint8_t xs[];       // [ST][STAGE]
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
        struct Weights {
            u32x4 w[2][2];
            uint32_t s[2][2];
        };
        Weights wb[ST];
        auto walk = [&](auto span) {
            using Sp = decltype(span);
            static_assert(Sp::rows * Sp::planes <= ROWS && P % Sp::planes == 0, "whole planes in a stage");
            // the x copies of this lane: 16 bytes of one row each
            const uint16_t *src[Sp::copies];
            int piece[Sp::copies], xrow[Sp::copies];
#pragma unroll
            for (int j = 0; j < Sp::copies; ++j) {
                const int n = (j * kMxgWaves + wave) * 4 + (lane >> 4);
                xrow[j] = tile.row0 + min(n % Sp::rows, tile.nrows - 1);
            }
            mx_x_rows(p, xrow);
#pragma unroll
            for (int j = 0; j < Sp::copies; ++j) {
                const int n = (j * kMxgWaves + wave) * 4 + (lane >> 4);
                piece[j] = (lane & 15) ^ (n & 15);
                src[j] = p.x + (n / Sp::rows) * p.xplane + int64_t(xrow[j]) * p.xld + piece[j] * 8;
            }
            // steps: chunk c_lo + step / turns, plane step % turns (the weights again for each)
            constexpr int turns = P / Sp::planes;
            const int steps = (c_hi - c_lo) * turns;
            auto issue = [&](int step, auto slot) {
                const int c = c_lo + step / turns;
                constexpr int S = decltype(slot)::value;
#pragma unroll
                for (int j = 0; j < Sp::copies; ++j) {
                    // past the row's last block: zeros
                    const uint16_t *from = src[j] + (step % turns) * p.xplane + int64_t(c) * kMxChunk;
                    from = 4 * c + piece[j] / 4 < p.NB ? from : reinterpret_cast<const uint16_t *>(mxg_zeros);
                    __builtin_amdgcn_global_load_lds((global_void *)from,
                                                     (lds_void *)(xs + S * STAGE + (j * kMxgWaves + wave) * 1024), 16, 0, 0);
                }
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        wb[S].w[a][q] = *reinterpret_cast<const u32x4 *>(cb[a] + (wo[a] + uint32_t(c) * 1024u + q * 256u));
                        wb[S].s[a][q] = *reinterpret_cast<const uint32_t *>(sb[a] + (so[a] + uint32_t(c / 4) * 256u + q * 64u));
                    }
            };
            auto mul = [&](int step, auto slot) {
                constexpr int S = decltype(slot)::value;
                const Weights &d = wb[S];
                const int c = c_lo + step / turns;
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    float sc[2];
#pragma unroll
                    for (int a = 0; a < 2; ++a) {
                        const uint32_t b = (d.s[a][q] >> (8 * (c & 3))) & 255u;
                        nan[a] = nan[a] || b == 255u;
                        sc[a] = mx_scale(b == 255u ? 127u : b);
                    }
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        u32x4 wf[2];
#pragma unroll
                        for (int a = 0; a < 2; ++a) wf[a] = mx_decode8_op<OP>(d.w[a][q][h], sc[a]);
                        const int at = ((8 * g + 4 * q + h) ^ (lane & 15)) * 16 + r * 256;
#pragma unroll
                        for (int b = 0; b < Sp::copies / 2; ++b) {
                            const u32x4 xv = *reinterpret_cast<const u32x4 *>(xs + S * STAGE + b * 8192 + at);
#pragma unroll
                            for (int a = 0; a < 2; ++a)
                                acc[a][b % Sp::groups] = mx_mma32<OP>(wf[a], xv, acc[a][b % Sp::groups]);
                        }
                    }
                }
            };
            constexpr int OPS = Sp::copies + 8;           // loads of a stage
            using s0 = std::integral_constant<int, 0>;
            using s1 = std::integral_constant<int, 1>;
            using s2 = std::integral_constant<int, ST - 1>;
            // past the last step it is loaded again, into a slot that no step reads, and the steps run in
            // whole rounds of the slots: on every path a step issues the same loads, so that the counted
            // wait stands for the compiler as well (it adds none of its own)
            auto one = [&](int step, auto slot) {
                // this wave's loads of the step (those of the next may be on their way), then every
                // wave's; every wave is done with the slot that is filled next
                mxg_keep_order();
                wait_vmcnt<(ST - 2) * OPS>();
                __builtin_amdgcn_s_waitcnt(0xC07F);       // lgkmcnt(0): this wave's reads of that slot
                __builtin_amdgcn_s_barrier();             // (a __syncthreads would wait for every load)
                mxg_keep_order();
                issue(min(step + ST - 1, steps - 1),
                      std::integral_constant<int, (decltype(slot)::value + ST - 1) % ST>{});
                mxg_keep_order();
                if (step < steps) mul(step, slot);
            };
            if (steps <= 0) return;
            issue(0, s0{});
            mxg_keep_order();
            if constexpr (ST == 3) {
                issue(min(1, steps - 1), s1{});
                mxg_keep_order();
            }
#pragma unroll 1
            for (int step = 0; step < steps; step += ST) {
                one(step, s0{});
                one(step + 1, s1{});
                if constexpr (ST == 3) one(step + 2, s2{});
            }
            wait_vmem();
            if constexpr (Sp::half) {                     // the second plane's sums are 16 lanes further
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[a][0][i] += __shfl_xor(acc[a][0][i], 16);
            }
        };
        const int groups = (tile.nrows + 31) / 32;
        if (BT == 1 && P == 2 && tile.nrows <= 16) {
            if constexpr (BT == 1 && P == 2) walk(MxgSpan<BT, P, 0>{});
        } else if (BT > 1 && groups <= 1) walk(MxgSpan<BT, P, 1>{});
        else if (BT > 2 && groups == 2) walk(MxgSpan<BT, P, (BT > 2 ? 2 : BT)>{});
        else if (BT > 3 && groups == 3) walk(MxgSpan<BT, P, (BT > 3 ? 3 : BT)>{});
        else walk(MxgSpan<BT, P, BT>{});
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
    if (GLU && ow >= p.ocover) return;        // whole blocks of 32, as ow is
    int yrow[BT];
#pragma unroll
    for (int b = 0; b < BT; ++b) yrow[b] = tile.row0 + min(32 * b + r, tile.nrows - 1);
    mx_y_rows(p, yrow);
#pragma unroll
    for (int b = 0; b < BT; ++b) {
        const int n = 32 * b + r;
        if (n >= tile.nrows) continue;
        const int64_t yr = yrow[b];
        if constexpr (GLU) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int o = ow + 8 * j + 4 * g;
                float h[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float v = value(0, b, 4 * j + i), u = value(1, b, 4 * j + i);
                    h[i] = o + i < p.OUT ? mx_swiglu(v, u) : 0.f;
                }
                for (int pl = 0; pl < p.yp; ++pl) {
                    uint16_t q[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) q[i] = mx_plane_next(h[i]);
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
