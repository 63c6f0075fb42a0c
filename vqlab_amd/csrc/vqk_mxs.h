// Products of MXFP4 weights with few rows of x: the weights are streamed once
// past up to 16 * NT rows.
//
//     y[n, o] = sum_k x[n, k] * W[o, k]
//
// A workgroup keeps its tile of x in registers and walks over weight rows, so
// its loop is the weight stream and little else. Eight waves: KW along k, NCW
// chunks of 128 each (x takes 16 * NCW * NT * P registers), and 8 / KW along the
// weight rows, 16 a step. The next step's weights (16 bytes a lane and chunk, a
// contiguous KB a wave) load while the last ones are decoded and multiplied. The
// fp32 sums of KW > 1 waves meet in LDS in wave order, two buffers in turn, one
// barrier a step.
// x comes straight from its rows where a tile has at most two, and otherwise
// through LDS, copied in whole lines and read in operand order (16 rows read
// directly cost 64 L1 cycles a load: 8 us of a 20-row product).
// Bound by HBM: a wave decodes and multiplies a 16 x 128 piece (1088 bytes) in
// ~100 cycles, several times the rate at which it can arrive.
#pragma once

#include "vqk_mx.h"

namespace vqk {

constexpr int kMxsWaves = 8;

struct MxsArgs {
    const uint8_t *codes[2], *scales[2];
    int64_t OUT, E;
    int32_t RT, NC, NB;
    const uint16_t *x;
    int64_t xld, xplane;
    int64_t N;
    int32_t xkrep;
    const int32_t *ids, *order, *meta, *ntiles;
    void *y;
    int32_t y_type, yp, ysorted;
    int64_t ldy, yplane, ocover;              // columns of y to write (OUT, or its padding to whole blocks)
    int32_t nob;                              // workgroups per tile
    // k_mx_rows: waves along k, row steps per workgroup and in all, x through LDS
    int32_t kw, steps, total_steps, stage;
};

// Rows of x that a tile multiplies, and where they lie.
struct MxTile {
    int expert;                               // < 0: none (rows of zeros)
    int row0, nrows;
};
template <int ROWS>
__device__ __forceinline__ bool mx_tile(const MxsArgs &p, int t, MxTile *out) {
    if (p.meta) {
        if (t >= p.ntiles[0]) return false;
        *out = MxTile{p.meta[3 * t], p.meta[3 * t + 1], p.meta[3 * t + 2]};
        if (out->nrows < 1) return false;
    } else if (p.ids) {
        const int e = p.ids[t];
        *out = MxTile{e >= 0 && e < p.E ? e : -1, t, 1};
    } else {
        const int r = t * ROWS;
        *out = MxTile{0, r, int(min(int64_t(ROWS), p.N - r))};
    }
    out->expert = __builtin_amdgcn_readfirstlane(out->expert);
    out->row0 = __builtin_amdgcn_readfirstlane(out->row0);
    out->nrows = __builtin_amdgcn_readfirstlane(out->nrows);
    return true;
}
// Tile positions -> rows of x / of y, in place; the loads of one call run together.
template <int N>
__device__ __forceinline__ void mx_x_rows(const MxsArgs &p, int (&pos)[N]) {
    if (p.xkrep == 0) return;
    if (p.meta) {
#pragma unroll
        for (int i = 0; i < N; ++i) pos[i] = load_global(p.order, pos[i]);
    }
    if (p.xkrep != 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) pos[i] = int(uint32_t(pos[i]) / uint32_t(p.xkrep));
    }
}
template <int N>
__device__ __forceinline__ void mx_y_rows(const MxsArgs &p, int (&pos)[N]) {
    if (!p.meta || p.ysorted) return;
#pragma unroll
    for (int i = 0; i < N; ++i) pos[i] = load_global(p.order, pos[i]);
}

template <int OP>
__device__ __forceinline__ f32x4 mx_mma16(u32x4 x, u32x4 w, f32x4 c) {
    if constexpr (OP == kOpBF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mx_b8, x), __builtin_bit_cast(mx_b8, w), c,
                                                       0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, w), c, 0, 0, 0);
}
__device__ __forceinline__ float mx_swiglu(float g, float u) { return g / (1.f + __expf(-g)) * u; }

template <int OP, int NT, int P, int NCW, bool GLU>
__global__ void __launch_bounds__(64 * kMxsWaves, 2) k_mx_rows(const MxsArgs p) {
    constexpr int TT = GLU ? 2 : 1;
    // sums [2][8 waves][TT * NT][256] floats (KW > 1); before them x, [8 waves][16 rows][NCW * 256 bytes]
    extern __shared__ __align__(16) uint8_t smem[];
    float *red = reinterpret_cast<float *>(smem);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int KW = p.kw, RW = kMxsWaves / KW;
    const int kw = wave % KW, rw = wave / KW;
    const int t = int(blockIdx.x / unsigned(p.nob)), part = int(blockIdx.x % unsigned(p.nob));
    MxTile tile;
    if (!mx_tile<16 * NT>(p, t, &tile)) return;
    const int s_lo = part * p.steps, s_hi = min(p.total_steps, s_lo + p.steps);
    if (s_lo >= s_hi) return;

    const bool live = tile.expert >= 0;
    const int64_t ex = live ? tile.expert : 0;
    const uint8_t *cb[2], *sb[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        cb[a] = p.codes[a] + ex * mx_expert_codes(p.RT, p.NC);
        sb[a] = p.scales[a] + ex * mx_expert_scales(p.RT, p.NC);
    }
    // this wave's chunks: kw * NCW ..; past the last one the last stands in, and for a pair without
    // an expert expert 0: against x of zero, and under a scale of 1, because a weight of 2^128 or
    // more decodes to infinity, which zero does not cancel
    const uint32_t NC = uint32_t(p.NC), NC4 = (NC + 3) / 4;
    u32x4 w[TT][NCW], wn[TT][NCW];
    uint32_t sc[TT][NCW], scn[TT][NCW];
    auto load_w = [&](int step) {
        const uint32_t rt = uint32_t(min(step * RW + rw, p.RT - 1));
#pragma unroll
        for (int a = 0; a < TT; ++a)
#pragma unroll
            for (int c = 0; c < NCW; ++c) {
                const uint32_t ch = min(uint32_t(kw * NCW + c), NC - 1);
                wn[a][c] = *reinterpret_cast<const u32x4 *>(cb[a] + ((rt * NC + ch) * 64 + lane) * 16u);
                scn[a][c] = sb[a][((rt * NC4 + ch / 4) * 64 + lane) * 4 + ch % 4];
            }
    };
    load_w(s_lo);

    u32x4 xf[P][NT][NCW][4];
    auto x_in = [&](int c) { return 4 * (kw * NCW + c) + g < p.NB; };   // this lane's block of x exists
    if (p.stage) {                            // dense rows: a tile's lie one after the other
        uint8_t *xl = smem + wave * (NCW * 4096);
#pragma unroll
        for (int pl = 0; pl < P; ++pl)
#pragma unroll
            for (int b = 0; b < NT; ++b) {
#pragma unroll
                for (int i = 0; i < 4 * NCW; ++i) {
                    // LDS unit i * 64 + lane: row / 16-byte slot; the slot holds piece slot ^ row of the
                    // wave's part of that row (past the row's end its start: zeroed below)
                    const int u = i * 64 + lane, row = u / (16 * NCW), piece = (u % (16 * NCW)) ^ row;
                    const int64_t k = int64_t(kw) * NCW * kMxChunk + piece * 8;
                    if (b * 16 + row < tile.nrows) {          // else the unit stays as it is: zeroed below
                        const uint16_t *src = p.x + pl * p.xplane + int64_t(tile.row0 + b * 16 + row) * p.xld +
                                              (k < int64_t(p.NB) * kMxBlock ? k : 0);
                        __builtin_amdgcn_global_load_lds((global_void *)src, (lds_void *)(xl + i * 1024), 16, 0, 0);
                    }
                }
                wait_vmem();
#pragma unroll
                for (int c = 0; c < NCW; ++c)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const u32x4 v = *reinterpret_cast<const u32x4 *>(
                            xl + r * (NCW * 256) + (((c * 16 + g * 4 + k) ^ r) << 4));
                        xf[pl][b][c][k] = live && x_in(c) && b * 16 + r < tile.nrows ? v : u32x4{};
                    }
                __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): read before the next rows land
            }
        __syncthreads();                      // the sums use the same LDS
    } else {
        int xrow[NT];
#pragma unroll
        for (int b = 0; b < NT; ++b) xrow[b] = tile.row0 + min(b * 16 + r, tile.nrows - 1);
        mx_x_rows(p, xrow);
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            const bool row_in = live && b * 16 + r < tile.nrows;
            const uint16_t *xp = p.x + int64_t(xrow[b]) * p.xld;
#pragma unroll
            for (int pl = 0; pl < P; ++pl)
#pragma unroll
                for (int c = 0; c < NCW; ++c)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        xf[pl][b][c][k] = row_in && x_in(c)
                            ? *reinterpret_cast<const u32x4 *>(xp + pl * p.xplane +
                                                               (4 * (kw * NCW + c) + g) * kMxBlock + 8 * k)
                            : u32x4{};
        }
    }

    for (int step = s_lo; step < s_hi; ++step) {
#pragma unroll
        for (int a = 0; a < TT; ++a)
#pragma unroll
            for (int c = 0; c < NCW; ++c) {
                w[a][c] = wn[a][c];
                sc[a][c] = scn[a][c];
            }
        if (step + 1 < s_hi) load_w(step + 1);
        f32x4 acc[TT][NT];
#pragma unroll
        for (int a = 0; a < TT; ++a) {
            bool nan = false;
#pragma unroll
            for (int b = 0; b < NT; ++b) acc[a][b] = f32x4{};
#pragma unroll
            for (int c = 0; c < NCW; ++c) {
                const uint32_t e = live && uint32_t(kw * NCW + c) < NC ? sc[a][c] : 127u;
                nan = nan || e == 255u;
                const float s = mx_scale(e == 255u ? 127u : e);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const u32x4 wf = mx_decode8_op<OP>(w[a][c][k], s);
#pragma unroll
                    for (int pl = 0; pl < P; ++pl)
#pragma unroll
                        for (int b = 0; b < NT; ++b)
                            acc[a][b] = mx_mma16<OP>(xf[pl][b][c][k], wf, acc[a][b]);
                }
            }
            // a NaN block makes its whole output column NaN, whichever of its lane groups holds it
            if (__ballot(nan)) {
                int f = nan;
                f |= __shfl_xor(f, 16);
                f |= __shfl_xor(f, 32);
#pragma unroll
                for (int b = 0; b < NT; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[a][b][i] = f ? __uint_as_float(0x7fc00000u) : acc[a][b][i];
            }
        }
        auto put = [&](int row, int o, float v, float u) {
            int yr_[1] = {tile.row0 + row};
            mx_y_rows(p, yr_);
            const int64_t yr = yr_[0];
            if constexpr (GLU) {
                float h = o < p.OUT ? mx_swiglu(v, u) : 0.f;
                uint16_t *y = static_cast<uint16_t *>(p.y) + yr * p.ldy + o;
                for (int pl = 0; pl < p.yp; ++pl) y[pl * p.yplane] = mx_plane_next(h);
            } else {
                store_act(p.y, p.y_type, yr * p.ldy + o, v);
            }
        };
        if (KW == 1) {
            // register i of lane l: x row 4 * (l / 16) + i, weight row l % 16
            const int o = (step * RW + rw) * 16 + r;
#pragma unroll
            for (int b = 0; b < NT; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (b * 16 + 4 * g + i < tile.nrows && o < p.ocover)
                        put(b * 16 + 4 * g + i, o, acc[0][b][i], acc[TT - 1][b][i]);
            continue;
        }
        float *buf = red + (step & 1) * kMxsWaves * TT * NT * 256;
#pragma unroll
        for (int a = 0; a < TT; ++a)
#pragma unroll
            for (int b = 0; b < NT; ++b)
                *reinterpret_cast<f32x4 *>(buf + ((wave * TT + a) * NT + b) * 256 + lane * 4) = acc[a][b];
        __syncthreads();
        // outputs (x row, weight row) of the step, weight rows fastest
        const int n_out = 16 * RW;
        for (int e = threadIdx.x; e < n_out * min(tile.nrows, 16 * NT); e += 64 * kMxsWaves) {
            const int row = e / n_out, c = e - row * n_out, n = c & 15, m = row & 15, b = row >> 4;
            const int o = step * n_out + c;
            if (o >= p.ocover) continue;
            const float *src = buf + ((c >> 4) * KW * TT * NT + b) * 256 + ((m >> 2) * 16 + n) * 4 + (m & 3);
            float v = 0.f, u = 0.f;
            for (int k = 0; k < KW; ++k) {
                v += src[k * TT * NT * 256];
                if constexpr (GLU) u += src[(k * TT + 1) * NT * 256];
            }
            put(row, o, v, u);
        }
    }
}

// Kernel arguments of a call, and the tiles of `rows` x rows that it makes.
void mx_args(const MxCall &c, MxsArgs *a);
int64_t mx_tiles(const MxCall &c, int rows);
// Whether k_mx_rows takes a call in tiles of 16 * NT rows; its launch.
bool mx_rows_ok(const MxCall &c, int NT);
int mx_rows(const MxCall &c, int NT, hipStream_t st);

}  // namespace vqk
