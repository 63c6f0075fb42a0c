// Products of MXFP4 weights with a few rows at a time: each weight is read
// once for up to 16 * NT rows.
//
//     y[n, o] = sum_k x[n, k] * W[o, k]
//
// A workgroup takes 16 * MT weight rows (of each projection of a SwiGLU pair)
// and a tile of x rows; its waves split k by chunks of 128 (wave w takes
// chunks w, w + NW, ...: side by side they read whole lines of a row) and
// their fp32 sums meet in LDS, added in wave order. Weights go from global
// memory to matrix-core operands in registers (vqk_mx.h); x pieces come from
// L2 in the same order, so nothing is staged. Bound by the weight stream: a
// wave decodes and multiplies a 16 x 128 piece (1088 bytes) in ~100 cycles,
// several times the rate at which HBM delivers them.
#pragma once

#include "vqk_mx.h"

namespace vqk {

constexpr int kMxsMaxWaves = 8;

struct MxsArgs {
    const uint8_t *codes0, *scales0, *codes1, *scales1;
    int64_t NB, OUT, E;
    int32_t NC, nob;                          // chunks of k; output blocks of 16 * MT rows
    const uint16_t *x;
    int64_t xld, xplane;
    int64_t N, xkrep;
    const int32_t *ids, *order, *meta, *ntiles;
    void *y;
    int32_t y_type, yp, ysorted;
    int64_t ldy, yplane, ocover;              // columns of y to write (OUT, or its padding to whole blocks)
};

// Rows of x that a tile multiplies, and where they lie.
struct MxTile {
    int64_t expert;                           // < 0: no expert (rows of zeros)
    int64_t row0;
    int nrows;
};
template <int ROWS>
__device__ __forceinline__ bool mx_tile(const MxsArgs &p, int t, MxTile *out) {
    if (p.meta) {
        if (t >= p.ntiles[0]) return false;
        *out = MxTile{p.meta[3 * t], p.meta[3 * t + 1], p.meta[3 * t + 2]};
        if (out->nrows < 1) return false;
    } else if (p.ids) {
        const int64_t e = p.ids[t];
        *out = MxTile{e >= 0 && e < p.E ? e : -1, t, 1};
    } else {
        const int64_t r = int64_t(t) * ROWS;
        *out = MxTile{0, r, int(min(int64_t(ROWS), p.N - r))};
    }
    return true;
}
__device__ __forceinline__ int64_t mx_x_row(const MxsArgs &p, int64_t pos) {
    if (p.xkrep == 0) return pos;
    const int64_t pair = p.meta ? p.order[pos] : pos;
    return p.xkrep == 1 ? pair : pair / p.xkrep;
}
__device__ __forceinline__ int64_t mx_y_row(const MxsArgs &p, int64_t pos) {
    return p.meta && !p.ysorted ? p.order[pos] : pos;
}

template <int NT, int MT, bool GLU, int P>
__global__ void __launch_bounds__(64 * kMxsMaxWaves) k_mx_stream(const MxsArgs p) {
    constexpr int TT = GLU ? 2 * MT : MT;
    extern __shared__ __align__(16) float red[];      // [waves][TT * NT][256]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, NW = blockDim.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int ob = int(blockIdx.x % unsigned(p.nob)), t = int(blockIdx.x / unsigned(p.nob));
    MxTile tile;
    if (!mx_tile<16 * NT>(p, t, &tile)) return;
    const int o0 = ob * 16 * MT;

    f32x4 acc[TT][NT];
#pragma unroll
    for (int a = 0; a < TT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = f32x4{};
    bool nan[TT] = {};
    if (tile.expert >= 0) {
        const uint8_t *wp[TT], *sp[TT];
#pragma unroll
        for (int a = 0; a < TT; ++a) {
            const int64_t row = tile.expert * p.OUT + min(int64_t(o0 + (a % MT) * 16 + r), p.OUT - 1);
            wp[a] = (a < MT ? p.codes0 : p.codes1) + row * p.NB * 16;
            sp[a] = (a < MT ? p.scales0 : p.scales1) + row * p.NB;
        }
        const uint16_t *xp[NT];
#pragma unroll
        for (int b = 0; b < NT; ++b)
            xp[b] = p.x + mx_x_row(p, tile.row0 + min(b * 16 + r, tile.nrows - 1)) * p.xld;
        for (int c = wave; c < p.NC; c += NW) {
            const int64_t blk = 4 * c + g;
            const bool ok = blk < p.NB;
            u32x4 w[TT];
            uint32_t s[TT];
#pragma unroll
            for (int a = 0; a < TT; ++a) {
                w[a] = ok ? *reinterpret_cast<const u32x4 *>(wp[a] + blk * 16) : u32x4{};
                s[a] = ok ? sp[a][blk] : 127u;
            }
            u32x4 xf[P][NT][4];
#pragma unroll
            for (int pl = 0; pl < P; ++pl)
#pragma unroll
                for (int b = 0; b < NT; ++b)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        xf[pl][b][k] = ok ? *reinterpret_cast<const u32x4 *>(xp[b] + pl * p.xplane +
                                                                             blk * kMxBlock + 8 * k)
                                          : u32x4{};
#pragma unroll
            for (int a = 0; a < TT; ++a) {
                nan[a] = nan[a] || s[a] == 255u;
                const float sc = mx_scale(s[a] == 255u ? 127u : s[a]);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const mx_b8 wf = __builtin_bit_cast(mx_b8, mx_decode8(w[a][k], sc));
#pragma unroll
                    for (int pl = 0; pl < P; ++pl)
#pragma unroll
                        for (int b = 0; b < NT; ++b)
                            acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                __builtin_bit_cast(mx_b8, xf[pl][b][k]), wf, acc[a][b], 0, 0, 0);
                }
            }
        }
    }
    // a NaN block makes its whole output column NaN: any of the column's four lane groups may hold it
#pragma unroll
    for (int a = 0; a < TT; ++a) {
        int f = nan[a];
        f |= __shfl_xor(f, 16);
        f |= __shfl_xor(f, 32);
        if (f) {
#pragma unroll
            for (int b = 0; b < NT; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[a][b][i] = __uint_as_float(0x7fc00000u);
        }
#pragma unroll
        for (int b = 0; b < NT; ++b)
            *reinterpret_cast<f32x4 *>(red + ((wave * TT + a) * NT + b) * 256 + lane * 4) = acc[a][b];
    }
    __syncthreads();
    // element (m, n) of a tile: lane (m / 4) * 16 + n, register m % 4
    for (int e = threadIdx.x; e < MT * NT * 256; e += blockDim.x) {
        const int n = e & 15, a = (e >> 4) % MT, m = (e >> 4) / MT % 16, b = (e >> 8) / MT;
        const int row = b * 16 + m, o = o0 + a * 16 + n;
        if (row >= tile.nrows || o >= p.ocover) continue;
        const int off = ((m >> 2) * 16 + n) * 4 + (m & 3);
        float v = 0.f, u = 0.f;
        for (int w = 0; w < NW; ++w) v += red[((w * TT + a) * NT + b) * 256 + off];
        const int64_t yr = mx_y_row(p, tile.row0 + row);
        if constexpr (GLU) {
            for (int w = 0; w < NW; ++w) u += red[((w * TT + MT + a) * NT + b) * 256 + off];
            float h = o < p.OUT ? v / (1.f + __expf(-v)) * u : 0.f;
            for (int pl = 0; pl < p.yp; ++pl)
                static_cast<uint16_t *>(p.y)[pl * p.yplane + yr * p.ldy + o] = mx_plane_next(h);
        } else {
            store_act(p.y, p.y_type, yr * p.ldy + o, v);
        }
    }
}

// Kernel arguments of a call, and the tiles of `rows` x rows that it makes.
void mx_args(const MxCall &c, MxsArgs *a);
int64_t mx_tiles(const MxCall &c, int rows);
// Launches k_mx_stream for a call; NT row tiles of 16.
int mx_stream(const MxCall &c, int NT, hipStream_t st);

}  // namespace vqk
