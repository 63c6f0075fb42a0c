// Products of 8-bit weights with few rows of x: the weights are streamed once
// past up to 16 * NT rows, and again for the next ones.
//
//     y[n, o] = sum_b f[n, o, b] sum_{k in b} w8[o, k] x[n, k]
//     f = sw[o / 128, b], with x in 8 bits (or codes' values in 16) times sx[n, b]
//
// A workgroup keeps its tile of x in registers and walks over weight rows. Eight
// waves: KW along k, NCW blocks of 128 each, and 8 / KW along the weight rows, 16 a
// step. The next step's weights (two contiguous KB a block) load while the last ones
// are multiplied: 8-bit x by one instruction a block, 16-bit x by four after the
// codes are converted. The matrix cores take the weights as rows, so a lane holds
// four neighbouring outputs of one x row and that row's scales are one number a
// lane. The fp32 sums of KW > 1 waves meet in LDS in wave order, two buffers in
// turn, one barrier a step.
// Rows of more blocks than eight waves hold (kF8sWaves times the registers' NCW) are cut
// into ks ranges of k, a workgroup each, whose sums a second kernel adds up.
// x comes from its rows where there are one or two, otherwise through LDS, copied
// in whole lines (20 KB or less a wave at a time).
// Bound by HBM: 2 KB of weights take a wave 32 cycles (8-bit x) or 64 and the
// conversions (16-bit), a fraction of the time in which they can arrive. Measured:
// 5120 to 17408, 8 rows of 8 bits 17.5 us (5.1 TB/s), 20 rows 19.0 (4.7); one row of bf16,
// 4096 to 4096, 6.5 us, a chain of launch, first load, products and the waves' sum.
#pragma once

#include "vqk_f8t.h"

namespace vqk {

constexpr int kF8sWaves = 8;

struct F8sArgs {
    const uint8_t *codes;
    const float *scales;
    int64_t swo, swk;
    int64_t OUT, IN, N;
    int32_t RT, NC;
    const uint8_t *x;                         // codes, or 16-bit rows
    int64_t xld, xplane;                      // in bytes
    const float *sx;
    int64_t sn, sk;
    void *y;
    int32_t y_type;
    int32_t nob, kw, ks, steps, total_steps, stage;
    int32_t even, more;                       // blocks of a share of k (kw * ks of them), shares with one more
    float *part;                              // ks > 1: sums of each range of k, [ks][N][OUT]
};

// OP: kOpF16, kOpBF16, or kOpF8 (8-bit x).
template <int OP, int NT, int P, int NCW>
__global__ void __launch_bounds__(64 * kF8sWaves, 2) k_f8_rows(const F8sArgs p) {
    constexpr bool A8 = OP == kOpF8;
    constexpr int XB = A8 ? 128 : 256;        // bytes of a block of an x row
    constexpr int PC = XB / 64;               // 16-byte pieces of it that a lane holds
    extern __shared__ __align__(16) uint8_t smem[];
    float *red = reinterpret_cast<float *>(smem);       // sums [2][8 waves][NT][256]; before them x
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int KW = p.kw, RW = kF8sWaves / KW;
    const int kw = wave % KW, rw = wave / KW;
    const int t = int(blockIdx.x / unsigned(p.nob)) / p.ks, z = int(blockIdx.x / unsigned(p.nob)) % p.ks;
    const int part = int(blockIdx.x % unsigned(p.nob));
    const int row0 = t * 16 * NT, nrows = int(min(int64_t(16 * NT), p.N - row0));
    const int s_lo = part * p.steps, s_hi = min(p.total_steps, s_lo + p.steps);
    if (s_lo >= s_hi) return;

    // this wave's blocks: an even share of them all, NCW at most
    const int share = z * KW + kw;
    const int c0 = share * p.even + min(share, p.more), nc = p.even + (share < p.more);
    u32x4 wn[NCW][2];
    float swn[NCW];
    auto load_w = [&](int step) {
        const uint32_t rt = uint32_t(min(step * RW + rw, p.RT - 1));
#pragma unroll
        for (int c = 0; c < NCW; ++c) {
            const uint32_t ch = uint32_t(min(c0 + c, p.NC - 1));
            const uint8_t *at = p.codes + ((rt * uint32_t(p.NC) + ch) * 2048u + lane * 16u);
            wn[c][0] = *reinterpret_cast<const u32x4 *>(at);
            wn[c][1] = *reinterpret_cast<const u32x4 *>(at + 1024);
            swn[c] = p.scales[int64_t(rt >> 3) * p.swo + ch * p.swk];
        }
    };
    load_w(s_lo);

    // x: piece k of a lane is bytes g * XB / 4 + 16 k of its row's block (zero past the row's end)
    u32x4 xf[P][NT][NCW][PC];
    float sx[NT][NCW];
    const int64_t xbytes = A8 ? int64_t(p.NC) * 128 : p.IN * 2;
    if (p.stage) {
        uint8_t *xl = smem + wave * (NCW * 16 * XB);
#pragma unroll
        for (int pl = 0; pl < P; ++pl)
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                constexpr int UPR = NCW * XB / 16;          // 16-byte units of a row's part
                constexpr int MASK = UPR % 16 == 0 ? 15 : 7;
#pragma unroll
                for (int i = 0; i < UPR / 4; ++i) {
                    // LDS unit i * 64 + lane: row / slot; the slot holds piece slot ^ row of the wave's part
                    const int u = i * 64 + lane, row = u / UPR, slot = u % UPR;
                    const int piece = slot ^ (row & MASK);
                    const int64_t at = int64_t(c0) * XB + piece * 16;
                    const uint8_t *src = p.x + pl * p.xplane + int64_t(row0 + min(b * 16 + row, nrows - 1)) * p.xld +
                                         (at < xbytes ? at : 0);
                    __builtin_amdgcn_global_load_lds((global_void *)src, (lds_void *)(xl + i * 1024), 16, 0, 0);
                }
                wait_vmem();
#pragma unroll
                for (int c = 0; c < NCW; ++c)
#pragma unroll
                    for (int k = 0; k < PC; ++k) {
                        const int piece = c * (XB / 16) + g * PC + k;
                        const u32x4 v = *reinterpret_cast<const u32x4 *>(
                            xl + (r * UPR + (piece ^ (r & MASK))) * 16);
                        xf[pl][b][c][k] = int64_t(c0) * XB + piece * 16 < xbytes ? v : u32x4{};
                    }
                __builtin_amdgcn_s_waitcnt(0xC07F);         // lgkmcnt(0): read before the next rows land
            }
        __syncthreads();                                    // the sums use the same LDS
    } else {
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            const uint8_t *xp = p.x + int64_t(row0 + min(b * 16 + r, nrows - 1)) * p.xld;
#pragma unroll
            for (int pl = 0; pl < P; ++pl)
#pragma unroll
                for (int c = 0; c < NCW; ++c)
#pragma unroll
                    for (int k = 0; k < PC; ++k) {
                        const int64_t at = int64_t(c0 + c) * XB + (g * PC + k) * 16;
                        xf[pl][b][c][k] = at < xbytes ? *reinterpret_cast<const u32x4 *>(xp + pl * p.xplane + at) : u32x4{};
                    }
        }
    }
#pragma unroll
    for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int c = 0; c < NCW; ++c)
            sx[b][c] = p.sx ? p.sx[int64_t(row0 + min(b * 16 + r, nrows - 1)) * p.sn + int64_t(min(c0 + c, p.NC - 1)) * p.sk] : 1.f;

    for (int step = s_lo; step < s_hi; ++step) {
        u32x4 w[NCW][2];
        float sw[NCW];
#pragma unroll
        for (int c = 0; c < NCW; ++c) {
            w[c][0] = wn[c][0];
            w[c][1] = wn[c][1];
            sw[c] = swn[c];
        }
        if (step + 1 < s_hi) load_w(step + 1);
        f32x4 acc[NT];
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[b] = f32x4{};
#pragma unroll
        for (int c = 0; c < NCW; ++c) {
            if (c >= nc) break;                             // the same for the whole wave
            f32x4 s[NT];
            if constexpr (A8) {
#pragma unroll
                for (int b = 0; b < NT; ++b)
                    s[b] = f8_mma16(f8_pair(w[c][0], w[c][1]), f8_pair(xf[0][b][c][0], xf[0][b][c][1]));
            } else {
#pragma unroll
                for (int b = 0; b < NT; ++b) s[b] = f32x4{};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const u32x4 wf = f8_operand<OP>(w[c][k / 2][k % 2 * 2], w[c][k / 2][k % 2 * 2 + 1]);
#pragma unroll
                    for (int pl = 0; pl < P; ++pl)
#pragma unroll
                        for (int b = 0; b < NT; ++b) s[b] = mx_mma16<A8 ? kOpBF16 : OP>(wf, xf[pl][b][c][k], s[b]);
                }
            }
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                const float f = sw[c] * sx[b][c];
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[b][i] = __builtin_fmaf(f, s[b][i], acc[b][i]);
            }
        }
        // register i of lane l: weight row 4 * (l / 16) + i, x row l % 16
        auto put = [&](int n, int o, f32x4 v) {
            if (n >= nrows || o >= p.OUT) return;
            float q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = OP == kOpBF16 ? v[i] * kF8Up : v[i];
            const int64_t at = int64_t(row0 + n) * p.OUT + o;
            const int count = int(min(int64_t(4), p.OUT - o));
            if (p.ks > 1) {
                mx_store4(p.part, VQK_F32, int64_t(z) * p.N * p.OUT + at, q, count, (p.OUT & 3) == 0);
            } else {
                const bool al = (p.OUT & 3) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
                mx_store4(p.y, p.y_type, at, q, count, al);
            }
        };
        if (KW == 1) {
#pragma unroll
            for (int b = 0; b < NT; ++b) put(b * 16 + r, (step * RW + rw) * 16 + 4 * g, acc[b]);
            continue;
        }
        float *buf = red + (step & 1) * kF8sWaves * NT * 256;
#pragma unroll
        for (int b = 0; b < NT; ++b) *reinterpret_cast<f32x4 *>(buf + (wave * NT + b) * 256 + lane * 4) = acc[b];
        __syncthreads();
        // sums (row tile of the step, x tile, lane)
        for (int e = threadIdx.x; e < RW * NT * 64; e += 64 * kF8sWaves) {
            const int l = e & 63, b = (e >> 6) % NT, q = (e >> 6) / NT;
            f32x4 v{};
            for (int k = 0; k < KW; ++k) {
                const f32x4 a = *reinterpret_cast<const f32x4 *>(buf + ((q * KW + k) * NT + b) * 256 + l * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] += a[i];
            }
            put(b * 16 + (l & 15), (step * RW + q) * 16 + 4 * (l >> 4), v);
        }
    }
}

}  // namespace vqk
