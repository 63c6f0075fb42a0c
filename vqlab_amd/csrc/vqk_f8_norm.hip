// RMS norm of rows with the residual's addition in front, its output in 8 bits
// with scales or as it is, and its backward pass.
//
//     h = round(x + residual)          (the type of x; what the next layer adds to)
//     r = 1 / sqrt(sum_c h_c^2 / C + eps),   y = h r w
//     8 bits: s = max(amax / 448, 2^-126) over 128 of y, code = e4m3(y * (1 / s))
// and with the gradients dy and dh of both outputs, xhat = h r, g = dy w:
//     dx = dresidual = r (g - xhat sum_c g xhat / C) + dh,   dw = sum over rows of dy xhat
//
// Bound by memory: each input is read once and each output written once. A
// workgroup of W waves takes a row and holds it in registers, 8 neighbouring
// columns a piece: few rows are spread over as many waves as they have pieces
// (latency), many rows take two pieces a lane (fewer steps across waves for
// each row). A block of 128 is 16 lanes of one piece, so its largest magnitude
// takes four DPP steps. Squares are summed in fp64 (2^127 squared is no fp32
// number), everything else is fp32. dw: a workgroup adds up its rows in
// registers, the workgroups' sums meet in a fixed order.
// Measured: one row of 4096 to 8 bits 3.0 us, 2048 rows of 5120 fp16 18 (4.1 TB/s), 16384
// rows of 4096 bf16 with h 87 (6.2 TB/s, out of the MALL in part), backward 112
// (4.8 TB/s) and 6.2 for dw.
#include "vqk_f8.h"

namespace vqk {

constexpr int kNormMaxC = 16384, kNormMaxWaves = 16;      // 2 pieces a lane

struct NormArgs {
    const void *x, *res, *w;
    int64_t N, ldx, ldr;
    int32_t C, w_type;
    double eps;
    void *h, *y;                              // h: NULL without a residual; y: NULL for 8 bits
    float *r;                                 // [N] or NULL
    uint8_t *codes;                           // [N][C]
    float *scales;
    int64_t sn, sk;
    int64_t row0;                             // first row of this launch
};

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t(dpp_u<CTRL>(uint32_t(b >> 32))) << 32) | dpp_u<CTRL>(uint32_t(b)));
}
__device__ __forceinline__ double lane_f64(double v, int from) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(b)), from));
    return __builtin_bit_cast(double, (uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(b >> 32)), from))) << 32) | lo);
}
// Sum over the workgroup's W waves, in every thread; `part` is used by one call. The
// barrier waits for LDS alone: loads of the next row stay on their way.
__device__ __forceinline__ double norm_sum(double v, double (&part)[kNormMaxWaves]) {
    const int W = int(blockDim.x) >> 6;
    v += dpp_f64<kDppQuadXor1>(v);
    v += dpp_f64<kDppQuadXor2>(v);
    v += dpp_f64<kDppRowHalfMirror>(v);
    v += dpp_f64<kDppRowMirror>(v);
    v = (lane_f64(v, 0) + lane_f64(v, 16)) + (lane_f64(v, 32) + lane_f64(v, 48));
    if (W == 1) return v;
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);       // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    double s = 0.;
    for (int i = 0; i < W; ++i) s += part[i];
    return s;
}

__device__ __forceinline__ void norm_store8(void *y, int32_t type, int64_t at, const float (&v)[8], int n, bool vec) {
    const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
    if (vec && n >= 8 && type != VQK_F32) {
        u32x4 o;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint16_t lo = type == VQK_BF16 ? f32_to_bf16(v[2 * u]) : f32_to_h(v[2 * u]);
            const uint16_t hi = type == VQK_BF16 ? f32_to_bf16(v[2 * u + 1]) : f32_to_h(v[2 * u + 1]);
            o[u] = lo | (uint32_t(hi) << 16);
        }
        *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(y) + at) = o;
        return;
    }
    if (n > 0) mx_store4(y, type, at, a, min(n, 4), vec);
    if (n > 4) mx_store4(y, type, at + 4, b, min(n - 4, 4), vec);
}

template <int T>
__device__ __forceinline__ float round_to(float v) {
    if constexpr (T == VQK_F32) return v;
    return T == VQK_BF16 ? bf16_to_f32(f32_to_bf16(v)) : h_to_f32(f32_to_h(v));
}

template <int XT, int P, bool Q>
__global__ void __launch_bounds__(64 * kNormMaxWaves) k_rms(const NormArgs p, bool vec, bool vecw) {
    __shared__ double part[kNormMaxWaves];
    const int64_t row = p.row0 + blockIdx.x;
    float h[P][8], wt[P][8];
    double sum = 0.;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int k0 = (i * int(blockDim.x) + int(threadIdx.x)) * 8;
        mx_load8(p.x, XT, row * p.ldx, k0, p.C, vec, h[i]);
        mx_load8(p.w, p.w_type, 0, k0, p.C, vecw, wt[i]);
    }
    if (p.res) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int k0 = (i * int(blockDim.x) + int(threadIdx.x)) * 8;
            float a[8];
            mx_load8(p.res, XT, row * p.ldr, k0, p.C, vec, a);
#pragma unroll
            for (int u = 0; u < 8; ++u) h[i][u] = round_to<XT>(h[i][u] + a[u]);
            norm_store8(p.h, XT, row * p.C + k0, h[i], p.C - k0, vec);
        }
    }
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int u = 0; u < 8; ++u) sum = __builtin_fma(double(h[i][u]), double(h[i][u]), sum);
    sum = norm_sum(sum, part);
    const float r = float(1. / sqrt(sum / double(p.C) + p.eps));
    if (p.r && threadIdx.x == 0) p.r[row] = r;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int k0 = (i * int(blockDim.x) + int(threadIdx.x)) * 8;
        float y[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) y[u] = h[i][u] * r * wt[i][u];
        if constexpr (Q) {
            uint32_t m = 0;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                y[u] = k0 + u < p.C ? y[u] : 0.f;              // 0 * r is NaN where r is infinite
                m = max(m, __float_as_uint(y[u]) & 0x7fffffffu);
            }
            const float s = f8_scale(row16_max(m));
            const u32x2 c = f8_encode8(y, 1.f / s, s == s);
            if (k0 >= p.C) continue;
            uint8_t *dst = p.codes + row * p.C + k0;
            if (vec && k0 + 8 <= p.C) {
                *reinterpret_cast<u32x2 *>(dst) = c;
            } else {
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (k0 + u < p.C) dst[u] = uint8_t(c[u / 4] >> (8 * (u % 4)));
            }
            if ((threadIdx.x & 15) == 0) p.scales[row * p.sn + (k0 >> 7) * p.sk] = s;
        } else {
            norm_store8(p.y, XT, row * p.C + k0, y, p.C - k0, vec);
        }
    }
}

struct NormBwdArgs {
    const void *h, *w, *dy, *dh;              // dh: NULL for none
    int64_t N, ldh;
    int32_t C, w_type;
    const float *r;
    void *dx;
    float *part;                              // [gridDim.x][C]
};

// Eight neighbouring columns as they lie in memory, zeros past the row.
template <int XT> struct Raw8 { u32x4 a[XT == VQK_F32 ? 2 : 1]; };
template <int XT>
__device__ __forceinline__ Raw8<XT> raw_load8(const void *x, int64_t base, int k0, int C, bool vec) {
    Raw8<XT> o{};
    constexpr int E = XT == VQK_F32 ? 4 : 8;  // elements of 16 bytes
    if (vec) {
        if (k0 < C) {
            const u32x4 *from = reinterpret_cast<const u32x4 *>(static_cast<const uint8_t *>(x) + (base + k0) * (16 / E));
            o.a[0] = from[0];
            if constexpr (XT == VQK_F32) o.a[1] = from[1];
        }
        return o;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (k0 + i >= C) continue;
        if constexpr (XT == VQK_F32) o.a[i / 4][i % 4] = static_cast<const uint32_t *>(x)[base + k0 + i];
        else o.a[0][i / 2] |= uint32_t(static_cast<const uint16_t *>(x)[base + k0 + i]) << (16 * (i % 2));
    }
    return o;
}
template <int XT>
__device__ __forceinline__ float raw_at(const Raw8<XT> &r, int i) {
    if constexpr (XT == VQK_F32) return __uint_as_float(r.a[i / 4][i % 4]);
    const uint16_t h = uint16_t(r.a[0][i / 2] >> (16 * (i % 2)));
    return XT == VQK_BF16 ? bf16_to_f32(h) : h_to_f32(h);
}

// The next row is loaded while this one is worked on, as it lies in memory (half the
// registers of its values); rows of more than 8 waves leave no registers for that (the 128
// of 1024 threads: those kernels spill 3 to 11).
template <int XT, int P, int MAXW>
__global__ void __launch_bounds__(64 * MAXW) k_rms_bwd(const NormBwdArgs p, bool vec, bool vecw) {
    constexpr bool AHEAD = MAXW <= 8;
    __shared__ double part[2][kNormMaxWaves];
    float wt[P][8], dw[P][8] = {};
    Raw8<XT> h[P], dy[P], dh[P];
    auto load = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int k0 = (i * int(blockDim.x) + int(threadIdx.x)) * 8;
            h[i] = raw_load8<XT>(p.h, row * p.ldh, k0, p.C, vec);
            dy[i] = raw_load8<XT>(p.dy, row * p.C, k0, p.C, vec);
            dh[i] = p.dh ? raw_load8<XT>(p.dh, row * p.C, k0, p.C, vec) : Raw8<XT>{};
        }
    };
    if (AHEAD) load(blockIdx.x);              // no more workgroups than rows
#pragma unroll
    for (int i = 0; i < P; ++i) mx_load8(p.w, p.w_type, 0, (i * int(blockDim.x) + int(threadIdx.x)) * 8, p.C, vecw, wt[i]);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < p.N; row += gridDim.x, turn ^= 1) {
        Raw8<XT> ch[P], cdy[P], cdh[P];
        const float r = p.r[row];
        if (!AHEAD) load(row);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < P; ++i) {
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float d = raw_at(dy[i], u), xh = raw_at(h[i], u) * r;
                dw[i][u] = __builtin_fmaf(d, xh, dw[i][u]);
                dot = __builtin_fmaf(d * wt[i][u], xh, dot);
            }
            ch[i] = h[i];
            cdy[i] = dy[i];
            cdh[i] = dh[i];
        }
        if (AHEAD && row + gridDim.x < p.N) load(row + gridDim.x);
        const float mean = float(norm_sum(double(dot), part[turn]) / double(p.C));
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int k0 = (i * int(blockDim.x) + int(threadIdx.x)) * 8;
            float d[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) d[u] = r * (raw_at(cdy[i], u) * wt[i][u] - raw_at(ch[i], u) * r * mean) + raw_at(cdh[i], u);
            norm_store8(p.dx, XT, row * p.C + k0, d, p.C - k0, vec);
        }
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int k0 = (i * int(blockDim.x) + int(threadIdx.x)) * 8;
        norm_store8(p.part, VQK_F32, int64_t(blockIdx.x) * p.C + k0, dw[i], p.C - k0, vec);
    }
}

// dw from the workgroups' sums: 32 columns by 32 slices of the sums a workgroup.
__global__ void __launch_bounds__(1024) k_rms_dw(const float *part, int rows, int C, void *dw, int32_t type) {
    __shared__ double s[32][33];
    const int c = int(blockIdx.x) * 32 + (threadIdx.x & 31), t = threadIdx.x >> 5;
    double v = 0.;
    if (c < C)
        for (int i = t; i < rows; i += 32) v += double(part[int64_t(i) * C + c]);
    s[t][threadIdx.x & 31] = v;
    __syncthreads();
    for (int o = 16; o >= 1; o >>= 1) {
        if (t < o) s[t][threadIdx.x & 31] += s[t + o][threadIdx.x & 31];
        __syncthreads();
    }
    if (t == 0 && c < C) store_act(dw, type, c, float(s[0][threadIdx.x]));
}

// Waves to a row and pieces to a lane.
struct NormPlan { int w, p; };
// Rows up to which a row is spread over one piece a lane.
constexpr int64_t kNormSpreadRows = 1024;
static NormPlan norm_plan(int64_t N, int64_t C) {
    const int pieces = int((C + 511) / 512);
    // 2048 rows of 5120 fp16 to 8 bits: two pieces a lane 18.0 us, one 20.6, four 20.6
    const int p = N <= kNormSpreadRows && pieces <= kNormMaxWaves ? 1 : 2;
    return NormPlan{(pieces + p - 1) / p, p};
}
// The backward pass: two pieces a lane, as many workgroups as run at once, each of which
// leaves a row of sums (16384 rows of 4096, bf16: 2048 waves 117 us with the sums' sum,
// 1024 waves 134, 4096 waves 135).
static NormPlan norm_bwd_plan(int64_t C) {
    const int pieces = int((C + 511) / 512), p = pieces > 1 ? 2 : 1;
    return NormPlan{(pieces + p - 1) / p, p};
}
static int64_t norm_bwd_wgs(int64_t N, int64_t C) {
    const int64_t most = 2048 / norm_bwd_plan(C).w;
    return N < most ? N : most;
}

template <int XT, bool Q>
static int go_norm(NormArgs a, NormPlan pl, bool vec, bool vecw, hipStream_t st) {
    const dim3 block{unsigned(64 * pl.w)};
    const int64_t most = (INT64_C(1) << 31) / block.x;      // a launch has fewer than 2^32 threads
    for (; a.row0 < a.N; a.row0 += most) {
        const dim3 grid{unsigned(a.N - a.row0 < most ? a.N - a.row0 : most)};
        if (pl.p == 1) hipLaunchKernelGGL((k_rms<XT, 1, Q>), grid, block, 0, st, a, vec, vecw);
        else hipLaunchKernelGGL((k_rms<XT, 2, Q>), grid, block, 0, st, a, vec, vecw);
        const int rc = hip_status(hipGetLastError(), "norm launch");
        if (rc) return rc;
    }
    return VQK_OK;
}
template <int XT>
static int go_norm_bwd(const NormBwdArgs &a, NormPlan pl, unsigned wgs, bool vec, bool vecw, hipStream_t st) {
    const dim3 grid{wgs}, block{unsigned(64 * pl.w)};
    if (pl.p == 1) hipLaunchKernelGGL((k_rms_bwd<XT, 1, 1>), grid, block, 0, st, a, vec, vecw);
    else if (pl.w <= 8) hipLaunchKernelGGL((k_rms_bwd<XT, 2, 8>), grid, block, 0, st, a, vec, vecw);
    else hipLaunchKernelGGL((k_rms_bwd<XT, 2, kNormMaxWaves>), grid, block, 0, st, a, vec, vecw);
    return hip_status(hipGetLastError(), "norm gradient launch");
}

static int check_norm(int32_t type, int32_t w_type, int64_t N, int64_t C, double eps, const char *what) {
    if (!act_size(type) || !act_size(w_type)) return set_error(VQK_EINVAL, "%s: types %d, %d", what, type, w_type);
    if (N < 0 || N > INT32_MAX || C < 1) return set_error(VQK_EINVAL, "%s: N=%lld C=%lld", what, (long long)N, (long long)C);
    if (C > kNormMaxC) return set_error(VQK_ENOTIMPL, "%s: rows of %lld > %d", what, (long long)C, kNormMaxC);
    if (!(eps >= 0.)) return set_error(VQK_EINVAL, "%s: eps=%g", what, eps);
    return VQK_OK;
}

static bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace vqk

using namespace vqk;

extern "C" int vqk_rms_norm(const void *x, int32_t type, int64_t N, int64_t C, int64_t ldx, const void *residual,
                            int64_t ldr, const void *weight, int32_t w_type, double eps, void *h, void *y, float *r,
                            uint8_t *codes, float *scales, int64_t scale_row, int64_t scale_block, void *stream) {
    int rc = check_norm(type, w_type, N, C, eps, "rms norm");
    if (rc) return rc;
    if (ldx < C || (residual && ldr < C)) return set_error(VQK_EINVAL, "rms norm: rows of %lld apart by %lld, %lld", (long long)C, (long long)ldx, (long long)ldr);
    if ((y != nullptr) == (codes != nullptr) && N > 0) return set_error(VQK_EINVAL, "rms norm: one of y and codes");
    if (N == 0) return VQK_OK;
    if (!x || !weight || (residual && !h) || (codes && !scales)) return set_error(VQK_EINVAL, "rms norm: NULL pointer");
    if (scale_row < 0 || scale_block < 0) return set_error(VQK_EINVAL, "rms norm: negative stride of scales");
    const int esz = act_size(type);
    const NormArgs a{x, residual, weight, N, ldx, ldr, int32_t(C), w_type, eps, h, y, r, codes, scales, scale_row, scale_block, 0};
    const bool vec = C % 8 == 0 && al16(x) && (ldx * esz) % 16 == 0 &&
                     (!residual || (al16(residual) && (ldr * esz) % 16 == 0 && al16(h))) &&
                     (y ? al16(y) : (reinterpret_cast<uintptr_t>(codes) & 7) == 0);
    const NormPlan pl = norm_plan(N, C);
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (type) {
        case VQK_F16: return y ? go_norm<VQK_F16, false>(a, pl, vec, al16(weight), st) : go_norm<VQK_F16, true>(a, pl, vec, al16(weight), st);
        case VQK_BF16: return y ? go_norm<VQK_BF16, false>(a, pl, vec, al16(weight), st) : go_norm<VQK_BF16, true>(a, pl, vec, al16(weight), st);
        default: return y ? go_norm<VQK_F32, false>(a, pl, vec, al16(weight), st) : go_norm<VQK_F32, true>(a, pl, vec, al16(weight), st);
    }
}

extern "C" int vqk_rms_norm_backward_workspace(int64_t N, int64_t C, size_t *bytes) {
    const int rc = check_norm(VQK_F32, VQK_F32, N, C, 0., "rms norm backward");
    if (rc) return rc;
    if (!bytes) return set_error(VQK_EINVAL, "rms norm backward: NULL bytes");
    *bytes = size_t(norm_bwd_wgs(N, C)) * size_t(C) * 4;
    return VQK_OK;
}

extern "C" int vqk_rms_norm_backward(const void *h, int32_t type, int64_t N, int64_t C, int64_t ldh, const void *weight,
                                     int32_t w_type, const float *r, const void *dy, const void *dh, void *dx, void *dw,
                                     void *workspace, size_t ws_bytes, void *stream) {
    const int rc = check_norm(type, w_type, N, C, 0., "rms norm backward");
    if (rc) return rc;
    if (ldh < C) return set_error(VQK_EINVAL, "rms norm backward: rows of %lld apart by %lld", (long long)C, (long long)ldh);
    if (!dw || (N > 0 && (!h || !weight || !r || !dy || !dx))) return set_error(VQK_EINVAL, "rms norm backward: NULL pointer");
    const int64_t wgs = norm_bwd_wgs(N, C);
    const size_t need = size_t(wgs) * size_t(C) * 4;
    if (need && (!workspace || ws_bytes < need))
        return set_error(VQK_ENOSPACE, "rms norm backward: workspace %zu < %zu", ws_bytes, need);
    if (reinterpret_cast<uintptr_t>(workspace) & 15)
        return set_error(VQK_EINVAL, "rms norm backward: workspace must be 16-byte aligned");
    hipStream_t st = static_cast<hipStream_t>(stream);
    float *part = static_cast<float *>(workspace);
    if (N > 0) {
        const int esz = act_size(type);
        const NormBwdArgs a{h, weight, dy, dh, N, ldh, int32_t(C), w_type, r, dx, part};
        const bool vec = C % 8 == 0 && al16(h) && (ldh * esz) % 16 == 0 && al16(dy) && (!dh || al16(dh)) && al16(dx);
        const NormPlan pl = norm_bwd_plan(C);
        int e;
        switch (type) {
            case VQK_F16: e = go_norm_bwd<VQK_F16>(a, pl, unsigned(wgs), vec, al16(weight), st); break;
            case VQK_BF16: e = go_norm_bwd<VQK_BF16>(a, pl, unsigned(wgs), vec, al16(weight), st); break;
            default: e = go_norm_bwd<VQK_F32>(a, pl, unsigned(wgs), vec, al16(weight), st);
        }
        if (e) return e;
    }
    hipLaunchKernelGGL(k_rms_dw, dim3(unsigned((C + 31) / 32)), dim3(1024), 0, st, part, int(wgs), int(C), dw, w_type);
    return hip_status(hipGetLastError(), "norm weight gradient launch");
}
