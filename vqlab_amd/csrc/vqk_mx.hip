// MXFP4 quantisation: rows to 4-bit codes and scale bytes, and back.
//
//     s = max(floor(log2(max |v|)) - 2, -127) + 127,   code = e2m1(v / 2^(s - 127))
//
// rounded to nearest (ties to even), values past 6 to 6; a block with an
// infinity or NaN gets s = 255 and codes 0, and reads back as NaN.
// Bound by memory: 16 (bf16) or 32 bytes in and 4.25 out for 8 values. Four
// lanes share a block, 8 values each: the loads of a wave are contiguous, the
// largest magnitude takes two DPP steps inside the quad and the conversion is
// v_cvt_scalef32_pk_fp4_f32, two values an instruction.
#include "vqk_mx.h"

namespace vqk {

int make_mx_geom(const vqk_mx_weights *w, MxGeom *g, const char *what) {
    if (!w) return set_error(VQK_EINVAL, "%s: NULL weights", what);
    if (w->E < 1 || w->OUT < 1 || w->IN < 1 || w->E > INT32_MAX || w->OUT > INT32_MAX / 2 ||
        w->IN > INT32_MAX / 2)
        return set_error(VQK_EINVAL, "%s: bad shape E=%lld OUT=%lld IN=%lld", what, (long long)w->E,
                         (long long)w->OUT, (long long)w->IN);
    if (!w->codes || !w->scales) return set_error(VQK_EINVAL, "%s: codes and scales are required", what);
    if (reinterpret_cast<uintptr_t>(w->codes) & 15)
        return set_error(VQK_EINVAL, "%s: codes must be 16-byte aligned", what);
    if (reinterpret_cast<uintptr_t>(w->scales) & 3)
        return set_error(VQK_EINVAL, "%s: scales must be 4-byte aligned", what);
    *g = MxGeom{w->E, w->OUT, w->IN, (w->IN + kMxBlock - 1) / kMxBlock, (w->OUT + 15) / 16,
                (w->IN + kMxChunk - 1) / kMxChunk};
    // kernels reach an expert's weights by 32-bit offsets
    if (mx_expert_codes(g->RT, g->NC) > INT64_C(0xffffffff))
        return set_error(VQK_ENOTIMPL, "%s: an expert of 4 GB or more", what);
    return VQK_OK;
}

struct QuantArgs {
    const void *x;
    int64_t cols, ldx, NB, pieces;            // pieces of 8 values: rows * NB * 4
    int32_t permute;
    uint8_t *codes, *scales;
};

// FLAT: rows are whole blocks one after the other, so piece i is values
// 8i..8i+7 of x. Otherwise a piece finds its row by division.
template <int XT, bool FLAT, bool VEC>
__global__ void __launch_bounds__(256) k_mx_quant(const QuantArgs p) {
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < p.pieces; i += int64_t(gridDim.x) * 256) {
        float v[8];
        if constexpr (FLAT) {
            mx_load8(p.x, XT, 0, i * 8, p.pieces * 8, true, v);
        } else {
            const int64_t blk = i >> 2, row = blk / p.NB;
            mx_load8(p.x, XT, row * p.ldx, (blk - row * p.NB) * kMxBlock + (i & 3) * 8, p.cols, VEC, v);
        }
        uint32_t m = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) m = max(m, __float_as_uint(v[u]) & 0x7fffffffu);
        // pieces come in whole quads (pieces % 4 == 0 and 256 % 4 == 0): all four lanes are here
        const uint32_t s = mx_scale_byte(quad_max(m));
        reinterpret_cast<uint32_t *>(p.codes)[i] = mx_encode8(v, s);
        if ((i & 3) == 0) p.scales[p.permute ? mxf_scale_at(i >> 2) : i >> 2] = uint8_t(s);   // NB % 16 == 0 then
    }
}

template <int XT>
static int go_quant(const QuantArgs &a, hipStream_t st) {
    const int esz = XT == VQK_F32 ? 4 : 2;
    const bool al = (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
    const bool vec = al && (a.ldx * esz) % 16 == 0;
    const bool flat = vec && a.ldx == a.cols && a.cols == a.NB * kMxBlock;
    const int64_t wgs = (a.pieces + 255) / 256;
    const dim3 grid(unsigned(wgs < 16384 ? wgs : 16384));
    if (flat) hipLaunchKernelGGL((k_mx_quant<XT, true, true>), grid, dim3(256), 0, st, a);
    else if (vec) hipLaunchKernelGGL((k_mx_quant<XT, false, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_mx_quant<XT, false, false>), grid, dim3(256), 0, st, a);
    return hip_status(hipGetLastError(), "MXFP4 quantiser launch");
}

int launch_mx_quant(const void *x, int32_t type, int64_t rows, int64_t cols, int64_t ldx, int64_t NB,
                    bool permute, uint8_t *codes, uint8_t *scales, hipStream_t st) {
    const QuantArgs a{x, cols, ldx, NB, rows * NB * 4, permute, codes, scales};
    switch (type) {
        case VQK_F16: return go_quant<VQK_F16>(a, st);
        case VQK_BF16: return go_quant<VQK_BF16>(a, st);
        default: return go_quant<VQK_F32>(a, st);
    }
}

struct DequantArgs {
    const uint8_t *codes, *scales;
    int64_t cols, NB, pieces;
    void *out;
};

// The way back: a lane writes the 8 values of one word of codes.
template <int YT, bool FLAT>
__global__ void __launch_bounds__(256) k_mx_dequant(const DequantArgs p) {
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < p.pieces; i += int64_t(gridDim.x) * 256) {
        const uint32_t w = reinterpret_cast<const uint32_t *>(p.codes)[i];
        const uint32_t s = p.scales[i >> 2];
        const float sc = mx_scale(s == 255u ? 127u : s);
        typedef float f2 __attribute__((ext_vector_type(2)));
        f2 q[4];
        q[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 0);
        q[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 1);
        q[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 2);
        q[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, sc, 3);
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = s == 255u ? __uint_as_float(0x7fc00000u) : q[u / 2][u & 1];
        if constexpr (FLAT) {
            if constexpr (YT == VQK_F32) {
                float4 *o = reinterpret_cast<float4 *>(static_cast<float *>(p.out) + i * 8);
                o[0] = float4{v[0], v[1], v[2], v[3]};
                o[1] = float4{v[4], v[5], v[6], v[7]};
            } else {
                u32x4 o;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const uint16_t lo = YT == VQK_BF16 ? f32_to_bf16(v[2 * u]) : f32_to_h(v[2 * u]);
                    const uint16_t hi = YT == VQK_BF16 ? f32_to_bf16(v[2 * u + 1]) : f32_to_h(v[2 * u + 1]);
                    o[u] = lo | (uint32_t(hi) << 16);
                }
                *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(p.out) + i * 8) = o;
            }
        } else {
            const int64_t blk = i >> 2, row = blk / p.NB;
            const int64_t k0 = (blk - row * p.NB) * kMxBlock + (i & 3) * 8;
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (k0 + u < p.cols) store_act(p.out, YT, row * p.cols + k0 + u, v[u]);
        }
    }
}

template <int YT>
static int go_dequant(const DequantArgs &a, hipStream_t st) {
    const bool flat = (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 && a.cols % kMxBlock == 0;
    const int64_t wgs = (a.pieces + 255) / 256;
    const dim3 grid(unsigned(wgs < 16384 ? wgs : 16384));
    if (flat) hipLaunchKernelGGL((k_mx_dequant<YT, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_mx_dequant<YT, false>), grid, dim3(256), 0, st, a);
    return hip_status(hipGetLastError(), "MXFP4 dequantiser launch");
}

struct PlaneArgs {
    const void *x;
    int64_t N, IN, ldx, NB, pieces;
    uint16_t *out;
};

// Activations as exact bf16 planes; QUANT: the values of their MXFP4 form.
template <int XT, bool QUANT>
__global__ void __launch_bounds__(256) k_mx_planes(const PlaneArgs p, bool vec) {
    constexpr int P = QUANT ? 1 : mx_planes(XT);
    const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (i >= p.pieces) return;
    const int64_t blk = i >> 2, row = blk / p.NB;
    float v[8];
    mx_load8(p.x, XT, row * p.ldx, (blk - row * p.NB) * kMxBlock + (i & 3) * 8, p.IN, vec, v);
    if constexpr (QUANT) {
        uint32_t m = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) m = max(m, __float_as_uint(v[u]) & 0x7fffffffu);
        const uint32_t s = mx_scale_byte(quad_max(m));
        u32x4 o = mx_decode8(mx_encode8(v, s), mx_scale(s == 255u ? 127u : s));
        if (s == 255u) o = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
        *reinterpret_cast<u32x4 *>(p.out + i * 8) = o;
    } else {
#pragma unroll
        for (int pl = 0; pl < P; ++pl) {
            u32x4 o;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t lo = mx_plane_next(v[2 * u]);
                o[u] = lo | (uint32_t(mx_plane_next(v[2 * u + 1])) << 16);
            }
            *reinterpret_cast<u32x4 *>(p.out + pl * p.N * p.NB * kMxBlock + i * 8) = o;
        }
    }
}

int launch_mx_planes(const void *x, int32_t type, int64_t N, int64_t IN, int64_t ldx, bool quant,
                     uint16_t *out, hipStream_t st) {
    const int64_t NB = (IN + kMxBlock - 1) / kMxBlock;
    const PlaneArgs a{x, N, IN, ldx, NB, N * NB * 4, out};
    if (a.pieces == 0) return VQK_OK;
    const int64_t wgs = (a.pieces + 255) / 256;
    if (wgs > INT32_MAX) return set_error(VQK_ENOTIMPL, "activations too large");
    const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * act_size(type)) % 16 == 0;
    const dim3 grid{unsigned(wgs)}, b(256);
    if (quant) {
        switch (type) {
            case VQK_F16: hipLaunchKernelGGL((k_mx_planes<VQK_F16, true>), grid, b, 0, st, a, vec); break;
            case VQK_BF16: hipLaunchKernelGGL((k_mx_planes<VQK_BF16, true>), grid, b, 0, st, a, vec); break;
            default: hipLaunchKernelGGL((k_mx_planes<VQK_F32, true>), grid, b, 0, st, a, vec);
        }
    } else {
        switch (type) {
            case VQK_F16: hipLaunchKernelGGL((k_mx_planes<VQK_F16, false>), grid, b, 0, st, a, vec); break;
            case VQK_BF16: hipLaunchKernelGGL((k_mx_planes<VQK_BF16, false>), grid, b, 0, st, a, vec); break;
            default: hipLaunchKernelGGL((k_mx_planes<VQK_F32, false>), grid, b, 0, st, a, vec);
        }
    }
    return hip_status(hipGetLastError(), "activation plane launch");
}

// ------------------------------------------------------- operand order
struct PackArgs {
    const uint8_t *codes, *scales;
    int64_t E, OUT, NB, RT, NC, units;        // units of 16 bytes: E * RT * NC * 64
    uint8_t *pcodes, *pscales;
    int32_t *not_f16;
};

// One unit a thread: 16 bytes of codes from their row to their place.
__global__ void __launch_bounds__(256) k_mx_pack(const PackArgs p) {
    const int64_t u = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (u >= p.units) return;
    const int i = int(u & 63);
    const int64_t tile = u >> 6, c = tile % p.NC, et = tile / p.NC, rt = et % p.RT, e = et / p.RT;
    const int64_t row = rt * 16 + (i & 15), blk = 4 * c + (i >> 4);
    const bool in = row < p.OUT && blk < p.NB;
    const int64_t at = (e * p.OUT + row) * p.NB + blk;
    const u32x4 w = in ? reinterpret_cast<const u32x4 *>(p.codes)[at] : u32x4{};
    reinterpret_cast<u32x4 *>(p.pcodes)[u] = w;
    uint8_t *sc = p.pscales + ((et * ((p.NC + 3) / 4) + c / 4) * 64 + i) * 4;
    const uint32_t s = in ? p.scales[at] : 127u;
    sc[c & 3] = uint8_t(s);
    if (p.not_f16 && ((w.x | w.y | w.z | w.w) & 0x77777777u) != 0 && s != 255u &&
        (s < kMxF16ScaleMin || s > kMxF16ScaleMax))
        *p.not_f16 = 1;                       // every thread that writes it writes the same
    if (c == p.NC - 1)                        // the bytes of chunks past the end
        for (int j = int(c & 3) + 1; j < 4; ++j) sc[j] = 127;
}

}  // namespace vqk

using namespace vqk;

static int check_pack(int64_t E, int64_t OUT, int64_t IN) {
    if (E < 1 || OUT < 1 || IN < 1 || E > INT32_MAX || OUT > INT32_MAX / 2 || IN > INT32_MAX / 2)
        return set_error(VQK_EINVAL, "mx pack: bad shape E=%lld OUT=%lld IN=%lld", (long long)E, (long long)OUT,
                         (long long)IN);
    return VQK_OK;
}

extern "C" int vqk_mx_pack_bytes(int64_t E, int64_t OUT, int64_t IN, size_t *codes, size_t *scales) {
    const int rc = check_pack(E, OUT, IN);
    if (rc) return rc;
    if (!codes || !scales) return set_error(VQK_EINVAL, "mx pack: NULL sizes");
    const int64_t RT = (OUT + 15) / 16, NC = (IN + kMxChunk - 1) / kMxChunk;
    *codes = size_t(E) * mx_expert_codes(RT, NC);
    *scales = size_t(E) * mx_expert_scales(RT, NC);
    return VQK_OK;
}

extern "C" int vqk_mx_pack(const uint8_t *codes, const uint8_t *scales, int64_t E, int64_t OUT, int64_t IN,
                           uint8_t *pcodes, uint8_t *pscales, int32_t *not_f16, void *stream) {
    const int rc = check_pack(E, OUT, IN);
    if (rc) return rc;
    if (!codes || !scales || !pcodes || !pscales) return set_error(VQK_EINVAL, "mx pack: NULL pointer");
    if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(pcodes)) & 15)
        return set_error(VQK_EINVAL, "mx pack: codes must be 16-byte aligned");
    const int64_t RT = (OUT + 15) / 16, NC = (IN + kMxChunk - 1) / kMxChunk, units = E * RT * NC * 64;
    if ((units + 255) / 256 > INT32_MAX) return set_error(VQK_ENOTIMPL, "mx pack: weight too large");
    const PackArgs a{codes, scales, E, OUT, (IN + kMxBlock - 1) / kMxBlock, RT, NC, units, pcodes, pscales, not_f16};
    hipLaunchKernelGGL(k_mx_pack, dim3(unsigned((units + 255) / 256)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), a);
    return hip_status(hipGetLastError(), "MXFP4 pack launch");
}

extern "C" int vqk_mx_quantize(const void *x, int32_t x_type, int64_t rows, int64_t cols, int64_t ldx,
                               uint8_t *codes, uint8_t *scales, void *stream) {
    if (rows < 0 || cols < 0 || ldx < cols)
        return set_error(VQK_EINVAL, "mx quantize: bad shape rows=%lld cols=%lld ldx=%lld", (long long)rows,
                         (long long)cols, (long long)ldx);
    if (!act_size(x_type)) return set_error(VQK_EINVAL, "mx quantize: x type %d", x_type);
    if (rows == 0 || cols == 0) return VQK_OK;
    if (!x || !codes || !scales) return set_error(VQK_EINVAL, "mx quantize: NULL pointer");
    if (reinterpret_cast<uintptr_t>(codes) & 3)
        return set_error(VQK_EINVAL, "mx quantize: codes must be 4-byte aligned");
    return launch_mx_quant(x, x_type, rows, cols, ldx, (cols + kMxBlock - 1) / kMxBlock, false, codes, scales,
                           static_cast<hipStream_t>(stream));
}

extern "C" int vqk_mx_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t rows, int64_t cols,
                                 void *out, int32_t out_type, void *stream) {
    if (rows < 0 || cols < 0)
        return set_error(VQK_EINVAL, "mx dequantize: bad shape rows=%lld cols=%lld", (long long)rows,
                         (long long)cols);
    if (!act_size(out_type)) return set_error(VQK_EINVAL, "mx dequantize: output type %d", out_type);
    if (rows == 0 || cols == 0) return VQK_OK;
    if (!codes || !scales || !out) return set_error(VQK_EINVAL, "mx dequantize: NULL pointer");
    if (reinterpret_cast<uintptr_t>(codes) & 3)
        return set_error(VQK_EINVAL, "mx dequantize: codes must be 4-byte aligned");
    const int64_t NB = (cols + kMxBlock - 1) / kMxBlock;
    const DequantArgs a{codes, scales, cols, NB, rows * NB * 4, out};
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (out_type) {
        case VQK_F16: return go_dequant<VQK_F16>(a, st);
        case VQK_BF16: return go_dequant<VQK_BF16>(a, st);
        default: return go_dequant<VQK_F32>(a, st);
    }
}
