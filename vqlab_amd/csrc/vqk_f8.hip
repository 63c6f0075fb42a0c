// 8-bit rows and weights: quantisers, the way back, and the operand order of
// weights (straight, and transposed for the gradient of x).
//
//     s = max(amax / 448, 2^-126) of a block,   code = e4m3(v * (1 / s))
//
// rounded to nearest (ties to even); |v| * (1 / s) stays below 448 (1 + 2^-22),
// which rounds to 448. A block with an infinity or NaN gets the scale NaN and
// codes 0, and reads back as NaN. Bound by memory: a row's block is 16 lanes of
// 8 values, so a wave's loads are contiguous, and the largest magnitude takes
// four DPP steps inside the lanes' row. Measured: 2048 rows of 5120 bf16 9.6 us (3.3 TB/s,
// out of the MALL in part), 20 rows 3.2, back to bf16 8.4.
#include "vqk_f8.h"

namespace vqk {

int make_f8_geom(const vqk_f8_weights *w, F8Geom *g, const char *what) {
    if (!w) return set_error(VQK_EINVAL, "%s: NULL weights", what);
    if (w->OUT < 1 || w->IN < 1 || w->OUT > INT32_MAX / 2 || w->IN > INT32_MAX / 2)
        return set_error(VQK_EINVAL, "%s: bad shape OUT=%lld IN=%lld", what, (long long)w->OUT, (long long)w->IN);
    if (!w->codes || !w->scales) return set_error(VQK_EINVAL, "%s: codes and scales are required", what);
    if (reinterpret_cast<uintptr_t>(w->codes) & 15)
        return set_error(VQK_EINVAL, "%s: codes must be 16-byte aligned", what);
    if (reinterpret_cast<uintptr_t>(w->scales) & 3)
        return set_error(VQK_EINVAL, "%s: scales must be 4-byte aligned", what);
    *g = F8Geom{w->OUT, w->IN, (w->OUT + 15) / 16, (w->IN + 127) / 128};
    // kernels reach a weight's codes by 32-bit offsets
    if (f8_code_bytes(g->RT, g->NC) > INT64_C(0xffffffff))
        return set_error(VQK_ENOTIMPL, "%s: a weight of 4 GB or more", what);
    return VQK_OK;
}

// Sixteen lanes a block, 8 values each.
template <int XT, bool VEC>
__global__ void __launch_bounds__(256) k_f8_quant(const F8Quant p, int64_t NB, int64_t pieces) {
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < pieces; i += int64_t(gridDim.x) * 256) {
        const int64_t blk = i >> 4, row = blk / NB, b = blk - row * NB, k0 = b * kF8Block + (i & 15) * 8;
        float v[8];
        mx_load8(p.x, XT, row * p.ldx, k0, p.C, VEC, v);
        uint32_t m = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) m = max(m, __float_as_uint(v[u]) & 0x7fffffffu);
        // pieces come in whole blocks (pieces % 16 == 0 and 256 % 16 == 0): all sixteen lanes are here
        const float s = f8_scale(row16_max(m));
        const bool ok = s == s;
        const u32x2 c = f8_encode8(v, 1.f / s, ok);
        uint8_t *dst = p.codes + row * p.ldc + k0;
        if ((p.ldc & 7) == 0 && (reinterpret_cast<uintptr_t>(p.codes) & 7) == 0 && k0 + 8 <= p.cover) {
            *reinterpret_cast<u32x2 *>(dst) = c;
        } else {
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (k0 + u < p.cover) dst[u] = uint8_t(c[u / 4] >> (8 * (u % 4)));
        }
        if ((i & 15) == 0) p.scales[row * p.sn + b * p.sk] = s;
    }
}

int launch_f8_quant(const F8Quant &q, int32_t type, hipStream_t st) {
    const int64_t NB = (q.C + kF8Block - 1) / kF8Block, pieces = q.N * NB * 16;
    if (pieces == 0) return VQK_OK;
    const bool vec = (reinterpret_cast<uintptr_t>(q.x) & 15) == 0 && (q.ldx * act_size(type)) % 16 == 0;
    const int64_t wgs = (pieces + 255) / 256;
    const dim3 grid(unsigned(wgs < 16384 ? wgs : 16384));
#define VQK_GO(T)                                                                                              \
    if (vec) hipLaunchKernelGGL((k_f8_quant<T, true>), grid, dim3(256), 0, st, q, NB, pieces);                 \
    else hipLaunchKernelGGL((k_f8_quant<T, false>), grid, dim3(256), 0, st, q, NB, pieces)
    switch (type) {
        case VQK_F16: VQK_GO(VQK_F16); break;
        case VQK_BF16: VQK_GO(VQK_BF16); break;
        default: VQK_GO(VQK_F32);
    }
#undef VQK_GO
    return hip_status(hipGetLastError(), "8-bit quantiser launch");
}

struct F8WQuant {
    const void *w;
    int64_t OUT, IN, ldw;
    uint8_t *codes;                           // [OUT][IN]
    float *scales;                            // [ceil(OUT / 128)][ceil(IN / 128)]
};

// A block of 128 x 128 a workgroup: 16 lanes a row, 16 rows a round.
template <int XT, bool VEC>
__global__ void __launch_bounds__(256) k_f8_wquant(const F8WQuant p) {
    __shared__ uint32_t top[4];
    const int64_t o0 = int64_t(blockIdx.y) * kF8Block, k0 = int64_t(blockIdx.x) * kF8Block + (threadIdx.x & 15) * 8;
    float v[8][8];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int64_t o = o0 + j * 16 + (threadIdx.x >> 4);
#pragma unroll
        for (int u = 0; u < 8; ++u) v[j][u] = 0.f;
        if (o < p.OUT) mx_load8(p.w, XT, o * p.ldw, k0, p.IN, VEC, v[j]);
#pragma unroll
        for (int u = 0; u < 8; ++u) m = max(m, __float_as_uint(v[j][u]) & 0x7fffffffu);
    }
    m = wave_max_u32(m);
    if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
    __syncthreads();
    m = max(max(top[0], top[1]), max(top[2], top[3]));
    const float s = f8_scale(m), inv = 1.f / s;
    const bool ok = s == s;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int64_t o = o0 + j * 16 + (threadIdx.x >> 4);
        if (o >= p.OUT) continue;
        const u32x2 c = f8_encode8(v[j], inv, ok);
        uint8_t *dst = p.codes + o * p.IN + k0;
        if ((p.IN & 7) == 0 && (reinterpret_cast<uintptr_t>(p.codes) & 7) == 0 && k0 + 8 <= p.IN) {
            *reinterpret_cast<u32x2 *>(dst) = c;
        } else {
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (k0 + u < p.IN) dst[u] = uint8_t(c[u / 4] >> (8 * (u % 4)));
        }
    }
    if (threadIdx.x == 0) p.scales[int64_t(blockIdx.y) * gridDim.x + blockIdx.x] = s;
}

struct F8Dequant {
    const uint8_t *codes;
    int64_t ldc, rows, cols;
    const float *scales;
    int64_t so, sk;                           // floats between scales of neighbouring rows (or blocks of rows), blocks
    int32_t shift;                            // rows of a scale: 1 << shift
    void *out;
};

// Eight codes a thread.
template <int YT>
__global__ void __launch_bounds__(256) k_f8_dequant(const F8Dequant p, int64_t per, int64_t pieces, bool vin, bool vout) {
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < pieces; i += int64_t(gridDim.x) * 256) {
        const int64_t row = i / per, k0 = (i - row * per) * 8;
        const uint8_t *src = p.codes + row * p.ldc + k0;
        u32x2 c{};
        if (vin && k0 + 8 <= p.cols) c = *reinterpret_cast<const u32x2 *>(src);
        else
            for (int u = 0; u < 8; ++u)
                if (k0 + u < p.cols) c[u / 4] |= uint32_t(src[u]) << (8 * (u % 4));
        const float s = p.scales[(row >> p.shift) * p.so + (k0 >> 7) * p.sk];
        float v[8];
        f8_decode8(c, v);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            v[u] *= s;
            asm("" : "+v"(v[u]));             // an fp32 number, not one half of a multiplication that rounds to fp16
        }
        const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
        const int64_t at = row * p.cols + k0;
        const int n = int(min(int64_t(8), p.cols - k0));
        mx_store4(p.out, YT, at, a, min(n, 4), vout);
        if (n > 4) mx_store4(p.out, YT, at + 4, b, n - 4, vout);
    }
}

// ------------------------------------------------------------ operand order
struct F8Pack {
    const uint8_t *codes;                     // rows [OUT][IN]
    int64_t OUT, IN, NC, units;               // units of 16 bytes: RT * NC * 128
    uint8_t *out;
};

// One unit a thread; BACK: from operand order to rows.
template <bool BACK>
__global__ void __launch_bounds__(256) k_f8_pack(const F8Pack p, bool vec) {
    const int64_t u = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (u >= p.units) return;
    const int i = int(u & 63), h = int(u >> 6) & 1;
    const int64_t tile = u >> 7, c = tile % p.NC, rt = tile / p.NC;
    const int64_t row = rt * 16 + (i & 15), k = c * kF8Block + 32 * (i >> 4) + 16 * h;
    if constexpr (BACK) {
        if (row >= p.OUT) return;
        const u32x4 w = reinterpret_cast<const u32x4 *>(p.codes)[u];
        uint8_t *dst = p.out + row * p.IN + k;
        if (vec && k + 16 <= p.IN) *reinterpret_cast<u32x4 *>(dst) = w;
        else
            for (int b = 0; b < 16; ++b)
                if (k + b < p.IN) dst[b] = uint8_t(w[b / 4] >> (8 * (b % 4)));
    } else {
        u32x4 w{};
        const uint8_t *src = p.codes + row * p.IN + k;
        if (row < p.OUT) {
            if (vec && k + 16 <= p.IN) w = *reinterpret_cast<const u32x4 *>(src);
            else
                for (int b = 0; b < 16; ++b)
                    if (k + b < p.IN) w[b / 4] |= uint32_t(src[b]) << (8 * (b % 4));
        }
        reinterpret_cast<u32x4 *>(p.out)[u] = w;
    }
}

}  // namespace vqk

using namespace vqk;

extern "C" int vqk_f8_quantize(const void *x, int32_t x_type, int64_t rows, int64_t cols, int64_t ldx,
                               uint8_t *codes, float *scales, int64_t scale_row, int64_t scale_block, void *stream) {
    if (rows < 0 || cols < 0 || ldx < cols)
        return set_error(VQK_EINVAL, "f8 quantize: bad shape rows=%lld cols=%lld ldx=%lld", (long long)rows,
                         (long long)cols, (long long)ldx);
    if (!act_size(x_type)) return set_error(VQK_EINVAL, "f8 quantize: x type %d", x_type);
    if (rows == 0 || cols == 0) return VQK_OK;
    if (!x || !codes || !scales) return set_error(VQK_EINVAL, "f8 quantize: NULL pointer");
    if (scale_row < 0 || scale_block < 0) return set_error(VQK_EINVAL, "f8 quantize: negative stride of scales");
    const F8Quant q{x, rows, cols, ldx, codes, cols, cols, scales, scale_row, scale_block};
    return launch_f8_quant(q, x_type, static_cast<hipStream_t>(stream));
}

extern "C" int vqk_f8_quantize_weight(const void *w, int32_t w_type, int64_t OUT, int64_t IN, int64_t ldw,
                                      uint8_t *codes, float *scales, void *stream) {
    if (OUT < 0 || IN < 0 || ldw < IN)
        return set_error(VQK_EINVAL, "f8 quantize weight: bad shape OUT=%lld IN=%lld ld=%lld", (long long)OUT,
                         (long long)IN, (long long)ldw);
    const int esz = act_size(w_type);
    if (!esz) return set_error(VQK_EINVAL, "f8 quantize weight: type %d", w_type);
    if (OUT == 0 || IN == 0) return VQK_OK;
    if (!w || !codes || !scales) return set_error(VQK_EINVAL, "f8 quantize weight: NULL pointer");
    const int64_t ob = (OUT + 127) / 128, kb = (IN + 127) / 128;
    if (ob > 65535 || kb > INT32_MAX) return set_error(VQK_ENOTIMPL, "f8 quantize weight: OUT=%lld", (long long)OUT);
    const F8WQuant a{w, OUT, IN, ldw, codes, scales};
    const bool vec = (reinterpret_cast<uintptr_t>(w) & 15) == 0 && (ldw * esz) % 16 == 0;
    const dim3 grid{unsigned(kb), unsigned(ob)};
    hipStream_t st = static_cast<hipStream_t>(stream);
#define VQK_GO(T)                                                                      \
    if (vec) hipLaunchKernelGGL((k_f8_wquant<T, true>), grid, dim3(256), 0, st, a);    \
    else hipLaunchKernelGGL((k_f8_wquant<T, false>), grid, dim3(256), 0, st, a)
    switch (w_type) {
        case VQK_F16: VQK_GO(VQK_F16); break;
        case VQK_BF16: VQK_GO(VQK_BF16); break;
        default: VQK_GO(VQK_F32);
    }
#undef VQK_GO
    return hip_status(hipGetLastError(), "8-bit weight quantiser launch");
}

extern "C" int vqk_f8_dequantize(const uint8_t *codes, int64_t ldc, const float *scales, int64_t scale_row,
                                 int64_t scale_block, int32_t rows_per_scale, int64_t rows, int64_t cols, void *out,
                                 int32_t out_type, void *stream) {
    if (rows < 0 || cols < 0 || ldc < cols)
        return set_error(VQK_EINVAL, "f8 dequantize: bad shape rows=%lld cols=%lld ld=%lld", (long long)rows,
                         (long long)cols, (long long)ldc);
    if (!act_size(out_type)) return set_error(VQK_EINVAL, "f8 dequantize: output type %d", out_type);
    if (rows_per_scale != 1 && rows_per_scale != kF8Block)
        return set_error(VQK_EINVAL, "f8 dequantize: a scale for %d rows", rows_per_scale);
    if (scale_row < 0 || scale_block < 0) return set_error(VQK_EINVAL, "f8 dequantize: negative stride of scales");
    if (rows == 0 || cols == 0) return VQK_OK;
    if (!codes || !scales || !out) return set_error(VQK_EINVAL, "f8 dequantize: NULL pointer");
    const F8Dequant a{codes, ldc, rows, cols, scales, scale_row, scale_block, rows_per_scale == 1 ? 0 : 7, out};
    const int64_t per = (cols + 7) / 8, pieces = rows * per, wgs = (pieces + 255) / 256;
    const bool vin = (ldc & 7) == 0 && (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
    const bool vout = (cols & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    const dim3 grid(unsigned(wgs < 16384 ? wgs : 16384));
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (out_type) {
        case VQK_F16: hipLaunchKernelGGL((k_f8_dequant<VQK_F16>), grid, dim3(256), 0, st, a, per, pieces, vin, vout); break;
        case VQK_BF16: hipLaunchKernelGGL((k_f8_dequant<VQK_BF16>), grid, dim3(256), 0, st, a, per, pieces, vin, vout); break;
        default: hipLaunchKernelGGL((k_f8_dequant<VQK_F32>), grid, dim3(256), 0, st, a, per, pieces, vin, vout);
    }
    return hip_status(hipGetLastError(), "8-bit dequantiser launch");
}

static int check_pack(int64_t OUT, int64_t IN, int64_t *RT, int64_t *NC) {
    if (OUT < 1 || IN < 1 || OUT > INT32_MAX / 2 || IN > INT32_MAX / 2)
        return set_error(VQK_EINVAL, "f8 pack: bad shape OUT=%lld IN=%lld", (long long)OUT, (long long)IN);
    *RT = (OUT + 15) / 16;
    *NC = (IN + 127) / 128;
    if (f8_code_bytes(*RT, *NC) > INT64_C(0xffffffff))
        return set_error(VQK_ENOTIMPL, "f8 pack: a weight of 4 GB or more");
    return VQK_OK;
}

extern "C" int vqk_f8_pack_bytes(int64_t OUT, int64_t IN, size_t *bytes) {
    int64_t RT, NC;
    const int rc = check_pack(OUT, IN, &RT, &NC);
    if (rc) return rc;
    if (!bytes) return set_error(VQK_EINVAL, "f8 pack: NULL bytes");
    *bytes = size_t(f8_code_bytes(RT, NC));
    return VQK_OK;
}

static int f8_pack(const uint8_t *from, int64_t OUT, int64_t IN, uint8_t *to, bool back, void *stream) {
    int64_t RT, NC;
    const int rc = check_pack(OUT, IN, &RT, &NC);
    if (rc) return rc;
    if (!from || !to) return set_error(VQK_EINVAL, "f8 pack: NULL pointer");
    const uintptr_t packed = reinterpret_cast<uintptr_t>(back ? from : to), rows = reinterpret_cast<uintptr_t>(back ? to : from);
    if (packed & 15) return set_error(VQK_EINVAL, "f8 pack: packed codes must be 16-byte aligned");
    const F8Pack a{from, OUT, IN, NC, RT * NC * 128, to};
    const bool vec = (rows & 15) == 0 && (IN & 15) == 0;
    const dim3 grid(unsigned((a.units + 255) / 256));
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (back) hipLaunchKernelGGL((k_f8_pack<true>), grid, dim3(256), 0, st, a, vec);
    else hipLaunchKernelGGL((k_f8_pack<false>), grid, dim3(256), 0, st, a, vec);
    return hip_status(hipGetLastError(), "8-bit pack launch");
}

extern "C" int vqk_f8_pack(const uint8_t *codes, int64_t OUT, int64_t IN, uint8_t *packed, void *stream) {
    return f8_pack(codes, OUT, IN, packed, false, stream);
}
extern "C" int vqk_f8_unpack(const uint8_t *packed, int64_t OUT, int64_t IN, uint8_t *codes, void *stream) {
    return f8_pack(packed, OUT, IN, codes, true, stream);
}
