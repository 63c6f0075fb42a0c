// Dense linears with 8-bit weights: y = x . W^T of x as it is, of x quantised
// here, and of rows that are in 8 bits already; and the gradient of x,
// dx = dy . W.
//
// 8-bit rows run on the 8-bit matrix instructions where the output has 16 bits, and
// as the codes' values in bf16 where it has 32 (vqk_f8.h).
// bf16 x enters as it is, fp16 x too (every e4m3 code is an fp16 number), fp32 x as
// three exact bf16 planes. x that is a multiple of 8 wide is read in place (many rows:
// whole blocks wide), other x is laid out in the workspace first. The gradient sums over
// the weight's rows, along which its codes do not lie: they are transposed into the
// workspace, operand order to operand order, and the same products run on them with
// the strides of the scales exchanged.
#include "vqk_f8.h"

namespace vqk {

constexpr int64_t kMostWgs = (1 << 24) - 1;   // workgroups of 256: a launch has fewer than 2^32 threads

static size_t al256(size_t v) { return (v + 255) & ~size_t(255); }
static bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Rows [N][IN] to rows of whole blocks, zero past IN: 16-bit numbers as they are, fp32
// as three planes.
template <int XT>
__global__ void __launch_bounds__(256) k_f8_stage16(const void *x, int64_t N, int64_t IN, int64_t ld, uint16_t *out, bool vec) {
    const int64_t per = ld / 8, i = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (i >= N * per) return;
    const int64_t row = i / per, k0 = (i - row * per) * 8;
    if constexpr (XT == VQK_F32) {
        float v[8];
        mx_load8(x, XT, row * IN, k0, IN, vec, v);
#pragma unroll
        for (int pl = 0; pl < 3; ++pl) {
            u32x4 o;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t lo = mx_plane_next(v[2 * u]);
                o[u] = lo | (uint32_t(mx_plane_next(v[2 * u + 1])) << 16);
            }
            *reinterpret_cast<u32x4 *>(out + pl * N * ld + row * ld + k0) = o;
        }
    } else {
        const uint16_t *src = static_cast<const uint16_t *>(x) + row * IN + k0;
        u32x4 v{};
        if (vec && k0 + 8 <= IN) v = *reinterpret_cast<const u32x4 *>(src);
        else
            for (int u = 0; u < 8; ++u)
                if (k0 + u < IN) v[u / 2] |= uint32_t(src[u]) << (16 * (u & 1));
        *reinterpret_cast<u32x4 *>(out + row * ld + k0) = v;
    }
}

// 8-bit rows to whole blocks, zero past IN, and their scales block by block.
struct F8Stage {
    const uint8_t *codes;
    int64_t ldc, N, IN, NC;
    const float *scales;
    int64_t sn, sk;
    uint8_t *out;                             // [N][NC * 128]
    float *sout;                              // [NC][N], or NULL
};
// WIDE: as the codes' values in bf16, 2 bytes each.
template <bool WIDE>
__global__ void __launch_bounds__(256) k_f8_stage8(const F8Stage p, int64_t pieces) {
    const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (i >= pieces) return;
    const int64_t row = i / (p.NC * 8), q = i - row * (p.NC * 8), k0 = q * 16;
    u32x4 v{};
#pragma unroll
    for (int u = 0; u < 16; ++u)
        if (k0 + u < p.IN) v[u / 4] |= uint32_t(p.codes[row * p.ldc + k0 + u]) << (8 * (u & 3));
    if constexpr (WIDE) {
        u32x4 *dst = reinterpret_cast<u32x4 *>(p.out + (row * p.NC * 128 + k0) * 2);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            u32x4 o;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                o[2 * u] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * j + u], 1.f, false));
                o[2 * u + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * j + u], 1.f, true));
            }
            dst[j] = o;
        }
    } else {
        *reinterpret_cast<u32x4 *>(p.out + row * p.NC * 128 + k0) = v;
    }
    if ((q & 7) == 0 && p.sout) p.sout[(q >> 3) * p.N + row] = p.scales[row * p.sn + (q >> 3) * p.sk];
}

// ------------------------------------------------------- transposed codes
struct F8Trans {
    const uint8_t *codes;                     // [RT][NC][2][64][16]
    int32_t RT, NC, RTt, NCt;                 // RTt = ceil(IN / 16), NCt = ceil(OUT / 128)
    uint8_t *out;                             // [RTt][NCt][2][64][16]
};

// 128 x 128 codes through LDS: 16 k of a weight row in per unit, 4 x 16 codes
// turned by byte permutes, 16 weight rows of a k out. 5120 x 17408: 48 us (3.7 TB/s both ways).
__global__ void __launch_bounds__(256) k_f8_trans(const F8Trans p) {
    constexpr int LD = 144;
    __shared__ __align__(16) uint8_t tile[128 * LD];    // [weight row][k]
    const int kb = blockIdx.x, ob = blockIdx.y;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int u = j * 256 + threadIdx.x, i = u & 63, h = (u >> 6) & 1, rt = u >> 7;
        u32x4 w{};
        if (ob * 8 + rt < p.RT)
            w = *reinterpret_cast<const u32x4 *>(p.codes + (int64_t(ob * 8 + rt) * p.NC + kb) * 2048 + h * 1024 + i * 16);
        *reinterpret_cast<u32x4 *>(tile + (rt * 16 + (i & 15)) * LD + 32 * (i >> 4) + 16 * h) = w;
    }
    __syncthreads();
    const int k4 = threadIdx.x & 31, og = threadIdx.x >> 5;             // k 4 k4 .., weight rows 16 og ..
    u32x4 o[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        uint32_t a[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = *reinterpret_cast<const uint32_t *>(tile + (og * 16 + q * 4 + j) * LD + k4 * 4);
        // v_perm selects bytes 0-3 of its second operand, 4-7 of its first
        const uint32_t lo01 = __builtin_amdgcn_perm(a[1], a[0], 0x05010400u), hi01 = __builtin_amdgcn_perm(a[1], a[0], 0x07030602u);
        const uint32_t lo23 = __builtin_amdgcn_perm(a[3], a[2], 0x05010400u), hi23 = __builtin_amdgcn_perm(a[3], a[2], 0x07030602u);
        o[0][q] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100u);
        o[1][q] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302u);
        o[2][q] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100u);
        o[3][q] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302u);
    }
    const int rt = kb * 8 + k4 / 4;
    if (rt >= p.RTt) return;
    uint8_t *dst = p.out + (int64_t(rt) * p.NCt + ob) * 2048 + (og & 1) * 1024 + ((og >> 1) * 16 + (k4 & 3) * 4) * 16;
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<u32x4 *>(dst + j * 16) = o[j];
}

static int check_lin(const vqk_f8_weights *w, int64_t N, F8Geom *g, const char *what) {
    const int rc = make_f8_geom(w, g, what);
    if (rc) return rc;
    if (N < 0 || N > INT32_MAX / 2) return set_error(VQK_EINVAL, "%s: N=%lld", what, (long long)N);
    return VQK_OK;
}

// x as it is: its layout in the workspace, where it cannot be read in place (few rows are
// read in pieces of 8, many in whole blocks), then the K slices of tiles.
static int x_planes(int32_t type) { return type == VQK_F32 ? 3 : 1; }
struct PlainPlan { bool few, lay; size_t x, part; };
static PlainPlan plain_plan(const F8Geom &g, int32_t type, int64_t N) {
    F8Call c{};
    c.g = g;
    c.N = N;
    c.x.P = x_planes(type);
    c.x.op = type == VQK_F16 ? kOpF16 : kOpBF16;
    PlainPlan p{};
    p.few = f8_rows_ok(c);
    p.lay = type == VQK_F32 || g.IN % (p.few ? 8 : kF8Block);
    p.x = p.lay ? al256(size_t(N) * g.NC * 256 * c.x.P) : 0;
    p.part = p.few ? f8_rows_part(c) : f8_tiles_part(N, g, false, false, c.x.P);
    return p;
}
static size_t plain_bytes(const F8Geom &g, int32_t type, int64_t N) {
    const PlainPlan p = plain_plan(g, type, N);
    return p.x + p.part;
}
// 8-bit x that is not in place: rows of whole blocks and their scales (and for an fp32
// output the codes' values after them); then the K slices.
static bool wide_out(int32_t y_type) { return (y_type & ~VQK_VIA_F16) == VQK_F32; }
static size_t code_bytes(const F8Geom &g, int64_t N) { return al256(size_t(N) * g.NC * 128); }
static size_t scale_bytes(const F8Geom &g, int64_t N) { return al256(size_t(N) * g.NC * 4); }
static size_t rows_bytes(const F8Geom &g, int64_t N, int32_t y_type) {
    return code_bytes(g, N) + scale_bytes(g, N) + (wide_out(y_type) ? al256(size_t(N) * g.NC * 256) : 0);
}
struct A8Plan { bool few, place; size_t x, part; };
// ldc: bytes between rows that are in 8 bits already, 0 for rows quantised here.
static A8Plan a8_plan(const F8Geom &g, int64_t N, int64_t ldc, int32_t y_type) {
    const bool wide = wide_out(y_type);
    F8Call c{};
    c.g = g;
    c.N = N;
    c.a8 = !wide;
    c.x.P = 1;
    c.x.op = kOpBF16;
    A8Plan p{};
    p.few = f8_rows_ok(c);
    // in place, if a tile's rows are within reach of 32-bit offsets
    p.place = ldc && !wide && g.IN % 128 == 0 && ldc % 16 == 0 && ldc < (1 << 24);
    p.x = p.place ? 0 : rows_bytes(g, N, y_type);
    p.part = p.few ? f8_rows_part(c) : f8_tiles_part(N, g, !wide, true, 1);
    return p;
}
static size_t a8_bytes(const F8Geom &g, int64_t N, int64_t ldc, int32_t y_type) {
    const A8Plan p = a8_plan(g, N, ldc, y_type);
    return p.x + p.part;
}

static int check_ws(const char *what, size_t need, const void *ws, size_t ws_bytes) {
    if (need && (!ws || ws_bytes < need)) return set_error(VQK_ENOSPACE, "%s: workspace %zu < %zu", what, ws_bytes, need);
    if (reinterpret_cast<uintptr_t>(ws) & 255) return set_error(VQK_EINVAL, "%s: workspace must be 256-byte aligned", what);
    return VQK_OK;
}

// The product of x (16-byte aligned) as it is; ws: plain_bytes.
static int plain_product(F8Call c, const void *x, int32_t type, uint8_t *ws, hipStream_t st) {
    const int64_t N = c.N, IN = c.g.IN, ld = c.g.NC * kF8Block;
    const PlainPlan p = plain_plan(c.g, type, N);
    c.x = MxX{static_cast<const uint16_t *>(x), IN, 0, x_planes(type), type == VQK_F16 ? kOpF16 : kOpBF16};
    if (p.lay) {
        const int64_t wgs = (N * (ld / 8) + 255) / 256;
        if (wgs > kMostWgs) return set_error(VQK_ENOTIMPL, "f8 linear: %lld rows of %lld", (long long)N, (long long)IN);
        uint16_t *out = reinterpret_cast<uint16_t *>(ws);
        const bool vec = (IN * act_size(type)) % 16 == 0;
        if (type == VQK_F32) hipLaunchKernelGGL((k_f8_stage16<VQK_F32>), dim3(unsigned(wgs)), dim3(256), 0, st, x, N, IN, ld, out, vec);
        else hipLaunchKernelGGL((k_f8_stage16<VQK_F16>), dim3(unsigned(wgs)), dim3(256), 0, st, x, N, IN, ld, out, vec);   // 16 bits as they are
        const int rc = hip_status(hipGetLastError(), "x staging launch");
        if (rc) return rc;
        c.x.x = out;
        c.x.ld = ld;
        c.x.plane = N * ld;
        c.g.IN = ld;
    }
    float *part = p.part ? reinterpret_cast<float *>(ws + p.x) : nullptr;
    return p.few ? f8_rows(c, part, p.part, st) : f8_tiles(c, part, p.part, st);
}

// The product of 8-bit rows; ws: a8_bytes. here: they are whole blocks at its start, with
// their scales after them.
static int a8_product(F8Call c, const F8X &x, bool here, uint8_t *ws, hipStream_t st) {
    const int64_t N = c.N;
    const A8Plan p = a8_plan(c.g, N, here ? 0 : x.ld, c.y_type);
    const bool wide = wide_out(c.y_type);
    c.x8 = x;
    c.a8 = !wide;
    if (wide || !(p.place || here)) {
        uint8_t *to = wide ? ws + code_bytes(c.g, N) + scale_bytes(c.g, N) : ws;
        float *sx = reinterpret_cast<float *>(ws + code_bytes(c.g, N));
        const F8Stage s{x.codes, x.ld, N, c.g.IN, c.g.NC, x.scales, x.sn, x.sk, to, here ? nullptr : sx};
        const int64_t pieces = N * c.g.NC * 8, wgs = (pieces + 255) / 256;
        if (wgs > kMostWgs) return set_error(VQK_ENOTIMPL, "f8 linear: %lld rows of %lld", (long long)N, (long long)c.g.IN);
        if (wide) hipLaunchKernelGGL((k_f8_stage8<true>), dim3(unsigned(wgs)), dim3(256), 0, st, s, pieces);
        else hipLaunchKernelGGL((k_f8_stage8<false>), dim3(unsigned(wgs)), dim3(256), 0, st, s, pieces);
        const int rc = hip_status(hipGetLastError(), "8-bit row staging launch");
        if (rc) return rc;
        c.x8 = F8X{ws, c.g.NC * 128, here ? x.scales : sx, here ? x.sn : 1, here ? x.sk : N};
        if (wide) c.x = MxX{reinterpret_cast<uint16_t *>(to), c.g.NC * 128, 0, 1, kOpBF16};
    }
    if (wide) c.g.IN = c.g.NC * 128;          // x's rows are whole blocks, zero past the weight's columns
    float *part = p.part ? reinterpret_cast<float *>(ws + p.x) : nullptr;
    return p.few ? f8_rows(c, part, p.part, st) : f8_tiles(c, part, p.part, st);
}

static F8Call base_call(const vqk_f8_weights *w, const F8Geom &g, int64_t N, bool a8, void *y, int32_t y_type) {
    F8Call c{};
    c.codes = w->codes; c.scales = w->scales;
    c.swo = g.NC; c.swk = 1;
    c.g = g;
    c.N = N; c.a8 = a8;
    c.y = y; c.y_type = y_type;
    return c;
}

// The transposed weight: OUT and IN exchanged.
static F8Geom transposed(const F8Geom &g) { return F8Geom{g.IN, g.OUT, (g.IN + 15) / 16, (g.OUT + 127) / 128}; }

}  // namespace vqk

using namespace vqk;

static int check_act(int32_t act, int32_t x_type) {
    if (!act_size(x_type)) return set_error(VQK_EINVAL, "f8 linear: x type %d", x_type);
    return act == VQK_F8_ACT_NONE || act == VQK_F8_ACT_F8 ? VQK_OK : set_error(VQK_EINVAL, "f8 linear: activation form %d", act);
}

extern "C" int vqk_f8_linear_workspace(const vqk_f8_weights *w, int32_t x_type, int64_t N, int32_t act, int32_t y_type,
                                       size_t *bytes) {
    F8Geom g;
    int rc = check_lin(w, N, &g, "f8 linear");
    if (rc || (rc = check_act(act, x_type))) return rc;
    if (!out_size(y_type)) return set_error(VQK_EINVAL, "f8 linear: y type %d", y_type);
    if (!bytes) return set_error(VQK_EINVAL, "f8 linear: NULL bytes");
    *bytes = N == 0 ? 0 : (act == VQK_F8_ACT_F8 ? a8_bytes(g, N, 0, y_type) : plain_bytes(g, x_type, N));
    return VQK_OK;
}

extern "C" int vqk_f8_linear(const vqk_f8_weights *w, const void *x, int32_t x_type, int64_t N, int32_t act, void *y,
                             int32_t y_type, void *workspace, size_t ws_bytes, void *stream) {
    F8Geom g;
    int rc = check_lin(w, N, &g, "f8 linear");
    if (rc || (rc = check_act(act, x_type))) return rc;
    if (!out_size(y_type)) return set_error(VQK_EINVAL, "f8 linear: y type %d", y_type);
    if (N == 0) return VQK_OK;
    if (!x || !y) return set_error(VQK_EINVAL, "f8 linear: NULL pointer");
    if (act == VQK_F8_ACT_NONE && !al16(x)) return set_error(VQK_EINVAL, "f8 linear: x must be 16-byte aligned");
    const size_t need = act == VQK_F8_ACT_F8 ? a8_bytes(g, N, 0, y_type) : plain_bytes(g, x_type, N);
    if ((rc = check_ws("f8 linear", need, workspace, ws_bytes))) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    F8Call c = base_call(w, g, N, act == VQK_F8_ACT_F8, y, y_type);
    if (!c.a8) return plain_product(c, x, x_type, ws, st);
    float *sx = reinterpret_cast<float *>(ws + code_bytes(g, N));
    const F8Quant q{x, N, g.IN, g.IN, ws, g.NC * 128, g.NC * 128, sx, 1, N};
    if ((rc = launch_f8_quant(q, x_type, st))) return rc;
    return a8_product(c, F8X{ws, g.NC * 128, sx, 1, N}, true, ws, st);
}

extern "C" int vqk_f8_linear_rows_workspace(const vqk_f8_weights *w, int64_t ldc, int64_t N, int32_t y_type, size_t *bytes) {
    F8Geom g;
    const int rc = check_lin(w, N, &g, "f8 linear of rows");
    if (rc) return rc;
    if (!out_size(y_type)) return set_error(VQK_EINVAL, "f8 linear of rows: y type %d", y_type);
    if (ldc < g.IN) return set_error(VQK_EINVAL, "f8 linear of rows: rows %lld apart", (long long)ldc);
    if (!bytes) return set_error(VQK_EINVAL, "f8 linear of rows: NULL bytes");
    *bytes = N == 0 ? 0 : a8_bytes(g, N, ldc, y_type);
    return VQK_OK;
}

extern "C" int vqk_f8_linear_rows(const vqk_f8_weights *w, const uint8_t *codes, int64_t ldc, const float *scales,
                                  int64_t scale_row, int64_t scale_block, int64_t N, void *y, int32_t y_type,
                                  void *workspace, size_t ws_bytes, void *stream) {
    F8Geom g;
    int rc = check_lin(w, N, &g, "f8 linear of rows");
    if (rc) return rc;
    if (!out_size(y_type)) return set_error(VQK_EINVAL, "f8 linear of rows: y type %d", y_type);
    if (ldc < g.IN || scale_row < 0 || scale_block < 0)
        return set_error(VQK_EINVAL, "f8 linear of rows: strides %lld, %lld, %lld", (long long)ldc, (long long)scale_row, (long long)scale_block);
    if (N == 0) return VQK_OK;
    if (!codes || !scales || !y) return set_error(VQK_EINVAL, "f8 linear of rows: NULL pointer");
    if (!al16(codes)) return set_error(VQK_EINVAL, "f8 linear of rows: codes must be 16-byte aligned");
    if ((rc = check_ws("f8 linear of rows", a8_bytes(g, N, ldc, y_type), workspace, ws_bytes))) return rc;
    return a8_product(base_call(w, g, N, true, y, y_type), F8X{codes, ldc, scales, scale_row, scale_block}, false,
                      static_cast<uint8_t *>(workspace), static_cast<hipStream_t>(stream));
}

extern "C" int vqk_f8_linear_dx_workspace(const vqk_f8_weights *w, int32_t type, int64_t N, size_t *bytes) {
    F8Geom g;
    const int rc = check_lin(w, N, &g, "f8 linear dx");
    if (rc) return rc;
    if (!act_size(type)) return set_error(VQK_EINVAL, "f8 linear dx: type %d", type);
    if (!bytes) return set_error(VQK_EINVAL, "f8 linear dx: NULL bytes");
    const F8Geom t = transposed(g);
    *bytes = N == 0 ? 0 : al256(f8_code_bytes(t.RT, t.NC)) + plain_bytes(t, type, N);
    return VQK_OK;
}

extern "C" int vqk_f8_linear_dx(const vqk_f8_weights *w, const void *dy, int32_t type, int64_t N, void *dx,
                                int32_t dx_type, void *workspace, size_t ws_bytes, void *stream) {
    F8Geom g;
    int rc = check_lin(w, N, &g, "f8 linear dx");
    if (rc) return rc;
    if (!act_size(type) || !out_size(dx_type)) return set_error(VQK_EINVAL, "f8 linear dx: types %d, %d", type, dx_type);
    if (N == 0) return VQK_OK;
    if (!dy || !dx) return set_error(VQK_EINVAL, "f8 linear dx: NULL pointer");
    if (!al16(dy)) return set_error(VQK_EINVAL, "f8 linear dx: dy must be 16-byte aligned");
    const F8Geom t = transposed(g);
    const size_t codes = al256(f8_code_bytes(t.RT, t.NC));
    if (f8_code_bytes(t.RT, t.NC) > INT64_C(0xffffffff) || t.NC > 65535)
        return set_error(VQK_ENOTIMPL, "f8 linear dx: OUT=%lld IN=%lld", (long long)g.OUT, (long long)g.IN);
    if ((rc = check_ws("f8 linear dx", codes + plain_bytes(t, type, N), workspace, ws_bytes))) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    const F8Trans a{w->codes, int32_t(g.RT), int32_t(g.NC), int32_t(t.RT), int32_t(t.NC), ws};
    hipLaunchKernelGGL(k_f8_trans, dim3(unsigned(g.NC), unsigned(t.NC)), dim3(256), 0, st, a);
    if ((rc = hip_status(hipGetLastError(), "8-bit transposition launch"))) return rc;
    F8Call c = base_call(w, t, N, false, dx, dx_type);
    c.codes = ws;
    c.swo = 1; c.swk = g.NC;
    return plain_product(c, dy, type, ws + codes, st);
}
