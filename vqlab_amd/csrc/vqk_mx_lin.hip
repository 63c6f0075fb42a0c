// Dense linears with MXFP4 weights: y = x . W^T and the gradient of x,
// dx = dy . W.
//
// The forward product streams the weights past few rows (vqk_mxs.h) or
// multiplies tiles of many (vqk_mxg.h; 4-bit x: vqk_mxf.h). x that is bf16 (or
// fp16, for weights that are fp16 numbers), 16-byte aligned and whole blocks wide
// is read in place; other x is laid out
// once in the workspace as exact bf16 planes (vqk_mx.h). The gradient sums over the
// weight's rows, along which its codes do not lie: the weight is decoded,
// transposed, into the workspace as bf16 (exact) and multiplied by the
// matrix-core GEMM of the dense prefill path.
#include "vqk_mxs.h"

namespace vqk {

static size_t al256(size_t v) { return (v + 255) & ~size_t(255); }


// ------------------------------------------------------- transposed decode
struct DecTArgs {
    const uint8_t *codes, *scales;
    int64_t IN, RT, NC, KO;                   // KO: columns of one copy of the transposed weight
    int32_t P;
    uint16_t *out;                            // [IN][P * KO], zero past OUT
};

// 64 weight rows x one chunk through LDS: 16 bytes of codes in per thread,
// 16-byte pieces of a transposed row out.
__global__ void __launch_bounds__(256) k_mx_dec_t(const DecTArgs p) {
    __shared__ __align__(16) uint16_t tile[128][72];     // read in 16-byte pieces
    const int64_t o0 = int64_t(blockIdx.x) * 64, c = blockIdx.y, k0 = c * kMxChunk;
    {
        const int unit = threadIdx.x & 63, o = (threadIdx.x >> 6) * 16 + (unit & 15), g = unit >> 4;
        const int64_t rt = o0 / 16 + (threadIdx.x >> 6);
        const bool ok = rt < p.RT;
        const u32x4 w = ok ? *reinterpret_cast<const u32x4 *>(p.codes + ((rt * p.NC + c) * 64 + unit) * 16) : u32x4{};
        const uint32_t s = ok ? p.scales[((rt * ((p.NC + 3) / 4) + c / 4) * 64 + unit) * 4 + c % 4] : 127u;
        const float sc = mx_scale(s == 255u ? 127u : s);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const u32x4 v = mx_decode8(w[k], sc);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t q = s == 255u ? 0x7fc07fc0u : v[u];
                tile[g * 32 + k * 8 + 2 * u][o] = uint16_t(q & 0xffffu);
                tile[g * 32 + k * 8 + 2 * u + 1][o] = uint16_t(q >> 16);
            }
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 128 * 8; e += 256) {
        const int k = e >> 3, c = (e & 7) * 8;
        if (k0 + k >= p.IN) continue;
        const u32x4 v = *reinterpret_cast<const u32x4 *>(&tile[k][c]);
        uint16_t *dst = p.out + (k0 + k) * p.P * p.KO + o0 + c;
        for (int pl = 0; pl < p.P; ++pl) *reinterpret_cast<u32x4 *>(dst + pl * p.KO) = v;
    }
}

// dy rows as [plane 0 | plane 1 | ...] of KO columns each, zero past OUT.
struct DyArgs {
    const void *dy;
    int64_t N, OUT, KO;
    uint16_t *out;
};
template <int XT>
__global__ void __launch_bounds__(256) k_mx_dy(const DyArgs p, bool vec) {
    constexpr int P = mx_planes(XT);
    const int64_t per = p.KO / 8, i = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (i >= p.N * per) return;
    const int64_t row = i / per, c = (i - row * per) * 8;
    float v[8];
    mx_load8(p.dy, XT, row * p.OUT, c, p.OUT, vec, v);
#pragma unroll
    for (int pl = 0; pl < P; ++pl) {
        u32x4 o;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t lo = mx_plane_next(v[2 * u]);
            o[u] = lo | (uint32_t(mx_plane_next(v[2 * u + 1])) << 16);
        }
        *reinterpret_cast<u32x4 *>(p.out + (row * P + pl) * p.KO + c) = o;
    }
}

struct DxPlan {
    int64_t KO, P;
    bool direct;
    size_t dy, wt, part, total;               // offsets of the three areas
    GemmPlan gemm;
};
constexpr size_t kDxPartRoom = size_t(64) << 20;      // split-K partials that the GEMM may use
static DxPlan dx_plan(const MxGeom &g, const void *dy, int32_t type, int64_t N) {
    DxPlan d;
    d.KO = (g.OUT + 63) / 64 * 64;
    d.P = mx_planes(type);
    // sized without a pointer: dy is staged unless it can be read in place whatever its address
    d.direct = type == VQK_BF16 && g.OUT % 64 == 0 && dy && (reinterpret_cast<uintptr_t>(dy) & 15) == 0;
    d.gemm = plan_gemm(N, g.IN, d.P * d.KO, kDxPartRoom);
    d.dy = 0;
    d.wt = al256(size_t(N) * d.P * d.KO * 2);
    d.part = d.wt + al256(size_t(g.IN) * d.P * d.KO * 2);
    d.total = d.part + al256(d.gemm.part_bytes);
    return d;
}

static int check_lin(const vqk_mx_weights *w, int32_t x_type, int64_t N, MxGeom *g, const char *what) {
    const int rc = make_mx_geom(w, g, what);
    if (rc) return rc;
    if (g->E != 1) return set_error(VQK_EINVAL, "%s: E=%lld, a linear is one expert", what, (long long)g->E);
    if (!act_size(x_type)) return set_error(VQK_EINVAL, "%s: x type %d", what, x_type);
    if (N < 0 || N > INT32_MAX / 2) return set_error(VQK_EINVAL, "%s: N=%lld", what, (long long)N);
    return VQK_OK;
}

// Rows up to which the weights are streamed past all rows (vqk_mxs.h), where x
// fits its registers; more run as tiles.
constexpr int64_t kMxStreamRows = 32;
// Rows from which x that is quantised runs on the 4-bit matrix instructions;
// fewer enter as the values they are rounded to.
constexpr int64_t kMxfMinRows = 65;

// Workspace: x's planes, then the K slices of the many-row product.
static size_t lin_x_bytes(const MxGeom &g, int32_t x_type, int64_t N, int32_t act) {
    const int P = act == VQK_MX_ACT_MXFP4 ? 1 : mx_planes(x_type);
    return al256(size_t(N) * g.NB * kMxBlock * 2 * P);
}
// 4-bit x: rows of whole groups of four chunks.
static int64_t mxf_blocks(const MxGeom &g) { return (g.NB + 15) / 16 * 16; }
static size_t mxf_x_bytes(const MxGeom &g, int64_t N) { return al256(size_t(N) * mxf_blocks(g) * 17); }
static bool lin_4bit(int64_t N, int32_t act) { return act == VQK_MX_ACT_MXFP4 && N >= kMxfMinRows; }
static size_t lin_bytes(const MxGeom &g, int32_t x_type, int64_t N, int32_t act) {
    if (lin_4bit(N, act)) return mxf_x_bytes(g, N) + mxf_part_bytes(N, g);
    return lin_x_bytes(g, x_type, N, act) + mxg_part_bytes(N, g);
}

}  // namespace vqk

using namespace vqk;

static int check_act(int32_t act) {
    return act == VQK_MX_ACT_NONE || act == VQK_MX_ACT_MXFP4
               ? VQK_OK : set_error(VQK_EINVAL, "mx linear: activation form %d", act);
}

extern "C" int vqk_mx_linear_workspace(const vqk_mx_weights *w, int32_t x_type, int64_t N, int32_t act,
                                       size_t *bytes) {
    MxGeom g;
    int rc = check_lin(w, x_type, N, &g, "mx linear");
    if (rc || (rc = check_act(act))) return rc;
    if (!bytes) return set_error(VQK_EINVAL, "mx linear: NULL bytes");
    *bytes = lin_bytes(g, x_type, N, act);
    return VQK_OK;
}

extern "C" int vqk_mx_linear(const vqk_mx_weights *w, const void *x, int32_t x_type, int64_t N, int32_t act,
                             void *y, int32_t y_type, void *workspace, size_t ws_bytes, void *stream) {
    MxGeom g;
    int rc = check_lin(w, x_type, N, &g, "mx linear");
    if (rc || (rc = check_act(act))) return rc;
    if (!out_size(y_type)) return set_error(VQK_EINVAL, "mx linear: y type %d", y_type);
    if (N == 0) return VQK_OK;
    if (!x || !y) return set_error(VQK_EINVAL, "mx linear: NULL pointer");
    hipStream_t st = static_cast<hipStream_t>(stream);
    MxCall c{};
    c.codes[0] = w->codes; c.scales[0] = w->scales;
    c.g = g;
    c.N = N; c.xkrep = 1;
    c.y = y; c.y_type = y_type; c.ldy = g.OUT;
    const bool place = act == VQK_MX_ACT_NONE && mx_x_in_place(w, x, x_type);
    c.x.P = place || act == VQK_MX_ACT_MXFP4 ? 1 : mx_planes(x_type);
    c.x.op = place && x_type == VQK_F16 ? kOpF16 : kOpBF16;
    const int nt = N <= 16 ? 1 : 2;
    const bool stream_w = N <= kMxStreamRows && mx_rows_ok(c, nt);
    const size_t need = lin_bytes(g, x_type, N, act);
    if (!(place && stream_w) && need && (!workspace || ws_bytes < need))
        return set_error(VQK_ENOSPACE, "mx linear: workspace %zu < %zu", ws_bytes, need);
    if (reinterpret_cast<uintptr_t>(workspace) & 255)
        return set_error(VQK_EINVAL, "mx linear: workspace must be 256-byte aligned");
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    if (lin_4bit(N, act)) {
        const int64_t xNB = mxf_blocks(g);
        uint8_t *xsc = ws + size_t(N) * xNB * 16;
        if ((rc = launch_mx_quant(x, x_type, N, g.IN, g.IN, xNB, true, ws, xsc, st))) return rc;
        const size_t xb = mxf_x_bytes(g, N);
        const MxfCall f{w->codes, w->scales, g, N, xNB, ws, xsc, y, y_type};
        return mxf_gemm(f, need > xb ? reinterpret_cast<float *>(ws + xb) : nullptr, need - xb, st);
    }
    if (place) {
        c.x = MxX{static_cast<const uint16_t *>(x), g.IN, 0, 1, c.x.op};
    } else {
        uint16_t *xs = reinterpret_cast<uint16_t *>(ws);
        if ((rc = launch_mx_planes(x, x_type, N, g.IN, g.IN, act == VQK_MX_ACT_MXFP4, xs, st))) return rc;
        c.x = MxX{xs, g.NB * kMxBlock, N * g.NB * kMxBlock, c.x.P, kOpBF16};
    }
    if (stream_w) return mx_rows(c, nt, st);
    const size_t xb = lin_x_bytes(g, x_type, N, act);
    return mx_gemm(c, mxg_dense_rows(N), need > xb ? reinterpret_cast<float *>(ws + xb) : nullptr, need - xb, st);
}

extern "C" int vqk_mx_linear_dx_workspace(const vqk_mx_weights *w, int32_t type, int64_t N, size_t *bytes) {
    MxGeom g;
    const int rc = check_lin(w, type, N, &g, "mx linear dx");
    if (rc) return rc;
    if (!bytes) return set_error(VQK_EINVAL, "mx linear dx: NULL bytes");
    *bytes = N == 0 ? 0 : dx_plan(g, nullptr, type, N).total;
    return VQK_OK;
}

extern "C" int vqk_mx_linear_dx(const vqk_mx_weights *w, const void *dy, int32_t type, int64_t N, void *dx,
                                int32_t dx_type, void *workspace, size_t ws_bytes, void *stream) {
    MxGeom g;
    int rc = check_lin(w, type, N, &g, "mx linear dx");
    if (rc) return rc;
    if (!out_size(dx_type)) return set_error(VQK_EINVAL, "mx linear dx: dx type %d", dx_type);
    if (N == 0) return VQK_OK;
    if (!dy || !dx) return set_error(VQK_EINVAL, "mx linear dx: NULL pointer");
    const DxPlan d = dx_plan(g, dy, type, N);
    if (!workspace || ws_bytes < d.total)
        return set_error(VQK_ENOSPACE, "mx linear dx: workspace %zu < %zu", ws_bytes, d.total);
    if (reinterpret_cast<uintptr_t>(workspace) & 255)
        return set_error(VQK_EINVAL, "mx linear dx: workspace must be 256-byte aligned");
    hipStream_t st = static_cast<hipStream_t>(stream);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    const uint16_t *A = static_cast<const uint16_t *>(dy);
    if (!d.direct) {
        uint16_t *out = reinterpret_cast<uint16_t *>(ws + d.dy);
        const DyArgs a{dy, N, g.OUT, d.KO, out};
        const int64_t wgs = (N * (d.KO / 8) + 255) / 256;
        if (wgs > INT32_MAX) return set_error(VQK_ENOTIMPL, "mx linear dx: dy too large");
        const bool vec = (reinterpret_cast<uintptr_t>(dy) & 15) == 0 && (g.OUT * act_size(type)) % 16 == 0;
        const dim3 grid{unsigned(wgs)};
        switch (type) {
            case VQK_F16: hipLaunchKernelGGL((k_mx_dy<VQK_F16>), grid, dim3(256), 0, st, a, vec); break;
            case VQK_BF16: hipLaunchKernelGGL((k_mx_dy<VQK_BF16>), grid, dim3(256), 0, st, a, vec); break;
            default: hipLaunchKernelGGL((k_mx_dy<VQK_F32>), grid, dim3(256), 0, st, a, vec);
        }
        if ((rc = hip_status(hipGetLastError(), "dy staging launch"))) return rc;
        A = out;
    }
    uint16_t *wt = reinterpret_cast<uint16_t *>(ws + d.wt);
    const DecTArgs t{w->codes, w->scales, g.IN, g.RT, g.NC, d.KO, int32_t(d.P), wt};
    const int64_t gy = g.NC;
    if (gy > 65535) return set_error(VQK_ENOTIMPL, "mx linear dx: IN=%lld", (long long)g.IN);
    hipLaunchKernelGGL(k_mx_dec_t, dim3(unsigned(d.KO / 64), unsigned(gy)), dim3(256), 0, st, t);
    if ((rc = hip_status(hipGetLastError(), "transposed decode launch"))) return rc;
    return launch_hgemm(kOpBF16, d.gemm, A, wt, dx, dx_type, g.IN, 0, N, g.IN, d.P * d.KO,
                        d.gemm.part_bytes ? reinterpret_cast<float *>(ws + d.part) : nullptr, st);
}
