// Routed experts with MXFP4 weights: one projection for (token, expert) pairs,
// and the whole block of experts,
//     y_t = sum_j w_tj * down_e( silu(gate_e x_t) * (up_e x_t) ),  e = ids_tj.
//
// Few pairs run pair by pair; more are sorted by expert on the device, so that
// an expert's weights are read once for a tile of its rows. Gate and up are one
// launch whose epilogue leaves silu(g) * u as the bf16 planes that down reads
// (mx_h_planes); down leaves fp32 rows by pair, and the last kernel adds them in
// order of j.
#include "vqk_mxs.h"

namespace vqk {

static size_t al256(size_t v) { return (v + 255) & ~size_t(255); }

// Whether a routing runs pair by pair: the sort, its tiles and the pass that adds
// rows cost about 20 us more, and read weights at 5.3 TB/s instead of 3.6 and an
// expert's once. us per block, pair by pair / sorted: 256 experts of 2048 x 512
// (1.7 MB a pair), 64 pairs 36 / 52, 128 56 / 67; 512 of 4096 x 1024 (6.7 MB), 30
// pairs 57 / 70, 60 117 / 112; 64 of 4096 x 1024, 24 pairs 55 / 62, 48 87 / 82; 8 of
// 2048 x 1024, 16 pairs 21 / 42, 24 34 / 42.
static bool mx_by_pair(int64_t N, int64_t E, int64_t pair_bytes) {
    return N <= 16 || (N <= 2 * E && N * pair_bytes <= INT64_C(256) << 20);
}
static int64_t pair_bytes(const MxGeom &g) { return mx_expert_codes(g.RT, g.NC); }
constexpr int64_t kMxMaxExperts = 4096;

// Rows per tile of a sorted routing of N pairs over E experts. Tiles cost the rows
// they hold (in groups of 32), so a tile is as large as what an expert is likely to
// have. us per block in tiles of 32 / 64 / 128: 256 experts of 2048 x 512, 12 rows an
// expert 147 / 154 / 153, 20 162 / 156 / 158, 30 181 / 188 / 185, 40 227 / 215 / 207, 60
// 278 / 267 / 261; 64 of 4096 x 1024, 12 136 / 139 / 136, 30 159 / 160 / 156, 60 234 / 248 /
// 219; 512 of 4096 x 1024, 1.25 rows 497 / 545 / 549.
static int mx_tile_rows(int64_t N, int64_t E) {
    const int64_t avg = N / E;
    return avg <= 20 ? 32 : (avg <= 40 ? 64 : 128);
}
// One product: pairs stream the weights where x fits (vqk_mxs.h), tiles else.
static int run(const MxCall &c, int rows, hipStream_t st) {
    return c.ids && mx_rows_ok(c, 1) ? mx_rows(c, 1, st) : mx_gemm(c, rows, nullptr, 0, st);
}

// The SwiGLU rows that down reads, as bf16 planes: three (24 bits) for fp32 x, two
// (16 bits, bf16's range) for 16-bit x, however many pairs share the call. They are
// nobody's output: rounded to x's type as well, they would put an error as large as
// the outputs' own rounding under it (against 64 bits 0.0026 instead of 0.0017 for
// bf16), and fp16 rows end at 65504. The second plane is a second product in down: a
// block of 64 tokens through 512 experts 466 us instead of 459, of 2048 through 256
// 270 instead of 246.
constexpr int mx_h_planes(int32_t x_type) { return x_type == VQK_F32 ? 3 : 2; }

struct CombineArgs {
    const float *part;
    const int32_t *ids;
    const float *wts;
    int64_t T, H, E;
    int32_t k;
    void *y;
    int32_t y_type;
};

// y_t = sum_j w_tj part[t k + j]; pairs without an expert are not read.
__global__ void __launch_bounds__(256) k_mx_combine(const CombineArgs p) {
    const int64_t t = blockIdx.y;
    const int64_t h = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4;
    if (h >= p.H) return;
    float v[4] = {};
    const bool vec = p.H % 4 == 0;
    for (int j = 0; j < p.k; ++j) {
        const int64_t pair = t * p.k + j;
        const int64_t e = p.ids[pair];
        if (e < 0 || e >= p.E) continue;
        const float w = p.wts[pair];
        const float *src = p.part + pair * p.H + h;
        if (vec) {
            const float4 q = *reinterpret_cast<const float4 *>(src);
            v[0] += w * q.x; v[1] += w * q.y; v[2] += w * q.z; v[3] += w * q.w;
        } else {
            for (int u = 0; u < 4 && h + u < p.H; ++u) v[u] += w * src[u];
        }
    }
    for (int u = 0; u < 4 && h + u < p.H; ++u) store_act(p.y, p.y_type, t * p.H + h + u, v[u]);
}

struct DownArgs {
    const uint8_t *codes, *scales;
    int64_t E, OUT;
    int32_t RT, NC, NB, k;
    const uint16_t *h;                        // SwiGLU rows by pair
    int64_t hld, hplane;
    const int32_t *ids;
    const float *wts;
    void *y;
    int32_t y_type;
};

// Down and the weighted sum for few pairs: a workgroup takes 16 weight rows of
// every expert of one token, its waves share the (expert, chunk) units. A wave's
// matrix instructions see the pair's row in all 16 x rows (one line a load) and
// leave the sums of a unit, which enter with the pair's weight; the waves meet in
// LDS in wave order. Against down rows in fp32 and a pass that adds them: one launch
// and one round trip less (8 pairs of 512 -> 2048: 4.4 us for 4.2 + 4.5).
template <int P>
__global__ void __launch_bounds__(64 * kMxsWaves) k_mx_down(const DownArgs p) {
    __shared__ float red[kMxsWaves][16];
    constexpr int U = 2;                      // units in flight (four: 100 us for 89 with 40 pairs of 512 experts)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const int t = int(blockIdx.x / unsigned(p.RT)), rt = int(blockIdx.x % unsigned(p.RT));
    const uint32_t NC = uint32_t(p.NC), NC4 = (NC + 3) / 4;
    float acc = 0.f;
    bool nan = false;
    const int units = p.k * p.NC;
    for (int u0 = wave; u0 < units; u0 += U * kMxsWaves) {
        u32x4 w[U], x[U][P][4];
        uint32_t sc[U];
        float wt[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = min(u0 + i * kMxsWaves, units - 1), j = u / p.NC;
            const uint32_t c = uint32_t(u - j * p.NC);
            const int pair = t * p.k + j, e = p.ids[pair];
            const bool on = u0 + i * kMxsWaves < units && e >= 0 && e < p.E;
            const int64_t ex = on ? e : 0;
            wt[i] = on ? p.wts[pair] : 0.f;
            w[i] = *reinterpret_cast<const u32x4 *>(p.codes + ex * mx_expert_codes(p.RT, p.NC) +
                                                    ((uint32_t(rt) * NC + c) * 64 + lane) * 16u);
            sc[i] = p.scales[ex * mx_expert_scales(p.RT, p.NC) + ((uint32_t(rt) * NC4 + c / 4) * 64 + lane) * 4 + c % 4];
            const int blk = int(4 * c) + g;
            const bool in = on && blk < p.NB;
            const uint16_t *xp = p.h + int64_t(pair) * p.hld + (in ? blk : 0) * kMxBlock;
#pragma unroll
            for (int pl = 0; pl < P; ++pl)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const u32x4 v = *reinterpret_cast<const u32x4 *>(xp + pl * p.hplane + 8 * k);
                    x[i][pl][k] = in ? v : u32x4{};
                }
            if (!on) sc[i] = 127u;
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            nan = nan || sc[i] == 255u;
            const float s = mx_scale(sc[i] == 255u ? 127u : sc[i]);
            f32x4 d{};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const u32x4 wf = mx_decode8(w[i][k], s);
#pragma unroll
                for (int pl = 0; pl < P; ++pl) d = mx_mma16<kOpBF16>(x[i][pl][k], wf, d);
            }
            acc += wt[i] * d[0];              // a pair without an expert: 0 times rows of zeros
        }
    }
    int f = nan;
    f |= __shfl_xor(f, 16);
    f |= __shfl_xor(f, 32);
    if (lane < 16) red[wave][lane] = f ? __uint_as_float(0x7fc00000u) : acc;
    __syncthreads();
    const int64_t o = int64_t(rt) * 16 + threadIdx.x;
    if (threadIdx.x < 16 && o < p.OUT) {
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < kMxsWaves; ++i) v += red[i][threadIdx.x];
        store_act(p.y, p.y_type, t * p.OUT + o, v);
    }
}

static int check_pairs(int64_t T, int64_t N, int64_t E, const char *what) {
    if (T < 0 || N < 0 || N > INT32_MAX / 4) return set_error(VQK_EINVAL, "%s: T=%lld N=%lld", what, (long long)T, (long long)N);
    if (E > kMxMaxExperts) return set_error(VQK_ENOTIMPL, "%s: E=%lld > %lld", what, (long long)E, (long long)kMxMaxExperts);
    return VQK_OK;
}

// x rows in place, or laid out as planes at `ws` (bytes: plane_bytes).
static size_t plane_bytes(int64_t rows, int64_t NB, int P) { return al256(size_t(rows) * NB * kMxBlock * 2 * P); }
static int make_x(const vqk_mx_weights *w, bool place, const void *x, int32_t type, int64_t rows, int64_t NB,
                  uint16_t *ws, MxX *out, hipStream_t st) {
    if (place) {
        *out = MxX{static_cast<const uint16_t *>(x), w->IN, 0, 1, type == VQK_F16 ? kOpF16 : kOpBF16};
        return VQK_OK;
    }
    *out = MxX{ws, NB * kMxBlock, rows * NB * kMxBlock, mx_planes(type), kOpBF16};
    return launch_mx_planes(x, type, rows, w->IN, w->IN, false, ws, st);
}

static size_t sort_bytes(int64_t N, int64_t E, int64_t pb) {
    return mx_by_pair(N, E, pb) ? 0 : al256(seg_sort_bytes(N, E));
}
// Sets a call's routing from the ids: unsorted pairs, or sorted into `ws`.
static int set_routing(MxCall *c, bool by_pair, const int32_t *ids, int64_t N, int64_t E, int rows, void *ws,
                       hipStream_t st) {
    if (by_pair) {
        c->ids = ids;
        return VQK_OK;
    }
    const int rc = seg_sort(reinterpret_cast<const uint32_t *>(ids), N, E, rows, ws, st);
    const SegTiles t = seg_tiles(ws, N, E);
    c->order = t.order;
    c->meta = t.meta;
    c->ntiles = t.ntiles;
    return rc;
}

struct ExpertsPlan {
    int64_t N, IP;
    int P;
    bool by_pair;
    size_t x, h, part, sort, total;
};
static int plan_experts(const vqk_mx_weights *gate, const vqk_mx_weights *up, const vqk_mx_weights *down,
                        int32_t x_type, int64_t T, int32_t top_k, MxGeom *g1, MxGeom *g2, ExpertsPlan *p) {
    MxGeom gu;
    int rc;
    if ((rc = make_mx_geom(gate, g1, "mx experts: gate")) || (rc = make_mx_geom(up, &gu, "mx experts: up")) ||
        (rc = make_mx_geom(down, g2, "mx experts: down")))
        return rc;
    if (gu.E != g1->E || gu.OUT != g1->OUT || gu.IN != g1->IN || g2->E != g1->E || g2->IN != g1->OUT ||
        g2->OUT != g1->IN)
        return set_error(VQK_EINVAL, "mx experts: gate, up [E, I, H] and down [E, H, I] do not fit together");
    if (!act_size(x_type)) return set_error(VQK_EINVAL, "mx experts: x type %d", x_type);
    if (top_k < 1 || top_k > g1->E)
        return set_error(VQK_EINVAL, "mx experts: top_k=%d of %lld experts", top_k, (long long)g1->E);
    if (T < 0 || T > INT32_MAX / 4 / top_k) return set_error(VQK_EINVAL, "mx experts: T=%lld", (long long)T);
    p->N = T * top_k;
    if ((rc = check_pairs(T, p->N, g1->E, "mx experts"))) return rc;
    p->IP = g2->NB * kMxBlock;
    p->P = mx_planes(x_type);
    const int64_t pb = 2 * pair_bytes(*g1) + pair_bytes(*g2);
    p->by_pair = mx_by_pair(p->N, g1->E, pb);
    p->x = 0;
    p->h = plane_bytes(T, g1->NB, p->P);
    p->part = p->h + plane_bytes(p->N, g2->NB, mx_h_planes(x_type));
    p->sort = p->part + (p->by_pair ? 0 : al256(size_t(p->N) * g2->OUT * 4));
    p->total = p->sort + sort_bytes(p->N, g1->E, pb);
    return VQK_OK;
}

}  // namespace vqk

using namespace vqk;

extern "C" int vqk_mx_switch_workspace(const vqk_mx_weights *w, int32_t x_type, int64_t T, int64_t N,
                                       size_t *bytes) {
    MxGeom g;
    int rc = make_mx_geom(w, &g, "mx switch");
    if (rc || (rc = check_pairs(T, N, g.E, "mx switch"))) return rc;
    if (!act_size(x_type)) return set_error(VQK_EINVAL, "mx switch: x type %d", x_type);
    if (!bytes) return set_error(VQK_EINVAL, "mx switch: NULL bytes");
    *bytes = plane_bytes(T, g.NB, mx_planes(x_type)) + sort_bytes(N, g.E, 3 * pair_bytes(g));
    return VQK_OK;
}

extern "C" int vqk_mx_switch(const vqk_mx_weights *w, const void *x, int32_t x_type, int64_t T,
                             const int32_t *eidx, int64_t N, int64_t xkrep, void *y, int32_t y_type,
                             void *workspace, size_t ws_bytes, void *stream) {
    MxGeom g;
    int rc = make_mx_geom(w, &g, "mx switch");
    if (rc || (rc = check_pairs(T, N, g.E, "mx switch"))) return rc;
    if (!act_size(x_type)) return set_error(VQK_EINVAL, "mx switch: x type %d", x_type);
    if (!out_size(y_type)) return set_error(VQK_EINVAL, "mx switch: y type %d", y_type);
    if (xkrep < 1 || T > INT64_MAX / xkrep || N != T * xkrep)
        return set_error(VQK_EINVAL, "mx switch: N=%lld pairs for T=%lld rows x %lld", (long long)N,
                         (long long)T, (long long)xkrep);
    if (N == 0) return VQK_OK;
    if (!x || !eidx || !y) return set_error(VQK_EINVAL, "mx switch: NULL pointer");
    const size_t sort_at = plane_bytes(T, g.NB, mx_planes(x_type));
    const size_t need = sort_at + sort_bytes(N, g.E, 3 * pair_bytes(g));
    if (!workspace || ws_bytes < need)
        return set_error(VQK_ENOSPACE, "mx switch: workspace %zu < %zu", ws_bytes, need);
    if (reinterpret_cast<uintptr_t>(workspace) & 255)
        return set_error(VQK_EINVAL, "mx switch: workspace must be 256-byte aligned");
    hipStream_t st = static_cast<hipStream_t>(stream);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    MxCall c{};
    c.codes[0] = w->codes; c.scales[0] = w->scales;
    c.g = g;
    c.N = N; c.xkrep = xkrep;
    c.y = y; c.y_type = y_type; c.ldy = g.OUT;
    if ((rc = make_x(w, mx_x_in_place(w, x, x_type), x, x_type, T, g.NB, reinterpret_cast<uint16_t *>(ws),
                     &c.x, st))) return rc;
    const bool by_pair = mx_by_pair(N, g.E, 3 * pair_bytes(g));
    const int rows = mx_tile_rows(N, g.E);
    if ((rc = set_routing(&c, by_pair, eidx, N, g.E, rows, ws + sort_at, st))) return rc;
    return run(c, rows, st);
}

static int experts(const vqk_mx_weights *gate, const vqk_mx_weights *up, const vqk_mx_weights *down,
                   const MxGeom &g1, const MxGeom &g2, const ExpertsPlan &p, const void *x, int32_t x_type,
                   int64_t T, const int32_t *ids, const float *wts, int32_t top_k, void *y, int32_t y_type,
                   uint8_t *ws, hipStream_t st);

extern "C" int vqk_mx_experts_workspace(const vqk_mx_weights *gate, const vqk_mx_weights *up,
                                        const vqk_mx_weights *down, int32_t x_type, int64_t T,
                                        int32_t top_k, size_t *bytes) {
    MxGeom g1, g2;
    ExpertsPlan p;
    const int rc = plan_experts(gate, up, down, x_type, T, top_k, &g1, &g2, &p);
    if (rc) return rc;
    if (!bytes) return set_error(VQK_EINVAL, "mx experts: NULL bytes");
    *bytes = p.total;
    return VQK_OK;
}

extern "C" int vqk_mx_experts(const vqk_mx_weights *gate, const vqk_mx_weights *up,
                              const vqk_mx_weights *down, const void *x, int32_t x_type, int64_t T,
                              const int32_t *ids, const float *wts, int32_t top_k, void *y, int32_t y_type,
                              void *workspace, size_t ws_bytes, void *stream) {
    MxGeom g1, g2;
    ExpertsPlan p;
    int rc = plan_experts(gate, up, down, x_type, T, top_k, &g1, &g2, &p);
    if (rc) return rc;
    if (!out_size(y_type)) return set_error(VQK_EINVAL, "mx experts: y type %d", y_type);
    if (T == 0) return VQK_OK;
    if (!x || !ids || !wts || !y) return set_error(VQK_EINVAL, "mx experts: NULL pointer");
    if (!workspace || ws_bytes < p.total)
        return set_error(VQK_ENOSPACE, "mx experts: workspace %zu < %zu", ws_bytes, p.total);
    if (reinterpret_cast<uintptr_t>(workspace) & 255)
        return set_error(VQK_EINVAL, "mx experts: workspace must be 256-byte aligned");
    return experts(gate, up, down, g1, g2, p, x, x_type, T, ids, wts, top_k, y, y_type,
                   static_cast<uint8_t *>(workspace), static_cast<hipStream_t>(stream));
}

static int experts(const vqk_mx_weights *gate, const vqk_mx_weights *up, const vqk_mx_weights *down,
                   const MxGeom &g1, const MxGeom &g2, const ExpertsPlan &p, const void *x, int32_t x_type,
                   int64_t T, const int32_t *ids, const float *wts, int32_t top_k, void *y, int32_t y_type,
                   uint8_t *ws, hipStream_t st) {
    int rc;
    const int rows = mx_tile_rows(p.N, g1.E);
    MxCall c{};
    c.codes[0] = gate->codes; c.scales[0] = gate->scales;
    c.codes[1] = up->codes; c.scales[1] = up->scales;
    c.g = g1;
    c.N = p.N; c.xkrep = top_k;
    uint16_t *h = reinterpret_cast<uint16_t *>(ws + p.h);
    const bool place = mx_x_in_place(gate, x, x_type) && (x_type != VQK_F16 || up->f16_exact);
    if ((rc = make_x(gate, place, x, x_type, T, g1.NB, reinterpret_cast<uint16_t *>(ws), &c.x, st))) return rc;
    const int hp = mx_h_planes(x_type);
    c.y = h; c.ldy = p.IP; c.yplane = p.N * p.IP; c.yp = hp; c.ysorted = true;
    if ((rc = set_routing(&c, p.by_pair, ids, p.N, g1.E, rows, ws + p.sort, st))) return rc;
    if ((rc = run(c, rows, st))) return rc;
    MxCall d = c;                              // the same routing, over the SwiGLU rows
    d.codes[0] = down->codes; d.scales[0] = down->scales;
    d.codes[1] = nullptr; d.scales[1] = nullptr;
    d.g = g2;
    d.x = MxX{h, p.IP, p.N * p.IP, hp, kOpBF16};
    d.xkrep = 0;
    if (p.by_pair) {
        const DownArgs a{d.codes[0], d.scales[0], g2.E, g2.OUT, int32_t(g2.RT), int32_t(g2.NC), int32_t(g2.NB),
                         top_k, h, p.IP, p.N * p.IP, ids, wts, y, y_type};
        const int64_t grid = T * g2.RT;
        if (grid > INT32_MAX) return set_error(VQK_ENOTIMPL, "mx experts: grid too large");
        const dim3 gr{unsigned(grid)}, b(64 * kMxsWaves);
        if (hp == 2) hipLaunchKernelGGL((k_mx_down<2>), gr, b, 0, st, a);
        else hipLaunchKernelGGL((k_mx_down<3>), gr, b, 0, st, a);
        return hip_status(hipGetLastError(), "MXFP4 down launch");
    }
    float *part = reinterpret_cast<float *>(ws + p.part);
    d.y = part; d.y_type = VQK_F32; d.ldy = g2.OUT; d.ysorted = false;
    if ((rc = run(d, rows, st))) return rc;
    const CombineArgs a{part, ids, wts, T, g2.OUT, g1.E, top_k, y, y_type};
    for (int64_t t0 = 0; t0 < T; t0 += 65535) {          // grid.y holds 65535 tokens
        CombineArgs b = a;
        b.part += t0 * top_k * g2.OUT;
        b.ids += t0 * top_k;
        b.wts += t0 * top_k;
        b.y = static_cast<uint8_t *>(y) + t0 * g2.OUT * out_size(y_type);
        const int64_t n = T - t0 < 65535 ? T - t0 : 65535;
        hipLaunchKernelGGL(k_mx_combine, dim3(unsigned((g2.OUT + 1023) / 1024), unsigned(n)), dim3(256), 0, st, b);
        if ((rc = hip_status(hipGetLastError(), "combine launch"))) return rc;
    }
    return VQK_OK;
}

// The block of experts with its routing: ids and weights in the workspace.
static size_t ids_bytes(int64_t N) { return al256(size_t(N) * 4); }

extern "C" int vqk_mx_moe_workspace(const vqk_mx_weights *gate, const vqk_mx_weights *up,
                                    const vqk_mx_weights *down, int32_t x_type, int64_t T, int32_t top_k,
                                    size_t *bytes) {
    MxGeom g1, g2;
    ExpertsPlan p;
    const int rc = plan_experts(gate, up, down, x_type, T, top_k, &g1, &g2, &p);
    if (rc) return rc;
    if (!bytes) return set_error(VQK_EINVAL, "mx moe: NULL bytes");
    *bytes = p.total + 2 * ids_bytes(p.N);
    return VQK_OK;
}

extern "C" int vqk_mx_moe(const vqk_mx_weights *gate, const vqk_mx_weights *up, const vqk_mx_weights *down,
                          const void *x, int32_t x_type, int64_t T, const void *logits, int32_t l_type,
                          int64_t ld, const uint8_t *mask, int32_t top_k, int32_t norm_topk, void *y,
                          int32_t y_type, void *workspace, size_t ws_bytes, void *stream) {
    MxGeom g1, g2;
    ExpertsPlan p;
    int rc = plan_experts(gate, up, down, x_type, T, top_k, &g1, &g2, &p);
    if (rc) return rc;
    if (!out_size(y_type)) return set_error(VQK_EINVAL, "mx moe: y type %d", y_type);
    if (T == 0) return VQK_OK;
    if (!x || !logits || !y) return set_error(VQK_EINVAL, "mx moe: NULL pointer");
    const size_t need = p.total + 2 * ids_bytes(p.N);
    if (!workspace || ws_bytes < need) return set_error(VQK_ENOSPACE, "mx moe: workspace %zu < %zu", ws_bytes, need);
    if (reinterpret_cast<uintptr_t>(workspace) & 255)
        return set_error(VQK_EINVAL, "mx moe: workspace must be 256-byte aligned");
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    int32_t *ids = reinterpret_cast<int32_t *>(ws + p.total);
    float *wts = reinterpret_cast<float *>(ws + p.total + ids_bytes(p.N));
    rc = vqk_route(logits, l_type, T, g1.E, ld, mask, top_k, norm_topk, ids, wts, nullptr, nullptr, nullptr,
                   nullptr, 0, stream);
    if (rc) return rc;
    return experts(gate, up, down, g1, g2, p, x, x_type, T, ids, wts, top_k, y, y_type, ws,
                   static_cast<hipStream_t>(stream));
}
