// Launch of the many-row MXFP4 products (kernel in vqk_mxg.h).
#include "vqk_mxg.h"

namespace vqk {

struct MxRedArgs {
    const float *part;
    int64_t n, plane;                         // outputs; floats between slices
    int32_t splits, y_type;
    void *y;
};

// Sum of the K slices in slice order, four outputs a thread.
__global__ void __launch_bounds__(256) k_mx_reduce(const MxRedArgs p) {
    const int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4;
    if (i >= p.n) return;
    float v[4] = {};
    const int n = int(min(int64_t(4), p.n - i));
    const bool al = (p.plane & 3) == 0;
    for (int s = 0; s < p.splits; ++s) {
        const float *src = p.part + s * p.plane + i;
        if (al && n == 4) {
            const float4 q = *reinterpret_cast<const float4 *>(src);
            v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
        } else {
            for (int u = 0; u < n; ++u) v[u] += src[u];
        }
    }
    mx_store4(p.y, p.y_type, i, v, n, (reinterpret_cast<uintptr_t>(p.y) & 15) == 0);
}

int launch_mx_reduce(const float *part, int splits, int64_t n, void *y, int32_t y_type, hipStream_t st) {
    const MxRedArgs r{part, n, n, splits, y_type, y};
    const int64_t wgs = (n + 1023) / 1024;
    if (wgs > INT32_MAX) return set_error(VQK_ENOTIMPL, "MXFP4 product: too many outputs");
    hipLaunchKernelGGL(k_mx_reduce, dim3(unsigned(wgs)), dim3(256), 0, st, r);
    return hip_status(hipGetLastError(), "slice sum launch");
}

// K slices of a dense product of T tiles over NC chunks with n outputs, by an
// estimate of its time in us. One workgroup on a CU takes a chunk in t1, two
// together in t2 (128-row tiles: 2.2 and 3.6); slices are written and read as
// fp32 at ~4.5 TB/s and cost one more launch.
int mx_splits(int64_t T, int64_t NC, int64_t n, float t1, float t2) {
    int best = 1;
    float cost = -1.f;
    for (int s = 1; s <= 16 && (s == 1 || NC / s >= 4); ++s) {
        const int64_t wgs = T * s, per = (NC + s - 1) / s;
        const int64_t rounds = wgs / 512, rest = wgs % 512;
        float c = float(per) * (float(rounds) * t2 + (rest == 0 ? 0.f : (rest <= 256 ? t1 : t2)));
        if (s > 1) c += 3.f + float(s) * float(n) * 8.f / 4.5e6f;
        if (cost < 0.f || c < cost * 0.97f) {
            best = s;
            cost = c;
        }
    }
    return best;
}

static int dense_splits(int64_t N, const MxGeom &g) {
    const int rows = mxg_dense_rows(N);
    const float f = rows == 128 ? 1.f : (rows == 64 ? 0.7f : 0.55f);
    return mx_splits(((N + rows - 1) / rows) * ((g.OUT + kMxgRows - 1) / kMxgRows), g.NC, N * g.OUT, 2.2f * f,
                     3.6f * f);
}

int mxg_dense_rows(int64_t N) { return N <= 32 ? 32 : (N <= 64 ? 64 : 128); }

size_t mxg_part_bytes(int64_t N, const MxGeom &g) {
    const int s = dense_splits(N, g);
    return s > 1 ? size_t(s) * N * g.OUT * 4 : 0;
}

template <int OP, int BT, int ST, bool GLU, int P>
static int go(MxgArgs ga, int64_t tiles, hipStream_t st) {
    MxsArgs &a = ga.a;
    a.nob = int32_t((a.ocover + (GLU ? kMxgRows / 2 : kMxgRows) - 1) / (GLU ? kMxgRows / 2 : kMxgRows));
    const int64_t grid = int64_t(a.nob) * tiles * ga.splits;
    if (grid > INT32_MAX) return set_error(VQK_ENOTIMPL, "MXFP4 product: grid too large");
    ga.ntiles_host = int32_t(tiles);
    int rc = launch_with_lds<k_mx_gemm<OP, BT, ST, GLU, P>>(dim3(unsigned(grid)), dim3(64 * kMxgWaves),
                                                       size_t(ST) * 32 * BT * 256, st, ga);
    if (rc || ga.splits == 1) return rc;
    return launch_mx_reduce(ga.part, ga.splits, a.N * a.OUT, a.y, a.y_type, st);
}

template <int BT, int ST, bool GLU>
static int go_op(const MxgArgs &a, int op, int planes, int64_t tiles, hipStream_t st) {
    if (op == kOpF16) return go<kOpF16, BT, ST, GLU, 1>(a, tiles, st);
    if (planes == 1) return go<kOpBF16, BT, ST, GLU, 1>(a, tiles, st);
    return planes == 2 ? go<kOpBF16, BT, ST, GLU, 2>(a, tiles, st) : go<kOpBF16, BT, ST, GLU, 3>(a, tiles, st);
}
template <bool GLU>
static int go_bt(const MxgArgs &a, int op, int planes, int tile_rows, int64_t tiles, hipStream_t st) {
    // three stages where registers and LDS leave two workgroups a CU
    if (tile_rows <= 32) return go_op<1, 3, GLU>(a, op, planes, tiles, st);
    if (tile_rows <= 64) return go_op<2, 3, GLU>(a, op, planes, tiles, st);
    return go_op<4, 2, GLU>(a, op, planes, tiles, st);
}

// tile_rows: x rows per tile (32, 64 or 128; the sort's for a sorted routing).
int mx_gemm(const MxCall &c, int tile_rows, float *part, size_t part_bytes, hipStream_t st) {
    const bool glu = c.codes[1] != nullptr;
    MxgArgs ga{};
    mx_args(c, &ga.a);
    const int64_t tiles = mx_tiles(c, tile_rows);
    if (tiles == 0) return VQK_OK;
    ga.splits = 1;
    ga.per = ga.a.NC;
    if (part && !c.meta && !c.ids && !glu) {
        const int s = dense_splits(c.N, c.g);
        if (s > 1 && size_t(s) * c.N * c.g.OUT * 4 <= part_bytes) {
            ga.per = int32_t((ga.a.NC + s - 1) / s);
            ga.splits = int32_t((ga.a.NC + ga.per - 1) / ga.per);
            ga.part = part;
        }
    }
    return glu ? go_bt<true>(ga, c.x.op, c.x.P, tile_rows, tiles, st)
               : go_bt<false>(ga, c.x.op, c.x.P, tile_rows, tiles, st);
}

}  // namespace vqk
