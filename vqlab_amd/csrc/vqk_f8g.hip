// Launch of the many-row products of 8-bit weights with 16-bit x (kernel in vqk_f8g.h).
#include "vqk_f8g.h"

namespace vqk {

static int gemm_rows(int64_t N) { return N <= 32 ? 32 : (N <= 64 ? 64 : 96); }

// One workgroup on a CU takes a block of 128 k in 2.2 us, two together in 3.2.
static int gemm_splits(int64_t N, const F8Geom &g, int P) {
    const int rows = gemm_rows(N);
    const float f = (rows == 96 ? 1.f : (rows == 64 ? 0.75f : 0.6f)) * float(P);
    return mx_splits(((N + rows - 1) / rows) * ((g.OUT + kF8gRows - 1) / kF8gRows), g.NC, N * g.OUT, 2.2f * f, 3.2f * f);
}

size_t f8_gemm_part(int64_t N, const F8Geom &g, int P) {
    const int s = gemm_splits(N, g, P);
    return s > 1 ? size_t(s) * N * g.OUT * 4 : 0;
}

template <int OP, int BT, bool SX>
static int go(const F8gArgs &a, hipStream_t st) {
    const int64_t grid = int64_t(a.nt) * ((a.OUT + kF8gRows - 1) / kF8gRows) * a.splits;
    if (grid > INT32_MAX) return set_error(VQK_ENOTIMPL, "8-bit product: grid too large");
    const int rc = launch_with_lds<k_f8_gemm<OP, BT, SX>>(dim3(unsigned(grid)), dim3(64 * kF8gWaves), size_t(2) * 32 * BT * 256, st, a);
    if (rc || a.splits == 1) return rc;
    return launch_mx_reduce(a.part, a.splits, a.N * a.OUT, a.y, a.y_type, st);
}
template <int OP, bool SX>
static int go_bt(const F8gArgs &a, int rows, hipStream_t st) {
    if (rows == 32) return go<OP, 1, SX>(a, st);
    return rows == 64 ? go<OP, 2, SX>(a, st) : go<OP, 3, SX>(a, st);
}

int f8_gemm(const F8Call &c, float *part, size_t part_bytes, hipStream_t st) {
    F8gArgs a{};
    a.codes = c.codes; a.scales = c.scales; a.swo = c.swo; a.swk = c.swk;
    a.OUT = c.g.OUT; a.IN = c.g.IN; a.N = c.N;
    a.RT = int32_t(c.g.RT); a.NC = int32_t(c.g.NC); a.P = c.x.P;
    a.x = c.x.x; a.xld = c.x.ld; a.xplane = c.x.plane;
    a.y = c.y; a.y_type = c.y_type;
    const int rows = gemm_rows(c.N);
    a.nt = int32_t((c.N + rows - 1) / rows);
    a.splits = 1;
    a.per = a.NC;
    const int s = gemm_splits(c.N, c.g, c.x.P);
    if (s > 1 && part && size_t(s) * c.N * c.g.OUT * 4 <= part_bytes) {
        a.per = (a.NC + s - 1) / s;
        a.splits = (a.NC + a.per - 1) / a.per;
        a.part = part;
    }
    a.sx = c.x8.scales; a.sn = c.x8.sn; a.sk = c.x8.sk;
    if (a.sx) return go_bt<kOpBF16, true>(a, rows, st);
    return c.x.op == kOpF16 ? go_bt<kOpF16, false>(a, rows, st) : go_bt<kOpBF16, false>(a, rows, st);
}

}  // namespace vqk
