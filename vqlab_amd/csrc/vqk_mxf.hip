// Launch of the 4-bit by 4-bit products (kernel in vqk_mxf.h).
#include "vqk_mxf.h"

namespace vqk {

constexpr int kMxfRows = 128;

static int64_t mxf_tiles(int64_t N, int64_t OUT) {
    return ((N + kMxfRows - 1) / kMxfRows) * ((OUT + 255) / 256);
}

// In groups of four chunks: 3.6 us with one workgroup on a CU, 6.1 with two.
static int splits_of(int64_t N, const MxGeom &g) {
    return mx_splits(mxf_tiles(N, g.OUT), (g.NC + 3) / 4, N * g.OUT, 3.6f, 6.1f);
}

size_t mxf_part_bytes(int64_t N, const MxGeom &g) {
    const int s = splits_of(N, g);
    return s > 1 ? size_t(s) * N * g.OUT * 4 : 0;
}

int mxf_gemm(const MxfCall &c, float *part, size_t part_bytes, hipStream_t st) {
    MxfArgs a{};
    a.codes = c.codes; a.scales = c.scales; a.xcodes = c.xcodes; a.xscales = c.xscales;
    a.OUT = c.g.OUT; a.N = c.N; a.xNB = c.xNB;
    a.y = c.y; a.y_type = c.y_type;
    a.RT = int32_t(c.g.RT); a.NC = int32_t(c.g.NC);
    a.nt = int32_t((c.N + kMxfRows - 1) / kMxfRows);
    a.nob = int32_t((c.g.OUT + 255) / 256);
    const int groups = (a.NC + 3) / 4;
    a.splits = 1;
    a.per = groups;
    const int s = splits_of(c.N, c.g);
    if (s > 1 && part && size_t(s) * c.N * c.g.OUT * 4 <= part_bytes) {
        a.per = (groups + s - 1) / s;
        a.splits = (groups + a.per - 1) / a.per;
        a.part = part;
    }
    if (c.xNB * 16 * kMxfRows > INT64_C(0xffffffff))      // offsets inside a tile of x are 32 bits
        return set_error(VQK_ENOTIMPL, "4-bit product: rows of %lld blocks", (long long)c.xNB);
    const int64_t grid = int64_t(a.nt) * a.nob * a.splits;
    if (grid > INT32_MAX) return set_error(VQK_ENOTIMPL, "4-bit product: grid too large");
    const int rc = launch_with_lds<k_mxf_gemm<kMxfRows / 32, 2>>(dim3(unsigned(grid)), dim3(256),
                                                                size_t(2) * kMxfRows * 128, st, a);
    if (rc || a.splits == 1) return rc;
    return launch_mx_reduce(a.part, a.splits, c.N * c.g.OUT, c.y, c.y_type, st);
}

}  // namespace vqk
