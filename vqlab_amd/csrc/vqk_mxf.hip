// Launch of the 4-bit by 4-bit products (kernel in vqk_mxf.h).
#include "vqk_mxf.h"

namespace vqk {

constexpr int kMxfRows = 128;

bool mxf_ok(const uint8_t *scales, int64_t IN, int64_t N) {
    // a lane's four blocks of a chunk share one aligned load of scales
    return IN % 128 == 0 && (reinterpret_cast<uintptr_t>(scales) & 3) == 0 && N > 0;
}

static int64_t mxf_tiles(int64_t N, int64_t OUT) {
    return ((N + kMxfRows - 1) / kMxfRows) * ((OUT + 255) / 256);
}

size_t mxf_part_bytes(int64_t N, int64_t OUT, int64_t NB) {
    const int s = mxg_splits(mxf_tiles(N, OUT), (NB + 7) / 8);
    return s > 1 ? size_t(s) * N * OUT * 4 : 0;
}

int mxf_gemm(const MxfCall &c, float *part, size_t part_bytes, hipStream_t st) {
    MxfArgs a{};
    a.codes = c.codes; a.scales = c.scales; a.xcodes = c.xcodes; a.xscales = c.xscales;
    a.OUT = c.OUT; a.NB = c.NB; a.N = c.N; a.xNB = c.xNB;
    a.y = c.y; a.y_type = c.y_type;
    a.NC = int32_t((c.NB + 7) / 8);
    a.nt = int32_t((c.N + kMxfRows - 1) / kMxfRows);
    a.nob = int32_t((c.OUT + 255) / 256);
    a.splits = 1;
    a.per = a.NC;
    const int s = mxg_splits(mxf_tiles(c.N, c.OUT), a.NC);
    if (s > 1 && part && size_t(s) * c.N * c.OUT * 4 <= part_bytes) {
        a.per = (a.NC + s - 1) / s;
        a.splits = (a.NC + a.per - 1) / a.per;
        a.part = part;
    }
    const int64_t grid = int64_t(a.nt) * a.nob * a.splits;
    if (grid > INT32_MAX) return set_error(VQK_ENOTIMPL, "4-bit product: grid too large");
    const int rc = launch_with_lds<k_mxf_gemm<kMxfRows / 32, 2>>(dim3(unsigned(grid)), dim3(256),
                                                                size_t(2) * kMxfRows * 128, st, a);
    if (rc || a.splits == 1) return rc;
    return launch_mx_reduce(a.part, a.splits, c.N * c.OUT, c.y, c.y_type, st);
}

}  // namespace vqk
