// Launch of the products of 8-bit weights with many 8-bit rows (kernel in vqk_f8t.h).
#include "vqk_f8t.h"

namespace vqk {

static int tile_cols(int64_t N) { return N <= 64 ? 64 : (N <= 128 ? 128 : 256); }

// In blocks of 128 k: a workgroup alone on its CU (wider tiles leave room for no other).
static int tile_splits(int64_t N, const F8Geom &g) {
    const int bn = tile_cols(N);
    const int64_t T = ((N + bn - 1) / bn) * ((g.OUT + kF8tRows - 1) / kF8tRows);
    const float t = bn == 256 ? 1.6f : (bn == 128 ? 1.f : 0.8f);
    int best = 1;
    float cost = -1.f;
    for (int s = 1; s <= 16 && (s == 1 || g.NC / s >= 4); ++s) {
        const int64_t per = (g.NC + s - 1) / s, rounds = (T * s + 255) / 256;
        float c = float(per) * float(rounds) * t;
        if (s > 1) c += 3.f + float(s) * float(N) * float(g.OUT) * 8.f / 4.5e6f;
        if (cost < 0.f || c < cost * 0.97f) {
            best = s;
            cost = c;
        }
    }
    return best;
}

size_t f8_tiles_part(int64_t N, const F8Geom &g) {
    const int s = tile_splits(N, g);
    return s > 1 ? size_t(s) * N * g.OUT * 4 : 0;
}

template <int BN, int NST>
static int go(const F8tArgs &a, hipStream_t st) {
    const int64_t grid = int64_t(a.nt) * ((a.OUT + kF8tRows - 1) / kF8tRows) * a.splits;
    if (grid > INT32_MAX) return set_error(VQK_ENOTIMPL, "8-bit product: grid too large");
    const int rc = launch_with_lds<k_f8_tiles<BN, NST>>(dim3(unsigned(grid)), dim3(512),
                                                       size_t(NST) * ((kF8tRows + BN) * 64 + BN * 4), st, a);
    if (rc || a.splits == 1) return rc;
    return launch_mx_reduce(a.part, a.splits, a.N * a.OUT, a.y, a.y_type, st);
}

int f8_tiles(const F8Call &c, float *part, size_t part_bytes, hipStream_t st) {
    if (c.x8.ld * 256 > INT64_C(0xffffffff))              // offsets inside a tile of x are 32 bits
        return set_error(VQK_ENOTIMPL, "8-bit product: rows %lld apart", (long long)c.x8.ld);
    F8tArgs a{};
    a.codes = c.codes; a.scales = c.scales; a.swo = c.swo; a.swk = c.swk;
    a.OUT = c.g.OUT; a.N = c.N;
    a.RT = int32_t(c.g.RT); a.NC = int32_t(c.g.NC);
    a.x = c.x8.codes; a.xld = c.x8.ld;
    a.sx = c.x8.scales; a.sn = c.x8.sn; a.sk = c.x8.sk;
    a.y = c.y; a.y_type = c.y_type;
    const int bn = tile_cols(c.N);
    a.nt = int32_t((c.N + bn - 1) / bn);
    a.splits = 1;
    a.per = a.NC;
    const int s = tile_splits(c.N, c.g);
    if (s > 1 && part && size_t(s) * c.N * c.g.OUT * 4 <= part_bytes) {
        a.per = (a.NC + s - 1) / s;
        a.splits = (a.NC + a.per - 1) / a.per;
        a.part = part;
    }
    switch (bn) {
        case 64: return go<64, 4>(a, st);
        case 128: return go<128, 4>(a, st);
        default: return go<256, 4>(a, st);
    }
}

}  // namespace vqk
