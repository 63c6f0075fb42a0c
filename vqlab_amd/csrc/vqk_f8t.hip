// Launch of the products of 8-bit weights with many rows (kernels in vqk_f8t.h).
#include "vqk_f8t.h"

namespace vqk {

// Forms of x: 8-bit rows, 16-bit rows, and 8-bit codes as 16-bit values with scales.
enum { kX8, kX16, kX16S };
static int form_of(const F8Call &c) { return c.a8 ? kX8 : (c.x8.scales ? kX16S : kX16); }

// Time of a block of 128 k in us by the tile's x rows, one workgroup a CU (measured
// at 8192 -> 16384 and whole rounds).
struct TileTime { int bn; float us; };
constexpr TileTime kTiles8[] = {{256, 2.0f}, {192, 1.65f}, {128, 1.05f}, {64, 0.73f}};
constexpr TileTime kTiles16[] = {{192, 2.6f}, {128, 1.9f}, {64, 1.25f}};
struct TilePlan {
    int bn;
    int32_t tiles, full, splits, per;
    size_t part;
};

static int cus() {
    int n = 0, dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1) n = 256;
    return n;
}

// The tile and the cut of the last round of least estimated time: slices are written
// and read as fp32 at ~4.5 TB/s and cost one more launch.
static TilePlan tile_plan(int64_t N, const F8Geom &g, int form, int P) {
    const int C = cus();
    TilePlan best{};
    float cost = -1.f;
    const TileTime *k = form == kX8 ? kTiles8 : kTiles16;
    const int n = form == kX8 ? 4 : 3, steps = int(g.NC) * P;
    for (int i = form == kX16S ? 1 : 0; i < n; ++i) {
        const int bn = k[i].bn;
        const int64_t T = ((N + bn - 1) / bn) * ((g.OUT + kF8tRows - 1) / kF8tRows), rest = T % C;
        for (int s = 1; s <= 16 && (s == 1 || (rest && steps / s >= 4)); ++s) {
            const int per = (steps + s - 1) / s, slices = (steps + per - 1) / per;
            const int64_t cut = s == 1 ? 0 : rest, full = T - cut;
            float c = float((full + C - 1) / C) * float(steps) * k[i].us;
            if (cut)
                c += float((cut * slices + C - 1) / C) * float(per) * k[i].us + 3.f + float(cut * slices) * float(bn * kF8tRows) * 8.f / 4.5e6f;
            if (cost < 0.f || c < cost * 0.98f) {
                cost = c;
                best = TilePlan{bn, int32_t(T < INT32_MAX ? T : INT32_MAX), int32_t(full < INT32_MAX ? full : INT32_MAX), cut ? slices : 1, per,
                                cut ? size_t(cut) * slices * bn * kF8tRows * 4 : 0};
            }
        }
    }
    return best;
}

size_t f8_tiles_part(int64_t N, const F8Geom &g, bool a8, bool scaled, int P) {
    return tile_plan(N, g, a8 ? kX8 : (scaled ? kX16S : kX16), P).part;
}

template <int OP, int BN, bool SX, int NST>
static int go(const F8tArgs &a, hipStream_t st) {
    static_assert(NST * f8t_stage(OP, BN, SX) <= kLdsBytes, "the ring fits LDS");
    const int64_t grid = a.full + int64_t(a.tiles - a.full) * a.splits;
    if (a.tiles == INT32_MAX || grid >= 1 << 23) return set_error(VQK_ENOTIMPL, "8-bit product: grid too large");
    const int rc = launch_with_lds<k_f8_tiles<OP, BN, SX, NST>>(dim3(unsigned(grid)), dim3(512), size_t(NST) * f8t_stage(OP, BN, SX), st, a);
    if (rc || a.tiles == a.full) return rc;
    hipLaunchKernelGGL(k_f8_reduce<BN>, dim3(BN * kF8tRows / 1024, unsigned(a.tiles - a.full)), dim3(256), 0, st, a);
    return hip_status(hipGetLastError(), "slice sum launch");
}

template <int OP, bool SX>
static int go16(const F8tArgs &a, int bn, hipStream_t st) {
    switch (bn) {
        case 64: return go<OP, 64, SX, 3>(a, st);
        case 128: return go<OP, 128, SX, 2>(a, st);
        default:
            if constexpr (!SX) return go<OP, 192, SX, 2>(a, st);
            return set_error(VQK_EINVAL, "8-bit product: no tile of %d", bn);
    }
}

int f8_tiles(const F8Call &c, float *part, size_t part_bytes, hipStream_t st) {
    const int form = form_of(c), P = c.a8 ? 1 : c.x.P;
    F8tArgs a{};
    a.codes = c.codes; a.scales = c.scales; a.swo = c.swo; a.swk = c.swk;
    a.OUT = c.g.OUT; a.N = c.N;
    a.RT = int32_t(c.g.RT); a.NC = int32_t(c.g.NC); a.P = P;
    if (c.a8) {
        a.x = c.x8.codes; a.xld = c.x8.ld;
    } else {
        a.x = reinterpret_cast<const uint8_t *>(c.x.x); a.xld = c.x.ld * 2; a.xplane = c.x.plane * 2;
    }
    if (a.xld * 256 > INT64_C(0xffffffff))                // offsets inside a tile of x are 32 bits
        return set_error(VQK_ENOTIMPL, "8-bit product: rows %lld bytes apart", (long long)a.xld);
    a.sx = c.x8.scales; a.sn = c.x8.sn; a.sk = c.x8.sk;
    a.y = c.y; a.y_type = c.y_type;
    const TilePlan pl = tile_plan(c.N, c.g, form, P);
    if (pl.part > part_bytes || (pl.part && !part)) return set_error(VQK_ENOSPACE, "8-bit product: workspace %zu < %zu", part_bytes, pl.part);
    a.nt = int32_t((c.N + pl.bn - 1) / pl.bn);
    a.tiles = pl.tiles; a.full = pl.full; a.splits = pl.splits; a.per = pl.per;
    a.part = part;
    if (form == kX16S) return go16<kOpBF16, true>(a, pl.bn, st);
    if (form == kX16) return c.x.op == kOpF16 ? go16<kOpF16, false>(a, pl.bn, st) : go16<kOpBF16, false>(a, pl.bn, st);
    switch (pl.bn) {
        case 64: return go<kOpF8, 64, true, 3>(a, st);
        case 128: return go<kOpF8, 128, true, 3>(a, st);
        case 192: return go<kOpF8, 192, true, 2>(a, st);
        default: return go<kOpF8, 256, true, 2>(a, st);
    }
}

}  // namespace vqk
