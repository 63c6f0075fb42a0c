// Launch of the few-row MXFP4 products (kernel in vqk_mxs.h).
#include "vqk_mxs.h"

namespace vqk {

void mx_args(const MxCall &c, MxsArgs *a) {
    *a = MxsArgs{};
    for (int i = 0; i < 2; ++i) {
        a->codes[i] = c.codes[i];
        a->scales[i] = c.scales[i];
    }
    a->OUT = c.g.OUT; a->E = c.g.E;
    a->RT = int32_t(c.g.RT); a->NC = int32_t(c.g.NC); a->NB = int32_t(c.g.NB);
    a->x = c.x.x; a->xld = c.x.ld; a->xplane = c.x.plane;
    a->N = c.N; a->xkrep = int32_t(c.xkrep);
    a->ids = c.ids; a->order = c.order; a->meta = c.meta; a->ntiles = c.ntiles;
    a->y = c.y; a->y_type = c.y_type; a->yp = c.yp; a->ysorted = c.ysorted;
    a->ldy = c.ldy; a->yplane = c.yplane;
    a->ocover = c.codes[1] ? c.ldy : c.g.OUT;
}

int64_t mx_tiles(const MxCall &c, int rows) {
    if (c.ids) return c.N;
    const int64_t full = (c.N + rows - 1) / rows;
    return c.meta ? full + (c.N < c.g.E + 1 ? c.N : c.g.E + 1) : full;
}

// Chunks per wave that the registers hold: 16 per chunk and x operand, 9 for two
// buffers of weights, 200 in all. (20 rows of 5120 -> 17408, five chunks a wave at
// 210: 25.6 us, the tiles of vqk_mxg.h 20.4; four chunks, 4096 -> 4096: 8.5 and 14.7.)
constexpr int rows_cap(int xn, bool glu) { return 200 / (16 * xn + (glu ? 18 : 9)); }

// Waves along k and chunks per wave, or kw = 0 where x does not fit.
struct RowsPlan { int kw, ncw; };
static RowsPlan rows_plan(int64_t NC, int xn, bool glu, int64_t row_tiles) {
    const int cap = rows_cap(xn, glu);
    // about four chunks a wave keep enough weights in flight, and fewer waves along k save the sums;
    // a small product takes more of them, until each CU has a workgroup
    int kw = 1;
    while (kw < kMxsWaves && ((NC + kw - 1) / kw > (cap < 4 ? cap : 4) ||
                              (NC > kw && row_tiles * kw < 256 * kMxsWaves))) kw *= 2;
    const int64_t ncw = (NC + kw - 1) / kw;
    return ncw <= cap ? RowsPlan{kw, int(ncw)} : RowsPlan{0, 0};
}

// Dense x of more than two rows goes through LDS, which holds five chunks a wave;
// longer rows are left to the tiles.
static bool rows_stage(const MxCall &c) { return !c.ids && c.N > 2; }
constexpr int kStageChunks = kLdsBytes / (kMxsWaves * 4096);

bool mx_rows_ok(const MxCall &c, int NT) {
    if (c.meta || (NT != 1 && (NT != 2 || c.x.P != 1))) return false;
    const RowsPlan pl = rows_plan(c.g.NC, NT * c.x.P, c.codes[1] != nullptr, mx_tiles(c, 16 * NT) * c.g.RT);
    return pl.kw > 0 && (!rows_stage(c) || pl.ncw <= kStageChunks);
}

template <int OP, int NT, int P, int NCW, bool GLU>
static int go(MxsArgs a, int64_t tiles, int kw, hipStream_t st) {
    const int RW = kMxsWaves / kw;
    a.kw = kw;
    a.total_steps = int32_t((a.ocover + 16 * RW - 1) / (16 * RW));
    // row steps per workgroup: one round of workgroups, two to a CU where the registers let them
    const int64_t room = 45 + NCW * (16 * NT * P + (GLU ? 18 : 9)) <= 128 ? 512 : 256;
    const int64_t want = tiles > 0 ? (room + tiles - 1) / tiles : 1;
    int64_t steps = (a.total_steps + want - 1) / want;
    if (a.ids) steps = steps > 8 ? 8 : steps;      // pairs without an expert leave early
    a.steps = int32_t(steps);
    a.nob = int32_t((a.total_steps + steps - 1) / steps);
    const int64_t grid = int64_t(a.nob) * tiles;
    if (grid > INT32_MAX) return set_error(VQK_ENOTIMPL, "MXFP4 product: grid too large");
    const size_t sums = kw > 1 ? size_t(2) * kMxsWaves * (GLU ? 2 : 1) * NT * 1024 : 0;
    const size_t xl = a.stage ? size_t(kMxsWaves) * NCW * 4096 : 0;
    return launch_with_lds<k_mx_rows<OP, NT, P, NCW, GLU>>(dim3(unsigned(grid)), dim3(64 * kMxsWaves),
                                                       sums > xl ? sums : xl, st, a);
}

template <int OP, int NT, int P, bool GLU, int NCW = 1>
static int go_ncw(const MxsArgs &a, int64_t tiles, RowsPlan pl, hipStream_t st) {
    if (pl.ncw == NCW) return go<OP, NT, P, NCW, GLU>(a, tiles, pl.kw, st);
    if constexpr (NCW < rows_cap(NT * P, GLU)) return go_ncw<OP, NT, P, GLU, NCW + 1>(a, tiles, pl, st);
    return set_error(VQK_EINVAL, "MXFP4 product: no instance of %d chunks", pl.ncw);
}
template <int OP, int NT, int P>
static int go_glu(const MxsArgs &a, bool glu, int64_t tiles, RowsPlan pl, hipStream_t st) {
    return glu ? go_ncw<OP, NT, P, true>(a, tiles, pl, st) : go_ncw<OP, NT, P, false>(a, tiles, pl, st);
}

int mx_rows(const MxCall &c, int NT, hipStream_t st) {
    const bool glu = c.codes[1] != nullptr;
    MxsArgs a;
    mx_args(c, &a);
    const int64_t tiles = mx_tiles(c, 16 * NT);
    if (tiles == 0) return VQK_OK;
    const RowsPlan pl = rows_plan(c.g.NC, NT * c.x.P, glu, tiles * c.g.RT);
    a.stage = rows_stage(c);
    if (c.x.op == kOpF16)
        return NT == 2 ? go_glu<kOpF16, 2, 1>(a, glu, tiles, pl, st) : go_glu<kOpF16, 1, 1>(a, glu, tiles, pl, st);
    if (NT == 2) return go_glu<kOpBF16, 2, 1>(a, glu, tiles, pl, st);
    switch (c.x.P) {
        case 1: return go_glu<kOpBF16, 1, 1>(a, glu, tiles, pl, st);
        case 2: return go_glu<kOpBF16, 1, 2>(a, glu, tiles, pl, st);
        default: return go_glu<kOpBF16, 1, 3>(a, glu, tiles, pl, st);
    }
}

}  // namespace vqk
