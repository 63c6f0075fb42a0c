// Launch of the few-row MXFP4 products (kernel in vqk_mxs.h).
#include "vqk_mxs.h"

namespace vqk {

template <int NT, int MT, bool GLU, int P>
static int go(MxsArgs a, int64_t tiles, hipStream_t st) {
    const int64_t cover = a.ocover;
    a.nob = int32_t((cover + 16 * MT - 1) / (16 * MT));
    const int64_t grid = int64_t(a.nob) * tiles;
    if (grid > INT32_MAX) return set_error(VQK_ENOTIMPL, "MXFP4 product: grid too large");
    int nw = 1;                               // no wave without a chunk of k
    while (nw < kMxsMaxWaves && nw < a.NC) nw *= 2;
    const size_t lds = size_t(nw) * (GLU ? 2 : 1) * MT * NT * 1024;
    return launch_with_lds<k_mx_stream<NT, MT, GLU, P>>(dim3(unsigned(grid)), dim3(64 * nw), lds, st, a);
}

template <int NT, int MT, bool GLU>
static int go_p(const MxsArgs &a, int P, int64_t tiles, hipStream_t st) {
    switch (P) {
        case 1: return go<NT, MT, GLU, 1>(a, tiles, st);
        case 2: return go<NT, MT, GLU, 2>(a, tiles, st);
        default: return go<NT, MT, GLU, 3>(a, tiles, st);
    }
}

void mx_args(const MxCall &c, MxsArgs *a) {
    *a = MxsArgs{};
    a->codes0 = c.codes[0]; a->scales0 = c.scales[0];
    a->codes1 = c.codes[1]; a->scales1 = c.scales[1];
    a->NB = c.NB; a->OUT = c.OUT; a->E = c.E;
    a->NC = int32_t((c.NB + 3) / 4);
    a->x = c.x.x; a->xld = c.x.ld; a->xplane = c.x.plane;
    a->N = c.N; a->xkrep = c.xkrep;
    a->ids = c.ids; a->order = c.order; a->meta = c.meta; a->ntiles = c.ntiles;
    a->y = c.y; a->y_type = c.y_type; a->yp = c.yp; a->ysorted = c.ysorted;
    a->ldy = c.ldy; a->yplane = c.yplane;
    a->ocover = c.codes[1] ? c.ldy : c.OUT;
}

int64_t mx_tiles(const MxCall &c, int rows) {
    if (c.ids) return c.N;
    const int64_t full = (c.N + rows - 1) / rows;
    return c.meta ? full + (c.N < c.E + 1 ? c.N : c.E + 1) : full;
}

int mx_stream(const MxCall &c, int NT, hipStream_t st) {
    const bool glu = c.codes[1] != nullptr;
    MxsArgs a;
    mx_args(c, &a);
    const int64_t tiles = mx_tiles(c, 16 * NT);
    if (tiles == 0) return VQK_OK;
    if (glu) {
        switch (NT) {
            case 1: return go_p<1, 1, true>(a, c.x.P, tiles, st);
            case 2: return go_p<2, 1, true>(a, c.x.P, tiles, st);
            default: return go_p<4, 1, true>(a, c.x.P, tiles, st);
        }
    }
    switch (NT) {
        case 1: return go_p<1, 1, false>(a, c.x.P, tiles, st);
        case 2: return go_p<2, 2, false>(a, c.x.P, tiles, st);
        default: return go_p<4, 2, false>(a, c.x.P, tiles, st);
    }
}

}  // namespace vqk
