// Launch of the few-row products of 8-bit weights (kernel in vqk_f8s.h).
#include "vqk_f8s.h"

namespace vqk {

// Registers of a block: two buffers of weights and their scales, and x.
constexpr int f8s_regs(int op, int nt, int p) { return 18 + nt * (op == kOpF8 ? 9 : 16 * p + 1); }
// Blocks a wave that the registers hold.
constexpr int f8s_cap(int op, int nt, int p) { return 208 / f8s_regs(op, nt, p); }

struct F8sPlan { int kw, ncw, ks; };          // waves along k, blocks a wave at most, ranges of k
static F8sPlan f8s_plan(int64_t NC, int cap, int64_t row_tiles) {
    // about four blocks a wave keep enough weights in flight, and fewer waves along k save the sums;
    // a small product takes more of them, until each CU has a workgroup
    int kw = 1;
    while (kw < kF8sWaves && ((NC + kw - 1) / kw > (cap < 4 ? cap : 4) ||
                              (NC > kw && row_tiles * kw < 256 * kF8sWaves))) kw *= 2;
    const int64_t ks = (NC + kw * cap - 1) / (kw * cap);
    return F8sPlan{kw, int((NC + kw * ks - 1) / (kw * ks)), int(ks)};
}

static int call_op(const F8Call &c) { return c.a8 ? kOpF8 : c.x.op; }
static int call_p(const F8Call &c) { return c.a8 ? 1 : c.x.P; }
static int call_nt(const F8Call &c) { return c.N <= 16 || call_p(c) != 1 ? 1 : 2; }
static int64_t call_tiles(const F8Call &c) { return (c.N + 16 * call_nt(c) - 1) / (16 * call_nt(c)); }
static F8sPlan call_plan(const F8Call &c) {
    return f8s_plan(c.g.NC, f8s_cap(call_op(c), call_nt(c), call_p(c)), call_tiles(c) * c.g.RT);
}

// Up to one tile of x (fp32: three) always: the weights pass once. More while the passes over
// them stay short of what tiles of 256 weight rows cost in slices of k and their sum. bf16 x
// in us, this way / by tiles: 4096 squared, 64 rows 11.7 / 17.1, 128 rows (67 MB in all)
// 13.4 / 21.0, 192 (100 MB) 22.1 / 19.1; 1024 squared, 1024 rows (33 MB) 10.3 / 14.2; 512
// squared, 8192 rows (67 MB, 256 tiles) 14.0 / 12.0; 5120 to 17408, 64 rows (178 MB) 41 / 30.
// fp32 x: 4096 squared, 96 rows (100 MB) 29 / 32, 192 43 / 39; 5120 to 17408, 48 rows 54 / 61.
bool f8_rows_ok(const F8Call &c) {
    const int64_t tiles = call_tiles(c);
    const bool one = call_p(c) == 1;
    return tiles <= (one ? 1 : 3) || tiles * f8_code_bytes(c.g.RT, c.g.NC) <= (one ? (tiles <= 16 ? 72 : 36) : 96) << 20;
}

size_t f8_rows_part(const F8Call &c) {
    const F8sPlan pl = call_plan(c);
    return pl.ks > 1 ? size_t(pl.ks) * size_t(c.N) * size_t(c.g.OUT) * 4 : 0;
}

// Sum of the ranges of k in their order, four outputs a thread.
__global__ void __launch_bounds__(256) k_f8_rows_sum(const F8sArgs p) {
    const int64_t all = p.N * p.OUT, at = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4;
    if (at >= all) return;
    const int n = int(min(int64_t(4), all - at));
    float v[4] = {};
    for (int z = 0; z < p.ks; ++z) {
        const float *src = p.part + z * all + at;
        if (n == 4 && all % 4 == 0) {
            const float4 a = *reinterpret_cast<const float4 *>(src);
            v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        } else {
            for (int i = 0; i < n; ++i) v[i] += src[i];
        }
    }
    mx_store4(p.y, p.y_type, at, v, n, (reinterpret_cast<uintptr_t>(p.y) & 15) == 0);
}

template <int OP, int NT, int P, int NCW>
static int go(F8sArgs a, int64_t tiles, int kw, hipStream_t st) {
    const int RW = kF8sWaves / kw;
    a.kw = kw;
    a.even = a.NC / (kw * a.ks);
    a.more = a.NC % (kw * a.ks);
    a.total_steps = int32_t((a.OUT + 16 * RW - 1) / (16 * RW));
    // row steps per workgroup: one round of workgroups, two to a CU where the registers let them
    const int64_t room = 40 + NCW * f8s_regs(OP, NT, P) <= 128 ? 512 : 256;
    const int64_t want = room / (tiles * a.ks) > 0 ? room / (tiles * a.ks) : 1;
    const int64_t steps = (a.total_steps + want - 1) / want;
    a.steps = int32_t(steps);
    a.nob = int32_t((a.total_steps + steps - 1) / steps);
    const int64_t grid = int64_t(a.nob) * tiles * a.ks;
    if (grid >= 1 << 23) return set_error(VQK_ENOTIMPL, "8-bit product: grid too large");
    const size_t sums = kw > 1 ? size_t(2) * kF8sWaves * NT * 1024 : 0;
    const size_t xl = a.stage ? size_t(kF8sWaves) * NCW * 16 * (OP == kOpF8 ? 128 : 256) : 0;
    const int rc = launch_with_lds<k_f8_rows<OP, NT, P, NCW>>(dim3(unsigned(grid)), dim3(64 * kF8sWaves),
                                                              sums > xl ? sums : xl, st, a);
    if (rc || a.ks == 1) return rc;
    hipLaunchKernelGGL(k_f8_rows_sum, dim3(unsigned((a.N * a.OUT + 1023) / 1024)), dim3(256), 0, st, a);
    return hip_status(hipGetLastError(), "sum of ranges launch");
}

template <int OP, int NT, int P, int NCW = 1>
static int go_ncw(const F8sArgs &a, int64_t tiles, F8sPlan pl, hipStream_t st) {
    if (pl.ncw == NCW) return go<OP, NT, P, NCW>(a, tiles, pl.kw, st);
    if constexpr (NCW < f8s_cap(OP, NT, P)) return go_ncw<OP, NT, P, NCW + 1>(a, tiles, pl, st);
    return set_error(VQK_EINVAL, "8-bit product: no instance of %d blocks", pl.ncw);
}

int f8_rows(const F8Call &c, float *part, size_t part_bytes, hipStream_t st) {
    F8sArgs a{};
    a.codes = c.codes; a.scales = c.scales; a.swo = c.swo; a.swk = c.swk;
    a.OUT = c.g.OUT; a.IN = c.g.IN; a.N = c.N;
    a.RT = int32_t(c.g.RT); a.NC = int32_t(c.g.NC);
    a.sx = c.x8.scales; a.sn = c.x8.sn; a.sk = c.x8.sk;
    if (c.a8) {
        a.x = c.x8.codes; a.xld = c.x8.ld;
    } else {
        a.x = reinterpret_cast<const uint8_t *>(c.x.x); a.xld = c.x.ld * 2; a.xplane = c.x.plane * 2;
    }
    a.y = c.y; a.y_type = c.y_type;
    a.stage = c.N > 2;
    const int nt = call_nt(c), P = call_p(c);
    const F8sPlan pl = call_plan(c);
    const size_t need = f8_rows_part(c);
    if (need > part_bytes || (need && !part)) return set_error(VQK_ENOSPACE, "8-bit product: workspace %zu < %zu", part_bytes, need);
    a.ks = pl.ks;
    a.part = part;
    const int64_t tiles = call_tiles(c);
    switch (call_op(c)) {
        case kOpF8: return nt == 2 ? go_ncw<kOpF8, 2, 1>(a, tiles, pl, st) : go_ncw<kOpF8, 1, 1>(a, tiles, pl, st);
        case kOpF16: return nt == 2 ? go_ncw<kOpF16, 2, 1>(a, tiles, pl, st) : go_ncw<kOpF16, 1, 1>(a, tiles, pl, st);
        default: break;
    }
    if (nt == 2) return go_ncw<kOpBF16, 2, 1>(a, tiles, pl, st);
    return P == 1 ? go_ncw<kOpBF16, 1, 1>(a, tiles, pl, st) : go_ncw<kOpBF16, 1, 3>(a, tiles, pl, st);
}

}  // namespace vqk
