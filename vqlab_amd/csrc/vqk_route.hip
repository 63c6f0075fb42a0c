// Router of a mixture of experts: softmax top-k of the logits, tokens per
// expert, the balance and z losses, and the gradient of the logits.
//
//   p_t = softmax(l_t), ids_t = the top_k largest (ties to the lower id),
//   w_t = p_t[ids_t] (norm: divided by their sum)
//   over the n live tokens:  c_e = |{t : e in ids_t}|,  P_e = sum_t p_te / n
//   balance = E sum_e c_e / (n k) P_e          (1 where every expert gets its share)
//   z       = sum_t lse_t^2 / n,  lse_t = log sum_e exp(l_te)
// with gradients g_b, g_z and dw, and f_e = g_b E c_e / (n^2 k) (c takes none):
//   dl_te = p_te (f_e - sum_i f_i p_ti) + 2 g_z / n lse_t p_te
//         + norm: [e in ids_t] w_te (dw_te - sum_j w_tj dw_tj)
//           else: p_te ([e in ids_t] dw_te - sum_j w_tj dw_tj)
// A token whose mask is 0, or whose logits are all -inf, is not live: its ids
// are -1, its weights and its gradient 0. An expert at -inf is never chosen
// (id -1, weight 0 where fewer than top_k are left).
//
// Sixteen lanes take a token (k_route16, k_route_bwd16: up to 512 experts, top_k
// up to 16), four tokens a wave, so that the steps across lanes stay inside a
// DPP row and serve four tokens at once; larger shapes take a wave a token
// (k_route, k_route_bwd). The sums over tokens stay in registers until the wave's
// last token. All arithmetic is fp32 (the sums over workgroups and the losses
// fp64). Sums meet in a fixed order: every result is the same from call to call.
#include "vqk_route.h"

namespace vqk {

struct RouteArgs {
    const void *l;
    int64_t T, ld;
    int32_t E, k, norm;
    const uint8_t *mask;
    int32_t *ids;
    float *wts;
    float2 *saved;                            // [T] (max, 1 / sum), or NULL
    // training: per-workgroup partials [wgs][E] and [wgs]
    float *part_p, *part_z;
    int32_t *part_c, *part_n;
};

template <int LT, int NS>
__device__ __forceinline__ void route_load(const void *l, int64_t base, int E, int lane, float (&v)[NS]) {
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int e = lane * NS + i;
        v[i] = e < E ? load_act(l, LT, base + e) : -__builtin_inff();
    }
}

template <int LT, int NS, bool TRAIN>
__global__ void __launch_bounds__(kRouteThreads) k_route(const RouteArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    int32_t *cnt = reinterpret_cast<int32_t *>(smem);              // [E]
    float *psh = reinterpret_cast<float *>(smem) + p.E;            // [E]
    __shared__ float zsh[kRouteWaves];
    __shared__ int nsh[kRouteWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if constexpr (TRAIN) {
        for (int e = threadIdx.x; e < p.E; e += kRouteThreads) cnt[e] = 0;
        __syncthreads();
    }
    float psum[NS] = {};
    float zsum = 0.f;
    int live = 0;
    for (int64_t t = int64_t(blockIdx.x) * kRouteWaves + wave; t < p.T; t += int64_t(gridDim.x) * kRouteWaves) {
        float v[NS];
        route_load<LT, NS>(p.l, t * p.ld, p.E, lane, v);
        uint32_t key[NS], best = 0;
        bool isnan = false;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            key[i] = f32_key(v[i]);
            isnan = isnan || v[i] != v[i];
            best = max(best, key[i]);
        }
        best = wave_max_u32(best);
        const bool anynan = __ballot(isnan) != 0;
        const bool on = (!p.mask || p.mask[t] != 0) && (best > kKeyNegInf || anynan);
        if (!on) {
            if (lane < p.k) {
                p.ids[t * p.k + lane] = -1;
                p.wts[t * p.k + lane] = 0.f;
            }
            if (p.saved && lane == 0) p.saved[t] = float2{0.f, 0.f};
            continue;
        }
        const float m = key_f32(best);
        float ex[NS], total = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            ex[i] = route_exp(v[i] - m);
            total += ex[i];
        }
        total = wave_sum(total);
        const float inv = 1.f / total;
        int id = -1;                          // lane j: the j-th choice and its exp
        float we = 0.f;
        for (int j = 0; j < p.k; ++j) {
            uint32_t mine = 0;
#pragma unroll
            for (int i = 0; i < NS; ++i) mine = max(mine, key[i]);
            const uint32_t top = wave_max_u32(mine);
            if (top <= kKeyNegInf) break;
            const int src = __ffsll((unsigned long long)__ballot(mine == top)) - 1;
            int at = 0;
#pragma unroll
            for (int i = NS - 1; i >= 0; --i)
                if (key[i] == top) at = i;
            const int e = src * NS + __builtin_amdgcn_readlane(at, src);
            if (lane == src) {
#pragma unroll
                for (int i = 0; i < NS; ++i)
                    if (i == at) key[i] = 0;
            }
            if (lane == j) {
                id = e;
                we = route_exp(key_f32(top) - m);
            }
        }
        float w = we * inv;
        if (p.norm) {
            const float s = wave_sum(we);
            w = we / s;
        }
        if (anynan) w = __uint_as_float(0x7fc00000u);
        if (lane < p.k) {
            p.ids[t * p.k + lane] = id;
            p.wts[t * p.k + lane] = w;
            if (TRAIN && id >= 0) atomicAdd(&cnt[id], 1);
        }
        if constexpr (TRAIN) {
            const float lse = m + logf(total);
            zsum += lse * lse;
            ++live;
#pragma unroll
            for (int i = 0; i < NS; ++i) psum[i] += ex[i] * inv;
        }
        if (p.saved && lane == 0) p.saved[t] = float2{m, inv};
    }
    if constexpr (TRAIN) {
        // the waves' sums in wave order
        for (int w = 0; w < kRouteWaves; ++w) {
            if (wave == w) {
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    const int e = lane * NS + i;
                    if (e < p.E) psh[e] = w ? psh[e] + psum[i] : psum[i];
                }
                if (lane == 0) {
                    zsh[w] = zsum;
                    nsh[w] = live;
                }
            }
            __syncthreads();
        }
        for (int e = threadIdx.x; e < p.E; e += kRouteThreads) {
            p.part_p[int64_t(blockIdx.x) * p.E + e] = psh[e];
            p.part_c[int64_t(blockIdx.x) * p.E + e] = cnt[e];
        }
        if (threadIdx.x == 0) {
            float z = 0.f;
            int n = 0;
            for (int w = 0; w < kRouteWaves; ++w) {
                z += zsh[w];
                n += nsh[w];
            }
            p.part_z[blockIdx.x] = z;
            p.part_n[blockIdx.x] = n;
        }
    }
}

// ------------------------------------------------- sixteen lanes to a token
constexpr int kRoute16MaxE = 512, kRoute16MaxK = 16;
// Tokens from which they pay: below, a wave a token spreads wider and is less code
// to fetch (509 tokens of 512 experts: 11 us against 31; 2048 of 256: both 7;
// 65536 of 256: 118 against 52).
constexpr int64_t kRoute16MinT = 2048;
static bool route16_ok(int64_t T, int64_t E, int k) {
    return T >= kRoute16MinT && E <= kRoute16MaxE && k <= kRoute16MaxK;
}

// How the top k are found: each lane's largest key is ranked against the row's
// other 15 (rotations); the k-th largest of these bounds the k-th largest key
// from below, and the keys that reach it, about 11 of 256 at k = 8, are
// collected in LDS and ranked against each other, two a lane. More than 32
// candidates (many equal logits) are taken one by one instead.
template <int LT, int NS, bool VEC, bool TRAIN>
__global__ void __launch_bounds__(kRouteThreads) k_route16(const RouteArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    int32_t *cnt = reinterpret_cast<int32_t *>(smem);              // [E]
    float *psh = reinterpret_cast<float *>(smem) + p.E;            // [E]
    __shared__ uint64_t cands[kRouteWaves][4][kRouteCands];
    __shared__ float zsh[kRouteWaves];
    __shared__ int nsh[kRouteWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sub = lane & 15, grp = lane >> 4;
    if constexpr (TRAIN) {
        for (int e = threadIdx.x; e < p.E; e += kRouteThreads) {
            cnt[e] = 0;
            psh[e] = 0.f;
        }
        __syncthreads();
    }
    float psum[NS] = {};
    float zsum = 0.f;
    int nlive = 0;
    const int64_t stride = int64_t(gridDim.x) * kRouteWaves * 4;
    for (int64_t t0 = (int64_t(blockIdx.x) * kRouteWaves + wave) * 4; t0 < p.T; t0 += stride) {
        const int64_t t = t0 + grp;
        const bool in = t < p.T && (!p.mask || p.mask[t] != 0);
        float v[NS];
        route_load16<LT, NS, VEC>(p.l, t * p.ld, p.E, sub, in, v);
        uint32_t key[NS], lm = 0;
        bool isnan = false;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            key[i] = f32_key(v[i]);
            isnan = isnan || v[i] != v[i];
            lm = max(lm, key[i]);
        }
        const uint32_t best = row_max(lm);
        const bool anynan = ((__ballot(isnan) >> (grp * 16)) & 0xffffu) != 0;
        const bool live = in && (best > kKeyNegInf || anynan);
        const float m = live ? key_f32(best) : 0.f;
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            v[i] = live ? route_exp(v[i] - m) : 0.f;
            total += v[i];
        }
        total = row_sum(total);
        const float inv = live ? 1.f / total : 0.f;

        // the k-th largest lane maximum
        int rank = 0;
#define VQK_ROR(N) rank += dpp_u<0x120 + N>(lm) > lm;
        VQK_ROR(1) VQK_ROR(2) VQK_ROR(3) VQK_ROR(4) VQK_ROR(5) VQK_ROR(6) VQK_ROR(7) VQK_ROR(8)
        VQK_ROR(9) VQK_ROR(10) VQK_ROR(11) VQK_ROR(12) VQK_ROR(13) VQK_ROR(14) VQK_ROR(15)
#undef VQK_ROR
        const uint32_t thr = max(row_min(rank < p.k ? lm : 0xffffffffu), kKeyNegInf + 1);
        int run = 0;
        wave_lds_sync();                      // the last token's candidates are read
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const bool c = live && key[i] >= thr;
            const uint32_t gm = uint32_t(__ballot(c) >> (grp * 16)) & 0xffffu;
            const int pos = run + __popc(gm & ((1u << sub) - 1u));
            if (c && pos < kRouteCands)
                cands[wave][grp][pos] = (uint64_t(key[i]) << 32) | uint32_t(~(64 * (i / 4) + 4 * sub + i % 4));
            run += __popc(gm);
        }
        uint64_t c0 = 0, c1 = 0;              // this lane's candidates, or with their ranks settled
        int r0 = 0, r1 = 0;
        if (__ballot(run > kRouteCands) == 0) {
            wave_lds_sync();
            if (sub < run) c0 = cands[wave][grp][sub];
            if (sub + 16 < run) c1 = cands[wave][grp][sub + 16];
            r0 = c1 > c0;
            r1 = c0 > c1;
#define VQK_ROR(N)                                                                              \
    {                                                                                           \
        const uint64_t a = dpp_u64<0x120 + N>(c0), b = dpp_u64<0x120 + N>(c1);                  \
        r0 += int(a > c0) + int(b > c0);                                                        \
        r1 += int(a > c1) + int(b > c1);                                                        \
    }
            VQK_ROR(1) VQK_ROR(2) VQK_ROR(3) VQK_ROR(4) VQK_ROR(5) VQK_ROR(6) VQK_ROR(7) VQK_ROR(8)
            VQK_ROR(9) VQK_ROR(10) VQK_ROR(11) VQK_ROR(12) VQK_ROR(13) VQK_ROR(14) VQK_ROR(15)
#undef VQK_ROR
        } else {
            for (int j = 0; j < p.k; ++j) {   // one by one: the largest key, of equals the lowest id
                uint32_t kb = 0, eb = 0xffffffffu;
#pragma unroll
                for (int i = 0; i < NS; ++i)
                    if (live && key[i] > kb) {
                        kb = key[i];
                        eb = uint32_t(64 * (i / 4) + 4 * sub + i % 4);
                    }
                const uint32_t top = row_max(kb);
                const uint32_t e = row_min(kb == top ? eb : 0xffffffffu);
                if (top > kKeyNegInf && sub == j) c0 = (uint64_t(top) << 32) | uint32_t(~e);
#pragma unroll
                for (int i = 0; i < NS; ++i)
                    if (uint32_t(64 * (i / 4) + 4 * sub + i % 4) == e) key[i] = 0;
            }
            r0 = sub;                         // k <= 16: in order already
            r1 = kRouteCands;
            run = 16 - __popc(uint32_t(__ballot(c0 == 0) >> (grp * 16)) & 0xffffu);
        }
        const bool s0 = c0 != 0 && r0 < p.k, s1 = c1 != 0 && r1 < p.k;
        const float e0 = s0 ? route_exp(key_f32(uint32_t(c0 >> 32)) - m) : 0.f;
        const float e1 = s1 ? route_exp(key_f32(uint32_t(c1 >> 32)) - m) : 0.f;
        const float sum = row_sum(e0 + e1);
        if (t < p.T) {
            const float f = anynan && live ? __uint_as_float(0x7fc00000u) : (p.norm ? 1.f / sum : inv);
            auto put = [&](int rank_, uint64_t c, float e) {
                const int id = int(~uint32_t(c));
                p.ids[t * p.k + rank_] = id;
                p.wts[t * p.k + rank_] = e * f;
                if (TRAIN) atomicAdd(&cnt[id], 1);
            };
            if (s0) put(r0, c0, e0);
            if (s1) put(r1, c1, e1);
            if (sub >= run && sub < p.k) {
                p.ids[t * p.k + sub] = -1;
                p.wts[t * p.k + sub] = anynan && live ? __uint_as_float(0x7fc00000u) : 0.f;
            }
            if (p.saved && sub == 0) p.saved[t] = float2{m, inv};
        }
        if constexpr (TRAIN) {
            if (live) {
                const float lse = m + logf(total);
                if (sub == 0) {
                    zsum += lse * lse;
                    ++nlive;
                }
#pragma unroll
                for (int i = 0; i < NS; ++i) psum[i] += v[i] * inv;
            }
        }
    }
    if constexpr (TRAIN) {
        // the tokens' sums in order of wave and row of lanes
        for (int w = 0; w < kRouteWaves * 4; ++w) {
            if (wave == w / 4 && grp == w % 4) {
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    const int e = 64 * (i / 4) + 4 * sub + i % 4;
                    if (e < p.E) psh[e] += psum[i];
                }
            }
            if (w % 4 == 3) __syncthreads();
            else wave_lds_sync();
        }
        zsum = wave_sum(zsum);
        for (int o = 16; o < 64; o <<= 1) nlive += __shfl_xor(nlive, o);
        if (lane == 0) {
            zsh[wave] = zsum;
            nsh[wave] = nlive;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < p.E; e += kRouteThreads) {
            p.part_p[int64_t(blockIdx.x) * p.E + e] = psh[e];
            p.part_c[int64_t(blockIdx.x) * p.E + e] = cnt[e];
        }
        if (threadIdx.x == 0) {
            float z = 0.f;
            int n = 0;
            for (int w = 0; w < kRouteWaves; ++w) {
                z += zsh[w];
                n += nsh[w];
            }
            p.part_z[blockIdx.x] = z;
            p.part_n[blockIdx.x] = n;
        }
    }
}

// The partials of 16 experts a workgroup: 64 threads an expert group walk over
// the routing workgroups, then meet in LDS in a fixed order.
constexpr int kFinExperts = 16;
__global__ void __launch_bounds__(1024) k_route_experts(const FinishArgs p) {
    __shared__ double P[64][kFinExperts];
    __shared__ int C[64][kFinExperts];
    const int j = threadIdx.x % kFinExperts, s = threadIdx.x / kFinExperts;
    const int e = blockIdx.x * kFinExperts + j;
    double sum = 0.;
    int c = 0;
    if (e < p.E)
        for (int w = s; w < p.wgs; w += 64) {
            sum += p.part_p[int64_t(w) * p.E + e];
            c += p.part_c[int64_t(w) * p.E + e];
        }
    P[s][j] = sum;
    C[s][j] = c;
    __syncthreads();
    for (int o = 32; o >= 1; o >>= 1) {
        if (s < o) {
            P[s][j] += P[s + o][j];
            C[s][j] += C[s + o][j];
        }
        __syncthreads();
    }
    if (s == 0 && e < p.E) p.counts[e] = C[0][j];
    if (threadIdx.x == 0) {
        double d = 0.;
        for (int i = 0; i < kFinExperts; ++i) d += double(C[0][i]) * P[0][i];   // past E: 0
        p.dot[blockIdx.x] = d;
    }
}

// The losses from the sums of every group of experts and every workgroup.
__global__ void __launch_bounds__(512) k_route_losses(const FinishArgs p, int groups) {
    __shared__ double d[512], z[512];
    __shared__ int n[512];
    const int t = threadIdx.x;
    d[t] = t < groups ? p.dot[t] : 0.;        // kRouteMaxE / kFinExperts groups at most
    z[t] = 0.;
    n[t] = 0;
    for (int w = t; w < p.wgs; w += 512) {
        z[t] += double(p.part_z[w]);
        n[t] += p.part_n[w];
    }
    __syncthreads();
    for (int o = 256; o >= 1; o >>= 1) {
        if (t < o) {
            d[t] += d[t + o];
            z[t] += z[t + o];
            n[t] += n[t + o];
        }
        __syncthreads();
    }
    if (t == 0) {
        const double N = n[0];
        p.stats[0] = N > 0. ? float(double(p.E) * d[0] / (N * N * p.k)) : 0.f;
        p.stats[1] = N > 0. ? float(z[0] / N) : 0.f;
        p.stats[2] = float(N);
    }
}

struct RouteBwdArgs {
    const void *l;
    int64_t T, ld;
    int32_t E, k, norm;
    const int32_t *ids, *counts;
    const float *wts, *stats;
    const float2 *saved;
    const float *dw, *gb, *gz;                // NULL: no gradient of that output
    void *dl;
};

template <int LT, int NS>
__global__ void __launch_bounds__(kRouteThreads) k_route_bwd(const RouteBwdArgs p) {
    extern __shared__ __align__(16) float rows[];      // [waves][64 * NS]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float *row = rows + wave * 64 * NS;
    const float n = p.stats[2];
    const float fb = p.gb && n > 0.f ? p.gb[0] * (float(p.E) / (n * n * float(p.k))) : 0.f;
    const float fz = p.gz && n > 0.f ? 2.f * p.gz[0] / n : 0.f;
    float f[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int e = lane * NS + i;
        f[i] = e < p.E ? fb * float(p.counts[e]) : 0.f;
    }
    for (int64_t t = int64_t(blockIdx.x) * kRouteWaves + wave; t < p.T; t += int64_t(gridDim.x) * kRouteWaves) {
        const float2 sv = p.saved[t];
        if (sv.y == 0.f) {                    // not live (a live token's sum is at most E)
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (lane * NS + i < p.E) store_act(p.dl, LT, t * p.E + lane * NS + i, 0.f);
            continue;
        }
        float v[NS];
        route_load<LT, NS>(p.l, t * p.ld, p.E, lane, v);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            v[i] = route_exp(v[i] - sv.x) * sv.y;  // p
            dot += f[i] * v[i];
        }
        int id = -1;
        float wdw = 0.f, w = 0.f;
        if (p.dw && lane < p.k) {
            id = p.ids[t * p.k + lane];
            w = p.wts[t * p.k + lane];
            wdw = id >= 0 ? w * p.dw[t * p.k + lane] : 0.f;
        }
        dot = wave_sum(dot);
        const float s = wave_sum(wdw);
        const float lse = sv.x - logf(sv.y);
        const float sub = fz * lse - dot - (p.norm ? 0.f : s);
#pragma unroll
        for (int i = 0; i < NS; ++i) row[lane * NS + i] = 0.f;
        wave_lds_sync();
        if (id >= 0) row[id] = p.norm ? wdw - w * s : wdw;
        wave_lds_sync();
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const float d = v[i] * (f[i] + sub) + row[lane * NS + i];
            if (lane * NS + i < p.E) store_act(p.dl, LT, t * p.E + lane * NS + i, d);
        }
    }
}

template <int LT, int NS, bool VEC>
__global__ void __launch_bounds__(kRouteThreads) k_route_bwd16(const RouteBwdArgs p) {
    __shared__ __align__(16) float rows[kRouteWaves][4][16 * NS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sub = lane & 15, grp = lane >> 4;
    float *row = rows[wave][grp];
    const float n = p.stats[2];
    const float fb = p.gb && n > 0.f ? p.gb[0] * (float(p.E) / (n * n * float(p.k))) : 0.f;
    const float fz = p.gz && n > 0.f ? 2.f * p.gz[0] / n : 0.f;
    float f[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int e = 64 * (i / 4) + 4 * sub + i % 4;
        f[i] = e < p.E ? fb * float(p.counts[e]) : 0.f;
    }
    const int64_t stride = int64_t(gridDim.x) * kRouteWaves * 4;
    for (int64_t t0 = (int64_t(blockIdx.x) * kRouteWaves + wave) * 4; t0 < p.T; t0 += stride) {
        const int64_t t = t0 + grp;
        const bool in = t < p.T;
        const float2 sv = in ? p.saved[t] : float2{0.f, 0.f};
        const bool live = sv.y != 0.f;        // a live token's sum is at most E
        float v[NS];
        route_load16<LT, NS, VEC>(p.l, t * p.ld, p.E, sub, live, v);
        int id = -1;
        float wdw = 0.f, w = 0.f;
        if (p.dw && live && sub < p.k) {
            id = p.ids[t * p.k + sub];
            w = p.wts[t * p.k + sub];
            wdw = id >= 0 ? w * p.dw[t * p.k + sub] : 0.f;
        }
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            v[i] = live ? route_exp(v[i] - sv.x) * sv.y : 0.f;      // p
            dot += f[i] * v[i];
        }
        dot = row_sum(dot);
        const float s = row_sum(wdw);
        const float lse = sv.x - logf(sv.y);
        const float sub_ = fz * lse - dot - (p.norm ? 0.f : s);
#pragma unroll
        for (int q = 0; q < NS / 4; ++q) *reinterpret_cast<float4 *>(row + 64 * q + 4 * sub) = float4{0.f, 0.f, 0.f, 0.f};
        wave_lds_sync();
        if (id >= 0) row[id] = p.norm ? wdw - w * s : wdw;
        wave_lds_sync();
#pragma unroll
        for (int q = 0; q < NS / 4; ++q) {
            const int e = 64 * q + 4 * sub;
            const float4 a = *reinterpret_cast<const float4 *>(row + e);
            const float add[4] = {a.x, a.y, a.z, a.w};
            float d[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j] = live ? v[4 * q + j] * (f[4 * q + j] + sub_) + add[j] : 0.f;
            if (!in || e >= p.E) continue;
            if constexpr (VEC) {
                if constexpr (LT == VQK_F32) {
                    *reinterpret_cast<float4 *>(static_cast<float *>(p.dl) + t * p.E + e) = float4{d[0], d[1], d[2], d[3]};
                } else {
                    uint32_t h[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) h[j] = LT == VQK_BF16 ? f32_to_bf16(d[j]) : f32_to_h(d[j]);
                    u32x2 o;
                    o.x = h[0] | (h[1] << 16);
                    o.y = h[2] | (h[3] << 16);
                    *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(p.dl) + t * p.E + e) = o;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (e + j < p.E) store_act(p.dl, LT, t * p.E + e + j, d[j]);
            }
        }
    }
}

// Workgroups of the forward: one wave to four tokens (k_route16) or to one.
static int route_wgs(int64_t T, int64_t E, int k) {
    return route_wgs_of(T, route16_ok(T, E, k) ? 4 * kRouteWaves : kRouteWaves);
}

static int fin_groups(int64_t E) { return int((E + kFinExperts - 1) / kFinExperts); }
static_assert(kRouteMaxE / kFinExperts <= 512, "one thread each in k_route_losses");
// Workspace: the groups' fp64 sums, then the workgroups' partials.
size_t route_bytes(int64_t T, int64_t E) {          // for any top_k
    return size_t(fin_groups(E)) * 8 + size_t(route_wgs(T, E, kRouteMaxK)) * (size_t(E) * 8 + 8);
}

void route_parts(void *workspace, int64_t E, int wgs, FinishArgs *f, float **part_p, int32_t **part_c, float **part_z,
                 int32_t **part_n) {
    f->dot = static_cast<double *>(workspace);
    *part_p = reinterpret_cast<float *>(f->dot + fin_groups(E));
    *part_c = reinterpret_cast<int32_t *>(*part_p + size_t(wgs) * E);
    *part_z = reinterpret_cast<float *>(*part_c + size_t(wgs) * E);
    *part_n = reinterpret_cast<int32_t *>(*part_z + wgs);
    f->part_p = *part_p; f->part_c = *part_c; f->part_z = *part_z; f->part_n = *part_n;
    f->wgs = wgs;
    f->E = int32_t(E);
}

int route_finish(const FinishArgs &f, hipStream_t st) {
    const int groups = fin_groups(f.E);
    hipLaunchKernelGGL(k_route_experts, dim3(groups), dim3(1024), 0, st, f);
    const int rc = hip_status(hipGetLastError(), "router sums launch");
    if (rc) return rc;
    hipLaunchKernelGGL(k_route_losses, dim3(1), dim3(512), 0, st, f, groups);
    return hip_status(hipGetLastError(), "router losses launch");
}

template <int LT, int NS>
static int go_route(const RouteArgs &a, bool train, int wgs, hipStream_t st) {
    if (train) hipLaunchKernelGGL((k_route<LT, NS, true>), dim3(wgs), dim3(kRouteThreads), 8 * a.E, st, a);
    else hipLaunchKernelGGL((k_route<LT, NS, false>), dim3(wgs), dim3(kRouteThreads), 0, st, a);
    return hip_status(hipGetLastError(), "router launch");
}
template <int LT, int NS>
static int go_route_bwd(const RouteBwdArgs &a, int wgs, hipStream_t st) {
    hipLaunchKernelGGL((k_route_bwd<LT, NS>), dim3(wgs), dim3(kRouteThreads), kRouteWaves * 64 * NS * 4, st, a);
    return hip_status(hipGetLastError(), "router gradient launch");
}

bool route_vec(const void *l, int64_t ld, int64_t E, int lt) {
    return E % 4 == 0 && ld % 4 == 0 && (reinterpret_cast<uintptr_t>(l) & (lt == VQK_F32 ? 15 : 7)) == 0;
}
template <int LT, int NS>
static int go_route16(const RouteArgs &a, bool train, int wgs, hipStream_t st) {
    const bool vec = route_vec(a.l, a.ld, a.E, LT);
    const dim3 g(wgs), b(kRouteThreads);
    const size_t lds = train ? 8 * a.E : 0;
    if (train && vec) hipLaunchKernelGGL((k_route16<LT, NS, true, true>), g, b, lds, st, a);
    else if (train) hipLaunchKernelGGL((k_route16<LT, NS, false, true>), g, b, lds, st, a);
    else if (vec) hipLaunchKernelGGL((k_route16<LT, NS, true, false>), g, b, lds, st, a);
    else hipLaunchKernelGGL((k_route16<LT, NS, false, false>), g, b, lds, st, a);
    return hip_status(hipGetLastError(), "router launch");
}
template <int LT, int NS>
static int go_route_bwd16(const RouteBwdArgs &a, int wgs, hipStream_t st) {
    const bool vec = route_vec(a.l, a.ld, a.E, LT) && (reinterpret_cast<uintptr_t>(a.dl) & 15) == 0;
    if (vec) hipLaunchKernelGGL((k_route_bwd16<LT, NS, true>), dim3(wgs), dim3(kRouteThreads), 0, st, a);
    else hipLaunchKernelGGL((k_route_bwd16<LT, NS, false>), dim3(wgs), dim3(kRouteThreads), 0, st, a);
    return hip_status(hipGetLastError(), "router gradient launch");
}

// The smallest instance that holds E.
template <int LT>
static int route_ns(const RouteArgs &a, bool train, int wgs, hipStream_t st) {
    const int E = a.E;
    if (route16_ok(a.T, E, a.k)) {
        if (E <= 64) return go_route16<LT, 4>(a, train, wgs, st);
        if (E <= 128) return go_route16<LT, 8>(a, train, wgs, st);
        if (E <= 192) return go_route16<LT, 12>(a, train, wgs, st);
        if (E <= 256) return go_route16<LT, 16>(a, train, wgs, st);
        if (E <= 384) return go_route16<LT, 24>(a, train, wgs, st);
        return go_route16<LT, 32>(a, train, wgs, st);
    }
    if (E <= 64) return go_route<LT, 1>(a, train, wgs, st);
    if (E <= 128) return go_route<LT, 2>(a, train, wgs, st);
    if (E <= 256) return go_route<LT, 4>(a, train, wgs, st);
    if (E <= 512) return go_route<LT, 8>(a, train, wgs, st);
    if (E <= 1024) return go_route<LT, 16>(a, train, wgs, st);
    return go_route<LT, 32>(a, train, wgs, st);
}
template <int LT>
static int route_bwd_ns(const RouteBwdArgs &a, int wgs, hipStream_t st) {
    const int E = a.E;
    if (route16_ok(a.T, E, a.k)) {
        if (E <= 64) return go_route_bwd16<LT, 4>(a, wgs, st);
        if (E <= 128) return go_route_bwd16<LT, 8>(a, wgs, st);
        if (E <= 192) return go_route_bwd16<LT, 12>(a, wgs, st);
        if (E <= 256) return go_route_bwd16<LT, 16>(a, wgs, st);
        if (E <= 384) return go_route_bwd16<LT, 24>(a, wgs, st);
        return go_route_bwd16<LT, 32>(a, wgs, st);
    }
    if (E <= 64) return go_route_bwd<LT, 1>(a, wgs, st);
    if (E <= 128) return go_route_bwd<LT, 2>(a, wgs, st);
    if (E <= 256) return go_route_bwd<LT, 4>(a, wgs, st);
    if (E <= 512) return go_route_bwd<LT, 8>(a, wgs, st);
    if (E <= 1024) return go_route_bwd<LT, 16>(a, wgs, st);
    return go_route_bwd<LT, 32>(a, wgs, st);
}

int check_route(int32_t l_type, int64_t T, int64_t E, int64_t ld, int32_t k, const char *what) {
    if (!act_size(l_type)) return set_error(VQK_EINVAL, "%s: logits type %d", what, l_type);
    if (T < 0 || E < 1 || ld < E) return set_error(VQK_EINVAL, "%s: T=%lld E=%lld ld=%lld", what, (long long)T, (long long)E, (long long)ld);
    if (E > kRouteMaxE) return set_error(VQK_ENOTIMPL, "%s: E=%lld > %d", what, (long long)E, kRouteMaxE);
    if (k < 1 || k > E) return set_error(VQK_EINVAL, "%s: top_k=%d of %lld experts", what, k, (long long)E);
    if (k > kRouteMaxK) return set_error(VQK_ENOTIMPL, "%s: top_k=%d > %d", what, k, kRouteMaxK);
    return VQK_OK;
}

}  // namespace vqk

using namespace vqk;

extern "C" int vqk_route_workspace(int64_t T, int64_t E, size_t *bytes) {
    if (T < 0 || E < 1 || E > kRouteMaxE) return set_error(VQK_EINVAL, "route: T=%lld E=%lld", (long long)T, (long long)E);
    if (!bytes) return set_error(VQK_EINVAL, "route: NULL bytes");
    *bytes = route_bytes(T, E);
    return VQK_OK;
}

extern "C" int vqk_route(const void *logits, int32_t l_type, int64_t T, int64_t E, int64_t ld,
                         const uint8_t *mask, int32_t top_k, int32_t norm_topk, int32_t *ids, float *wts,
                         int32_t *counts, float *stats, float *saved, void *workspace, size_t ws_bytes,
                         void *stream) {
    int rc = check_route(l_type, T, E, ld, top_k, "route");
    if (rc) return rc;
    const bool train = counts || stats;
    if (train && (!counts || !stats)) return set_error(VQK_EINVAL, "route: counts and stats come together");
    if (T > 0 && (!logits || !ids || !wts)) return set_error(VQK_EINVAL, "route: NULL pointer");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int wgs = route_wgs(T, E, top_k);
    RouteArgs a{};
    a.l = logits; a.T = T; a.ld = ld;
    a.E = int32_t(E); a.k = top_k; a.norm = norm_topk;
    a.mask = mask; a.ids = ids; a.wts = wts;
    a.saved = reinterpret_cast<float2 *>(saved);
    if (reinterpret_cast<uintptr_t>(saved) & 7) return set_error(VQK_EINVAL, "route: saved must be 8-byte aligned");
    FinishArgs f{};
    if (train) {
        const size_t need = route_bytes(T, E);
        if (!workspace || ws_bytes < need) return set_error(VQK_ENOSPACE, "route: workspace %zu < %zu", ws_bytes, need);
        if (reinterpret_cast<uintptr_t>(workspace) & 15) return set_error(VQK_EINVAL, "route: workspace must be 16-byte aligned");
        route_parts(workspace, E, wgs, &f, &a.part_p, &a.part_c, &a.part_z, &a.part_n);
        f.k = top_k; f.counts = counts; f.stats = stats;
    }
    if (wgs) {
        switch (l_type) {
            case VQK_F16: rc = route_ns<VQK_F16>(a, train, wgs, st); break;
            case VQK_BF16: rc = route_ns<VQK_BF16>(a, train, wgs, st); break;
            default: rc = route_ns<VQK_F32>(a, train, wgs, st);
        }
        if (rc) return rc;
    }
    return train ? route_finish(f, st) : VQK_OK;
}

extern "C" int vqk_route_backward(const void *logits, int32_t l_type, int64_t T, int64_t E, int64_t ld,
                                  int32_t top_k, int32_t norm_topk, const int32_t *ids, const float *wts,
                                  const int32_t *counts, const float *stats, const float *saved,
                                  const float *dw, const float *dbalance, const float *dz, void *dlogits,
                                  void *stream) {
    const int rc = check_route(l_type, T, E, ld, top_k, "route backward");
    if (rc) return rc;
    if (T == 0) return VQK_OK;
    if (!logits || !ids || !wts || !counts || !stats || !saved || !dlogits)
        return set_error(VQK_EINVAL, "route backward: NULL pointer");
    if (reinterpret_cast<uintptr_t>(saved) & 7)
        return set_error(VQK_EINVAL, "route backward: saved must be 8-byte aligned");
    RouteBwdArgs a{};
    a.l = logits; a.T = T; a.ld = ld;
    a.E = int32_t(E); a.k = top_k; a.norm = norm_topk;
    a.ids = ids; a.counts = counts; a.wts = wts; a.stats = stats;
    a.saved = reinterpret_cast<const float2 *>(saved);
    a.dw = dw; a.gb = dbalance; a.gz = dz;
    a.dl = dlogits;
    const int per = route16_ok(T, E, top_k) ? 4 * kRouteWaves : kRouteWaves;
    const int64_t w = (T + per - 1) / per;
    const int wgs = int(w < 2048 ? w : 2048);
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (l_type) {
        case VQK_F16: return route_bwd_ns<VQK_F16>(a, wgs, st);
        case VQK_BF16: return route_bwd_ns<VQK_BF16>(a, wgs, st);
        default: return route_bwd_ns<VQK_F32>(a, wgs, st);
    }
}
