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
// One wave takes a token: lane i holds experts i * NS .. i * NS + NS - 1, so
// equal logits go to the lower id by the first lane of a ballot, and the sums
// over tokens stay in the lane's registers until the wave's last token. All
// arithmetic is fp32 (the sums over workgroups and the losses fp64). Sums meet
// in a fixed order: every result is the same from call to call.
#include "vqk_common.h"

namespace vqk {

constexpr int kRouteWaves = 4;
constexpr int kRouteThreads = kRouteWaves * kWave;
constexpr int kRouteMaxWgs = 512;
constexpr int kRouteMaxE = 2048;
constexpr int kRouteMaxK = 64;
constexpr uint32_t kKeyNegInf = 0x007fffffu;           // f32_key(-inf); NaN maps below it

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
            ex[i] = expf(v[i] - m);
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
                we = expf(key_f32(top) - m);
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

struct FinishArgs {
    const float *part_p, *part_z;
    const int32_t *part_c, *part_n;
    int32_t wgs, E, k;
    int32_t *counts;
    float *stats;                             // balance, z, n
};

// One workgroup: the partials of every expert in workgroup order, then the losses.
__global__ void __launch_bounds__(1024) k_route_finish(const FinishArgs p) {
    __shared__ double dsum[1024], zred[1024];
    __shared__ int nred[1024];
    const int tid = threadIdx.x;
    double z = 0., dot = 0.;
    int n = 0;
    for (int w = tid; w < p.wgs; w += 1024) {
        z += p.part_z[w];
        n += p.part_n[w];
    }
    for (int e = tid; e < p.E; e += 1024) {
        double P = 0.;
        int c = 0;
        for (int w = 0; w < p.wgs; ++w) {
            P += p.part_p[int64_t(w) * p.E + e];
            c += p.part_c[int64_t(w) * p.E + e];
        }
        p.counts[e] = c;
        dot += double(c) * P;
    }
    dsum[tid] = dot;
    zred[tid] = z;
    nred[tid] = n;
    __syncthreads();
    for (int o = 512; o >= 1; o >>= 1) {
        if (tid < o) {
            dsum[tid] += dsum[tid + o];
            zred[tid] += zred[tid + o];
            nred[tid] += nred[tid + o];
        }
        __syncthreads();
    }
    if (tid == 0) {
        const double N = nred[0];
        p.stats[0] = N > 0. ? float(double(p.E) * dsum[0] / (N * N * p.k)) : 0.f;
        p.stats[1] = N > 0. ? float(zred[0] / N) : 0.f;
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
            v[i] = expf(v[i] - sv.x) * sv.y;  // p
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
        __builtin_amdgcn_wave_barrier();
        if (id >= 0) row[id] = p.norm ? wdw - w * s : wdw;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const float d = v[i] * (f[i] + sub) + row[lane * NS + i];
            if (lane * NS + i < p.E) store_act(p.dl, LT, t * p.E + lane * NS + i, d);
        }
    }
}

static int route_wgs(int64_t T) {
    const int64_t w = (T + kRouteWaves - 1) / kRouteWaves;
    return int(w < kRouteMaxWgs ? w : kRouteMaxWgs);
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

// Experts per lane: the smallest instance that holds E.
#define VQK_ROUTE_NS(CALL)                                                                      \
    do {                                                                                        \
        if (E <= 64) return CALL(1);                                                            \
        if (E <= 128) return CALL(2);                                                           \
        if (E <= 256) return CALL(4);                                                           \
        if (E <= 512) return CALL(8);                                                           \
        if (E <= 1024) return CALL(16);                                                         \
        return CALL(32);                                                                        \
    } while (0)
template <int LT>
static int route_ns(const RouteArgs &a, bool train, int wgs, hipStream_t st) {
    const int E = a.E;
#define C(NS) go_route<LT, NS>(a, train, wgs, st)
    VQK_ROUTE_NS(C);
#undef C
}
template <int LT>
static int route_bwd_ns(const RouteBwdArgs &a, int wgs, hipStream_t st) {
    const int E = a.E;
#define C(NS) go_route_bwd<LT, NS>(a, wgs, st)
    VQK_ROUTE_NS(C);
#undef C
}

static int check_route(int32_t l_type, int64_t T, int64_t E, int64_t ld, int32_t k, const char *what) {
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
    *bytes = size_t(route_wgs(T)) * (size_t(E) * 8 + 8);
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
    const int wgs = route_wgs(T);
    RouteArgs a{};
    a.l = logits; a.T = T; a.ld = ld;
    a.E = int32_t(E); a.k = top_k; a.norm = norm_topk;
    a.mask = mask; a.ids = ids; a.wts = wts;
    a.saved = reinterpret_cast<float2 *>(saved);
    if (reinterpret_cast<uintptr_t>(saved) & 7) return set_error(VQK_EINVAL, "route: saved must be 8-byte aligned");
    if (train && wgs) {
        const size_t need = size_t(wgs) * (size_t(E) * 8 + 8);
        if (!workspace || ws_bytes < need) return set_error(VQK_ENOSPACE, "route: workspace %zu < %zu", ws_bytes, need);
        if (reinterpret_cast<uintptr_t>(workspace) & 15) return set_error(VQK_EINVAL, "route: workspace must be 16-byte aligned");
        a.part_p = static_cast<float *>(workspace);
        a.part_c = reinterpret_cast<int32_t *>(a.part_p + size_t(wgs) * E);
        a.part_z = reinterpret_cast<float *>(a.part_c + size_t(wgs) * E);
        a.part_n = reinterpret_cast<int32_t *>(a.part_z + wgs);
    }
    if (wgs) {
        switch (l_type) {
            case VQK_F16: rc = route_ns<VQK_F16>(a, train, wgs, st); break;
            case VQK_BF16: rc = route_ns<VQK_BF16>(a, train, wgs, st); break;
            default: rc = route_ns<VQK_F32>(a, train, wgs, st);
        }
        if (rc) return rc;
    }
    if (!train) return VQK_OK;
    const FinishArgs f{a.part_p, a.part_z, a.part_c, a.part_n, wgs, int32_t(E), top_k, counts, stats};
    hipLaunchKernelGGL(k_route_finish, dim3(1), dim3(1024), 0, st, f);
    return hip_status(hipGetLastError(), "router sums launch");
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
    const int64_t w = (T + kRouteWaves - 1) / kRouteWaves;
    const int wgs = int(w < 2048 ? w : 2048);
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (l_type) {
        case VQK_F16: return route_bwd_ns<VQK_F16>(a, wgs, st);
        case VQK_BF16: return route_bwd_ns<VQK_BF16>(a, wgs, st);
        default: return route_bwd_ns<VQK_F32>(a, wgs, st);
    }
}
