// Routing by scores with a bias and groups of experts, with what training it needs:
// tokens per expert, the balance and z losses, the gradient of the logits.
//
//   s = sigmoid(l) or softmax(l),  c = s + bias (the bias alone steers the choice)
//   a group's score: the sum of its group_top (1 or 2) largest c, of the experts that can be chosen
//   ids = the top_k largest c in the top_groups best groups; ties to the lower group, the lower id
//   w = scale s[ids] (norm: scale s / sum of the chosen s)
//   balance = E sum_e c_e / (n k) mean_t p_te,  p = s / sum s;   z = mean_t lse_t^2
// with gradients g_b, g_z and dw, and f_e = g_b E c_e / (n^2 k):
//   u_e = p_e (f_e - sum_i f_i p_i) + [e in ids] (norm: w_e dw_e - w_e / scale sum_j w_j dw_j,
//                                                 else: w_e dw_e)
//   sigmoid: dl_e = (1 - s_e) u_e;  softmax: dl_e = u_e - (norm: 0, else: p_e sum_j w_j dw_j)
//   and 2 g_z / n lse softmax(l)_e
//
// Which of two scores is larger is a question of 64 bits: in 32, one in some
// hundred tokens has two near enough to come out in the other order. The choice
// (choose64) evaluates scores in fp64, a wave a token. From 4096 tokens sixteen lanes
// take a token in fp32 (k_group16) with a bound on its errors, and only tokens with two
// scores closer than that, where it matters, are chosen again by choose64. Without a
// bias experts of equal group are in the order of their logits, which is exact.
// A sigmoid row far below zero (largest logit under -40) has s = e^l to within fp64's
// rounding: its weights and p are a softmax, and nothing divides by a vanishing sum.
// Sums over tokens stay in registers until the wave's last token and meet in a fixed
// order: every result is the same from call to call.
// Bound by instructions: 65536 tokens over 256 experts in 8 groups read 67 MB in 70 us
// (1800 vector instructions for four tokens, issued 65 % of the time at three waves a
// SIMD), the gradient moves twice that in 37 (3.6 TB/s). 64 tokens: 8.9 us, one wave's
// chain of loads, fp64 exponentials, groups and k maxima.
#include "vqk_gemv.h"
#include "vqk_route.h"

namespace vqk {

constexpr int kGroupMaxGroups = 64;
constexpr int kGroup16MaxE = 512, kGroup16MaxK = 15, kGroup16MaxG = 16;   // a lane for the best left out, too
// Tokens from which sixteen lanes take one: choices over 256 experts in 8 groups, us by a
// wave / by sixteen lanes: 2048 tokens 9.0 / 13.0 (a second look's latency), 4096 13.0 / 13.1,
// 8192 20 / 15.5, 16384 39 / 20; over 64 experts 4096 tokens 8.1 / 6.5.
constexpr int64_t kGroup16MinT = 4096;
constexpr float kFarLogit = -40.f;

struct GroupArgs {
    const void *l;
    int64_t T, ld;
    int32_t E, k, norm;
    const uint8_t *mask;
    const float *bias;                        // [E] or NULL
    int32_t G, top_groups, group_top, gs;     // gs = E / G
    float scale;
    int32_t *ids;
    float *wts;
    float4 *saved;                            // [T] (max, 1 / sum exp, 1 / sum sigmoid, 0), or NULL
    float *part_p, *part_z;                   // training: per-workgroup partials [wgs][E] and [wgs]
    int32_t *part_c, *part_n;
};

// 1 / x for x in [1, 2]: the reciprocal instruction and one step of Newton's.
__device__ __forceinline__ float rcp12(float x) {
    const float r = __builtin_amdgcn_rcpf(x);
    return __builtin_fmaf(__builtin_fmaf(-x, r, 1.f), r, r);
}
// sigmoid(l) and 1 - sigmoid(l), both to their own last bits (a NaN stays).
__device__ __forceinline__ float2 sigmoid2(float l) {
    const float e = route_exp(-__builtin_fabsf(l)), r = rcp12(1.f + e);
    return l >= 0.f ? float2{r, e * r} : float2{e * r, r};
}
// The same exponential and sigmoid without a branch and with 0 for a NaN (1 - sigmoid: 1).
__device__ __forceinline__ float exp0(float d) { return route_exp_in(__builtin_fmaxf(d, -200.f)); }
__device__ __forceinline__ float2 sigmoid0(float l) {
    const float e = exp0(-__builtin_fabsf(l)), r = rcp12(1.f + e);
    return float2{(l >= 0.f ? 1.f : e) * r, (l >= 0.f ? e : 1.f) * r};
}
__device__ __forceinline__ float pick(uint32_t mask, float a, float b) {        // bits of a where mask has them, of b elsewhere
    return __uint_as_float((mask & __float_as_uint(a)) | (~mask & __float_as_uint(b)));
}

__device__ __forceinline__ uint64_t f64_key(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.);               // -0 as 0
    return v != v ? 0 : ((b >> 63) ? ~b : (b | (uint64_t(1) << 63)));
}
constexpr uint64_t kKey64NegInf = 0x000fffffffffffffull;                   // f64_key(-inf)

__device__ __forceinline__ double shfl_f64(double v, int from) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __shfl(uint32_t(b), from), hi = __shfl(uint32_t(b >> 32), from);
    return __builtin_bit_cast(double, (uint64_t(hi) << 32) | lo);
}
// From a lane that the whole wave agrees on.
__device__ __forceinline__ uint32_t lane_u32(uint32_t v, int from) { return uint32_t(__builtin_amdgcn_readlane(int(v), from)); }
__device__ __forceinline__ double lane_f64(double v, int from) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t(lane_u32(uint32_t(b >> 32), from)) << 32) | lane_u32(uint32_t(b), from));
}

// The experts' biases as choose64 takes them.
template <int NS>
__device__ __forceinline__ void wave_bias(const GroupArgs &p, int lane, float (&bias)[NS]) {
#pragma unroll
    for (int i = 0; i < NS; ++i) bias[i] = p.bias && lane + 64 * i < p.E ? p.bias[lane + 64 * i] : 0.f;
}

// The choice for one token by a whole wave: lane holds logits v[i] of experts lane +
// 64 i (-inf past E) and their biases, m is the largest; lds: E doubles. Returns the
// lane's choice (lane j the j-th), -1 for none, and its logit. 64 tokens are a matter of
// latency: the lanes share out the groups' experts, and of the wave's reductions only
// the high word's is made unless two lanes hold the same.
template <int NS, bool SIG>
__device__ int choose64(const GroupArgs &p, const float (&v)[NS], const float (&bias)[NS], float m, double *lds, int lane, float *l) {
    double s[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) s[i] = 0.;
    if (p.bias || p.G > 1) {
        double total = 1.;
        if constexpr (!SIG) {
            total = 0.;
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                s[i] = v[i] == v[i] ? exp(double(v[i]) - double(m)) : 0.;
                total += s[i];
            }
            for (int o = 1; o < 64; o <<= 1) total += shfl_f64(total, lane ^ o);
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            s[i] = SIG ? 1. / (1. + exp(-double(v[i]))) : s[i] / total;
            if (p.bias) s[i] += double(bias[i]);
        }
    }
    uint64_t key[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        // a logit of -inf or NaN, a bias of -inf or NaN: never chosen
        const bool can = lane + 64 * i < p.E && v[i] > -__builtin_inff() && s[i] > -__builtin_inf();
        key[i] = can ? f64_key(p.bias ? s[i] : double(v[i])) : 0;
        if (p.G > 1 && lane + 64 * i < p.E) lds[lane + 64 * i] = can ? s[i] : -__builtin_inf();
    }
    if (p.G > 1) {
        const int lg = 31 - __builtin_clz(64 / p.G);        // 2^lg lanes to a group
        const int mine = lane >> lg, part = lane & ((1 << lg) - 1);
        wave_lds_sync();
        double a = -__builtin_inf(), b = a;   // the group's two largest
        if (mine < p.G)
            for (int j = part; j < p.gs; j += 1 << lg) {
                const double c = lds[mine * p.gs + j];
                b = c > a ? a : (c > b ? c : b);
                a = c > a ? c : a;
            }
        for (int o = 1; o < 1 << lg; o <<= 1) {
            const double a2 = shfl_f64(a, lane ^ o), b2 = shfl_f64(b, lane ^ o);
            const double lo = a2 > a ? a : a2;
            b = b2 > b ? b2 : b;
            b = lo > b ? lo : b;
            a = a2 > a ? a2 : a;
        }
        const double sum = p.group_top == 2 && b > -__builtin_inf() ? a + b : a;
        int rank = 0;
        for (int j = 0; j < p.G; ++j) {
            const double o = lane_f64(sum, j << lg);
            rank += o > sum || (o == sum && j < mine);
        }
        const uint64_t kept = __ballot(mine < p.G && rank < p.top_groups);
        wave_lds_sync();
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int e = lane + 64 * i;
            if (e >= p.E || !((kept >> ((e / p.gs) << lg)) & 1)) key[i] = 0;
        }
    }
    int id = -1;
    for (int j = 0; j < p.k; ++j) {
        uint64_t mine = 0;
        int at = 0;
#pragma unroll
        for (int i = NS - 1; i >= 0; --i)
            if (key[i] >= mine) {
                mine = key[i];
                at = i;
            }
        const uint32_t top = wave_max_u32(uint32_t(mine >> 32));
        uint64_t who = __ballot(uint32_t(mine >> 32) == top);
        if (who & (who - 1)) {                // more than one: by the low word, then by the id
            const bool first = uint32_t(mine >> 32) == top;
            const uint32_t low = wave_max_u32(first ? uint32_t(mine) : 0u);
            const bool both = first && uint32_t(mine) == low;
            const int e = int(wave_min_u32(both ? uint32_t(lane + 64 * at) : 0xffffffffu));
            who = __ballot(both && lane + 64 * at == e);
        }
        const int from = __builtin_ctzll(who);
        const uint64_t best = (uint64_t(top) << 32) | lane_u32(uint32_t(mine), from);
        if (best <= kKey64NegInf) break;
        const int e = from + 64 * int(lane_u32(uint32_t(at), from));
        float le = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            if (e >> 6 == i) le = __uint_as_float(lane_u32(__float_as_uint(v[i]), from));
            if (lane + 64 * i == e) key[i] = 0;
        }
        if (lane == j) {
            id = e;
            *l = le;
        }
    }
    return id;
}

// Weight of the choice `id` with logit l (id < 0: 0), from sums over the lanes of a
// token; sum and biggest: reductions over those lanes.
template <bool SIG, typename Sum, typename Big>
__device__ __forceinline__ float group_weight(const GroupArgs &p, int id, float l, float m, float inv, Sum sum, Big biggest) {
    if (p.norm) {
        const float top = biggest(id >= 0 ? l : -__builtin_inff());
        const bool far = !SIG || top < kFarLogit;
        const float e = id < 0 ? 0.f : (far ? route_exp(l - top) : sigmoid2(l).x);
        const float t = sum(e);
        return id < 0 ? 0.f : e / t * p.scale;
    }
    return id < 0 ? 0.f : (SIG ? sigmoid2(l).x : route_exp(l - m) * inv) * p.scale;
}

// ------------------------------------------------------- a wave to a token
// Logits of token t, their largest and whether one is NaN; false: the token is not live.
template <int LT, int NS>
__device__ __forceinline__ bool wave_token(const GroupArgs &p, int64_t t, int lane, float (&v)[NS], float *m, bool *anynan) {
    uint32_t best = 0;
    bool isnan = false;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int e = lane + 64 * i;
        v[i] = e < p.E ? load_act(p.l, LT, t * p.ld + e) : -__builtin_inff();
        isnan = isnan || v[i] != v[i];
        best = max(best, f32_key(v[i]));
    }
    best = wave_max_u32(best);
    *anynan = __ballot(isnan) != 0;
    *m = key_f32(best);
    return (!p.mask || p.mask[t] != 0) && (best > kKeyNegInf || *anynan);
}

// The choice and its weights, written; inv: 1 / sum exp(l - m) where it is known (softmax).
template <int NS, bool SIG>
__device__ __forceinline__ void wave_choose(const GroupArgs &p, int64_t t, int lane, const float (&v)[NS], float m, float inv,
                                            bool anynan, const float (&bias)[NS], double *lds, int32_t *cnt) {
    float l = 0.f;
    const int id = choose64<NS, SIG>(p, v, bias, m, lds, lane, &l);
    float w = group_weight<SIG>(p, id, l, m, inv, [](float x) { return wave_sum(x); }, [](float x) { return wave_max(x); });
    if (anynan) w = __uint_as_float(0x7fc00000u);
    if (lane < p.k) {
        p.ids[t * p.k + lane] = id;
        p.wts[t * p.k + lane] = w;
        if (cnt && id >= 0) atomicAdd(&cnt[id], 1);
    }
}

template <int NS>
__device__ __forceinline__ float wave_total(const float (&v)[NS], float m) {
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i) total += route_exp(v[i] - m);
    return wave_sum(total);
}

template <int LT, int NS, bool SIG, bool TRAIN>
__global__ void __launch_bounds__(kRouteThreads) k_group_wave(const GroupArgs p) {
    extern __shared__ __align__(16) uint8_t smem[];
    double *lds = reinterpret_cast<double *>(smem) + (threadIdx.x >> 6) * p.E;     // [waves][E]
    int32_t *cnt = reinterpret_cast<int32_t *>(smem + kRouteWaves * 8 * size_t(p.E));   // TRAIN: [E], [E]
    float *psh = reinterpret_cast<float *>(cnt + p.E);
    __shared__ float zsh[kRouteWaves];
    __shared__ int nsh[kRouteWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if constexpr (TRAIN) {
        for (int e = threadIdx.x; e < p.E; e += kRouteThreads) cnt[e] = 0;
        __syncthreads();
    }
    float bias[NS], psum[NS] = {};
    wave_bias(p, lane, bias);
    float zsum = 0.f;
    int live = 0;
    for (int64_t t = int64_t(blockIdx.x) * kRouteWaves + wave; t < p.T; t += int64_t(gridDim.x) * kRouteWaves) {
        float v[NS], m;
        bool anynan;
        if (!wave_token<LT>(p, t, lane, v, &m, &anynan)) {
            if (lane < p.k) {
                p.ids[t * p.k + lane] = -1;
                p.wts[t * p.k + lane] = 0.f;
            }
            if (p.saved && lane == 0) p.saved[t] = float4{0.f, 0.f, 0.f, 0.f};
            continue;
        }
        float total = 0.f, inv = 0.f, sums = 0.f;
        if constexpr (!SIG || TRAIN) {
            total = wave_total(v, m);
            inv = 1.f / total;
        }
        wave_choose<NS, SIG>(p, t, lane, v, m, inv, anynan, bias, lds, TRAIN ? cnt : nullptr);
        if constexpr (TRAIN) {
            const float lse = m + logf(total);
            zsum += lse * lse;
            ++live;
            const bool far = !SIG || m < kFarLogit;
            float f = inv;
            if (!far) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < NS; ++i) s += sigmoid2(v[i]).x;
                sums = f = 1.f / wave_sum(s);
            }
#pragma unroll
            for (int i = 0; i < NS; ++i) psum[i] += (far ? route_exp(v[i] - m) : sigmoid2(v[i]).x) * f;
        }
        if (p.saved && lane == 0) p.saved[t] = float4{m, inv, sums, 0.f};
    }
    if constexpr (TRAIN) {
        for (int w = 0; w < kRouteWaves; ++w) {             // the waves' sums in wave order
            if (wave == w) {
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    const int e = lane + 64 * i;
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

// Logits expert(i) of the row at `base`, -inf for those past E and where the token is not
// `in` (base: 0): whole, aligned fours fetched and later turned into values, or one by
// one. All loads are issued before the first is used: an address past the row is replaced
// by the row's own start.
template <int LT> using RowFour = std::conditional_t<LT == VQK_F32, u32x4, u32x2>;
template <int LT, int NS, typename Expert>
__device__ __forceinline__ void row_fetch(const void *l, int64_t base, int E, Expert expert, RowFour<LT> (&f)[NS / 4]) {
    using T = std::conditional_t<LT == VQK_F32, float, uint16_t>;
    const T *row = static_cast<const T *>(l) + base;
#pragma unroll
    for (int q = 0; q < NS / 4; ++q) {
        const int e = expert(4 * q);
        f[q] = *reinterpret_cast<const RowFour<LT> *>(row + (e < E ? e : 0));
    }
}
template <int LT, int NS, typename Expert>
__device__ __forceinline__ void row_values(const RowFour<LT> (&f)[NS / 4], int E, bool in, Expert expert, float (&v)[NS]) {
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const RowFour<LT> w = f[i / 4];
        if constexpr (LT == VQK_F32) {
            v[i] = __uint_as_float(w[i % 4]);
        } else {
            const uint16_t h = uint16_t(w[i % 4 / 2] >> (16 * (i & 1)));
            v[i] = LT == VQK_BF16 ? bf16_to_f32(h) : h_to_f32(h);
        }
        v[i] = in && expert(i / 4 * 4) < E ? v[i] : -__builtin_inff();
    }
}
template <int LT, int NS, typename Expert>
__device__ __forceinline__ void row_each(const void *l, int64_t base, int E, bool in, Expert expert, float (&v)[NS]) {
    using T = std::conditional_t<LT == VQK_F32, float, uint16_t>;
    const T *row = static_cast<const T *>(l) + base;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int e = expert(i);
        v[i] = load_act(row, LT, e < E ? e : 0);
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) v[i] = in && expert(i) < E ? v[i] : -__builtin_inff();
}

// ------------------------------------------------- sixteen lanes to a token
// Bounds of what fp32 may get wrong in a comparison of two c (smax: the row's
// largest s): a sigmoid is 4 units of 2^-23 off at most, a softmax 2^-18 of itself
// (its sum adds up E terms, 32 in a lane), the sum with the bias half a unit. An
// exponential below 2^-126 comes out as 0, which costs a sigmoid up to that much whatever
// smax is: four times it, two scores to a group's sum on each side of the comparison.
template <bool SIG>
__device__ __forceinline__ float group_tol(float smax, float c) {
    return (SIG ? __builtin_fmaf(0x1p-19f, smax, 0x1p-124f) : 0x1p-16f * smax) + 0x1p-21f * __builtin_fabsf(c);
}

// Lane `sub` of a token holds in value 4 q + j expert 64 q + 4 ((sub + 4 q) % 16) + j:
// whole lines a load, and the lanes of a group shift from one 64 to the next, so that
// the experts of few groups are not all in the same lanes.
__device__ __forceinline__ int group16_expert(int i, int sub) { return 64 * (i / 4) + 4 * ((sub + i / 4 * 4) & 15) + i % 4; }
// The top k as in k_route16: the k-th largest lane maximum bounds them from below,
// what reaches it is collected in LDS and ranked, two candidates a lane. One more than
// top_k is looked at: the best that is left out.
constexpr int kSecondLook = -2;                // ids[t][0] of a token that choose64 is to choose for

template <int LT, int NS, bool SIG, bool TRAIN>
__global__ void __launch_bounds__(kRouteThreads, NS <= 16 ? 3 : 1) k_group16(const GroupArgs p, bool vec) {
    extern __shared__ __align__(16) uint8_t smem[];
    // [waves]: four tokens' scores, as floats or the two largest of every four; choose64: E doubles
    float *csh = reinterpret_cast<float *>(smem) + (threadIdx.x >> 6) * 64 * NS;
    int32_t *cnt = reinterpret_cast<int32_t *>(smem + kRouteWaves * 256 * NS);           // TRAIN: [16 NS], [16 NS]
    float *psh = reinterpret_cast<float *>(cnt + 16 * NS);
    __shared__ __align__(16) float bsh[16 * NS];
    __shared__ uint64_t cands[kRouteWaves][4][kRouteCands];
    __shared__ uint64_t sel[kRouteWaves][4][kGroup16MaxK + 1];
    __shared__ float zsh[kRouteWaves];
    __shared__ int nsh[kRouteWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sub0 = lane & 15, grp = lane >> 4;
    if constexpr (TRAIN) {
        for (int e = threadIdx.x; e < 16 * NS; e += kRouteThreads) {
            cnt[e] = 0;
            psh[e] = 0.f;
        }
        __syncthreads();
    }
    // experts past E have logits of -inf: whatever their bias and group, they are not chosen
    for (int e = threadIdx.x; e < 16 * NS; e += kRouteThreads) bsh[e] = p.bias ? p.bias[min(e, p.E - 1)] : 0.f;
    __syncthreads();
    uint32_t gid[NS / 4] = {};                // the experts' groups, four to a word
    const uint32_t per = ((1u << 20) + p.gs - 1) / p.gs;    // e / gs = e per >> 20: e and gs are at most 512
#pragma unroll
    for (int i = 0; i < NS; ++i) gid[i / 4] |= (uint32_t(group16_expert(i, sub0)) * per >> 20) << (8 * (i % 4));
    const bool fours = p.gs % 4 == 0;
    float psum[NS] = {};
    float zsum = 0.f;
    int nlive = 0;
    const int64_t t00 = (int64_t(blockIdx.x) * kRouteWaves + wave) * 4, stride = int64_t(gridDim.x) * kRouteWaves * 4;
    // the next four tokens' logits are on their way while these are ranked
    RowFour<LT> ahead[NS / 4];
    bool in_next = false;
    auto fetch = [&](int64_t t0, int sub, int E) {
        const int64_t t = t0 + grp;
        in_next = t < p.T && (!p.mask || p.mask[t] != 0);
        if (vec) row_fetch<LT, NS>(p.l, in_next ? t * p.ld : 0, E, [=](int i) { return group16_expert(i, sub); }, ahead);
    };
    fetch(t00, sub0, p.E);                    // past the last token: the first row's
    for (int64_t t0 = t00; t0 < p.T; t0 += stride) {
        const int64_t t = t0 + grp;
        float v[NS], c[NS];
        int E = p.E, sub = sub0;
        asm volatile("" : "+s"(E), "+v"(sub));              // masks and places made anew: kept over the loop they spill
        const bool in = in_next;
        const auto expert = [=](int i) { return group16_expert(i, sub); };
        if (vec) row_values<LT, NS>(ahead, E, in, expert, v);
        else row_each<LT, NS>(p.l, in ? t * p.ld : 0, E, in, expert, v);
        fetch(t0 + stride, sub, E);
        float best = -__builtin_inff();
        bool isnan = false;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            isnan = isnan || v[i] != v[i];
            best = fmaxf(best, v[i]);         // of a NaN and a number the number
        }
        best = key_f32(row_max(f32_key(best)));
        const bool anynan = ((__ballot(isnan) >> (grp * 16)) & 0xffffu) != 0;
        const bool live = in && (best > -__builtin_inff() || anynan);
        const float m = best > -__builtin_inff() ? best : 0.f;
        const bool far = !SIG || m < kFarLogit;             // p: a softmax
        float lse = 0.f, inv = 0.f, sums = 0.f;
        if constexpr (!SIG) {
            float total = 0.f;
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                c[i] = exp0(v[i] - m);
                total += c[i];
            }
            total = row_sum(total);
            inv = live ? 1.f / total : 0.f;
            lse = m + logf(total);
            const float f = anynan && live ? __uint_as_float(0x7fc00000u) : inv;
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                if constexpr (TRAIN) psum[i] = __builtin_fmaf(c[i], f, psum[i]);
                c[i] *= inv;
            }
        } else {
            // e^l of the sigmoid's own e^-|l|, unless a row's largest is too far from 0 for its sum
            float total = 0.f, s = 0.f;
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const float e = exp0(-__builtin_fabsf(v[i])), x = rcp12(1.f + e);
                const bool up = v[i] >= 0.f;
                c[i] = (up ? 1.f : e) * x;
                if constexpr (TRAIN) {
                    s += c[i];
                    total += up ? __builtin_amdgcn_rcpf(e) : e;
                }
            }
            if constexpr (TRAIN) {
                const bool odd = live && !(__builtin_fabsf(m) < -kFarLogit);
                sums = live && !far ? 1.f / row_sum(s) : 0.f;
                if (__ballot(odd) == 0) {
                    total = row_sum(total);
                    const float em = exp0(-__builtin_fabsf(m));
                    inv = live ? (m >= 0.f ? 1.f : em) / (total * (m >= 0.f ? em : 1.f)) : 0.f;
                    lse = logf(total);
                    sums = anynan && live ? __uint_as_float(0x7fc00000u) : sums;
#pragma unroll
                    for (int i = 0; i < NS; ++i) psum[i] = __builtin_fmaf(c[i], sums, psum[i]);
                } else {
                    total = 0.f;
#pragma unroll
                    for (int i = 0; i < NS; ++i) total += exp0(v[i] - m);
                    total = row_sum(total);
                    inv = live ? 1.f / total : 0.f;
                    lse = m + logf(total);
                    float f = far ? inv : sums;             // 0 where the token is not live
                    f = anynan && live ? __uint_as_float(0x7fc00000u) : f;
#pragma unroll
                    for (int i = 0; i < NS; ++i) psum[i] = __builtin_fmaf(far ? exp0(v[i] - m) : c[i], f, psum[i]);
                }
            }
        }
        const float smax = SIG ? sigmoid2(m).x : inv;
        if (anynan) lse = inv = sums = __uint_as_float(live ? 0x7fc00000u : 0u);
        if constexpr (TRAIN) {
            zsum += live && sub == 0 ? lse * lse : 0.f;
            nlive += live && sub == 0;
        }
        float bias[NS];
#pragma unroll
        for (int q = 0; q < NS / 4; ++q)
            *reinterpret_cast<float4 *>(bias + 4 * q) = *reinterpret_cast<const float4 *>(bsh + group16_expert(4 * q, sub));
        uint32_t key[NS], lm = 0;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            c[i] += bias[i];
            const bool can = live && v[i] > -__builtin_inff() && c[i] > -__builtin_inff();
            const uint32_t b = __float_as_uint((p.bias ? c[i] : v[i]) + 0.f);      // -0 as 0
            key[i] = can ? b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u) : 0u;    // f32_key of a number
            c[i] = can ? c[i] : -__builtin_inff();
        }
        bool amb = false;                                   // fp32 does not say which is larger
        if (p.G > 1) {
            float a = -__builtin_inff(), b = a;             // the group's two largest
            wave_lds_sync();                                // the last tokens' scores are read
            if (fours) {
                float2 *mine = reinterpret_cast<float2 *>(csh) + grp * 4 * NS;
#pragma unroll
                for (int w = 0; w < NS / 4; ++w) {
                    const float hi0 = fmaxf(c[4 * w], c[4 * w + 1]), lo0 = fminf(c[4 * w], c[4 * w + 1]);
                    const float hi1 = fmaxf(c[4 * w + 2], c[4 * w + 3]), lo1 = fminf(c[4 * w + 2], c[4 * w + 3]);
                    mine[group16_expert(4 * w, sub) / 4] = float2{fmaxf(hi0, hi1), fmaxf(fminf(hi0, hi1), fmaxf(lo0, lo1))};
                }
                wave_lds_sync();
                if (sub < p.G) {
                    const int n = p.gs / 4;
                    int at = sub % n;                       // lanes start at banks of their own
                    for (int j = 0; j < n; ++j) {
                        const float2 x = mine[sub * n + at];
                        at = at + 1 == n ? 0 : at + 1;
                        b = fmaxf(fmaxf(b, x.y), fminf(a, x.x));
                        a = fmaxf(a, x.x);
                    }
                }
            } else {
                float *mine = csh + grp * 16 * NS;
#pragma unroll
                for (int i = 0; i < NS; ++i) mine[group16_expert(i, sub)] = c[i];
                wave_lds_sync();
                if (sub < p.G) {
                    int at = sub % p.gs;
                    for (int j = 0; j < p.gs; ++j) {
                        const float x = mine[sub * p.gs + at];
                        at = at + 1 == p.gs ? 0 : at + 1;
                        b = fmaxf(b, fminf(a, x));
                        a = fmaxf(a, x);
                    }
                }
            }
            const float g = p.group_top == 2 && b > -__builtin_inff() ? a + b : a;
            const uint32_t gk = sub < p.G ? f32_key(g) : 0u;
            const uint64_t gl = (uint64_t(gk) << 32) | uint32_t(15 - sub);
            int rank = 0;
#define VQK_ROR(N) rank += dpp_u64<0x120 + N>(gl) > gl;
            VQK_ROR(1) VQK_ROR(2) VQK_ROR(3) VQK_ROR(4) VQK_ROR(5) VQK_ROR(6) VQK_ROR(7) VQK_ROR(8)
            VQK_ROR(9) VQK_ROR(10) VQK_ROR(11) VQK_ROR(12) VQK_ROR(13) VQK_ROR(14) VQK_ROR(15)
#undef VQK_ROR
            const bool keep = sub < p.G && rank < p.top_groups;
            const uint32_t kept = uint32_t(__ballot(keep) >> (grp * 16)) & 0xffffu;
            const uint32_t worst = row_min(keep ? gk : 0xffffffffu), next = row_max(sub < p.G && !keep ? gk : 0u);
            // of a sum each part is as far off as c may be
            const float mag = p.group_top == 2 ? __builtin_fabsf(a) + (b > -__builtin_inff() ? __builtin_fabsf(b) : 0.f) : __builtin_fabsf(a);
            const float most = key_f32(row_max(sub < p.G && a > -__builtin_inff() ? f32_key(mag) : f32_key(0.f)));
            if (next > kKeyNegInf) amb = !(key_f32(worst) - key_f32(next) > 4.f * group_tol<SIG>(smax, most));
#pragma unroll
            for (int i = 0; i < NS; ++i) key[i] &= uint32_t(-int32_t((kept >> ((gid[i / 4] >> (8 * (i % 4))) & 31u)) & 1u));
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) lm = max(lm, key[i]);
        // the k-th largest lane maximum; with a bias one rank further, so that the best left out is a
        // candidate too
        const int want = p.bias ? p.k + 1 : p.k;
        int rank = 0;
#define VQK_ROR(N) rank += dpp_u<0x120 + N>(lm) > lm;
        VQK_ROR(1) VQK_ROR(2) VQK_ROR(3) VQK_ROR(4) VQK_ROR(5) VQK_ROR(6) VQK_ROR(7) VQK_ROR(8)
        VQK_ROR(9) VQK_ROR(10) VQK_ROR(11) VQK_ROR(12) VQK_ROR(13) VQK_ROR(14) VQK_ROR(15)
#undef VQK_ROR
        const uint32_t thr = max(row_min(rank < want ? lm : 0xffffffffu), kKeyNegInf + 1);
        int mine = 0;                                       // this lane's candidates, and those of the lanes before
#pragma unroll
        for (int i = 0; i < NS; ++i) mine += key[i] >= thr;
        int upto = mine;
        upto += int(__builtin_amdgcn_update_dpp(0, upto, 0x111, 0xf, 0xf, true));           // row_shr:1, zeros in
        upto += int(__builtin_amdgcn_update_dpp(0, upto, 0x112, 0xf, 0xf, true));
        upto += int(__builtin_amdgcn_update_dpp(0, upto, 0x114, 0xf, 0xf, true));
        upto += int(__builtin_amdgcn_update_dpp(0, upto, 0x118, 0xf, 0xf, true));
        const int run = int(row_max(uint32_t(upto)));
        int pos = upto - mine;
        wave_lds_sync();                                    // the last token's candidates are read
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (key[i] >= thr) {
                if (pos < kRouteCands) cands[wave][grp][pos] = (uint64_t(key[i]) << 32) | uint32_t(~group16_expert(i, sub));
                ++pos;
            }
        if (sub <= p.k) sel[wave][grp][sub] = 0;
        wave_lds_sync();
        const uint64_t c0 = sub < run ? cands[wave][grp][sub] : 0;
        int r0 = 0;
        if (__ballot(run > 16) == 0) {
#define VQK_ROR(N) r0 += dpp_u64<0x120 + N>(c0) > c0;
            VQK_ROR(1) VQK_ROR(2) VQK_ROR(3) VQK_ROR(4) VQK_ROR(5) VQK_ROR(6) VQK_ROR(7) VQK_ROR(8)
            VQK_ROR(9) VQK_ROR(10) VQK_ROR(11) VQK_ROR(12) VQK_ROR(13) VQK_ROR(14) VQK_ROR(15)
#undef VQK_ROR
        } else {
            const uint64_t c1 = sub + 16 < run && sub + 16 < kRouteCands ? cands[wave][grp][sub + 16] : 0;
            r0 = c1 > c0;
            int r1 = c0 > c1;
#define VQK_ROR(N)                                                                              \
    {                                                                                           \
        const uint64_t a = dpp_u64<0x120 + N>(c0), b = dpp_u64<0x120 + N>(c1);                  \
        r0 += int(a > c0) + int(b > c0);                                                        \
        r1 += int(a > c1) + int(b > c1);                                                        \
    }
            VQK_ROR(1) VQK_ROR(2) VQK_ROR(3) VQK_ROR(4) VQK_ROR(5) VQK_ROR(6) VQK_ROR(7) VQK_ROR(8)
            VQK_ROR(9) VQK_ROR(10) VQK_ROR(11) VQK_ROR(12) VQK_ROR(13) VQK_ROR(14) VQK_ROR(15)
#undef VQK_ROR
            if (c1 != 0 && r1 <= p.k) sel[wave][grp][r1] = c1;
        }
        if (c0 != 0 && r0 <= p.k) sel[wave][grp][r0] = c0;
        wave_lds_sync();
        const uint64_t got = sub < p.k ? sel[wave][grp][sub] : 0, next = sub < p.k ? sel[wave][grp][sub + 1] : 0;
        const int id = got ? int(~uint32_t(got)) : -1;
        const float l = id >= 0 ? load_act(p.l, LT, t * p.ld + id) : 0.f;
        if (p.bias) {
            bool near = false;
            if (next) {
                // equal logits under equal biases are a tie, and the lower id comes first already
                const int e = int(~uint32_t(next));
                const float x = key_f32(uint32_t(got >> 32)), y = key_f32(uint32_t(next >> 32));
                near = !(x - y > 2.f * group_tol<SIG>(smax, x)) &&
                       !(l == load_act(p.l, LT, t * p.ld + e) && p.bias[id] == p.bias[e]);
            }
            amb = amb || ((__ballot(near) >> (grp * 16)) & 0xffffu) != 0;
        }
        amb = live && (amb || run > kRouteCands);
        float w = group_weight<SIG>(p, id, l, m, inv, [](float x) { return row_sum(x); },
                                    [](float x) { return key_f32(row_max(f32_key(x))); });
        if (anynan && live) w = __uint_as_float(0x7fc00000u);
        if (t < p.T && sub < p.k) {
            p.ids[t * p.k + sub] = amb ? kSecondLook : id;
            p.wts[t * p.k + sub] = w;
            if (TRAIN && id >= 0 && !amb) atomicAdd(&cnt[id], 1);
        }
        if (p.saved && t < p.T && sub == 0) p.saved[t] = live ? float4{m, inv, sums, 0.f} : float4{0.f, 0.f, 0.f, 0.f};
    }
    if constexpr (TRAIN) {
        for (int w = 0; w < kRouteWaves * 4; ++w) {         // the tokens' sums in order of wave and row of lanes
            if (wave == w / 4 && grp == w % 4) {
#pragma unroll
                for (int i = 0; i < NS; ++i) psh[group16_expert(i, sub0)] += psum[i];
            }
            if (w % 4 == 3) __syncthreads();
            else wave_lds_sync();
        }
    }
    // the second look, at this wave's own tokens
    __syncthreads();
    for (int64_t t0 = t00; t0 < p.T; t0 += stride) {
        const uint64_t again = __ballot(sub0 == 0 && t0 + grp < p.T && p.ids[(t0 + grp) * p.k] == kSecondLook);
        for (int g = 0; g < 4; ++g) {
            if (!((again >> (16 * g)) & 1)) continue;
            float v[NS / 4], near[NS / 4], m;
            bool anynan;
            wave_token<LT>(p, t0 + g, lane, v, &m, &anynan);
            wave_bias(p, lane, near);
            wave_lds_sync();
            wave_choose<NS / 4, SIG>(p, t0 + g, lane, v, m, SIG ? 0.f : 1.f / wave_total(v, m), anynan, near,
                                     reinterpret_cast<double *>(csh), TRAIN ? cnt : nullptr);
        }
    }
    if constexpr (TRAIN) {
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

// ---------------------------------------------------------------- gradient
struct GroupBwdArgs {
    const void *l;
    int64_t T, ld;
    int32_t E, k, norm;
    float scale;
    const int32_t *ids, *counts;
    const float *wts, *stats;
    const float4 *saved;
    const float *dw, *gb, *gz;                // NULL: no gradient of that output
    void *dl;
};

// L = 16 lanes to a token (four a wave) or 64; lane `sub` holds experts 4 L q + 4 sub + j.
template <int LT, int NS, int L, bool SIG>
__global__ void __launch_bounds__(kRouteThreads) k_group_bwd(const GroupBwdArgs p, bool vec) {
    extern __shared__ __align__(16) float rows[];           // [waves][64 / L][L * NS]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sub = lane % L, grp = lane / L;
    float *row = rows + (wave * (64 / L) + grp) * (L * NS);
    const float n = p.stats[2];
    const float fb = p.gb && n > 0.f ? p.gb[0] * (float(p.E) / (n * n * float(p.k))) : 0.f;
    const float fz = p.gz && n > 0.f ? 2.f * p.gz[0] / n : 0.f;
    auto sum = [](float x) { return L == 16 ? row_sum(x) : wave_sum(x); };
    float f[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int e = 4 * L * (i / 4) + 4 * sub + i % 4;
        f[i] = e < p.E ? fb * float(p.counts[e]) : 0.f;
    }
    const int64_t stride = int64_t(gridDim.x) * kRouteWaves * (64 / L);
    for (int64_t t0 = (int64_t(blockIdx.x) * kRouteWaves + wave) * (64 / L); t0 < p.T; t0 += stride) {
        const int64_t t = t0 + grp;
        const bool in = t < p.T;
        const float4 sv = in ? p.saved[t] : float4{0.f, 0.f, 0.f, 0.f};
        const bool live = sv.y != 0.f;        // a live token's sum is at most E
        float v[NS];
        const auto expert = [=](int i) { return 4 * L * (i / 4) + 4 * sub + i % 4; };
        if (vec) {
            RowFour<LT> f4[NS / 4];
            row_fetch<LT, NS>(p.l, live ? t * p.ld : 0, p.E, expert, f4);
            row_values<LT, NS>(f4, p.E, live, expert, v);
        } else {
            row_each<LT, NS>(p.l, live ? t * p.ld : 0, p.E, live, expert, v);
        }
        int id = -1;
        float wdw = 0.f, w = 0.f;
        if (p.dw && live && sub < p.k) {
            id = p.ids[t * p.k + sub];
            w = p.wts[t * p.k + sub];
            wdw = id >= 0 ? w * p.dw[t * p.k + sub] : 0.f;
        }
        const float s = sum(wdw);
        const float lse = sv.x - logf(sv.y);
        const bool far = !SIG || sv.x < kFarLogit;
        const uint32_t fm = far ? 0xffffffffu : 0u;
        // softmax, p and 1 - sigmoid; a token that is not live has sums of 0 and logits of -inf
        float x[NS], pr[SIG ? NS : 1], to1[SIG ? NS : 1];
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            x[i] = exp0(v[i] - sv.x) * sv.y;
            if constexpr (SIG) {
                const float2 g = sigmoid0(v[i]);
                pr[i] = pick(fm, x[i], g.x * sv.z);
                to1[i] = g.y;
            }
            dot += f[i] * (SIG ? pr[SIG ? i : 0] : x[i]);
        }
        dot = sum(dot);
        const float sub_ = fz * lse - (SIG || p.norm ? 0.f : s);
#pragma unroll
        for (int q = 0; q < NS / 4; ++q) *reinterpret_cast<float4 *>(row + 4 * L * q + 4 * sub) = float4{0.f, 0.f, 0.f, 0.f};
        wave_lds_sync();
        if (id >= 0) row[id] = p.norm ? wdw - w / p.scale * s : wdw;
        wave_lds_sync();
#pragma unroll
        for (int q = 0; q < NS / 4; ++q) {
            const int e = 4 * L * q + 4 * sub;
            const float4 a = *reinterpret_cast<const float4 *>(row + e);
            const float add[4] = {a.x, a.y, a.z, a.w};
            float d[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = 4 * q + j;
                if constexpr (SIG) d[j] = to1[i] * (pr[i] * (f[i] - dot) + add[j]) + x[i] * sub_;
                else d[j] = x[i] * (f[i] - dot + sub_) + add[j];
                d[j] = live ? d[j] : 0.f;
            }
            if (!in || e >= p.E) continue;
            if (vec) {
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

// ------------------------------------------------------------------ launch
static bool group16_ok(int64_t T, int64_t E, int k, int G) {
    return T >= kGroup16MinT && E <= kGroup16MaxE && k <= kGroup16MaxK && G <= kGroup16MaxG;
}

template <int LT, int NS, bool SIG>
static int go_wave(const GroupArgs &a, bool train, int wgs, hipStream_t st) {
    const size_t lds = kRouteWaves * 8 * size_t(a.E) + (train ? 8 * size_t(a.E) : 0);
    if (train) return launch_with_lds<k_group_wave<LT, NS, SIG, true>>(dim3(wgs), dim3(kRouteThreads), lds, st, a);
    return launch_with_lds<k_group_wave<LT, NS, SIG, false>>(dim3(wgs), dim3(kRouteThreads), lds, st, a);
}
template <int LT, int NS, bool SIG>
static int go_16(const GroupArgs &a, bool train, int wgs, hipStream_t st) {
    const size_t lds = kRouteWaves * 256 * NS + (train ? 128 * NS : 0);
    const bool vec = route_vec(a.l, a.ld, a.E, LT);
    if (train) hipLaunchKernelGGL((k_group16<LT, NS, SIG, true>), dim3(wgs), dim3(kRouteThreads), lds, st, a, vec);
    else hipLaunchKernelGGL((k_group16<LT, NS, SIG, false>), dim3(wgs), dim3(kRouteThreads), lds, st, a, vec);
    return hip_status(hipGetLastError(), "router launch");
}
template <int LT, bool SIG>
static int go_group(const GroupArgs &a, bool train, int wgs, hipStream_t st) {
    const int E = a.E;
    if (group16_ok(a.T, E, a.k, a.G)) {
        if (E <= 64) return go_16<LT, 4, SIG>(a, train, wgs, st);
        if (E <= 128) return go_16<LT, 8, SIG>(a, train, wgs, st);
        if (E <= 192) return go_16<LT, 12, SIG>(a, train, wgs, st);
        if (E <= 256) return go_16<LT, 16, SIG>(a, train, wgs, st);
        if (E <= 384) return go_16<LT, 24, SIG>(a, train, wgs, st);
        return go_16<LT, 32, SIG>(a, train, wgs, st);
    }
    if (E <= 64) return go_wave<LT, 1, SIG>(a, train, wgs, st);
    if (E <= 128) return go_wave<LT, 2, SIG>(a, train, wgs, st);
    if (E <= 256) return go_wave<LT, 4, SIG>(a, train, wgs, st);
    if (E <= 512) return go_wave<LT, 8, SIG>(a, train, wgs, st);
    if (E <= 1024) return go_wave<LT, 16, SIG>(a, train, wgs, st);
    return go_wave<LT, 32, SIG>(a, train, wgs, st);
}

template <int LT, int NS, int L, bool SIG>
static int go_bwd(const GroupBwdArgs &a, int wgs, hipStream_t st) {
    const bool vec = route_vec(a.l, a.ld, a.E, LT) && (reinterpret_cast<uintptr_t>(a.dl) & 15) == 0;
    hipLaunchKernelGGL((k_group_bwd<LT, NS, L, SIG>), dim3(wgs), dim3(kRouteThreads), kRouteWaves * 64 * NS * 4, st, a, vec);
    return hip_status(hipGetLastError(), "router gradient launch");
}
template <int LT, bool SIG>
static int go_group_bwd(const GroupBwdArgs &a, bool rows16, int wgs, hipStream_t st) {
    const int E = a.E;
    if (rows16) {
        if (E <= 64) return go_bwd<LT, 4, 16, SIG>(a, wgs, st);
        if (E <= 128) return go_bwd<LT, 8, 16, SIG>(a, wgs, st);
        if (E <= 192) return go_bwd<LT, 12, 16, SIG>(a, wgs, st);
        if (E <= 256) return go_bwd<LT, 16, 16, SIG>(a, wgs, st);
        if (E <= 384) return go_bwd<LT, 24, 16, SIG>(a, wgs, st);
        return go_bwd<LT, 32, 16, SIG>(a, wgs, st);
    }
    if (E <= 256) return go_bwd<LT, 4, 64, SIG>(a, wgs, st);
    if (E <= 512) return go_bwd<LT, 8, 64, SIG>(a, wgs, st);
    if (E <= 1024) return go_bwd<LT, 16, 64, SIG>(a, wgs, st);
    return go_bwd<LT, 32, 64, SIG>(a, wgs, st);
}

static int check_form(const vqk_route_form *f, int64_t E, int32_t k, const char *what) {
    if (!f) return set_error(VQK_EINVAL, "%s: NULL form", what);
    if (f->score != VQK_SCORE_SOFTMAX && f->score != VQK_SCORE_SIGMOID) return set_error(VQK_EINVAL, "%s: score %d", what, f->score);
    if (f->groups < 1 || E % f->groups || f->top_groups < 1 || f->top_groups > f->groups)
        return set_error(VQK_EINVAL, "%s: %d of %d groups of %lld experts", what, f->top_groups, f->groups, (long long)E);
    if (f->groups > kGroupMaxGroups) return set_error(VQK_ENOTIMPL, "%s: %d groups > %d", what, f->groups, kGroupMaxGroups);
    if (f->group_top != 1 && f->group_top != 2) return set_error(VQK_ENOTIMPL, "%s: a group's score from %d experts", what, f->group_top);
    if (int64_t(k) > f->top_groups * (E / f->groups))
        return set_error(VQK_EINVAL, "%s: top_k=%d of %lld experts in %d groups", what, k, (long long)(f->top_groups * (E / f->groups)), f->top_groups);
    if (!(f->scale > 0.f) || f->scale > 3.4028234e38f) return set_error(VQK_EINVAL, "%s: scale %g", what, double(f->scale));
    return VQK_OK;
}

}  // namespace vqk

using namespace vqk;

extern "C" int vqk_route_grouped(const void *logits, int32_t l_type, int64_t T, int64_t E, int64_t ld,
                                 const uint8_t *mask, const vqk_route_form *form, int32_t top_k, int32_t norm_topk,
                                 int32_t *ids, float *wts, int32_t *counts, float *stats, float *saved, void *workspace,
                                 size_t ws_bytes, void *stream) {
    int rc = check_route(l_type, T, E, ld, top_k, "route");
    if (rc || (rc = check_form(form, E, top_k, "route"))) return rc;
    const bool train = counts || stats;
    if (train && (!counts || !stats)) return set_error(VQK_EINVAL, "route: counts and stats come together");
    if (T > 0 && (!logits || !ids || !wts)) return set_error(VQK_EINVAL, "route: NULL pointer");
    if (reinterpret_cast<uintptr_t>(saved) & 15) return set_error(VQK_EINVAL, "route: saved must be 16-byte aligned");
    hipStream_t st = static_cast<hipStream_t>(stream);
    GroupArgs a{};
    a.l = logits; a.T = T; a.ld = ld;
    a.E = int32_t(E); a.k = top_k; a.norm = norm_topk;
    a.mask = mask; a.bias = form->bias;
    a.G = form->groups; a.top_groups = form->top_groups; a.group_top = form->group_top; a.gs = int32_t(E / form->groups);
    if (a.top_groups == a.G) a.G = a.top_groups = 1, a.gs = int32_t(E);       // every group is kept
    a.scale = form->scale;
    a.ids = ids; a.wts = wts;
    a.saved = reinterpret_cast<float4 *>(saved);
    const int wgs = route_wgs_of(T, group16_ok(T, E, top_k, a.G) ? 4 * kRouteWaves : kRouteWaves);
    FinishArgs f{};
    if (train) {
        const size_t need = route_bytes(T, E);
        if (!workspace || ws_bytes < need) return set_error(VQK_ENOSPACE, "route: workspace %zu < %zu", ws_bytes, need);
        if (reinterpret_cast<uintptr_t>(workspace) & 15) return set_error(VQK_EINVAL, "route: workspace must be 16-byte aligned");
        route_parts(workspace, E, wgs, &f, &a.part_p, &a.part_c, &a.part_z, &a.part_n);
        f.k = top_k; f.counts = counts; f.stats = stats;
    }
    if (wgs) {
        const bool sig = form->score == VQK_SCORE_SIGMOID;
        switch (l_type) {
            case VQK_F16: rc = sig ? go_group<VQK_F16, true>(a, train, wgs, st) : go_group<VQK_F16, false>(a, train, wgs, st); break;
            case VQK_BF16: rc = sig ? go_group<VQK_BF16, true>(a, train, wgs, st) : go_group<VQK_BF16, false>(a, train, wgs, st); break;
            default: rc = sig ? go_group<VQK_F32, true>(a, train, wgs, st) : go_group<VQK_F32, false>(a, train, wgs, st);
        }
        if (rc) return rc;
    }
    return train ? route_finish(f, st) : VQK_OK;
}

extern "C" int vqk_route_grouped_backward(const void *logits, int32_t l_type, int64_t T, int64_t E, int64_t ld,
                                          const vqk_route_form *form, int32_t top_k, int32_t norm_topk,
                                          const int32_t *ids, const float *wts, const int32_t *counts,
                                          const float *stats, const float *saved, const float *dw,
                                          const float *dbalance, const float *dz, void *dlogits, void *stream) {
    int rc = check_route(l_type, T, E, ld, top_k, "route backward");
    if (rc || (rc = check_form(form, E, top_k, "route backward"))) return rc;
    if (T == 0) return VQK_OK;
    if (!logits || !ids || !wts || !counts || !stats || !saved || !dlogits)
        return set_error(VQK_EINVAL, "route backward: NULL pointer");
    if (reinterpret_cast<uintptr_t>(saved) & 15)
        return set_error(VQK_EINVAL, "route backward: saved must be 16-byte aligned");
    GroupBwdArgs a{};
    a.l = logits; a.T = T; a.ld = ld;
    a.E = int32_t(E); a.k = top_k; a.norm = norm_topk; a.scale = form->scale;
    a.ids = ids; a.counts = counts; a.wts = wts; a.stats = stats;
    a.saved = reinterpret_cast<const float4 *>(saved);
    a.dw = dw; a.gb = dbalance; a.gz = dz;
    a.dl = dlogits;
    const bool rows16 = group16_ok(T, E, top_k, 1);
    const int per = rows16 ? 4 * kRouteWaves : kRouteWaves;
    const int wgs = route_wgs_of(T, per);     // resident at once: 65536 tokens over 256 experts 38 us, in 2048 workgroups 45
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool sig = form->score == VQK_SCORE_SIGMOID;
    switch (l_type) {
        case VQK_F16: return sig ? go_group_bwd<VQK_F16, true>(a, rows16, wgs, st) : go_group_bwd<VQK_F16, false>(a, rows16, wgs, st);
        case VQK_BF16: return sig ? go_group_bwd<VQK_BF16, true>(a, rows16, wgs, st) : go_group_bwd<VQK_BF16, false>(a, rows16, wgs, st);
        default: return sig ? go_group_bwd<VQK_F32, true>(a, rows16, wgs, st) : go_group_bwd<VQK_F32, false>(a, rows16, wgs, st);
    }
}
