// What the routing kernels share: reductions inside a row of 16 lanes, loads of
// logits, the sums over tokens that both forms of routing leave to be finished.
#pragma once

#include "vqk_common.h"

namespace vqk {

constexpr int kRouteWaves = 4;
constexpr int kRouteThreads = kRouteWaves * kWave;
constexpr int kRouteMaxWgs = 768;              // three waves a SIMD: the registers of k_route16
constexpr int kRouteMaxE = 2048;
constexpr int kRouteMaxK = 64;
constexpr int kRouteCands = 32;                 // candidates of a token that sixteen lanes rank
constexpr uint32_t kKeyNegInf = 0x007fffffu;           // f32_key(-inf); NaN maps below it

// What a wave's lanes wrote to LDS before, its other lanes read after. The hardware
// keeps a wave's LDS accesses in order; the fences, which cost no instruction, hold
// the compiler to it.
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// e^d for -200 <= d <= 0: 2^(d log2 e), the product's rounding error carried along.
__device__ __forceinline__ float route_exp_in(float d) {
    constexpr float hi = 1.44269502162933349609375f, lo = 1.92596299113e-8f;   // log2 e = hi + lo
    const float t = d * hi, r = __builtin_fmaf(d, hi, -t) + d * lo;
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e, 0.693147182f * r, e);
}
// d <= 0: e^-200 is 0 already (and -inf leaves no NaN; a NaN stays).
__device__ __forceinline__ float route_exp(float d) { return route_exp_in(d < -200.f ? -200.f : d); }

template <int CTRL>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
    return (uint64_t(dpp_u<CTRL>(uint32_t(v >> 32))) << 32) | dpp_u<CTRL>(uint32_t(v));
}
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    v = max(v, dpp_u<kDppQuadXor1>(v));
    v = max(v, dpp_u<kDppQuadXor2>(v));
    v = max(v, dpp_u<kDppRowHalfMirror>(v));
    return max(v, dpp_u<kDppRowMirror>(v));
}
__device__ __forceinline__ uint32_t row_min(uint32_t v) {
    v = min(v, dpp_u<kDppQuadXor1>(v));
    v = min(v, dpp_u<kDppQuadXor2>(v));
    v = min(v, dpp_u<kDppRowHalfMirror>(v));
    return min(v, dpp_u<kDppRowMirror>(v));
}
// Both partners add the same two values, so every lane ends with the same sum.
__device__ __forceinline__ float row_sum(float v) {
    v += dpp_f<kDppQuadXor1>(v);
    v += dpp_f<kDppQuadXor2>(v);
    v += dpp_f<kDppRowHalfMirror>(v);
    return v + dpp_f<kDppRowMirror>(v);
}

// Lane `sub` of a token holds experts 64 q + 4 sub + j in value 4 q + j: whole
// lines a load. VEC: fours are aligned and whole.
template <int LT, int NS, bool VEC>
__device__ __forceinline__ void route_load16(const void *l, int64_t base, int E, int sub, bool in, float (&v)[NS]) {
#pragma unroll
    for (int q = 0; q < NS / 4; ++q) {
        const int e = 64 * q + 4 * sub;
        if constexpr (VEC) {
            if (in && e < E) {
                if constexpr (LT == VQK_F32) {
                    const float4 f = *reinterpret_cast<const float4 *>(static_cast<const float *>(l) + base + e);
                    v[4 * q] = f.x; v[4 * q + 1] = f.y; v[4 * q + 2] = f.z; v[4 * q + 3] = f.w;
                } else {
                    const u32x2 f = *reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(l) + base + e);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint16_t h = uint16_t(f[j / 2] >> (16 * (j & 1)));
                        v[4 * q + j] = LT == VQK_BF16 ? bf16_to_f32(h) : h_to_f32(h);
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * q + j] = -__builtin_inff();
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[4 * q + j] = in && e + j < E ? load_act(l, LT, base + e + j) : -__builtin_inff();
        }
    }
}

struct FinishArgs {
    const float *part_p, *part_z;
    const int32_t *part_c, *part_n;
    int32_t wgs, E, k;
    double *dot;                              // [groups] sums of c_e P_e
    int32_t *counts;
    float *stats;                             // balance, z, n
};
// counts, balance, z and n from the workgroups' partials.
int route_finish(const FinishArgs &f, hipStream_t st);
// Workgroups of a forward call that gives `per` tokens to one.
inline int route_wgs_of(int64_t T, int per) {
    const int64_t w = (T + per - 1) / per;
    return int(w < kRouteMaxWgs ? w : kRouteMaxWgs);
}
// Workspace of T tokens over E experts in either form, and where its parts lie.
size_t route_bytes(int64_t T, int64_t E);
void route_parts(void *workspace, int64_t E, int wgs, FinishArgs *f, float **part_p, int32_t **part_c, float **part_z,
                 int32_t **part_n);
// Fours of logits can be loaded (and of the gradient stored) at once.
bool route_vec(const void *l, int64_t ld, int64_t E, int lt);
int check_route(int32_t l_type, int64_t T, int64_t E, int64_t ld, int32_t k, const char *what);

}  // namespace vqk
