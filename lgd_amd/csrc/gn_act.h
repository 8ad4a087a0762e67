// Shared pieces of the channels-last GroupNorm + activation: gn_act.hip (streaming, any size) and gn_slab.hip (one pass, a group per workgroup).
#pragma once
#include "vec16.h"

namespace lgd {

enum GaAct { kActNone = 0, kActRelu = 1, kActSilu = 2 };

// gamma / beta in any of the three types; null: the neutral value
__device__ __forceinline__ float ga_param(const void* p, int type, int c, float none) {
    if (!p) return none;
    if (type == LGD_F32) return static_cast<const float*>(p)[c];
    if (type == LGD_BF16) return (float)static_cast<const __bf16*>(p)[c];
    return (float)static_cast<const _Float16*>(p)[c];
}
// the same for N channels as raw words, so that all the loads are on their way together (a load and its conversion per channel wait for each other:
// 16 of them took 3 us of an 8 us kernel)
template <int N> __device__ __forceinline__ void ga_param_words(const void* p, int type, const int (&c)[N], uint32_t (&w)[N]) {
    if (!p) return;
    if (type == LGD_F32) {
        #pragma unroll
        for (int i = 0; i < N; ++i) w[i] = static_cast<const uint32_t*>(p)[c[i]];
    } else {
        #pragma unroll
        for (int i = 0; i < N; ++i) w[i] = static_cast<const uint16_t*>(p)[c[i]];
    }
}
template <int N> __device__ __forceinline__ void ga_param_values(const void* p, int type, const uint32_t (&w)[N], float none, float (&v)[N]) {
    if (!p) {
        #pragma unroll
        for (int i = 0; i < N; ++i) v[i] = none;
    } else if (type == LGD_F32) {
        #pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __builtin_bit_cast(float, w[i]);
    } else if (type == LGD_BF16) {
        #pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __builtin_bit_cast(float, w[i] << 16);
    } else {
        #pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]);
    }
}
__device__ __forceinline__ void ga_param_store(void* p, int type, int c, float v) {
    if (type == LGD_F32) static_cast<float*>(p)[c] = v;
    else if (type == LGD_BF16) static_cast<__bf16*>(p)[c] = (__bf16)v;
    else static_cast<_Float16*>(p)[c] = (_Float16)v;
}

// fp64 -> fp32 as a rounding of its own: in front of one to fp16 the compiler makes both a single fp64 -> fp16 conversion, 25 instructions instead of 2
__device__ __forceinline__ float ga_single(double d) {
    float f = (float)d;
    asm("" : "+v"(f));
    return f;
}

// sigmoid: v_exp_f32 and v_rcp_f32 (one ulp each); z = -inf gives 0, +inf gives 1
__device__ __forceinline__ float ga_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896341f * z)); }

template <int ACT> __device__ __forceinline__ float ga_act(float z) {
    if (ACT == kActRelu) return z <= 0.f ? 0.f : z;   // NaN passes, as torch.relu
    if (ACT == kActSilu) return z * ga_sigmoid(z);
    return z;
}

// The backward's constants of a group: mean = hi + lo and
// 1/deviation = r + rl are pairs of fp32 words: xh = (x - hi) r - lo r is as good as the fp64 form (x - hi is exact near the mean)
struct GaGroup { float hi, lo, r, rl, nlr; };
__device__ __forceinline__ GaGroup ga_group(double m, double r) {
    GaGroup k;
    k.hi = (float)m; k.lo = (float)(m - (double)k.hi);
    k.r = (float)r; k.rl = (float)(r - (double)k.r);
    k.nlr = -k.lo * k.r;
    return k;
}
__device__ __forceinline__ float ga_xhat(float x, const GaGroup& k) { return __builtin_fmaf(x - k.hi, k.r, k.nlr); }

// g = dy act'(z).  ReLU: z in fp32 is within 2^-21 (|xh gamma| + |beta|) of its value; where that leaves the sign open (one element in 10^5 or so)
// it is computed again in fp64
template <int ACT> __device__ __forceinline__ float ga_grad(float dy, float x, float xh, const GaGroup& k, float ga, float be) {
    if (ACT == kActNone) return dy;
    const float z = __builtin_fmaf(xh, ga, be);
    if (ACT == kActRelu) {
        bool off = z <= 0.f;
        if (!(fabsf(z) > 9.5367431640625e-7f * (fabsf(xh * ga) + fabsf(be)))) {
            float hi = k.hi, lo = k.lo, r = k.r, rl = k.rl, a = ga, b = be;
            asm volatile("" : "+v"(hi), "+v"(lo), "+v"(r), "+v"(rl), "+v"(a), "+v"(b));   // keeps their fp64 forms out of the loop's registers
            off = fma(((double)x - ((double)hi + (double)lo)) * ((double)r + (double)rl), (double)a, (double)b) <= 0.0;
        }
        return off ? 0.f : dy;   // NaN passes dy, as torch
    }
    const float s = ga_sigmoid(z);
    return dy * __builtin_fmaf(z * s, 1.f - s, s);
}

// a call as the one-pass kernels take it (checked by the caller); they return false where the call is not theirs
struct GaCall {
    const void* const* x;
    const void* const* dy;
    void* const* out;
    const int32_t* hw;
    int L, B, C, G, dtype, act, ptype;
    double eps;
    const void* gamma;
    const void* beta;
    double* stats;
    double* csum;       // backward: [L*B][C][2]
    void* dgamma;
    void* dbeta;
};
bool ga_slab_takes(const int32_t* hw, int L, int B, int C, int G, int dtype);
bool ga_slab_fwd(const GaCall& c, hipStream_t s);
bool ga_slab_bwd(const GaCall& c, hipStream_t s);

}  // namespace lgd
