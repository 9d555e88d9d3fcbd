// What the group norm's kernels share (ksr_group_norm.hip: chunks of an image; ksr_group_norm_one.hip: a group in registers).
#pragma once
#include "ksr.h"
#include "ksr_common.h"

struct GnArgs {
    const void* x; const void* dy; void* out;          // out: y (forward) or dx (backward), dense
    const float* w; const float* b;                    // [C] or null
    float* stats;                                      // [B][G][2]: mean, 1 / sqrt(var + eps)
    float* part;                                       // per-chunk partial results
    float* coef;                                       // backward: [B][G][2] mean(w dz), mean(w dz xhat)
    float* chsum;                                      // backward: [B][2][C] sum dz, sum dz xhat
    float* dw; float* db;
    long xs_b, xs_p, ds_b, ds_p;                       // image and pixel strides of x, dy in elements
    long B, S, chunk, nchunk;
    int C, G, Cg, CB, nblk, GB, CV, PL;                // channels per block, blocks, group slots per block, vectors, pixel lanes
    int all;                                           // backward: these are all images of the call, not a range of them
    int past;                                          // write the result past the caches
    int join;                                          // the pass that uses the chunks' results joins them itself
    float eps;
};

namespace {


template <int BYTES> struct RawOf;
template <> struct RawOf<16> { typedef ksr_u32x4_t T; };
template <> struct RawOf<8> { typedef unsigned T __attribute__((ext_vector_type(2))); };
template <> struct RawOf<4> { typedef unsigned T; };
template <> struct RawOf<2> { typedef unsigned short T; };

template <class T, int VEC> struct Vec {
    typedef typename RawOf<sizeof(T) * VEC>::T Raw;
    static __device__ __forceinline__ void unpack(const Raw& r, float (&v)[VEC]) {
        T t[VEC];
        __builtin_memcpy(t, &r, sizeof(r));
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = (float)t[i];
    }
    static __device__ __forceinline__ Raw pack(const float (&v)[VEC]) {      // bf16: rounded to nearest even, once
        T t[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) t[i] = (T)v[i];
        Raw r;
        __builtin_memcpy(&r, t, sizeof(r));
        return r;
    }
};

// What the activation is taken of, from xhat = (x - mean) * rstd: one expression for forward and backward, so that ReLU's mask is
// that of the result (as fmaf(x - mean, w * rstd, b) a value next to 0 may have the other sign)
__device__ __forceinline__ float gn_z(float xhat, float w, float b) { return fmaf(xhat, w, b); }

// SiLU and the normal density in GELU's slope take e^u as 2^(u log2 e) (v_exp_f32) with the argument rounded once, and 1 / v by
// v_rcp_f32: the argument's rounding is |u| 2^-24 of the value, which in SiLU comes to at most z^2 e^-|z| 2^-24 < 0.55 2^-24.  Only
// values that are small themselves lose bits (z = -30: 2e-6 of 3e-12), for a quarter of what a library's exp costs.
template <int ACT> __device__ __forceinline__ float act_of(float z) {
    if constexpr (ACT == KSR_ACT_RELU) return z < 0.f ? 0.f : z;                // NaN stays NaN
    else if constexpr (ACT == KSR_ACT_SILU) return z * ksr_sigmoid(z);
    else if constexpr (ACT == KSR_ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    else return z;
}
template <int ACT> __device__ __forceinline__ float act_slope(float z) {
    if constexpr (ACT == KSR_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    else if constexpr (ACT == KSR_ACT_SILU) {
        const float s = ksr_sigmoid(z);
        return s * (1.f + z * (1.f - s));
    } else if constexpr (ACT == KSR_ACT_GELU)
        return 0.5f * (1.f + erff(z * 0.70710678118654752f)) +
               z * 0.39894228040143268f * __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z);
    else return 1.f;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
    return v;
}


}  // namespace

// ksr_group_norm_one.hip: whether a (image, group) fits one workgroup's registers, and the launches if it does
bool ksr_gn_one_fits(const GnArgs& a, int esize, bool backward, int& vec, int& per_vec);
int ksr_gn_one_fwd(GnArgs& a, int act, bool bf16, int vec, int per_vec, hipStream_t st);
int ksr_gn_one_bwd(GnArgs& a, int act, bool bf16, int vec, int per_vec, hipStream_t st);
