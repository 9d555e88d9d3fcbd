// Group norm with an activation on channels-last tensors [B, S, C] (S pixels, C channels, G groups of Cg = C / G):
//   mu, var over the S x Cg values of (image, group);  xhat = (x - mu) / sqrt(var + eps);  z = w xhat + b;  y = act(z)
// and its backward
//   dz = dy act'(z);  db = sum dz;  dw = sum dz xhat;  dx = rstd (w dz - mean(w dz) - xhat mean(w dz xhat)).
// All of it is bound by memory: the arithmetic is about 10 (30) operations per element.
//
// Layout of the work: a workgroup takes a chunk of pixels of one image and a block of CB <= 256 vectors of VEC channels; a
// thread keeps one channel vector and walks pixels, so that 16-byte loads of neighbouring lanes are neighbours in memory
// whatever Cg is, and the affine constants are read once.
// Statistics: per thread and tile the mean and the sum of squared differences from it, joined by
//   M2 = M2a + M2b + d^2 na nb / (na + nb):
// E[x^2] - mu^2 would lose everything where |mu| >> sigma.  fp32 throughout.  Every sum has a fixed order: results do not
// change from run to run.
#include "ksr_common.h"

namespace {

constexpr int THREADS = 256;

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
    float eps;
};

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

// Where this workgroup and thread work: blockIdx.x = (image * nblk + channel block) * nchunk + chunk.
template <int VEC> struct Place {
    long b, chunk, p0, p1;
    int blk, c0, cb, tv, pl;
    bool active;
    __device__ __forceinline__ Place(const GnArgs& a, long wg) {
        chunk = wg % a.nchunk;
        const long r = wg / a.nchunk;
        blk = (int)(r % a.nblk);
        b = r / a.nblk;
        c0 = blk * a.CB;
        cb = a.C - c0 < a.CB ? a.C - c0 : a.CB;
        tv = (int)threadIdx.x % a.CV;
        pl = (int)threadIdx.x / a.CV;
        active = pl < a.PL && tv * VEC < cb;
        p0 = chunk * a.chunk;
        p1 = p0 + a.chunk < a.S ? p0 + a.chunk : a.S;
    }
    // the r-th of a thread's pixels in flight, held inside the chunk: loads need no branch, what is loaded twice is not used
    __device__ __forceinline__ long pixel(long base, int r, int PL) const {
        const long p = base + (long)r * PL;
        return p < p1 ? p : p1 - 1;
    }
};

// vectors in flight per thread: 64 bytes of 16-byte loads, eight of the narrower ones
template <class T, int VEC> constexpr int in_flight() { return sizeof(T) * VEC == 16 ? 4 : 8; }

// ------------------------------------------------------------------------------------------------ statistics
// ONE: a vector's channels belong to one group (Cg % VEC == 0): one (mean, M2) per thread instead of one per channel.
template <class T, int VEC, bool ONE>
__global__ void __launch_bounds__(THREADS) gn_stats_kernel(GnArgs a) {
    constexpr int NE = ONE ? 1 : VEC, R = in_flight<T, VEC>();
    typedef Vec<T, VEC> V;
    __shared__ float smean[THREADS * NE], sm2[THREADS * NE], sn[THREADS];
    const Place<VEC> w(a, blockIdx.x);
    float mean[NE], m2[NE], n = 0.f;                    // n: values behind each of the NE entries
#pragma unroll
    for (int i = 0; i < NE; ++i) mean[i] = m2[i] = 0.f;
    if (w.active) {
        const T* src = reinterpret_cast<const T*>(a.x) + w.b * a.xs_b + w.c0 + w.tv * VEC;
        for (long base = w.p0 + w.pl; base < w.p1; base += (long)R * a.PL) {
            typename V::Raw raw[R];
            int cnt = 0;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                raw[r] = *reinterpret_cast<const typename V::Raw*>(src + w.pixel(base, r, a.PL) * a.xs_p);
                cnt += base + (long)r * a.PL < w.p1;
            }
            float v[R][VEC], s[NE], q[NE];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                V::unpack(raw[r], v[r]);
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[r][i] = r < cnt ? v[r][i] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < NE; ++i) s[i] = q[i] = 0.f;
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < VEC; ++i) s[ONE ? 0 : i] += v[r][i];
            const float nt = (float)(cnt * (ONE ? VEC : 1)), rn = 1.f / nt;
#pragma unroll
            for (int i = 0; i < NE; ++i) s[i] *= rn;                     // the tile's mean
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float d = r < cnt ? v[r][i] - s[ONE ? 0 : i] : 0.f;
                    q[ONE ? 0 : i] = fmaf(d, d, q[ONE ? 0 : i]);
                }
            const float f = nt / (n + nt);
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const float d = s[i] - mean[i];
                mean[i] = fmaf(d, f, mean[i]);
                m2[i] += fmaf(d, d * f * n, q[i]);
            }
            n += nt;
        }
    }
    if (w.active) {
        if (w.tv == 0) sn[w.pl] = n;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int e = (w.pl * a.CV + w.tv) * NE + i;
            smean[e] = mean[i];
            sm2[e] = m2[i];
        }
    }
    __syncthreads();
    // a wave per group that this channel block touches: join the entries of its channels and the pixel lanes
    const int lane = threadIdx.x & 63, per = ONE ? VEC : 1;
    const int g0 = w.c0 / a.Cg, g1 = (w.c0 + w.cb - 1) / a.Cg;
    for (int g = g0 + ((int)threadIdx.x >> 6); g <= g1; g += THREADS / 64) {
        const int lo = (g * a.Cg > w.c0 ? g * a.Cg - w.c0 : 0) / per;
        const int hi = ((g + 1) * a.Cg < w.c0 + w.cb ? (g + 1) * a.Cg - w.c0 : w.cb) / per, ne = hi - lo;
        float cnt = 0.f, sum = 0.f;
        for (int e = lane; e < a.PL * ne; e += 64) {
            const int pl = e / ne;
            cnt += sn[pl];
            sum = fmaf(sn[pl], smean[pl * a.CV * NE + lo + e - pl * ne], sum);
        }
        cnt = wave_sum(cnt);
        const float m = wave_sum(sum) / cnt;
        float q = 0.f;
        for (int e = lane; e < a.PL * ne; e += 64) {
            const int pl = e / ne, k = pl * a.CV * NE + lo + e - pl * ne;
            const float d = smean[k] - m;
            q += fmaf(sn[pl] * d, d, sm2[k]);
        }
        q = wave_sum(q);
        if (lane == 0) {
            float* o = a.part + 2 * (((w.b * a.nchunk + w.chunk) * a.nblk + w.blk) * a.GB + (g - g0));
            o[0] = m;
            o[1] = q;
        }
    }
}

// one wave per (image, group): joins the chunks' (mean, M2)
__global__ void __launch_bounds__(THREADS) gn_stats_join_kernel(GnArgs a) {
    const long i = (long)blockIdx.x * (THREADS / 64) + (threadIdx.x >> 6);
    if (i >= a.B * a.G) return;
    const long b = i / a.G;
    const int g = (int)(i % a.G), lane = threadIdx.x & 63;
    const int k0 = g * a.Cg / a.CB, k1 = ((g + 1) * a.Cg - 1) / a.CB, nk = k1 - k0 + 1;
    float m = 0.f, q = 0.f;
    const float rn = 1.f / ((float)a.S * (float)a.Cg);
    for (int pass = 0; pass < 2; ++pass) {
        float s = 0.f;
        for (long e = lane; e < a.nchunk * nk; e += 64) {
            const long chunk = e / nk;
            const int blk = k0 + (int)(e - chunk * nk), c0 = blk * a.CB;
            const long left = a.S - chunk * a.chunk;
            const int hi = (g + 1) * a.Cg < c0 + a.CB ? (g + 1) * a.Cg : c0 + a.CB, lo = g * a.Cg > c0 ? g * a.Cg : c0;
            const float n = (float)(left < a.chunk ? left : a.chunk) * (float)(hi - lo);
            const float* p = a.part + 2 * (((b * a.nchunk + chunk) * a.nblk + blk) * a.GB + (g - c0 / a.Cg));
            if (pass == 0) s = fmaf(n * rn, p[0], s);
            else { const float d = p[0] - m; s += fmaf(n * d, d, p[1]); }
        }
        if (pass == 0) m = wave_sum(s); else q = wave_sum(s);
    }
    if (lane == 0) {
        a.stats[2 * i] = m;
        a.stats[2 * i + 1] = 1.f / sqrtf(fmaf(q, rn, a.eps));
    }
}

// the thread's channels: mean, rstd of their groups, weight and bias
template <int VEC> struct Affine {
    float mean[VEC], rstd[VEC], w[VEC], b[VEC];
    __device__ __forceinline__ Affine(const GnArgs& a, long img, int c) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float* s = a.stats + 2 * (img * a.G + (c + i) / a.Cg);
            mean[i] = s[0];
            rstd[i] = s[1];
            w[i] = a.w ? a.w[c + i] : 1.f;
            b[i] = a.b ? a.b[c + i] : 0.f;
        }
    }
};

// ------------------------------------------------------------------------------------------------ y = act(w xhat + b)
template <class T, int VEC, int ACT>
__global__ void __launch_bounds__(THREADS) gn_apply_kernel(GnArgs a) {
    constexpr int R = in_flight<T, VEC>();
    typedef Vec<T, VEC> V;
    const Place<VEC> w(a, blockIdx.x);
    if (!w.active) return;
    const int c = w.c0 + w.tv * VEC;
    Affine<VEC> k(a, w.b, c);
#pragma unroll
    for (int i = 0; i < VEC; ++i) k.w[i] *= k.rstd[i];
    const T* src = reinterpret_cast<const T*>(a.x) + w.b * a.xs_b + c;
    T* dst = reinterpret_cast<T*>(a.out) + w.b * a.S * a.C + c;
    for (long base = w.p0 + w.pl; base < w.p1; base += (long)R * a.PL) {
        typename V::Raw raw[R];
#pragma unroll
        for (int r = 0; r < R; ++r)
            raw[r] = *reinterpret_cast<const typename V::Raw*>(src + w.pixel(base, r, a.PL) * a.xs_p);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (base + (long)r * a.PL < w.p1) {
                float v[VEC];
                V::unpack(raw[r], v);
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[i] = act_of<ACT>(fmaf(v[i] - k.mean[i], k.w[i], k.b[i]));
                *reinterpret_cast<typename V::Raw*>(dst + (base + (long)r * a.PL) * a.C) = V::pack(v);
            }
    }
}

// ------------------------------------------------------------------------------------------------ backward
// per chunk and channel: sum dz, sum dz xhat
template <class T, int VEC, int ACT>
__global__ void __launch_bounds__(THREADS) gn_bwd_reduce_kernel(GnArgs a) {
    constexpr int R = in_flight<T, VEC>() / 2;
    typedef Vec<T, VEC> V;
    __shared__ float s1[THREADS * VEC], s2[THREADS * VEC];
    const Place<VEC> w(a, blockIdx.x);
    float d1[VEC], d2[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) d1[i] = d2[i] = 0.f;
    const int c = w.c0 + w.tv * VEC;
    if (w.active) {
        const Affine<VEC> k(a, w.b, c);
        const T* src = reinterpret_cast<const T*>(a.x) + w.b * a.xs_b + c;
        const T* gsrc = reinterpret_cast<const T*>(a.dy) + w.b * a.ds_b + c;
        for (long base = w.p0 + w.pl; base < w.p1; base += (long)R * a.PL) {
            typename V::Raw raw[R], graw[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                raw[r] = *reinterpret_cast<const typename V::Raw*>(src + w.pixel(base, r, a.PL) * a.xs_p);
                graw[r] = *reinterpret_cast<const typename V::Raw*>(gsrc + w.pixel(base, r, a.PL) * a.ds_p);
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (base + (long)r * a.PL < w.p1) {
                    float v[VEC], g[VEC];
                    V::unpack(raw[r], v);
                    V::unpack(graw[r], g);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float xh = (v[i] - k.mean[i]) * k.rstd[i];
                        const float dz = g[i] * act_slope<ACT>(fmaf(xh, k.w[i], k.b[i]));
                        d1[i] += dz;
                        d2[i] = fmaf(dz, xh, d2[i]);
                    }
                }
        }
    }
    // pairwise over the pixel lanes
    const int e = (w.pl * a.CV + w.tv) * VEC;
    for (int n = a.PL; n > 1;) {
        const int half = (n + 1) >> 1;
        if (w.active && w.pl >= half && w.pl < n)
#pragma unroll
            for (int i = 0; i < VEC; ++i) { s1[e + i] = d1[i]; s2[e + i] = d2[i]; }
        __syncthreads();
        if (w.active && w.pl + half < n) {
            const int o = e + half * a.CV * VEC;
#pragma unroll
            for (int i = 0; i < VEC; ++i) { d1[i] += s1[o + i]; d2[i] += s2[o + i]; }
        }
        __syncthreads();
        n = half;
    }
    if (w.active && w.pl == 0) {
        float* o = a.part + 2 * (w.b * a.nchunk + w.chunk) * a.C + c;
#pragma unroll
        for (int i = 0; i < VEC; ++i) { o[i] = d1[i]; o[a.C + i] = d2[i]; }
    }
}

// one workgroup per (image, group): sums the chunks per channel (chsum) and forms mean(w dz), mean(w dz xhat) (coef).
// TC lanes walk the group's channels, THREADS / TC the chunks.
__global__ void __launch_bounds__(THREADS) gn_bwd_join_kernel(GnArgs a, int TC) {
    __shared__ float s1[THREADS], s2[THREADS];
    const long b = blockIdx.x / a.G;
    const int g = (int)(blockIdx.x % a.G), t = threadIdx.x, tc = t % TC, tk = t / TC, NK = THREADS / TC;
    float g1 = 0.f, g2 = 0.f;
    for (int cc = 0; cc < a.Cg; cc += TC) {
        const bool ok = cc + tc < a.Cg;
        const int c = g * a.Cg + cc + tc;
        float v1 = 0.f, v2 = 0.f;
        if (ok)
            for (long k = tk; k < a.nchunk; k += NK) {
                const float* p = a.part + 2 * (b * a.nchunk + k) * a.C + c;
                v1 += p[0];
                v2 += p[a.C];
            }
        s1[t] = v1;
        s2[t] = v2;
        __syncthreads();
        for (int h = NK >> 1; h > 0; h >>= 1) {
            if (tk < h) { s1[t] += s1[t + h * TC]; s2[t] += s2[t + h * TC]; }
            __syncthreads();
        }
        if (ok && tk == 0) {
            a.chsum[2 * b * a.C + c] = s1[t];
            a.chsum[(2 * b + 1) * a.C + c] = s2[t];
            const float w = a.w ? a.w[c] : 1.f;
            g1 = fmaf(w, s1[t], g1);
            g2 = fmaf(w, s2[t], g2);
        }
        __syncthreads();
    }
    s1[t] = g1;                      // zero outside tk == 0
    s2[t] = g2;
    __syncthreads();
    if (t < 64) {
        float v1 = t < TC ? s1[t] : 0.f, v2 = t < TC ? s2[t] : 0.f;
        v1 = wave_sum(v1);
        v2 = wave_sum(v2);
        if (t == 0) {
            const float rn = 1.f / ((float)a.S * (float)a.Cg);
            a.coef[2 * (long)blockIdx.x] = v1 * rn;
            a.coef[2 * (long)blockIdx.x + 1] = v2 * rn;
        }
    }
}

// dw, db: chsum over the images; 16 channels x 16 image lanes per workgroup
__global__ void __launch_bounds__(THREADS) gn_bwd_params_kernel(GnArgs a) {
    __shared__ float s1[THREADS], s2[THREADS];
    const int t = threadIdx.x, c = blockIdx.x * 16 + (t & 15), tb = t >> 4;
    float v1 = 0.f, v2 = 0.f;
    if (c < a.C)
        for (long b = tb; b < a.B; b += 16) {
            v1 += a.chsum[2 * b * a.C + c];
            v2 += a.chsum[(2 * b + 1) * a.C + c];
        }
    s1[t] = v1;
    s2[t] = v2;
    __syncthreads();
    for (int h = 8; h > 0; h >>= 1) {
        if (tb < h) { s1[t] += s1[t + 16 * h]; s2[t] += s2[t + 16 * h]; }
        __syncthreads();
    }
    if (tb == 0 && c < a.C) {
        if (a.db) a.db[c] = s1[t];
        if (a.dw) a.dw[c] = s2[t];
    }
}

template <class T, int VEC, int ACT>
__global__ void __launch_bounds__(THREADS) gn_bwd_dx_kernel(GnArgs a) {
    constexpr int R = in_flight<T, VEC>() / 2;
    typedef Vec<T, VEC> V;
    const Place<VEC> w(a, blockIdx.x);
    if (!w.active) return;
    const int c = w.c0 + w.tv * VEC;
    const Affine<VEC> k(a, w.b, c);
    float q1[VEC], q2[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const float* s = a.coef + 2 * (w.b * a.G + (c + i) / a.Cg);
        q1[i] = s[0];
        q2[i] = s[1];
    }
    const T* src = reinterpret_cast<const T*>(a.x) + w.b * a.xs_b + c;
    const T* gsrc = reinterpret_cast<const T*>(a.dy) + w.b * a.ds_b + c;
    T* dst = reinterpret_cast<T*>(a.out) + w.b * a.S * a.C + c;
    for (long base = w.p0 + w.pl; base < w.p1; base += (long)R * a.PL) {
        typename V::Raw raw[R], graw[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            raw[r] = *reinterpret_cast<const typename V::Raw*>(src + w.pixel(base, r, a.PL) * a.xs_p);
            graw[r] = *reinterpret_cast<const typename V::Raw*>(gsrc + w.pixel(base, r, a.PL) * a.ds_p);
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (base + (long)r * a.PL < w.p1) {
                float v[VEC], g[VEC];
                V::unpack(raw[r], v);
                V::unpack(graw[r], g);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float xh = (v[i] - k.mean[i]) * k.rstd[i];
                    const float dz = g[i] * act_slope<ACT>(fmaf(xh, k.w[i], k.b[i]));
                    v[i] = k.rstd[i] * (fmaf(dz, k.w[i], -q1[i]) - xh * q2[i]);
                }
                *reinterpret_cast<typename V::Raw*>(dst + (base + (long)r * a.PL) * a.C) = V::pack(v);
            }
    }
}

// ------------------------------------------------------------------------------------------------ host
// Number of workgroups that the chunks of a pass aim at: eight 256-thread workgroups on each of 256 CUs
constexpr long AIM_WGS = 2048;

// Split of [B, S, C] for a vector of `vec` channels, `inflight` pixels a thread holds at once
void split(GnArgs& a, int vec, int inflight) {
    const int vectors = a.C / vec;
    a.nblk = (vectors + THREADS - 1) / THREADS;
    a.CV = (vectors + a.nblk - 1) / a.nblk;
    a.CB = a.CV * vec;
    a.nblk = (a.C + a.CB - 1) / a.CB;
    a.PL = THREADS / a.CV;
    a.GB = (a.CB - 1) / a.Cg + 2;
    if (a.GB > a.G) a.GB = a.G;
    const long tile = (long)a.PL * inflight, tiles = (a.S + tile - 1) / tile;
    long want = AIM_WGS / (a.B * a.nblk > AIM_WGS ? AIM_WGS : a.B * a.nblk);
    if (want < 1) want = 1;
    if (want > tiles) want = tiles;
    a.chunk = (tiles + want - 1) / want * tile;
    a.nchunk = (a.S + a.chunk - 1) / a.chunk;
}

// most chunks that split() makes for any vector width
long max_parts(long B, long S, int C, int G, bool backward) {
    long most = 0;
    for (int vec = 1; vec <= 8; vec *= 2)
        for (int fl = 2; fl <= 8; fl *= 2) {
            if (C % vec) continue;
            GnArgs a{};
            a.B = B; a.S = S; a.C = C; a.G = G; a.Cg = C / G;
            split(a, vec, fl);
            const long n = B * a.nchunk * 2 * (backward ? C : (long)a.nblk * a.GB);
            if (n > most) most = n;
        }
    return most;
}

bool aligned(const void* p, long bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }

// widest vector (8, 2, 1 bf16 or 4, 1 fp32) that divides the channels, the strides and every address
int vec_of(const GnArgs& a, int esize, bool backward) {
    for (int vec = 16 / esize; vec > 1; vec = (esize == 2 && vec == 8) ? 2 : 1) {
        const long bytes = (long)vec * esize;
        bool ok = a.C % vec == 0 && a.xs_b % vec == 0 && a.xs_p % vec == 0 && aligned(a.x, bytes) && aligned(a.out, bytes);
        if (backward) ok = ok && a.ds_b % vec == 0 && a.ds_p % vec == 0 && aligned(a.dy, bytes);
        if (ok) return vec;
    }
    return 1;
}

template <class T, int VEC> int run_fwd(GnArgs& a, int act, hipStream_t st) {
    split(a, VEC, in_flight<T, VEC>());
    const dim3 grid((unsigned)(a.B * a.nblk * a.nchunk)), block(THREADS);
    if (a.Cg % VEC == 0) hipLaunchKernelGGL((gn_stats_kernel<T, VEC, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((gn_stats_kernel<T, VEC, false>), grid, block, 0, st, a);
    KSR_LAUNCH_CHECK("group_norm_fwd");
    hipLaunchKernelGGL(gn_stats_join_kernel, dim3((unsigned)((a.B * a.G + 3) / 4)), block, 0, st, a);
    KSR_LAUNCH_CHECK("group_norm_fwd");
    switch (act) {
        case KSR_ACT_NONE: hipLaunchKernelGGL((gn_apply_kernel<T, VEC, KSR_ACT_NONE>), grid, block, 0, st, a); break;
        case KSR_ACT_RELU: hipLaunchKernelGGL((gn_apply_kernel<T, VEC, KSR_ACT_RELU>), grid, block, 0, st, a); break;
        case KSR_ACT_SILU: hipLaunchKernelGGL((gn_apply_kernel<T, VEC, KSR_ACT_SILU>), grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL((gn_apply_kernel<T, VEC, KSR_ACT_GELU>), grid, block, 0, st, a); break;
    }
    KSR_LAUNCH_CHECK("group_norm_fwd");
    return KSR_OK;
}

template <class T, int VEC, int ACT> int run_bwd_act(GnArgs& a, hipStream_t st) {
    split(a, VEC, in_flight<T, VEC>() / 2);
    const dim3 grid((unsigned)(a.B * a.nblk * a.nchunk)), block(THREADS);
    hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, VEC, ACT>), grid, block, 0, st, a);
    KSR_LAUNCH_CHECK("group_norm_bwd");
    int tc = 1;
    while (tc < a.Cg && tc < 64) tc *= 2;
    hipLaunchKernelGGL(gn_bwd_join_kernel, dim3((unsigned)(a.B * a.G)), block, 0, st, a, tc);
    KSR_LAUNCH_CHECK("group_norm_bwd");
    if (a.dw || a.db) {
        hipLaunchKernelGGL(gn_bwd_params_kernel, dim3((unsigned)((a.C + 15) / 16)), block, 0, st, a);
        KSR_LAUNCH_CHECK("group_norm_bwd");
    }
    if (a.out) {
        hipLaunchKernelGGL((gn_bwd_dx_kernel<T, VEC, ACT>), grid, block, 0, st, a);
        KSR_LAUNCH_CHECK("group_norm_bwd");
    }
    return KSR_OK;
}
template <class T, int VEC> int run_bwd(GnArgs& a, int act, hipStream_t st) {
    switch (act) {
        case KSR_ACT_NONE: return run_bwd_act<T, VEC, KSR_ACT_NONE>(a, st);
        case KSR_ACT_RELU: return run_bwd_act<T, VEC, KSR_ACT_RELU>(a, st);
        case KSR_ACT_SILU: return run_bwd_act<T, VEC, KSR_ACT_SILU>(a, st);
        default: return run_bwd_act<T, VEC, KSR_ACT_GELU>(a, st);
    }
}

int check_shape(const char* what, int64_t B, int64_t S, int C, int G) {
    KSR_CHECK_ARG(B >= 0 && S >= 0 && C > 0 && G > 0 && C % G == 0, "%s: [%lld, %lld, %d] in %d groups", what, (long long)B,
                  (long long)S, C, G);
    KSR_UNSUPPORTED(B > (1 << 24) || S > (1ll << 40) || B * (int64_t)G > (1ll << 30) || B * ((C + 255) / 256) > (1ll << 30),
                    "%s: [%lld, %lld, %d] is beyond the launch limits", what, (long long)B, (long long)S, C);
    return KSR_OK;
}

}  // namespace

extern "C" int64_t ksr_group_norm_ws_floats(int64_t B, int64_t S, int C, int G, int backward) {
    if (check_shape("group_norm_ws_floats", B, S, C, G) != KSR_OK) return -1;
    if (B == 0 || S == 0) return 0;
    return max_parts(B, S, C, G, backward != 0) + (backward ? 2 * B * G + 2 * B * C : 0);
}

extern "C" int ksr_group_norm_fwd(const void* x, int64_t x_image_stride, int64_t x_pixel_stride, const float* weight, const float* bias,
                                  void* y, float* stats, float* ws, int64_t B, int64_t S, int C, int G, float eps, int act, int bf16,
                                  hipStream_t stream) {
    if (int rc = check_shape("group_norm_fwd", B, S, C, G)) return rc;
    KSR_CHECK_ARG(act >= KSR_ACT_NONE && act <= KSR_ACT_GELU, "group_norm_fwd: activation %d", act);
    KSR_CHECK_ARG(eps >= 0.f, "group_norm_fwd: eps = %g", (double)eps);
    if (B == 0 || S == 0) return KSR_OK;
    KSR_CHECK_ARG(x && y && stats && ws, "group_norm_fwd: null pointer");
    KSR_CHECK_ARG(x_pixel_stride >= 0 && x_image_stride >= 0, "group_norm_fwd: negative stride");
    KSR_CHECK_ARG(aligned(x, bf16 ? 2 : 4) && aligned(y, bf16 ? 2 : 4), "group_norm_fwd: misaligned pointer");
    GnArgs a{};
    a.x = x; a.out = y; a.w = weight; a.b = bias; a.stats = stats; a.part = ws;
    a.xs_b = x_image_stride; a.xs_p = x_pixel_stride;
    a.B = B; a.S = S; a.C = C; a.G = G; a.Cg = C / G; a.eps = eps;
    const int vec = vec_of(a, bf16 ? 2 : 4, false);
    if (bf16) return vec == 8 ? run_fwd<__bf16, 8>(a, act, stream) : vec == 2 ? run_fwd<__bf16, 2>(a, act, stream) : run_fwd<__bf16, 1>(a, act, stream);
    return vec == 4 ? run_fwd<float, 4>(a, act, stream) : run_fwd<float, 1>(a, act, stream);
}

extern "C" int ksr_group_norm_bwd(const void* x, int64_t x_image_stride, int64_t x_pixel_stride, const void* dy, int64_t dy_image_stride,
                                  int64_t dy_pixel_stride, const float* weight, const float* bias, const float* stats, void* dx,
                                  float* dweight, float* dbias, float* ws, int64_t B, int64_t S, int C, int G, int act, int bf16,
                                  hipStream_t stream) {
    if (int rc = check_shape("group_norm_bwd", B, S, C, G)) return rc;
    KSR_CHECK_ARG(act >= KSR_ACT_NONE && act <= KSR_ACT_GELU, "group_norm_bwd: activation %d", act);
    GnArgs a{};
    a.x = x; a.dy = dy; a.out = dx; a.w = weight; a.b = bias; a.stats = const_cast<float*>(stats); a.dw = dweight; a.db = dbias;
    a.xs_b = x_image_stride; a.xs_p = x_pixel_stride; a.ds_b = dy_image_stride; a.ds_p = dy_pixel_stride;
    a.B = B; a.S = S; a.C = C; a.G = G; a.Cg = C / G;
    if (B == 0 || S == 0) {                               // empty sums
        a.B = 0;
        if (!dweight && !dbias) return KSR_OK;
        hipLaunchKernelGGL(gn_bwd_params_kernel, dim3((unsigned)((C + 15) / 16)), dim3(THREADS), 0, stream, a);
        KSR_LAUNCH_CHECK("group_norm_bwd");
        return KSR_OK;
    }
    KSR_CHECK_ARG(x && dy && stats && ws, "group_norm_bwd: null pointer");
    KSR_CHECK_ARG(x_pixel_stride >= 0 && x_image_stride >= 0 && dy_pixel_stride >= 0 && dy_image_stride >= 0, "group_norm_bwd: negative stride");
    KSR_CHECK_ARG(aligned(x, bf16 ? 2 : 4) && aligned(dy, bf16 ? 2 : 4) && aligned(dx, bf16 ? 2 : 4), "group_norm_bwd: misaligned pointer");
    a.coef = ws;
    a.chsum = a.coef + 2 * B * G;
    a.part = a.chsum + 2 * B * C;
    const int vec = vec_of(a, bf16 ? 2 : 4, true);
    if (bf16) return vec == 8 ? run_bwd<__bf16, 8>(a, act, stream) : vec == 2 ? run_bwd<__bf16, 2>(a, act, stream) : run_bwd<__bf16, 1>(a, act, stream);
    return vec == 4 ? run_bwd<float, 4>(a, act, stream) : run_bwd<float, 1>(a, act, stream);
}
