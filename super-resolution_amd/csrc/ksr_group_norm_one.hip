// Group norm in one pass, for a (image, group) that fits the registers of one workgroup: x (and dy) are read once and held as they
// were read, statistics and sums are formed from the registers, y (dx) is written - one launch forward, one or two backward, the
// least traffic there is (ksr_group_norm.hip reads x twice, x and dy twice).  256 bytes per thread forward, 128 + 128 backward:
// 65536 fp32 (131072 bf16) values per workgroup of 1024 threads, half of it backward.
// Variance: the mean first, then squared differences from it.  A vector of VEC channels lies inside one group (NE = 1), or holds
// NE = VEC / Cg whole groups.  Neighbouring groups, which share cache lines, run on one XCD.
#include "ksr_group_norm.h"

namespace {

template <class T, int VEC, int NE, int TH> struct One {
    long b;
    int blk, c0, tv, pl, PL;
    bool active;
    __device__ __forceinline__ explicit One(const GnArgs& a) {
        const unsigned id = ksr_xcd_contiguous(blockIdx.x, gridDim.x);
        blk = (int)(id % (unsigned)a.nblk);
        b = (long)(id / (unsigned)a.nblk);
        c0 = blk * a.CB;
        if constexpr (NE > 1) { tv = 0; pl = (int)threadIdx.x; PL = TH; active = true; }      // one vector holds the block
        else { tv = (int)threadIdx.x % a.CV; pl = (int)threadIdx.x / a.CV; PL = a.PL; active = pl < PL; }
    }
};

// From here on the registers may hold anything as far as the compiler knows: it would otherwise keep every unpacked value from one
// pass over them to the next (twice the registers of bf16 data) and spill.
template <int R, class Raw> __device__ __forceinline__ void forget(Raw (&raw)[R]) {
    if constexpr (sizeof(Raw) >= 4)
#pragma unroll
        for (int r = 0; r < R; ++r) asm volatile("" : "+v"(raw[r]));
}

// sums of N values over the workgroup, in every thread; a fixed order
template <int N, int TH> __device__ __forceinline__ void block_sum(float (&v)[N], float (*lds)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) v[i] += __shfl_xor(v[i], m, 64);
    __syncthreads();                                   // lds may still be read from the sum before
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) lds[threadIdx.x >> 6][i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = 0.f;
#pragma unroll
        for (int w = 0; w < TH / 64; ++w) v[i] += lds[w][i];
    }
}

template <class T, int VEC, int NE, int R, int TH, int ACT>
__global__ void __launch_bounds__(TH) gn_one_fwd_kernel(GnArgs a) {
    typedef Vec<T, VEC> V;
    constexpr int PE = VEC / NE;                       // channels of a vector per group
    __shared__ float red[TH / 64][NE];
    const One<T, VEC, NE, TH> w(a);
    const int c = w.c0 + w.tv * VEC;
    const T* src = reinterpret_cast<const T*>(a.x) + w.b * a.xs_b + c;
    const int S = (int)a.S;
    typename V::Raw raw[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (r * w.PL < S) {
            const int p = w.pl + r * w.PL;
            raw[r] = *reinterpret_cast<const typename V::Raw*>(src + (long)(p < S ? p : S - 1) * a.xs_p);
        }
    float mean[NE], m2[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) mean[e] = m2[e] = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (r * w.PL < S) {
            float v[VEC];
            V::unpack(raw[r], v);
            const bool ok = w.active && w.pl + r * w.PL < S;
#pragma unroll
            for (int i = 0; i < VEC; ++i) mean[i / PE] += ok ? v[i] : 0.f;
        }
    const float rn = 1.f / ((float)S * (float)a.Cg);
    block_sum<NE, TH>(mean, red);
    forget<R>(raw);
#pragma unroll
    for (int e = 0; e < NE; ++e) mean[e] *= rn;
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (r * w.PL < S) {
            float v[VEC];
            V::unpack(raw[r], v);
            const bool ok = w.active && w.pl + r * w.PL < S;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float d = ok ? v[i] - mean[i / PE] : 0.f;
                m2[i / PE] = fmaf(d, d, m2[i / PE]);
            }
        }
    block_sum<NE, TH>(m2, red);
    forget<R>(raw);
    float rstd[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) {
        rstd[e] = 1.f / sqrtf(fmaf(m2[e], rn, a.eps));
        if (threadIdx.x == 0) {
            float* s = a.stats + 2 * (w.b * a.G + (long)w.blk * NE + e);
            s[0] = mean[e];
            s[1] = rstd[e];
        }
    }
    if (!w.active) return;
    float k[VEC], b[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        k[i] = a.w ? a.w[c + i] : 1.f;
        b[i] = a.b ? a.b[c + i] : 0.f;
    }
    T* dst = reinterpret_cast<T*>(a.out) + w.b * a.S * a.C + c;
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (w.pl + r * w.PL < S) {
            float v[VEC];
            V::unpack(raw[r], v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = act_of<ACT>(gn_z((v[i] - mean[i / PE]) * rstd[i / PE], k[i], b[i]));
            *reinterpret_cast<typename V::Raw*>(dst + (long)(w.pl + r * w.PL) * a.C) = V::pack(v);
        }
}

template <class T, int VEC, int NE, int R, int TH, int ACT>
__global__ void __launch_bounds__(TH) gn_one_bwd_kernel(GnArgs a) {
    typedef Vec<T, VEC> V;
    constexpr int PE = VEC / NE;
    __shared__ float red[TH / 64][2 * NE];
    __shared__ float s1[TH * VEC / 2], s2[TH * VEC / 2];
    const One<T, VEC, NE, TH> w(a);
    const int c = w.c0 + w.tv * VEC, S = (int)a.S;
    const T* src = reinterpret_cast<const T*>(a.x) + w.b * a.xs_b + c;
    const T* gsrc = reinterpret_cast<const T*>(a.dy) + w.b * a.ds_b + c;
    typename V::Raw raw[R], graw[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (r * w.PL < S) {
            const int p = w.pl + r * w.PL;
            raw[r] = *reinterpret_cast<const typename V::Raw*>(src + (long)(p < S ? p : S - 1) * a.xs_p);
            graw[r] = *reinterpret_cast<const typename V::Raw*>(gsrc + (long)(p < S ? p : S - 1) * a.ds_p);
        }
    float mean[NE], rstd[NE], wt[VEC], bs[VEC], d1[VEC], d2[VEC], q[2 * NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) {
        const float* s = a.stats + 2 * (w.b * a.G + (long)w.blk * NE + e);
        mean[e] = s[0];
        rstd[e] = s[1];
        q[e] = q[NE + e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        wt[i] = a.w ? a.w[c + i] : 1.f;
        bs[i] = a.b ? a.b[c + i] : 0.f;
        d1[i] = d2[i] = 0.f;
    }
    auto dz_of = [&](const typename V::Raw& rx, const typename V::Raw& rg, float (&xh)[VEC], float (&dz)[VEC]) {
        V::unpack(rx, xh);
        V::unpack(rg, dz);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            xh[i] = (xh[i] - mean[i / PE]) * rstd[i / PE];
            dz[i] *= act_slope<ACT>(gn_z(xh[i], wt[i], bs[i]));
        }
    };
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (r * w.PL < S) {
            float xh[VEC], dz[VEC];
            dz_of(raw[r], graw[r], xh, dz);
            const bool ok = w.active && w.pl + r * w.PL < S;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                dz[i] = ok ? dz[i] : 0.f;
                d1[i] += dz[i];
                d2[i] += ok ? dz[i] * xh[i] : 0.f;
            }
        }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        q[i / PE] = fmaf(wt[i], d1[i], q[i / PE]);
        q[NE + i / PE] = fmaf(wt[i], d2[i], q[NE + i / PE]);
    }
    if (a.out) {
        block_sum<2 * NE, TH>(q, red);
        forget<R>(raw);
        forget<R>(graw);
        const float rn = 1.f / ((float)S * (float)a.Cg);
        T* dst = reinterpret_cast<T*>(a.out) + w.b * a.S * a.C + c;
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (w.active && w.pl + r * w.PL < S) {
                float xh[VEC], dz[VEC];
                dz_of(raw[r], graw[r], xh, dz);
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    xh[i] = rstd[i / PE] * (fmaf(dz[i], wt[i], -q[i / PE] * rn) - xh[i] * (q[NE + i / PE] * rn));
                *reinterpret_cast<typename V::Raw*>(dst + (long)(w.pl + r * w.PL) * a.C) = V::pack(xh);
            }
    }
    if (!a.chsum) return;
    // per channel: pairwise over the pixel lanes
    const int e = w.pl * (NE > 1 ? 1 : a.CV) + w.tv;
    for (int n = w.PL; n > 1;) {
        const int half = (n + 1) >> 1, off = half * (NE > 1 ? 1 : a.CV);
        __syncthreads();
        if (w.active && w.pl >= half && w.pl < n)
#pragma unroll
            for (int i = 0; i < VEC; ++i) { s1[(e - off) * VEC + i] = d1[i]; s2[(e - off) * VEC + i] = d2[i]; }
        __syncthreads();
        if (w.active && w.pl + half < n)
#pragma unroll
            for (int i = 0; i < VEC; ++i) { d1[i] += s1[e * VEC + i]; d2[i] += s2[e * VEC + i]; }
        n = half;
    }
    if (w.active && w.pl == 0) {
        // one image: these are the parameters' gradients
        const bool only = a.all && a.B == 1;
        float* o1 = only ? a.db : a.chsum + 2 * w.b * a.C;
        float* o2 = only ? a.dw : a.chsum + (2 * w.b + 1) * a.C;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            if (o1) o1[c + i] = d1[i];
            if (o2) o2[c + i] = d2[i];
        }
    }
}

// bytes a thread holds of each tensor: at most 40 (20) vectors of them, less where the statistics of four groups or more need room.
// Of the workgroups of 1024 threads (128 registers each) the bf16 ones in vectors of 8 still spill: forward with eight groups a
// vector (one channel each) 150 registers, backward 4 to 41 by activation and groups; the others none.
constexpr int hold(bool bwd, int bytes, int ne) { return bwd ? (bytes < 8 ? 20 * bytes : 128) : (bytes < 8 ? 40 * bytes : ne >= 4 ? 128 : 256); }

template <class T, int VEC, int NE, int TH, int HOLD, bool BWD> int launch(const GnArgs& a, int act, hipStream_t st) {
    constexpr int R = HOLD / (int)(sizeof(T) * VEC);
    const dim3 grid((unsigned)(a.B * a.nblk)), block(TH);
#define KSR_GN_ONE(A)                                                                                                          \
    do {                                                                                                                       \
        if constexpr (BWD) hipLaunchKernelGGL((gn_one_bwd_kernel<T, VEC, NE, R, TH, A>), grid, block, 0, st, a);               \
        else hipLaunchKernelGGL((gn_one_fwd_kernel<T, VEC, NE, R, TH, A>), grid, block, 0, st, a);                             \
    } while (0)
    switch (act) {
        case KSR_ACT_NONE: KSR_GN_ONE(KSR_ACT_NONE); break;
        case KSR_ACT_RELU: KSR_GN_ONE(KSR_ACT_RELU); break;
        case KSR_ACT_SILU: KSR_GN_ONE(KSR_ACT_SILU); break;
        default: KSR_GN_ONE(KSR_ACT_GELU); break;
    }
#undef KSR_GN_ONE
    KSR_LAUNCH_CHECK("group_norm");
    return KSR_OK;
}

// 256 threads where that is enough for the group, 1024 otherwise
template <class T, int VEC, int NE, bool BWD> int sized(GnArgs& a, int act, hipStream_t st) {
    constexpr int SMALL = 16 * (sizeof(T) * VEC) < 64 ? 16 * (sizeof(T) * VEC) : 64;
    constexpr long few = SMALL / (long)(sizeof(T) * VEC);
    a.CV = a.CB / VEC;
    if (NE == 1 ? a.CV <= 256 && a.S <= few * (256 / a.CV) : a.S <= few * 256) {
        a.PL = NE == 1 ? 256 / a.CV : 256;
        return launch<T, VEC, NE, 256, SMALL, BWD>(a, act, st);
    }
    a.PL = NE == 1 ? 1024 / a.CV : 1024;
    return launch<T, VEC, NE, 1024, hold(BWD, sizeof(T) * VEC, NE), BWD>(a, act, st);
}

template <bool BWD> int run(GnArgs& a, int act, bool bf16, int vec, int ne, hipStream_t st) {
    a.CB = ne > 1 ? vec : a.Cg;
    a.nblk = a.C / a.CB;
    if (bf16) {
        if (vec == 8) return ne == 1 ? sized<__bf16, 8, 1, BWD>(a, act, st) : ne == 2 ? sized<__bf16, 8, 2, BWD>(a, act, st) : ne == 4 ? sized<__bf16, 8, 4, BWD>(a, act, st) : sized<__bf16, 8, 8, BWD>(a, act, st);
        return vec == 4 ? sized<__bf16, 4, 1, BWD>(a, act, st) : vec == 2 ? sized<__bf16, 2, 1, BWD>(a, act, st) : sized<__bf16, 1, 1, BWD>(a, act, st);
    }
    if (vec == 4) return ne == 1 ? sized<float, 4, 1, BWD>(a, act, st) : ne == 2 ? sized<float, 4, 2, BWD>(a, act, st) : sized<float, 4, 4, BWD>(a, act, st);
    return vec == 2 ? sized<float, 2, 1, BWD>(a, act, st) : sized<float, 1, 1, BWD>(a, act, st);
}

bool aligned(const void* p, long bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }

}  // namespace

bool ksr_gn_one_fits(const GnArgs& a, int esize, bool backward, int& vec, int& ne) {
    // the widest vector that divides strides and addresses and lies in one group, or (16 bytes) holds whole ones
    for (vec = 16 / esize; vec >= 1; vec /= 2) {
        const long bytes = (long)vec * esize;
        if (a.C % vec || a.xs_b % vec || a.xs_p % vec || !aligned(a.x, bytes) || !aligned(a.out, bytes)) continue;
        if (backward && (a.ds_b % vec || a.ds_p % vec || !aligned(a.dy, bytes))) continue;
        if (a.Cg % vec == 0) { ne = 1; break; }
        if (bytes == 16 && vec % a.Cg == 0) { ne = vec / a.Cg; break; }
    }
    if (vec < 1) return false;
    const long cv = ne > 1 ? 1 : a.Cg / vec;
    if (cv > 1024) return false;
    if (a.S > hold(backward, vec * esize, ne) / ((long)vec * esize) * (1024 / cv)) return false;
    // One workgroup has one CU's arithmetic: where there are fewer than 192 of them, a group is taken in one pass up to 16384 values
    // (27 workgroups of 71610 bf16 values with GELU: 31.8 us; in chunks over the whole chip: 13 us)
    const long values = a.S * (ne > 1 ? vec : a.Cg);
    if (a.B * (a.C / (ne > 1 ? vec : a.Cg)) < 192 && values > 16384) return false;
    // Under 16 bytes of a pixel per group (one or two channels that no vector holds together with their neighbours) a workgroup
    // uses little of each cache line it loads: for small tensors only
    return (ne > 1 ? vec : a.Cg) * esize >= 16 || a.S * a.C <= (1 << 18);
}
int ksr_gn_one_fwd(GnArgs& a, int act, bool bf16, int vec, int ne, hipStream_t st) { return run<false>(a, act, bf16, vec, ne, st); }
int ksr_gn_one_bwd(GnArgs& a, int act, bool bf16, int vec, int ne, hipStream_t st) { return run<true>(a, act, bf16, vec, ne, st); }
