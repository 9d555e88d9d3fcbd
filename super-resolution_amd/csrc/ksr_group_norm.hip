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
#include "ksr_group_norm.h"

namespace {

constexpr int THREADS = 256;

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

template <class V, class T> __device__ __forceinline__ typename V::Raw ld(const T* p) { return *reinterpret_cast<const typename V::Raw*>(p); }
// Results past the caches where they are large: the pass that writes them reads x (and dy) a second time, and what of it the
// caches still hold stays there (4 x 512 x 512 x 128 bf16: 155 instead of 174 us).  Smaller results are left to whoever reads next.
template <class V, bool PAST, class T> __device__ __forceinline__ void put(T* p, const typename V::Raw& v) {
    if constexpr (PAST) __builtin_nontemporal_store(v, reinterpret_cast<typename V::Raw*>(p));
    else *reinterpret_cast<typename V::Raw*>(p) = v;
}

// vectors in flight per thread: 64 bytes of 16-byte loads, eight of the narrower ones
template <class T, int VEC> constexpr int in_flight() { return sizeof(T) * VEC == 16 ? 4 : 8; }

// ------------------------------------------------------------------------------------------------ statistics
// NE: entries (mean, M2) of a thread, each over the gcd(VEC, Cg) = VEC / NE neighbouring channels that always share a group
template <class T, int VEC, int NE>
__global__ void __launch_bounds__(THREADS) gn_stats_kernel(GnArgs a) {
    constexpr int PE = VEC / NE, R = in_flight<T, VEC>();
    typedef Vec<T, VEC> V;
    __shared__ float smean[THREADS * NE], sm2[THREADS * NE], sn[THREADS];
    const Place<VEC> w(a, blockIdx.x);
    float mean[NE], m2[NE], n = 0.f;                    // n: values behind each of the NE entries
#pragma unroll
    for (int i = 0; i < NE; ++i) mean[i] = m2[i] = 0.f;
    if (w.active) {
        const T* src = reinterpret_cast<const T*>(a.x) + w.b * a.xs_b + w.c0 + w.tv * VEC;
        typename V::Raw next[R];
#pragma unroll
        for (int r = 0; r < R; ++r) next[r] = ld<V>(src + w.pixel(w.p0 + w.pl, r, a.PL) * a.xs_p);
        for (long base = w.p0 + w.pl; base < w.p1; base += (long)R * a.PL) {
            float v[R][VEC], s[NE], q[NE];
            int cnt = 0;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                V::unpack(next[r], v[r]);
                const bool ok = base + (long)r * a.PL < w.p1;
                cnt += ok;
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[r][i] = ok ? v[r][i] : 0.f;
            }
            // the next tile is on its way while this one is summed
#pragma unroll
            for (int r = 0; r < R; ++r) next[r] = ld<V>(src + w.pixel(base + (long)R * a.PL, r, a.PL) * a.xs_p);
#pragma unroll
            for (int i = 0; i < NE; ++i) s[i] = q[i] = 0.f;
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < VEC; ++i) s[i / PE] += v[r][i];
            const float nt = (float)(cnt * PE), rn = 1.f / nt;
#pragma unroll
            for (int i = 0; i < NE; ++i) s[i] *= rn;                     // the tile's mean
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float d = r < cnt ? v[r][i] - s[i / PE] : 0.f;
                    q[i / PE] = fmaf(d, d, q[i / PE]);
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
    // L lanes per group that this channel block touches, all groups at once if they are few enough: join the entries of its
    // channels and the pixel lanes
    const int g0 = w.c0 / a.Cg, g1 = (w.c0 + w.cb - 1) / a.Cg;
    int L = 64;
    while (L > 4 && THREADS / L <= g1 - g0) L >>= 1;
    const int lane = threadIdx.x & (L - 1);
    auto sum_of = [&](float v) {
        for (int m = L >> 1; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
        return v;
    };
    for (int g = g0 + (int)threadIdx.x / L; g <= g1; g += THREADS / L) {
        const int lo = (g * a.Cg > w.c0 ? g * a.Cg - w.c0 : 0) / PE;
        const int hi = ((g + 1) * a.Cg < w.c0 + w.cb ? (g + 1) * a.Cg - w.c0 : w.cb) / PE, ne = hi - lo;
        float cnt = 0.f, sum = 0.f;
        for (int e = lane; e < a.PL * ne; e += L) {
            const int pl = e / ne;
            cnt += sn[pl];
            sum = fmaf(sn[pl], smean[pl * a.CV * NE + lo + e - pl * ne], sum);
        }
        cnt = sum_of(cnt);
        const float m = sum_of(sum) / cnt;
        float q = 0.f;
        for (int e = lane; e < a.PL * ne; e += L) {
            const int pl = e / ne, k = pl * a.CV * NE + lo + e - pl * ne;
            const float d = smean[k] - m;
            q += fmaf(sn[pl] * d, d, sm2[k]);
        }
        q = sum_of(q);
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

// The same inside the pass that uses it, where an image has few chunks: all groups of the image (G <= 256, one channel block) to
// st, 256 / 2^k lanes per group; saves a launch.
__device__ __forceinline__ void join_stats(const GnArgs& a, long b, float2* st, float (*lds)[3]) {
    int tg = 1;
    while (tg < a.G) tg *= 2;
    const int t = threadIdx.x, g = t & (tg - 1), k0 = t / tg, kl = THREADS / tg;
    float n = 0.f, m = 0.f, q = 0.f;
    if (g < a.G)
#pragma unroll 4
        for (int c = k0; c < (int)a.nchunk; c += kl) {
            const float2 p = *reinterpret_cast<const float2*>(a.part + 2 * ((b * a.nchunk + c) * a.GB + g));
            const long left = a.S - c * a.chunk;
            const float nc = (float)(left < a.chunk ? left : a.chunk) * (float)a.Cg, f = nc / (n + nc), d = p.x - m;
            m = fmaf(d, f, m);
            q += fmaf(d, d * f * n, p.y);
            n += nc;
        }
    for (int h = kl >> 1; h > 0; h >>= 1) {
        if (k0 >= h && k0 < 2 * h) { lds[t][0] = n; lds[t][1] = m; lds[t][2] = q; }
        __syncthreads();
        if (k0 < h) {
            const float* o = lds[t + h * tg];
            if (o[0] > 0.f) {
                const float f = o[0] / (n + o[0]), d = o[1] - m;
                m = fmaf(d, f, m);
                q += fmaf(d, d * f * n, o[2]);
                n += o[0];
            }
        }
        __syncthreads();
    }
    if (k0 == 0 && g < a.G) st[g] = make_float2(m, 1.f / sqrtf(fmaf(q, 1.f / n, a.eps)));
    __syncthreads();
}

// the thread's channels: mean, rstd of their groups (stats: of the image), weight and bias
template <int VEC> struct Affine {
    float mean[VEC], rstd[VEC], w[VEC], b[VEC];
    __device__ __forceinline__ Affine(const GnArgs& a, const float* stats, int c) {
        int g = c / a.Cg, r = c - g * a.Cg;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float* s = stats + 2 * g;
            if (++r == a.Cg) { r = 0; ++g; }
            mean[i] = s[0];
            rstd[i] = s[1];
            w[i] = a.w ? a.w[c + i] : 1.f;
            b[i] = a.b ? a.b[c + i] : 0.f;
        }
    }
};

// ------------------------------------------------------------------------------------------------ y = act(w xhat + b)
template <class T, int VEC, int ACT, bool PAST>
__global__ void __launch_bounds__(THREADS) gn_apply_kernel(GnArgs a) {
    constexpr int R = in_flight<T, VEC>();
    typedef Vec<T, VEC> V;
    __shared__ float2 st[THREADS];
    __shared__ float lds[THREADS][3];
    // the chunks that were read last are the likeliest to be in the caches still
    const Place<VEC> w(a, (long)gridDim.x - 1 - blockIdx.x);
    const float* stats = a.stats + 2 * w.b * a.G;
    if (a.join) {
        join_stats(a, w.b, st, lds);
        stats = reinterpret_cast<const float*>(st);
        if (w.chunk == 0 && (int)threadIdx.x < a.G) reinterpret_cast<float2*>(a.stats)[w.b * a.G + threadIdx.x] = st[threadIdx.x];
    }
    if (!w.active) return;
    const int c = w.c0 + w.tv * VEC;
    const Affine<VEC> k(a, stats, c);
    const T* src = reinterpret_cast<const T*>(a.x) + w.b * a.xs_b + c;
    T* dst = reinterpret_cast<T*>(a.out) + w.b * a.S * a.C + c;
    typename V::Raw next[R];
#pragma unroll
    for (int r = 0; r < R; ++r) next[r] = ld<V>(src + w.pixel(w.p0 + w.pl, r, a.PL) * a.xs_p);
    for (long base = w.p0 + w.pl; base < w.p1; base += (long)R * a.PL) {
        typename V::Raw raw[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            raw[r] = next[r];
            next[r] = ld<V>(src + w.pixel(base + (long)R * a.PL, r, a.PL) * a.xs_p);
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (base + (long)r * a.PL < w.p1) {
                float v[VEC];
                V::unpack(raw[r], v);
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[i] = act_of<ACT>(gn_z((v[i] - k.mean[i]) * k.rstd[i], k.w[i], k.b[i]));
                put<V, PAST>(dst + (base + (long)r * a.PL) * a.C, V::pack(v));
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
        const Affine<VEC> k(a, a.stats + 2 * w.b * a.G, c);
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
                        const float dz = g[i] * act_slope<ACT>(gn_z(xh, k.w[i], k.b[i]));
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
    #pragma unroll 4
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

// dw, db: [rows][2][C] sums (images, or their chunks) over the rows; 2^k >= C channels (at most 64) per workgroup, the other
// lanes along the rows
__device__ __forceinline__ void sum_params(const GnArgs& a, const float* rows, long n, int wg, float (*lds)[2]) {
    int tc = 1;
    while (tc < a.C && tc < 64) tc *= 2;
    const int t = threadIdx.x, c = wg * tc + (t & (tc - 1)), k0 = t / tc, kl = THREADS / tc;
    float v1 = 0.f, v2 = 0.f;
    if (c < a.C)
#pragma unroll 4
        for (long k = k0; k < n; k += kl) {
            v1 += rows[2 * k * a.C + c];
            v2 += rows[(2 * k + 1) * a.C + c];
        }
    lds[t][0] = v1;
    lds[t][1] = v2;
    __syncthreads();
    for (int h = kl >> 1; h > 0; h >>= 1) {
        if (k0 < h) { lds[t][0] += lds[t + h * tc][0]; lds[t][1] += lds[t + h * tc][1]; }
        __syncthreads();
    }
    if (k0 == 0 && c < a.C) {
        if (a.db) a.db[c] = lds[t][0];
        if (a.dw) a.dw[c] = lds[t][1];
    }
}
int params_wgs(int C) {
    int tc = 1;
    while (tc < C && tc < 64) tc *= 2;
    return (C + tc - 1) / tc;
}

__global__ void __launch_bounds__(THREADS) gn_bwd_params_kernel(GnArgs a) {
    __shared__ float lds[THREADS][2];
    sum_params(a, a.chsum, a.B, (int)blockIdx.x, lds);
}

// gn_bwd_join_kernel's coefficients inside the pass that uses them, where an image has few chunks and channels (C <= 256, one
// block): st[g] = mean(w dz), mean(w dz xhat)
__device__ __forceinline__ void join_coef(const GnArgs& a, long b, float2* st, float (*lds)[2]) {
    int tc = 1;
    while (tc < a.C) tc *= 2;
    const int t = threadIdx.x, c = t & (tc - 1), k0 = t / tc, kl = THREADS / tc;
    float v1 = 0.f, v2 = 0.f;
    if (c < a.C)
#pragma unroll 4
        for (int k = k0; k < (int)a.nchunk; k += kl) {
            const float* p = a.part + 2 * (b * a.nchunk + k) * a.C + c;
            v1 += p[0];
            v2 += p[a.C];
        }
    const float w = c < a.C && a.w ? a.w[c] : 1.f;
    lds[t][0] = v1 * w;
    lds[t][1] = v2 * w;
    __syncthreads();
    for (int h = kl >> 1; h > 0; h >>= 1) {
        if (k0 < h) { lds[t][0] += lds[t + h * tc][0]; lds[t][1] += lds[t + h * tc][1]; }
        __syncthreads();
    }
    if (t < a.G) {
        float s1 = 0.f, s2 = 0.f;
        for (int i = 0; i < a.Cg; ++i) { s1 += lds[t * a.Cg + i][0]; s2 += lds[t * a.Cg + i][1]; }
        const float rn = 1.f / ((float)a.S * (float)a.Cg);
        st[t] = make_float2(s1 * rn, s2 * rn);
    }
    __syncthreads();
}

// dx; the last workgroups (with a.dw or a.db) sum the parameters' gradients
template <class T, int VEC, int ACT, bool PAST>
__global__ void __launch_bounds__(THREADS) gn_bwd_dx_kernel(GnArgs a) {
    constexpr int R = in_flight<T, VEC>() / 2;
    typedef Vec<T, VEC> V;
    __shared__ float2 st[THREADS];
    __shared__ float lds[THREADS][2];
    const long work = a.out ? a.B * a.nblk * a.nchunk : 0;
    if ((long)blockIdx.x >= work) {
        if (a.join) sum_params(a, a.part, a.B * a.nchunk, (int)(blockIdx.x - work), lds);
        else sum_params(a, a.chsum, a.B, (int)(blockIdx.x - work), lds);
        return;
    }
    const Place<VEC> w(a, work - 1 - blockIdx.x);
    const float* coef = a.coef + 2 * w.b * a.G;
    if (a.join) {
        join_coef(a, w.b, st, lds);
        coef = reinterpret_cast<const float*>(st);
    }
    if (!w.active) return;
    const int c = w.c0 + w.tv * VEC;
    const Affine<VEC> k(a, a.stats + 2 * w.b * a.G, c);
    float q1[VEC], q2[VEC];
    int g = c / a.Cg, r = c - g * a.Cg;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const float* s = coef + 2 * g;
        if (++r == a.Cg) { r = 0; ++g; }
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
            raw[r] = ld<V>(src + w.pixel(base, r, a.PL) * a.xs_p);
            graw[r] = ld<V>(gsrc + w.pixel(base, r, a.PL) * a.ds_p);
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
                    const float dz = g[i] * act_slope<ACT>(gn_z(xh, k.w[i], k.b[i]));
                    v[i] = k.rstd[i] * (fmaf(dz, k.w[i], -q1[i]) - xh * q2[i]);
                }
                put<V, PAST>(dst + (base + (long)r * a.PL) * a.C, V::pack(v));
            }
    }
}

// ------------------------------------------------------------------------------------------------ host
// Number of workgroups that the chunks of a pass aim at: eight 256-thread workgroups on each of 256 CUs; fewer, down to two, where
// a workgroup would have less than MIN_TILES turns of its loop, whose start and join then cost more than its work
// (2 x 128 x 128 x 320 bf16, one turn: statistics and result 10.2 + 17.4 us; three: 8.9 + 12.4 us).
constexpr long AIM_WGS = 2048, LEAST_WGS = 512, MIN_TILES = 8;
// Chunks that the pass which uses their results joins itself, rather than a launch in between: as many values a workgroup reads
constexpr long JOIN_VALUES = 4096;
constexpr int64_t PAST_BYTES = 64 << 20;            // results of a quarter of the last-level cache or more are written past it

// Split of [B, S, C] for a vector of `vec` channels, `inflight` pixels a thread holds at once.  A chunk has G (forward) or C
// (backward) results; half as many chunks as would fit are taken if they can be joined without a launch (one channel block, at
// most THREADS results) and each CU still has a workgroup (the case above: one launch of 6 us less, 1 us more in each pass).
void split(GnArgs& a, int vec, int inflight, bool backward) {
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
    const long few = tiles / MIN_TILES, least = LEAST_WGS / (a.B * a.nblk);
    if (want > few) want = few > least ? few : least;
    const int results = backward ? a.C : a.G;
    const long joined = JOIN_VALUES / results;
    const bool joins = a.nblk == 1 && results <= THREADS;
    if (joins && want > joined && want <= 2 * joined && 2 * joined * a.B >= LEAST_WGS) want = joined;
    if (want < 1) want = 1;
    if (want > tiles) want = tiles;
    a.chunk = (tiles + want - 1) / want * tile;
    a.nchunk = (a.S + a.chunk - 1) / a.chunk;
    a.join = joins && a.nchunk * results <= JOIN_VALUES;
}

// most chunks that split() makes for any vector width
long max_parts(long B, long S, int C, int G, bool backward) {
    long most = 0;
    for (int vec = 1; vec <= 8; vec *= 2)
        for (int fl = 2; fl <= 8; fl *= 2) {
            if (C % vec) continue;
            GnArgs a{};
            a.B = B; a.S = S; a.C = C; a.G = G; a.Cg = C / G;
            split(a, vec, fl, backward);
            const long n = B * a.nchunk * 2 * (backward ? C : (long)a.nblk * a.GB);
            if (n > most) most = n;
        }
    return most;
}

bool aligned(const void* p, long bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }

// widest vector that divides the channels, the strides and every address
int vec_of(const GnArgs& a, int esize, bool backward) {
    for (int vec = 16 / esize; vec > 1; vec /= 2) {
        const long bytes = (long)vec * esize;
        bool ok = a.C % vec == 0 && a.xs_b % vec == 0 && a.xs_p % vec == 0 && aligned(a.x, bytes) && aligned(a.out, bytes);
        if (backward) ok = ok && a.ds_b % vec == 0 && a.ds_p % vec == 0 && aligned(a.dy, bytes);
        if (ok) return vec;
    }
    return 1;
}

template <class T, int VEC> void stats(const GnArgs& a, dim3 grid, hipStream_t st) {
    const dim3 block(THREADS);
    int per = VEC;                                      // gcd(VEC, Cg): VEC is a power of two
    while (a.Cg % per) per >>= 1;
    if (per == VEC) hipLaunchKernelGGL((gn_stats_kernel<T, VEC, 1>), grid, block, 0, st, a);
    else if (VEC > 2 && 2 * per == VEC) hipLaunchKernelGGL((gn_stats_kernel<T, VEC, (VEC > 2 ? 2 : 1)>), grid, block, 0, st, a);
    else if (VEC > 4 && 4 * per == VEC) hipLaunchKernelGGL((gn_stats_kernel<T, VEC, (VEC > 4 ? 4 : 1)>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((gn_stats_kernel<T, VEC, VEC>), grid, block, 0, st, a);
}

template <class T, int VEC, int ACT> void apply(const GnArgs& a, dim3 grid, hipStream_t st) {
    if (a.past) hipLaunchKernelGGL((gn_apply_kernel<T, VEC, ACT, true>), grid, dim3(THREADS), 0, st, a);
    else hipLaunchKernelGGL((gn_apply_kernel<T, VEC, ACT, false>), grid, dim3(THREADS), 0, st, a);
}

template <class T, int VEC> int run_fwd(GnArgs& a, int act, hipStream_t st) {
    split(a, VEC, in_flight<T, VEC>(), false);
    const dim3 grid((unsigned)(a.B * a.nblk * a.nchunk)), block(THREADS);
    stats<T, VEC>(a, grid, st);
    KSR_LAUNCH_CHECK("group_norm_fwd");
    if (!a.join) {
        hipLaunchKernelGGL(gn_stats_join_kernel, dim3((unsigned)((a.B * a.G + 3) / 4)), block, 0, st, a);
        KSR_LAUNCH_CHECK("group_norm_fwd");
    }
    switch (act) {
        case KSR_ACT_NONE: apply<T, VEC, KSR_ACT_NONE>(a, grid, st); break;
        case KSR_ACT_RELU: apply<T, VEC, KSR_ACT_RELU>(a, grid, st); break;
        case KSR_ACT_SILU: apply<T, VEC, KSR_ACT_SILU>(a, grid, st); break;
        default: apply<T, VEC, KSR_ACT_GELU>(a, grid, st); break;
    }
    KSR_LAUNCH_CHECK("group_norm_fwd");
    return KSR_OK;
}

template <class T, int VEC, int ACT> int run_bwd_act(GnArgs& a, hipStream_t st) {
    split(a, VEC, in_flight<T, VEC>() / 2, true);
    if (!a.all) a.join = 0;                             // the images' channel sums are needed beyond this launch
    const dim3 block(THREADS);
    const long work = a.B * a.nblk * a.nchunk;
    hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, VEC, ACT>), dim3((unsigned)work), block, 0, st, a);
    KSR_LAUNCH_CHECK("group_norm_bwd");
    if (!a.join) {
        int tc = 1;
        while (tc < a.Cg && tc < 64) tc *= 2;
        hipLaunchKernelGGL(gn_bwd_join_kernel, dim3((unsigned)(a.B * a.G)), block, 0, st, a, tc);
        KSR_LAUNCH_CHECK("group_norm_bwd");
    }
    const long wgs = (a.out ? work : 0) + (a.all && (a.dw || a.db) ? params_wgs(a.C) : 0);
    if (wgs) {
        if (a.past) hipLaunchKernelGGL((gn_bwd_dx_kernel<T, VEC, ACT, true>), dim3((unsigned)wgs), block, 0, st, a);
        else hipLaunchKernelGGL((gn_bwd_dx_kernel<T, VEC, ACT, false>), dim3((unsigned)wgs), block, 0, st, a);
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

// A launch holds fewer than 2^32 threads.  No kernel has more workgroups per image than max(G, C / 256), beyond the few thousand of
// small batches; they have 256 threads, 1024 only where a group of an image has more than 256 values.
long images_at_once(int64_t S, int C, int G) {
    const long threads = S > 256 || S * (C / G) > 256 ? 1024 : 256, per = G > (C + 255) / 256 ? G : (C + 255) / 256;
    return ((1l << 32) / threads - 1 - 4096) / per;
}

int check_shape(const char* what, int64_t B, int64_t S, int C, int G) {
    KSR_CHECK_ARG(B >= 0 && S >= 0 && C > 0 && G > 0 && C % G == 0, "%s: [%lld, %lld, %d] in %d groups", what, (long long)B,
                  (long long)S, C, G);
    KSR_UNSUPPORTED(B > (1 << 24) || S > (1ll << 40) || B * (int64_t)G > (1ll << 30) || B * ((C + 255) / 256) > (1ll << 30),
                    "%s: [%lld, %lld, %d] is beyond the launch limits", what, (long long)B, (long long)S, C);
    KSR_UNSUPPORTED(images_at_once(S, C, G) < 1, "%s: an image [%lld, %d] in %d groups is beyond the launch limits", what, (long long)S, C, G);
    return KSR_OK;
}

// the images in as many equal ranges as images_at_once() asks for: images of a range, f(first image, images) for each
long range_of(int64_t B, int64_t S, int C, int G) {
    const long most = images_at_once(S, C, G), n = (B + most - 1) / most;
    return (B + n - 1) / n;
}
template <class F> int for_ranges(int64_t B, int64_t S, int C, int G, F f) {
    const long nb = range_of(B, S, C, G);
    for (long b0 = 0; b0 < B; b0 += nb)
        if (int rc = f(b0, nb < B - b0 ? nb : B - b0)) return rc;
    return KSR_OK;
}

}  // namespace

extern "C" int64_t ksr_group_norm_ws_floats(int64_t B, int64_t S, int C, int G, int backward) {
    if (check_shape("group_norm_ws_floats", B, S, C, G) != KSR_OK) return -1;
    if (B == 0 || S == 0) return 0;
    int64_t most = 0;
    for_ranges(B, S, C, G, [&](long, long n) {
        const int64_t parts = max_parts(n, S, C, G, backward != 0);
        if (parts > most) most = parts;
        return KSR_OK;
    });
    return most + (backward ? 2 * B * G + 2 * B * C : 0);
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
    const int es = bf16 ? 2 : 4;
    return for_ranges(B, S, C, G, [&](long b0, long n) {
        GnArgs a{};
        a.x = reinterpret_cast<const char*>(x) + b0 * x_image_stride * es; a.out = reinterpret_cast<char*>(y) + b0 * S * C * es;
        a.w = weight; a.b = bias; a.stats = stats + 2 * b0 * G; a.part = ws;
        a.xs_b = x_image_stride; a.xs_p = x_pixel_stride;
        a.B = n; a.S = S; a.C = C; a.G = G; a.Cg = C / G; a.eps = eps;
        a.past = n * S * C * es >= PAST_BYTES;
        int vec, ne;
        if (ksr_gn_one_fits(a, es, false, vec, ne)) return ksr_gn_one_fwd(a, act, bf16 != 0, vec, ne, stream);
        vec = vec_of(a, es, false);
        if (bf16)
            return vec == 8 ? run_fwd<__bf16, 8>(a, act, stream) : vec == 4 ? run_fwd<__bf16, 4>(a, act, stream) : vec == 2 ? run_fwd<__bf16, 2>(a, act, stream) : run_fwd<__bf16, 1>(a, act, stream);
        return vec == 4 ? run_fwd<float, 4>(a, act, stream) : vec == 2 ? run_fwd<float, 2>(a, act, stream) : run_fwd<float, 1>(a, act, stream);
    });
}

extern "C" int ksr_group_norm_bwd(const void* x, int64_t x_image_stride, int64_t x_pixel_stride, const void* dy, int64_t dy_image_stride,
                                  int64_t dy_pixel_stride, const float* weight, const float* bias, const float* stats, void* dx,
                                  float* dweight, float* dbias, float* ws, int64_t B, int64_t S, int C, int G, int act, int bf16,
                                  hipStream_t stream) {
    if (int rc = check_shape("group_norm_bwd", B, S, C, G)) return rc;
    KSR_CHECK_ARG(act >= KSR_ACT_NONE && act <= KSR_ACT_GELU, "group_norm_bwd: activation %d", act);
    if (B == 0 || S == 0) {                               // empty sums
        GnArgs a{};
        a.C = C; a.dw = dweight; a.db = dbias;
        if (!dweight && !dbias) return KSR_OK;
        hipLaunchKernelGGL(gn_bwd_params_kernel, dim3((unsigned)params_wgs(C)), dim3(THREADS), 0, stream, a);
        KSR_LAUNCH_CHECK("group_norm_bwd");
        return KSR_OK;
    }
    KSR_CHECK_ARG(x && dy && stats && ws, "group_norm_bwd: null pointer");
    KSR_CHECK_ARG(x_pixel_stride >= 0 && x_image_stride >= 0 && dy_pixel_stride >= 0 && dy_image_stride >= 0, "group_norm_bwd: negative stride");
    KSR_CHECK_ARG(aligned(x, bf16 ? 2 : 4) && aligned(dy, bf16 ? 2 : 4) && aligned(dx, bf16 ? 2 : 4), "group_norm_bwd: misaligned pointer");
    const int es = bf16 ? 2 : 4;
    float* const coef = ws;
    float* const chsum = coef + 2 * B * G;
    bool later = false;                                   // the parameters' gradients are left to be summed over the images
    const int rc = for_ranges(B, S, C, G, [&](long b0, long n) {
        GnArgs a{};
        a.x = reinterpret_cast<const char*>(x) + b0 * x_image_stride * es; a.dy = reinterpret_cast<const char*>(dy) + b0 * dy_image_stride * es;
        a.out = dx ? reinterpret_cast<char*>(dx) + b0 * S * C * es : nullptr;
        a.w = weight; a.b = bias; a.stats = const_cast<float*>(stats) + 2 * b0 * G; a.dw = dweight; a.db = dbias;
        a.xs_b = x_image_stride; a.xs_p = x_pixel_stride; a.ds_b = dy_image_stride; a.ds_p = dy_pixel_stride;
        a.B = n; a.S = S; a.C = C; a.G = G; a.Cg = C / G;
        a.past = n * S * C * es >= PAST_BYTES;
        a.all = n == B;
        a.coef = coef + 2 * b0 * G; a.chsum = chsum + 2 * b0 * C; a.part = chsum + 2 * B * C;
        int vec, ne;
        if (ksr_gn_one_fits(a, es, true, vec, ne)) {
            if (!dweight && !dbias) a.chsum = nullptr;
            later = B > 1 && a.chsum;
            return ksr_gn_one_bwd(a, act, bf16 != 0, vec, ne, stream);
        }
        later = !a.all && (dweight || dbias);
        vec = vec_of(a, es, true);
        if (bf16)
            return vec == 8 ? run_bwd<__bf16, 8>(a, act, stream) : vec == 4 ? run_bwd<__bf16, 4>(a, act, stream) : vec == 2 ? run_bwd<__bf16, 2>(a, act, stream) : run_bwd<__bf16, 1>(a, act, stream);
        return vec == 4 ? run_bwd<float, 4>(a, act, stream) : vec == 2 ? run_bwd<float, 2>(a, act, stream) : run_bwd<float, 1>(a, act, stream);
    });
    if (rc || !later) return rc;
    GnArgs a{};
    a.B = B; a.C = C; a.chsum = chsum; a.dw = dweight; a.db = dbias;
    hipLaunchKernelGGL(gn_bwd_params_kernel, dim3((unsigned)params_wgs(C)), dim3(THREADS), 0, stream, a);
    KSR_LAUNCH_CHECK("group_norm_bwd");
    return KSR_OK;
}
