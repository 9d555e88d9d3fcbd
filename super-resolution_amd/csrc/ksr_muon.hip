// Orthogonalisation of matrices by Newton-Schulz products, and the Muon update that uses it.
//   X0 = U / (|U|_F + eps), transposed where U has more rows than columns: X [m, n], m <= n; then `steps` times
//   A = X X^T,   B = b A + c A^2,   X <- a X + B X;      Muon: W <- (1 - lr wd) W - lr scale X.
// Arithmetic: 2 m^2 n for A and 2 m^3 for A^2 (both symmetric: half of it is computed) and 2 m^2 n for B X.
//
// All products run on the f16 matrix cores with fp32 accumulation.  Numbers are held as S x value (S = 2^10, X0 by a power of
// two of its own) in one f16 plane, or as hi + lo in two:
//   SPLIT   operands hi + lo (22 bits), three products hi hi + hi lo + lo hi: as close to 64 bits as fp32 products, at 5 times
//           the fp32 matrix instruction's rate (the dropped lo lo is below 2^-22 of a product).  For fp32 results.
//   single  operands rounded to f16 (11 bits).  For bf16 results: 8 bits.
// What a single f16 rounding would lose is kept out of it: diagonals of A and B, which are far larger than the rest, stay in
// fp32 vectors (A = D + R, A^2 = D^2 + D R + R D + R^2; B likewise), and the linear term a X + diag(B) X takes X as hi + lo.
// With that the single form is 2e-4 to 9e-4 off the 64-bit result (plain f16 products: 4e-3, bf16 products: 3e-2), less than the
// 1.7e-3 of rounding the result to bf16.
#include "ksr_common.h"
#include "ksr.h"

#include <math.h>

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));

constexpr float S = 1024.f, INV_S = 1.f / 1024.f;     // values up to 30 (checked on the host) fit f16
constexpr int MAX_STEPS = 32, MAX_MATS = 40;
constexpr int NORM_PARTS = 64;                        // partial sums of squares per matrix (large path)

struct Mat {
    const void* src;          // U, or the gradient
    void* dst;                // the orthogonalised matrix (dense, type of src), or the weight to update (fp32, dense)
    float* mom;               // Muon: momentum (fp32, dense)
    long rs, cs, bs;          // strides of src in elements: row, column, matrix
    int rows, cols, batch, first;
};

struct Step {
    int steps, bf16, muon, nesterov;
    float a, b, c, eps, gain;             // gain: most by which a step multiplies a singular value
    float momentum, grad_scale, lr, wd, scale;
    const float* lr_dev;                  // replaces lr
};

struct Mats { Mat m[MAX_MATS]; int count; Step s; };

__device__ __forceinline__ const Mat& find(const Mats& p, int i, int& sub) {
    int k = 0;
    while (k + 1 < p.count && i >= p.m[k + 1].first) ++k;
    sub = i - p.m[k].first;
    return p.m[k];
}

// What a call reads and writes: fp32 -> fp32, bf16 -> bf16, or gradient and momentum -> weight
enum { F32, BF16, MUON };
int mode_of(const Step& s) { return s.muon ? MUON : s.bf16 ? BF16 : F32; }

// value of U at (r, c) of matrix `sub`; WRITE: the momentum is updated (once per step and element).
// Muon: m <- momentum m + g and U = g + momentum m (Nesterov) or m, as ug g + um m
template <int MODE, bool WRITE>
__device__ __forceinline__ float load_u(const Step& s, const Mat& m, int sub, int r, int c) {
    const long o = (long)sub * m.bs + (long)r * m.rs + (long)c * m.cs;
    if constexpr (MODE == BF16) return (float)reinterpret_cast<const __bf16*>(m.src)[o];
    const float g = reinterpret_cast<const float*>(m.src)[o];
    if constexpr (MODE == F32) return g;
    float* mp = m.mom + ((long)sub * m.rows + r) * m.cols + c;
    const float gs = g * s.grad_scale;
    float mo = *mp;
    if (WRITE) {
        mo = fmaf(s.momentum, mo, gs);
        *mp = mo;
    }
    return s.nesterov ? fmaf(s.momentum, mo, gs) : mo;
}

// W <- keep W - rate X, or the result itself
struct Apply {
    float keep, rate;
    __device__ __forceinline__ Apply(const Step& s, const Mat& m) {
        const float lr = s.lr_dev ? *s.lr_dev : s.lr;
        keep = 1.f - lr * s.wd;
        rate = lr * s.scale * sqrtf((float)(m.rows > m.cols ? m.rows : m.cols));
    }
    template <int MODE> __device__ __forceinline__ void store(const Mat& m, long o, float v) const {
        if constexpr (MODE == MUON) {
            float* w = reinterpret_cast<float*>(m.dst) + o;
            *w = fmaf(-rate, v, *w * keep);
        } else if constexpr (MODE == BF16) reinterpret_cast<__bf16*>(m.dst)[o] = (__bf16)v;
        else reinterpret_cast<float*>(m.dst)[o] = v;
    }
};

// Scales of one matrix from the sum of its squares: U is stored as 2^e U (norm in [2^14, 2^15)), X_k as X_k / xi[k].
// xi[k] = 2^-10, smaller by a power of two while X_k is still tiny (a norm below eps), so that f16 keeps its bits.
__device__ __forceinline__ float scales(const Step& s, double sumsq, int& e) {
    const double norm = sqrt(sumsq);
    e = 0;
    if (!(norm < INFINITY)) return NAN;              // infinities and NaN: everything becomes NaN
    if (norm > 0) { (void)frexp(norm, &e); e = 15 - e; }
    return (float)(ldexp(1.0 / (norm + (double)s.eps), -e));
}
__device__ __forceinline__ float scale_of(const Step& s, double sumsq, int k) {
    const double norm = sqrt(sumsq), nu = norm / (norm + (double)s.eps);
    double lg = nu > 0 ? -log2(nu) - k * (double)log2f(s.gain) : 0.0;
    lg = lg > 0 ? (lg < 100 ? floor(lg) : 100.0) : 0.0;
    return (float)ldexp(1.0, -10 - (int)lg);
}

__device__ __forceinline__ float scaled(float u, int e) {       // u 2^e, also where 2^e is beyond a float's range
    return ldexpf(u, e);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
    return v;
}

// ================================================================================================ small matrices
// m <= 64, n <= 1024: one workgroup of eight waves per matrix runs the whole iteration.  X stays in registers: a wave owns NS
// slabs of 32 columns in the accumulator layout of v_mfma_f32_32x32x16 (lane = column, register r = row 8 (r/4) + 4 (lane/32) +
// r%4), which is the B operand's layout for the next product when both operands take k in that order.  Always SPLIT (the time
// is latency).  LDS: partial sums of A per wave, R and B in hi and lo, one slab per wave on its way to X X^T.
constexpr int LD = 72;                                  // halves per row of R, B and a slab: 144 bytes

struct SmallLds {
    union {
        float part[8][3 * 1024];                        // 96 KB: A's three 32 x 32 tiles per wave
        _Float16 slab[8][2][32 * LD];                   // 72 KB: [column][row], hi and lo
    };
    _Float16 r[2][64 * LD], bm[2][64 * LD];             // 36 KB
    float d[64], ae[64];                                // diagonal of A; a + diagonal of B
    double sq[8];
};

__device__ __forceinline__ int acc_row(int r, int lane) { return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3); }

__device__ __forceinline__ f32x16 mfma(const h8& a, const h8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// (hi + lo)(hi + lo) without lo lo
__device__ __forceinline__ f32x16 mfma3(const h8& ah, const h8& al, const h8& bh, const h8& bl, f32x16 c) {
    c = mfma(al, bh, c);
    c = mfma(ah, bl, c);
    return mfma(ah, bh, c);
}

__device__ __forceinline__ h4 lds_tr4(const _Float16* p) {      // transposed read: see frag_of_slab
    const s4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p));
    h4 o;
    __builtin_memcpy(&o, &v, 8);
    return o;
}
// Operand of X X^T from a slab stored [column][row]: lane = row 32 t + lane%32, k = columns 16 s + 8 (lane/32) .. + 7.
// The transposed read hands lane i of a 16-lane group column i of the 4 x 16 block whose row q starts at lane 4 q + p's address.
__device__ __forceinline__ h8 frag_of_slab(const _Float16* slab, int t, int s, int lane) {
    const int grp = lane >> 4, li = lane & 15, q = li >> 2, pp = li & 3;
    const _Float16* p = slab + (16 * s + 8 * (grp >> 1) + q) * LD + 32 * t + 16 * (grp & 1) + 4 * pp;
    const h4 lo = lds_tr4(p), hi = lds_tr4(p + 4 * LD);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
// rows of R or B as an operand with k in natural order / in accumulator order (see above)
__device__ __forceinline__ h8 frag_row(const _Float16* mat, int t, int s, int lane) {
    return *reinterpret_cast<const h8*>(mat + (32 * t + (lane & 31)) * LD + 16 * s + 8 * (lane >> 5));
}
__device__ __forceinline__ h8 frag_row_acc(const _Float16* mat, int t, int s, int lane) {
    const _Float16* p = mat + (32 * t + (lane & 31)) * LD + 16 * s + 4 * (lane >> 5);
    const h4 x = *reinterpret_cast<const h4*>(p), y = *reinterpret_cast<const h4*>(p + 8);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ void put2(_Float16 (&mat)[2][64 * LD], int r, int c, float v) {
    const _Float16 hi = (_Float16)v;
    mat[0][r * LD + c] = hi;
    mat[1][r * LD + c] = (_Float16)(v - (float)hi);
}

template <int MODE, int NS>
__device__ __forceinline__ void small_body(const Mats& p, const Mat& mt, int sub, SmallLds& L) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31;
    const bool tall = mt.rows > mt.cols;
    const int m = tall ? mt.cols : mt.rows, n = tall ? mt.rows : mt.cols, slabs = (n + 31) >> 5;
    // sum of squares, the momentum updated on the way; neighbouring threads along U's contiguous dimension
    double sq = 0;
    {
        const bool by_col = mt.cs <= mt.rs;
        const int inner = by_col ? mt.cols : mt.rows, total = mt.rows * mt.cols;
        for (int t = threadIdx.x; t < total; t += 512) {
            const int o = t / inner, i = t - o * inner;
            const double u = load_u<MODE, true>(p.s, mt, sub, by_col ? o : i, by_col ? i : o);
            sq = fma(u, u, sq);
        }
    }
    sq = wave_sum(sq);
    if (lane == 0) L.sq[wave] = sq;
    __threadfence_block();
    __syncthreads();
    double total = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) total += L.sq[w];
    int e;
    float xi = scales(p.s, total, e);
    // slab s of this wave: columns 32 (wave + 8 s) ..
    h8 xh[NS][4], xl[NS][4];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int j = 32 * (wave + 8 * s) + col, jc = j < n ? j : n - 1;
#pragma unroll
        for (int r = 0; r < 32; ++r) {
            const int i = 32 * (r >> 4) + acc_row(r & 15, lane), ic = i < m ? i : m - 1;
            const float u = load_u<MODE, false>(p.s, mt, sub, tall ? jc : ic, tall ? ic : jc);
            const float v = i < m && j < n ? scaled(u, e) : 0.f;
            const _Float16 hi = (_Float16)v;
            xh[s][r >> 3][r & 7] = hi;
            xl[s][r >> 3][r & 7] = (_Float16)(v - (float)hi);
            if ((r & 7) == 7) __builtin_amdgcn_sched_barrier(0);      // eight loads in flight: more addresses would spill
        }
    }
    const Apply ap(p.s, mt);
    const int lane0 = lane;
    for (int k = 0; k < p.s.steps; ++k) {
        // an index the compiler cannot follow: it would otherwise keep every address and bound of the last step's stores (more
        // than 256 registers) through all steps
        int lane = lane0;
        asm volatile("" : "+v"(lane));
        const int col = lane & 31;
        // ---- A = X X^T: each wave over its own columns
        f32x16 acc[3] = {};
#pragma unroll
        for (int s = 0; s < NS; ++s)
            if (wave + 8 * s < slabs) {
#pragma unroll
                for (int pl = 0; pl < 2; ++pl)
#pragma unroll
                    for (int q = 0; q < 8; ++q) {          // four rows 32 (q/4) + 8 (q%4) + 4 (lane/32) .. of the lane's column
                        const h8& v = pl ? xl[s][q >> 1] : xh[s][q >> 1];
                        const h4 w = (q & 1) ? __builtin_shufflevector(v, v, 4, 5, 6, 7) : __builtin_shufflevector(v, v, 0, 1, 2, 3);
                        *reinterpret_cast<h4*>(&L.slab[wave][pl][col * LD + 32 * (q >> 2) + 8 * (q & 3) + 4 * (lane >> 5)]) = w;
                    }
                asm volatile("" ::: "memory");             // a wave's LDS accesses are in order; its slab is its own
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    h8 fh[2], fl[2];
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        fh[t] = frag_of_slab(L.slab[wave][0], t, ks, lane);
                        fl[t] = frag_of_slab(L.slab[wave][1], t, ks, lane);
                    }
                    acc[0] = mfma3(fh[0], fl[0], fh[0], fl[0], acc[0]);
                    acc[1] = mfma3(fh[1], fl[1], fh[0], fl[0], acc[1]);
                    acc[2] = mfma3(fh[1], fl[1], fh[1], fl[1], acc[2]);
                }
                asm volatile("" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
            }
        __syncthreads();                                   // slabs are read: their LDS becomes the partial sums'
        if (wave < slabs)
#pragma unroll
            for (int t = 0; t < 3; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) L.part[wave][(t * 16 + r) * 64 + lane] = acc[t][r];
        __syncthreads();
        const int nw = slabs < 8 ? slabs : 8;
        const float xi2 = xi * xi;
#pragma unroll
        for (int q = 0; q < 6; ++q) {
            const int tr = wave + 8 * q, t = tr >> 4, r = tr & 15;
            float v = 0.f;
            for (int w = 0; w < nw; ++w) v += L.part[w][tr * 64 + lane];
            v *= xi2;
            const int i = (t > 0 ? 32 : 0) + acc_row(r, lane), j = (t > 1 ? 32 : 0) + col;
            const bool diag = i == j;
            if (diag) L.d[i] = v;
            if (t == 1 || i >= j) {                        // the lower triangle decides both
                const float w = diag ? 0.f : v * S;
                put2(L.r, i, j, w);
                if (!diag) put2(L.r, j, i, w);
            }
        }
        __syncthreads();
        // ---- B = b A + c A^2, one 32 x 32 tile for each of three waves
        if (wave < 3) {
            const int ti = wave > 0 ? 1 : 0, tj = wave > 1 ? 1 : 0;
            f32x16 g = {};
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
                g = mfma3(frag_row(L.r[0], ti, ks, lane), frag_row(L.r[1], ti, ks, lane), frag_row(L.r[0], tj, ks, lane),
                          frag_row(L.r[1], tj, ks, lane), g);
            const int j = 32 * tj + col;
            const float dj = L.d[j];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int i = 32 * ti + acc_row(r, lane);
                const float di = L.d[i], sq2 = g[r] * (INV_S * INV_S);
                if (i == j) {
                    L.ae[i] = p.s.a + p.s.b * di + p.s.c * (di * di + sq2);
                    put2(L.bm, i, i, 0.f);
                } else if (i > j) {
                    const float rij = ((float)L.r[0][i * LD + j] + (float)L.r[1][i * LD + j]) * INV_S;
                    const float v = S * (p.s.b * rij + p.s.c * ((di + dj) * rij + sq2));
                    put2(L.bm, i, j, v);
                    put2(L.bm, j, i, v);
                }
            }
        }
        __syncthreads();
        // ---- X <- (a + diag B) X + B X
        const float xn = k + 1 < p.s.steps ? scale_of(p.s, total, k + 1) : 1.f, rn = 1.f / xn, alpha = xi * INV_S;
        const bool last = k + 1 == p.s.steps;
#pragma unroll
        for (int s = 0; s < NS; ++s)
            if (wave + 8 * s < slabs) {
                f32x16 x[2] = {};
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        x[t] = mfma3(frag_row_acc(L.bm[0], t, ks, lane), frag_row_acc(L.bm[1], t, ks, lane), xh[s][ks], xl[s][ks], x[t]);
                const int j = 32 * (wave + 8 * s) + col;
#pragma unroll
                for (int r = 0; r < 32; ++r) {
                    const int i = 32 * (r >> 4) + acc_row(r & 15, lane);
                    const float old = ((float)xh[s][r >> 3][r & 7] + (float)xl[s][r >> 3][r & 7]) * xi;
                    const float v = fmaf(L.ae[i], old, x[r >> 4][r & 15] * alpha);
                    if (last) {
                        if (i < m && j < n) ap.store<MODE>(mt, ((long)sub * mt.rows + (tall ? j : i)) * mt.cols + (tall ? i : j), v);
                    } else {
                        const float w = v * rn;
                        const _Float16 hi = (_Float16)w;
                        xh[s][r >> 3][r & 7] = hi;
                        xl[s][r >> 3][r & 7] = (_Float16)(w - (float)hi);
                    }
                    if ((r & 7) == 7) __builtin_amdgcn_sched_barrier(0);
                }
            }
        xi = xn;
    }
}

template <int MODE>
__global__ void __launch_bounds__(512) ns_small_kernel(Mats p) {
    __shared__ SmallLds L;
    int sub;
    const Mat& mt = find(p, (int)blockIdx.x, sub);
    const int n = mt.rows > mt.cols ? mt.rows : mt.cols;
    if (n <= 256) small_body<MODE, 1>(p, mt, sub, L);
    else if (n <= 512) small_body<MODE, 2>(p, mt, sub, L);
    else small_body<MODE, 4>(p, mt, sub, L);
}

// ================================================================================================ large matrices
// Buffers of one matrix, padded to the tile in both directions with zeros that every step reproduces (A, B and X of a zero row
// or column are zero), so that no product needs a bounds check:  X [mp][np] and X^T [np][mp] (twice), R and B [mp][mp].  With X
// in both orders each of the three products contracts the contiguous dimension of both operands.
struct Large {
    char* ws;
    long per;                       // bytes per matrix
    long o_x, o_xt[2], o_r, o_b, o_d, o_e, o_xi, o_sq;
    int m, n, mp, np, tall, tile, batch, base;   // base: index of the first matrix of this launch among p.m
};

struct NormArgs { Mats p; Large l; };

// partial sums of squares (64-bit), the momentum update on the way
template <int MODE>
__global__ void __launch_bounds__(256) ns_norm_kernel(NormArgs a) {
    __shared__ double sq[4];
    int sub;
    const Mat& mt = find(a.p, a.l.base + (int)blockIdx.y, sub);
    // threads walk the contiguous dimension of U
    const bool by_col = mt.cs <= mt.rs;
    const int inner = by_col ? mt.cols : mt.rows, outer = by_col ? mt.rows : mt.cols;
    double s = 0;
    for (int o = blockIdx.x; o < outer; o += NORM_PARTS)
        for (int i = threadIdx.x; i < inner; i += 256) {
            const double u = load_u<MODE, true>(a.p.s, mt, sub, by_col ? o : i, by_col ? i : o);
            s = fma(u, u, s);
        }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) sq[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0)
        reinterpret_cast<double*>(a.l.ws + (long)blockIdx.y * a.l.per + a.l.o_sq)[blockIdx.x] = sq[0] + sq[1] + sq[2] + sq[3];
}

// X0 in both orders, a 64 x 64 tile per workgroup
template <int MODE, bool SPLIT>
__global__ void __launch_bounds__(256) ns_prepare_kernel(NormArgs a) {
    __shared__ _Float16 tile[2][64][72];
    int sub;
    const Mat& mt = find(a.p, a.l.base + (int)blockIdx.z, sub);
    char* ws = a.l.ws + (long)blockIdx.z * a.l.per;
    const double* part = reinterpret_cast<const double*>(ws + a.l.o_sq);
    double total = 0;
    for (int i = 0; i < NORM_PARTS; ++i) total += part[i];
    int e;
    const float xi0 = scales(a.p.s, total, e);
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x <= a.p.s.steps)
        reinterpret_cast<float*>(ws + a.l.o_xi)[threadIdx.x] = threadIdx.x == 0 ? xi0 : scale_of(a.p.s, total, threadIdx.x);
    const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
    const bool across = (mt.cs <= mt.rs) != (a.l.tall != 0);             // whether columns of X are contiguous in U
    for (int t = threadIdx.x; t < 4096; t += 256) {
        const int i = across ? t >> 6 : t & 63, j = across ? t & 63 : t >> 6, gi = i0 + i, gj = j0 + j;
        float v = 0.f;
        if (gi < a.l.m && gj < a.l.n) v = scaled(load_u<MODE, false>(a.p.s, mt, sub, a.l.tall ? gj : gi, a.l.tall ? gi : gj), e);
        const _Float16 hi = (_Float16)v;
        tile[0][i][j] = hi;
        tile[1][i][j] = (_Float16)(v - (float)hi);
    }
    __syncthreads();
    const long plane = (long)a.l.mp * a.l.np;
    _Float16* xt = reinterpret_cast<_Float16*>(ws + a.l.o_xt[0]);
    _Float16* x = reinterpret_cast<_Float16*>(ws + a.l.o_x);
#pragma unroll
    for (int pl = 0; pl < 2; ++pl)
        for (int t = threadIdx.x; t < 4096; t += 256) {
            if (SPLIT || pl == 0) x[pl * plane + (long)(i0 + (t >> 6)) * a.l.np + j0 + (t & 63)] = tile[pl][t >> 6][t & 63];
            xt[pl * plane + (long)(j0 + (t >> 6)) * a.l.mp + i0 + (t & 63)] = tile[pl][t & 63][t >> 6];
        }
}

// One product of a step, C[i][j] = sum_k P[i][k] Q[j][k], and what follows it:
//   A_OF_X      P = Q = X, tiles of the lower triangle:   R = A - diag A (both triangles), d = diag A
//   B_OF_A      P = Q = R, tiles of the lower triangle:   B - diag B, e = a + diag B
//   X_NEXT      P = B, Q = X^T:                            X, X^T
//   X_LAST      the same, result or weight update; TALL: P = X^T, Q = B, so that lanes run along U's rows either way
// Four waves, each (TILE / 2)^2 of the TILE^2 outputs; two stages of BK columns of P and Q in LDS, filled by LDS-DMA one stage
// ahead.  Rows of a stage hold 16-byte chunks in an order that depends on the row (chunk c of row r at c ^ f(r)), so that the
// eight lanes that read at once hit all banks.
enum { A_OF_X, B_OF_A, X_NEXT, X_LAST };

struct GemmArgs { Mats p; Large l; int k; };

template <int TILE, bool SPLIT, int KIND>
__global__ void __launch_bounds__(256, 2) ns_gemm_kernel(GemmArgs a) {
    constexpr int BK = SPLIT ? 32 : 64, NP = SPLIT ? 2 : 1, W = TILE / 2, NT = W / 32, CH = BK / 8;
    constexpr int OPBYTES = TILE * BK * 2, STAGE = 2 * NP * OPBYTES;
    constexpr int STG = TILE + 8;                                       // halves per row of the output tile in LDS
    constexpr int LDS_BYTES = 2 * STAGE > TILE * STG * 2 ? 2 * STAGE : TILE * STG * 2;
    __shared__ __attribute__((aligned(16))) char lds[LDS_BYTES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = wave >> 1, wc = wave & 1;
    char* ws = a.l.ws + (long)blockIdx.y * a.l.per;
    const Large& l = a.l;
    const bool swap = KIND == X_LAST && l.tall;
    const int mt = l.mp / TILE;
    int ti, tj;
    if constexpr (KIND == A_OF_X || KIND == B_OF_A) {
        const int t = (int)ksr_xcd_contiguous(blockIdx.x, gridDim.x);
        ti = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
        while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
        while (ti * (ti + 1) / 2 > t) --ti;
        tj = t - ti * (ti + 1) / 2;
    } else {
        const int t = (int)ksr_xcd_contiguous(blockIdx.x, gridDim.x);
        if (swap) { ti = t / mt; tj = t % mt; } else { ti = t % mt; tj = t / mt; }
    }
    const _Float16* R = reinterpret_cast<const _Float16*>(ws + l.o_r);
    const _Float16* xt = reinterpret_cast<const _Float16*>(ws + l.o_xt[a.k & 1]);
    const _Float16 *P, *Q;
    long pp, qp;                                        // distance of the lo plane
    int K;
    if constexpr (KIND == A_OF_X) { P = Q = reinterpret_cast<const _Float16*>(ws + l.o_x); K = l.np; pp = qp = (long)l.mp * l.np; }
    else if constexpr (KIND == B_OF_A) { P = Q = R; K = l.mp; pp = qp = (long)l.mp * l.mp; }
    else {
        const _Float16* B = reinterpret_cast<const _Float16*>(ws + l.o_b);
        P = swap ? xt : B; Q = swap ? B : xt; K = l.mp;
        pp = swap ? (long)l.np * l.mp : (long)l.mp * l.mp;
        qp = swap ? (long)l.mp * l.mp : (long)l.np * l.mp;
    }
    P += (long)ti * TILE * K;
    Q += (long)tj * TILE * K;
    // LDS-DMA: one instruction of a wave brings 64 chunks of 16 bytes; lane -> (row, slot), the chunk that belongs there
    constexpr int ROWS = 64 / CH, NI = TILE / ROWS / 4;                 // rows per instruction, instructions per wave and operand plane
    const int drow = lane / CH, dslot = lane % CH;
    auto f = [](int row) { return CH == 8 ? (row & 7) : ((row >> 1) & 3); };
    auto fill = [&](int st, int kt) {
#pragma unroll
        for (int op = 0; op < 2; ++op)
#pragma unroll
            for (int pl = 0; pl < NP; ++pl)
#pragma unroll
                for (int q = 0; q < NI; ++q) {
                    const int row = (wave * NI + q) * ROWS + drow;
                    const _Float16* src = (op ? Q + pl * qp : P + pl * pp) + (long)row * K + kt * BK + 8 * (dslot ^ f(row));
                    ksr_dma16<false>(src, lds + st * STAGE + (op * NP + pl) * OPBYTES + (wave * NI + q) * 1024);
                }
    };
    auto frag = [&](int st, int op, int pl, int row, int ks) {
        const int chunk = (2 * ks + (lane >> 5)) ^ f(row);
        return *reinterpret_cast<const h8*>(lds + st * STAGE + (op * NP + pl) * OPBYTES + row * (BK * 2) + 16 * chunk);
    };
    // hi lo + lo hi have accumulators of their own: added to the large sum one by one they would round it three times a step
    f32x16 acc[NT][NT] = {}, low[SPLIT ? NT : 1][SPLIT ? NT : 1] = {};
    const int nk = K / BK;
    fill(0, 0);
    for (int kt = 0; kt < nk; ++kt) {
        ksr_dma_barrier();                              // this stage has landed, the other one has been read by every wave
        if (kt + 1 < nk) fill((kt + 1) & 1, kt + 1);
        const int st = kt & 1;
#pragma unroll
        for (int ks = 0; ks < BK / 16; ++ks) {
            h8 ph[NT], qh[NT], pl[NT], ql[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                ph[t] = frag(st, 0, 0, wr * W + 32 * t + (lane & 31), ks);
                qh[t] = frag(st, 1, 0, wc * W + 32 * t + (lane & 31), ks);
                if constexpr (SPLIT) {
                    pl[t] = frag(st, 0, 1, wr * W + 32 * t + (lane & 31), ks);
                    ql[t] = frag(st, 1, 1, wc * W + 32 * t + (lane & 31), ks);
                }
            }
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
                for (int y = 0; y < NT; ++y) {
                    acc[x][y] = mfma(ph[x], qh[y], acc[x][y]);
                    if constexpr (SPLIT) {
                        low[x][y] = mfma(ph[x], ql[y], low[x][y]);
                        low[x][y] = mfma(pl[x], qh[y], low[x][y]);
                    }
                }
        }
    }
    if constexpr (SPLIT)
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int y = 0; y < NT; ++y) acc[x][y] += low[x][y];
    ksr_lds_barrier();                                  // LDS is free for the output tile
    // ---- values
    const float* xis = reinterpret_cast<const float*>(ws + l.o_xi);
    float* dv = reinterpret_cast<float*>(ws + l.o_d);
    float* ev = reinterpret_cast<float*>(ws + l.o_e);
    const Step& sp = a.p.s;
    const float xi = xis[a.k], rn = KIND == X_NEXT ? 1.f / xis[a.k + 1] : 1.f;
    int sub = 0;
    const Mat& mat = find(a.p, l.base + (int)blockIdx.y, sub);
    const Apply ap(sp, mat);
    const int mode = sp.muon ? MUON : sp.bf16 ? BF16 : F32;
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int y = 0; y < NT; ++y)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row0 = ti * TILE + wr * W + 32 * x + 8 * q + 4 * (lane >> 5), c = tj * TILE + wc * W + 32 * y + (lane & 31);
                float v[4];
#pragma unroll
                for (int z = 0; z < 4; ++z) v[z] = acc[x][y][4 * q + z];
                if constexpr (KIND == A_OF_X) {
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        v[z] *= xi * xi;
                        if (row0 + z == c) { dv[c] = v[z]; v[z] = 0.f; }
                        v[z] *= S;
                    }
                } else if constexpr (KIND == B_OF_A) {
                    const h4 rh = *reinterpret_cast<const h4*>(R + (long)c * l.mp + row0);       // R is symmetric
                    h4 rl = {};
                    if constexpr (SPLIT) rl = *reinterpret_cast<const h4*>(R + pp + (long)c * l.mp + row0);
                    const float dc = dv[c];
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const float di = dv[row0 + z], r = ((float)rh[z] + (float)rl[z]) * INV_S, sq = v[z] * (INV_S * INV_S);
                        if (row0 + z == c) {
                            ev[c] = sp.a + sp.b * di + sp.c * (di * di + sq);
                            v[z] = 0.f;
                        } else v[z] = S * (sp.b * r + sp.c * ((di + dc) * r + sq));
                    }
                } else {
                    const float alpha = xi * INV_S;
                    const long plane = (long)l.mp * l.np;
                    if (!swap) {                        // rows are i, columns j
                        const h4 xh = *reinterpret_cast<const h4*>(xt + (long)c * l.mp + row0), xl = *reinterpret_cast<const h4*>(xt + plane + (long)c * l.mp + row0);
#pragma unroll
                        for (int z = 0; z < 4; ++z) v[z] = fmaf(ev[row0 + z], ((float)xh[z] + (float)xl[z]) * xi, v[z] * alpha);
                    } else {
                        const float ec = ev[c];
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            const long o = (long)(row0 + z) * l.mp + c;
                            v[z] = fmaf(ec, ((float)xt[o] + (float)xt[plane + o]) * xi, v[z] * alpha);
                        }
                    }
                    if constexpr (KIND == X_LAST) {
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            const int r = row0 + z;     // rows and columns of the result are those of U either way
                            if (r < mat.rows && c < mat.cols) {
                                const long o = ((long)sub * mat.rows + r) * mat.cols + c;
                                if (mode == F32) ap.store<F32>(mat, o, v[z]);
                                else if (mode == BF16) ap.store<BF16>(mat, o, v[z]);
                                else ap.store<MUON>(mat, o, v[z]);
                            }
                        }
                    } else {
#pragma unroll
                        for (int z = 0; z < 4; ++z) v[z] *= rn;
                    }
                }
#pragma unroll
                for (int z = 0; z < 4; ++z) acc[x][y][4 * q + z] = v[z];
            }
    if constexpr (KIND == X_LAST) return;
    // ---- the tile and its transpose, hi and lo, through LDS: 16-byte stores of whole rows
    _Float16* stage = reinterpret_cast<_Float16*>(lds);
    _Float16 *out, *outt;
    long ld, ldt, plane;
    constexpr int planes = (KIND == X_NEXT || SPLIT) ? 2 : 1;
    if constexpr (KIND == X_NEXT) {
        out = reinterpret_cast<_Float16*>(ws + l.o_x); outt = reinterpret_cast<_Float16*>(ws + l.o_xt[(a.k + 1) & 1]);
        ld = l.np; ldt = l.mp; plane = (long)l.mp * l.np;
    } else {
        out = outt = reinterpret_cast<_Float16*>(ws + (KIND == A_OF_X ? l.o_r : l.o_b));
        ld = ldt = l.mp; plane = (long)l.mp * l.mp;
    }
#pragma unroll
    for (int pl = 0; pl < planes; ++pl)
#pragma unroll
        for (int tr = 0; tr < 2; ++tr) {
            if (tr == 1 && KIND != X_NEXT && ti == tj) continue;
            if (tr == 0 && pl == 1 && !SPLIT) continue;              // X's lo is only read through X^T (the linear term)
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
                for (int y = 0; y < NT; ++y)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int r = wr * W + 32 * x + 8 * q + 4 * (lane >> 5), c = wc * W + 32 * y + (lane & 31);
                        h4 w;
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            const float v = acc[x][y][4 * q + z];
                            const _Float16 hi = (_Float16)v;
                            w[z] = pl ? (_Float16)(v - (float)hi) : hi;
                        }
                        if (tr) *reinterpret_cast<h4*>(stage + c * STG + r) = w;
                        else {
#pragma unroll
                            for (int z = 0; z < 4; ++z) stage[(r + z) * STG + c] = w[z];
                        }
                    }
            __syncthreads();
            _Float16* o = (tr ? outt : out) + pl * plane;
            const long lo = tr ? ldt : ld;
            const int r0 = (tr ? tj : ti) * TILE, c0 = (tr ? ti : tj) * TILE;
            for (int t = threadIdx.x; t < TILE * (TILE / 8); t += 256) {
                const int r = t / (TILE / 8), c = t % (TILE / 8) * 8;
                *reinterpret_cast<uint4*>(o + (long)(r0 + r) * lo + c0 + c) = *reinterpret_cast<const uint4*>(stage + r * STG + c);
            }
            __syncthreads();
        }
}

// ------------------------------------------------------------------------------------------------ host
bool is_small(int rows, int cols) { return rows < cols ? rows <= 64 && cols <= 1024 : cols <= 64 && rows <= 1024; }

int tile_of(int m, int n) { return (long)((m + 127) / 128) * ((n + 127) / 128) >= 128 ? 128 : 64; }

long align256(long v) { return (v + 255) / 256 * 256; }

void plan(Large& l, int rows, int cols, bool split) {
    l = Large{};
    l.tall = rows > cols;
    l.m = l.tall ? cols : rows;
    l.n = l.tall ? rows : cols;
    const int tile = l.tile = tile_of(l.m, l.n);
    l.mp = (l.m + tile - 1) / tile * tile;
    l.np = (l.n + tile - 1) / tile * tile;
    const long xp = 2l * l.mp * l.np, ap = 2l * l.mp * l.mp;
    long o = 0;
    l.o_x = o; o += align256(xp * (split ? 2 : 1));
    l.o_xt[0] = o; o += align256(2 * xp);
    l.o_xt[1] = o; o += align256(2 * xp);
    l.o_r = o; o += align256(ap * (split ? 2 : 1));
    l.o_b = o; o += align256(ap * (split ? 2 : 1));
    l.o_d = o; o += align256(4l * l.mp);
    l.o_e = o; o += align256(4l * l.mp);
    l.o_xi = o; o += align256(4l * (MAX_STEPS + 1));
    l.o_sq = o; o += align256(8l * NORM_PARTS);
    l.per = o;
}

constexpr long WS_CAP = 1l << 30;           // matrices of one shape that run together: as many as fit 1 GiB, at least one
constexpr int BATCH_CAP = 16384;

long together(const Large& l, long count) {
    long n = WS_CAP / l.per;
    if (n < 1) n = 1;
    if (n > BATCH_CAP) n = BATCH_CAP;
    return n < count ? n : count;
}

// Largest singular value that each step can reach from [0, 1], and that A and B stay inside f16's range
bool bounded(float a, float b, float c, int steps, float& gain) {
    double top = 1.0, g = fabs((double)a);
    for (int k = 0; k < steps; ++k) {
        double next = 0;
        for (int i = 0; i <= 512; ++i) {
            const double s = top * 1.02 * i / 512, s2 = s * s, f = a + b * s2 + c * s2 * s2;
            if (fabs(f) > g) g = fabs(f);
            if (fabs(f) * s > next) next = fabs(f) * s;
            if (!(s2 <= 30) || !(fabs(b * s2 + c * s2 * s2) <= 30) || !(fabs(f) * s <= 30)) return false;
        }
        top = next;
    }
    gain = (float)(g > 1 ? g : 1);
    return true;
}

template <int MODE, bool SPLIT> void start_large(const NormArgs& na, hipStream_t st) {
    const Large& l = na.l;
    hipLaunchKernelGGL((ns_norm_kernel<MODE>), dim3(NORM_PARTS, (unsigned)l.batch), dim3(256), 0, st, na);
    hipLaunchKernelGGL((ns_prepare_kernel<MODE, SPLIT>), dim3((unsigned)(l.np / 64), (unsigned)(l.mp / 64), (unsigned)l.batch), dim3(256), 0, st, na);
}

template <int TILE, bool SPLIT> int run_large(const Mats& p, Large l, hipStream_t st) {
    NormArgs na{p, l};
    const int mode = mode_of(p.s);
    if (mode == F32) start_large<F32, SPLIT>(na, st);
    else if (mode == BF16) start_large<BF16, SPLIT>(na, st);
    else start_large<MUON, SPLIT>(na, st);
    KSR_LAUNCH_CHECK("muon_batch");
    const int mt = l.mp / TILE, nt = l.np / TILE;
    const dim3 tri((unsigned)(mt * (mt + 1) / 2), (unsigned)l.batch), full((unsigned)(mt * nt), (unsigned)l.batch);
    for (int k = 0; k < p.s.steps; ++k) {
        GemmArgs g{p, l, k};
        hipLaunchKernelGGL((ns_gemm_kernel<TILE, SPLIT, A_OF_X>), tri, dim3(256), 0, st, g);
        hipLaunchKernelGGL((ns_gemm_kernel<TILE, SPLIT, B_OF_A>), tri, dim3(256), 0, st, g);
        if (k + 1 < p.s.steps) hipLaunchKernelGGL((ns_gemm_kernel<TILE, SPLIT, X_NEXT>), full, dim3(256), 0, st, g);
        else hipLaunchKernelGGL((ns_gemm_kernel<TILE, SPLIT, X_LAST>), full, dim3(256), 0, st, g);
        KSR_LAUNCH_CHECK("muon_batch");
    }
    return KSR_OK;
}

}  // namespace

namespace {

int check_shapes(const KsrMatrix* mats, int count) {
    KSR_CHECK_ARG(count >= 0 && (mats || count == 0), "muon_batch: null pointer");
    for (int i = 0; i < count; ++i) {
        const KsrMatrix& q = mats[i];
        KSR_CHECK_ARG(q.rows >= 0 && q.cols >= 0 && q.batch >= 0, "muon_batch: matrix %d is [%d, %d, %d]", i, q.batch, q.rows, q.cols);
        KSR_UNSUPPORTED(q.rows > (1 << 20) || q.cols > (1 << 20) || (q.rows > (1 << 15) && q.cols > (1 << 15)),
                        "muon_batch: matrix %d is [%d, %d]: sides up to 2^20, the shorter one up to 2^15", i, q.rows, q.cols);
        KSR_UNSUPPORTED(q.batch > (1 << 24), "muon_batch: %d matrices in one batch (up to 2^24)", q.batch);
    }
    return KSR_OK;
}

bool empty(const KsrMatrix& q) { return !q.rows || !q.cols || !q.batch; }

int check_mats(const KsrMatrix* mats, int count, int bf16, bool muon) {
    if (int rc = check_shapes(mats, count)) return rc;
    for (int i = 0; i < count; ++i) {
        const KsrMatrix& q = mats[i];
        if (empty(q)) continue;
        KSR_CHECK_ARG(q.src && q.dst && (!muon || q.momentum), "muon_batch: null pointer in matrix %d", i);
        KSR_CHECK_ARG(q.row_stride >= 0 && q.col_stride >= 0 && q.batch_stride >= 0, "muon_batch: negative stride in matrix %d", i);
        const uintptr_t es = bf16 ? 2 : 4;
        KSR_CHECK_ARG((uintptr_t)q.src % es == 0 && (uintptr_t)q.dst % es == 0 && (!muon || (uintptr_t)q.momentum % 4 == 0),
                      "muon_batch: misaligned pointer in matrix %d", i);
    }
    return KSR_OK;
}

}  // namespace

extern "C" int64_t ksr_muon_ws_bytes(const KsrMatrix* mats, int count, int split) {
    if (check_shapes(mats, count) != KSR_OK) return -1;
    int64_t most = 0;
    for (int i = 0; i < count; ++i) {
        if (empty(mats[i]) || is_small(mats[i].rows, mats[i].cols)) continue;
        int64_t same = 0;                    // matrices of this shape in the list run together
        for (int j = 0; j < count; ++j)
            if (!empty(mats[j]) && mats[j].rows == mats[i].rows && mats[j].cols == mats[i].cols) same += mats[j].batch;
        Large l;
        plan(l, mats[i].rows, mats[i].cols, split != 0);
        const int64_t need = together(l, same) * l.per;
        if (need > most) most = need;
    }
    return most;
}

extern "C" int ksr_muon_batch(const KsrMatrix* mats, int count, int bf16, int split, int muon, int steps, float a, float b, float c,
                              float eps, float momentum, int nesterov, float grad_scale, float lr, const float* lr_dev,
                              float weight_decay, float scale, void* ws, int64_t ws_bytes, hipStream_t stream) {
    if (int rc = check_mats(mats, count, bf16, muon != 0)) return rc;
    KSR_CHECK_ARG(!(muon && bf16), "muon_batch: the update takes fp32 gradients, momenta and weights");
    KSR_CHECK_ARG(steps >= 1 && steps <= MAX_STEPS, "muon_batch: %d steps (1 to %d)", steps, MAX_STEPS);
    KSR_CHECK_ARG(eps >= 0.f && eps < INFINITY, "muon_batch: eps = %g", (double)eps);
    Mats p{};
    p.s = Step{steps, bf16, muon, nesterov, a, b, c, eps, 1.f, momentum, grad_scale, lr, weight_decay, scale, lr_dev};
    KSR_UNSUPPORTED(!bounded(a, b, c, steps, p.s.gain), "muon_batch: with coefficients (%g, %g, %g) %d steps leave the range of the products (30)",
                    (double)a, (double)b, (double)c, steps);
    KSR_CHECK_ARG(ws_bytes >= ksr_muon_ws_bytes(mats, count, split), "muon_batch: the workspace has %lld bytes, %lld are needed",
                  (long long)ws_bytes, (long long)ksr_muon_ws_bytes(mats, count, split));
    KSR_CHECK_ARG((ws || ws_bytes == 0) && reinterpret_cast<uintptr_t>(ws) % 16 == 0, "muon_batch: null or misaligned workspace");
    auto add = [&](const KsrMatrix& q, int first) {
        Mat& m = p.m[p.count++];
        m = Mat{q.src, q.dst, q.momentum, (long)q.row_stride, (long)q.col_stride, (long)q.batch_stride, q.rows, q.cols, q.batch, first};
    };
    auto small = [&](const KsrMatrix& q) { return is_small(q.rows, q.cols); };
    // every small matrix of the list in one launch (of up to MAX_MATS entries)
    for (int i = 0; i < count;) {
        p.count = 0;
        int64_t total = 0;
        for (; i < count && p.count < MAX_MATS; ++i) {
            if (empty(mats[i]) || !small(mats[i])) continue;
            add(mats[i], (int)total);
            total += mats[i].batch;
        }
        if (!p.count) continue;
        const int mode = mode_of(p.s);
        if (mode == F32) hipLaunchKernelGGL(ns_small_kernel<F32>, dim3((unsigned)total), dim3(512), 0, stream, p);
        else if (mode == BF16) hipLaunchKernelGGL(ns_small_kernel<BF16>, dim3((unsigned)total), dim3(512), 0, stream, p);
        else hipLaunchKernelGGL(ns_small_kernel<MUON>, dim3((unsigned)total), dim3(512), 0, stream, p);
        KSR_LAUNCH_CHECK("muon_batch");
    }
    // large ones: all of one shape together
    for (int i = 0; i < count; ++i) {
        if (empty(mats[i]) || small(mats[i])) continue;
        bool seen = false;
        for (int j = 0; j < i; ++j) seen = seen || (!empty(mats[j]) && mats[j].rows == mats[i].rows && mats[j].cols == mats[i].cols);
        if (seen) continue;
        Large l;
        plan(l, mats[i].rows, mats[i].cols, split != 0);
        l.ws = reinterpret_cast<char*>(ws);
        for (int j = i; j < count;) {
            p.count = 0;
            int64_t total = 0;
            for (; j < count && p.count < MAX_MATS; ++j) {
                if (empty(mats[j]) || mats[j].rows != mats[i].rows || mats[j].cols != mats[i].cols) continue;
                add(mats[j], (int)total);
                total += mats[j].batch;
            }
            if (!p.count) break;
            const long at_once = together(l, total);
            for (int64_t base = 0; base < total; base += at_once) {
                l.base = (int)base;
                l.batch = (int)(total - base < at_once ? total - base : at_once);
                int rc;
                if (split) rc = l.tile == 128 ? run_large<128, true>(p, l, stream) : run_large<64, true>(p, l, stream);
                else rc = l.tile == 128 ? run_large<128, false>(p, l, stream) : run_large<64, false>(p, l, stream);
                if (rc) return rc;
            }
        }
    }
    return KSR_OK;
}
