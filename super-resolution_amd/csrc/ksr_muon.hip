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
constexpr int SMALL_WGS = 1 << 22;                    // workgroups (of 512 threads) of a launch: it holds fewer than 2^32 threads

struct Mat {
    const void* src;          // U, or the gradient
    void* dst;                // the orthogonalised matrix (dense, type of src), or the weight to update (fp32, dense)
    float* mom;               // Muon: momentum (fp32, dense)
    long rs, cs, bs;          // strides of src in elements: row, column, matrix
    int rows, cols, batch, first;
    int sub0;                 // small matrices: index in the batch of the launch's first one
};

struct Step {
    int steps, bf16, muon, nesterov;
    float a, b, c, eps, log2_gain;        // gain: most by which a step multiplies a singular value
    float momentum, grad_scale, lr, wd, scale;
    const float* lr_dev;                  // replaces lr
};

struct Mats { Mat m[MAX_MATS]; int count; Step s; };

__device__ __forceinline__ const Mat& find(const Mats& p, int i, int& sub) {
    int k = 0;
    while (k + 1 < p.count && i >= p.m[k + 1].first) ++k;
    sub = p.m[k].sub0 + i - p.m[k].first;
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
    // the weights of several results are read before the first is written: a load behind a store would wait for it
    template <int MODE> __device__ __forceinline__ float old(const Mat& m, long o) const {
        return MODE == MUON ? reinterpret_cast<const float*>(m.dst)[o] : 0.f;
    }
    __device__ __forceinline__ float updated(float v, float w) const { return fmaf(-rate, v, w * keep); }
    template <int MODE> __device__ __forceinline__ void store(const Mat& m, long o, float v, float w) const {
        if constexpr (MODE == MUON) reinterpret_cast<float*>(m.dst)[o] = updated(v, w);
        else if constexpr (MODE == BF16) reinterpret_cast<__bf16*>(m.dst)[o] = (__bf16)v;
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
// -log2 of the norm of X0, and from it xi[k], k > 0
__device__ __forceinline__ double log_norm(const Step& s, double sumsq) {
    const double norm = sqrt(sumsq), nu = norm / (norm + (double)s.eps);
    return nu > 0 ? -log2(nu) : 0.0;
}
__device__ __forceinline__ float scale_at(const Step& s, double lg, int k) {
    const float f = (float)lg - (float)k * s.log2_gain;
    return ldexpf(INV_S, -(int)(f > 0.f ? (f < 100.f ? floorf(f) : 100.f) : 0.f));      // NaN: 1
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
// r%4), which is the B operand's layout for the next product when both operands take k in that order.  Always SPLIT: the time
// is latency (one wave or two per SIMD, three or four barriers a step), not matrix work.  fp32, five steps: 26 us for 64 x 64, 97 us
// for 1 or 16 of 64 x 1024; as large matrices 245 to 265 us, in 17 launches.  Four slabs (513 columns and more) do not fit 256
// registers: 34 (Muon 110, bf16 26) are spilled.
// The 64 x 64 matrices A and A^2 are four 32 x 32 tiles of four waves; both triangles are computed, so that a wave writes its
// tile's transpose in 8-byte pieces and nothing else (symmetric up to the rounding of hi lo + lo hi).  For X X^T the slabs pass
// through LDS, eight at a time, the upper four waves taking slabs 4 to 7 of them.
constexpr int LD = 72;                                  // halves per row of R, B and a slab: 144 bytes

struct SmallLds {
    _Float16 slab[8][2][32 * LD];                       // 72 KB: [column][row], hi and lo
    float red[4][16][64];                               // 16 KB: the upper waves' sums
    _Float16 r[2][64 * LD], bm[2][64 * LD];             // 36 KB
    float d[64], ae[64];                                // diagonal of A; a + diagonal of B
    double sq[8];
};

__device__ __forceinline__ int acc_row(int r, int lane) { return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3); }

__device__ __forceinline__ f32x16 mfma(const h8& a, const h8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
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
// four values as hi and lo to row j, columns i .. i + 3
__device__ __forceinline__ void put4(_Float16 (&mat)[2][64 * LD], int j, int i, const float (&v)[4]) {
    h4 hi, lo;
#pragma unroll
    for (int z = 0; z < 4; ++z) {
        hi[z] = (_Float16)v[z];
        lo[z] = (_Float16)(v[z] - (float)hi[z]);
    }
    *reinterpret_cast<h4*>(&mat[0][j * LD + i]) = hi;
    *reinterpret_cast<h4*>(&mat[1][j * LD + i]) = lo;
}

// four neighbours of a dense row, fp32 or bf16
template <int MODE> __device__ __forceinline__ void load4(const void* p, long o, float* v) {
    if constexpr (MODE == BF16) {
        const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const __bf16*>(p) + o);
        v[0] = __uint_as_float(w.x << 16); v[1] = __uint_as_float(w.x & 0xffff0000u);
        v[2] = __uint_as_float(w.y << 16); v[3] = __uint_as_float(w.y & 0xffff0000u);
    } else {
        const float4 w = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + o);
        v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    }
}
template <int MODE> __device__ __forceinline__ void store4(void* p, long o, const float* v) {
    if constexpr (MODE == BF16) {
        __bf16 w[4];
#pragma unroll
        for (int z = 0; z < 4; ++z) w[z] = (__bf16)v[z];
        __builtin_memcpy(__builtin_assume_aligned(reinterpret_cast<__bf16*>(p) + o, 8), w, 8);
    } else *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + o) = make_float4(v[0], v[1], v[2], v[3]);
}

// Four rows of X that a lane holds are neighbours in U where U is transposed and dense: in single values each of a wave's loads
// would touch 64 lines (16 matrices of up to 192 x 64, Muon: 58 us so, 46 us in fours)
template <int MODE> __device__ __forceinline__ bool in_fours(const Mat& m) {
    constexpr uintptr_t bytes = MODE == BF16 ? 8 : 16;
    return m.rows > m.cols && m.cs == 1 && m.cols % 4 == 0 && m.rs % 4 == 0 && m.bs % 4 == 0 && (uintptr_t)m.src % bytes == 0 &&
           (uintptr_t)m.dst % bytes == 0 && (MODE != MUON || (uintptr_t)m.mom % 16 == 0);
}

template <int MODE, int NS>
__device__ __forceinline__ void small_body(const Step& st, const Mat& mt, int sub, SmallLds& L) {
    const int lane0 = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool tall = mt.rows > mt.cols;
    const int m = tall ? mt.cols : mt.rows, n = tall ? mt.rows : mt.cols, slabs = (n + 31) >> 5;
    const Apply ap(st, mt);
    const bool fours = in_fours<MODE>(mt);
    // slab s of this wave: columns 32 (wave + 8 s) ..; all loads are in flight together
    h8 xh[NS][4], xl[NS][4];
    float xi;
    double lg;
    {
        const int lane = lane0, col = lane & 31;
        float u[NS][32];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int j = 32 * (wave + 8 * s) + col, jc = j < n ? j : n - 1;
            float mo[MODE == MUON ? 32 : 1];
            if (fours) {
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const int i = 32 * (q >> 2) + acc_row(4 * (q & 3), lane), ic = i < m ? i : 0;
                    load4<MODE>(mt.src, (long)sub * mt.bs + (long)jc * mt.rs + ic, &u[s][4 * q]);
                    if constexpr (MODE == MUON) load4<MUON>(mt.mom, ((long)sub * mt.rows + jc) * mt.cols + ic, &mo[4 * q]);
                }
            } else
#pragma unroll
            for (int r = 0; r < 32; ++r) {
                const int i = 32 * (r >> 4) + acc_row(r & 15, lane), ic = i < m ? i : m - 1;
                const int row = tall ? jc : ic, c = tall ? ic : jc;
                const long o = (long)sub * mt.bs + (long)row * mt.rs + (long)c * mt.cs;
                if constexpr (MODE == BF16) u[s][r] = (float)reinterpret_cast<const __bf16*>(mt.src)[o];
                else u[s][r] = reinterpret_cast<const float*>(mt.src)[o];
                if constexpr (MODE == MUON) mo[r] = mt.mom[((long)sub * mt.rows + row) * mt.cols + c];
            }
            if constexpr (MODE == MUON) {               // every element has one lane; what a lane beyond the matrix read is dropped below
#pragma unroll
                for (int r = 0; r < 32; ++r) {
                    const float gs = u[s][r] * st.grad_scale;
                    mo[r] = fmaf(st.momentum, mo[r], gs);
                    u[s][r] = st.nesterov ? fmaf(st.momentum, mo[r], gs) : mo[r];
                }
                if (fours) {
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const int i = 32 * (q >> 2) + acc_row(4 * (q & 3), lane);
                        if (i < m && j < n) store4<MUON>(mt.mom, ((long)sub * mt.rows + j) * mt.cols + i, &mo[4 * q]);
                    }
                } else
#pragma unroll
                for (int r = 0; r < 32; ++r) {
                    const int i = 32 * (r >> 4) + acc_row(r & 15, lane);
                    if (i < m && j < n) mt.mom[((long)sub * mt.rows + (tall ? j : i)) * mt.cols + (tall ? i : j)] = mo[r];
                }
                if (NS > 1) __builtin_amdgcn_sched_barrier(0);
            }
        }
        double sq = 0;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int j = 32 * (wave + 8 * s) + col;
#pragma unroll
            for (int r = 0; r < 32; ++r) {
                const int i = 32 * (r >> 4) + acc_row(r & 15, lane);
                if (!(i < m && j < n)) u[s][r] = 0.f;
                sq = fma((double)u[s][r], (double)u[s][r], sq);
            }
        }
        sq = wave_sum(sq);
        if (lane == 0) L.sq[wave] = sq;
        __syncthreads();
        double total = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) total += L.sq[w];
        int e;
        xi = scales(st, total, e);
        lg = log_norm(st, total);
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int r = 0; r < 32; ++r) {
                const float v = scaled(u[s][r], e);
                const _Float16 hi = (_Float16)v;
                xh[s][r >> 3][r & 7] = hi;
                xl[s][r >> 3][r & 7] = (_Float16)(v - (float)hi);
            }
    }
    for (int k = 0; k < st.steps; ++k) {
        // an index the compiler cannot follow: it would otherwise keep every address and bound of the last step's stores (more
        // than 256 registers) through all steps
        int lane = lane0;
        asm volatile("" : "+v"(lane));
        const int col = lane & 31, half = lane >> 5, ti = (wave >> 1) & 1, tj = wave & 1;
        // ---- A = X X^T
        f32x16 acc = {}, low = {};
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            if (s) __syncthreads();                        // the slabs of the round before are read
#pragma unroll
            for (int pl = 0; pl < 2; ++pl)
#pragma unroll
                for (int q = 0; q < 8; ++q) {              // four rows 32 (q/4) + 8 (q%4) + 4 (lane/32) .. of the lane's column
                    const h8& v = pl ? xl[s][q >> 1] : xh[s][q >> 1];
                    const h4 w = (q & 1) ? __builtin_shufflevector(v, v, 4, 5, 6, 7) : __builtin_shufflevector(v, v, 0, 1, 2, 3);
                    *reinterpret_cast<h4*>(&L.slab[wave][pl][col * LD + 32 * (q >> 2) + 8 * (q & 3) + 4 * half]) = w;
                }
            __syncthreads();
            const int first = 4 * (wave >> 2), left = slabs - 8 * s;
            for (int w = first; w < first + 4 && w < left; ++w)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    const h8 ph = frag_of_slab(L.slab[w][0], ti, ks, lane), pl = frag_of_slab(L.slab[w][1], ti, ks, lane);
                    const h8 qh = frag_of_slab(L.slab[w][0], tj, ks, lane), ql = frag_of_slab(L.slab[w][1], tj, ks, lane);
                    acc = mfma(ph, qh, acc);
                    low = mfma(ph, ql, low);
                    low = mfma(pl, qh, low);
                }
        }
        acc += low;
        if (slabs > 4) {                                   // the upper waves' half
            if (wave >= 4)
#pragma unroll
                for (int r = 0; r < 16; ++r) L.red[wave - 4][r][lane] = acc[r];
            __syncthreads();
        }
        if (wave < 4) {
            if (slabs > 4)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[r] += L.red[wave][r][lane];
            const float xi2 = xi * xi;
            const int j = 32 * tj + col;
            float dj = 0.f;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int i = 32 * ti + 8 * g + 4 * half;
                float v[4];
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    v[z] = acc[4 * g + z] * xi2;
                    dj = i + z == j ? v[z] : dj;
                    v[z] = i + z == j ? 0.f : v[z] * S;
                }
                put4(L.r, j, i, v);
            }
            if (ti == tj && ((col >> 2) & 1) == half) L.d[j] = dj;       // the lane that holds (j, j)
        }
        __syncthreads();
        // ---- B = b A + c A^2; what multiplies X itself, a + diag B, already in the scales of the old and the new X
        const bool last = k + 1 == st.steps;
        const float xn = last ? 1.f : scale_at(st, lg, k + 1), rn = 1.f / xn;
        if (wave < 4) {
            f32x16 g0 = {}, g1 = {};
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                const h8 ph = frag_row(L.r[0], ti, ks, lane), pl = frag_row(L.r[1], ti, ks, lane);
                const h8 qh = frag_row(L.r[0], tj, ks, lane), ql = frag_row(L.r[1], tj, ks, lane);
                g0 = mfma(ph, qh, g0);
                g1 = mfma(ph, ql, g1);
                g1 = mfma(pl, qh, g1);
            }
            g0 += g1;
            const int j = 32 * tj + col;
            const float dj = L.d[j];
            float ej = 0.f;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int i = 32 * ti + 8 * g + 4 * half;
                const h4 rh = *reinterpret_cast<const h4*>(&L.r[0][j * LD + i]), rl = *reinterpret_cast<const h4*>(&L.r[1][j * LD + i]);
                const float4 d4 = *reinterpret_cast<const float4*>(&L.d[i]);
                const float di[4] = {d4.x, d4.y, d4.z, d4.w};
                float v[4];
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    const float rij = ((float)rh[z] + (float)rl[z]) * INV_S, sq2 = g0[4 * g + z] * (INV_S * INV_S);
                    ej = i + z == j ? sq2 : ej;
                    v[z] = i + z == j ? 0.f : S * (st.b * rij + st.c * ((di[z] + dj) * rij + sq2));
                }
                put4(L.bm, j, i, v);
            }
            if (ti == tj && ((col >> 2) & 1) == half) L.ae[j] = (st.a + st.b * dj + st.c * (dj * dj + ej)) * (xi * rn);
        }
        __syncthreads();
        // ---- X <- (a + diag B) X + B X.  The products with a lo part go into the accumulators before those of the hi parts: the
        // large sum is rounded four times, not twelve.  fmaf on f16 values is one mixed-precision instruction.
        const float alpha = xi * rn * INV_S;
#pragma unroll
        for (int s = 0; s < NS; ++s)
            if (wave + 8 * s < slabs) {
                f32x16 x[2] = {};
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        x[t] = mfma(frag_row_acc(L.bm[0], t, ks, lane), xl[s][ks], x[t]);
                        x[t] = mfma(frag_row_acc(L.bm[1], t, ks, lane), xh[s][ks], x[t]);
                    }
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                    for (int t = 0; t < 2; ++t) x[t] = mfma(frag_row_acc(L.bm[0], t, ks, lane), xh[s][ks], x[t]);
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    const float4 e4 = *reinterpret_cast<const float4*>(&L.ae[32 * (g >> 2) + 8 * (g & 3) + 4 * half]);
                    const float ae[4] = {e4.x, e4.y, e4.z, e4.w};
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const int r = 4 * g + z;
                        x[g >> 2][r & 15] = fmaf((float)xh[s][r >> 3][r & 7], ae[z], fmaf((float)xl[s][r >> 3][r & 7], ae[z], x[g >> 2][r & 15] * alpha));
                    }
                }
                if (last) {
                    const int j = 32 * (wave + 8 * s) + col;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        float w[16];
                        if (fours) {
                            const long row = ((long)sub * mt.rows + (j < n ? j : n - 1)) * mt.cols;
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const int i = 32 * t + acc_row(4 * q, lane);
                                if constexpr (MODE == MUON) load4<MUON>(mt.dst, row + (i < m ? i : 0), &w[4 * q]);
                            }
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const int i = 32 * t + acc_row(4 * q, lane);
                                float v[4];
#pragma unroll
                                for (int z = 0; z < 4; ++z) v[z] = MODE == MUON ? ap.updated(x[t][4 * q + z], w[4 * q + z]) : x[t][4 * q + z];
                                if (i < m && j < n) store4<MODE>(mt.dst, row + i, v);
                            }
                            continue;
                        }
                        auto place_of = [&](int i, int jj) { return ((long)sub * mt.rows + (tall ? jj : i)) * mt.cols + (tall ? i : jj); };
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int i = 32 * t + acc_row(r, lane);
                            w[r] = ap.old<MODE>(mt, place_of(i < m ? i : m - 1, j < n ? j : n - 1));
                        }
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int i = 32 * t + acc_row(r, lane);
                            if (i < m && j < n) ap.store<MODE>(mt, place_of(i, j), x[t][r], w[r]);
                        }
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 32; ++r) {
                        const float v = x[r >> 4][r & 15];
                        const _Float16 hi = (_Float16)v;
                        xh[s][r >> 3][r & 7] = hi;
                        xl[s][r >> 3][r & 7] = (_Float16)fmaf((float)hi, -1.f, v);
                    }
                }
                if (NS > 1) __builtin_amdgcn_sched_barrier(0);
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
    if (n <= 256) small_body<MODE, 1>(p.s, mt, sub, L);
    else if (n <= 512) small_body<MODE, 2>(p.s, mt, sub, L);
    else small_body<MODE, 4>(p.s, mt, sub, L);
}

// ================================================================================================ large matrices
// All matrices of a call that are not small run together, whatever their shapes: per step one launch for A, one for B and one for
// the next X, over the tiles of all of them.
// Layout of every plane: blocks of 32 columns, row after row within a block, so that 16 rows of a block are 1 KB without a gap: the
// products are bound by their loads from the L2 (2 x 2048 x 2048 fp32: 1530 us with whole rows, 1470 us with blocks).
// Buffers of one matrix, padded to the tile in both directions with zeros that every step reproduces (A, B and X of a zero row
// or column are zero), so that no product needs a bounds check:  X [mp][np] and X^T [np][mp] (twice), R and B [mp][mp].  With X
// in both orders each of the three products contracts the contiguous dimension of both operands.
constexpr int MAX_LARGE = 24;
constexpr int NORM_PARTS = 1024;                         // partial sums of squares per matrix, at most
constexpr int CUS = 256, SLOTS = 1024, COUNTERS = 4 * SLOTS;      // partial sums of products that are cut along k: room for SLOTS wide tiles

struct LMat {
    long off;                       // of the first matrix's buffers in the workspace
    int m, n, mp, np, tall;
    int sub0, nsub;                 // matrices sub0 .. sub0 + nsub - 1 of the entry's batch
    int parts;
    int first, sym, full[2];        // matrices, tiles of the lower triangles, of X and of the result in the entries before this one
};
struct Large {
    char* ws;
    long o_part;                    // COUNTERS counters, then fp32 partial tiles
    int count, tile, split;
    LMat e[MAX_LARGE];
};

__device__ __forceinline__ long place(int rows, int r, int k) { return ((long)(k >> 5) * rows + r) * 32 + (k & 31); }

__host__ __device__ inline long align256(long v) { return (v + 255) / 256 * 256; }
struct Offsets {
    long x, xt0, xt1, r, b, d, e, xi, sq, per;
    __host__ __device__ Offsets(int mp, int np, bool split) {
        const long xp = 2l * mp * np, ap = 2l * mp * mp;
        long o = 0;
        x = o; o += align256(xp * (split ? 2 : 1));
        xt0 = o; o += align256(2 * xp);
        xt1 = o; o += align256(2 * xp);
        r = o; o += align256(ap * (split ? 2 : 1));
        b = o; o += align256(ap * (split ? 2 : 1));
        d = o; o += align256(4l * mp);
        e = o; o += align256(4l * mp);
        xi = o; o += align256(4l * (MAX_STEPS + 1));
        sq = o; o += align256(8l * NORM_PARTS);
        per = o;
    }
    __device__ __forceinline__ long xt(int k) const { return (k & 1) ? xt1 : xt0; }       // X^T before step k
};

struct LargeArgs { Step s; Large l; Mat m[MAX_LARGE]; int k, whole, cut; };

// partial sums of squares (64-bit), the momentum update on the way; grid (NORM_PARTS, matrices)
template <int MODE>
__global__ void __launch_bounds__(256) ns_norm_kernel(LargeArgs a) {
    __shared__ double sq[4];
    int q = 0;
    while (q + 1 < a.l.count && (int)blockIdx.y >= a.l.e[q + 1].first) ++q;
    const LMat& le = a.l.e[q];
    const Mat& mt = a.m[q];
    if ((int)blockIdx.x >= le.parts) return;
    const int at = (int)blockIdx.y - le.first, sub = le.sub0 + at;
    // threads walk the contiguous dimension of U, TX of them along it and 256 / TX along the other
    const bool by_col = mt.cs <= mt.rs;
    const int inner = by_col ? mt.cols : mt.rows, outer = by_col ? mt.rows : mt.cols;
    const long os = by_col ? mt.rs : mt.cs, is = by_col ? mt.cs : mt.rs, base = (long)sub * mt.bs;
    // four at a time where the addresses allow it
    const uintptr_t bytes = MODE == BF16 ? 8 : 16;
    const bool vec = is == 1 && inner % 4 == 0 && os % 4 == 0 && base % 4 == 0 && (uintptr_t)mt.src % bytes == 0 &&
                     (MODE != MUON || (by_col && (uintptr_t)mt.mom % 16 == 0));
    const int cols = vec ? inner / 4 : inner;
    int tx = 1;
    while (tx < 256 && tx < cols) tx *= 2;
    const int ty = 256 / tx, x0 = (int)threadIdx.x % tx, y0 = (int)threadIdx.x / tx;
    double s = 0;
    for (int o = (int)blockIdx.x * ty + y0; o < outer; o += le.parts * ty) {
        if (vec) {
#pragma unroll 4
            for (int i = x0; i < cols; i += tx) {
                float u[4];
                const long at4 = base + (long)o * os + 4l * i;
                if constexpr (MODE == BF16) {
                    const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const __bf16*>(mt.src) + at4);
                    u[0] = __uint_as_float(w.x << 16); u[1] = __uint_as_float(w.x & 0xffff0000u);
                    u[2] = __uint_as_float(w.y << 16); u[3] = __uint_as_float(w.y & 0xffff0000u);
                } else {
                    const float4 w = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(mt.src) + at4);
                    u[0] = w.x; u[1] = w.y; u[2] = w.z; u[3] = w.w;
                }
                if constexpr (MODE == MUON) {
                    float4* mp = reinterpret_cast<float4*>(mt.mom + ((long)sub * mt.rows + o) * mt.cols + 4l * i);
                    float4 w = *mp;
                    float* mo = &w.x;
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const float gs = u[z] * a.s.grad_scale;
                        mo[z] = fmaf(a.s.momentum, mo[z], gs);
                        u[z] = a.s.nesterov ? fmaf(a.s.momentum, mo[z], gs) : mo[z];
                    }
                    *mp = w;
                }
#pragma unroll
                for (int z = 0; z < 4; ++z) s = fma((double)u[z], (double)u[z], s);
            }
        } else {
#pragma unroll 4
            for (int i = x0; i < cols; i += tx) {
                const double u = load_u<MODE, true>(a.s, mt, sub, by_col ? o : i, by_col ? i : o);
                s = fma(u, u, s);
            }
        }
    }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) sq[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        const Offsets of(le.mp, le.np, a.l.split != 0);
        reinterpret_cast<double*>(a.l.ws + le.off + at * of.per + of.sq)[blockIdx.x] = sq[0] + sq[1] + sq[2] + sq[3];
    }
}

// X0 in both orders, a 64 x 64 tile per workgroup; the counters of the split products are cleared here
template <int MODE, bool SPLIT>
__global__ void __launch_bounds__(256) ns_prepare_kernel(LargeArgs a) {
    __shared__ _Float16 tile[2][64][72];
    __shared__ double part[4];
    int q = 0;
    while (q + 1 < a.l.count && (int)blockIdx.y >= a.l.e[q + 1].first) ++q;
    const LMat& le = a.l.e[q];
    const Mat& mt = a.m[q];
    const int at = (int)blockIdx.y - le.first, sub = le.sub0 + at;
    const int nj = le.np / 64, ni = le.mp / 64;
    if (blockIdx.x == 0 && blockIdx.y == 0)
        for (int t = threadIdx.x; t < COUNTERS; t += 256) reinterpret_cast<int*>(a.l.ws + a.l.o_part)[t] = 0;
    if ((int)blockIdx.x >= ni * nj) return;
    const Offsets of(le.mp, le.np, SPLIT);
    char* ws = a.l.ws + le.off + at * of.per;
    // the tile's values are on their way while the norm is added up
    const int i0 = (int)blockIdx.x / nj * 64, j0 = (int)blockIdx.x % nj * 64;
    const bool across = (mt.cs <= mt.rs) != (le.tall != 0);             // whether columns of X are contiguous in U
    float u[16];
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        const int t = (int)threadIdx.x + 256 * w, i = i0 + (across ? t >> 6 : t & 63), j = j0 + (across ? t & 63 : t >> 6);
        const int ic = i < le.m ? i : le.m - 1, jc = j < le.n ? j : le.n - 1;
        u[w] = load_u<MODE, false>(a.s, mt, sub, le.tall ? jc : ic, le.tall ? ic : jc);
        u[w] = i < le.m && j < le.n ? u[w] : 0.f;
    }
    double total = 0;
    for (int i = threadIdx.x; i < le.parts; i += 256) total += reinterpret_cast<const double*>(ws + of.sq)[i];
    total = wave_sum(total);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = total;
    __syncthreads();
    total = part[0] + part[1] + part[2] + part[3];
    int e;
    const float xi0 = scales(a.s, total, e);
    if (blockIdx.x == 0 && (int)threadIdx.x <= a.s.steps)
        reinterpret_cast<float*>(ws + of.xi)[threadIdx.x] = threadIdx.x == 0 ? xi0 : scale_at(a.s, log_norm(a.s, total), (int)threadIdx.x);
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        const int t = (int)threadIdx.x + 256 * w, i = across ? t >> 6 : t & 63, j = across ? t & 63 : t >> 6;
        const float v = scaled(u[w], e);
        const _Float16 hi = (_Float16)v;
        tile[0][i][j] = hi;
        tile[1][i][j] = (_Float16)(v - (float)hi);
    }
    __syncthreads();
    const long plane = (long)le.mp * le.np;
    _Float16* xt = reinterpret_cast<_Float16*>(ws + of.xt0);
    _Float16* x = reinterpret_cast<_Float16*>(ws + of.x);
#pragma unroll
    for (int pl = 0; pl < 2; ++pl)
        for (int t = threadIdx.x; t < 4096; t += 256) {
            const int r = (t >> 5) & 63, k = (t >> 11) * 32 + (t & 31);
            if (SPLIT || pl == 0) x[pl * plane + place(le.mp, i0 + r, j0 + k)] = tile[pl][r][k];
            xt[pl * plane + place(le.np, j0 + r, i0 + k)] = tile[pl][k][r];
        }
}

// One product of a step, C[i][j] = sum_k P[i][k] Q[j][k], and what follows it:
//   A_OF_X      P = Q = X, tiles of the lower triangle:   R = A - diag A (exactly symmetric), d = diag A
//   B_OF_A      P = Q = R, tiles of the lower triangle:   B - diag B, e = a + diag B
//   X_NEXT      P = B, Q = X^T:                            X, X^T
//   X_LAST      the same, result or weight update; TALL: P = X^T, Q = B, so that lanes run along U's rows either way
// Workgroups of TM x TN outputs, each wave WM x WN of them; NST stages of BK columns of P and Q in LDS, filled by LDS-DMA ahead of
// their use.  What bounds large products is that traffic from the L2 and the MALL (4096 x 4096, X in 128 x 128 tiles: 178 us; 157 us
// without the matrix instructions, 111 us without the loads); of small ones a third is the epilogue, which few workgroups share.
// Rows of a stage hold 16-byte chunks in an order that depends on the row (chunk c of row r at c ^ f(r)), so that the eight lanes
// that read at once hit all banks.
// Sums: along k in chunks of `chunk_of` columns; a chunk's sum is added to the tile's in the order of k.  Shorter chains of
// roundings, and the result does not depend on who computes which chunk.  X of single operands has one chain instead (the
// 256 x 256 tile has no registers for a second sum) and is never cut, so that a tile of any size gives the same bits.  bf16 squares,
// against chains and cuts that followed the tile: 1536 339 us for 369, 1792 424 for 599, 2560 723 for 864, but 2100 579 for 534
// and 2944 1027 for 938, whose 128 x 128 tiles just pass a multiple of the workgroups that run at once.
// Work split: of T tiles the first `whole` = 256 floor(T / 256) have a workgroup each; each chunk of the others has one of its
// own (`cut`), so that a round that is not full still occupies the chip (528 tiles would otherwise take as long as 768).  Such a
// workgroup leaves its fp32 sums in the workspace; the one that arrives last adds them in order and goes on with the tile.
enum { A_OF_X, B_OF_A, X_NEXT, X_LAST };
template <bool SPLIT, int KIND> constexpr bool folds() { return SPLIT || KIND == A_OF_X || KIND == B_OF_A; }

// 512 columns, more where there would be over 64 chunks; of the unpadded length, so that the tile makes no difference
__host__ __device__ inline int chunk_of(int k) {
    int c = 512;
    while (k > 64 * c) c *= 2;
    return c;
}

// tiles of a product: of the lower triangle, or of X (of U, transposed or not; the last row and column of tiles may be cut off)
template <int TM, int TN, int KIND> __host__ __device__ inline int tiles_of(const LMat& e) {
    if (KIND == A_OF_X || KIND == B_OF_A) return e.mp / TM * (e.mp / TM + 1) / 2;
    const bool swap = KIND == X_LAST && e.tall;
    return ((swap ? e.np : e.mp) + TM - 1) / TM * (((swap ? e.mp : e.np) + TN - 1) / TN);
}

template <int TM, int TN, int WM, int WN, int BK, int NST, bool SPLIT, int KIND>
__global__ void __launch_bounds__(TM / WM * (TN / WN) * 64, TM / WM * (TN / WN) == 4 ? 2 : 1) ns_gemm_kernel(LargeArgs a) {
    constexpr int WC = TN / WN, WAVES = TM / WM * WC, TH = 64 * WAVES;
    constexpr int NP = SPLIT ? 2 : 1, MT = WM / 32, NT = WN / 32, CH = BK / 8;
    constexpr bool WIDE = TM > 128 || TN > 128;                          // buffers are padded to 128: the last tile may be cut off
    constexpr int PBYTES = TM * BK * 2, QBYTES = TN * BK * 2, STAGE = NP * (PBYTES + QBYTES);
    constexpr int HALVES = NST * STAGE >= TM * (TN + 8) * 2 && NST * STAGE >= TN * (TM + 8) * 2 ? 1 : 2;      // the output tile reuses the stages
    static_assert(NST * STAGE >= TM / HALVES * (TN + 8) * 2 && NST * STAGE >= TN * (TM / HALVES + 8) * 2 && TM / HALVES >= WM, "output tile");
    static_assert((TM == TN && !WIDE && HALVES == 1) || KIND == X_NEXT || KIND == X_LAST, "a triangle of square tiles that fit the stages");
    __shared__ __attribute__((aligned(16))) char lds[NST * STAGE];
    __shared__ int arrived;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = wave / WC, wc = wave % WC;
    constexpr bool SYM = KIND == A_OF_X || KIND == B_OF_A, FOLD = folds<SPLIT, KIND>();
    int t, slice = 0, slices = 1, slot = 0, q = 0;      // slot: of the tile's first partial sums
    if ((int)blockIdx.x < a.whole) {
        t = (int)ksr_xcd_contiguous(blockIdx.x, (unsigned)a.whole);
        while (q + 1 < a.l.count && t >= (SYM ? a.l.e[q + 1].sym : a.l.e[q + 1].full[KIND == X_LAST])) ++q;
    } else {
        // entries whose tiles are cut: each with its own number of chunks
        int rest = (int)blockIdx.x - a.whole;
        for (;; ++q) {
            const LMat& e = a.l.e[q];
            const int first = SYM ? e.sym : e.full[KIND == X_LAST], tiles = e.nsub * tiles_of<TM, TN, KIND>(e);
            const int from = a.whole > first ? a.whole : first, cut = first + tiles - from;       // tiles of this entry in the rest
            if (cut <= 0) continue;
            const int ch = chunk_of(KIND == A_OF_X ? e.n : e.m), kp = KIND == A_OF_X ? e.np : e.mp, n = a.cut ? (kp + ch - 1) / ch : 1;
            if (rest < cut * n || q + 1 == a.l.count) {
                slices = n;
                slice = rest % n;
                slot = (int)blockIdx.x - a.whole - slice;
                t = from + rest / n;
                break;
            }
            rest -= cut * n;
        }
    }
    const LMat& l = a.l.e[q];
    t -= SYM ? l.sym : l.full[KIND == X_LAST];
    const bool swap = KIND == X_LAST && l.tall;
    const int mt = ((swap ? l.np : l.mp) + TM - 1) / TM, per = tiles_of<TM, TN, KIND>(l);
    const int at = t / per, sub = l.sub0 + at;
    t -= at * per;
    const Offsets of(l.mp, l.np, SPLIT);
    char* ws = a.l.ws + l.off + at * of.per;
    int ti, tj;
    if constexpr (SYM) {                                // ti + 1 tiles in row ti
        ti = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
        while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
        while (ti * (ti + 1) / 2 > t) --ti;
        tj = t - ti * (ti + 1) / 2;
    } else { ti = t % mt; tj = t / mt; }
    const _Float16* R = reinterpret_cast<const _Float16*>(ws + of.r);
    const _Float16* xt = reinterpret_cast<const _Float16*>(ws + of.xt(a.k));
    const _Float16 *P, *Q;
    long pp, qp;                                        // distance of the lo plane
    int K, pr, qr;                                      // columns, rows of P's and Q's planes
    if constexpr (KIND == A_OF_X) { P = Q = reinterpret_cast<const _Float16*>(ws + of.x); K = l.np; pr = qr = l.mp; pp = qp = (long)l.mp * l.np; }
    else if constexpr (KIND == B_OF_A) { P = Q = R; K = pr = qr = l.mp; pp = qp = (long)l.mp * l.mp; }
    else {
        const _Float16* B = reinterpret_cast<const _Float16*>(ws + of.b);
        P = swap ? xt : B; Q = swap ? B : xt; K = l.mp;
        pr = swap ? l.np : l.mp;
        qr = swap ? l.mp : l.np;
        pp = (long)pr * K;
        qp = (long)qr * K;
    }
    P += (long)ti * TM * 32;
    Q += (long)tj * TN * 32;
    // rows of P and Q that exist: fewer than the tile's in the last one of an odd number of 128s
    const int rows = pr - ti * TM, cols = qr - tj * TN;
    // LDS-DMA: one instruction of a wave brings 64 chunks of 16 bytes; lane -> (row, slot), the chunk that belongs there
    constexpr int ROWS = 64 / CH, PI = TM / ROWS / WAVES, QI = TN / ROWS / WAVES;        // rows per instruction, instructions per wave and plane
    constexpr int PER_STAGE = NP * (PI + QI);                           // a wave's instructions per stage
    const int drow = lane / CH, dslot = lane % CH;
    auto f = [](int row) { return CH == 8 ? (row & 7) : ((row >> 1) & 3); };
    auto fill = [&](int kt) {
        char* to = lds + kt % NST * STAGE;
#pragma unroll
        for (int pl = 0; pl < NP; ++pl) {
#pragma unroll
            for (int i = 0; i < PI; ++i) {
                const int row = (wave * PI + i) * ROWS + drow;
                const _Float16* src = P + pl * pp + place(pr, !WIDE || row < rows ? row : 0, kt * BK + 8 * (dslot ^ f(row)));
                ksr_dma16<false>(src, to + pl * PBYTES + (wave * PI + i) * 1024);
            }
#pragma unroll
            for (int i = 0; i < QI; ++i) {
                const int row = (wave * QI + i) * ROWS + drow;
                const _Float16* src = Q + pl * qp + place(qr, TN <= 128 || row < cols ? row : 0, kt * BK + 8 * (dslot ^ f(row)));
                ksr_dma16<false>(src, to + NP * PBYTES + pl * QBYTES + (wave * QI + i) * 1024);
            }
        }
    };
    auto frag = [&](int st, int at_byte, int row, int ks) {
        const int chunk = (2 * ks + (lane >> 5)) ^ f(row);
        return *reinterpret_cast<const h8*>(lds + st * STAGE + at_byte + row * (BK * 2) + 16 * chunk);
    };
    f32x16 acc[MT][NT] = {}, sum[FOLD ? MT : 1][FOLD ? NT : 1] = {};
    const int chunk = chunk_of(KIND == A_OF_X ? l.n : l.m) / BK, nk = K / BK;
    const int k0 = slices > 1 ? slice * chunk : 0, k1 = slices > 1 && k0 + chunk < nk ? k0 + chunk : nk;
    h8 ph[2][MT], qh[2][NT], pl[2][SPLIT ? MT : 1], ql[2][SPLIT ? NT : 1];
    // Two sets of operands: 16 columns are multiplied while the next 16 come out of LDS, also across a stage's end, so that the
    // barrier and the LDS' latency lie behind matrix work
    auto stage_ready = [&](int kt) {
        // stage kt has landed (of the NST - 2 younger ones this wave's transfers may be in flight, if there are that many), and
        // every wave has read all of stage kt - 1, whose place the next one takes
        if (kt + NST - 2 < k1) ksr_dma_barrier_but<PER_STAGE*(NST - 2)>();
        else ksr_dma_barrier();
        if (kt + NST - 1 < k1) fill(kt + NST - 1);
    };
    auto load = [&](int set, int kt, int ks) {
        const int st = kt % NST;
#pragma unroll
        for (int x = 0; x < MT; ++x) {
            ph[set][x] = frag(st, 0, wr * WM + 32 * x + (lane & 31), ks);
            if constexpr (SPLIT) pl[set][x] = frag(st, PBYTES, wr * WM + 32 * x + (lane & 31), ks);
        }
#pragma unroll
        for (int y = 0; y < NT; ++y) {
            qh[set][y] = frag(st, NP * PBYTES, wc * WN + 32 * y + (lane & 31), ks);
            if constexpr (SPLIT) ql[set][y] = frag(st, NP * PBYTES + QBYTES, wc * WN + 32 * y + (lane & 31), ks);
        }
    };
    for (int kt = k0; kt < k0 + NST - 1 && kt < k1; ++kt) fill(kt);
    stage_ready(k0);
    load(0, k0, 0);
    for (int c0 = k0; c0 < k1; c0 += chunk) {           // k0 is the start of a chunk
        const int c1 = FOLD && c0 + chunk < k1 ? c0 + chunk : k1;
        for (int kt = c0; kt < c1; ++kt)
#pragma unroll
            for (int ks = 0; ks < BK / 16; ++ks) {
                const int set = ks & 1;
                if (ks + 1 < BK / 16) load(set ^ 1, kt, ks + 1);
                else if (kt + 1 < k1) {
                    stage_ready(kt + 1);
                    load(set ^ 1, kt + 1, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int x = 0; x < MT; ++x)
#pragma unroll
                    for (int y = 0; y < NT; ++y) {
                        if constexpr (SPLIT) {
                            acc[x][y] = mfma(ph[set][x], ql[set][y], acc[x][y]);
                            acc[x][y] = mfma(pl[set][x], qh[set][y], acc[x][y]);
                        }
                        acc[x][y] = mfma(ph[set][x], qh[set][y], acc[x][y]);
                    }
                __builtin_amdgcn_sched_barrier(0);
            }
        if constexpr (!FOLD) break;
        else
#pragma unroll
            for (int x = 0; x < MT; ++x)
#pragma unroll
                for (int y = 0; y < NT; ++y) {
                    sum[x][y] += acc[x][y];
                    acc[x][y] = f32x16{};
                }
    }
    if constexpr (FOLD)
#pragma unroll
        for (int x = 0; x < MT; ++x)
#pragma unroll
            for (int y = 0; y < NT; ++y) acc[x][y] = sum[x][y];
    if (FOLD && slices > 1) {
        int* counter = reinterpret_cast<int*>(a.l.ws + a.l.o_part) + slot;
        float* part = reinterpret_cast<float*>(a.l.ws + a.l.o_part + 4l * COUNTERS) + (long)slot * TM * TN + threadIdx.x;
        float* own = part + (long)slice * TM * TN;
#pragma unroll
        for (int x = 0; x < MT; ++x)
#pragma unroll
            for (int y = 0; y < NT; ++y)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    __hip_atomic_store(own + ((x * NT + y) * 16 + r) * TH, acc[x][y][r], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // Device-scope accesses go past the caches of the eight dies, and a wave's are complete when its count of outstanding ones
        // is 0: the sums are in place before the arrival is counted.  (A release fence would write back a whole L2 per workgroup.)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) arrived = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (arrived != slices - 1) return;
        if (threadIdx.x == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);       // for the next launch
#pragma unroll
        for (int x = 0; x < MT; ++x)
#pragma unroll
            for (int y = 0; y < NT; ++y) acc[x][y] = f32x16{};
        for (int w = 0; w < slices; ++w)
#pragma unroll
            for (int x = 0; x < MT; ++x)
#pragma unroll
                for (int y = 0; y < NT; ++y)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        acc[x][y][r] += __hip_atomic_load(part + (long)w * TM * TN + ((x * NT + y) * 16 + r) * TH, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    ksr_lds_barrier();                                  // LDS is free for the output tile
    // ---- values
    const float* xis = reinterpret_cast<const float*>(ws + of.xi);
    float* dv = reinterpret_cast<float*>(ws + of.d);
    float* ev = reinterpret_cast<float*>(ws + of.e);
    const Step& sp = a.s;
    const float xi = xis[a.k], rn = KIND == X_NEXT ? 1.f / xis[a.k + 1] : 1.f;
    const Mat& mat = a.m[q];
    const Apply ap(sp, mat);
    const int mode = sp.muon ? MUON : sp.bf16 ? BF16 : F32;
#pragma unroll
    for (int x = 0; x < MT; ++x)
#pragma unroll
        for (int y = 0; y < NT; ++y) {
            float w[KIND == X_LAST ? 16 : 1];
            if constexpr (KIND == X_LAST)
                if (mode == MUON) {
                    const int c = tj * TN + wc * WN + 32 * y + (lane & 31), cc = c < mat.cols ? c : mat.cols - 1;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int r = ti * TM + wr * WM + 32 * x + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
                        w[i] = ap.old<MUON>(mat, ((long)sub * mat.rows + (r < mat.rows ? r : mat.rows - 1)) * mat.cols + cc);
                    }
                }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int row0 = ti * TM + wr * WM + 32 * x + 8 * g + 4 * (lane >> 5), c = tj * TN + wc * WN + 32 * y + (lane & 31);
                float v[4];
#pragma unroll
                for (int z = 0; z < 4; ++z) v[z] = acc[x][y][4 * g + z];
                if constexpr (KIND == A_OF_X) {
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        v[z] *= xi * xi;
                        if (row0 + z == c) { dv[c] = v[z]; v[z] = 0.f; }
                        v[z] *= S;
                    }
                } else if constexpr (KIND == B_OF_A) {
                    const h4 rh = *reinterpret_cast<const h4*>(R + place(l.mp, c, row0));       // R is symmetric
                    h4 rl = {};
                    if constexpr (SPLIT) rl = *reinterpret_cast<const h4*>(R + pp + place(l.mp, c, row0));
                    const float dc = dv[c];
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const float di = dv[row0 + z], r = ((float)rh[z] + (float)rl[z]) * INV_S, sq = v[z] * (INV_S * INV_S);
                        if (row0 + z == c) {
                            ev[c] = sp.a + sp.b * di + sp.c * (di * di + sq);
                            v[z] = 0.f;
                        } else v[z] = S * (sp.b * r + sp.c * ((di + dc) * r + sq));
                    }
                } else if (!WIDE || (row0 - ti * TM < rows && c - tj * TN < cols)) {
                    const float alpha = xi * INV_S;
                    const long plane = (long)l.mp * l.np;
                    if (!swap) {                        // rows are i, columns j
                        const h4 xh = *reinterpret_cast<const h4*>(xt + place(l.np, c, row0)), xl = *reinterpret_cast<const h4*>(xt + plane + place(l.np, c, row0));
#pragma unroll
                        for (int z = 0; z < 4; ++z) v[z] = fmaf(ev[row0 + z], ((float)xh[z] + (float)xl[z]) * xi, v[z] * alpha);
                    } else {
                        const float ec = ev[c];
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            const long o = place(l.np, row0 + z, c);
                            v[z] = fmaf(ec, ((float)xt[o] + (float)xt[plane + o]) * xi, v[z] * alpha);
                        }
                    }
                    if constexpr (KIND == X_LAST) {
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            const int r = row0 + z;     // rows and columns of the result are those of U either way
                            if (r < mat.rows && c < mat.cols) {
                                const long o = ((long)sub * mat.rows + r) * mat.cols + c;
                                if (mode == F32) ap.store<F32>(mat, o, v[z], 0.f);
                                else if (mode == BF16) ap.store<BF16>(mat, o, v[z], 0.f);
                                else ap.store<MUON>(mat, o, v[z], w[KIND == X_LAST ? 4 * g + z : 0]);
                            }
                        }
                    } else {
#pragma unroll
                        for (int z = 0; z < 4; ++z) v[z] *= rn;
                    }
                }
#pragma unroll
                for (int z = 0; z < 4; ++z) acc[x][y][4 * g + z] = v[z];
                if (WIDE && g == 3) __builtin_amdgcn_sched_barrier(0);        // more of X^T in flight would spill
            }
        }
    if constexpr (KIND == X_LAST) return;
    // ---- the tile and its transpose, hi and lo, through LDS: 16-byte stores of whole rows
    _Float16* stage = reinterpret_cast<_Float16*>(lds);
    _Float16 *out, *outt;
    long plane;
    int onr, ort;                                       // rows of the planes that are written
    constexpr int planes = (KIND == X_NEXT || SPLIT) ? 2 : 1;
    if constexpr (KIND == X_NEXT) {
        out = reinterpret_cast<_Float16*>(ws + of.x); outt = reinterpret_cast<_Float16*>(ws + of.xt(a.k + 1));
        onr = l.mp; ort = l.np; plane = (long)l.mp * l.np;
    } else {
        out = outt = reinterpret_cast<_Float16*>(ws + (KIND == A_OF_X ? of.r : of.b));
        onr = ort = l.mp; plane = (long)l.mp * l.mp;
    }
#pragma unroll
    for (int pl = 0; pl < planes; ++pl)
#pragma unroll
        for (int tr = 0; tr < 2; ++tr) {
            if (tr == 0 && pl == 1 && !SPLIT) continue;              // X's lo is only read through X^T (the linear term)
#pragma unroll
            for (int half = 0; half < HALVES; ++half) {
                constexpr int HM = TM / HALVES;                      // rows of the tile in LDS at a time
                if constexpr (WIDE)                                       // nothing rounded is kept for the next round: it would spill
#pragma unroll
                    for (int x = 0; x < MT; ++x)
#pragma unroll
                        for (int y = 0; y < NT; ++y) asm volatile("" : "+v"(acc[x][y]));
                if (HALVES == 1 || wr * WM / HM == half)
#pragma unroll
                    for (int x = 0; x < MT; ++x)
#pragma unroll
                        for (int y = 0; y < NT; ++y)
#pragma unroll
                            for (int g = 0; g < 4; ++g) {
                                const int r = wr * WM - half * HM + 32 * x + 8 * g + 4 * (lane >> 5), c = wc * WN + 32 * y + (lane & 31);
                                h4 w;
#pragma unroll
                                for (int z = 0; z < 4; ++z) {
                                    const float v = acc[x][y][4 * g + z];
                                    const _Float16 hi = (_Float16)v;
                                    w[z] = pl ? (_Float16)(v - (float)hi) : hi;
                                }
                                if (tr) *reinterpret_cast<h4*>(stage + c * (HM + 8) + r) = w;
                                else {
#pragma unroll
                                    for (int z = 0; z < 4; ++z) stage[(r + z) * (TN + 8) + c] = w[z];
                                }
                            }
                ksr_lds_barrier();                                       // stores of the tile stay in flight across it
                _Float16* o = (tr ? outt : out) + pl * plane;
                const int i0 = ti * TM + half * HM, j0 = tj * TN, of_rows = tr ? ort : onr;
                constexpr int PITCH_N = TN + 8, PITCH_M = HM + 8;
                const int height = tr ? TN : HM, pitch = tr ? PITCH_M : PITCH_N;
                for (int w = threadIdx.x; w < HM * TN / 8; w += TH) {
                    const int r = (w >> 2) % height, c = (w >> 2) / height * 32 + (w & 3) * 8;        // along a block of 32 columns
                    const int i = tr ? c : r, j = tr ? r : c;        // row and column of the product's tile
                    _Float16* to = o + place(of_rows, (tr ? j0 : i0) + r, (tr ? i0 : j0) + c);
                    if constexpr (SYM) {
                        // Above the diagonal stand the transposes of what is below it, in the diagonal's own tiles too: what these
                        // computed there has hi lo and lo hi added in the other order, and where they end depends on the tile
                        if (ti == tj) {
                            if (tr ? c <= r : c > r) continue;
                            if (SPLIT && !tr && c + 7 > r) {            // eight columns across the diagonal
                                h8 v;
#pragma unroll
                                for (int z = 0; z < 8; ++z) v[z] = stage[(c + z > r ? c + z : r) * pitch + (c + z > r ? r : c + z)];
                                *reinterpret_cast<h8*>(to) = v;
                                continue;
                            }
                        }
                    } else if (WIDE && !(half * HM + i < rows && j < cols)) continue;      // beyond an odd number of 128s
                    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(stage + r * pitch + c);
                }
                ksr_lds_barrier();
            }
        }
}

// ------------------------------------------------------------------------------------------------ host
bool is_small(int rows, int cols) { return rows < cols ? rows <= 64 && cols <= 1024 : cols <= 64 && rows <= 1024; }
bool empty(const KsrMatrix& q) { return !q.rows || !q.cols || !q.batch; }

// Matrices that run together: as many as fit 1 GiB of buffers, at least one.  (entry, index in its batch) of the first one that
// is left is advanced; returns the bytes the group needs, 0 at the end of the list.
constexpr long WS_CAP = 1l << 30;

long next_group(const KsrMatrix* mats, int count, bool split, int& entry, int& sub, Large& l, Mat* m) {
    const int entry0 = entry, sub0 = sub;
    l.count = 0;
    l.split = split;
    for (int pass = 0; pass < 2; ++pass) {
        // the tile: 128 where that gives at least 128 tiles of X.  A wide tile reads less, many narrow ones fill the chip: 12 matrices
        // with 466 wide tiles: X 42 us so and 61 us with narrow ones; 777 x 2051 (119 wide tiles) is latency, 14 us narrow
        l.tile = pass == 0 ? 128 : 64;
        l.count = 0;
        entry = entry0;
        sub = sub0;
        long off = 0;
        int matrices = 0;
        long full = 0;
        for (; entry < count && l.count < MAX_LARGE; ++entry, sub = 0) {
            const KsrMatrix& k = mats[entry];
            if (empty(k) || is_small(k.rows, k.cols)) continue;
            LMat& e = l.e[l.count];
            e.tall = k.rows > k.cols;
            e.m = e.tall ? k.cols : k.rows;
            e.n = e.tall ? k.rows : k.cols;
            e.mp = (e.m + l.tile - 1) / l.tile * l.tile;
            e.np = (e.n + l.tile - 1) / l.tile * l.tile;
            const long per = Offsets(e.mp, e.np, split).per, mt = e.mp / l.tile, nt = e.np / l.tile;
            long room = (WS_CAP - off) / per;
            if (room < 1) {
                if (l.count) break;
                room = 1;
            }
            if (room > 60000 - matrices) room = 60000 - matrices;               // the grid's second dimension
            if (room < 1) break;
            const int left = k.batch - sub;
            e.nsub = left < room ? left : (int)room;
            e.sub0 = sub;
            const long elements = (long)e.m * e.n;
            e.parts = elements / 4096 < 1 ? 1 : elements / 4096 < NORM_PARTS ? (int)(elements / 4096) : NORM_PARTS;
            e.off = off;
            e.first = matrices;
            m[l.count++] = Mat{k.src, k.dst, k.momentum, (long)k.row_stride, (long)k.col_stride, (long)k.batch_stride, k.rows, k.cols, k.batch, 0, 0};
            off += e.nsub * per;
            matrices += e.nsub;
            full += e.nsub * mt * nt;
            if (e.nsub < left) { sub += e.nsub; break; }
        }
        if (!l.count) return 0;
        l.o_part = off;
        if (pass == 1 || full >= 128) break;
    }
    return l.o_part + 4l * COUNTERS + 4l * SLOTS * l.tile * l.tile;
}

// Largest singular value that each step can reach from [0, 1], and that A and B stay inside f16's range
bool bounded(float a, float b, float c, int steps, float& log2_gain) {
    double top = 1.0, g = fabs((double)a);
    for (int k = 0; k < steps; ++k) {
        double next = 0;
        for (int i = 0; i <= 128; ++i) {
            const double s = top * 1.02 * i / 128, s2 = s * s, f = a + b * s2 + c * s2 * s2;
            if (fabs(f) > g) g = fabs(f);
            if (fabs(f) * s > next) next = fabs(f) * s;
            if (!(s2 <= 30) || !(fabs(b * s2 + c * s2 * s2) <= 30) || !(fabs(f) * s <= 30)) return false;
        }
        top = next;
    }
    log2_gain = (float)(g > 1 ? log2(g) : 0);
    return true;
}

template <int MODE, bool SPLIT> void start_large(const LargeArgs& a, hipStream_t st) {
    unsigned matrices = 0, parts = 1, tiles = 1;
    for (int i = 0; i < a.l.count; ++i) {
        const LMat& e = a.l.e[i];
        matrices = (unsigned)(e.first + e.nsub);
        if ((unsigned)e.parts > parts) parts = (unsigned)e.parts;
        const unsigned t = (unsigned)((long)(e.mp / 64) * (e.np / 64));
        if (t > tiles) tiles = t;
    }
    hipLaunchKernelGGL((ns_norm_kernel<MODE>), dim3(parts, matrices), dim3(256), 0, st, a);
    hipLaunchKernelGGL((ns_prepare_kernel<MODE, SPLIT>), dim3(tiles, matrices), dim3(256), 0, st, a);
}

template <int TM, int TN, int WM, int WN, int BK, int NST, bool SPLIT, int KIND> void product(LargeArgs& a, hipStream_t st) {
    constexpr bool SYM = KIND == A_OF_X || KIND == B_OF_A;
    int tiles = 0;
    for (int i = 0; i < a.l.count; ++i) {
        LMat& e = a.l.e[i];
        (SYM ? e.sym : e.full[KIND == X_LAST]) = tiles;
        tiles += e.nsub * tiles_of<TM, TN, KIND>(e);
    }
    a.whole = tiles / CUS * CUS;
    long cut = 0;                                       // workgroups if every chunk of the rest has one
    for (int i = 0; i < a.l.count; ++i) {
        const LMat& e = a.l.e[i];
        const int first = SYM ? e.sym : e.full[KIND == X_LAST], from = a.whole > first ? a.whole : first, n = first + e.nsub * tiles_of<TM, TN, KIND>(e) - from;
        const int ch = chunk_of(KIND == A_OF_X ? e.n : e.m), kp = KIND == A_OF_X ? e.np : e.mp;
        if (n > 0) cut += (long)n * ((kp + ch - 1) / ch);
    }
    // Cut only what is worth its traffic: four chunks or more, or fewer tiles than CUs (429 tiles of 832 columns in two chunks: 20 us,
    // uncut 14 us), and no single chains (see above)
    a.cut = folds<SPLIT, KIND>() && cut <= COUNTERS && cut * TM * TN <= (long)SLOTS * a.l.tile * a.l.tile && (tiles < CUS || cut >= 4l * (tiles - a.whole));
    hipLaunchKernelGGL((ns_gemm_kernel<TM, TN, WM, WN, BK, NST, SPLIT, KIND>), dim3((unsigned)(a.cut ? a.whole + cut : tiles)), dim3(TM / WM * (TN / WN) * 64), 0, st, a);
}

template <int TM, int TN, int KIND> long tiles_in(const Large& l) {
    long n = 0;
    for (int i = 0; i < l.count; ++i) n += (long)l.e[i].nsub * tiles_of<TM, TN, KIND>(l.e[i]);
    return n;
}

// The tile of a product, by the number of tiles (us; f fp32 and SPLIT, b bf16 and single):
//   A and B: 64 x 64 below 160 tiles of 128 x 128.  136 tiles (2048 x 2048), A: f 61 against 68, b 28 against 35; 113 of 12 matrices
//   512 wide, B: f 21 against 34.  210 tiles (2560 x 2560), A: f 115 against 88, b 46 against 37.
//   X: 256 x 256 (b, 8 waves) where rounds of 256 workgroups are 85 % full, never cut.  256 tiles: 156, in 128 x 128 183; 304 tiles:
//   282 against 230; 36 tiles, cut: 143 against 30.  SPLIT 256 x 128: 112 against 114 at 256 tiles, 214 against 171 at 384: not used.
//   64 x 64 does not pay: 144 tiles of 128 x 128 (1536 x 1536): f 45 against 61, b 30 against 28; 256 tiles: f 69 against 92, b 34 against 45.
// Stages: two of 64 columns (four of 32, A b at 4096: 110 against 102); SPLIT two of 32 (three: 95 against 77).  64 x 64: three, so
// that three workgroups share a CU (four: A at 1024 x 4096 f 45 against 39, b 27 against 23; two: 777 x 2051 b 255 against 245).
template <bool SPLIT, int KIND> void product_of_size(LargeArgs& a, hipStream_t st) {
    constexpr int BK = SPLIT ? 32 : 64;
    if (a.l.tile == 64) return product<64, 64, 32, 32, BK, 3, SPLIT, KIND>(a, st);
    if constexpr (KIND == A_OF_X || KIND == B_OF_A) {
        if (tiles_in<128, 128, KIND>(a.l) < 5 * CUS / 8) return product<64, 64, 32, 32, BK, 3, SPLIT, KIND>(a, st);
    } else if constexpr (!SPLIT) {
        const long wide = tiles_in<256, 256, KIND>(a.l);
        if (20 * wide >= 17 * ((wide + CUS - 1) / CUS * CUS)) return product<256, 256, 128, 64, 32, 4, false, KIND>(a, st);
    }
    product<128, 128, 64, 64, BK, 2, SPLIT, KIND>(a, st);
}

template <bool SPLIT> int run_large(LargeArgs& a, hipStream_t st) {
    const int mode = mode_of(a.s);
    if (mode == F32) start_large<F32, SPLIT>(a, st);
    else if (mode == BF16) start_large<BF16, SPLIT>(a, st);
    else start_large<MUON, SPLIT>(a, st);
    KSR_LAUNCH_CHECK("muon_batch");
    for (a.k = 0; a.k < a.s.steps; ++a.k) {
        product_of_size<SPLIT, A_OF_X>(a, st);
        product_of_size<SPLIT, B_OF_A>(a, st);
        if (a.k + 1 < a.s.steps) product_of_size<SPLIT, X_NEXT>(a, st);
        else product_of_size<SPLIT, X_LAST>(a, st);
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
    Large l;
    Mat m[MAX_LARGE];
    for (int entry = 0, sub = 0; entry < count;) {
        const int64_t need = next_group(mats, count, split != 0, entry, sub, l, m);
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
    p.s = Step{steps, bf16, muon, nesterov, a, b, c, eps, 0.f, momentum, grad_scale, lr, weight_decay, scale, lr_dev};
    KSR_UNSUPPORTED(!bounded(a, b, c, steps, p.s.log2_gain), "muon_batch: with coefficients (%g, %g, %g) %d steps leave the range of the products (30)",
                    (double)a, (double)b, (double)c, steps);
    KSR_CHECK_ARG(ws_bytes >= ksr_muon_ws_bytes(mats, count, split), "muon_batch: the workspace has %lld bytes, %lld are needed",
                  (long long)ws_bytes, (long long)ksr_muon_ws_bytes(mats, count, split));
    KSR_CHECK_ARG((ws || ws_bytes == 0) && reinterpret_cast<uintptr_t>(ws) % 16 == 0, "muon_batch: null or misaligned workspace");
    // every small matrix of the list in one launch, of up to MAX_MATS entries and SMALL_WGS matrices; `sub`: what of entry i is done
    for (int i = 0, sub = 0; i < count;) {
        p.count = 0;
        int total = 0;
        for (; i < count && p.count < MAX_MATS && total < SMALL_WGS; ++i, sub = 0) {
            const KsrMatrix& q = mats[i];
            if (empty(q) || !is_small(q.rows, q.cols)) continue;
            const int left = q.batch - sub, n = left < SMALL_WGS - total ? left : SMALL_WGS - total;
            p.m[p.count++] = Mat{q.src, q.dst, q.momentum, (long)q.row_stride, (long)q.col_stride, (long)q.batch_stride, q.rows, q.cols, q.batch, total, sub};
            total += n;
            if (n < left) { sub += n; break; }
        }
        if (!p.count) continue;
        const int mode = mode_of(p.s);
        if (mode == F32) hipLaunchKernelGGL(ns_small_kernel<F32>, dim3((unsigned)total), dim3(512), 0, stream, p);
        else if (mode == BF16) hipLaunchKernelGGL(ns_small_kernel<BF16>, dim3((unsigned)total), dim3(512), 0, stream, p);
        else hipLaunchKernelGGL(ns_small_kernel<MUON>, dim3((unsigned)total), dim3(512), 0, stream, p);
        KSR_LAUNCH_CHECK("muon_batch");
    }
    LargeArgs g{};
    g.s = p.s;
    g.l.ws = reinterpret_cast<char*>(ws);
    for (int entry = 0, sub = 0; entry < count;) {
        if (!next_group(mats, count, split != 0, entry, sub, g.l, g.m)) break;
        int rc;
        rc = split ? run_large<true>(g, stream) : run_large<false>(g, stream);
        if (rc) return rc;
    }
    return KSR_OK;
}
