// Low-rank adapters of many requests beside a shared projection (the heads of models/humaniflow_model.py:232-252 with the weights of one trained model and a
// small difference to them for every subject, camera or data set):
//
//   l = ids[m] (negative: no adapter)      t[m] = s_l A_l x[m]              (r values, 32 bits, kept for the backward pass)
//   y[m] = W x[m] + b + B_l t[m]           W (N, K), A (L, r, K), B (L, N, r)
//   u[m] = s_l B_l^T dy[m]                 dx[m] = W^T dy[m] + A_l^T u[m]
//   dA_l = sum_{m: ids[m] = l} u[m] x[m]^T      dB_l = sum dy[m] t[m]^T     (an adapter without rows: zero)
//
// Three forms by the number of rows:
//   one to four (a single image): one launch of dot products.
//   few rows (M <= kFewRows: a batch of images): the weights are read once and bound everything.  32 x 32 tiles straight from global memory on the fp32 MFMA, the
//     reduction split over waves and work-groups until the chip is full; the rows' own adapters are dot products of the rows; one joining launch
//     adds the partial sums (a fixed order), the bias and the adapters' part.  Two launches.
//   many rows: rows are put in the order of their adapters (a plan of two index arrays), and a tile of 128 rows treats its few adapters as more columns of
//     the reduction: [x, t] . [W, B_l]^T, with t zero in the columns of the other rows' adapters.
// Everything is accumulated in 32 bits.  bfloat16 operands of the many-row form are exact; t and u enter it as a high and a low bfloat16 (16 bits of mantissa),
// so the adapters' part loses nothing against the output's own rounding.
#include <algorithm>
#include <type_traits>
#include "hmf_common.h"

namespace hmf {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short bf16_t;

constexpr int kFewRows = 256;          // also the most rows of one piece of a gradient sum (LDS list)
constexpr int kMaxRank = 64;

__device__ __forceinline__ float up(float v) { return v; }
__device__ __forceinline__ float up(bf16_t h) { return __uint_as_float((unsigned)h << 16); }
__device__ __forceinline__ bf16_t to_bf16(float f) { return __builtin_bit_cast(bf16_t, (__bf16)f); }      // nearest even, one instruction (a NaN stays one)
// a number less its nearest bfloat16 (exact; an infinity or NaN leaves nothing): 8 of its 24 bits at a time
__device__ __forceinline__ float bf16_left(float v) {
    const bf16_t h = to_bf16(v);
    return (h & 0x7f80u) == 0x7f80u ? 0.f : v - up(h);
}
__device__ __forceinline__ void down(float* p, float v) { *p = v; }
__device__ __forceinline__ void down(bf16_t* p, float v) { *p = to_bf16(v); }

// Four consecutive elements at p as floats, `n` of them valid and zero behind; n <= 0: none.  Every load is made, at the last valid place where its own is none (at least one
// element, VEC: four, lies in front of p + n): behind conditions each would be waited for before the next (4 rows, 1,940 -> 1,379, rank 15, bfloat16: 78 us).
// VEC: the caller guarantees alignment, and n is a multiple of 4.
template <bool VEC, typename T> __device__ __forceinline__ f32x4 load4(const T* p, int n) {
    typedef __attribute__((ext_vector_type(4))) T t4;
    t4 h;
    if (VEC) h = *(const t4*)(p + (n > 0 ? 0 : n - 4));
    else
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = p[min(k, n - 1)];
    f32x4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = k < n ? up((T)h[k]) : 0.f;
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ bool finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ bool finite(bf16_t v) { return (v & 0x7f80u) != 0x7f80u; }
__device__ __forceinline__ float nan32() { return __uint_as_float(0x7fc00000u); }

template <typename T> struct AdArgs {
    const T *x, *w, *bias, *a, *b, *dy;       // forward: x; backward: dy (x of the gradients: AdGrad)
    const float* scale;
    const int* ids;
    T *y, *dx;
    float *t, *u, *partial;
    long long ldx;
    int M, K, N, r, L, ksplit, kw;            // kw: reduction elements of one wave of one split (a multiple of 8)
};

// ---------------------------------------------------------------------------------------------------
// few rows
// ---------------------------------------------------------------------------------------------------
// t[m][j] = s_l sum_k x[m][k] A[l][j][k]: one work-group per row, four ranks of a wave at a time, lanes along K
template <typename T, bool VEC>
__device__ __forceinline__ void low_row(const AdArgs<T>& a, int m, float* t) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int l = a.ids[m];
    if (l < 0 || l >= a.L) {                                               // no adapter: zero; an id that no adapter has: NaN, so that it is seen
        for (int j = threadIdx.x; j < a.r; j += 256) t[j] = l < 0 ? 0.f : nan32();
        return;
    }
    const T* xr = a.x + (long long)m * a.ldx;
    const T* al = a.a + (long long)l * a.r * a.K;
    const float s = a.scale[l];
    for (int j0 = wave * 4; j0 < a.r; j0 += 16) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int k0 = lane * 4; k0 - lane * 4 < a.K; k0 += 512) {          // ten loads in flight
            f32x4 xv[2], av[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = k0 + 256 * h;
                xv[h] = load4<VEC>(xr + k, a.K - k);
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) av[h][jj] = load4<VEC>(al + (long long)min(j0 + jj, a.r - 1) * a.K + k, a.K - k);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int jj = 0; jj < 4; ++jj)
                    acc[jj] = fmaf(xv[h][0], av[h][jj][0], fmaf(xv[h][1], av[h][jj][1], fmaf(xv[h][2], av[h][jj][2], fmaf(xv[h][3], av[h][jj][3], acc[jj]))));
        }
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
            const float v = wave_sum(acc[jj]);
            if (lane == 0 && j0 + jj < a.r) t[j0 + jj] = s * v;
        }
    }
}

// u[m][j] = s_l sum_n dy[m][n] B[l][n][j]: lane = (row n of a group, rank j), so that B is read in order; the waves take a quarter of N each
template <typename T>
__device__ __forceinline__ void up_row(const AdArgs<T>& a, int m, float* red) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int l = a.ids[m];
    if (l < 0 || l >= a.L) {
        for (int j = threadIdx.x; j < a.r; j += 256) a.u[(long long)m * a.r + j] = l < 0 ? 0.f : nan32();
        return;
    }
    const int per = 64 / a.r, j = lane % a.r, g = lane / a.r;              // r <= 64
    const T* dr = a.dy + (long long)m * a.N;
    const T* bl = a.b + (long long)l * a.N * a.r;
    float acc = 0.f;
    if (g < per)
        for (int nb = wave * per + g; nb < a.N; nb += 4 * per * 16) {      // 16 rows of B in flight (one: 1,378 outputs at rank 63 took 54 us)
            T d[16], b[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const int n = min(nb + 4 * per * k, a.N - 1);
                d[k] = dr[n];
                b[k] = bl[(long long)n * a.r + j];
            }
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (nb + 4 * per * k < a.N) acc = fmaf(up(d[k]), up(b[k]), acc);
        }
    red[wave * 64 + lane] = acc;
    __syncthreads();
    if (threadIdx.x < a.r) {
        float v = 0.f;
        for (int w = 0; w < 4; ++w)
            for (int q = 0; q < per; ++q) v += red[w * 64 + q * a.r + threadIdx.x];
        a.u[(long long)m * a.r + threadIdx.x] = a.scale[l] * v;
    }
}

// partial[ks][m][o] = sum over the split's reduction range of  in[m][c] w(o, c);  NT: w(o, c) = W[o][c] (forward), else W[c][o] (backward).
// The weight is the MFMA's A operand (rows o), the activations its B operand (columns m); a group of 8 reduction elements is 4 MFMA steps whose two lane halves
// hold elements 4 q + step.
template <typename T, bool NT, bool VEC>
__device__ __forceinline__ void base_tile(const AdArgs<T>& a, const T* in, long long ldin, int O, int Cn, int ot, int ks, int mt, float* red) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 31, q = lane >> 5;
    const int o = ot * 32 + i, m = mt * 32 + i;
    const int c0 = (ks * 4 + wave) * a.kw, c1 = min(c0 + a.kw, Cn);
    const T* ir = in + (long long)min(m, a.M - 1) * ldin;
    const int oc = min(o, O - 1);
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
    constexpr int U = 4;                                                   // groups of 8 in flight: 128 bytes of a fp32 weight row
    for (int c = c0; c < c1; c += 8 * U) {
        f32x4 wv[U], xv[U];
#pragma unroll
        for (int g = 0; g < U; ++g) {
            const int cc = c + 8 * g + 4 * q, n = c1 - cc;
            xv[g] = load4<VEC>(ir + cc, n);
            if (NT) {
                wv[g] = load4<VEC>(a.w + (long long)oc * Cn + cc, n);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const T h = a.w[(long long)min(cc + e, c1 - 1) * O + oc];
                    wv[g][e] = e < n ? up(h) : 0.f;
                }
            }
        }
#pragma unroll
        for (int g = 0; g < U; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(wv[g][e], xv[g][e], acc, 0, 0, 0);
    }
    // acc[e] of lane (m, q) is output 8 (e >> 2) + 4 q + (e & 3): the four waves meet in LDS
#pragma unroll
    for (int e = 0; e < 16; ++e) red[(wave * 32 + 8 * (e >> 2) + 4 * q + (e & 3)) * 33 + i] = acc[e];
    __syncthreads();
    const int oo = threadIdx.x & 31;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int mm = (threadIdx.x >> 5) + 8 * s;
        if (mt * 32 + mm < a.M && ot * 32 + oo < O) {
            const float v = ((red[oo * 33 + mm] + red[(32 + oo) * 33 + mm]) + red[(64 + oo) * 33 + mm]) + red[(96 + oo) * 33 + mm];
            a.partial[((long long)ks * a.M + mt * 32 + mm) * O + ot * 32 + oo] = v;
        }
    }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void k_ad_few(const AdArgs<T> a, int tiles_o, int tiles_m) {
    __shared__ float red[4 * 32 * 33];
    const int nb = tiles_o * a.ksplit * tiles_m;
    if ((int)blockIdx.x >= nb) {
        low_row<T, VEC>(a, blockIdx.x - nb, a.t + (long long)(blockIdx.x - nb) * a.r);
        return;
    }
    const int ot = blockIdx.x % tiles_o, rest = blockIdx.x / tiles_o;
    base_tile<T, true, VEC>(a, a.x, a.ldx, a.N, a.K, ot, rest % a.ksplit, rest / a.ksplit, red);
}

// One to four rows (a single image): everything in ONE launch, since a second one costs as much as the work.  A work-group finds the rows' t itself -- A_l is read once per
// work-group, from L2 -- and then its waves two outputs each, lanes along K.  1 row, 2,048 -> 1,024, rank 16 in 32 bits: 7.6 us, and two launches of 9 us in all in the form below.
constexpr int kOneRows = 4, kOneBytes = 512 << 10, kOneOdd = 64 << 10;      // rows; bytes of A that a work-group reads for them, and where it reads them element by
// element: a width, pitch or address that is no multiple of four elements (4 rows, 1,941 -> 1,379, rank 15: 56 us, 18 below; 2,048 -> 1,024, rank 16, of a wider view: 55 us,
// 19 below; 4 rows, 1,001 -> 64, rank 8, bfloat16: 16 us, 18 below)
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void k_ad_one(const AdArgs<T> a) {
    __shared__ float st[kOneRows][kMaxRank];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n0 = blockIdx.x * 8 + wave * 2;
    // the outputs' own products first: their loads are on their way while t is found
    float y[kOneRows][2];
#pragma unroll
    for (int m = 0; m < kOneRows; ++m) y[m][0] = y[m][1] = 0.f;
    const T *w0 = a.w + (long long)min(n0, a.N - 1) * a.K, *w1 = a.w + (long long)min(n0 + 1, a.N - 1) * a.K;
    for (int k0 = lane * 4; k0 - lane * 4 < a.K; k0 += 1024) {             // the weight's loads of four steps in flight
        f32x4 u0[4], u1[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const int k = k0 + 256 * h;
            u0[h] = load4<VEC>(w0 + k, a.K - k);
            u1[h] = load4<VEC>(w1 + k, a.K - k);
        }
#pragma unroll
        for (int m = 0; m < kOneRows; ++m) {
            if (m >= a.M) break;
            f32x4 xv[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) xv[h] = load4<VEC>(a.x + m * a.ldx + k0 + 256 * h, a.K - k0 - 256 * h);
#pragma unroll
            for (int h = 0; h < 4; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y[m][0] = fmaf(xv[h][e], u0[h][e], y[m][0]);
                    y[m][1] = fmaf(xv[h][e], u1[h][e], y[m][1]);
                }
        }
    }
    for (int m = 0; m < a.M; ++m) {
        low_row<T, VEC>(a, m, st[m]);
        if (a.t && blockIdx.x == 0) {
            __syncthreads();
            for (int j = threadIdx.x; j < a.r; j += 256) a.t[(long long)m * a.r + j] = st[m][j];
        }
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < kOneRows; ++m) {
        if (m >= a.M) break;
        const int l = a.ids[m];
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            const int n = n0 + o;
            float v = wave_sum(y[m][o]);
            float d = 0.f;
            if (l >= 0 && l < a.L && n < a.N && lane < a.r) d = st[m][lane] * up(a.b[((long long)l * a.N + n) * a.r + lane]);      // r <= 64: a rank per lane
            v += wave_sum(d);
            if (lane == 0 && n < a.N) {
                if (a.bias) v += up(a.bias[n]);
                down(a.y + (long long)m * a.N + n, l >= a.L ? nan32() : v);
            }
        }
    }
}

// sum of n values `stride` apart, eight loads in flight (a plain loop waits for every one: 16 splits took 7 us)
__device__ __forceinline__ float sum_strided(const float* p, int n, long long stride) {
    float v = 0.f;
    for (int k0 = 0; k0 < n; k0 += 8) {
        float q[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) q[k] = p[(long long)min(k0 + k, n - 1) * stride];
#pragma unroll
        for (int k = 0; k < 8; ++k) v += k0 + k < n ? q[k] : 0.f;
    }
    return v;
}
// sum_j low[j] w[j * stride], eight loads of each in flight
template <typename T> __device__ __forceinline__ float dot_strided(const float* low, const T* w, int r, long long stride) {
    float v = 0.f;
    for (int j0 = 0; j0 < r; j0 += 8) {
        float a[8];
        T b[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            a[k] = low[min(j0 + k, r - 1)];
            b[k] = w[(long long)min(j0 + k, r - 1) * stride];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (j0 + k < r) v = fmaf(a[k], up(b[k]), v);
    }
    return v;
}

// y = partial sums + bias + B_l t
template <typename T>
__global__ __launch_bounds__(64) void k_ad_join(const AdArgs<T> a) {
    const long long e = (long long)blockIdx.x * 64 + threadIdx.x, n_all = (long long)a.M * a.N;
    if (e >= n_all) return;
    const int m = (int)(e / a.N), n = (int)(e - (long long)m * a.N);
    const int l = a.ids[m];
    float v = sum_strided(a.partial + e, a.ksplit, n_all);
    if (a.bias) v += up(a.bias[n]);
    if (l >= a.L) v = nan32();
    else if (l >= 0) v += dot_strided(a.t + (long long)m * a.r, a.b + ((long long)l * a.N + n) * a.r, a.r, 1);
    down(a.y + e, v);
}

// ---------------------------------------------------------------------------------------------------
// gradients of the adapters: G[j][c] = sum over an adapter's rows of p[m][j] z[m][c], p (M, r) in 32 bits;  dA: p = u, z = x (or its 8-bit checkpoint);  dB^T: p = t, z = dy.
// A work-group owns (adapter, piece of <= 256 of its rows, 128 columns, 16 ranks); its waves take a part of the rows each, 4 rows per 16 x 16 x 4 MFMA step, and every lane
// eight columns, 8 i .. 8 i + 7 where z is aligned (one load of 8 to 32 bytes feeds eight MFMA tiles); they meet in LDS in a fixed order.  In bfloat16 z is exact in 16 bits (a
// checkpoint's value too), so p goes in as three parts of 8 bits
// and 32 rows take three 16 x 16 x 32 steps, a fifth of the matrix time.  More pieces than one: partial sums in the
// workspace, joined by k_ad_grad_join.  Tiles of 32 ranks (32 x 32 x 2) waste half the matrix work at the usual ranks of up to 16.
// ---------------------------------------------------------------------------------------------------
struct AdGrad {
    const float* p;                    // pitch ldp
    const void* z;                     // rows of pitch ldz, or the codes (M, C)
    const unsigned char* exps;         // with codes
    void* out;                         // (L, r, C), or (L, C, r) with trans
    float* part;                       // [pieces of adapters that have several][r][C]
    long long ldz, ldp;
    int C, Cp, trans, blocks;          // columns, columns that may be read; blocks: blocks of 128 columns x 16 ranks, columns first
};

// Eight elements of a row of z, as they lie in memory: consecutive ones (`load`), or, where the rows are not aligned, every sixteenth (`load_any`, in order over the
// lanes; a row of 1,230 in 32 bits, 462 rows, 40 adapters, consecutive: 47 us).  Past the last column there is no promise but that the memory is there (nothing of it is stored).
template <typename T, bool ACT8> struct Z8;
template <typename T> struct Z8<T, false> {
    typedef __attribute__((ext_vector_type(8))) T v8;
    v8 d;
    static __device__ __forceinline__ bool aligned(const AdGrad& g) { return g.ldz % (16 / sizeof(T)) == 0 && g.Cp % 8 == 0 && ((uintptr_t)g.z & 15) == 0; }
    __device__ __forceinline__ void load(const AdGrad& g, int m, int c) {
        const uint4* p = (const uint4*)((const T*)g.z + (long long)m * g.ldz + min(c, g.Cp - 8));
        uint4 h[sizeof(T) / 2];
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; ++k) h[k] = p[k];
        __builtin_memcpy(&d, h, sizeof(d));
    }
    __device__ __forceinline__ void load_any(const AdGrad& g, int m, int c) {
#pragma unroll
        for (int k = 0; k < 8; ++k) d[k] = ((const T*)g.z)[(long long)m * g.ldz + min(c + 16 * k, g.C - 1)];
    }
    __device__ __forceinline__ void keep(bool in) {
#pragma unroll
        for (int k = 0; k < 8; ++k) d[k] = in ? d[k] : (T)0;
    }
    __device__ __forceinline__ float get(int k) const { return up((T)d[k]); }
    __device__ __forceinline__ bf16_t half(int k) const { return d[k]; }   // bfloat16 alone
    static __device__ __forceinline__ float one(const AdGrad& g, int m, int c) { return up(((const T*)g.z)[(long long)m * g.ldz + c]); }
};
template <typename T> struct Z8<T, true> {
    unsigned int w[2], e[2];
    static __device__ __forceinline__ bool aligned(const AdGrad& g) { return g.C % 8 == 0 && ((uintptr_t)g.z & 7) == 0 && ((uintptr_t)g.exps & 7) == 0; }
    __device__ __forceinline__ void load(const AdGrad& g, int m, int c) {
        const int at = min(c, g.C - 8);
        const uint2 a = *(const uint2*)((const unsigned char*)g.z + (long long)m * g.C + at), b = *(const uint2*)(g.exps + (long long)(m >> 5) * g.C + at);
        w[0] = a.x; w[1] = a.y; e[0] = b.x; e[1] = b.y;
    }
    __device__ __forceinline__ void load_any(const AdGrad& g, int m, int c) {
        w[0] = w[1] = e[0] = e[1] = 0u;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int at = min(c + 16 * k, g.C - 1);
            w[k >> 2] |= (unsigned)((const unsigned char*)g.z)[(long long)m * g.C + at] << (8 * (k & 3));
            e[k >> 2] |= (unsigned)g.exps[(long long)(m >> 5) * g.C + at] << (8 * (k & 3));
        }
    }
    __device__ __forceinline__ void keep(bool in) {
        w[0] = in ? w[0] : 0u;
        w[1] = in ? w[1] : 0u;
    }
    __device__ __forceinline__ float get(int k) const {
        const int q = (int)(signed char)(w[k >> 2] >> (8 * (k & 3)));
        const float step = __uint_as_float((unsigned)max((int)((e[k >> 2] >> (8 * (k & 3))) & 0xffu) - 6, 0) << 23);
        return q == -128 ? nan32() : (float)q * step;
    }
    __device__ __forceinline__ bf16_t half(int k) const { return (bf16_t)(__float_as_uint(get(k)) >> 16); }      // exact: seven bits times a power of two
    static __device__ __forceinline__ float one(const AdGrad& g, int m, int c) {
        Z8<T, true> z;
        z.w[0] = ((const unsigned char*)g.z)[(long long)m * g.C + c];
        z.e[0] = g.exps[(long long)(m >> 5) * g.C + c];
        return z.get(0);
    }
};

constexpr int kGradLds = 4 * 32 * 64;                                     // floats
// T: type of z and of the gradients; ACT8: z is a checkpoint.  Four waves (4,096 rows, 2,048 -> 1,024, 16 adapters, bfloat16: 12.7 us; eight, of which a CU holds
// one work-group: 14.7, and 16.6 with z and p in 32 bits)
template <typename T, bool ACT8>
__device__ __forceinline__ void grad_piece(const AdGrad& g, int r, const int* rows, int n, int l, long long piece, bool whole, int block, float* red) {
    const int ncb = (g.C + 127) / 128, cb = block % ncb, j0 = block / ncb * 16;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
    if (n == 0) {                                                          // an adapter without rows has one piece: its part of the result is zero
        const int c0 = cb * 128, w = min(128, g.C - c0), nj = min(16, r - j0);
        for (int e = threadIdx.x; e < 128 * 16; e += 256) {
            const int jj = g.trans ? e & 15 : e >> 7, cc = g.trans ? e >> 4 : e & 127;      // along what lies next to each other
            if (jj < nj && cc < w) down((T*)g.out + (g.trans ? ((long long)l * g.C + c0 + cc) * r + j0 + jj : ((long long)l * r + j0 + jj) * g.C + c0 + cc), 0.f);
        }
        return;
    }
    const bool vec = Z8<T, ACT8>::aligned(g);
    const int c = cb * 128 + (vec ? 8 * i : i), cs = vec ? 1 : 16;         // a lane's columns: c, c + cs ..
    const int per = ((n + 3) / 4 + 3) & ~3, r0 = wave * per, r1 = min(r0 + per, n);
    const int j = min(j0 + i, r - 1);
    f32x4 acc[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    constexpr int U = 8;
    constexpr bool B16 = sizeof(T) == 2;
    auto place = [&](int s) { return B16 ? 8 * q + s : 4 * s + q; };       // of a lane's row s among the 32; bfloat16: the eight that its operand holds
    for (int rr = r0; rr < r1; rr += 4 * U) {
        Z8<T, ACT8> z[U];
        float pv[U];
        int m[U];
#pragma unroll
        for (int s = 0; s < U; ++s) m[s] = rows[min(rr + place(s), r1 - 1)];
        if (vec) {                                                         // every load is made, behind conditions each would be waited for before the next
#pragma unroll
            for (int s = 0; s < U; ++s) z[s].load(g, m[s], c);
        } else {
#pragma unroll
            for (int s = 0; s < U; ++s) z[s].load_any(g, m[s], c);
        }
#pragma unroll
        for (int s = 0; s < U; ++s) pv[s] = g.p[(long long)m[s] * g.ldp + j];
#pragma unroll
        for (int s = 0; s < U; ++s) {
            const bool in = rr + place(s) < r1;
            z[s].keep(in);                                                 // not an infinity of the last row times zero
            pv[s] = in && j0 + i < r ? pv[s] : 0.f;
        }
        if constexpr (B16) {
            u16x8 part[3];                                                 // smallest first
#pragma unroll
            for (int k = 2; k >= 0; --k)
#pragma unroll
                for (int s = 0; s < U; ++s) {
                    part[k][s] = to_bf16(pv[s]);
                    pv[s] = bf16_left(pv[s]);
                }
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                u16x8 v;
#pragma unroll
                for (int s = 0; s < U; ++s) v[s] = z[s].half(t);
#pragma unroll
                for (int k = 0; k < 3; ++k)
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, part[k]), __builtin_bit_cast(bf16x8, v), acc[t], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int s = 0; s < U; ++s)
#pragma unroll
                for (int t = 0; t < 8; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(pv[s], z[s].get(t), acc[t], 0, 0, 0);
        }
    }
    // element e of tile t: rank j0 + 4 q + e of column c + t cs
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[(wave * 32 + t * 4 + e) * 64 + lane] = acc[t][e];
    __syncthreads();
    auto total = [&](int t, int e) {
        const int at = (t * 4 + e) * 64 + lane;
        float v = red[at];
#pragma unroll
        for (int w = 1; w < 4; ++w) v += red[at + w * 32 * 64];
        if constexpr (B16) {                                           // an infinity of z times the parts of p may be a NaN, and a p near the largest float's first
            const int jj = j0 + 4 * q + e, cc = c + t * cs;            // part an infinity, where their own product is neither
            if (!finite(v) && jj < r && cc < g.C) {
                v = 0.f;
#pragma unroll 4
                for (int k = 0; k < n; ++k) v = fmaf(g.p[(long long)rows[k] * g.ldp + jj], Z8<T, ACT8>::one(g, rows[k], cc), v);
            }
        }
        return v;
    };
    if (whole && g.trans) {                                            // a wave: two columns, four ranks each
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
            const int t = 2 * wave + t2, jj = j0 + 4 * q;
            T* po = (T*)g.out + ((long long)l * g.C + c + t * cs) * r + jj;
            T h[4] __attribute__((aligned(16)));
#pragma unroll
            for (int e = 0; e < 4; ++e) down(h + e, total(t, e));
            if (c + t * cs < g.C) {
                if (r % 4 == 0 && ((uintptr_t)g.out & (4 * sizeof(T) - 1)) == 0) {
                    if (jj < r) {
                        if (sizeof(T) == 4) *(uint4*)po = *(const uint4*)h;
                        else *(uint2*)po = *(const uint2*)h;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (jj + e < r) po[e] = h[e];
                }
            }
        }
    } else {                                                           // a wave: rank j0 + 4 q + wave, eight columns
        const int e = wave, jj = j0 + 4 * q + e;
        float v[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) v[t] = total(t, e);
        if (jj < r) {
            if (!whole) {
                float* po = g.part + (piece * r + jj) * g.C + c;
#pragma unroll
                for (int t = 0; t < 8; ++t)
                    if (c + t * cs < g.C) po[t * cs] = v[t];
            } else {
                T* po = (T*)g.out + ((long long)l * r + jj) * g.C + c;
                T h[8] __attribute__((aligned(16)));
#pragma unroll
                for (int t = 0; t < 8; ++t) down(h + t, v[t]);
                if (vec && g.C % 8 == 0 && ((uintptr_t)g.out & 15) == 0) {
                    if (c < g.C) {
#pragma unroll
                        for (int k = 0; k < (int)sizeof(h) / 16; ++k) *((uint4*)po + k) = *((const uint4*)h + k);
                    }
                } else {
#pragma unroll
                    for (int t = 0; t < 8; ++t)
                        if (c + t * cs < g.C) po[t * cs] = h[t];
                }
            }
        }
    }
}

// rows of adapter l among the first M <= kFewRows ids, in order, into LDS; returns their number (256 threads)
__device__ __forceinline__ int rows_of(const int* ids, int M, int l, int* rows, int* cnt) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool mine = (int)threadIdx.x < M && ids[threadIdx.x] == l;
    const unsigned long long b = __ballot(mine);
    if (lane == 0) cnt[wave] = __popcll(b);
    __syncthreads();
    int base = 0;
    for (int w = 0; w < wave; ++w) base += cnt[w];
    if (mine) rows[base + __popcll(b & ((1ull << lane) - 1ull))] = threadIdx.x;
    const int n = cnt[0] + cnt[1] + cnt[2] + cnt[3];
    __syncthreads();
    return n;
}

// few rows, backward, first launch: dx's partial sums, u, dB
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void k_ad_few_back(const AdArgs<T> a, const AdGrad db, int tiles_o, int tiles_m) {
    __shared__ float red[kGradLds];
    __shared__ int rows[kFewRows], cnt[4];
    const int nb = a.dx ? tiles_o * a.ksplit * tiles_m : 0;
    int id = blockIdx.x;
    if (id < nb) {
        const int ot = id % tiles_o, rest = id / tiles_o;
        base_tile<T, false, VEC>(a, a.dy, a.N, a.K, a.N, ot, rest % a.ksplit, rest / a.ksplit, red);
        return;
    }
    id -= nb;
    if (id < a.M) {
        up_row<T>(a, id, red);
        return;
    }
    id -= a.M;
    const int l = id / db.blocks;
    const int n = rows_of(a.ids, a.M, l, rows, cnt);
    grad_piece<T, false>(db, a.r, rows, n, l, 0, true, id - l * db.blocks, red);
}

// second launch: dx = partial sums + A_l^T u, dA
template <typename T, bool ACT8>
__global__ __launch_bounds__(256) void k_ad_few_back2(const AdArgs<T> a, const AdGrad da, int join_wgs) {
    __shared__ float red[kGradLds];
    __shared__ int rows[kFewRows], cnt[4];
    int id = blockIdx.x;
    if (id < join_wgs) {
        const long long e = (long long)id * 256 + threadIdx.x, n_all = (long long)a.M * a.K;
        if (e >= n_all) return;
        const int m = (int)(e / a.K), k = (int)(e - (long long)m * a.K);
        const int l = a.ids[m];
        float v = sum_strided(a.partial + e, a.ksplit, n_all);
        if (l >= a.L) v = nan32();
        else if (l >= 0) v += dot_strided(a.u + (long long)m * a.r, a.a + (long long)l * a.r * a.K + k, a.r, a.K);
        down(a.dx + e, v);
        return;
    }
    id -= join_wgs;
    const int l = id / da.blocks;
    const int n = rows_of(a.ids, a.M, l, rows, cnt);
    grad_piece<T, ACT8>(da, a.r, rows, n, l, 0, true, id - l * da.blocks, red);
}

// ---------------------------------------------------------------------------------------------------
// many rows
// ---------------------------------------------------------------------------------------------------
// First launch: the rows' order by adapter, and the copies of operands that the tiles below need in another layout.
//   order: the rows by adapter (those without one last), each adapter's in their own order; key: their ids in that order;  seg[l]: where adapter l begins (seg[L]:
//     rows without, seg[L + 1] = M).  Work-group l counts the rows in front of its own adapter's, then places these: its sixteen waves take a range of the rows
//     each, nothing is shared between work-groups.
//   Copies: dst[b][r][c] (pitch ldd, columns past C zero) = src[b][r][c] or, transposed, src[b][c][r], through LDS.
struct AdCopy {
    const void* src;
    void* dst;
    long long lds_, ldd, sbs, dbs;         // row pitches and batch strides of source and destination
    int R, C, Cp, trans, tiles, tr, tc;     // destination rows, columns, padded columns; tiles = batches * tr * tc
};
struct AdPrep {
    const int* ids;
    int *order, *key, *seg;
    int M, L, ncopy;
    AdCopy copy[3];
};

constexpr int kPrep = 1024;                // threads: the plan of some thousand rows is two rounds of loads, not thirty
template <typename T>
__global__ __launch_bounds__(kPrep) void k_ad_prep(const AdPrep a) {
    __shared__ T s[64][257];
    __shared__ int cnt[32];
    int id = blockIdx.x;
    if (id <= a.L) {
        const int l = id, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int per = ((a.M + 15) / 16 + 63) / 64 * 64, m0 = wave * per, m1 = min(m0 + per, a.M);
        constexpr int U = 8;
        int less = 0, mine = 0;
        for (int mb = m0; mb < m1; mb += 64 * U) {
            int v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = a.ids[min(mb + 64 * u + lane, m1 - 1)];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool in = mb + 64 * u + lane < m1;
                const int key = (v[u] < 0 || v[u] >= a.L) ? a.L : v[u];
                less += in && key < l;
                mine += in && key == l;
            }
        }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) {
            less += __shfl_xor(less, d);
            mine += __shfl_xor(mine, d);
        }
        if (lane == 0) { cnt[wave] = less; cnt[16 + wave] = mine; }
        __syncthreads();
        int at = 0;
        for (int w = 0; w < 16; ++w) at += cnt[w];
        if (threadIdx.x == 0) {
            a.seg[l] = at;
            if (l == a.L) a.seg[l + 1] = a.M;
        }
        for (int w = 0; w < wave; ++w) at += cnt[16 + w];
        for (int mb = m0; mb < m1; mb += 64 * U) {
            int v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = a.ids[min(mb + 64 * u + lane, m1 - 1)];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int m = mb + 64 * u + lane, key = (v[u] < 0 || v[u] >= a.L) ? a.L : v[u];
                const bool in = m < m1 && key == l;
                const unsigned long long b = __ballot(in);
                if (in) {
                    const int p = at + __popcll(b & ((1ull << lane) - 1ull));
                    a.order[p] = m;
                    a.key[p] = v[u];
                }
                at += __popcll(b);
            }
        }
        return;
    }
    id -= a.L + 1;
    int k = 0;
    while (k < a.ncopy && id >= a.copy[k].tiles) id -= a.copy[k++].tiles;
    if (k >= a.ncopy) return;
    const AdCopy& c = a.copy[k];
    const int bt = id / (c.tr * c.tc), rest = id - bt * c.tr * c.tc, ir = rest / c.tc, ic = rest - ir * c.tc;
    const T* src = (const T*)c.src + bt * c.sbs;
    T* dst = (T*)c.dst + bt * c.dbs;
    const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
    T v[16];                                                                // sixteen elements of a thread in flight: no load behind a condition
    if (!c.trans) {                                                         // 256 rows x 64 columns
        const int r0 = ir * 256 + y, cc = ic * 64 + x;
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = src[(long long)min(r0 + 16 * j, c.R - 1) * c.lds_ + min(cc, c.C - 1)];
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (r0 + 16 * j < c.R && cc < c.Cp) dst[(long long)(r0 + 16 * j) * c.ldd + cc] = cc < c.C ? v[j] : (T)0;
        return;
    }
    const int r0 = ir * 64, c0 = ic * 256;                                  // 64 rows x 256 columns of the destination
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = src[(long long)min(c0 + y + 16 * j, c.C - 1) * c.lds_ + min(r0 + x, c.R - 1)];
#pragma unroll
    for (int j = 0; j < 16; ++j) s[x][y + 16 * j] = c0 + y + 16 * j < c.C ? v[j] : (T)0;
    __syncthreads();
    const int xc = threadIdx.x & 255, yr = threadIdx.x >> 8;
#pragma unroll
    for (int j = 0; j < 16; ++j)
        if (r0 + yr + 4 * j < c.R && c0 + xc < c.Cp) dst[(long long)(r0 + yr + 4 * j) * c.ldd + c0 + xc] = s[yr + 4 * j][xc];
}

// Whether any of the 16 bytes of u and v holds an exponent of all ones: an infinity or a NaN.  ONES: the exponents' bits in a word, LOW: their lowest ones, which added to
// an exponent of all ones carry into the sign's place and no further.
template <unsigned ONES, unsigned LOW, typename F> __device__ __forceinline__ bool odd16(F u, F v) {
    const uint4 a = __builtin_bit_cast(uint4, u), b = __builtin_bit_cast(uint4, v);
    const unsigned s = ((a.x & ONES) + LOW) | ((a.y & ONES) + LOW) | ((a.z & ONES) + LOW) | ((a.w & ONES) + LOW) | ((b.x & ONES) + LOW) | ((b.y & ONES) + LOW) |
                       ((b.z & ONES) + LOW) | ((b.w & ONES) + LOW);
    return (s & (ONES + LOW)) != 0u;
}
// What the two types differ in.  A fragment is 16 bytes of a row in both.
template <typename T> struct Mma;
template <> struct Mma<float> {
    static constexpr int E = 4, HL = 1, STEPS = 4;                          // elements of 16 bytes; columns of the reduction per rank; MFMA steps of 32 bytes
    typedef f32x4 frag;
    // 32 bytes of both operands' rows: 4 steps of the 32 x 32 x 2 MFMA, lane half q holds elements 4 q .. 4 q + 3
    static __device__ __forceinline__ f32x16 mma32(frag a, frag b, f32x16 c, int e) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0); }
    // 64 bytes: 4 steps of the 16 x 16 x 4 MFMA, lane quarter holds its 16 bytes
    static __device__ __forceinline__ f32x4 mma16(frag a, frag b, f32x4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ float part(float v, int) { return v; }
    static __device__ __forceinline__ bool any_odd(frag u, frag v) { return odd16<0x7f800000u, 0x00800000u>(u, v); }
};
template <> struct Mma<bf16_t> {
    static constexpr int E = 8, HL = 2, STEPS = 1;
    typedef u16x8 frag;
    static __device__ __forceinline__ f32x16 mma32(frag a, frag b, f32x16 c, int) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mma16(frag a, frag b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ bf16_t part(float v, int lo) { return to_bf16(lo ? bf16_left(v) : v); }      // high half, and what it leaves
    static __device__ __forceinline__ bool any_odd(frag u, frag v) { return odd16<0x7f807f80u, 0x00800080u>(u, v); }
};

// Piece z of the order: segment l (of n) has max(MIN, ceil(rows / R)) pieces of R rows, one behind the other.  All lanes of a wave return the same: the segment, how many
// pieces it has, this one's first place and its end; l = n: no such piece.  PART: and `part`, its number among the pieces of segments that have several.
template <int R, int MIN, bool PART>
__device__ __forceinline__ void find_piece(const int* seg, int n, int z, int& l, int& np, int& at, int& end, int& part) {
    const int lane = threadIdx.x & 63;
    int base = 0, pbase = 0;
    for (int l0 = 0; l0 < n; l0 += 64) {
        const int li = l0 + lane;
        const int s0 = seg[min(li, n)], s1 = seg[min(li + 1, n)], rows = s1 - s0;
        const int mine = li < n ? max(MIN, (rows + R - 1) / R) : 0;
        int incl = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(incl, d);
            if (lane >= d) incl += o;
        }
        const unsigned long long over = __ballot(base + incl > z);
        const int k = over ? __ffsll((long long)over) - 1 : 64;              // the piece's segment in these 64
        if (PART) {
            int before = lane < k && mine > 1 ? mine : 0;
#pragma unroll
            for (int d = 32; d >= 1; d >>= 1) before += __shfl_xor(before, d);
            pbase += before;
        }
        if (over) {
            l = l0 + k;
            np = __shfl(mine, k);
            const int nth = z - (base + __shfl(incl, k) - np);
            at = __shfl(s0, k) + nth * R;
            end = min(at + R, __shfl(s1, k));
            part = pbase + nth;
            return;
        }
        base += __shfl(incl, 63);
    }
    l = n;
    np = at = end = part = 0;
}

typedef __attribute__((address_space(3))) void* ad_lds_t;
typedef const __attribute__((address_space(1))) void* ad_glb_t;
// one LDS-DMA request: lane l's 16 bytes at g land at dst + 16 l
static __device__ __forceinline__ void ad_dma16(const char* g, void* dst) { __builtin_amdgcn_global_load_lds((ad_glb_t)g, (ad_lds_t)dst, 16, 0, 0); }
#define HMF_AD_VMCNT(n) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory")

// low[m][j] = s_l sum_c in[m][c] v[l][j][c]:  t (in = x, v = A) and u (in = dy, v = B^T).  A work-group owns up to 16 rows of one adapter; its sixteen waves take a
// part of the reduction each (16 rows x 16 ranks per MFMA) and meet in LDS in a fixed order.  Operands go through LDS by DMA although nothing is used twice: the MFMA's
// operand layout has 16 rows in 16 neighbouring lanes, and a load of 16 bytes per lane in that layout takes the address unit 64 cycles instead of 16 (4,096 rows
// of 2,048 in bfloat16: 11.6 us, and twice that in 32 bits).  C: whole chunks.
struct AdLow {
    const void *in, *v;
    const float* scale;
    const int *order, *key, *seg;
    float *low, *t;                         // (M, rp), rp = r rounded up to 4, zeros behind r; t: a copy (M, r) for the caller, or null
    long long ldin, ldv;                    // row pitches; v: (L r) rows
    int M, C, r, rp, L;
};
template <typename T>
__global__ __launch_bounds__(1024) void k_ad_low(const AdLow a) {
    typedef Mma<T> X;
    typedef typename X::frag frag;
    constexpr int U = 4;                                                    // groups of 64 bytes in flight per wave and operand
    __shared__ __attribute__((aligned(16))) char smem[16 * 2 * U * 1024];
    float* red = (float*)smem;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, q = lane >> 4;
    int ad, np, first, end, part;
    find_piece<16, 0, false>(a.seg, a.L + 1, blockIdx.x, ad, np, first, end, part);      // the rows without an adapter are the last segment
    if (ad > a.L) return;
    ad = __builtin_amdgcn_readfirstlane(ad);
    const bool live = first + i < end;
    const int p = min(first + i, end - 1), m = a.order[p];                         // places past the segment's last row repeat it and write nothing
    if (ad == a.L) {                                                        // no adapter: zero; an id that no adapter has: NaN
        if (live && q == 0)
            for (int j = wave; j < a.rp; j += 16) {
                const float v = a.key[p] < 0 ? 0.f : nan32();
                a.low[(long long)m * a.rp + j] = v;
                if (a.t && j < a.r) a.t[(long long)m * a.r + j] = v;
            }
        return;
    }
    const float s = a.scale[ad];
    const int ng = a.C / (4 * X::E), per = (ng + 15) / 16, g0 = wave * per, g1 = min(g0 + per, ng);         // groups of 64 bytes
    // DMA: lane brings piece (lane & 3) ^ s of row lane >> 2, s = (row >> 2) & 3; fragment (i, q) lies in slot q ^ s of row i
    const int dr = lane >> 2, dc = (lane & 3) ^ ((dr >> 2) & 3);
    const char* xr = (const char*)((const T*)a.in + (long long)__shfl(m, dr) * a.ldin) + 16 * dc;
    char* mine = smem + wave * 2 * U * 1024;
    const char* fr = mine + i * 64 + ((q ^ ((i >> 2) & 3)) * 16);
    for (int j0 = 0; j0 < a.r; j0 += 16) {
        const char* vr = (const char*)((const T*)a.v + ((long long)ad * a.r + min(j0 + dr, a.r - 1)) * a.ldv) + 16 * dc;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int g = g0; g < g1; g += U) {
#pragma unroll
            for (int h = 0; h < U; ++h)
                if (g + h < g1) {                                           // wave-uniform
                    ad_dma16(xr + (long long)(g + h) * 64, mine + h * 1024);
                    ad_dma16(vr + (long long)(g + h) * 64, mine + (U + h) * 1024);
                }
            HMF_AD_VMCNT(0);
#pragma unroll
            for (int h = 0; h < U; ++h)
                if (g + h < g1) acc = X::mma16(*(const frag*)(fr + (U + h) * 1024), *(const frag*)(fr + h * 1024), acc);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");               // read before the next round overwrites
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 4; ++e) red[wave * 256 + e * 64 + lane] = acc[e];
        __syncthreads();
        if (wave < 4) {                                                     // wave w finishes element w: rank j0 + 4 q + w of row i
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < 16; ++w) v += red[w * 256 + tid];
            const int j = j0 + 4 * q + wave;
            if (live && j < a.rp) {
                a.low[(long long)m * a.rp + j] = j < a.r ? s * v : 0.f;
                if (a.t && j < a.r) a.t[(long long)m * a.r + j] = s * v;
            }
        }
        __syncthreads();
    }
}

// out[m][o] = sum_c in[m][c] w[o][c] (+ bias[o]) + sum_j low[m][j] v[l][o][j]: forward in = x, w = W, low = t, v = B; backward in = dy, w = W^T, low = u, v = A^T.
template <typename T> struct AdGemm {
    const T *in, *w, *bias, *v;
    const float* low;
    const int *order, *key;
    T* out;
    long long ldin, ldw, vl, vo, vj;        // pitches; strides of v
    int M, C, O, r, rp, L, tiles_o;         // C: whole chunks; rp: low's pitch
    float* partial;                         // with several splits of the reduction (gridDim.y): [split][M][O]
    int per;                                // chunks of a split
};

// BT x BT tile, 4 waves of (BT / 2) x (BT / 2); a ring of 4 LDS stages of one chunk (RB bytes of every row of both operands) filled by LDS-DMA three chunks ahead:
// with one chunk ahead through registers a chunk of the 128-tile took 2.2 us, the latency of its loads; so 0.46 us (32 KB read from and 16 KB written to LDS
// for 512 cycles of MFMA).  The 16-byte slot c of row r lies at slot c ^ swizzle(r) (the DMA writes in lane order, so the source address is permuted): a
// fragment read hits every bank once.  RB = 128 (whole lines, one work-group per CU at BT = 128) where a CU has one tile; RB = 64 (half the LDS: two work-groups
// per CU, one's start and end under the other's products) where it has more.
// After the shared weight's chunks come the adapters': 16-byte piece P of a row belongs to the tile's adapter list[P / pp] and holds E of its ranks (bfloat16: the
// high halves of all ranks, then the low ones).  The rows of other adapters hold zeros there,
// and a zero times an infinity or a NaN of a weight would reach them: such weights are staged as zeros and added to their own rows at the end, and so are values of low
// that are not finite or, in bfloat16, become infinite there (from 3.39e38 on).
template <typename T, int BT, int RB>
__global__ __launch_bounds__(256) void k_ad_gemm(const AdGemm<T> a) {
    typedef Mma<T> X;
    typedef typename X::frag frag;
    constexpr int E = X::E, S = 4, PR = RB / 16, G = RB / 32;               // 16-byte pieces and MFMA groups of a row's chunk
    constexpr int ND = BT * RB / 4096;                                      // DMA requests of a wave, operand and chunk (1 KB each)
    constexpr int NT = BT / 64;                                             // MFMA tiles of a wave, each way
    constexpr int NS = BT * PR / 256;                                       // pieces of a thread, operand and chunk
    constexpr int OP = BT * RB, STAGE = 2 * OP;                             // bytes
    auto swizzle = [](int row) { return RB == 128 ? (row >> 1) & 7 : (row >> 2) & 3; };
    __shared__ __attribute__((aligned(16))) char smem[S * STAGE + (3 * BT + 4) * 4];      // one object: a second one makes hipcc wait for the DMA before every read
    int* rowid = (int*)(smem + S * STAGE);
    int *slot = rowid + BT, *list = slot + BT, *nlist = list + BT, *odd = nlist + 2;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 31, q = lane >> 5;
    // XCD x (work-groups go round robin) gets a contiguous run of tiles, the tiles of one row panel next to each other
    const int all = gridDim.x, t8 = all >> 3, id = (all & 7) ? blockIdx.x : (blockIdx.x & 7) * t8 + (blockIdx.x >> 3);
    const int ot = id % a.tiles_o, mt = id / a.tiles_o;
    const int o0 = ot * BT, p0 = mt * BT;
    // the tile's rows and its distinct adapters, in order
    if (tid == 0) *odd = 0;
    bool first = false;
    int l = -1, before = 0;
    if (tid < BT) {
        const int p = min(p0 + tid, a.M - 1), prev = max(p - 1, 0);
        const int m = a.order[p], id = a.key[p], idp = a.key[prev];
        const bool in = p0 + tid < a.M;
        l = (in && id >= 0) ? (id < a.L ? id : -2) : -1;
        first = l >= 0 && (tid == 0 || l != idp);
        const unsigned long long b = __ballot(first);
        before = __popcll(b & ((2ull << lane) - 1ull));                     // first rows of this wave up to and including this one
        rowid[tid] = in ? m : -1 - m;                                       // places past the last row read it and store nothing
        if (lane == 0) nlist[wave] = __popcll(b);
    }
    __syncthreads();
    const int n0 = nlist[0], nad = n0 + (BT > 64 ? nlist[1] : 0);
    if (tid < BT) {                                                         // a second wave's leading rows may continue the first one's last adapter: place n0 - 1
        const int at = before - 1 + (wave > 0 ? n0 : 0);
        slot[tid] = l >= 0 ? at : l;                                        // -1: no adapter, -2: an id that no adapter has
        if (first) list[at] = l;
    }
    __syncthreads();
    // chunks of this split; 16-byte pieces of an adapter's ranks, of an adapter, of all (the first split's), and their chunks
    const int cfirst = blockIdx.y * a.per, kc = min(a.per, a.C * (int)sizeof(T) / RB - cfirst);
    const int pr = (a.r + E - 1) / E, pp = pr * X::HL, ext = blockIdx.y == 0 ? nad * pp : 0, ne = (ext + PR - 1) / PR;

    // DMA sources: request d of wave w brings rows 64 / PR (w ND + d) ..; rows that are not there read a valid one, whose results are not stored
    const char *gw[ND], *gx[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        const int row = (wave * ND + d) * (64 / PR) + lane / PR, c = (lane % PR) ^ swizzle(row);
        gw[d] = (const char*)(a.w + (long long)min(o0 + row, a.O - 1) * a.ldw) + 16 * c + (long long)cfirst * RB;
        const int m = rowid[row];
        gx[d] = (const char*)(a.in + (long long)(m < 0 ? -1 - m : m) * a.ldin) + 16 * c + (long long)cfirst * RB;
    }
    auto issue = [&](int c, int lo, int hi) {
        char* st = smem + (c & (S - 1)) * STAGE + wave * ND * 1024;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            if (d < lo || d >= hi) continue;
            ad_dma16(gw[d] + (long long)c * RB, st + d * 1024);
            ad_dma16(gx[d] + (long long)c * RB, st + OP + d * 1024);
        }
    };
    // The adapters' chunks go through registers: raw values first, so that the first of them are loaded under the main loop.  A thread's pieces lie in the same column.
    // Every load is made, from a place that is there, and what does not belong is zeroed at the stash: behind a condition of its own each would be waited for before
    // the next (4,096 rows, 2,048 -> 1,024, bfloat16, with the conversions and the bias's loads as straight: 37 -> 25 us).
    frag ew[NS];
    f32x4 ex[NS][E / 4];
    const bool vec_v = a.vj == 1 && a.r % E == 0 && ((uintptr_t)a.v & 15) == 0;
    int elo = 0, ead = 0, ej0 = 0;                                          // of the fetched pieces: which half, whose, first rank
    bool elive = false;
    auto fetch = [&](int c) {
        const int P = c * PR + tid % PR, ad = min(P, ext - 1) / pp, rem = min(P, ext - 1) - ad * pp;
        elo = rem >= pr;
        ej0 = (elo ? rem - pr : rem) * E;
        ead = ad;
        elive = P < ext;
        const T *vb = a.v + (long long)list[ad] * a.vl, *pv[NS];
        const float* pl[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int row = (tid + 256 * s) / PR;
            pv[s] = vb + (long long)min(o0 + row, a.O - 1) * a.vo;
            pl[s] = a.low + (long long)max(rowid[row], 0) * a.rp;
        }
        if (vec_v) {
#pragma unroll
            for (int s = 0; s < NS; ++s) ew[s] = *(const frag*)(pv[s] + ej0);
        } else {
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int k = 0; k < E; ++k) ew[s][k] = pv[s][min(ej0 + k, a.r - 1) * a.vj];
        }
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int k = 0; k < E; k += 4) ex[s][k / 4] = *(const f32x4*)(pl[s] + min(ej0 + k, a.rp - 4));
    };
    auto stash = [&](int st) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int e = tid + 256 * s, row = e / PR, at = row * RB + ((e % PR) ^ swizzle(row)) * 16;
            const bool mine = elive && slot[row] == ead, out = elive && o0 + row < a.O;
            frag zw, zx;
#pragma unroll
            for (int k = 0; k < E; ++k) {
                zw[k] = out && ej0 + k < a.r ? ew[s][k] : (T)0;
                zx[k] = X::part(mine && ej0 + k < a.r ? ex[s][k / 4][k & 3] : 0.f, elo);
            }
            if (X::any_odd(zw, zx)) {
                *odd = 1;
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    if (!finite(zw[k])) zw[k] = 0;
                    if (!finite(zx[k])) zx[k] = 0;
                }
            }
            *(frag*)(smem + st * STAGE + at) = zw;
            *(frag*)(smem + st * STAGE + OP + at) = zx;
        }
    };
    f32x16 acc[NT][NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int v = 0; v < NT; ++v)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[t][v][e] = 0.f;
    const int wo = (wave & 1) * (BT / 2), wm = (wave >> 1) * (BT / 2);
    const char *pw = smem + (wo + i) * RB, *px = smem + OP + (wm + i) * RB;
    int go[G];
#pragma unroll
    for (int g = 0; g < G; ++g) go[g] = ((2 * g + q) ^ swizzle(i)) * 16;
    frag fw[2][NT], fx[2][NT];
    auto frags = [&](int st, int g) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            fw[g & 1][t] = *(const frag*)(pw + st * STAGE + go[g] + t * 32 * RB);
            fx[g & 1][t] = *(const frag*)(px + st * STAGE + go[g] + t * 32 * RB);
        }
    };
    auto mma = [&](int g) {                                                 // step by step over the tiles: the next MFMA is never the one that waits for the last
#pragma unroll
        for (int e = 0; e < X::STEPS; ++e)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int v = 0; v < NT; ++v) acc[t][v] = X::mma32(fw[g & 1][t], fx[g & 1][v], acc[t][v], e);
    };
#pragma unroll
    for (int c = 0; c < S - 1; ++c)
        if (c < kc) issue(c, 0, ND);
    if (ne > 0) fetch(0);                                                   // behind the first requests: the counts waited for below are then only stricter than they say
    // One chunk: its own fragments group by group, each read under the MFMAs of the group before; chunk c + 1 is there too (at most the one behind it is on its way),
    // so the next chunk's first fragments are read under this one's last MFMAs and the matrix pipe does not drain at the barrier.
    auto iteration = [&](int c, auto MORE) {
        constexpr bool more = decltype(MORE)::value;
        if (more) HMF_AD_VMCNT(2 * ND);
        else HMF_AD_VMCNT(0);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int st = c & (S - 1);
        constexpr int nm = NT * NT * X::STEPS;
        auto group = [&](auto index) {
            constexpr int g = decltype(index)::value;
            if (g + 1 < G) frags(st, g + 1);
            else if (more || c + 1 < kc) frags((c + 1) & (S - 1), 0);
            mma(g);
            if (more && g < ND) issue(c + S - 1, g, g + 1);                 // into the stage that everybody has read (chunk c - 1)
            // order: an MFMA on the fragments at hand, the next fragments' reads, the DMA requests, the other MFMAs (the compiler waits for all reads at once:
            // reads issued in front of the first MFMA would be waited for there)
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * NT, 0);
            if (more && g < ND) __builtin_amdgcn_sched_group_barrier(0x010, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, nm - 1, 0);
        };
        group(std::integral_constant<int, 0>{});
        group(std::integral_constant<int, 1>{});
        if constexpr (G == 4) {
            group(std::integral_constant<int, 2>{});
            group(std::integral_constant<int, 3>{});
        }
    };
    if (kc >= S - 1) HMF_AD_VMCNT(2 * 2 * ND);                              // the first chunk
    else HMF_AD_VMCNT(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    frags(0, 0);
    int c = 0;
    for (; c + S - 1 < kc; ++c) iteration(c, std::true_type{});
    for (; c < kc; ++c) iteration(c, std::false_type{});
    auto compute = [&](int st) {
        frags(st, 0);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            if (g + 1 < G) frags(st, g + 1);
            mma(g);
        }
    };
    for (int e = 0; e < ne; ++e) {
        __syncthreads();
        stash(0);
        __syncthreads();
        if (e + 1 < ne) fetch(e + 1);
        compute(0);
    }
    __syncthreads();
    // Epilogue through LDS: lane (m = column i) holds outputs 8 (e >> 2) + 4 q + (e & 3); every wave turns its own tile round and stores 16 bytes per lane, whole rows of
    // BT / 2 outputs.
    const bool any_odd = *odd != 0;
    constexpr int H = BT / 2, PF = H + 4;                                   // outputs of a wave's rows, pitch in floats
    static_assert(4 * 32 * PF * 4 <= S * STAGE, "the turned tiles lie in the ring");
    float* tw = (float*)smem + wave * 32 * PF;
    constexpr int LPR = H / E, RPI = 64 / LPR;                              // lanes of a row, rows of an instruction
    const int oc = (lane % LPR) * E, o = o0 + wo + oc;
    const bool vec = a.O % E == 0 && ((uintptr_t)a.out & 15) == 0;
    float bv[E];
#pragma unroll
    for (int k = 0; k < E; ++k) bv[k] = 0.f;
    if (a.bias && !a.partial) {                                             // from places that are there: behind conditions each is waited for
        T bt[E];
#pragma unroll
        for (int k = 0; k < E; ++k) bt[k] = a.bias[min(o + k, a.O - 1)];
#pragma unroll
        for (int k = 0; k < E; ++k) bv[k] = up(bt[k]);
    }
#pragma unroll
    for (int v = 0; v < NT; ++v) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4)
                *(f32x4*)(tw + i * PF + 32 * t + 8 * e4 + 4 * q) = f32x4{acc[t][v][4 * e4], acc[t][v][4 * e4 + 1], acc[t][v][4 * e4 + 2], acc[t][v][4 * e4 + 3]};
#pragma unroll
        for (int s = 0; s < 32 / RPI; ++s) {
            const int row = s * RPI + lane / LPR, at = wm + 32 * v + row, m = rowid[at];
            float z[E];
#pragma unroll
            for (int k = 0; k < E; k += 4) {
                const f32x4 u = *(const f32x4*)(tw + row * PF + oc + k);
#pragma unroll
                for (int e = 0; e < 4; ++e) z[k + e] = u[e] + bv[k + e];
            }
            if (m < 0 || o >= a.O) continue;
            const int sl = slot[at];
            if (sl == -2 || any_odd) {
                const int id = sl >= 0 ? list[sl] : -1;
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    if (sl == -2) z[k] = nan32();
                    else if (id >= 0 && o + k < a.O)
                        for (int j = 0; j < a.r; ++j) {
                            const T vv = a.v[id * a.vl + (o + k) * a.vo + j * a.vj];
                            const float lv = a.low[(long long)m * a.rp + j];
                            if (!finite(vv) || !finite(X::part(lv, 0))) z[k] = fmaf(lv, up(vv), z[k]);
                        }
                }
            }
            if (a.partial) {
                float* pp_ = a.partial + ((long long)blockIdx.y * a.M + m) * a.O + o;
#pragma unroll
                for (int k = 0; k < E; ++k)
                    if (o + k < a.O) pp_[k] = z[k];
                continue;
            }
            T h[E] __attribute__((aligned(16)));
#pragma unroll
            for (int k = 0; k < E; ++k) down(h + k, z[k]);
            T* po = a.out + (long long)m * a.O + o;
            if (vec) *(uint4*)po = *(const uint4*)h;
            else
#pragma unroll
                for (int k = 0; k < E; ++k)
                    if (o + k < a.O) po[k] = h[k];
        }
    }
}

// out = the splits' sums, in order, + bias
template <typename T>
__global__ __launch_bounds__(256) void k_ad_sum(const float* __restrict__ partial, int splits, const T* __restrict__ bias, T* __restrict__ out, long long n, int O) {
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long long)gridDim.x * 256) {
        float v = partial[e];
#pragma unroll 4
        for (int k = 1; k < splits; ++k) v += partial[(long long)k * n + e];
        if (bias) v += up(bias[e % O]);
        down(out + e, v);
    }
}

template <typename T, bool ACT8>
__global__ __launch_bounds__(256) void k_ad_grads(const AdGrad da, const AdGrad db, const int* __restrict__ order, const int* __restrict__ seg, int r, int L) {
    __shared__ float red[kGradLds];
    __shared__ int rows[kFewRows];
    int l, np, s0, end, part;
    find_piece<kFewRows, 1, true>(seg, L, blockIdx.y, l, np, s0, end, part);
    if (l >= L) return;
    const int n = end - s0;
    if ((int)threadIdx.x < n) rows[threadIdx.x] = order[s0 + threadIdx.x];
    __syncthreads();
    const int cb = blockIdx.x;
    if (cb < da.blocks) grad_piece<T, ACT8>(da, r, rows, n, l, part, np == 1, cb, red);
    else grad_piece<T, false>(db, r, rows, n, l, part, np == 1, cb - da.blocks, red);
}

// sums of the adapters that had several pieces, in the pieces' order; a column of work-groups per adapter, gone at once where there is nothing to add
template <typename T>
__global__ __launch_bounds__(256) void k_ad_grad_join(const AdGrad da, const AdGrad db, const int* __restrict__ seg, int r, int L) {
    const int l = blockIdx.y, mine = seg[l + 1] - seg[l];
    if (mine <= kFewRows) return;
    const int lane = threadIdx.x & 63, np = (mine + kFewRows - 1) / kFewRows;
    int first = 0;                                                         // pieces in front of this adapter's, of adapters that have several
    for (int l0 = 0; l0 < l; l0 += 64) {
        const int li = l0 + lane, rows = li < l ? seg[li + 1] - seg[li] : 0;
        int v = rows > kFewRows ? (rows + kFewRows - 1) / kFewRows : 0;
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
        first += v;
    }
    const long long na = (long long)r * da.C, n = na + (long long)r * db.C;
    for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < n; at += (long long)gridDim.x * 256) {
        const AdGrad& g = at < na ? da : db;
        const long long e = at < na ? at : at - na;
        const float v = sum_strided(g.part + (long long)first * r * g.C + e, np, (long long)r * g.C);
        const int j = (int)(e / g.C), c = (int)(e - (long long)j * g.C);
        if (g.trans) down((T*)g.out + ((long long)l * g.C + c) * r + j, v);
        else down((T*)g.out + ((long long)l * r + j) * g.C + c, v);
    }
}

// ---------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------
static inline bool off16(const void* p) { return ((uintptr_t)p & 15) != 0; }
static inline size_t al(size_t v) { return align_up(v, 256); }
static inline int blocks_of(long long n, int per) { return (int)((n + per - 1) / per); }

// work-groups of a reduction: enough of them for two per CU, at least 32 elements for each of the four waves
static void few_split(int M, int O, int Cn, int* ksplit, int* kw) {
    const int tiles = blocks_of(O, 32) * blocks_of(M, 32);
    const int most = std::max(1, blocks_of(Cn, 128));
    const int ks = std::max(1, std::min(most, 512 / std::max(1, tiles)));
    *kw = (blocks_of(Cn, 4 * ks) + 31) / 32 * 32;
    *ksplit = blocks_of(Cn, 4 * *kw);
}

// Tiles of 128 where they fill three quarters of the CUs, else of 64; where those leave CUs idle too, the reduction is split until two work-groups go on each CU, but
// not under 8 chunks in 32 bits (512 rows, 2,048 -> 1,024, 128 tiles: 42 us unsplit, 27 us and 4 us for the sum in four) and 32 in bfloat16, whose chunk takes an
// eighth of the matrix time (15 us unsplit, 14 + 4 us in two).  Chunks of 64 bytes (k_ad_gemm's RB) where a CU has several tiles and their rows are short, up to
// 2,048 bytes (3,000 rows, 1,024 -> 2,048, 1.5 tiles a CU, bfloat16: 26.7 us, 30.2 in chunks of 128; 8,192 rows, 2,048 -> 2,048: 82 and 77 us).
static void gemm_shape(int M, int O, int Cp, size_t z, int* bt, int* rb, int* splits, int* per) {
    const long long big = (long long)blocks_of(M, 128) * blocks_of(O, 128);
    *bt = big >= 192 ? 128 : 64;
    *rb = big > 256 && z == 2 && Cp * z <= 2048 ? 64 : 128;
    const int kc = (int)(Cp * z / *rb), tiles = blocks_of(M, *bt) * blocks_of(O, *bt);
    const int want = tiles >= 256 || *bt == 128 ? 1 : std::max(1, std::min(kc / (z == 4 ? 8 : 32), 512 / tiles));
    *per = blocks_of(kc, want);
    *splits = blocks_of(kc, *per);
}
static size_t gemm_partial(int M, int O, int Cp, size_t z) {
    int bt, rb, splits, per;
    gemm_shape(M, O, Cp, z, &bt, &rb, &splits, &per);
    return splits > 1 ? (size_t)splits * M * O * 4 : 0;
}
// the many-row form's rows: whole chunks of 128 bytes, 16-byte aligned
static inline int padded(int C, size_t z) { const int bk = (int)(128 / z); return (C + bk - 1) / bk * bk; }
static inline int rank_pitch(int r) { return (r + 3) & ~3; }
// how the forward's operands lie: which of them the many-row form has to copy into whole chunks of aligned rows, and whether the few-row forms can read four elements at a
// time (load4's VEC)
struct FwdLayout { bool x, w, a, vec; };
constexpr FwdLayout kAnyLayout{true, true, true, false};
static FwdLayout fwd_layout(const void* x, long long ldx, const void* w, const void* a, int K, size_t z) {
    const bool odd = K != padded(K, z);
    return {odd || ldx % (long long)(16 / z) != 0 || off16(x), odd || off16(w), odd || off16(a),
            K % 4 == 0 && ldx % 4 == 0 && !(((uintptr_t)x | (uintptr_t)w | (uintptr_t)a) & (4 * z - 1))};
}
// one launch for one to four rows: no workspace (an allocation is 1.3 us of 12)
static inline bool one_launch(int M, int K, int r, size_t z, bool vec) {
    return M <= kOneRows && (long long)M * r * K * (int)z <= (vec ? kOneBytes : kOneOdd);
}
struct FwdWs { size_t t, partial, order, key, seg, xp, wp, ap, total; };
static FwdWs fwd_ws(int M, int K, int N, int r, int L, size_t z, const FwdLayout& in) {
    FwdWs w{};
    size_t o = 0;
    if (one_launch(M, K, r, z, in.vec)) return w;
    w.t = o; o += al((size_t)M * rank_pitch(r) * 4);
    if (M <= kFewRows) {
        int ks, kw;
        few_split(M, N, K, &ks, &kw);
        w.partial = o; o += al((size_t)ks * M * N * 4);
    } else {
        const size_t Kp = padded(K, z);
        w.order = o; o += al((size_t)M * 4);
        w.key = o; o += al((size_t)M * 4);
        w.seg = o; o += al((size_t)(L + 2) * 4);
        w.xp = o; o += in.x ? al(M * Kp * z) : 0;
        w.wp = o; o += in.w ? al(N * Kp * z) : 0;
        w.ap = o; o += in.a ? al((size_t)L * r * Kp * z) : 0;
        w.partial = o; o += al(gemm_partial(M, N, (int)Kp, z));
    }
    w.total = o;
    return w;
}
struct BwdWs { size_t u, partial, order, key, seg, wt, bt, dyp, part_a, part_b, total; };
static BwdWs bwd_ws(int M, int K, int N, int r, int L, size_t z, bool dx) {
    BwdWs w{};
    size_t o = 0;
    w.u = o; o += al((size_t)M * rank_pitch(r) * 4);
    if (M <= kFewRows) {
        int ks, kw;
        few_split(M, K, N, &ks, &kw);
        w.partial = o; o += dx ? al((size_t)ks * M * K * 4) : 0;
    } else {
        // adapters of several pieces have over kFewRows rows each, and less than one piece each beyond their rows'
        const size_t pieces = (size_t)std::min(L, M / (kFewRows + 1)) + M / kFewRows, Np = padded(N, z);
        w.order = o; o += al((size_t)M * 4);
        w.key = o; o += al((size_t)M * 4);
        w.seg = o; o += al((size_t)(L + 2) * 4);
        w.wt = o; o += dx ? al(K * Np * z) : 0;
        w.bt = o; o += al((size_t)L * r * Np * z);
        w.dyp = o; o += N == (int)Np ? 0 : al(M * Np * z);
        w.partial = o; o += dx ? al(gemm_partial(M, K, (int)Np, z)) : 0;
        w.part_a = o; o += al(pieces * r * K * 4);
        w.part_b = o; o += al(pieces * r * N * 4);
    }
    w.total = o;
    return w;
}

static int check_sizes(const char* who, int M, int K, int N, int r, int L) {
    if (M < 0 || K < 1 || N < 1 || r < 1 || L < 1) return fail(HMF_ERR_INVALID, "%s: M=%d K=%d N=%d r=%d L=%d", who, M, K, N, r, L);
    if (r > kMaxRank) return fail(HMF_ERR_UNSUPPORTED, "%s: rank %d, built up to %d", who, r, kMaxRank);
    // a grid has under 2^32 threads in a dimension, and its y extent is 16 bits
    const long long c = std::max(K, N) + 128ll, tc = c / 64 + 1, most = 4194303;                      // work-groups of 1,024
    const bool few = M <= kFewRows;
    if (L > 65535 || (long long)L + M / kFewRows > 65535 || (few && (M * c > 0xffffff00ll || L * (c / 128 + 1) * (r / 16 + 1) > 4 * most - c)) ||
        (!few && (long long)L + 1 + (M / 64 + 1) * tc + (N / 64 + 1) * (long long)(K / 64 + 3) + std::max((long long)L * r / 64 + 1, (long long)L) * tc > most))
        return fail(HMF_ERR_UNSUPPORTED, "%s: M=%d K=%d N=%d r=%d L=%d exceed the grid", who, M, K, N, r, L);
    return HMF_OK;
}

static AdCopy copy_job(const void* src, void* dst, long long lds_, long long ldd, long long sbs, long long dbs, int batches, int R, int C, int Cp, int trans) {
    AdCopy c{src, dst, lds_, ldd, sbs, dbs, R, C, Cp, trans, 0, blocks_of(R, trans ? 64 : 256), blocks_of(Cp, trans ? 256 : 64)};
    c.tiles = batches * c.tr * c.tc;
    return c;
}
template <typename T> static int prepare(const AdPrep& p, hipStream_t st) {
    long long wgs = p.L + 1;
    for (int k = 0; k < p.ncopy; ++k) wgs += p.copy[k].tiles;
    hipLaunchKernelGGL(k_ad_prep<T>, dim3((unsigned)wgs), dim3(kPrep), 0, st, p);
    HMF_LAUNCH_CHECK();
    return HMF_OK;
}
template <typename T> static int gemm(AdGemm<T>& m, void* partial, hipStream_t st) {
    int bt, rb, splits;
    gemm_shape(m.M, m.O, m.C, sizeof(T), &bt, &rb, &splits, &m.per);
    m.tiles_o = blocks_of(m.O, bt);
    m.partial = splits > 1 ? (float*)partial : nullptr;
    const dim3 grid(m.tiles_o * blocks_of(m.M, bt), splits);
    if (bt == 64) hipLaunchKernelGGL((k_ad_gemm<T, 64, 128>), grid, dim3(256), 0, st, m);
    else if (rb == 128) hipLaunchKernelGGL((k_ad_gemm<T, 128, 128>), grid, dim3(256), 0, st, m);
    else hipLaunchKernelGGL((k_ad_gemm<T, 128, 64>), grid, dim3(256), 0, st, m);
    HMF_LAUNCH_CHECK();
    if (splits > 1) {
        const long long n = (long long)m.M * m.O;
        hipLaunchKernelGGL(k_ad_sum<T>, dim3((unsigned)std::min<long long>((n + 255) / 256, 4096)), dim3(256), 0, st, m.partial, splits, m.bias, m.out, n, m.O);
        HMF_LAUNCH_CHECK();
    }
    return HMF_OK;
}

template <typename T>
static int forward_t(const T* x, long long ldx, const T* w, const T* bias, const T* a, const T* b, const float* scale, const int* ids, int M, int K, int N, int r, int L,
                     T* y, float* t, char* ws, hipStream_t st) {
    const FwdLayout in = fwd_layout(x, ldx, w, a, K, sizeof(T));
    const FwdWs o = fwd_ws(M, K, N, r, L, sizeof(T), in);
    AdArgs<T> g{};
    g.x = x; g.ldx = ldx; g.w = w; g.bias = bias; g.a = a; g.b = b; g.scale = scale; g.ids = ids; g.y = y; g.t = t ? t : (float*)(ws + o.t);
    g.M = M; g.K = K; g.N = N; g.r = r; g.L = L;
    if (one_launch(M, K, r, sizeof(T), in.vec)) {
        g.t = t;
        if (in.vec) hipLaunchKernelGGL((k_ad_one<T, true>), dim3(blocks_of(N, 8)), dim3(256), 0, st, g);
        else hipLaunchKernelGGL((k_ad_one<T, false>), dim3(blocks_of(N, 8)), dim3(256), 0, st, g);
        HMF_LAUNCH_CHECK();
        return HMF_OK;
    }
    if (M <= kFewRows) {
        few_split(M, N, K, &g.ksplit, &g.kw);
        g.partial = (float*)(ws + o.partial);
        const int to = blocks_of(N, 32), tm = blocks_of(M, 32);
        const dim3 grid(to * g.ksplit * tm + M);
        if (in.vec) hipLaunchKernelGGL((k_ad_few<T, true>), grid, dim3(256), 0, st, g, to, tm);
        else hipLaunchKernelGGL((k_ad_few<T, false>), grid, dim3(256), 0, st, g, to, tm);
        HMF_LAUNCH_CHECK();
        hipLaunchKernelGGL(k_ad_join<T>, dim3(blocks_of((long long)M * N, 64)), dim3(64), 0, st, g);
        HMF_LAUNCH_CHECK();
        return HMF_OK;
    }
    // x, W and A as whole chunks of aligned rows: themselves, or copies
    const int Kp = padded(K, sizeof(T));
    AdPrep pr{};
    pr.ids = ids; pr.order = (int*)(ws + o.order); pr.key = (int*)(ws + o.key); pr.seg = (int*)(ws + o.seg); pr.M = M; pr.L = L;
    AdLow lo{};
    lo.in = x; lo.ldin = ldx; lo.v = a; lo.ldv = K;
    AdGemm<T> m{};
    m.w = w; m.ldw = K;
    if (in.x) {
        pr.copy[pr.ncopy++] = copy_job(x, ws + o.xp, ldx, Kp, 0, 0, 1, M, K, Kp, 0);
        lo.in = ws + o.xp; lo.ldin = Kp;
    }
    if (in.w) {
        pr.copy[pr.ncopy++] = copy_job(w, ws + o.wp, K, Kp, 0, 0, 1, N, K, Kp, 0);
        m.w = (const T*)(ws + o.wp); m.ldw = Kp;
    }
    if (in.a) {
        pr.copy[pr.ncopy++] = copy_job(a, ws + o.ap, K, Kp, 0, 0, 1, L * r, K, Kp, 0);
        lo.v = ws + o.ap; lo.ldv = Kp;
    }
    if (int rc = prepare<T>(pr, st)) return rc;
    lo.scale = scale; lo.order = pr.order; lo.key = pr.key; lo.seg = pr.seg; lo.low = (float*)(ws + o.t); lo.t = t; lo.M = M; lo.C = Kp; lo.r = r;
    lo.rp = rank_pitch(r); lo.L = L;
    hipLaunchKernelGGL(k_ad_low<T>, dim3(L + 1 + M / 16), dim3(1024), 0, st, lo);
    HMF_LAUNCH_CHECK();
    m.in = (const T*)lo.in; m.ldin = lo.ldin; m.bias = bias; m.v = b; m.vl = (long long)N * r; m.vo = r; m.vj = 1; m.low = lo.low; m.rp = lo.rp; m.order = pr.order; m.key = pr.key; m.out = y;
    m.M = M; m.C = Kp; m.O = N; m.r = r; m.L = L;
    return gemm<T>(m, ws + o.partial, st);
}

template <typename T>
static int backward_t(const T* dy, const void* x, long long ldx, const unsigned char* exps, const float* t, const T* w, const T* a, const T* b, const float* scale,
                      const int* ids, int M, int K, int N, int r, int L, T* dx, T* da, T* db, char* ws, hipStream_t st) {
    const BwdWs o = bwd_ws(M, K, N, r, L, sizeof(T), dx != nullptr);
    AdArgs<T> g{};
    g.dy = dy; g.w = w; g.a = a; g.b = b; g.scale = scale; g.ids = ids; g.dx = dx; g.u = (float*)(ws + o.u);
    g.M = M; g.K = K; g.N = N; g.r = r; g.L = L;
    AdGrad ga{}, gb{};
    ga.p = g.u; ga.ldp = r; ga.z = x; ga.exps = exps; ga.out = da; ga.ldz = ldx; ga.C = ga.Cp = K; ga.trans = 0; ga.blocks = blocks_of(K, 128) * blocks_of(r, 16);
    gb.p = t; gb.ldp = r; gb.z = dy; gb.out = db; gb.ldz = N; gb.C = gb.Cp = N; gb.trans = 1; gb.blocks = blocks_of(N, 128) * blocks_of(r, 16);
    const bool vec = N % 4 == 0;                                           // dy itself is 16-byte aligned
    if (M <= kFewRows) {
        few_split(M, K, N, &g.ksplit, &g.kw);
        g.partial = (float*)(ws + o.partial);
        const int to = blocks_of(K, 32), tm = blocks_of(M, 32), nb = dx ? to * g.ksplit * tm : 0;
        const dim3 grid(nb + M + L * gb.blocks);
        if (vec) hipLaunchKernelGGL((k_ad_few_back<T, true>), grid, dim3(256), 0, st, g, gb, to, tm);
        else hipLaunchKernelGGL((k_ad_few_back<T, false>), grid, dim3(256), 0, st, g, gb, to, tm);
        HMF_LAUNCH_CHECK();
        const int jw = dx ? blocks_of((long long)M * K, 256) : 0;
        const dim3 grid2(jw + L * ga.blocks);
        if (exps) hipLaunchKernelGGL((k_ad_few_back2<T, true>), grid2, dim3(256), 0, st, g, ga, jw);
        else hipLaunchKernelGGL((k_ad_few_back2<T, false>), grid2, dim3(256), 0, st, g, ga, jw);
        HMF_LAUNCH_CHECK();
        return HMF_OK;
    }
    // W^T and B^T, dy as whole chunks of aligned rows
    const int Np = padded(N, sizeof(T));
    AdPrep pr{};
    pr.ids = ids; pr.order = (int*)(ws + o.order); pr.key = (int*)(ws + o.key); pr.seg = (int*)(ws + o.seg); pr.M = M; pr.L = L;
    pr.copy[pr.ncopy++] = copy_job(b, ws + o.bt, r, Np, (long long)N * r, (long long)r * Np, L, r, N, Np, 1);
    if (dx) pr.copy[pr.ncopy++] = copy_job(w, ws + o.wt, K, Np, 0, 0, 1, K, N, Np, 1);
    const T* dyp = dy;
    if (N != Np) {
        pr.copy[pr.ncopy++] = copy_job(dy, ws + o.dyp, N, Np, 0, 0, 1, M, N, Np, 0);
        dyp = (const T*)(ws + o.dyp);
        gb.z = dyp; gb.ldz = Np; gb.Cp = Np;                               // the padded rows serve dB's aligned loads too
    }
    if (int rc = prepare<T>(pr, st)) return rc;
    AdLow lo{};
    lo.in = dyp; lo.ldin = Np; lo.v = ws + o.bt; lo.ldv = Np; lo.scale = scale; lo.order = pr.order; lo.key = pr.key; lo.seg = pr.seg; lo.low = g.u; lo.M = M; lo.C = Np; lo.r = r;
    lo.rp = rank_pitch(r); lo.L = L;
    ga.ldp = lo.rp;
    hipLaunchKernelGGL(k_ad_low<T>, dim3(L + 1 + M / 16), dim3(1024), 0, st, lo);
    HMF_LAUNCH_CHECK();
    if (dx) {
        AdGemm<T> m{};
        m.in = dyp; m.ldin = Np; m.w = (const T*)(ws + o.wt); m.ldw = Np; m.v = a; m.vl = (long long)r * K; m.vo = 1; m.vj = K; m.low = g.u; m.rp = lo.rp; m.order = pr.order; m.key = pr.key;
        m.out = dx; m.M = M; m.C = Np; m.O = K; m.r = r; m.L = L;
        if (int rc = gemm<T>(m, ws + o.partial, st)) return rc;
    }
    const int *order = pr.order, *seg = pr.seg;
    ga.part = (float*)(ws + o.part_a);
    gb.part = (float*)(ws + o.part_b);
    const dim3 grid(ga.blocks + gb.blocks, L + M / kFewRows);
    if (exps) hipLaunchKernelGGL((k_ad_grads<T, true>), grid, dim3(256), 0, st, ga, gb, order, seg, r, L);
    else hipLaunchKernelGGL((k_ad_grads<T, false>), grid, dim3(256), 0, st, ga, gb, order, seg, r, L);
    HMF_LAUNCH_CHECK();
    hipLaunchKernelGGL(k_ad_grad_join<T>, dim3(std::min(256, blocks_of((long long)r * (K + N), 256)), L), dim3(256), 0, st, ga, gb, seg, r, L);
    HMF_LAUNCH_CHECK();
    return HMF_OK;
}

}  // namespace hmf

using namespace hmf;

extern "C" {

size_t hmf_adapted_linear_workspace_bytes(int M, int K, int N, int r, int L, int bf16) {
    if (M < 1 || K < 1 || N < 1 || r < 1 || L < 1) return 0;
    return fwd_ws(M, K, N, r, L, bf16 ? 2 : 4, kAnyLayout).total;
}

size_t hmf_adapted_linear_workspace_bytes_for(const void* x, long long ldx, const void* w, const void* a, int M, int K, int N, int r, int L, int bf16) {
    if (M < 1 || K < 1 || N < 1 || r < 1 || L < 1) return 0;
    const size_t z = bf16 ? 2 : 4;
    return fwd_ws(M, K, N, r, L, z, fwd_layout(x, ldx, w, a, K, z)).total;
}

int hmf_adapted_linear(const void* x, long long ldx, const void* w, const void* bias, const void* a, const void* b, const float* scale, const int* ids, int M, int K,
                       int N, int r, int L, int bf16, void* y, float* t, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_sizes("hmf_adapted_linear", M, K, N, r, L)) return rc;
    if (M == 0) return HMF_OK;
    if (!x || !w || !a || !b || !scale || !ids || !y || ldx < K) return fail(HMF_ERR_INVALID, "hmf_adapted_linear: null argument or ldx=%lld < K=%d", ldx, K);
    const size_t need = hmf_adapted_linear_workspace_bytes_for(x, ldx, w, a, M, K, N, r, L, bf16);
    if (need && (!workspace || workspace_bytes < need || off16(workspace)))
        return fail(HMF_ERR_WORKSPACE, "hmf_adapted_linear: workspace %zu < %zu bytes (16-byte aligned)", workspace_bytes, need);
    hipStream_t st = (hipStream_t)stream;
    if (bf16)
        return forward_t<bf16_t>((const bf16_t*)x, ldx, (const bf16_t*)w, (const bf16_t*)bias, (const bf16_t*)a, (const bf16_t*)b, scale, ids, M, K, N, r, L, (bf16_t*)y, t,
                                 (char*)workspace, st);
    return forward_t<float>((const float*)x, ldx, (const float*)w, (const float*)bias, (const float*)a, (const float*)b, scale, ids, M, K, N, r, L, (float*)y, t,
                            (char*)workspace, st);
}

size_t hmf_adapted_linear_backward_workspace_bytes(int M, int K, int N, int r, int L, int bf16) {
    if (M < 1 || K < 1 || N < 1 || r < 1 || L < 1) return 0;
    return bwd_ws(M, K, N, r, L, bf16 ? 2 : 4, true).total;
}

size_t hmf_adapted_linear_backward_workspace_bytes_for(int M, int K, int N, int r, int L, int bf16, int need_dx) {
    if (M < 1 || K < 1 || N < 1 || r < 1 || L < 1) return 0;
    return bwd_ws(M, K, N, r, L, bf16 ? 2 : 4, need_dx != 0).total;
}

int hmf_adapted_linear_backward(const void* dy, const void* x, long long ldx, const unsigned char* exps, const float* t, const void* w, const void* a, const void* b,
                                const float* scale, const int* ids, int M, int K, int N, int r, int L, int bf16, void* dx, void* da, void* db, void* workspace,
                                size_t workspace_bytes, void* stream) {
    if (int rc = check_sizes("hmf_adapted_linear_backward", M, K, N, r, L)) return rc;
    if (M < 1) return fail(HMF_ERR_INVALID, "hmf_adapted_linear_backward: no rows");
    if (!dy || !x || !t || !w || !a || !b || !scale || !ids || !da || !db || (exps ? ldx != K : ldx < K))
        return fail(HMF_ERR_INVALID, "hmf_adapted_linear_backward: null argument, or ldx=%lld with K=%d (a checkpoint is contiguous)", ldx, K);
    if (off16(dy)) return fail(HMF_ERR_INVALID, "hmf_adapted_linear_backward: dy must be 16-byte aligned");
    const size_t need = bwd_ws(M, K, N, r, L, bf16 ? 2 : 4, dx != nullptr).total;
    if (!workspace || workspace_bytes < need || off16(workspace))
        return fail(HMF_ERR_WORKSPACE, "hmf_adapted_linear_backward: workspace %zu < %zu bytes (16-byte aligned)", workspace_bytes, need);
    hipStream_t st = (hipStream_t)stream;
    if (bf16)
        return backward_t<bf16_t>((const bf16_t*)dy, x, ldx, exps, t, (const bf16_t*)w, (const bf16_t*)a, (const bf16_t*)b, scale, ids, M, K, N, r, L, (bf16_t*)dx, (bf16_t*)da,
                                  (bf16_t*)db, (char*)workspace, st);
    return backward_t<float>((const float*)dy, x, ldx, exps, t, (const float*)w, (const float*)a, (const float*)b, scale, ids, M, K, N, r, L, (float*)dx, (float*)da,
                             (float*)db, (char*)workspace, st);
}

}  // extern "C"
