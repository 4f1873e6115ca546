// Low-rank adapters of many requests beside a shared projection (the heads of models/humaniflow_model.py:232-252 with the weights of one trained model and a
// small difference to them for every subject, camera or data set):
//
//   l = ids[m] (negative: no adapter)      t[m] = s_l A_l x[m]              (r values, 32 bits, kept for the backward pass)
//   y[m] = W x[m] + b + B_l t[m]           W (N, K), A (L, r, K), B (L, N, r)
//   u[m] = s_l B_l^T dy[m]                 dx[m] = W^T dy[m] + A_l^T u[m]
//   dA_l = sum_{m: ids[m] = l} u[m] x[m]^T      dB_l = sum dy[m] t[m]^T     (an adapter without rows: zero)
//
// Two forms by the number of rows:
//   few rows (M <= kFewRows: a batch of images): the weights are read once and bound everything.  32 x 32 tiles straight from global memory on the fp32 MFMA, the
//     reduction split over waves and work-groups until the chip is full; the rows' own adapters are dot products of the rows; one joining launch
//     adds the partial sums (a fixed order), the bias and the adapters' part.  Two launches.
//   many rows: rows are put in the order of their adapters (a plan of two index arrays), and a tile of 128 rows treats its few adapters as more columns of
//     the reduction: [x, t] . [W, B_l]^T, with t zero in the columns of the other rows' adapters.
// Everything is accumulated in 32 bits.  bfloat16 operands of the many-row form are exact; t and u enter it as a high and a low bfloat16 (16 bits of mantissa),
// so the adapters' part loses nothing against the output's own rounding.
#include <algorithm>
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
__device__ __forceinline__ bf16_t to_bf16(float f) {                       // nearest even, a NaN stays one
    const unsigned int u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (bf16_t)((u >> 16) | 0x40u);
    return (bf16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ void down(float* p, float v) { *p = v; }
__device__ __forceinline__ void down(bf16_t* p, float v) { *p = to_bf16(v); }

// four consecutive elements at p as floats, `n` of them valid (VEC: the caller guarantees alignment, and n is 0 or >= 4)
template <bool VEC> __device__ __forceinline__ f32x4 load4(const float* p, int n) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (VEC) {
        if (n > 0) v = *(const f32x4*)p;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < n) v[k] = p[k];
    }
    return v;
}
template <bool VEC> __device__ __forceinline__ f32x4 load4(const bf16_t* p, int n) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (VEC) {
        if (n > 0) {
            const u16x4 h = *(const u16x4*)p;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = up(h[k]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < n) v[k] = up(p[k]);
    }
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
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
__device__ __forceinline__ void low_row(const AdArgs<T>& a, int m) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int l = a.ids[m];
    if (l < 0 || l >= a.L) {                                               // no adapter: zero; an id that no adapter has: NaN, so that it is seen
        for (int j = threadIdx.x; j < a.r; j += 256) a.t[(long long)m * a.r + j] = l < 0 ? 0.f : nan32();
        return;
    }
    const T* xr = a.x + (long long)m * a.ldx;
    const T* al = a.a + (long long)l * a.r * a.K;
    const float s = a.scale[l];
    for (int j0 = wave * 4; j0 < a.r; j0 += 16) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int k = lane * 4; k < a.K; k += 256) {
            const f32x4 xv = load4<VEC>(xr + k, a.K - k);
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
                const int j = min(j0 + jj, a.r - 1);
                const f32x4 av = load4<VEC>(al + (long long)j * a.K + k, a.K - k);
                acc[jj] = fmaf(xv[0], av[0], fmaf(xv[1], av[1], fmaf(xv[2], av[2], fmaf(xv[3], av[3], acc[jj]))));
            }
        }
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
            const float v = wave_sum(acc[jj]);
            if (lane == 0 && j0 + jj < a.r) a.t[(long long)m * a.r + j0 + jj] = s * v;
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
        for (int n = wave * per + g; n < a.N; n += 4 * per) acc = fmaf(up(dr[n]), up(bl[(long long)n * a.r + j]), acc);
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
                for (int e = 0; e < 4; ++e) wv[g][e] = e < n ? up(a.w[(long long)(cc + e) * O + oc]) : 0.f;
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
        low_row<T, VEC>(a, blockIdx.x - nb);
        return;
    }
    const int ot = blockIdx.x % tiles_o, rest = blockIdx.x / tiles_o;
    base_tile<T, true, VEC>(a, a.x, a.ldx, a.N, a.K, ot, rest % a.ksplit, rest / a.ksplit, red);
}

// y = partial sums + bias + B_l t
template <typename T>
__global__ __launch_bounds__(256) void k_ad_join(const AdArgs<T> a) {
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x, n_all = (long long)a.M * a.N;
    if (e >= n_all) return;
    const int m = (int)(e / a.N), n = (int)(e - (long long)m * a.N);
    float v = a.partial[e];
    for (int k = 1; k < a.ksplit; ++k) v += a.partial[(long long)k * n_all + e];
    if (a.bias) v += up(a.bias[n]);
    const int l = a.ids[m];
    if (l >= a.L) v = nan32();
    else if (l >= 0) {
        const T* br = a.b + ((long long)l * a.N + n) * a.r;
        const float* tr = a.t + (long long)m * a.r;
        float d = 0.f;
        for (int j = 0; j < a.r; ++j) d = fmaf(tr[j], up(br[j]), d);
        v += d;
    }
    down(a.y + e, v);
}

// ---------------------------------------------------------------------------------------------------
// gradients of the adapters: G[j][c] = sum over an adapter's rows of p[m][j] z[m][c], p (M, r) in 32 bits;  dA: p = u, z = x (or its 8-bit checkpoint);  dB^T: p = t, z = dy.
// A work-group owns (adapter, piece of <= 256 of its rows, 128 columns); its waves take a quarter of the rows each, 2 rows per MFMA step, and every lane the four
// columns 4 i .. 4 i + 3 (one vector load feeds four MFMA tiles); they meet in LDS in a fixed order.  More pieces than one: partial sums in the workspace,
// joined by k_ad_grad_join.
// ---------------------------------------------------------------------------------------------------
struct AdGrad {
    const float* p;
    const void* z;                     // rows of pitch ldz, or the codes (M, C)
    const unsigned char* exps;         // with codes
    void* out;                         // (L, r, C), or (L, C, r) with trans
    float* part;                       // [pieces][r][C]
    long long ldz;
    int C, trans, blocks;              // blocks: column blocks of 128
};

template <typename T> __device__ __forceinline__ f32x4 z4(const AdGrad& g, int m, int c, int n, bool vec) {
    const T* p = (const T*)g.z + (long long)m * g.ldz + c;
    return vec ? load4<true>(p, n) : load4<false>(p, n);
}
__device__ __forceinline__ f32x4 z4_act8(const AdGrad& g, int m, int c, int n, bool vec) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    const signed char* pc = (const signed char*)g.z + (long long)m * g.C + c;
    const unsigned char* pe = g.exps + (long long)(m >> 5) * g.C + c;
    unsigned int w = 0u, e = 0u;
    if (vec) {
        if (n > 0) { w = *(const unsigned int*)pc; e = *(const unsigned int*)pe; }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < n) { w |= (unsigned)(unsigned char)pc[k] << (8 * k); e |= (unsigned)pe[k] << (8 * k); }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int q = (int)(signed char)(w >> (8 * k));
        const float step = __uint_as_float((unsigned)max((int)((e >> (8 * k)) & 0xffu) - 6, 0) << 23);
        v[k] = q == -128 ? nan32() : (float)q * step;
    }
    return v;
}

// T: type of z and of the gradients; ACT8: z is a checkpoint
template <typename T, bool ACT8>
__device__ __forceinline__ void grad_piece(const AdGrad& g, int r, const int* rows, int n, int l, long long piece, bool whole, int cb, float* red) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 31, q = lane >> 5;
    const int c = cb * 128 + 4 * i, cn = g.C - c;
    const int esz = ACT8 ? 1 : (int)sizeof(T);
    const bool vec = (ACT8 ? g.C : g.ldz) % 4 == 0 && g.C % 4 == 0 && ((uintptr_t)g.z & (4 * esz - 1)) == 0 && (!ACT8 || ((uintptr_t)g.exps & 3) == 0);
    const int quarter = ((n + 3) / 4 + 1) & ~1, r0 = wave * quarter, r1 = min(r0 + quarter, n);
    for (int j0 = 0; j0 < r; j0 += 32) {
        const bool jin = j0 + i < r;
        f32x16 acc[4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[t][e] = 0.f;
        constexpr int U = 4;
        for (int rr = r0; rr < r1; rr += 2 * U) {
            f32x4 zv[U];
            float pv[U];
#pragma unroll
            for (int s = 0; s < U; ++s) {
                const int at = rr + 2 * s + q;
                const bool in = at < r1;
                const int m = rows[in ? at : 0];
                pv[s] = (in && jin) ? g.p[(long long)m * r + j0 + i] : 0.f;
                zv[s] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (in) zv[s] = ACT8 ? z4_act8(g, m, c, cn, vec) : z4<T>(g, m, c, cn, vec);
            }
#pragma unroll
            for (int s = 0; s < U; ++s)
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(pv[s], zv[s][t], acc[t], 0, 0, 0);
        }
        // rank 8 (e >> 2) + 4 q + (e & 3) of column 4 i + t
        __syncthreads();
        if (wave > 0)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) red[((wave - 1) * 64 + t * 16 + e) * 64 + lane] = acc[t][e];
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int j = j0 + 8 * (e >> 2) + 4 * q + (e & 3);
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int at = (t * 16 + e) * 64 + lane;
                    const float v = ((acc[t][e] + red[at]) + red[64 * 64 + at]) + red[2 * 64 * 64 + at];
                    if (j < r && t < cn) {
                        if (!whole) g.part[(piece * r + j) * g.C + c + t] = v;
                        else if (g.trans) down((T*)g.out + ((long long)l * g.C + c + t) * r + j, v);
                        else down((T*)g.out + ((long long)l * r + j) * g.C + c + t, v);
                    }
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
    __shared__ float red[3 * 64 * 64];
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
    __shared__ float red[3 * 64 * 64];
    __shared__ int rows[kFewRows], cnt[4];
    int id = blockIdx.x;
    if (id < join_wgs) {
        const long long e = (long long)id * 256 + threadIdx.x, n_all = (long long)a.M * a.K;
        if (e >= n_all) return;
        const int m = (int)(e / a.K), k = (int)(e - (long long)m * a.K);
        float v = a.partial[e];
        for (int s = 1; s < a.ksplit; ++s) v += a.partial[(long long)s * n_all + e];
        const int l = a.ids[m];
        if (l >= a.L) v = nan32();
        else if (l >= 0) {
            const T* ar = a.a + (long long)l * a.r * a.K + k;
            const float* ur = a.u + (long long)m * a.r;
            float d = 0.f;
            for (int j = 0; j < a.r; ++j) d = fmaf(ur[j], up(ar[(long long)j * a.K]), d);
            v += d;
        }
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
// order: the rows by adapter (those without one last), each adapter's in their own order;  seg[l]: where adapter l begins (seg[L]: rows without, seg[L + 1] = M).
// Work-group l counts the rows in front of its own, then places them; nothing is shared between work-groups.
__global__ __launch_bounds__(256) void k_ad_plan(const int* __restrict__ ids, int M, int L, int* __restrict__ order, int* __restrict__ seg) {
    __shared__ int cnt[4];
    const int l = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int less = 0;
    for (int m = threadIdx.x; m < M; m += 256) {
        const int v = ids[m], key = (v < 0 || v >= L) ? L : v;
        less += key < l;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) less += __shfl_xor(less, d);
    if (lane == 0) cnt[wave] = less;
    __syncthreads();
    int at = cnt[0] + cnt[1] + cnt[2] + cnt[3];
    if (threadIdx.x == 0) {
        seg[l] = at;
        if (l == L) seg[L + 1] = M;
    }
    for (int m0 = 0; m0 < M; m0 += 256) {
        const int m = m0 + threadIdx.x;
        bool mine = false;
        if (m < M) {
            const int v = ids[m], key = (v < 0 || v >= L) ? L : v;
            mine = key == l;
        }
        const unsigned long long b = __ballot(mine);
        __syncthreads();
        if (lane == 0) cnt[wave] = __popcll(b);
        __syncthreads();
        int base = at;
        for (int w = 0; w < wave; ++w) base += cnt[w];
        if (mine) order[base + __popcll(b & ((1ull << lane) - 1ull))] = m;
        at += cnt[0] + cnt[1] + cnt[2] + cnt[3];
    }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void k_ad_low(const AdArgs<T> a) { low_row<T, VEC>(a, blockIdx.x); }

template <typename T>
__global__ __launch_bounds__(256) void k_ad_up(const AdArgs<T> a) {
    __shared__ float red[256];
    up_row<T>(a, blockIdx.x, red);
}

// out[b][c][r] = in[b][r][c], 32 x 32 tiles
template <typename T>
__global__ __launch_bounds__(256) void k_ad_transpose(const T* __restrict__ in, T* __restrict__ out, int R, int C, int tc, int tr) {
    __shared__ T s[32][33];
    const int id = blockIdx.x, c0 = (id % tc) * 32, r0 = (id / tc) % tr * 32;
    const long long base = (long long)(id / (tc * tr)) * R * C;
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (r0 + y + 8 * k < R && c0 + x < C) s[y + 8 * k][x] = in[base + (long long)(r0 + y + 8 * k) * C + c0 + x];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (c0 + y + 8 * k < C && r0 + x < R) out[base + (long long)(c0 + y + 8 * k) * R + r0 + x] = s[x][y + 8 * k];
}

// out[m][o] = sum_c in[m][c] w[o][c] (+ bias[o]) + sum_j low[m][j] v[l][o][j]: forward in = x, w = W, low = t, v = B; backward in = dy, w = W^T, low = u, v = A^T.
template <typename T> struct AdGemm {
    const T *in, *w, *bias, *v;
    const float* low;
    const int *ids, *order;
    T* out;
    long long ldin;
    int M, C, O, r, L, tiles_o;
};

template <typename T> struct Mma;
template <> struct Mma<float> {                                            // 8 reduction elements: 4 steps of the 32 x 32 x 2 MFMA, lane half q holds 4 q .. 4 q + 3
    static constexpr int BK = 32, G = 8, E = 4, HL = 1;                     // E: elements of 16 bytes; HL: columns of the reduction per rank
    typedef f32x4 frag;
    static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ float part(float v, int) { return v; }
};
template <> struct Mma<bf16_t> {                                           // 16 reduction elements: one 32 x 32 x 16 MFMA, lane half q holds 8 q .. 8 q + 7
    static constexpr int BK = 64, G = 16, E = 8, HL = 2;
    typedef u16x8 frag;
    static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ bf16_t part(float v, int lo) {       // high half, and what it leaves
        const bf16_t h = to_bf16(v);
        return lo ? ((h & 0x7f80u) == 0x7f80u ? (bf16_t)0 : to_bf16(v - up(h))) : h;      // an infinity (or NaN) leaves nothing
    }
};
__device__ __forceinline__ bool finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ bool finite(bf16_t v) { return (v & 0x7f80u) != 0x7f80u; }

// 128 x 128 tile, 4 waves of 64 x 64 (2 x 2 MFMA tiles), two LDS stages of one chunk (BK reduction elements) each, rows padded by 16 bytes.  Chunks past the
// shared weight's are the adapters': element e belongs to the tile's adapter list[e / rr], rank e % rr.  The rows of other adapters hold zeros there, and a zero
// times an infinity or a NaN of a weight would reach them: such weights are staged as zeros and added to their own rows at the end.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void k_ad_gemm(const AdGemm<T> a) {
    typedef Mma<T> X;
    typedef typename X::frag frag;
    constexpr int BK = X::BK, E = X::E, P = BK + E;                         // pitch of an LDS row
    constexpr int SEG = BK / E, NS = 128 * SEG / 256;                       // 16-byte pieces of a row; pieces per thread and operand
    __shared__ __attribute__((aligned(16))) T sw[2][128 * P], sx[2][128 * P];
    __shared__ int rowid[128], slot[128], list[128], nlist[2], odd;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 31, q = lane >> 5;
    const int ot = blockIdx.x % a.tiles_o, mt = blockIdx.x / a.tiles_o;
    const int o0 = ot * 128, p0 = mt * 128;
    // the tile's rows and its distinct adapters, in order
    if (tid == 0) odd = 0;
    if (tid < 128) {
        const int p = p0 + tid;
        const int m = p < a.M ? a.order[p] : -1;
        int l = m >= 0 ? a.ids[m] : -1;
        if (l >= a.L) l = -1;
        const int prev = (tid > 0 && p < a.M) ? a.ids[a.order[p - 1]] : -1;
        const bool first = l >= 0 && l != prev;
        const unsigned long long b = __ballot(first);
        const int before = __popcll(b & ((2ull << lane) - 1ull));           // first rows up to and including this one
        rowid[tid] = m;
        if (lane == 0) nlist[wave] = __popcll(b);
        slot[tid] = l >= 0 ? before - 1 : -1000;                            // of this wave's list; the second wave's is moved below
        if (first) list[wave * 64 + before - 1] = l;
    }
    __syncthreads();
    // the second wave's first rows may continue the first wave's last adapter: then before - 1 = -1 is that adapter's place once moved
    const int n0 = nlist[0], n1 = nlist[1];
    int moved = 0;
    if (tid >= 64 && tid < 128) moved = list[tid];
    __syncthreads();
    if (tid >= 64 && tid < 128) {
        if (tid - 64 < n1) list[n0 + tid - 64] = moved;
        slot[tid] += n0;
    }
    __syncthreads();
    const int rr = a.r * X::HL, ext = (n0 + n1) * rr;
    const int kc = (a.C + BK - 1) / BK, nc = kc + (ext + BK - 1) / BK;

    frag gw[NS], gx[NS];
    auto fetch = [&](int c) {
        if (c < kc) {
            const int cb = c * BK;
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const int e = tid + 256 * s, row = e / SEG, cc = cb + (e % SEG) * E;
                const int o = o0 + row, m = rowid[row];
                frag zw, zx;
#pragma unroll
                for (int k = 0; k < E; ++k) { zw[k] = 0; zx[k] = 0; }
                const T* pw = a.w + (long long)o * a.C + cc;
                const T* px = a.in + (long long)m * a.ldin + cc;
                if (VEC) {
                    if (o < a.O && cc < a.C) zw = *(const frag*)pw;
                    if (m >= 0 && cc < a.C) zx = *(const frag*)px;
                } else {
#pragma unroll
                    for (int k = 0; k < E; ++k) {
                        if (o < a.O && cc + k < a.C) zw[k] = pw[k];
                        if (m >= 0 && cc + k < a.C) zx[k] = px[k];
                    }
                }
                gw[s] = zw;
                gx[s] = zx;
            }
        } else {
            const int eb = (c - kc) * BK;
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const int e = tid + 256 * s, row = e / SEG;
                const int o = o0 + row, m = rowid[row], sl = slot[row];
                frag zw, zx;
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    const int el = eb + (e % SEG) * E + k, ad = el / rr, jj = el - ad * rr, lo = jj >= a.r, j = lo ? jj - a.r : jj;
                    zw[k] = 0;
                    zx[k] = 0;
                    if (el < ext) {
                        if (o < a.O) {
                            zw[k] = a.v[((long long)list[ad] * a.O + o) * a.r + j];
                            if (!finite(zw[k])) { zw[k] = 0; odd = 1; }
                        }
                        if (ad == sl) zx[k] = X::part(a.low[(long long)m * a.r + j], lo);
                    }
                }
                gw[s] = zw;
                gx[s] = zx;
            }
        }
    };
    auto stash = [&](int b) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int e = tid + 256 * s, at = (e / SEG) * P + (e % SEG) * E;
            *(frag*)&sw[b][at] = gw[s];
            *(frag*)&sx[b][at] = gx[s];
        }
    };
    f32x16 acc[2][2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[t][v][e] = 0.f;
    const int wo = (wave & 1) * 64, wm = (wave >> 1) * 64;
    fetch(0);
    stash(0);
    __syncthreads();
    for (int c = 0; c < nc; ++c) {
        const int b = c & 1;
        if (c + 1 < nc) fetch(c + 1);
#pragma unroll
        for (int g = 0; g < BK / X::G; ++g) {
            frag fw[2], fx[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                fw[t] = *(const frag*)&sw[b][(wo + 32 * t + i) * P + g * X::G + q * E];
                fx[t] = *(const frag*)&sx[b][(wm + 32 * t + i) * P + g * X::G + q * E];
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int v = 0; v < 2; ++v) acc[t][v] = X::mma(fw[t], fx[v], acc[t][v]);
        }
        if (c + 1 < nc) stash(b ^ 1);
        __syncthreads();
    }
    // lane (m = column i) holds outputs 8 (e >> 2) + 4 q + (e & 3): four consecutive ones per store
    const bool vec = a.O % 4 == 0 && ((uintptr_t)a.out & (4 * sizeof(T) - 1)) == 0;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const int m = rowid[wm + 32 * v + i];
        if (m < 0) continue;
        const int l = a.ids[m];
        const bool bad = l >= a.L;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4) {
                const int o = o0 + wo + 32 * t + 8 * e4 + 4 * q;
                float z[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    z[e] = acc[t][v][4 * e4 + e];
                    if (a.bias && o + e < a.O) z[e] += up(a.bias[o + e]);
                    if (bad) z[e] = nan32();
                    if (odd && l >= 0 && !bad && o + e < a.O)
                        for (int j = 0; j < a.r; ++j) {
                            const T vv = a.v[((long long)l * a.O + o + e) * a.r + j];
                            if (!finite(vv)) z[e] = fmaf(a.low[(long long)m * a.r + j], up(vv), z[e]);
                        }
                }
                T* po = a.out + (long long)m * a.O + o;
                if (vec) {
                    if (o < a.O) {
                        T h[4] __attribute__((aligned(16)));
#pragma unroll
                        for (int e = 0; e < 4; ++e) down(h + e, z[e]);
                        if (sizeof(T) == 4) *(uint4*)po = *(const uint4*)h;
                        else *(uint2*)po = *(const uint2*)h;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (o + e < a.O) down(po + e, z[e]);
                }
            }
    }
}

// Piece z of the adapters' rows: adapter l has max(1, ceil(rows / kFewRows)) of them, one behind the other.  All threads return the same; l = L: no such piece.
__device__ __forceinline__ void find_piece(const int* seg, int L, int z, int& l, int& p, int& n, int& first) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int l0 = 0; l0 < L; l0 += 64) {
        const int li = l0 + lane;
        const int rows = li < L ? seg[li + 1] - seg[li] : 0;
        const int np = li < L ? max(1, (rows + kFewRows - 1) / kFewRows) : 0;
        int incl = np;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(incl, d);
            if (lane >= d) incl += o;
        }
        const unsigned long long over = __ballot(base + incl > z);
        if (over) {
            const int k = __ffsll((long long)over) - 1;
            l = l0 + k;
            const int np_k = __shfl(np, k);
            first = base + __shfl(incl, k) - np_k;
            p = z - first;
            n = np_k;
            return;
        }
        base += __shfl(incl, 63);
    }
    l = L;
    p = n = first = 0;
}

template <typename T, bool ACT8>
__global__ __launch_bounds__(256) void k_ad_grads(const AdGrad da, const AdGrad db, const int* __restrict__ order, const int* __restrict__ seg, int r, int L) {
    __shared__ float red[3 * 64 * 64];
    __shared__ int rows[kFewRows];
    int l, p, np, first;
    find_piece(seg, L, blockIdx.y, l, p, np, first);
    if (l >= L) return;
    const int s0 = seg[l] + p * kFewRows, n = min(kFewRows, seg[l + 1] - s0);
    if ((int)threadIdx.x < n) rows[threadIdx.x] = order[s0 + threadIdx.x];
    __syncthreads();
    const int cb = blockIdx.x;
    if (cb < da.blocks) grad_piece<T, ACT8>(da, r, rows, n, l, blockIdx.y, np == 1, cb, red);
    else grad_piece<T, false>(db, r, rows, n, l, blockIdx.y, np == 1, cb - da.blocks, red);
}

// sums of the adapters that had several pieces, in the pieces' order; one work-group per (adapter, 256 elements of dA_l or dB_l)
template <typename T>
__global__ __launch_bounds__(256) void k_ad_grad_join(const AdGrad da, const AdGrad db, const int* __restrict__ seg, int r, int L, int wa) {
    const int l = blockIdx.y;
    if (seg[l + 1] - seg[l] <= kFewRows) return;
    int first = 0, np = 0;
    {                                                                      // pieces in front of this adapter's
        const int lane = threadIdx.x & 63;
        for (int l0 = 0; l0 < l; l0 += 64) {
            const int li = l0 + lane;
            int v = li < l ? max(1, (seg[li + 1] - seg[li] + kFewRows - 1) / kFewRows) : 0;
#pragma unroll
            for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
            first += v;
        }
        np = (seg[l + 1] - seg[l] + kFewRows - 1) / kFewRows;
    }
    const bool is_a = (int)blockIdx.x < wa;
    const AdGrad& g = is_a ? da : db;
    const long long e = (long long)(is_a ? blockIdx.x : blockIdx.x - wa) * 256 + threadIdx.x, n = (long long)r * g.C;
    if (e >= n) return;
    float v = 0.f;
    for (int p = 0; p < np; ++p) v += g.part[(long long)(first + p) * n + e];
    const int j = (int)(e / g.C), c = (int)(e - (long long)j * g.C);
    if (g.trans) down((T*)g.out + ((long long)l * g.C + c) * r + j, v);
    else down((T*)g.out + ((long long)l * r + j) * g.C + c, v);
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

struct FwdWs { size_t t, partial, order, seg, total; };
static FwdWs fwd_ws(int M, int K, int N, int r, int L) {
    FwdWs w{};
    size_t o = 0;
    w.t = o; o += al((size_t)M * r * 4);
    if (M <= kFewRows) {
        int ks, kw;
        few_split(M, N, K, &ks, &kw);
        w.partial = o; o += al((size_t)ks * M * N * 4);
    } else {
        w.order = o; o += al((size_t)M * 4);
        w.seg = o; o += al((size_t)(L + 2) * 4);
    }
    w.total = o;
    return w;
}
struct BwdWs { size_t u, partial, order, seg, wt, at, part_a, part_b, total; };
static BwdWs bwd_ws(int M, int K, int N, int r, int L, int bf16) {
    BwdWs w{};
    size_t o = 0;
    const size_t z = bf16 ? 2 : 4;
    w.u = o; o += al((size_t)M * r * 4);
    if (M <= kFewRows) {
        int ks, kw;
        few_split(M, K, N, &ks, &kw);
        w.partial = o; o += al((size_t)ks * M * K * 4);
    } else {
        const size_t pieces = (size_t)L + M / kFewRows;
        w.order = o; o += al((size_t)M * 4);
        w.seg = o; o += al((size_t)(L + 2) * 4);
        w.wt = o; o += al((size_t)N * K * z);
        w.at = o; o += al((size_t)L * r * K * z);
        w.part_a = o; o += al(pieces * r * K * 4);
        w.part_b = o; o += al(pieces * r * N * 4);
    }
    w.total = o;
    return w;
}

static int check_sizes(const char* who, int M, int K, int N, int r, int L) {
    if (M < 0 || K < 1 || N < 1 || r < 1 || L < 1) return fail(HMF_ERR_INVALID, "%s: M=%d K=%d N=%d r=%d L=%d", who, M, K, N, r, L);
    if (r > kMaxRank) return fail(HMF_ERR_UNSUPPORTED, "%s: rank %d, built up to %d", who, r, kMaxRank);
    if (L > 65535 || M > (1 << 30) || (long long)blocks_of(M, 128) * blocks_of(std::max(N, K), 128) > 0x7fffffffLL || (long long)L + M / kFewRows > 65535)
        return fail(HMF_ERR_UNSUPPORTED, "%s: M=%d K=%d N=%d L=%d exceed the grid", who, M, K, N, L);
    return HMF_OK;
}

template <typename T>
static int forward_t(const T* x, long long ldx, const T* w, const T* bias, const T* a, const T* b, const float* scale, const int* ids, int M, int K, int N, int r, int L,
                     T* y, float* t, char* ws, hipStream_t st) {
    const FwdWs o = fwd_ws(M, K, N, r, L);
    AdArgs<T> g{};
    g.x = x; g.ldx = ldx; g.w = w; g.bias = bias; g.a = a; g.b = b; g.scale = scale; g.ids = ids; g.y = y; g.t = t ? t : (float*)(ws + o.t);
    g.M = M; g.K = K; g.N = N; g.r = r; g.L = L;
    const int V = 16 / (int)sizeof(T);
    const bool vec = K % V == 0 && ldx % V == 0 && !off16(x) && !off16(w) && !off16(a);
    if (M <= kFewRows) {
        few_split(M, N, K, &g.ksplit, &g.kw);
        g.partial = (float*)(ws + o.partial);
        const int to = blocks_of(N, 32), tm = blocks_of(M, 32);
        const dim3 grid(to * g.ksplit * tm + M);
        if (vec) hipLaunchKernelGGL((k_ad_few<T, true>), grid, dim3(256), 0, st, g, to, tm);
        else hipLaunchKernelGGL((k_ad_few<T, false>), grid, dim3(256), 0, st, g, to, tm);
        HMF_LAUNCH_CHECK();
        hipLaunchKernelGGL(k_ad_join<T>, dim3(blocks_of((long long)M * N, 256)), dim3(256), 0, st, g);
        HMF_LAUNCH_CHECK();
        return HMF_OK;
    }
    int *order = (int*)(ws + o.order), *seg = (int*)(ws + o.seg);
    hipLaunchKernelGGL(k_ad_plan, dim3(L + 1), dim3(256), 0, st, ids, M, L, order, seg);
    HMF_LAUNCH_CHECK();
    if (vec) hipLaunchKernelGGL((k_ad_low<T, true>), dim3(M), dim3(256), 0, st, g);
    else hipLaunchKernelGGL((k_ad_low<T, false>), dim3(M), dim3(256), 0, st, g);
    HMF_LAUNCH_CHECK();
    AdGemm<T> m{};
    m.in = x; m.ldin = ldx; m.w = w; m.bias = bias; m.v = b; m.low = g.t; m.ids = ids; m.order = order; m.out = y;
    m.M = M; m.C = K; m.O = N; m.r = r; m.L = L; m.tiles_o = blocks_of(N, 128);
    const dim3 grid(m.tiles_o * blocks_of(M, 128));
    if (vec) hipLaunchKernelGGL((k_ad_gemm<T, true>), grid, dim3(256), 0, st, m);
    else hipLaunchKernelGGL((k_ad_gemm<T, false>), grid, dim3(256), 0, st, m);
    HMF_LAUNCH_CHECK();
    return HMF_OK;
}

template <typename T>
static int backward_t(const T* dy, const void* x, long long ldx, const unsigned char* exps, const float* t, const T* w, const T* a, const T* b, const float* scale,
                      const int* ids, int M, int K, int N, int r, int L, T* dx, T* da, T* db, char* ws, hipStream_t st) {
    const BwdWs o = bwd_ws(M, K, N, r, L, sizeof(T) == 2);
    AdArgs<T> g{};
    g.dy = dy; g.w = w; g.a = a; g.b = b; g.scale = scale; g.ids = ids; g.dx = dx; g.u = (float*)(ws + o.u);
    g.M = M; g.K = K; g.N = N; g.r = r; g.L = L;
    AdGrad ga{}, gb{};
    ga.p = g.u; ga.z = x; ga.exps = exps; ga.out = da; ga.ldz = ldx; ga.C = K; ga.trans = 0; ga.blocks = blocks_of(K, 128);
    gb.p = t; gb.z = dy; gb.out = db; gb.ldz = N; gb.C = N; gb.trans = 1; gb.blocks = blocks_of(N, 128);
    const int V = 16 / (int)sizeof(T);
    const bool vec = N % V == 0 && !off16(dy);
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
    int *order = (int*)(ws + o.order), *seg = (int*)(ws + o.seg);
    hipLaunchKernelGGL(k_ad_plan, dim3(L + 1), dim3(256), 0, st, ids, M, L, order, seg);
    HMF_LAUNCH_CHECK();
    hipLaunchKernelGGL(k_ad_up<T>, dim3(M), dim3(256), 0, st, g);
    HMF_LAUNCH_CHECK();
    if (dx) {
        T *wt = (T*)(ws + o.wt), *at = (T*)(ws + o.at);
        const int tk = blocks_of(K, 32);
        hipLaunchKernelGGL(k_ad_transpose<T>, dim3(tk * blocks_of(N, 32)), dim3(256), 0, st, w, wt, N, K, tk, blocks_of(N, 32));
        HMF_LAUNCH_CHECK();
        hipLaunchKernelGGL(k_ad_transpose<T>, dim3(tk * blocks_of(r, 32) * L), dim3(256), 0, st, a, at, r, K, tk, blocks_of(r, 32));
        HMF_LAUNCH_CHECK();
        AdGemm<T> m{};
        m.in = dy; m.ldin = N; m.w = wt; m.v = at; m.low = g.u; m.ids = ids; m.order = order; m.out = dx;
        m.M = M; m.C = N; m.O = K; m.r = r; m.L = L; m.tiles_o = blocks_of(K, 128);
        const dim3 grid(m.tiles_o * blocks_of(M, 128));
        if (vec) hipLaunchKernelGGL((k_ad_gemm<T, true>), grid, dim3(256), 0, st, m);
        else hipLaunchKernelGGL((k_ad_gemm<T, false>), grid, dim3(256), 0, st, m);
        HMF_LAUNCH_CHECK();
    }
    ga.part = (float*)(ws + o.part_a);
    gb.part = (float*)(ws + o.part_b);
    const dim3 grid(ga.blocks + gb.blocks, L + M / kFewRows);
    if (exps) hipLaunchKernelGGL((k_ad_grads<T, true>), grid, dim3(256), 0, st, ga, gb, order, seg, r, L);
    else hipLaunchKernelGGL((k_ad_grads<T, false>), grid, dim3(256), 0, st, ga, gb, order, seg, r, L);
    HMF_LAUNCH_CHECK();
    const int wa = blocks_of((long long)r * K, 256), wb = blocks_of((long long)r * N, 256);
    hipLaunchKernelGGL(k_ad_grad_join<T>, dim3(wa + wb, L), dim3(256), 0, st, ga, gb, seg, r, L, wa);
    HMF_LAUNCH_CHECK();
    return HMF_OK;
}

}  // namespace hmf

using namespace hmf;

extern "C" {

size_t hmf_adapted_linear_workspace_bytes(int M, int K, int N, int r, int L) {
    if (M < 1 || K < 1 || N < 1 || r < 1 || L < 1) return 0;
    return fwd_ws(M, K, N, r, L).total;
}

int hmf_adapted_linear(const void* x, long long ldx, const void* w, const void* bias, const void* a, const void* b, const float* scale, const int* ids, int M, int K,
                       int N, int r, int L, int bf16, void* y, float* t, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_sizes("hmf_adapted_linear", M, K, N, r, L)) return rc;
    if (M == 0) return HMF_OK;
    if (!x || !w || !a || !b || !scale || !ids || !y || ldx < K) return fail(HMF_ERR_INVALID, "hmf_adapted_linear: null argument or ldx=%lld < K=%d", ldx, K);
    const size_t need = fwd_ws(M, K, N, r, L).total;
    if (!workspace || workspace_bytes < need || off16(workspace))
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
    return bwd_ws(M, K, N, r, L, bf16).total;
}

int hmf_adapted_linear_backward(const void* dy, const void* x, long long ldx, const unsigned char* exps, const float* t, const void* w, const void* a, const void* b,
                                const float* scale, const int* ids, int M, int K, int N, int r, int L, int bf16, void* dx, void* da, void* db, void* workspace,
                                size_t workspace_bytes, void* stream) {
    if (int rc = check_sizes("hmf_adapted_linear_backward", M, K, N, r, L)) return rc;
    if (M < 1) return fail(HMF_ERR_INVALID, "hmf_adapted_linear_backward: no rows");
    if (!dy || !x || !t || !w || !a || !b || !scale || !ids || !da || !db || (exps ? ldx != K : ldx < K))
        return fail(HMF_ERR_INVALID, "hmf_adapted_linear_backward: null argument, or ldx=%lld with K=%d (a checkpoint is contiguous)", ldx, K);
    const size_t need = bwd_ws(M, K, N, r, L, bf16).total;
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
