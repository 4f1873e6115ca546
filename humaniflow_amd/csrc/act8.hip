// 8-bit activation checkpoints: what a training step keeps of an activation between its forward and its backward pass, and the BatchNorm + ReLU
// backward that reads them (models/resnet.py under train(); the 32-bit forms are in encoder_train.hip).
//
// A checkpoint of rows x (M, C) is, for blocks of 32 consecutive rows of ONE column (a channel: its own scale, and 32 neighbouring pixels):
//   exps  uint8 [ceil(M/32)][C]   E = ((bits(amax) + 0x10000) >> 23) clamped to [7, 254]: the exponent field of the block's largest finite magnitude,
//                                 one more where that magnitude would round to 128 steps;  step = 2^(E - 133)
//   codes int8  [M][C]            rint(x / step), |code| <= 127; -128 marks a value that was not finite (it comes back as NaN)
// The step is a power of two, so x / step is exact and the code's rounding (to nearest even) is the only one: |x - code * step| <= step / 2, between
// amax / 254 and amax / 127.  A scale of amax / 127 would gain half a bit on average and cost a division and a rounding that depends on how the
// division is done; a power of two gives the same codes in any arithmetic and a scale of one byte (1.03 bytes per element in all).
//   bits  uint32 [ceil(M/32)][C]  bit i of word t: the ReLU's input was positive in row 32 t + i (exact: the backward mask is that of the forward pass)
//
// All kernels are streams over the data, bound by HBM.  A wave owns a tile of 32 rows x 64 channels: lane = 4 channels (16 lanes: 256 consecutive
// bytes of a row) x a quarter of the rows (row 4 i + q), so a tile is 8 independent 16-byte loads per lane and the block maximum needs two shuffles per
// channel; with the 32 rows of a block in one lane (no shuffle) the tensor of the last layer (4,608 x 512) is 288 waves on 1,024 SIMDs.
#include <algorithm>
#include <type_traits>
#include "hmf_common.h"

namespace hmf {

typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));

constexpr float kMagic = 12582912.0f;           // 1.5 * 2^23: v + kMagic holds rint(v) in its low bits, |v| < 2^22

__device__ __forceinline__ unsigned int mag_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// magnitude of a finite value as bits (they order like the magnitudes), 0 for infinities and NaN
__device__ __forceinline__ unsigned int fin_mag(float v) {
    const unsigned int m = mag_bits(v);
    return m < 0x7f800000u ? m : 0u;
}
__device__ __forceinline__ int exp_of(unsigned int amax_bits) { return min(max((int)((amax_bits + 0x10000u) >> 23), 7), 254); }
__device__ __forceinline__ float inv_step(int E) { return __uint_as_float((unsigned)(260 - E) << 23); }      // 2^(133 - E)
__device__ __forceinline__ float step_of(int E) { return __uint_as_float((unsigned)max(E - 6, 0) << 23); }   // 2^(E - 133)
__device__ __forceinline__ unsigned int code_of(float v, float inv) {
    const float q = __builtin_amdgcn_fmed3f(v * inv, -127.f, 127.f) + kMagic;      // the clamp acts only where E itself was clamped
    return mag_bits(v) < 0x7f800000u ? (__float_as_uint(q) & 0xffu) : 0x80u;
}
__device__ __forceinline__ unsigned int pack4(unsigned int a, unsigned int b, unsigned int c, unsigned int d) { return a | (b << 8) | (c << 16) | (d << 24); }
__device__ __forceinline__ float value_of(unsigned int word, int k, float step) {
    const int c = (int)(signed char)(word >> (8 * k));
    return c == -128 ? __uint_as_float(0x7fc00000u) : (float)c * step;
}
// a word of codes without the marker -128 (values_of's fast side): plain conversions
__device__ __forceinline__ bool has_marker(unsigned int word) {
    const unsigned int x = word ^ 0x80808080u;
    return ((x - 0x01010101u) & ~x & 0x80808080u) != 0u;
}
template <bool MARKED> __device__ __forceinline__ float value_minus(unsigned int word, int k, float step, float sub) {
    const int c = (int)(signed char)(word >> (8 * k));
    const float v = fmaf((float)c, step, -sub);                            // the product is exact: one rounding
    return MARKED && c == -128 ? __uint_as_float(0x7fc00000u) : v;
}
// v where bit b (a constant after unrolling) of the word is set, else 0: two integer operations
__device__ __forceinline__ float where_bit(unsigned int word, int b, float v) {
    return __uint_as_float(__float_as_uint(v) & (unsigned)__builtin_amdgcn_sbfe((int)word, b, 1));
}
__device__ __forceinline__ unsigned int max_over_quarters(unsigned int m) {
    m = max(m, (unsigned)__shfl_xor((int)m, 16));
    return max(m, (unsigned)__shfl_xor((int)m, 32));
}
__device__ __forceinline__ float bf16_to_f32(unsigned short h) { return __uint_as_float((unsigned)h << 16); }
__device__ __forceinline__ unsigned short f32_to_bf16(float f) { return __builtin_bit_cast(unsigned short, (__bf16)f); }      // nearest even

// NT: past the caches.  A map of more than half the Infinity Cache (256 MB) is gone from it before its reader comes, and only pushes out what the next kernels
// read: the backward of 294,912 x 256 takes 247 us with, 269 us without; a small map's reader finds it there.  (The forward's map: 202 us without, 207 us with.)
constexpr long long kStreamBytes = 128ll << 20;
template <bool NT> __device__ __forceinline__ void store4(float* p, f32x4 v) {
    if (NT) __builtin_nontemporal_store(v, (f32x4*)p);
    else *(f32x4*)p = v;
}

// lane's V consecutive columns of one row: 16 bytes
template <bool BF16> struct Row;
template <> struct Row<false> {
    static constexpr int V = 4;
    f32x4 d;
    __device__ __forceinline__ void load(const void* p, long long o) { d = *(const f32x4*)((const float*)p + o); }
    __device__ __forceinline__ float get(int k) const { return d[k]; }
    __device__ __forceinline__ void set(int k, float v) { d[k] = v; }
    __device__ __forceinline__ void store(void* p, long long o) const { *(f32x4*)((float*)p + o) = d; }
};
template <> struct Row<true> {
    static constexpr int V = 8;
    u16x8 d;
    __device__ __forceinline__ void load(const void* p, long long o) { d = *(const u16x8*)((const unsigned short*)p + o); }
    __device__ __forceinline__ float get(int k) const { return bf16_to_f32(d[k]); }
    __device__ __forceinline__ void set(int k, float v) { d[k] = f32_to_bf16(v); }
    __device__ __forceinline__ void store(void* p, long long o) const { *(u16x8*)((unsigned short*)p + o) = d; }
};

// ---------------------------------------------------------------------------------------------------
// pack / unpack of plain rows.  Aligned form: C a multiple of V (4 floats / 8 bfloat16), rows 16-byte aligned.  Tile of a wave: 32 rows x 16 V columns.
// ---------------------------------------------------------------------------------------------------
template <bool BF16>
__global__ __launch_bounds__(256) void k_act8_pack(const void* __restrict__ x, long long ld, int M, int C, unsigned char* __restrict__ codes,
                                                   unsigned char* __restrict__ exps, int ct, long long tiles) {
    constexpr int V = Row<BF16>::V;
    const long long tile = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tile >= tiles) return;
    const int lane = threadIdx.x & 63, q = lane >> 4;
    const int t = (int)(tile / ct), c = (int)(tile - (long long)t * ct) * 16 * V + (lane & 15) * V;
    const bool live = c < C;                                          // C is a multiple of V: a lane's columns are all in or all out
    const int m0 = t * 32 + q;
    Row<BF16> r[8];
    bool in[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {                                     // what is not there reads the last row (of this block) or column: no load behind a condition
        in[i] = live && m0 + 4 * i < M;
        r[i].load(x, (long long)min(m0 + 4 * i, M - 1) * ld + min(c, C - V));
    }
    unsigned int top[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        top[k] = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) top[k] = max(top[k], fin_mag(r[i].get(k)));
    }
    float inv[V];
    unsigned int E[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        E[k] = (unsigned)exp_of(max_over_quarters(top[k]));
        inv[k] = inv_step((int)E[k]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (in[i]) {
            unsigned int w[V / 4];
#pragma unroll
            for (int j = 0; j < V / 4; ++j)
                w[j] = pack4(code_of(r[i].get(4 * j), inv[4 * j]), code_of(r[i].get(4 * j + 1), inv[4 * j + 1]), code_of(r[i].get(4 * j + 2), inv[4 * j + 2]),
                             code_of(r[i].get(4 * j + 3), inv[4 * j + 3]));
            unsigned int* o = (unsigned int*)(codes + (long long)(m0 + 4 * i) * C + c);
#pragma unroll
            for (int j = 0; j < V / 4; ++j) o[j] = w[j];
        }
    if (live && q == 0) {
        unsigned int* o = (unsigned int*)(exps + (long long)t * C + c);
#pragma unroll
        for (int j = 0; j < V / 4; ++j) o[j] = pack4(E[4 * j], E[4 * j + 1], E[4 * j + 2], E[4 * j + 3]);
    }
}

template <bool BF16>
__global__ __launch_bounds__(256) void k_act8_unpack(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ exps, int M, int C,
                                                     void* __restrict__ out, int ct, long long tiles) {
    constexpr int V = Row<BF16>::V;
    const long long tile = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tile >= tiles) return;
    const int lane = threadIdx.x & 63, q = lane >> 4;
    const int t = (int)(tile / ct), c = (int)(tile - (long long)t * ct) * 16 * V + (lane & 15) * V;
    if (c >= C) return;
    const int m0 = t * 32 + q;
    const unsigned int* pe = (const unsigned int*)(exps + (long long)t * C + c);
    unsigned int e[V / 4], w[8][V / 4];
#pragma unroll
    for (int j = 0; j < V / 4; ++j) e[j] = pe[j];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (m0 + 4 * i < M) {
            const unsigned int* p = (const unsigned int*)(codes + (long long)(m0 + 4 * i) * C + c);
#pragma unroll
            for (int j = 0; j < V / 4; ++j) w[i][j] = p[j];
        }
    float st[V];
#pragma unroll
    for (int k = 0; k < V; ++k) st[k] = step_of((int)((e[k / 4] >> (8 * (k & 3))) & 0xffu));
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (m0 + 4 * i < M) {
            Row<BF16> r;
#pragma unroll
            for (int k = 0; k < V; ++k) r.set(k, value_of(w[i][k / 4], k & 3, st[k]));
            r.store(out, (long long)(m0 + 4 * i) * C + c);
        }
}

// Any width, pitch and alignment: lane = one column, the 32 rows of a block in the lane (64 consecutive elements of a row per load)
template <bool BF16>
__global__ __launch_bounds__(256) void k_act8_pack_any(const void* __restrict__ x, long long ld, int M, int C, unsigned char* __restrict__ codes,
                                                       unsigned char* __restrict__ exps, int ct, long long tiles) {
    const long long tile = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tile >= tiles) return;
    const int t = (int)(tile / ct), c = (int)(tile - (long long)t * ct) * 64 + (threadIdx.x & 63);
    if (c >= C) return;
    const int m0 = t * 32, n = min(32, M - m0);
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const long long o = (long long)(m0 + min(i, n - 1)) * ld + c;
        v[i] = BF16 ? bf16_to_f32(((const unsigned short*)x)[o]) : ((const float*)x)[o];
    }
    unsigned int top = 0u;
#pragma unroll
    for (int i = 0; i < 32; ++i) top = max(top, fin_mag(v[i]));
    const int E = exp_of(top);
    const float inv = inv_step(E);
#pragma unroll
    for (int i = 0; i < 32; ++i)
        if (i < n) codes[(long long)(m0 + i) * C + c] = (unsigned char)code_of(v[i], inv);
    exps[(long long)t * C + c] = (unsigned char)E;
}

template <bool BF16>
__global__ __launch_bounds__(256) void k_act8_unpack_any(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ exps, int M, int C,
                                                         void* __restrict__ out, int ct, long long tiles) {
    const long long tile = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tile >= tiles) return;
    const int t = (int)(tile / ct), c = (int)(tile - (long long)t * ct) * 64 + (threadIdx.x & 63);
    if (c >= C) return;
    const int m0 = t * 32, n = min(32, M - m0);
    const float st = step_of(exps[(long long)t * C + c]);
    unsigned char w[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) w[i] = i < n ? codes[(long long)(m0 + i) * C + c] : 0;
#pragma unroll
    for (int i = 0; i < 32; ++i)
        if (i < n) {
            const float v = value_of(w[i], 0, st);
            const long long o = (long long)(m0 + i) * C + c;
            if (BF16) ((unsigned short*)out)[o] = f32_to_bf16(v);
            else ((float*)out)[o] = v;
        }
}

// ---------------------------------------------------------------------------------------------------
// BatchNorm affine (+ identity) (+ ReLU) that leaves the checkpoint of its input y (and of its output) behind: one pass over y and the identity.
//   v = fma(y, scale[c], shift[c]) + res;   out = relu ? max(v, 0) : v  (a NaN stays one);   bits = v > 0
// A separate checkpoint pass would read y (and out) again: 4 (8) more bytes per element.
// ---------------------------------------------------------------------------------------------------
template <bool RES, bool RELU, bool KEEP>
__global__ __launch_bounds__(256) void k_bn_apply8(const float* __restrict__ y, const float* __restrict__ scale, const float* __restrict__ shift,
                                                   const float* __restrict__ res, float* __restrict__ out, unsigned char* __restrict__ codes,
                                                   unsigned char* __restrict__ exps, unsigned int* __restrict__ bits, unsigned char* __restrict__ ocodes,
                                                   unsigned char* __restrict__ oexps, int M, int C, int ct, long long tiles) {
    const long long tile = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tile >= tiles) return;
    const int lane = threadIdx.x & 63, q = lane >> 4;
    const int t = (int)(tile / ct), c = (int)(tile - (long long)t * ct) * 64 + (lane & 15) * 4;
    const int m0 = t * 32 + q;
    const f32x4 sc = *(const f32x4*)(scale + c), sh = *(const f32x4*)(shift + c);
    f32x4 v[8], r[8];
    bool in[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        in[i] = m0 + 4 * i < M;
        const long long o = (long long)(m0 + 4 * i) * C + c;
        v[i] = in[i] ? *(const f32x4*)(y + o) : f32x4{0.f, 0.f, 0.f, 0.f};
        if (RES) r[i] = in[i] ? *(const f32x4*)(res + o) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    unsigned int top[4] = {0u, 0u, 0u, 0u}, otop[4] = {0u, 0u, 0u, 0u}, on[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) top[k] = max(top[k], fin_mag(v[i][k]));
    float inv[4];
    unsigned int E[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        E[k] = (unsigned)exp_of(max_over_quarters(top[k]));
        inv[k] = inv_step((int)E[k]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (in[i]) {
            const long long o = (long long)(m0 + 4 * i) * C + c;
            *(unsigned int*)(codes + o) = pack4(code_of(v[i][0], inv[0]), code_of(v[i][1], inv[1]), code_of(v[i][2], inv[2]), code_of(v[i][3], inv[3]));
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float a = fmaf(v[i][k], sc[k], sh[k]);
                if (RES) a = __fadd_rn(a, r[i][k]);
                if (RELU) {
                    on[k] |= (a > 0.f ? 1u : 0u) << (4 * i + q);
                    a = (a != a) ? a : fmaxf(a, 0.f);
                }
                v[i][k] = a;
                if (KEEP) otop[k] = max(otop[k], fin_mag(a));
            }
            *(f32x4*)(out + o) = v[i];
        }
    if (q == 0) *(unsigned int*)(exps + (long long)t * C + c) = pack4(E[0], E[1], E[2], E[3]);
    if (RELU) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            on[k] |= (unsigned)__shfl_xor((int)on[k], 16);
            on[k] |= (unsigned)__shfl_xor((int)on[k], 32);
        }
        if (q == 1) *(uint4*)(bits + (long long)t * C + c) = make_uint4(on[0], on[1], on[2], on[3]);
    }
    if (KEEP) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            E[k] = (unsigned)exp_of(max_over_quarters(otop[k]));
            inv[k] = inv_step((int)E[k]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (in[i])
                *(unsigned int*)(ocodes + (long long)(m0 + 4 * i) * C + c) =
                    pack4(code_of(v[i][0], inv[0]), code_of(v[i][1], inv[1]), code_of(v[i][2], inv[2]), code_of(v[i][3], inv[3]));
        if (q == 2) *(unsigned int*)(oexps + (long long)t * C + c) = pack4(E[0], E[1], E[2], E[3]);
    }
}

// The activation behind such a unit, rebuilt for the next layer's weight gradient: max(fma(yq, scale, shift), 0) where the bit is set, 0 elsewhere
// (bits null: the affine alone).  A value that was not finite stays a NaN.
__global__ __launch_bounds__(256) void k_act8_restore(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ exps,
                                                      const unsigned int* __restrict__ bits, const float* __restrict__ scale, const float* __restrict__ shift,
                                                      float* __restrict__ out, int M, int C, int ct, long long tiles) {
    const long long tile = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tile >= tiles) return;
    const int lane = threadIdx.x & 63, q = lane >> 4;
    const int t = (int)(tile / ct), c = (int)(tile - (long long)t * ct) * 64 + (lane & 15) * 4;
    const int m0 = t * 32 + q;
    const f32x4 sc = *(const f32x4*)(scale + c), sh = *(const f32x4*)(shift + c);
    const unsigned int e = *(const unsigned int*)(exps + (long long)t * C + c);
    uint4 b = make_uint4(~0u, ~0u, ~0u, ~0u);
    if (bits) b = *(const uint4*)(bits + (long long)t * C + c);
    const unsigned int on[4] = {b.x, b.y, b.z, b.w};
    const float floor_ = bits ? 0.f : -INFINITY;
    unsigned int w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = *(const unsigned int*)(codes + (long long)min(m0 + 4 * i, M - 1) * C + c);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (m0 + 4 * i < M) {
            f32x4 o;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float a = fmaf(value_of(w[i], k, step_of((int)((e >> (8 * k)) & 0xffu))), sc[k], sh[k]);
                o[k] = (a != a) ? a : (((on[k] >> (4 * i + q)) & 1u) ? fmaxf(a, floor_) : 0.f);
            }
            *(f32x4*)(out + (long long)(m0 + 4 * i) * C + c) = o;
        }
}

// ---------------------------------------------------------------------------------------------------
// BatchNorm (+ ReLU) backward from the checkpoint: gz = bit ? g : 0, xhat = (yq - mean) rstd,
//   sg = sum gz, sgx = sum gz xhat (over the M rows);  gy = gamma rstd (gz - sg / M - xhat sgx / M);  d gamma = sgx, d beta = sg.
// Two passes over g (4 bytes) and the checkpoint (1.16 bytes) where the 32-bit form reads g, out and y (12 bytes) in each.  A lane adds its rows of one
// tile run in 32 bits, everything above that in 64 bits and in a fixed order (partial sums per work-group, no atomics): results repeat bit for bit.
// ---------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_bn8_reduce(const float* __restrict__ g, const unsigned char* __restrict__ codes, const unsigned char* __restrict__ exps,
                                                    const unsigned int* __restrict__ bits, const float* __restrict__ mean, const float* __restrict__ rstd, int M,
                                                    int C, int tiles_per_wg, double* __restrict__ part) {
    __shared__ double red[2][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
    const int c = blockIdx.x * 64 + (lane & 15) * 4;
    const f32x4 mu = *(const f32x4*)(mean + c), rs = *(const f32x4*)(rstd + c);
    const int nt = (M + 31) / 32, t_end = min(((int)blockIdx.y + 1) * tiles_per_wg, nt);
    double S[4] = {0.0, 0.0, 0.0, 0.0}, SX[4] = {0.0, 0.0, 0.0, 0.0};
    for (int t = blockIdx.y * tiles_per_wg + wave; t < t_end; t += 4) {
        const int m0 = t * 32 + q;
        f32x4 gv[8];
        unsigned int w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool in = m0 + 4 * i < M;
            const long long o = (long long)(m0 + 4 * i) * C + c;
            gv[i] = in ? *(const f32x4*)(g + o) : f32x4{0.f, 0.f, 0.f, 0.f};
            w[i] = in ? *(const unsigned int*)(codes + o) : 0u;
        }
        const unsigned int e = *(const unsigned int*)(exps + (long long)t * C + c);
        uint4 b = make_uint4(~0u, ~0u, ~0u, ~0u);
        if (bits) b = *(const uint4*)(bits + (long long)t * C + c);
        const unsigned int on[4] = {b.x >> q, b.y >> q, b.z >> q, b.w >> q};
        auto add = [&](auto MARKED) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float st = step_of((int)((e >> (8 * k)) & 0xffu));
                float s = 0.f, sx = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float gz = where_bit(on[k], 4 * i, gv[i][k]);
                    s += gz;
                    sx = fmaf(gz, value_minus<decltype(MARKED)::value>(w[i], k, st, mu[k]), sx);
                }
                S[k] += (double)s;
                SX[k] += (double)(sx * rs[k]);
            }
        };
        bool marked = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) marked |= has_marker(w[i]);
        if (__any(marked)) add(std::true_type{});
        else add(std::false_type{});
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        S[k] += __shfl_xor(S[k], 16);
        S[k] += __shfl_xor(S[k], 32);
        SX[k] += __shfl_xor(SX[k], 16);
        SX[k] += __shfl_xor(SX[k], 32);
    }
    if (q == 0)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            red[0][wave][lane * 4 + k] = S[k];
            red[1][wave][lane * 4 + k] = SX[k];
        }
    __syncthreads();
    if (threadIdx.x < 128) {
        const int which = threadIdx.x >> 6, cc = threadIdx.x & 63;
        part[((long long)blockIdx.y * 2 + which) * C + blockIdx.x * 64 + cc] =
            ((red[which][0][cc] + red[which][1][cc]) + red[which][2][cc]) + red[which][3][cc];
    }
}

// coef[0][c] = gamma rstd, coef[1][c] = sg / M, coef[2][c] = sgx / M; 64 lanes per channel walk the partial sums, four channels a work-group (16 lanes: 576 partial sums
// of 256 channels took 14 us)
__global__ __launch_bounds__(256) void k_bn8_finalize(const double* __restrict__ part, int nparts, int M, int C, const float* __restrict__ gamma,
                                                      const float* __restrict__ rstd, float* __restrict__ g_gamma, float* __restrict__ g_beta,
                                                      float* __restrict__ coef) {
    __shared__ double red[2][64][5];
    const int cl = threadIdx.x & 3, j = threadIdx.x >> 2, c = blockIdx.x * 4 + cl;
    double s = 0.0, sx = 0.0;
    for (int p0 = j; p0 < nparts; p0 += 64 * 4) {
        double v[4], w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const long long p = min(p0 + 64 * k, nparts - 1);
            v[k] = part[p * 2 * C + c];
            w[k] = part[(p * 2 + 1) * C + c];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (p0 + 64 * k < nparts) { s += v[k]; sx += w[k]; }
    }
    red[0][j][cl] = s;
    red[1][j][cl] = sx;
    __syncthreads();
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        if (j < d) {
            red[0][j][cl] += red[0][j + d][cl];
            red[1][j][cl] += red[1][j + d][cl];
        }
        __syncthreads();
    }
    if (j == 0) {
        const double a = red[0][0][cl], b = red[1][0][cl];
        g_beta[c] = (float)a;
        g_gamma[c] = (float)b;
        coef[c] = gamma[c] * rstd[c];
        coef[C + c] = (float)(a / M);
        coef[2 * C + c] = (float)(b / M);
    }
}

// What the second pass needs to add the partial sums itself (FOLD): every wave those of its 64 channels, 1 KB for each work-group of the first pass.
struct Bn8Fold {
    const double* part;
    const float* gamma;
    float *g_gamma, *g_beta;
    int nparts;
};
template <bool GZ, bool NT, bool FOLD>
__global__ __launch_bounds__(256) void k_bn8_apply(const float* __restrict__ g, const unsigned char* __restrict__ codes, const unsigned char* __restrict__ exps,
                                                   const unsigned int* __restrict__ bits, const float* __restrict__ mean, const float* __restrict__ rstd,
                                                   const float* __restrict__ coef, float* __restrict__ gy, float* __restrict__ gz_out, int M, int C, int ct,
                                                   long long tiles, const Bn8Fold f) {
    // last tile first: the reduction ended there, and what it read last is still in the Infinity Cache
    const long long tile = tiles - 1 - ((long long)blockIdx.x * 4 + (threadIdx.x >> 6));
    if (tile < 0) return;
    const int lane = threadIdx.x & 63, q = lane >> 4;
    const int t = (int)(tile / ct), c = (int)(tile - (long long)t * ct) * 64 + (lane & 15) * 4;
    const int m0 = t * 32 + q;
    f32x4 gv[8];
    unsigned int w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        w[i] = 0u;
        if (m0 + 4 * i < M) {
            const long long o = (long long)(m0 + 4 * i) * C + c;
            gv[i] = *(const f32x4*)(g + o);
            w[i] = *(const unsigned int*)(codes + o);
        }
    }
    const unsigned int e = *(const unsigned int*)(exps + (long long)t * C + c);
    uint4 b = make_uint4(~0u, ~0u, ~0u, ~0u);
    if (bits) b = *(const uint4*)(bits + (long long)t * C + c);
    const unsigned int on[4] = {b.x >> q, b.y >> q, b.z >> q, b.w >> q};
    const f32x4 mu = *(const f32x4*)(mean + c), rs = *(const f32x4*)(rstd + c);
    f32x4 ca, cs, cx;
    if (FOLD) {                                                            // lane = one of the wave's 64 channels, then handed to the lanes that use it
        const int ch = c - (lane & 15) * 4 + lane;
        double a = 0.0, b2 = 0.0;
        for (int p0 = 0; p0 < f.nparts; p0 += 8) {
            double v[8], x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const long long p = min(p0 + k, f.nparts - 1);
                v[k] = f.part[p * 2 * C + ch];
                x[k] = f.part[(p * 2 + 1) * C + ch];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (p0 + k < f.nparts) { a += v[k]; b2 += x[k]; }
        }
        const float fa = f.gamma[ch] * rstd[ch], fs = (float)(a / M), fx = (float)(b2 / M);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            ca[k] = __shfl(fa, (lane & 15) * 4 + k);
            cs[k] = __shfl(fs, (lane & 15) * 4 + k);
            cx[k] = __shfl(fx, (lane & 15) * 4 + k);
        }
        if (t == 0) {
            f.g_beta[ch] = (float)a;
            f.g_gamma[ch] = (float)b2;
        }
    } else {
        ca = *(const f32x4*)(coef + c);
        cs = *(const f32x4*)(coef + C + c);
        cx = *(const f32x4*)(coef + 2 * C + c);
    }
    float st[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) st[k] = step_of((int)((e >> (8 * k)) & 0xffu));
    auto write = [&](auto MARKED) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (m0 + 4 * i < M) {
                f32x4 z, o;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float xh = value_minus<decltype(MARKED)::value>(w[i], k, st[k], mu[k]) * rs[k];
                    z[k] = where_bit(on[k], 4 * i, gv[i][k]);
                    o[k] = ca[k] * ((z[k] - cs[k]) - xh * cx[k]);
                }
                const long long at = (long long)(m0 + 4 * i) * C + c;
                store4<NT>(gy + at, o);
                if (GZ) store4<NT>(gz_out + at, z);
            }
    };
    bool marked = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) marked |= has_marker(w[i]);
    if (__any(marked)) write(std::true_type{});
    else write(std::false_type{});
}

// Tiles of 32 rows per work-group of the reduction: enough work-groups for the 256 CUs first, then up to 16 tiles (512 rows) each
static int bn8_tiles_per_wg(int M, int C) {
    const int nt = (M + 31) / 32;
    const long long cols = C / 64;
    int per = (int)std::min<long long>(16, (nt * cols + 2047) / 2048);
    per = std::max(8, (per + 3) / 4 * 4);
    while ((long long)((nt + per - 1) / per) > 65535) per *= 2;                // the grid's y extent
    return per;
}
constexpr long long kFoldReads = 64 << 10;      // wave reads of 1 KB: 64 MB
static int bn8_parts(int M, int C) { const int per = bn8_tiles_per_wg(M, C); return ((M + 31) / 32 + per - 1) / per; }

static inline bool misaligned(const void* p, unsigned a) { return ((uintptr_t)p & (a - 1)) != 0; }
constexpr long long kMaxTiles = 4LL * 16777215;                            // four tiles to a work-group of 256: a grid has under 2^32 threads
constexpr int kMaxRows = 0x7fffff00;                                       // row numbers are ints

}  // namespace hmf

using namespace hmf;

extern "C" {

int hmf_act8_pack(const void* x, long long ld, int bf16, int M, int C, signed char* codes, unsigned char* exps, void* stream) {
    if (M < 0 || C < 0 || ld < C) return fail(HMF_ERR_INVALID, "hmf_act8_pack: M=%d C=%d ld=%lld", M, C, ld);
    if (M == 0 || C == 0) return HMF_OK;
    if (!x || !codes || !exps) return fail(HMF_ERR_INVALID, "hmf_act8_pack: null argument");
    const int V = bf16 ? 8 : 4;
    const bool fast = C % V == 0 && ld % V == 0 && !misaligned(x, 16) && !misaligned(codes, 4) && !misaligned(exps, 4);
    const int cols = fast ? 16 * V : 64, ct = (C + cols - 1) / cols;
    const long long tiles = ((long long)M + 31) / 32 * ct;
    if (M > kMaxRows || tiles > kMaxTiles) return fail(HMF_ERR_UNSUPPORTED, "hmf_act8_pack: M=%d C=%d exceeds the grid", M, C);
    const dim3 grid((unsigned)((tiles + 3) / 4)), block(256);
    hipStream_t st = (hipStream_t)stream;
    unsigned char* cd = (unsigned char*)codes;
    if (fast && bf16) hipLaunchKernelGGL(k_act8_pack<true>, grid, block, 0, st, x, ld, M, C, cd, exps, ct, tiles);
    else if (fast) hipLaunchKernelGGL(k_act8_pack<false>, grid, block, 0, st, x, ld, M, C, cd, exps, ct, tiles);
    else if (bf16) hipLaunchKernelGGL(k_act8_pack_any<true>, grid, block, 0, st, x, ld, M, C, cd, exps, ct, tiles);
    else hipLaunchKernelGGL(k_act8_pack_any<false>, grid, block, 0, st, x, ld, M, C, cd, exps, ct, tiles);
    HMF_LAUNCH_CHECK();
    return HMF_OK;
}

int hmf_act8_unpack(const signed char* codes, const unsigned char* exps, int M, int C, void* x, int bf16, void* stream) {
    if (M < 0 || C < 0) return fail(HMF_ERR_INVALID, "hmf_act8_unpack: M=%d C=%d", M, C);
    if (M == 0 || C == 0) return HMF_OK;
    if (!x || !codes || !exps) return fail(HMF_ERR_INVALID, "hmf_act8_unpack: null argument");
    const int V = bf16 ? 8 : 4;
    const bool fast = C % V == 0 && !misaligned(x, 16) && !misaligned(codes, 4) && !misaligned(exps, 4);
    const int cols = fast ? 16 * V : 64, ct = (C + cols - 1) / cols;
    const long long tiles = ((long long)M + 31) / 32 * ct;
    if (M > kMaxRows || tiles > kMaxTiles) return fail(HMF_ERR_UNSUPPORTED, "hmf_act8_unpack: M=%d C=%d exceeds the grid", M, C);
    const dim3 grid((unsigned)((tiles + 3) / 4)), block(256);
    hipStream_t st = (hipStream_t)stream;
    const unsigned char* cd = (const unsigned char*)codes;
    if (fast && bf16) hipLaunchKernelGGL(k_act8_unpack<true>, grid, block, 0, st, cd, exps, M, C, x, ct, tiles);
    else if (fast) hipLaunchKernelGGL(k_act8_unpack<false>, grid, block, 0, st, cd, exps, M, C, x, ct, tiles);
    else if (bf16) hipLaunchKernelGGL(k_act8_unpack_any<true>, grid, block, 0, st, cd, exps, M, C, x, ct, tiles);
    else hipLaunchKernelGGL(k_act8_unpack_any<false>, grid, block, 0, st, cd, exps, M, C, x, ct, tiles);
    HMF_LAUNCH_CHECK();
    return HMF_OK;
}

int hmf_bn_apply_act8(const float* y, const float* scale, const float* shift, const float* residual, float* out, signed char* codes, unsigned char* exps,
                      unsigned int* bits, signed char* out_codes, unsigned char* out_exps, int M, int C, int relu, void* stream) {
    if (!y || !scale || !shift || !out || !codes || !exps || M <= 0 || C <= 0 || C % 64 || (relu && !bits) || (!relu && bits) || (!out_codes != !out_exps))
        return fail(HMF_ERR_INVALID, "hmf_bn_apply_act8: bad args (C %% 64 == 0; bits with relu and only then; out_codes and out_exps together)");
    if (misaligned(y, 16) || misaligned(scale, 16) || misaligned(shift, 16) || misaligned(residual, 16) || misaligned(out, 16) || misaligned(codes, 4) ||
        misaligned(exps, 4) || misaligned(bits, 16) || misaligned(out_codes, 4) || misaligned(out_exps, 4))
        return fail(HMF_ERR_INVALID, "hmf_bn_apply_act8: float tensors and bits must be 16-byte aligned, codes and exps 4-byte");
    const int ct = C / 64;
    const long long tiles = ((long long)M + 31) / 32 * ct;
    if (M > kMaxRows || tiles > kMaxTiles) return fail(HMF_ERR_UNSUPPORTED, "hmf_bn_apply_act8: M=%d C=%d exceeds the grid", M, C);
    const dim3 grid((unsigned)((tiles + 3) / 4)), block(256);
    hipStream_t st = (hipStream_t)stream;
    unsigned char *cd = (unsigned char*)codes, *oc = (unsigned char*)out_codes;
#define HMF_BN8(RES, RELU, KEEP) hipLaunchKernelGGL((k_bn_apply8<RES, RELU, KEEP>), grid, block, 0, st, y, scale, shift, residual, out, cd, exps, bits, oc, out_exps, M, C, ct, tiles)
    const int sel = (residual ? 4 : 0) | (relu ? 2 : 0) | (out_codes ? 1 : 0);
    switch (sel) {
        case 0: HMF_BN8(false, false, false); break;
        case 1: HMF_BN8(false, false, true); break;
        case 2: HMF_BN8(false, true, false); break;
        case 3: HMF_BN8(false, true, true); break;
        case 4: HMF_BN8(true, false, false); break;
        case 5: HMF_BN8(true, false, true); break;
        case 6: HMF_BN8(true, true, false); break;
        default: HMF_BN8(true, true, true); break;
    }
#undef HMF_BN8
    HMF_LAUNCH_CHECK();
    return HMF_OK;
}

int hmf_act8_restore_activation(const signed char* codes, const unsigned char* exps, const unsigned int* bits, const float* scale, const float* shift, float* x,
                                int M, int C, void* stream) {
    if (!codes || !exps || !scale || !shift || !x || M <= 0 || C <= 0 || C % 64)
        return fail(HMF_ERR_INVALID, "hmf_act8_restore_activation: bad args (C %% 64 == 0 required)");
    if (misaligned(codes, 4) || misaligned(exps, 4) || misaligned(bits, 16) || misaligned(scale, 16) || misaligned(shift, 16) || misaligned(x, 16))
        return fail(HMF_ERR_INVALID, "hmf_act8_restore_activation: float tensors and bits must be 16-byte aligned, codes and exps 4-byte");
    const int ct = C / 64;
    const long long tiles = ((long long)M + 31) / 32 * ct;
    if (M > kMaxRows || tiles > kMaxTiles) return fail(HMF_ERR_UNSUPPORTED, "hmf_act8_restore_activation: M=%d C=%d exceeds the grid", M, C);
    hipLaunchKernelGGL(k_act8_restore, dim3((unsigned)((tiles + 3) / 4)), dim3(256), 0, (hipStream_t)stream, (const unsigned char*)codes, exps, bits, scale, shift,
                       x, M, C, ct, tiles);
    HMF_LAUNCH_CHECK();
    return HMF_OK;
}

size_t hmf_bn_backward_act8_workspace_bytes(int M, int C) {
    if (M <= 0 || M > kMaxRows || C <= 0 || C % 64) return 0;
    return (size_t)bn8_parts(M, C) * 2 * C * sizeof(double) + (size_t)3 * C * sizeof(float);
}

int hmf_bn_backward_act8(const float* g, const signed char* codes, const unsigned char* exps, const unsigned int* bits, const float* mean, const float* rstd,
                         const float* gamma, float* gy, float* gz, float* g_gamma, float* g_beta, int M, int C, void* workspace, size_t workspace_bytes,
                         void* stream) {
    if (!g || !codes || !exps || !mean || !rstd || !gamma || !gy || !g_gamma || !g_beta || M <= 0 || C <= 0 || C % 64)
        return fail(HMF_ERR_INVALID, "hmf_bn_backward_act8: bad args (C %% 64 == 0 required)");
    if (misaligned(g, 16) || misaligned(codes, 4) || misaligned(exps, 4) || misaligned(bits, 16) || misaligned(mean, 16) || misaligned(rstd, 16) ||
        misaligned(gy, 16) || misaligned(gz, 16) || misaligned(workspace, 16))
        return fail(HMF_ERR_INVALID, "hmf_bn_backward_act8: float tensors, bits and workspace must be 16-byte aligned, codes and exps 4-byte");
    const size_t need = hmf_bn_backward_act8_workspace_bytes(M, C);
    if (!workspace || workspace_bytes < need) return fail(HMF_ERR_WORKSPACE, "hmf_bn_backward_act8: workspace %zu < %zu bytes", workspace_bytes, need);
    const int per = bn8_tiles_per_wg(M, C), parts = bn8_parts(M, C), ct = C / 64;
    if (M > kMaxRows || (long long)((M + 31) / 32) * ct > kMaxTiles) return fail(HMF_ERR_UNSUPPORTED, "hmf_bn_backward_act8: M=%d C=%d exceeds the grid", M, C);
    double* part = (double*)workspace;
    float* coef = (float*)(part + (size_t)parts * 2 * C);
    hipStream_t st = (hipStream_t)stream;
    const unsigned char* cd = (const unsigned char*)codes;
    hipLaunchKernelGGL(k_bn8_reduce, dim3(ct, parts), dim3(256), 0, st, g, cd, exps, bits, mean, rstd, M, C, per, part);
    HMF_LAUNCH_CHECK();
    const long long tiles = ((long long)M + 31) / 32 * ct;
    // A launch of its own for the partial sums costs 3 us and the call's host time another 3; adding them in every wave of the second pass costs their reads.
    const bool nt = (long long)M * C * 4 > kStreamBytes, fold = !nt && tiles * parts <= kFoldReads;
    if (!fold) {
        hipLaunchKernelGGL(k_bn8_finalize, dim3(C / 4), dim3(256), 0, st, part, parts, M, C, gamma, rstd, g_gamma, g_beta, coef);
        HMF_LAUNCH_CHECK();
    }
    const Bn8Fold f{part, gamma, g_gamma, g_beta, parts};
    const dim3 grid((unsigned)((tiles + 3) / 4)), block(256);
#define HMF_BN8A(GZ, NT, FOLD) hipLaunchKernelGGL((k_bn8_apply<GZ, NT, FOLD>), grid, block, 0, st, g, cd, exps, bits, mean, rstd, coef, gy, gz, M, C, ct, tiles, f)
    if (gz && nt) HMF_BN8A(true, true, false);
    else if (nt) HMF_BN8A(false, true, false);
    else if (gz && fold) HMF_BN8A(true, false, true);
    else if (gz) HMF_BN8A(true, false, false);
    else if (fold) HMF_BN8A(false, false, true);
    else HMF_BN8A(false, false, false);
#undef HMF_BN8A
    HMF_LAUNCH_CHECK();
    return HMF_OK;
}

}  // extern "C"
