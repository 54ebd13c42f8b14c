// Cross entropy of a row's unembedding, without the [rows, vocabulary] logits, and its gradient (gfx950).
//
//   l[m][v] = sum_d x[m][d] W[d][v] + b[v]          lse[m] = log sum_v exp l[m][v]
//   loss[m] = lse[m] - l[m][t_m]                    (0 where t_m is the ignored index)
//   G[m][v] = g_m (exp(l[m][v] - lse[m]) - [v = t_m])        dx = G W^T      dW = x^T G      db = sum_m G
//
// Bound by the matrix pipe: 2 M D V operations forward; backward makes the logits again (2 M D V) and adds two products of
// the same size.  Forward: the tile of logits stays in the accumulators, only its rows' maximum and sum of exponentials leave
// the workgroup.  Backward, in pieces of the vocabulary: G of a piece goes to the workspace in 16 bits (fp32: two fp16
// planes), and the two products read it from there.
#include <new>

#include "unembed_gemm.h"

using namespace unembed_gemm;

namespace {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float read_elem(const void *p, int elem, long long i) {
    if (elem == TSC_ELEM_F32) return ((const float *)p)[i];
    if (elem == TSC_ELEM_BF16) return (float)((const __bf16 *)p)[i];
    return (float)((const _Float16 *)p)[i];
}
__device__ __forceinline__ void write_elem(void *p, int elem, long long i, float v) {
    if (elem == TSC_ELEM_F32) ((float *)p)[i] = v;
    else if (elem == TSC_ELEM_BF16) ((__bf16 *)p)[i] = (__bf16)v;
    else ((_Float16 *)p)[i] = (_Float16)v;
}
__device__ __forceinline__ short bits(_Float16 v) { return __builtin_bit_cast(short, v); }
__device__ __forceinline__ short bits(__bf16 v) { return __builtin_bit_cast(short, v); }

// power of two s that brings a magnitude into [2^13, 2^14) when divided by s (1 for 0, infinities and NaN)
__device__ __forceinline__ float pow2_scale(float top) {
    if (!(top > 0.f) || !(top < __builtin_inff())) return 1.f;
    const int e = (int)(__float_as_uint(top) >> 23) - 13;  // biased exponent of s; 1: the smallest normal
    return __uint_as_float((unsigned)(e < 1 ? 1 : e) << 23);
}
// h1 + h2 / 2048 = v to 22 bits.  A value that fp16 does not hold (it is not finite, or NaN) goes to h1 alone.
__device__ __forceinline__ void split(float v, short &h1, short &h2) {
    const _Float16 a = (_Float16)v;
    const float r = (v - (float)a) * 2048.f;
    h1 = bits(a);
    h2 = fabsf((float)a) < __builtin_inff() ? bits((_Float16)r) : (short)0;
}

// ------------------------------------------------------------------------------------------------ operands
__global__ __launch_bounds__(1024) void absmax_kernel(const float *w, long long rows, long long cols, long long ld, unsigned *top) {
    float m = 0.f;
    for (long long r = blockIdx.x; r < rows; r += gridDim.x)
        for (long long c = threadIdx.x; c < cols; c += 1024) {
            const float v = fabsf(w[r * ld + c]);
            m = v < __builtin_inff() ? fmaxf(m, v) : m;
        }
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    __shared__ float s[16];
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) m = fmaxf(m, s[i]);
        atomicMax(top, __float_as_uint(m));  // non-negative floats order like their bits; a maximum has no order of arrival
    }
}
__global__ void wscale_kernel(float *wscale) {  // wscale[0]: the maximum's bits -> s; reset to the neutral 1 where all is 0
    wscale[0] = pow2_scale(wscale[0]);
}
__global__ void fill_kernel(float *p, float v, long long n) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = v;
}
// (the lowest finite fp32 and bf16 values mean -inf: their product with log2 e would overflow half way)
__global__ void bias_kernel(const void *b, int elem, int V, int n, float *out) {
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v >= n) return;
    const float x = v < V ? (b ? read_elem(b, elem, v) : 0.f) : -__builtin_inff();
    out[v] = x < -1e38f ? -__builtin_inff() : x;
}

// out[r][c] = in[r * sr + c * sc], c < C, zero up to the pitch (of a plane); one of sr, sc is 1
__global__ __launch_bounds__(256) void pack_w_kernel(const void *in, int elem, long long sr, long long sc, int R, int C, int Cp,
                                                     const float *wscale, short *out) {
    __shared__ float t[64][65];
    const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64, a = threadIdx.x & 63, b = threadIdx.x >> 6;
    for (int i = b; i < 64; i += 4) {
        const int r = sc == 1 ? r0 + i : r0 + a, c = sc == 1 ? c0 + a : c0 + i;
        const float v = r < R && c < C ? read_elem(in, elem, r * sr + c * sc) : 0.f;
        t[sc == 1 ? i : a][sc == 1 ? a : i] = v;
    }
    __syncthreads();
    const int planes = elem == TSC_ELEM_F32 ? 2 : 1;
    const float inv = elem == TSC_ELEM_F32 ? 1.f / wscale[0] : 1.f;
    for (int i = b; i < 64; i += 4) {
        const int r = r0 + i, c = c0 + a;
        if (r >= R || c >= Cp) continue;
        const float v = t[i][a];
        short *o = out + (long long)r * planes * Cp + c;
        if (elem == TSC_ELEM_F32) split(v * inv, o[0], o[Cp]);
        else o[0] = elem == TSC_ELEM_BF16 ? bits((__bf16)v) : bits((_Float16)v);
    }
}

__device__ __forceinline__ long long row_at(const TscRows &r, long long row) {
    return (row / r.inner) * r.outer_stride + (row % r.inner) * r.inner_stride;
}

// One wave a row: x[m] / s_m in planes of Dp elements, rows behind M (up to Mp) and rows without a loss zero; s_m to xscale.
__global__ __launch_bounds__(256) void pack_x_kernel(const TscRows x, int elem, int M, int Mp, int D, int Dp, const long long *targets,
                                                     long long ignore, short *out, float *xscale) {
    const int m = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (m >= Mp) return;
    const int planes = elem == TSC_ELEM_F32 ? 2 : 1;
    short *o = out + (long long)m * planes * Dp;
    const bool live = m < M && (!targets || targets[m] != ignore);
    const long long at = live ? row_at(x, m) : 0;
    float s = 1.f;
    if (elem == TSC_ELEM_F32) {
        float top = 0.f;
        if (live)
            for (int d = lane; d < D; d += 64) {
                const float v = fabsf(((const float *)x.data)[at + d]);
                top = v < __builtin_inff() ? fmaxf(top, v) : top;
            }
        for (int k = 32; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor(top, k));
        s = pow2_scale(top);
    }
    if (lane == 0 && m < M) xscale[m] = s;
    const float inv = 1.f / s;
    for (int d = lane; d < Dp; d += 64) {
        const bool in = live && d < D;
        if (elem == TSC_ELEM_F32) split(in ? ((const float *)x.data)[at + d] * inv : 0.f, o[d], o[Dp + d]);
        else o[d] = in ? ((const short *)x.data)[at + d] : (short)0;
    }
}

// rowf[m] = g_m s_m S (0 without a loss, NaN with a target outside the vocabulary), post[0] = 1 / S.  S = 1 for bf16, whose
// range is fp32's; for the fp16 planes the power of two that keeps |G'| = |rowf (p - [v = t])| within 2^14.
__global__ __launch_bounds__(1024) void row_factor_kernel(const float *g, const float *xscale, const long long *targets, long long ignore,
                                                          int V, int M, int f16, float *rowf, float *post) {
    __shared__ float s[17];
    float top = 0.f;
    if (f16)
        for (int m = threadIdx.x; m < M; m += 1024)
            if (targets[m] != ignore) {
                const float v = fabsf(g[m] * xscale[m]);
                top = v < __builtin_inff() ? fmaxf(top, v) : top;
            }
    for (int k = 32; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor(top, k));
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
        const float q = f16 ? pow2_scale(top) : 1.f;
        s[16] = 1.f / q;
        post[0] = q;
    }
    __syncthreads();
    for (int m = threadIdx.x; m < M; m += 1024) {
        const long long t = targets[m];
        rowf[m] = t == ignore ? 0.f : t < 0 || t >= V ? __builtin_nanf("") : g[m] * xscale[m] * s[16];
    }
}

// ------------------------------------------------------------------------------------------------ products
// Tiles of a launch: workgroups b and b + 8 share an XCD, so each XCD gets a run of neighbouring tiles, and within a run
// eight tiles of i go with every tile of j: the operands of the 32 tiles resident on an XCD fit its L2.
__device__ __forceinline__ void tile_of(int b, int ti, int tj, int &i, int &j) {
    const int n = ti * tj, x = b & 7, q = b >> 3;
    const int t = x * (n >> 3) + (x < (n & 7) ? x : (n & 7)) + q;
    const int g = t / (8 * tj), r = t - g * 8 * tj, gi = ti - g * 8 < 8 ? ti - g * 8 : 8;
    i = g * 8 + r % gi;
    j = r / gi;
}

// (reference, sum of 2^(l - reference)) of two sets of logits; a set of nothing but -inf is (-inf, 0)
__device__ __forceinline__ float2 merge(float2 a, float2 b) {
    const float t = fmaxf(a.x, b.x);
    return make_float2(t, t > -__builtin_inff() ? a.y * exp2_(a.x - t) + b.y * exp2_(b.x - t) : a.y + b.y);
}

struct LogitArgs {
    Operand W, x;       // i = v, j = m
    int nk, passes, ti, tj, v0;  // v0: first entry of the piece (tiles are counted from it)
    int M, V;
    const float *bias;   // -inf behind V
    const float *wscale, *xscale;  // null: 1
    const long long *targets;
    long long ignore;
    // forward
    float2 *part;        // [ti][M]: maximum, sum of exp2((l - maximum) log2 e)
    float *hit;          // [M]
    // backward
    const float *lse, *rowf;
    short *G;            // [Mp][ldg], second plane at gplane
    long long ldg, gplane;
    int Mp, f16, planes;
    float *dbias;        // [tj][ldg] or null
    const float *g;      // d(loss) of the rows
};

template <class C, bool F16, bool GRAD> __global__ __launch_bounds__(C::NT) void logits_kernel(const LogitArgs a) {
    typedef Gemm<C, false, F16> G;
    __shared__ __attribute__((aligned(16))) char lds[G::LDS_BYTES];
    int bi, bj;
    tile_of(blockIdx.x, a.ti, a.tj, bi, bj);
    const int i0 = a.v0 + bi * C::BI, j0 = bj * C::BJ;
    f32x16 acc[C::WI][C::WJ];
    G::run(a.W, a.x, i0, j0, 0, a.nk, a.passes, lds, acc);
    const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave / C::VJ, wi0 = i0 + wi * (C::WI * 32), wj0 = j0 + (wave % C::VJ) * (C::WJ * 32);
    const float ws = a.wscale ? a.wscale[0] : 1.f;
    float sc[C::WJ];
    long long tg[C::WJ];
#pragma unroll
    for (int q = 0; q < C::WJ; ++q) {
        const int m = wj0 + q * 32 + li, mc = m < a.M ? m : a.M - 1;
        sc[q] = a.xscale ? a.xscale[mc] * ws : 1.f;
        tg[q] = m < a.M ? a.targets[mc] : -1;
    }
    // logits in place of the products
#pragma unroll
    for (int p = 0; p < C::WI; ++p)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const f32x4 b = *(const f32x4 *)(a.bias + wi0 + p * 32 + 8 * s + 4 * lh);
#pragma unroll
            for (int q = 0; q < C::WJ; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[p][q][s * 4 + e] = fmaf(acc[p][q][s * 4 + e], sc[q], b[e]);
        }
    if constexpr (!GRAD) {
        __syncthreads();  // the operand tiles are no longer read: their place takes the waves' parts
        float2 *sm = (float2 *)lds;
#pragma unroll
        for (int q = 0; q < C::WJ; ++q) {
            float top = acc[0][q][0];
#pragma unroll
            for (int p = 0; p < C::WI; ++p)
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, acc[p][q][r]);
            top = fmaxf(top, __shfl_xor(top, 32));
            const float ref = top > -__builtin_inff() ? top * LOG2E : 0.f;  // nothing but -inf: the sum is 0
            float sum = 0.f;
#pragma unroll
            for (int p = 0; p < C::WI; ++p)
#pragma unroll
                for (int r = 0; r < 16; ++r) sum += exp2_(fmaf(acc[p][q][r], LOG2E, -ref));
            sum += __shfl_xor(sum, 32);
            const int jl = wj0 - j0 + q * 32 + li;
            if (lh == 0) sm[wi * C::BJ + jl] = make_float2(top > -__builtin_inff() ? ref : -__builtin_inff(), sum);
            // the target's logit, where it is one of this wave's
            const long long at = tg[q] - wi0;
            const bool mine = at >= 0 && at < C::WI * 32 && tg[q] < a.V && ((at >> 2) & 1) == lh;
            if (__builtin_amdgcn_ballot_w64(mine)) {
#pragma unroll
                for (int p = 0; p < C::WI; ++p)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (mine && at == p * 32 + block_row(r, lh)) a.hit[wj0 + q * 32 + li] = acc[p][q][r];
            }
        }
        __syncthreads();
        for (int jl = threadIdx.x; jl < C::BJ; jl += C::NT) {
            if (j0 + jl >= a.M) continue;
            float2 v = sm[jl];
#pragma unroll
            for (int w = 1; w < C::VI; ++w) {
                const float2 u = sm[w * C::BJ + jl];
                v = merge(v, u);
            }
            a.part[(long long)bi * a.M + j0 + jl] = v;
        }
    } else {
        float db[C::WI][16];
        if (a.dbias)
#pragma unroll
            for (int p = 0; p < C::WI; ++p)
#pragma unroll
                for (int r = 0; r < 16; ++r) db[p][r] = 0.f;
#pragma unroll
        for (int q = 0; q < C::WJ; ++q) {
            const int m = wj0 + q * 32 + li, mc = m < a.M ? m : a.M - 1;
            const bool live = m < a.M && tg[q] != a.ignore;
            const float lse2 = a.lse[mc] * LOG2E, f = a.rowf[mc], g = a.dbias ? a.g[mc] : 0.f;
            const long long at = tg[q] - wi0;
            short *row = a.G + (long long)m * a.ldg + (wi0 - a.v0) + 4 * lh;
#pragma unroll
            for (int p = 0; p < C::WI; ++p)
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    short h1[4], h2[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = s * 4 + e, v = p * 32 + block_row(r, lh);
                        float d = exp2_(fmaf(acc[p][q][r], LOG2E, -lse2));
                        d -= at == v ? 1.f : 0.f;
                        const float w = live ? d * f : 0.f;
                        if (a.dbias) db[p][r] += live ? d * g : 0.f;
                        if (!F16) h1[e] = bits((__bf16)w);
                        else if (a.planes == 2) split(w, h1[e], h2[e]);
                        else h1[e] = bits((_Float16)w);
                    }
                    if (m < a.Mp) {
                        *(s16x4 *)(row + p * 32 + 8 * s) = (s16x4){h1[0], h1[1], h1[2], h1[3]};
                        if (a.planes == 2) *(s16x4 *)(row + a.gplane + p * 32 + 8 * s) = (s16x4){h2[0], h2[1], h2[2], h2[3]};
                    }
                }
        }
        if (a.dbias) {  // over the wave's rows (lanes), then over the waves beside it
            __syncthreads();
            float *sm = (float *)lds;
#pragma unroll
            for (int p = 0; p < C::WI; ++p)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float v = db[p][r];
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor(v, o);
                    if (li == 0) sm[(wave % C::VJ) * C::BI + wi * (C::WI * 32) + p * 32 + block_row(r, lh)] = v;
                }
            __syncthreads();
            for (int il = threadIdx.x; il < C::BI; il += C::NT) {
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < C::VJ; ++w) v += sm[w * C::BI + il];
                a.dbias[(long long)bj * a.ldg + bi * C::BI + il] = v;
            }
        }
    }
}

// lse and loss of the rows from the tiles' parts: one wave a row
__global__ __launch_bounds__(256) void loss_kernel(const float2 *part, int n, int M, int V, const float *hit, const long long *targets,
                                                   long long ignore, float *loss, float *lse) {
    const int m = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (m >= M) return;
    float2 all = make_float2(-__builtin_inff(), 0.f);
    for (int i = lane; i < n; i += 64) all = merge(all, part[(long long)i * M + m]);
    for (int o = 32; o > 0; o >>= 1) all = merge(all, make_float2(__shfl_xor(all.x, o), __shfl_xor(all.y, o)));
    if (lane) return;
    const float l = (all.x + __log2f(all.y)) * LN2;
    const long long t = targets[m];
    lse[m] = l;
    loss[m] = t == ignore ? 0.f : t < 0 || t >= V ? __builtin_nanf("") : l - hit[m];
}

struct SumArgs {  // dx: C[z][i][j] = (or +=) the z-th part of the k-steps
    Operand A, B;
    int nk, per, passes, ti, tj, I, J, add;
    float *out;
};
template <class C, bool F16> __global__ __launch_bounds__(C::NT) void sum_kernel(const SumArgs a) {
    typedef Gemm<C, false, F16> G;
    __shared__ __attribute__((aligned(16))) char lds[G::LDS_BYTES];
    int bi, bj;
    tile_of(blockIdx.x, a.ti, a.tj, bi, bj);
    const int k0 = blockIdx.y * a.per, k1 = k0 + a.per < a.nk ? k0 + a.per : a.nk;
    f32x16 acc[C::WI][C::WJ];
    G::run(a.A, a.B, bi * C::BI, bj * C::BJ, k0, k1, a.passes, lds, acc);
    const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5, wave = threadIdx.x >> 6;
    const int wi0 = bi * C::BI + (wave / C::VJ) * (C::WI * 32), wj0 = bj * C::BJ + (wave % C::VJ) * (C::WJ * 32);
#pragma unroll
    for (int p = 0; p < C::WI; ++p)
#pragma unroll
        for (int q = 0; q < C::WJ; ++q)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int i = wi0 + p * 32 + block_row(r, lh), j = wj0 + q * 32 + li;
                if (i >= a.I || j >= a.J) continue;
                float *o = a.out + ((long long)blockIdx.y * a.I + i) * a.J + j;
                *o = a.add ? *o + acc[p][q][r] : acc[p][q][r];
            }
}
// dx[m][d] = sum over z, with the scales undone
__global__ __launch_bounds__(256) void dx_kernel(const float *part, int n, int M, int D, const float *wscale, const float *xscale,
                                                 const float *post, const long long *targets, long long ignore, int elem, void *dx) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)M * D) return;
    const int m = (int)(i / D);
    float v = 0.f;
    for (int z = 0; z < n; ++z) v += part[(long long)z * M * D + i];
    v *= post[0];
    if (wscale) v = v * wscale[0] / xscale[m];
    write_elem(dx, elem, i, targets[m] == ignore ? 0.f : v);
}

struct OutArgs {  // dW: both operands k-major
    Operand A, B;
    int nk, passes, ti, tj, I, J;
    const float *post;
    void *out;
    long long ld;
    int elem;
};
template <class C, bool F16> __global__ __launch_bounds__(C::NT) void out_kernel(const OutArgs a) {
    typedef Gemm<C, true, F16> G;
    __shared__ __attribute__((aligned(16))) char lds[G::LDS_BYTES];
    int bi, bj;
    tile_of(blockIdx.x, a.ti, a.tj, bi, bj);
    f32x16 acc[C::WI][C::WJ];
    G::run(a.A, a.B, bi * C::BI, bj * C::BJ, 0, a.nk, a.passes, lds, acc);
    const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5, wave = threadIdx.x >> 6;
    const int wi0 = bi * C::BI + (wave / C::VJ) * (C::WI * 32), wj0 = bj * C::BJ + (wave % C::VJ) * (C::WJ * 32);
    const float post = a.post[0];
#pragma unroll
    for (int p = 0; p < C::WI; ++p)
#pragma unroll
        for (int q = 0; q < C::WJ; ++q)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int i = wi0 + p * 32 + block_row(r, lh), j = wj0 + q * 32 + li;
                if (i < a.I && j < a.J) write_elem(a.out, a.elem, i * a.ld + j, acc[p][q][r] * post);
            }
}
__global__ __launch_bounds__(256) void dbias_kernel(const float *part, int n, long long ld, int J, int elem, void *out, long long at) {
    const int j = blockIdx.x * 256 + threadIdx.x;
    if (j >= J) return;
    float v = 0.f;
    for (int i = 0; i < n; ++i) v += part[i * ld + j];
    write_elem(out, elem, at + j, v);
}
__global__ void zero_elem_kernel(void *p, int elem, long long n) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i < n) write_elem(p, elem, i, 0.f);
}

inline int cdiv(long long a, long long b) { return (int)((a + b - 1) / b); }
inline long long up(long long a, long long b) { return (a + b - 1) / b * b; }

constexpr long long PIECE_BYTES = 1ll << 30;  // G of one piece of the vocabulary

}  // namespace

struct tsc_unembed {
    int D, V, elem, belem, planes, Dp, Vp, Vb;  // paddings: 64 for a product's k, 256 for the bias a tile reads
    long long sd, sv;                    // strides of W (elements): one of them is 1
    const void *W, *bias;                // borrowed
    short *Wt, *Wd;                      // [V][planes * Dp] and [D][planes * Vp]
    float *bias32, *wscale;
};

// ------------------------------------------------------------------------------------------------ handle
int tsc_unembed_destroy_(tsc_unembed *h) {
    if (!h) return TSC_OK;
    if (h->Wt) (void)hipFree(h->Wt);
    if (h->Wd) (void)hipFree(h->Wd);
    if (h->bias32) (void)hipFree(h->bias32);
    if (h->wscale) (void)hipFree(h->wscale);
    delete h;
    return TSC_OK;
}

void tsc_unembed_shape_(const tsc_unembed *h, int *elem, int *D, int *V) { *elem = h->elem; *D = h->D; *V = h->V; }

int tsc_unembed_refresh_(tsc_unembed *h, hipStream_t s) {
    hipLaunchKernelGGL(bias_kernel, dim3(cdiv(h->Vb, 256)), dim3(256), 0, s, h->bias, h->belem, h->V, h->Vb, h->bias32);
    if (h->elem == TSC_ELEM_F32) {
        hipLaunchKernelGGL(fill_kernel, dim3(1), dim3(256), 0, s, h->wscale, 0.f, 1ll);
        const long long rows = h->sv == 1 ? h->D : h->V, cols = h->sv == 1 ? h->V : h->D, ld = h->sv == 1 ? h->sd : h->sv;
        hipLaunchKernelGGL(absmax_kernel, dim3((int)(rows < 1024 ? rows : 1024)), dim3(1024), 0, s, (const float *)h->W, rows, cols, ld, (unsigned *)h->wscale);
        hipLaunchKernelGGL(wscale_kernel, dim3(1), dim3(1), 0, s, h->wscale);
    }
    hipLaunchKernelGGL(pack_w_kernel, dim3(h->Dp / 64, cdiv(h->V, 64)), dim3(256), 0, s, h->W, h->elem, h->sv, h->sd, h->V, h->D, h->Dp, h->wscale, h->Wt);
    hipLaunchKernelGGL(pack_w_kernel, dim3(h->Vp / 64, cdiv(h->D, 64)), dim3(256), 0, s, h->W, h->elem, h->sd, h->sv, h->D, h->V, h->Vp, h->wscale, h->Wd);
    TSC_HIP_CHECK(hipGetLastError());
    return TSC_OK;
}

int tsc_unembed_create_(tsc_unembed **out, int D, int V, int elem, const void *W, long long sd, long long sv, const void *bias, int belem, hipStream_t s) {
    tsc_unembed *h = new (std::nothrow) tsc_unembed();
    if (!h) return tsc_fail(TSC_ERR_HIP, "out of host memory");
    h->D = D; h->V = V; h->elem = elem; h->belem = belem; h->planes = elem == TSC_ELEM_F32 ? 2 : 1;
    h->Dp = (int)up(D, BK); h->Vp = (int)up(V, 256); h->Vb = h->Vp + 256;
    h->sd = sd; h->sv = sv; h->W = W; h->bias = bias;
    hipError_t e = hipMalloc((void **)&h->Wt, (size_t)V * h->planes * h->Dp * 2);
    if (e == hipSuccess) e = hipMalloc((void **)&h->Wd, (size_t)D * h->planes * h->Vp * 2);
    if (e == hipSuccess) e = hipMalloc((void **)&h->bias32, (size_t)h->Vb * 4);
    if (e == hipSuccess) e = hipMalloc((void **)&h->wscale, 256);
    int rc = e == hipSuccess ? tsc_unembed_refresh_(h, s) : tsc_fail(TSC_ERR_HIP, "hipMalloc of the unembedding's operands failed: %s", hipGetErrorString(e));
    if (rc != TSC_OK) {
        tsc_unembed_destroy_(h);
        return rc;
    }
    *out = h;
    return TSC_OK;
}

// ------------------------------------------------------------------------------------------------ launches
namespace {

// What a call keeps in its workspace, in this order (each part starts at a multiple of 256 bytes)
struct Plan {
    int Mp, tile, bi, bj, ti, tj;      // logits: i = v (of a piece), j = m
    int Vc, pieces;                    // backward: entries of a piece
    int z, per;                        // dx: parts of a piece's k-steps, k-steps of a part
    long long xp, xscale, part, hit, rowf, post, g, db, dx, bytes;
};
int tile_for(long long I, long long J) {
    if (J <= 64) return 2;
    return (long long)cdiv(I, 256) * cdiv(J, 256) >= 256 ? 0 : 1;  // the large tile once it fills the chip
}
void tile_size(int t, int &bi, int &bj) {
    bi = t == 0 ? 256 : 128;
    bj = t == 0 ? 256 : t == 1 ? 128 : 64;
}
Plan plan(const tsc_unembed *h, long long M, bool backward, bool want_x, bool want_b) {
    Plan p{};
    p.Mp = (int)up(M, BK);
    p.Vc = h->Vp;
    if (backward) {
        const long long fit = PIECE_BYTES / (2ll * h->planes * p.Mp) / 256 * 256;
        p.Vc = (int)(fit < 256 ? 256 : fit < h->Vp ? fit : h->Vp);
    }
    p.pieces = cdiv(h->V, p.Vc);
    p.tile = tile_for(p.Vc < h->V ? p.Vc : h->V, M);
    tile_size(p.tile, p.bi, p.bj);
    p.ti = cdiv(p.Vc < h->V ? p.Vc : h->V, p.bi);
    p.tj = cdiv(M, p.bj);
    long long at = 0;
    auto take = [&](long long n) { const long long q = at; at = up(at + n, 256); return q; };
    p.xp = take(2ll * h->planes * p.Mp * h->Dp);
    p.xscale = take(4 * M);
    if (!backward) {
        p.part = take(8ll * p.ti * M);
        p.hit = take(4 * M);
    } else {
        p.rowf = take(4 * M);
        p.post = take(4);
        p.g = take(2ll * h->planes * p.Mp * p.Vc);
        if (want_b) p.db = take(4ll * p.tj * p.Vc);
        if (want_x) {
            const int nk = p.Vc / BK, t = tile_for(M, h->D) == 0 ? 0 : 1;
            int bi, bj;
            tile_size(t, bi, bj);
            const long long tiles = (long long)cdiv(M, bi) * cdiv(h->D, bj);
            long long z = cdiv(t == 0 ? 256 : 512, tiles);
            if (z > nk / 8) z = nk / 8;
            if (z < 1) z = 1;
            p.per = cdiv(nk, z);
            p.z = cdiv(nk, p.per);
            p.dx = take(4ll * p.z * M * h->D);
        }
    }
    p.bytes = at;
    return p;
}

template <bool F16, bool GRAD> int launch_logits(int tile, const LogitArgs &a, hipStream_t s) {
    const dim3 grid(a.ti * a.tj);
    if (tile == 0) hipLaunchKernelGGL((logits_kernel<TileLarge, F16, GRAD>), grid, dim3(TileLarge::NT), 0, s, a);
    else if (tile == 1) hipLaunchKernelGGL((logits_kernel<TileMedium, F16, GRAD>), grid, dim3(TileMedium::NT), 0, s, a);
    else hipLaunchKernelGGL((logits_kernel<TileSkinny, F16, GRAD>), grid, dim3(TileSkinny::NT), 0, s, a);
    TSC_HIP_CHECK(hipGetLastError());
    return TSC_OK;
}
LogitArgs logit_args(const tsc_unembed *h, const Plan &p, char *ws, int M, const long long *targets, long long ignore) {
    LogitArgs a{};
    a.W = {h->Wt, (long long)h->planes * h->Dp, h->Dp, h->V};
    a.x = {(const short *)(ws + p.xp), (long long)h->planes * h->Dp, h->Dp, M};
    a.nk = h->Dp / BK; a.passes = h->planes == 2 ? 3 : 1;
    a.ti = p.ti; a.tj = p.tj; a.M = M; a.V = h->V;
    a.bias = h->bias32;
    a.wscale = h->planes == 2 ? h->wscale : nullptr;
    a.xscale = h->planes == 2 ? (const float *)(ws + p.xscale) : nullptr;
    a.targets = targets; a.ignore = ignore; a.planes = h->planes;
    return a;
}

}  // namespace

size_t tsc_unembed_workspace_(const tsc_unembed *h, long long M, int backward, int want_x, int want_b) {
    return M < 1 ? 0 : (size_t)plan(h, M, backward, want_x, want_b).bytes;
}

int tsc_launch_unembed_loss(const tsc_unembed *h, const TscRows &x, int M, const long long *targets, long long ignore, float *loss,
                            float *lse, char *ws, hipStream_t s) {
    const Plan p = plan(h, M, false, false, false);
    hipLaunchKernelGGL(pack_x_kernel, dim3(cdiv(p.Mp, 4)), dim3(256), 0, s, x, h->elem, M, p.Mp, h->D, h->Dp, (const long long *)nullptr, ignore,
                       (short *)(ws + p.xp), (float *)(ws + p.xscale));
    LogitArgs a = logit_args(h, p, ws, M, targets, ignore);
    a.part = (float2 *)(ws + p.part);
    a.hit = (float *)(ws + p.hit);
    const int rc = h->elem == TSC_ELEM_BF16 ? launch_logits<false, false>(p.tile, a, s) : launch_logits<true, false>(p.tile, a, s);
    if (rc) return rc;
    hipLaunchKernelGGL(loss_kernel, dim3(cdiv(M, 4)), dim3(256), 0, s, a.part, p.ti, M, h->V, a.hit, targets, ignore, loss, lse);
    TSC_HIP_CHECK(hipGetLastError());
    return TSC_OK;
}

int tsc_launch_unembed_backward(const tsc_unembed *h, const float *g, const TscRows &x, int M, const long long *targets, long long ignore,
                                const float *lse, void *dx, void *dW, void *db, char *ws, hipStream_t s) {
    const bool f16 = h->elem != TSC_ELEM_BF16;
    if (M == 0) {
        if (dW) hipLaunchKernelGGL(zero_elem_kernel, dim3(cdiv((long long)h->D * h->V, 256)), dim3(256), 0, s, dW, h->elem, (long long)h->D * h->V);
        if (db) hipLaunchKernelGGL(zero_elem_kernel, dim3(cdiv(h->V, 256)), dim3(256), 0, s, db, h->belem, (long long)h->V);
        TSC_HIP_CHECK(hipGetLastError());
        return TSC_OK;
    }
    const Plan p = plan(h, M, true, dx != nullptr, db != nullptr);
    short *xp = (short *)(ws + p.xp), *G = (short *)(ws + p.g);
    float *xscale = (float *)(ws + p.xscale), *rowf = (float *)(ws + p.rowf), *post = (float *)(ws + p.post), *dxp = (float *)(ws + p.dx);
    hipLaunchKernelGGL(pack_x_kernel, dim3(cdiv(p.Mp, 4)), dim3(256), 0, s, x, h->elem, M, p.Mp, h->D, h->Dp, targets, ignore, xp, xscale);
    hipLaunchKernelGGL(row_factor_kernel, dim3(1), dim3(1024), 0, s, g, xscale, targets, ignore, h->V, M, f16, rowf, post);
    LogitArgs a = logit_args(h, p, ws, M, targets, ignore);
    a.lse = lse; a.rowf = rowf; a.G = G; a.ldg = p.Vc; a.gplane = (long long)p.Mp * p.Vc; a.Mp = p.Mp; a.f16 = f16;
    a.dbias = db ? (float *)(ws + p.db) : nullptr;
    a.g = g;
    const long long xld = (long long)h->planes * h->Dp;
    for (int c = 0; c < p.pieces; ++c) {
        const int v0 = c * p.Vc, nv = h->V - v0 < p.Vc ? h->V - v0 : p.Vc, nvp = (int)up(nv, p.bi);
        a.v0 = v0;
        a.ti = nvp / p.bi;
        int rc = f16 ? launch_logits<true, true>(p.tile, a, s) : launch_logits<false, true>(p.tile, a, s);
        if (rc) return rc;
        if (db) hipLaunchKernelGGL(dbias_kernel, dim3(cdiv(nv, 256)), dim3(256), 0, s, a.dbias, p.tj, a.ldg, nv, h->belem, db, (long long)v0);
        if (dx) {
            SumArgs q{};
            q.A = {G, p.Vc, a.gplane, M};
            q.B = {h->Wd + v0, (long long)h->planes * h->Vp, h->Vp, h->D};
            q.nk = nvp / BK; q.per = p.per; q.passes = a.passes; q.I = M; q.J = h->D; q.add = c > 0; q.out = dxp;
            const int t = tile_for(M, h->D) == 0 ? 0 : 1;
            int bi, bj;
            tile_size(t, bi, bj);
            q.ti = cdiv(M, bi); q.tj = cdiv(h->D, bj);
            const dim3 grid(q.ti * q.tj, c == 0 ? p.z : cdiv(q.nk, p.per));
            if (t == 0) {
                if (f16) hipLaunchKernelGGL((sum_kernel<TileLarge, true>), grid, dim3(TileLarge::NT), 0, s, q);
                else hipLaunchKernelGGL((sum_kernel<TileLarge, false>), grid, dim3(TileLarge::NT), 0, s, q);
            } else {
                if (f16) hipLaunchKernelGGL((sum_kernel<TileMedium, true>), grid, dim3(TileMedium::NT), 0, s, q);
                else hipLaunchKernelGGL((sum_kernel<TileMedium, false>), grid, dim3(TileMedium::NT), 0, s, q);
            }
        }
        if (dW) {
            OutArgs q{};
            const Operand X = {xp, xld, h->Dp, h->D}, Gk = {G, p.Vc, a.gplane, nv};
            const bool by_d = h->sv == 1;  // dW is dense in W's order: [D][V] or [V][D]
            q.A = by_d ? X : Gk;
            q.B = by_d ? Gk : X;
            q.nk = p.Mp / BK; q.passes = a.passes; q.I = by_d ? h->D : nv; q.J = by_d ? nv : h->D;
            q.post = post; q.elem = h->elem; q.ld = by_d ? h->V : h->D;
            const long long first = by_d ? v0 : (long long)v0 * h->D;
            q.out = (char *)dW + first * (h->elem == TSC_ELEM_F32 ? 4 : 2);
            const int t = tile_for(q.I, q.J) == 0 ? 0 : 1;
            int bi, bj;
            tile_size(t, bi, bj);
            q.ti = cdiv(q.I, bi); q.tj = cdiv(q.J, bj);
            const dim3 grid(q.ti * q.tj);
            if (t == 0) {
                if (f16) hipLaunchKernelGGL((out_kernel<TileLarge, true>), grid, dim3(TileLarge::NT), 0, s, q);
                else hipLaunchKernelGGL((out_kernel<TileLarge, false>), grid, dim3(TileLarge::NT), 0, s, q);
            } else {
                if (f16) hipLaunchKernelGGL((out_kernel<TileMedium, true>), grid, dim3(TileMedium::NT), 0, s, q);
                else hipLaunchKernelGGL((out_kernel<TileMedium, false>), grid, dim3(TileMedium::NT), 0, s, q);
            }
        }
        TSC_HIP_CHECK(hipGetLastError());
    }
    if (dx) hipLaunchKernelGGL(dx_kernel, dim3(cdiv((long long)M * h->D, 256)), dim3(256), 0, s, dxp, p.z, M, h->D,
                               a.wscale, a.xscale, post, targets, ignore, h->elem, dx);
    TSC_HIP_CHECK(hipGetLastError());
    return TSC_OK;
}
