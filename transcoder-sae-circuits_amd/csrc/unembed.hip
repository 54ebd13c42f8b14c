// Cross entropy of a row's unembedding, without the [rows, vocabulary] logits, and its gradient (gfx950).
//
//   l[m][v] = sum_d x[m][d] W[d][v] + b[v]          lse[m] = log sum_v exp l[m][v]
//   loss[m] = lse[m] - l[m][t_m]                    (0 where t_m is the ignored index)
//   G[m][v] = g_m (exp(l[m][v] - lse[m]) - [v = t_m])        dx = G W^T      dW = x^T G      db = sum_m G
//
// Bound by the matrix pipe: 2 M D V operations forward; backward makes the logits again (2 M D V) and adds two products of
// the same size.  Forward: the tile of logits stays in the accumulators, only its rows' maximum and sum of exponentials leave
// the workgroup.  Backward, in pieces of the vocabulary: G of a piece goes to the workspace in 16 bits (fp32: two fp16
// planes), and the two products read it from there.  One entry carries most of a row of G, the target's, so what is lost of
// it in 16 bits is lost of the row's gradient: as much as the result's own rounding loses on the average of many rows, up to
// twice that in a single one.  So what the rounding took of it is kept as a number a row; dx adds it times W's row t, and dW's
// column t adds it times the row (target_rows_kernel).  Up to 64 rows of 16-bit elements, whose time is W's way from memory,
// keep what the rounding took of all entries (rows 2 m: G_m, 2 m + 1: its remainder), and both products run over twice as many
// rows.
#include <mutex>
#include <new>
#include <type_traits>

#include "unembed_gemm.h"

using namespace unembed_gemm;

namespace {

constexpr int FEW_ROWS = 64;  // a tile's rows where W's way from memory is what takes the time
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

// power of two s that brings a magnitude into [2^14, 2^15) when divided by s (1 for 0, infinities and NaN)
__device__ __forceinline__ float pow2_scale(float top) {
    if (!(top > 0.f) || !(top < __builtin_inff())) return 1.f;
    const int e = (int)(__float_as_uint(top) >> 23) - 14;  // biased exponent of s; 1: the smallest normal
    return __uint_as_float((unsigned)(e < 1 ? 1 : e) << 23);
}
// h1 + h2 = v (unembed_gemm.h).  A value that fp16 does not hold (it is not finite, or NaN) goes to h1 alone.
__device__ __forceinline__ void split(float v, short &h1, short &h2) {
    const _Float16 a = (_Float16)v;
    h1 = bits(a);
    h2 = fabsf((float)a) < __builtin_inff() ? bits((_Float16)(v - (float)a)) : (short)0;
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

// 16 bytes of elements at an element's alignment
template <class T> struct __attribute__((packed, aligned(sizeof(T)))) Vec { T e[16 / sizeof(T)]; };

// out[r][c] = in[r * sr + c * sc], c < C, zero up to the pitch Cp; one of sr, sc is 1.  64 x 64 elements a workgroup, 16 bytes
// a lane on both sides.  T: float (two planes) or the bits of a 16-bit type.
template <class T> __global__ __launch_bounds__(256) void pack_w_kernel(const T *in, long long sr, long long sc, int R, int C, int Cp,
                                                                        const float *wscale, short *out) {
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int VE = 16 / sizeof(T), PER = 64 / VE;
    __shared__ T t[64][64 + 4 / sizeof(T)];
    const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
    for (int i = threadIdx.x; i < 64 * PER; i += 256) {
        const int line = i / PER, at = i % PER * VE;  // along the axis of stride 1
        const int r = r0 + (sc == 1 ? line : at), c = c0 + (sc == 1 ? at : line);
        const T *p = in + r * sr + c * sc;
        if (sc == 1 ? r < R && c + VE <= C : c < C && r + VE <= R) {
            const Vec<T> v = *(const Vec<T> *)p;
#pragma unroll
            for (int e = 0; e < VE; ++e) t[sc == 1 ? line : at + e][sc == 1 ? at + e : line] = v.e[e];
        } else {
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const bool ok = sc == 1 ? r < R && c + e < C : c < C && r + e < R;
                t[sc == 1 ? line : at + e][sc == 1 ? at + e : line] = ok ? p[e] : (T)0;
            }
        }
    }
    __syncthreads();
    const float inv = SPLIT ? 1.f / wscale[0] : 1.f;
    for (int i = threadIdx.x; i < 64 * 8; i += 256) {  // 8 elements of a row (Cp is a multiple of 64)
        const int line = i / 8, at = i % 8 * 8, r = r0 + line, c = c0 + at;
        if (r >= R) continue;
        s16x8 h1, h2;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            short x, y = 0;
            if constexpr (SPLIT) split(t[line][at + e] * inv, x, y);
            else x = t[line][at + e];
            h1[e] = x;
            h2[e] = y;
        }
        short *o = out + (SPLIT ? (long long)r * 2 * Cp + (c >> 5) * 64 + (c & 31) : (long long)r * Cp + c);
        *(s16x8 *)o = h1;
        if constexpr (SPLIT) *(s16x8 *)(o + 32) = h2;
    }
}

__device__ __forceinline__ long long row_at(const TscRows &r, long long row) {
    return (row / r.inner) * r.outer_stride + (row % r.inner) * r.inner_stride;
}

// One wave a row, n rows one after the other: x[m] / s_m, pitch Dp, rows behind M (up to Mp) and rows without a loss zero; s_m
// to xscale (fp32); `copies` of each row one after the other.  With gtop: it takes the largest |g_m| s_m, from which G is scaled (a
// maximum does not depend on the order of the atomics; one a workgroup, only where it raises the value).  A row of fp32 without
// elements has no scale (0 in xscale, see row_scale) and must not count as one of scale 1, 2^13 times that of common rows: its
// |g_m| goes to gtop[1], which counts where there are no others.
template <class T> __global__ __launch_bounds__(256) void pack_x_kernel(const TscRows x, int M, int Mp, int D, int Dp, int n, int copies, const long long *targets,
                                                                        long long ignore, const float *g, short *out, float *xscale, unsigned *gtop) {
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int VE = 16 / sizeof(T);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float most[2] = {0.f, 0.f};
    for (int m = (blockIdx.x * 4 + wave) * n, end = m + n < Mp ? m + n : Mp; m < end; ++m) {
        short *o = out + (long long)m * (SPLIT ? 2 : copies) * Dp;
        const bool live = m < M && (!targets || targets[m] != ignore);
        const T *p = (const T *)x.data + (live ? row_at(x, m) : 0);
        float s = 1.f;
        bool empty = false;
        auto load = [&](int d) __attribute__((always_inline)) {
            Vec<T> v;
            if (live && d + VE <= D) {
                v = *(const Vec<T> *)(p + d);
            } else {
#pragma unroll
                for (int e = 0; e < VE; ++e) v.e[e] = live && d + e < D ? p[d + e] : (T)0;
            }
            return v;
        };
        constexpr int HELD = SPLIT ? 4 : 1;  // vectors a lane that are read once, all at the same time (for few rows that is what counts)
        Vec<T> held[HELD];
#pragma unroll
        for (int i = 0; i < HELD; ++i) held[i] = load((i * 64 + lane) * VE);
        if constexpr (SPLIT) {
            float top = 0.f;
            auto take = [&](const Vec<T> &v) __attribute__((always_inline)) {
#pragma unroll
                for (int e = 0; e < VE; ++e) top = fabsf(v.e[e]) < __builtin_inff() ? fmaxf(top, fabsf(v.e[e])) : top;
            };
#pragma unroll
            for (int i = 0; i < HELD; ++i) take(held[i]);
            for (int d = (HELD * 64 + lane) * VE; d < D; d += 64 * VE) take(load(d));
            for (int k = 32; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor(top, k));
            s = pow2_scale(top);
            empty = gtop && live && top == 0.f;
            if (lane == 0 && m < M) xscale[m] = empty ? 0.f : s;
        }
        if (gtop && live) {
            const float v = fabsf(g[m] * s);
            if (v < __builtin_inff()) {
                if (empty) most[1] = fmaxf(most[1], v);
                else most[0] = fmaxf(most[0], v);
            }
        }
        const float inv = 1.f / s;
        auto store = [&](int d, const Vec<T> &v) __attribute__((always_inline)) {
            if constexpr (SPLIT) {
                s16x4 h1, h2;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    short a, b;
                    split(v.e[e] * inv, a, b);
                    h1[e] = a;
                    h2[e] = b;
                }
                short *q = o + (d >> 5) * 64 + (d & 31);
                *(s16x4 *)q = h1;
                *(s16x4 *)(q + 32) = h2;
            } else {
                for (int k = 0; k < copies; ++k) *(Vec<T> *)(o + (long long)k * Dp + d) = v;
            }
        };
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if ((i * 64 + lane) * VE < Dp) store((i * 64 + lane) * VE, held[i]);
        for (int d = (HELD * 64 + lane) * VE; d < Dp; d += 64 * VE) store(d, load(d));
    }
    if (!gtop) return;
    __shared__ float all[2][4];
    if (lane == 0)
        for (int i = 0; i < 2; ++i) all[i][wave] = most[i];
    __syncthreads();
    if (threadIdx.x >= (SPLIT ? 2 : 1)) return;
    const float *a = all[threadIdx.x];
    const unsigned top = __float_as_uint(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])));
    if (top > __atomic_load_n(gtop + threadIdx.x, __ATOMIC_RELAXED)) atomicMax(gtop + threadIdx.x, top);
}

// G' = G s_m S in 16 bits: S is 1 for bf16, whose range is fp32's, and for the fp16 planes the power of two that keeps |G'| =
// |g_m| s_m S |p - [v = t]| below 2^15.  This is 1 / S.
__device__ __forceinline__ float g_unit(const unsigned *gtop) { return gtop ? pow2_scale(__uint_as_float(gtop[0] ? gtop[0] : gtop[1])) : 1.f; }
// s_m of a row of x in the backward pass.  One without elements is 0 at any scale; it takes the power of two that brings |g_m| s_m
// next to the largest of the others, so that its entries of G are held like theirs.
__device__ __forceinline__ float row_scale(float s, const unsigned *gtop, float g) {
    if (s > 0.f || !gtop[0] || !(fabsf(g) > 0.f) || !(fabsf(g) < __builtin_inff())) return s > 0.f ? s : 1.f;
    const int e = (int)(__float_as_uint(__uint_as_float(gtop[0]) / fabsf(g)) >> 23);
    return __uint_as_float((unsigned)(e < 1 ? 1 : e > 254 ? 254 : e) << 23);
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

__device__ __forceinline__ void clear(f32x16 &v) {
#pragma unroll
    for (int r = 0; r < 16; ++r) v[r] = 0.f;
}
// (reference, sum of 2^(l - reference)) of two sets of logits; a set of nothing but -inf is (-inf, 0)
__device__ __forceinline__ float2 merge(float2 a, float2 b) {
    const float t = fmaxf(a.x, b.x);
    return make_float2(t, t > -__builtin_inff() ? a.y * exp2_(a.x - t) + b.y * exp2_(b.x - t) : a.y + b.y);
}

struct LogitArgs {
    Operand W, x;
    int nk;
    int nm, ns, nv, v0;  // blocks of rows, streams of a block, tiles of the vocabulary (counted from entry v0)
    int M, V;
    const float *bias;                  // -inf behind V
    const float *wscale, *xscale;       // null: 1
    const long long *targets;
    long long ignore;
    // forward
    float2 *part;        // [ns][M]: reference, sum of 2^(l log2 e - reference)
    float *hit;          // [M]
    // backward
    const float *lse, *g;    // of the rows: kept, and d(loss)
    const unsigned *gtop;    // g_unit, row_scale
    short *G;            // [Mp][PLANES * ldg]
    long long ldg;
    int rest;            // of a row's remainder behind the row (elements); FEW rows of 16-bit elements
    float *left;         // or [M]: the remainder of the target's entry alone; more of them; null: not wanted
    int Mp;              // rows of G that are wanted (32 at a time are written)
    float *dbias;        // [parts of the rows][ldg] or null
};

// Forward, i = v, j = m: a lane holds 16 WI logits of one row for each of its WJ columns.  The workgroup walks every ns-th
// tile of the vocabulary for one block of rows.  The first tile's maximum becomes the row's reference; from then on a tile
// costs an fma, an exponential and an add an element: sums of 2^(l - reference) are exact enough whatever the later maxima
// are, as long as nothing overflows (the tile is then repeated with its own maximum) -- what underflows is below 2^-126 of a
// term that is already in the sum.  (fp32 at LARGE: 13 registers do not fit; the loop over k touches none of them, a tile's end
// reads eight back.)
template <class C, bool F16, bool SPLIT> __global__ __launch_bounds__(C::NT, C::OCC) void loss_logits_kernel(const LogitArgs a) {
    typedef Gemm<C, false, F16, SPLIT ? 2 : 1> G;
    __shared__ __attribute__((aligned(16))) char lds[G::LDS_BYTES];
    int bj, st;
    tile_of(blockIdx.x, a.nm, a.ns, bj, st);
    const int j0 = bj * C::BJ;
    const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave / C::VJ, wj0 = j0 + (wave % C::VJ) * (C::WJ * 32);
    float sc[C::WJ], ref[C::WJ], sum[C::WJ];
    int tg[C::WJ];
#pragma unroll
    for (int q = 0; q < C::WJ; ++q) {
        const int m = wj0 + q * 32 + li, mc = m < a.M ? m : a.M - 1;
        sc[q] = SPLIT ? a.xscale[mc] * a.wscale[0] : 1.f;
        const long long t = a.targets[mc];
        tg[q] = m < a.M && t >= 0 && t < a.V ? (int)t : -1;
        ref[q] = -__builtin_inff();
        sum[q] = 0.f;
    }
    auto tile = [&](int t) { return TileAt{(st + t * a.ns) * C::BI, j0}; };
    auto first = [&](int t) { return (st + t * a.ns) * C::BI + wi * (C::WI * 32); };
    auto begin = [&](int t, f32x16 (&acc)[C::WI][C::WJ]) __attribute__((always_inline)) {
        const float *b0 = a.bias + first(t) + 4 * lh;
#pragma unroll
        for (int p = 0; p < C::WI; ++p)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const f32x4 b = SPLIT ? (f32x4){0.f, 0.f, 0.f, 0.f} : *(const f32x4 *)(b0 + p * 32 + 8 * s);
#pragma unroll
                for (int q = 0; q < C::WJ; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[p][q][s * 4 + e] = b[e];  // products start from the bias
            }
    };
    auto done = [&](int t, f32x16 (&acc)[C::WI][C::WJ]) __attribute__((always_inline)) {
        const int wi0 = first(t);
        if (SPLIT) {
#pragma unroll
            for (int p = 0; p < C::WI; ++p) {
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const f32x4 b = *(const f32x4 *)(a.bias + wi0 + 4 * lh + p * 32 + 8 * s);
#pragma unroll
                    for (int q = 0; q < C::WJ; ++q)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[p][q][s * 4 + e] = fmaf(acc[p][q][s * 4 + e], sc[q], b[e]);
                }
                __builtin_amdgcn_sched_barrier(0);  // (block by block: together the temporaries spill)
            }
        }
#pragma unroll
        for (int q = 0; q < C::WJ; ++q) {
            float part[4];
            auto add = [&](float r) {
                part[0] = part[1] = part[2] = part[3] = 0.f;
#pragma unroll
                for (int p = 0; p < C::WI; ++p) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) part[e & 3] += exp2_(fmaf(acc[p][q][e], LOG2E, -r));
                    __builtin_amdgcn_sched_barrier(0);
                }
                return (part[0] + part[1]) + (part[2] + part[3]);
            };
            float s = add(ref[q] > -__builtin_inff() ? ref[q] : 0.f);
            const bool ok = ref[q] > -__builtin_inff() && s < 0x1p100f;
            if (__builtin_amdgcn_ballot_w64(!ok)) {
                float top = acc[0][q][0];
#pragma unroll
                for (int p = 0; p < C::WI; ++p)
#pragma unroll
                    for (int e = 0; e < 16; ++e) top = fmaxf(top, acc[p][q][e]);
                const float r = ok ? ref[q] : top > -__builtin_inff() ? fmaxf(ref[q], top * LOG2E) : ref[q];
                s = add(r > -__builtin_inff() ? r : 0.f);  // (nothing but -inf so far: the sum is 0)
                if (ref[q] > -__builtin_inff()) sum[q] *= exp2_(ref[q] - r);
                ref[q] = r;
            }
            sum[q] += s;
            // the target's logit, where it is one of this wave's
            const int at = tg[q] - wi0 - 4 * lh;  // a lane's entries: block_row(r, 0) of each block
            const bool mine = tg[q] >= 0 && at >= 0 && at < C::WI * 32 && (at & 4) == 0;
            if (__builtin_amdgcn_ballot_w64(mine)) {
#pragma unroll
                for (int p = 0; p < C::WI; ++p)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (mine && at == p * 32 + block_row(r, 0)) a.hit[wj0 + q * 32 + li] = acc[p][q][r];
            }
        }
    };
    G::run(a.W, a.x, (a.nv - st + a.ns - 1) / a.ns, tile, 0, a.nk, lds, begin, done);
    __syncthreads();  // the operand tiles are no longer read: their place takes the waves' parts
    float2 *sm = (float2 *)lds;
#pragma unroll
    for (int q = 0; q < C::WJ; ++q) {
        const float2 v = merge(make_float2(ref[q], sum[q]), make_float2(__shfl_xor(ref[q], 32), __shfl_xor(sum[q], 32)));
        if (lh == 0) sm[wi * C::BJ + wj0 - j0 + q * 32 + li] = v;
    }
    __syncthreads();
    for (int jl = threadIdx.x; jl < C::BJ; jl += C::NT) {
        if (j0 + jl >= a.M) continue;
        float2 v = sm[jl];
#pragma unroll
        for (int w = 1; w < C::VI; ++w) v = merge(v, sm[w * C::BJ + jl]);
        a.part[(long long)st * a.M + j0 + jl] = v;
    }
}

// Backward, i = m, j = v: a lane holds one entry of the vocabulary and 16 WI rows of it, so db is a sum over its registers,
// and two neighbouring lanes exchange halves to store two entries of a row each.  The rows' constants lie in LDS.
template <class C, bool F16, bool SPLIT> __global__ __launch_bounds__(C::NT, C::OCC) void grad_logits_kernel(const LogitArgs a) {
    typedef Gemm<C, false, F16, SPLIT ? 2 : 1> G;
    __shared__ __attribute__((aligned(16))) char lds[G::LDS_BYTES];
    __shared__ __attribute__((aligned(16))) float r_lse[C::BI], r_f[C::BI], r_sc[SPLIT ? C::BI : 4], r_inv[SPLIT ? C::BI : 4];
    __shared__ __attribute__((aligned(16))) int r_t[C::BI];
    int bi, st;
    tile_of(blockIdx.x, a.nm, a.ns, bi, st);
    const int i0 = bi * C::BI;
    const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave / C::VJ, wr = wi * (C::WI * 32), wj = (wave % C::VJ) * (C::WJ * 32);
    const float unit = 1.f / g_unit(a.gtop);
    for (int i = threadIdx.x; i < C::BI; i += C::NT) {
        const int m = i0 + i, mc = m < a.M ? m : a.M - 1;
        const long long t = a.targets[mc];
        const bool live = m < a.M && t != a.ignore;
        // rows without a loss: every exponential is 2^-inf = 0
        r_lse[i] = live ? a.lse[mc] * LOG2E : __builtin_inff();
        const bool known = t >= 0 && t < a.V;
        const float s = SPLIT ? row_scale(a.xscale[mc], a.gtop, a.g[mc]) : 1.f;
        r_f[i] = !live ? 0.f : known ? a.g[mc] * s * unit : __builtin_nanf("");
        r_t[i] = live && known ? (int)t - a.v0 : -1;
        if (SPLIT) {
            r_sc[i] = a.xscale[mc] * a.wscale[0] * LOG2E;  // (0 for a row without elements, whose products are 0)
            r_inv[i] = 1.f / s;
        }
    }
    __syncthreads();
    const unsigned sel = lane & 1 ? 0x03020706u : 0x05040100u;  // of (neighbour's pair : own pair)
    auto tile = [&](int t) { return TileAt{i0, a.v0 + (st + t * a.ns) * C::BJ}; };
    auto first = [&](int t) { return (st + t * a.ns) * C::BJ + wj; };  // in the piece
    // (products that start from the bias would save an add an element, but make the compiler spill the sums)
    auto begin = [&](int, f32x16 (&acc)[C::WI][C::WJ]) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < C::WI; ++p)
#pragma unroll
            for (int q = 0; q < C::WJ; ++q) clear(acc[p][q]);
    };
    auto done = [&](int t, f32x16 (&acc)[C::WI][C::WJ]) __attribute__((always_inline)) {
        const int v = first(t);
        // blocks that hold a target: bit q * WI + p
        unsigned hot = 0;
#pragma unroll
        for (int i = 0; i < C::WI * 32; i += 64) {
            const int at = r_t[wr + i + (i + lane < C::WI * 32 ? lane : 0)] - v;
#pragma unroll
            for (int q = 0; q < C::WJ; ++q) {
                const unsigned long long m = __builtin_amdgcn_ballot_w64(at >= q * 32 && at < q * 32 + 32);
                hot |= ((unsigned)m ? 1u << (q * C::WI + i / 32) : 0u) | (i + 32 < C::WI * 32 && (m >> 32) ? 2u << (q * C::WI + i / 32) : 0u);
            }
        }
        constexpr int PL = SPLIT ? 2 : 1;
        constexpr bool REST = !SPLIT && C::BI <= FEW_ROWS;
        long long ld2 = a.ldg * 2 * PL;
        asm volatile("" : "+s"(ld2));  // (else the distances of all rows are computed once and spilled)
        // a lane stores row (lane & 1) of a pair of rows, columns col & ~1 and the next
        char *base = (char *)(a.G + ((long long)(i0 + wr) * a.ldg + v) * PL);
        const unsigned lane_at = (unsigned)((4 * lh + (lane & 1)) * (int)a.ldg * PL + (li & ~1)) * 2u;
        float db[C::WJ], b2[C::WJ];
#pragma unroll
        for (int q = 0; q < C::WJ; ++q) {
            b2[q] = a.bias[a.v0 + v + q * 32 + li] * LOG2E;
            db[q] = 0.f;
        }
        // four rows (8 s .. of block p) by the wave's columns from block q0 on; again: once more, with the targets taken off
        auto quad = [&](auto again_, int p, int s, int q0, int q1) __attribute__((always_inline)) {
            constexpr bool AGAIN = decltype(again_)::value;
            int at = wr + p * 32 + 8 * s + 4 * lh;
            if (AGAIN) asm volatile("" : "+v"(at));  // (else everything of the first time is kept for the second, and spilled)
            const f32x4 l = *(const f32x4 *)&r_lse[at], f = *(const f32x4 *)&r_f[at];
            f32x4 sc, inv;
            if (SPLIT) sc = *(const f32x4 *)&r_sc[at], inv = *(const f32x4 *)&r_inv[at];
            char *row = base + (p * 32 + 8 * s) * ld2;
#pragma unroll
            for (int q = q0; q < q1; ++q) {
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = acc[p][q][s * 4 + e];
                    w[e] = exp2_(fmaf(x, SPLIT ? sc[e] : LOG2E, b2[q]) - l[e]);
                    if (AGAIN) {
                        const float hit = r_t[at + e] == v + q * 32 + li ? 1.f : 0.f;
                        w[e] -= hit;
                        db[q] -= SPLIT ? hit * f[e] * inv[e] : hit * f[e];
                    }
                    w[e] *= f[e];
                    if (!AGAIN) db[q] = SPLIT ? fmaf(w[e], inv[e], db[q]) : db[q] + w[e];
                }
                if constexpr (AGAIN && !SPLIT && !REST) {
                    if (a.left)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (r_t[at + e] == v + q * 32 + li) a.left[i0 + at + e] = w[e] - (F16 ? (float)(_Float16)w[e] : (float)(__bf16)w[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    auto put = [&](unsigned own, char *to) __attribute__((always_inline)) {
                        const unsigned other = __builtin_amdgcn_update_dpp(0, own, 0xB1, 0xF, 0xF, true);  // lane ^ 1
                        *(unsigned *)(to + e * ld2 + q * 64 * PL + lane_at) = __builtin_amdgcn_perm(other, own, sel);
                    };
                    const f32x2 pair = {w[e], w[e + 1]};
                    if constexpr (F16) {
                        const f16x2 h = __builtin_convertvector(pair, f16x2);
                        put(__builtin_bit_cast(unsigned, h), row);
                        if constexpr (SPLIT) {  // h2 is held times 2048
                            const f32x2 r = {fmaf((float)h[0], -2048.f, pair[0] * 2048.f), fmaf((float)h[1], -2048.f, pair[1] * 2048.f)};
                            put(__builtin_bit_cast(unsigned, __builtin_convertvector(r, f16x2)), row + 64);
                        } else if constexpr (REST) put(__builtin_bit_cast(unsigned, __builtin_convertvector(pair - __builtin_convertvector(h, f32x2), f16x2)), row + 2 * a.rest);
                    } else {
                        const bf16x2 h = __builtin_convertvector(pair, bf16x2);
                        put(__builtin_bit_cast(unsigned, h), row);
                        if constexpr (REST) put(__builtin_bit_cast(unsigned, __builtin_convertvector(pair - __builtin_convertvector(h, f32x2), bf16x2)), row + 2 * a.rest);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);  // (quad by quad: together the temporaries spill)
        };
#pragma unroll
        for (int p = 0; p < C::WI; ++p) {
            if (i0 + wr + p * 32 >= a.Mp) break;
#pragma unroll
            for (int s = 0; s < 4; ++s) quad(std::false_type(), p, s, 0, C::WJ);
        }
        // The few blocks with a target are stored twice, by the same lanes: a test in the loop above would cost every block more
        if (hot) {
#pragma unroll
            for (int p = 0; p < C::WI; ++p)
#pragma unroll
                for (int q = 0; q < C::WJ; ++q)
                    if (hot >> (q * C::WI + p) & 1)
#pragma unroll
                        for (int s = 0; s < 4; ++s) quad(std::true_type(), p, s, q, q + 1);
        }
        if (a.dbias)
#pragma unroll
            for (int q = 0; q < C::WJ; ++q) {
                db[q] += __shfl_xor(db[q], 32);
                if (lh == 0) a.dbias[(long long)(bi * C::VI + wi) * a.ldg + v + q * 32 + li] = db[q];
            }
    };
    G::run(a.x, a.W, (a.nv - st + a.ns - 1) / a.ns, tile, 0, a.nk, lds, begin, done);
}

// lse and loss of the rows from the streams' parts: a wave a row, or (LANE) a lane, whose loads are then whole lines: many rows
// have few streams (65536 rows of 4: 5 us against 32 as waves)
template <bool LANE> __global__ __launch_bounds__(256) void loss_kernel(const float2 *part, int n, int M, int V, const float *hit, const long long *targets,
                                                                        long long ignore, float *loss, float *lse) {
    const int lane = threadIdx.x & 63, m = LANE ? blockIdx.x * 256 + threadIdx.x : blockIdx.x * 4 + (threadIdx.x >> 6);
    if (m >= M) return;
    const long long t = targets[m];
    const float h = hit[m];  // (nothing where the target is no entry)
    float2 all = make_float2(-__builtin_inff(), 0.f);
    constexpr int STEP = LANE ? 1 : 64;
    for (int i = LANE ? 0 : lane; i < n; i += 8 * STEP) {  // (the loads of eight parts under way at once)
        float2 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = i + STEP * k < n ? part[(long long)(i + STEP * k) * M + m] : make_float2(-__builtin_inff(), 0.f);
#pragma unroll
        for (int k = 0; k < 8; ++k) all = merge(all, v[k]);
    }
    if constexpr (!LANE) {
        for (int o = 32; o > 0; o >>= 1) all = merge(all, make_float2(__shfl_xor(all.x, o), __shfl_xor(all.y, o)));
        if (lane) return;
    }
    const float l = (all.x + __log2f(all.y)) * LN2;
    lse[m] = l;
    loss[m] = t == ignore ? 0.f : t < 0 || t >= V ? __builtin_nanf("") : l - h;
}

// What G's rounding took of the targets' entries, for dW: sums[slot[v]][d] = sum of left[m] x[m][d] over the rows m whose target
// is v, for every one of the tokens v0 .. v1 - 1 that has a row; slot[v] is the first of them, or v itself (BY_TOKEN: of more
// rows than tokens), and -1 where v has none.  A workgroup looks through the targets for those among its TOKENS tokens and keeps
// their rows in order, so that every sum has a fixed order; where the list could overflow it is added up first, and the next one
// goes on from there.  A wave takes the rows of a token one after the other, all waves together those of a token that has many,
// and join what they have.
// Bound by latency (a target's way from memory, a row's, the sums' back).  Measured: 16384 rows x 768 of 50257 tokens 47 us,
// 1999 x 1001 of 32003 11 us.
constexpr int TOKENS = 128, LIST = 4096, MANY = 32;
template <class T, bool BY_TOKEN> __global__ __launch_bounds__(1024) void target_rows_kernel(const long long *targets, long long ignore, const float *left,
                                                                                             const short *x, long long ld, int M, int D, int v0, int v1,
                                                                                             float *sums, int *slot) {
    constexpr int WAVES = 16, PER = 4, STEP = PER * 1024;
    static_assert(LIST >= STEP, "a step's rows fit");
    __shared__ int row_of[LIST], first[TOKENS], many[TOKENS], before[PER * WAVES];
    __shared__ unsigned char token_of[LIST];
    __shared__ __attribute__((aligned(16))) float part[WAVES][512];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int e0 = v0 + blockIdx.x * TOKENS, ne = v1 - e0 < TOKENS ? v1 - e0 : TOKENS;
    if (threadIdx.x < TOKENS) first[threadIdx.x] = -1, many[threadIdx.x] = 0;
    // acc += left x of token e's rows, 8 elements a lane from c and C - 1 times 512 behind it, of the rows at from .. from + 63,
    // from + step .. of the list's n; the first of these rows (the whole wave goes through them; lanes behind the row's end
    // read its beginning, for nothing)
    auto walk = [&](auto &acc, int e, int n, int from, int step, int c) __attribute__((always_inline)) {
        constexpr int C = sizeof(acc) / sizeof(acc[0]), AT_ONCE = 4 / C;  // rows on their way
        int d[C], row = -1;
#pragma unroll
        for (int h = 0; h < C; ++h) d[h] = c + h * 512 + lane * 8 < D ? c + h * 512 + lane * 8 : 0;
        for (int p = from; p < n; p += step) {
            unsigned long long mine = __builtin_amdgcn_ballot_w64(p + lane < n && token_of[p + lane < n ? p + lane : 0] == e);
            while (mine) {
                Vec<T> v[AT_ONCE][C];
                float f[AT_ONCE];
                int m = 0;
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i) {
                    const bool there = mine != 0;
                    if (there) m = __builtin_amdgcn_readfirstlane(row_of[p + __builtin_ctzll(mine)]);  // (else: the last one again, times 0)
                    if (row < 0) row = m;
                    mine &= mine - 1;
                    f[i] = there ? left[m] : 0.f;
#pragma unroll
                    for (int h = 0; h < C; ++h) v[i][h] = *(const Vec<T> *)(x + (long long)m * ld + d[h]);
                }
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
                    for (int h = 0; h < C; ++h)
#pragma unroll
                        for (int k = 0; k < 8; ++k) acc[h][k] = fmaf(f[i], (float)v[i][h].e[k], acc[h][k]);
            }
        }
        return row;
    };
    auto put = [&](int m, bool more, int d, const float (&acc)[8]) __attribute__((always_inline)) {
        float *to = sums + (long long)m * D + d;
        if (d + 8 <= D) {
#pragma unroll
            for (int k = 0; k < 8; k += 4) {
                Vec<float> v = {{acc[k], acc[k + 1], acc[k + 2], acc[k + 3]}};
                if (more) {
                    const Vec<float> u = *(const Vec<float> *)(to + k);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v.e[i] += u.e[i];
                }
                *(Vec<float> *)(to + k) = v;
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (d + k < D) to[k] = more ? to[k] + acc[k] : acc[k];
        }
    };
    auto add_up = [&](int n) {  // the n rows of the list
        unsigned long long few[TOKENS / 64], lots[TOKENS / 64];  // tokens with rows in the list
#pragma unroll
        for (int b = 0; b < TOKENS / 64; ++b) {
            const int count = many[b * 64 + lane];
            few[b] = __builtin_amdgcn_ballot_w64(count > 0 && count <= MANY) & (0x0001000100010001ull << wave);  // (this wave's)
            lots[b] = __builtin_amdgcn_ballot_w64(count > MANY);
        }
        static_assert(WAVES == 16 && TOKENS == 128, "every 16th token of two words");
        auto next_of = [](unsigned long long (&set)[2]) __attribute__((always_inline)) {  // takes the first token out; -1: none
            const int e = set[0] ? __builtin_ctzll(set[0]) : set[1] ? 64 + __builtin_ctzll(set[1]) : -1;
            set[1] &= set[0] ? ~0ull : set[1] - 1;
            set[0] &= set[0] - 1;
            return e;
        };
        for (int e = next_of(few); e >= 0; e = next_of(few)) {
            const int known = __builtin_amdgcn_readfirstlane(first[e]);
            int m = known;
            for (int c = 0; c < D; c += 1024) {
                float acc[2][8] = {};
                const int row = walk(acc, e, n, 0, 64, c);
                if (m < 0) m = BY_TOKEN ? e0 + e : row;
                put(m, known >= 0, c + lane * 8, acc[0]);
                put(m, known >= 0, c + 512 + lane * 8, acc[1]);
            }
            if (lane == 0) first[e] = m;
        }
        for (int e = next_of(lots); e >= 0; e = next_of(lots)) {
            const int known = __builtin_amdgcn_readfirstlane(first[e]);
            int m = BY_TOKEN ? e0 + e : known;
            for (int p = 0; m < 0; p += 64) {  // (there is one)
                const unsigned long long mine = __builtin_amdgcn_ballot_w64(p + lane < n && token_of[p + lane < n ? p + lane : 0] == e);
                if (mine) m = __builtin_amdgcn_readfirstlane(row_of[p + __builtin_ctzll(mine)]);
            }
            for (int c = 0; c < D; c += 512) {
                float acc[1][8] = {};
                walk(acc, e, n, wave * 64, 1024, c);
                *(f32x4 *)&part[wave][lane * 8] = (f32x4){acc[0][0], acc[0][1], acc[0][2], acc[0][3]};
                *(f32x4 *)&part[wave][lane * 8 + 4] = (f32x4){acc[0][4], acc[0][5], acc[0][6], acc[0][7]};
                __syncthreads();
                if (threadIdx.x < 512 && c + (int)threadIdx.x < D) {
                    float v = 0.f;
#pragma unroll
                    for (int w = 0; w < WAVES; ++w) v += part[w][threadIdx.x];
                    float *to = sums + (long long)m * D + c + threadIdx.x;
                    *to = known >= 0 ? *to + v : v;
                }
                __syncthreads();
            }
            if (threadIdx.x == 0) first[e] = m;
        }
        __syncthreads();  // the list and the counts are no longer read
        if (threadIdx.x < TOKENS) many[threadIdx.x] = 0;
    };
    int n = 0;
    long long next[PER];
    auto load = [&](int r) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const long long m = (long long)r + i * 1024 + threadIdx.x;
            next[i] = m < M ? targets[m] : ignore;
        }
    };
    load(0);
    for (int r = 0; r < M; r += STEP) {
        int token[PER], at[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const long long t = next[i];
            token[i] = t != ignore && t >= e0 && t < e0 + ne ? (int)(t - e0) : -1;
        }
        if (r + STEP < M) load(r + STEP);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const unsigned long long found = __builtin_amdgcn_ballot_w64(token[i] >= 0);
            at[i] = __popcll(found & ((1ull << lane) - 1));
            if (lane == 0) before[i * WAVES + wave] = __popcll(found);
        }
        __syncthreads();
        // how many were found before each of this wave's 64 (a lane a count: PER * WAVES of them)
        static_assert(PER * WAVES == 64, "a lane a count");
        const int count = before[lane];
        int upto = count;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const int u = __shfl_up(upto, o);
            if (lane >= o) upto += u;
        }
        const int total = __shfl(upto, 63);
        if (total) {  // (of the whole workgroup)
            if (n + total > LIST) {
                add_up(n);
                n = 0;
                __syncthreads();
            }
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int from = __shfl(upto - count, i * WAVES + wave);
                if (token[i] >= 0) {
                    row_of[n + from + at[i]] = r + i * 1024 + threadIdx.x;
                    token_of[n + from + at[i]] = token[i];
                    atomicAdd(&many[token[i]], 1);  // (a count has no order)
                }
            }
            n += total;
        }
        __syncthreads();  // the list is there, and the counts are no longer read
    }
    if (n) add_up(n);
    __syncthreads();
    if (threadIdx.x < ne) slot[e0 + threadIdx.x] = first[threadIdx.x];
}
// The targets' part of a product of dW (target_rows_kernel), slot: of its first token; null: none
struct Targets {
    const float *sums;
    const int *slot;
    int by_col;  // the vocabulary is the product's columns
};

struct SumArgs {  // C[z][i][j] = (or +=) the z-th part of the k-steps; pair: of rows 2 i and 2 i + 1 of A
    Operand A, B;
    int nk, per, ti, tj, I, J, add, pair;
    float *out;
};
struct OutArgs {  // C[i][j] * g_unit, in the elements' type
    Operand A, B;
    int nk, ti, tj, I, J;
    const unsigned *gtop;
    void *out;
    long long ld;
    Targets more;
};
template <class C, bool KMAJOR, bool F16, int PLANES, int SCALED> __global__ __launch_bounds__(C::NT, C::OCC) void sum_kernel(const SumArgs a) {
    typedef Gemm<C, KMAJOR, F16, PLANES, SCALED> G;
    __shared__ __attribute__((aligned(16))) char lds[G::LDS_BYTES];
    int bi, bj;
    tile_of(blockIdx.x, a.ti, a.tj, bi, bj);
    const int k0 = blockIdx.y * a.per, k1 = k0 + a.per < a.nk ? k0 + a.per : a.nk;
    const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5, wave = threadIdx.x >> 6;
    const int wi0 = bi * C::BI + (wave / C::VJ) * (C::WI * 32), wj0 = bj * C::BJ + (wave % C::VJ) * (C::WJ * 32);
    auto begin = [&](int, f32x16 (&acc)[C::WI][C::WJ]) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < C::WI; ++p)
#pragma unroll
            for (int q = 0; q < C::WJ; ++q) clear(acc[p][q]);
    };
    auto done = [&](int, f32x16 (&acc)[C::WI][C::WJ]) __attribute__((always_inline)) {
        float *o = a.out + ((long long)blockIdx.y * a.I + wi0 + 4 * lh) * a.J + wj0 + li;
        if (PLANES == 1 && a.pair) {
            o -= (long long)(wi0 / 2 + 2 * lh) * a.J;
#pragma unroll
            for (int p = 0; p < C::WI; ++p)
#pragma unroll
                for (int q = 0; q < C::WJ; ++q)
#pragma unroll
                    for (int r = 0; r < 16; r += 2) {
                        if ((wi0 + p * 32 + block_row(r, lh)) / 2 >= a.I || wj0 + q * 32 + li >= a.J) continue;
                        float *to = o + (long long)((p * 32 + block_row(r, 0)) / 2) * a.J + q * 32;
                        const float v = acc[p][q][r] + acc[p][q][r + 1];
                        *to = a.add ? *to + v : v;
                    }
            return;
        }
#pragma unroll
        for (int p = 0; p < C::WI; ++p)
#pragma unroll
            for (int q = 0; q < C::WJ; ++q)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    if (wi0 + p * 32 + block_row(r, lh) >= a.I || wj0 + q * 32 + li >= a.J) continue;
                    float *to = o + (long long)(p * 32 + block_row(r, 0)) * a.J + q * 32;
                    *to = a.add ? *to + acc[p][q][r] : acc[p][q][r];
                }
    };
    G::run(a.A, a.B, 1, [&](int) { return TileAt{bi * C::BI, bj * C::BJ}; }, k0, k1, lds, begin, done);
}
template <class C, bool F16, int PLANES, int SCALED> __global__ __launch_bounds__(C::NT, C::OCC) void out_kernel(const OutArgs a) {
    typedef Gemm<C, true, F16, PLANES, SCALED> G;
    __shared__ __attribute__((aligned(16))) char lds[G::LDS_BYTES];
    int bi, bj;
    tile_of(blockIdx.x, a.ti, a.tj, bi, bj);
    const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5, wave = threadIdx.x >> 6;
    const int wi0 = bi * C::BI + (wave / C::VJ) * (C::WI * 32), wj0 = bj * C::BJ + (wave % C::VJ) * (C::WJ * 32);
    constexpr int ELEM = PLANES == 2 ? TSC_ELEM_F32 : F16 ? TSC_ELEM_F16 : TSC_ELEM_BF16;  // (a type that is asked for at every store costs more than the store)
    const float post = g_unit(a.gtop);
    __shared__ int slots[PLANES == 1 ? (C::BI > C::BJ ? C::BI : C::BJ) : 1];  // of the tile's part of the vocabulary
    if (PLANES == 1 && a.more.slot) {
        const int at = a.more.by_col ? bj * C::BJ : bi * C::BI, n = a.more.by_col ? a.J : a.I;
        for (int i = threadIdx.x; i < (a.more.by_col ? C::BJ : C::BI); i += C::NT) slots[i] = at + i < n ? a.more.slot[at + i] : -1;
        __syncthreads();
    }
    auto begin = [&](int, f32x16 (&acc)[C::WI][C::WJ]) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < C::WI; ++p)
#pragma unroll
            for (int q = 0; q < C::WJ; ++q) clear(acc[p][q]);
    };
    auto done = [&](int, f32x16 (&acc)[C::WI][C::WJ]) __attribute__((always_inline)) {
        const long long at = (long long)(wi0 + 4 * lh) * a.ld + wj0 + li;
        auto put = [&](int p, int q, int r, float v) __attribute__((always_inline)) {
            if (wi0 + p * 32 + block_row(r, lh) < a.I && wj0 + q * 32 + li < a.J)
                write_elem(a.out, ELEM, at + (long long)(p * 32 + block_row(r, 0)) * a.ld + q * 32, v * post);
        };
        // The targets' part is added on the way out (sums that change in a branch are copied, and spilled): block by block, the
        // next one's loads in front of a block's stores, behind which they would have to wait, and a row's blocks one after the other,
        // so that the halves of a line leave together: 1999 x 1001 x 32003 136 us.
        constexpr int N = C::WI * C::WJ, AHEAD = 2;
        float v[AHEAD][16];
        if (PLANES == 1 && a.more.slot && a.more.by_col) {
            auto load = [&](int b) __attribute__((always_inline)) {
                const int p = b / C::WJ, q = b % C::WJ, from = slots[wj0 - bj * C::BJ + q * 32 + li];
                const float *s = a.more.sums + (long long)(from < 0 ? 0 : from) * a.I + wi0 + p * 32 + 4 * lh;
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const int i = wi0 + p * 32 + block_row(r, lh);
                    Vec<float> u = {};
                    if (from >= 0 && i + 4 <= a.I) {
                        u = *(const Vec<float> *)(s + block_row(r, 0));
                    } else if (from >= 0) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (i + e < a.I) u.e[e] = s[block_row(r, 0) + e];
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[b % AHEAD][r + e] = u.e[e];
                }
            };
#pragma unroll
            for (int b = 0; b < AHEAD - 1; ++b) load(b);
#pragma unroll
            for (int b = 0; b < N; ++b) {
                if (b + AHEAD - 1 < N) load(b + AHEAD - 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int r = 0; r < 16; ++r) put(b / C::WJ, b % C::WJ, r, acc[b / C::WJ][b % C::WJ][r] + v[b % AHEAD][r]);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else if (PLANES == 1 && a.more.slot) {
            auto load = [&](int b) __attribute__((always_inline)) {
                const int p = b / C::WJ, j = wj0 + b % C::WJ * 32 + li;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int from = slots[wi0 - bi * C::BI + p * 32 + block_row(r, lh)];
                    v[b % AHEAD][r] = from >= 0 && j < a.J ? a.more.sums[(long long)from * a.J + j] : 0.f;
                }
            };
#pragma unroll
            for (int b = 0; b < AHEAD - 1; ++b) load(b);
#pragma unroll
            for (int b = 0; b < N; ++b) {
                if (b + AHEAD - 1 < N) load(b + AHEAD - 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int r = 0; r < 16; ++r) put(b / C::WJ, b % C::WJ, r, acc[b / C::WJ][b % C::WJ][r] + v[b % AHEAD][r]);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
#pragma unroll
            for (int p = 0; p < C::WI; ++p)
#pragma unroll
                for (int q = 0; q < C::WJ; ++q)
#pragma unroll
                    for (int r = 0; r < 16; ++r) put(p, q, r, acc[p][q][r]);
        }
    };
    G::run(a.A, a.B, 1, [&](int) { return TileAt{bi * C::BI, bj * C::BJ}; }, 0, a.nk, lds, begin, done);
}
// v = the sum of n parts, `step` apart, of 4 neighbouring elements at p (fewer where only `rest` are left).  SHARED: the four
// waves of the workgroup take every fourth part each, and the first one, for which this is true, gets the sums.
template <bool SHARED> __device__ __forceinline__ bool sum_parts(const float *p, int n, long long step, int rest, float (&red)[3][256], float (&v)[4]) {
    const int lane = threadIdx.x & 63, wave = SHARED ? threadIdx.x >> 6 : 0;
    constexpr int W = SHARED ? 4 : 1;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = 0.f;
    if (rest >= 4) {
#pragma unroll 4
        for (int z = wave; z < n; z += W) {
            const Vec<float> u = *(const Vec<float> *)(p + z * step);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += u.e[e];
        }
    } else {
        for (int e = 0; e < rest; ++e)
            for (int z = wave; z < n; z += W) v[e] += p[z * step + e];
    }
    if constexpr (SHARED) {
        if (wave)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[wave - 1][e * 64 + lane] = v[e];
        __syncthreads();
        if (wave) return false;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (v[e] + red[0][e * 64 + lane]) + (red[1][e * 64 + lane] + red[2][e * 64 + lane]);
    }
    return true;
}
// C[i][j] = sum over z of part[z][i][j] times g_unit, 4 elements a lane: a dW whose k-steps were split
template <bool SHARED> __global__ __launch_bounds__(256) void join_kernel(const float *part, int n, int I, int J, const Targets more, const unsigned *gtop,
                                                                          void *out, long long ld, int elem) {
    __shared__ float red[3][256];
    const int i = blockIdx.x, j = SHARED ? blockIdx.y * 256 + (threadIdx.x & 63) * 4 : (blockIdx.y * 256 + threadIdx.x) * 4;
    float v[4];
    if (!sum_parts<SHARED>(part + (long long)i * J + j, n, (long long)I * J, J - j, red, v)) return;
    if (more.slot) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (j + e < J) {
                const int from = more.slot[more.by_col ? j + e : i];
                if (from >= 0) v[e] += more.by_col ? more.sums[(long long)from * I + i] : more.sums[(long long)from * J + j + e];
            }
    }
    const float unit = g_unit(gtop);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (j + e < J) write_elem(out, elem, i * ld + j + e, v[e] * unit);
}
// dx[m][d] = sum over z, with the scales undone: 256 elements of a row a workgroup, whose waves share the parts, or a wave (few
// parts, many rows: what takes the time is the way from a row's target to its row of W)
template <bool SHARED> __global__ __launch_bounds__(256) void dx_kernel(const float *part, int n, int M, int D, const float *wscale, const float *xscale,
                                                 const unsigned *gtop, const float *g, const long long *targets, long long ignore,
                                                 const float *left, const short *Wt, long long wt_ld, int V, int elem, void *dx) {
    __shared__ float red[3][256];
    const int m = SHARED ? blockIdx.x : blockIdx.x * 4 + (threadIdx.x >> 6), d = blockIdx.y * 256 + (threadIdx.x & 63) * 4;
    if (!SHARED && m >= M) return;
    const long long t = targets[m];
    const bool live = t != ignore;
    struct __attribute__((packed, aligned(2))) Four { short e[4]; } u = {};
    float v[4], rest = 0.f;
    if (left && live && t >= 0 && t < V && (!SHARED || threadIdx.x < 64)) {  // (on their way while the parts are summed)
        rest = left[m];
        const short *p = Wt + t * wt_ld + d;
        if (d + 4 <= D) {
            u = *(const Four *)p;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e < D) u.e[e] = p[e];
        }
    }
    if (!sum_parts<SHARED>(part + (long long)m * D + d, n, (long long)M * D, D - d, red, v)) return;
    const float unit = g_unit(gtop), ws = wscale ? wscale[0] : 1.f, xs = wscale ? 1.f / row_scale(xscale[m], gtop, g[m]) : 1.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float w = elem == TSC_ELEM_BF16 ? (float)__builtin_bit_cast(__bf16, u.e[e]) : (float)__builtin_bit_cast(_Float16, u.e[e]);
        if (d + e < D) write_elem(dx, elem, (long long)m * D + d + e, live ? fmaf(rest, w, v[e]) * unit * ws * xs : 0.f);
    }
}
// db[at + j] = sum over the parts, 64 columns x 16 parts a workgroup
__global__ __launch_bounds__(1024) void dbias_kernel(const float *part, int n, long long ld, int J, const unsigned *gtop, int elem, void *out,
                                                     long long at) {
    __shared__ float red[16][64];
    const int c = threadIdx.x & 63, p = threadIdx.x >> 6, j = blockIdx.x * 64 + c;
    float v = 0.f;
    if (j < J)
        for (int i = p; i < n; i += 16) v += part[i * ld + j];
    red[p][c] = v;
    __syncthreads();
    if (p || j >= J) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) v += red[i][c];
    write_elem(out, elem, at + j, v * g_unit(gtop));
}
__global__ void zero_elem_kernel(void *p, int elem, long long n) {  // (a launch holds fewer than 2^32 threads, dW up to 2^35 elements)
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) write_elem(p, elem, i, 0.f);
}

inline int cdiv(long long a, long long b) { return (int)((a + b - 1) / b); }
inline long long up(long long a, long long b) { return (a + b - 1) / b * b; }

constexpr long long PIECE_BYTES = 1ll << 31;  // G of one piece of the vocabulary
constexpr long long MAX_LD = 1 << 22;         // a tile's 256 rows lie within 2^31 bytes

}  // namespace

struct tsc_unembed {
    int D, V, elem, belem, planes, Dp, Vp, Vb;  // paddings: 64 for a product's k, 256 for the bias a tile reads
    long long sd, sv;                    // strides of W (elements): one of them is 1
    const void *W, *bias;                // borrowed
    const short *Wt, *Wd;                // [V][planes * Dp] and [D][planes * Vp], or W itself where it can be read as it is
    long long wt_ld, wd_ld;
    bool own_t, own_d;
    float *bias32, *wscale;
    mutable std::mutex lock;             // of what follows
    hipEvent_t laid;                     // behind the last layout that was not captured
    mutable bool pending;                // ... which may still run
};

namespace {

bool capturing(hipStream_t s) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(s, &st) == hipSuccess) return st != hipStreamCaptureStatusNone;
    (void)hipGetLastError();
    return false;
}

// Work on s comes after the layout, whichever stream that runs on.  A captured stream cannot wait for one outside the
// capture: the layout has to be over by then.
int after_layout(const tsc_unembed *h, hipStream_t s) {
    std::lock_guard<std::mutex> own(h->lock);
    if (!h->pending) return TSC_OK;
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;  // (asking for an event's state would end somebody's capture otherwise)
    TSC_HIP_CHECK(hipThreadExchangeStreamCaptureMode(&mode));
    const hipError_t e = hipEventQuery(h->laid);
    TSC_HIP_CHECK(hipThreadExchangeStreamCaptureMode(&mode));
    if (e == hipSuccess) {
        h->pending = false;
        return TSC_OK;
    }
    (void)hipGetLastError();
    if (e != hipErrorNotReady) return tsc_fail(TSC_ERR_HIP, "hipEventQuery failed: %s", hipGetErrorString(e));
    if (capturing(s)) return tsc_fail(TSC_ERR_ARG, "the unembedding is still being laid out: synchronize before the capture");
    TSC_HIP_CHECK(hipStreamWaitEvent(s, h->laid, 0));
    return TSC_OK;
}

}  // namespace

// ------------------------------------------------------------------------------------------------ handle
int tsc_unembed_destroy_(tsc_unembed *h) {
    if (!h) return TSC_OK;
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;  // (a handle may be dropped while somebody captures)
    const bool relaxed = hipThreadExchangeStreamCaptureMode(&mode) == hipSuccess;
    if (h->own_t && h->Wt) (void)hipFree((void *)h->Wt);
    if (h->own_d && h->Wd) (void)hipFree((void *)h->Wd);
    if (h->bias32) (void)hipFree(h->bias32);
    if (h->wscale) (void)hipFree(h->wscale);
    if (h->laid) (void)hipEventDestroy(h->laid);
    if (relaxed) (void)hipThreadExchangeStreamCaptureMode(&mode);
    delete h;
    return TSC_OK;
}

void tsc_unembed_shape_(const tsc_unembed *h, int *elem, int *D, int *V) { *elem = h->elem; *D = h->D; *V = h->V; }

int tsc_unembed_refresh_(tsc_unembed *h, hipStream_t s) {
    const int rc = after_layout(h, s);  // (two at once would meet in the scale)
    if (rc) return rc;
    hipLaunchKernelGGL(bias_kernel, dim3(cdiv(h->Vb, 256)), dim3(256), 0, s, h->bias, h->belem, h->V, h->Vb, h->bias32);
    if (h->elem == TSC_ELEM_F32) {
        hipLaunchKernelGGL(fill_kernel, dim3(1), dim3(256), 0, s, h->wscale, 0.f, 1ll);
        const long long rows = h->sv == 1 ? h->D : h->V, cols = h->sv == 1 ? h->V : h->D, ld = h->sv == 1 ? h->sd : h->sv;
        hipLaunchKernelGGL(absmax_kernel, dim3((int)(rows < 1024 ? rows : 1024)), dim3(1024), 0, s, (const float *)h->W, rows, cols, ld, (unsigned *)h->wscale);
        hipLaunchKernelGGL(wscale_kernel, dim3(1), dim3(1), 0, s, h->wscale);
    }
    auto pack = [&](long long sr, long long sc, int R, int C, int Cp, short *out) {
        const dim3 grid(Cp / 64, cdiv(R, 64));
        if (h->elem == TSC_ELEM_F32) hipLaunchKernelGGL((pack_w_kernel<float>), grid, dim3(256), 0, s, (const float *)h->W, sr, sc, R, C, Cp, h->wscale, out);
        else hipLaunchKernelGGL((pack_w_kernel<short>), grid, dim3(256), 0, s, (const short *)h->W, sr, sc, R, C, Cp, (const float *)nullptr, out);
    };
    if (h->own_t) pack(h->sv, h->sd, h->V, h->D, h->Dp, (short *)h->Wt);
    if (h->own_d) pack(h->sd, h->sv, h->D, h->V, h->Vp, (short *)h->Wd);
    TSC_HIP_CHECK(hipGetLastError());
    if (capturing(s)) return TSC_OK;  // (nothing has been laid out yet)
    std::lock_guard<std::mutex> own(h->lock);
    TSC_HIP_CHECK(hipEventRecord(h->laid, s));
    h->pending = true;
    return TSC_OK;
}

int tsc_unembed_create_(tsc_unembed **out, int D, int V, int elem, const void *W, long long sd, long long sv, const void *bias, int belem, hipStream_t s) {
    if (capturing(s)) return tsc_fail(TSC_ERR_ARG, "an unembedding cannot be made inside a capture: make it before");
    tsc_unembed *h = new (std::nothrow) tsc_unembed();
    if (!h) return tsc_fail(TSC_ERR_HIP, "out of host memory");
    h->D = D; h->V = V; h->elem = elem; h->belem = belem; h->planes = elem == TSC_ELEM_F32 ? 2 : 1;
    h->Dp = (int)up(D, BK); h->Vp = (int)up(V, 256); h->Vb = h->Vp + 256;
    h->sd = sd; h->sv = sv; h->W = W; h->bias = bias;
    // 16-bit weights in the order and at the alignment that a product reads are read where they are
    const bool plain = elem != TSC_ELEM_F32 && (uintptr_t)W % 16 == 0;
    h->own_t = !(plain && sd == 1 && D % BK == 0 && sv % 8 == 0 && sv <= MAX_LD);
    h->own_d = !(plain && sv == 1 && V % BK == 0 && sd % 8 == 0 && sd <= MAX_LD);
    h->wt_ld = h->own_t ? (long long)h->planes * h->Dp : sv;
    h->wd_ld = h->own_d ? (long long)h->planes * h->Vp : sd;
    hipError_t e = hipSuccess;
    if (!h->own_t) h->Wt = (const short *)W;
    else e = hipMalloc((void **)&h->Wt, (size_t)V * h->planes * h->Dp * 2);
    if (!h->own_d) h->Wd = (const short *)W;
    else if (e == hipSuccess) e = hipMalloc((void **)&h->Wd, (size_t)D * h->planes * h->Vp * 2);
    if (e == hipSuccess) e = hipMalloc((void **)&h->bias32, (size_t)h->Vb * 4);
    if (e == hipSuccess) e = hipMalloc((void **)&h->wscale, 256);
    if (e == hipSuccess) e = hipEventCreateWithFlags(&h->laid, hipEventDisableTiming);
    int rc = e == hipSuccess ? tsc_unembed_refresh_(h, s) : tsc_fail(TSC_ERR_HIP, "making the unembedding's operands failed: %s", hipGetErrorString(e));
    if (rc != TSC_OK) {
        tsc_unembed_destroy_(h);
        return rc;
    }
    *out = h;
    return TSC_OK;
}

// ------------------------------------------------------------------------------------------------ launches
namespace {

// Tiles of a launch.  LARGE: one workgroup a CU; MEDIUM: two; FEW (64 rows of x at most): three.
enum { LARGE, MEDIUM, FEW };
constexpr int CUS = 256;
struct Shape {
    int kind, bi, bj, slots;
};
Shape shape_of(int kind) {  // bi: rows of x (products of logits), or of the result
    return kind == LARGE ? Shape{LARGE, 256, 256, CUS} : kind == MEDIUM ? Shape{MEDIUM, 128, 128, 2 * CUS} : Shape{FEW, 64, 128, 3 * CUS};
}

// Logits: blocks of rows x streams of vocabulary tiles.  A stream's length times the rounds of workgroups is what a CU does;
// at least four streams a block where there are many blocks, so that the tiles resident on an XCD share its L2.
struct Streams {
    Shape s;
    int nm, nv, ns;
};
Streams streams(long long M, long long V) {
    Streams r{};
    r.s = shape_of(M <= FEW_ROWS ? FEW : cdiv(M, 256) * (long long)cdiv(V, 256) >= CUS ? LARGE : MEDIUM);
    r.nm = cdiv(M, r.s.bi);
    r.nv = cdiv(V, r.s.bj);
    long long best = -1;
    for (int ns = r.nv < 4 ? r.nv : 4; ns <= r.nv; ++ns) {
        const long long cost = (long long)cdiv((long long)r.nm * ns, r.s.slots) * cdiv(r.nv, ns);
        if (best < 0 || cost < best) best = cost, r.ns = ns;
        if ((long long)r.nm * ns >= 4ll * r.s.slots) break;
    }
    return r;
}

// A product of I x J with nk k-steps: tiles and the parts that its k-steps are split into, by the time of the slowest CU
// (64 k of a LARGE tile take 1.8 us, of a MEDIUM one, two of which share a CU, 1.1; three times that with two planes; a
// tile begins and ends in 4) plus the traffic of the fp32 parts.
struct Split {
    Shape s;
    int ti, tj, z, per;
    double cost;
};
Split split_of(long long I, long long J, int nk, int planes, bool always_parts) {
    Split best{};
    double least = 0;
    for (int kind : {LARGE, MEDIUM}) {
        Split r{};
        r.s = shape_of(kind);
        r.ti = cdiv(I, r.s.bi);
        r.tj = cdiv(J, r.s.bj);
        const double step = (kind == LARGE ? 1.8e-6 : 1.1e-6) * (planes == 2 ? 3 : 1), start = 4e-6, part = (double)I * J * 8 / 5e12;
        for (int z = 1; z <= 128 && z <= nk; ++z) {
            r.per = cdiv(nk, z);
            r.z = cdiv(nk, r.per);
            const double cost = (double)cdiv((long long)r.ti * r.tj * r.z, r.s.slots) * (r.per * step + start) +
                                (r.z > 1 || always_parts ? r.z * part : 0);
            if (least == 0 || cost < least) least = r.cost = cost, best = r;
        }
    }
    return best;
}

// What a call keeps in its workspace (each part starts at a multiple of 256 bytes)
struct Plan {
    int Mp;
    int copies;      // backward: rows of G a row (2: its remainder too), and of x
    bool left_wanted, targets_wanted;  // what 16 bits take of the targets' entries: kept; summed by token for dW
    Streams st;
    int Vc, pieces;  // backward: entries of a piece
    Split dx;        // of a whole piece
    long long xp, xscale, part, hit, gtop, left, sums, slot, g, db, dxp, dwp, bytes;
};
// dW of nv entries of the vocabulary: as many of them as fill whole rounds of the chip in one piece, the rest (or all of them,
// where that is cheaper) with their k-steps split.
struct DwPlan {
    int n[2];  // entries of each part
    Split w[2];
};
DwPlan dw_plan(const tsc_unembed *h, long long rows, int nv) {
    const int nk = (int)(rows / BK), dt = cdiv(h->D, 256);
    auto of = [&](int n) { return h->sv == 1 ? split_of(h->D, n, nk, h->planes, false) : split_of(n, h->D, nk, h->planes, false); };
    DwPlan r{{nv, 0}, {of(nv), {}}};
    const int rounds = (int)((long long)dt * cdiv(nv, 256) / CUS), main = rounds * CUS / dt * 256;
    if (rounds < 1 || main >= nv) return r;
    const DwPlan two{{main, nv - main}, {of(main), of(nv - main)}};
    return two.w[0].cost + two.w[1].cost < r.w[0].cost ? two : r;
}
Plan plan(const tsc_unembed *h, long long M, bool backward, bool want_x, bool want_w, bool want_b) {
    Plan p{};
    p.Mp = (int)up(M, BK);
    p.copies = backward && h->planes == 1 && M <= FEW_ROWS ? 2 : 1;
    const int rows = p.copies * p.Mp;
    int nv = h->V;
    if (backward) {
        const int all = cdiv(h->V, 256);
        const long long fit = PIECE_BYTES / (2ll * h->planes * rows * 256);
        const int vt = (int)(fit < 1 ? 1 : fit < all ? fit : all);
        p.Vc = vt * 256;
        p.pieces = cdiv(h->V, p.Vc);
        if (p.Vc < nv) nv = p.Vc;
    }
    p.st = streams(M, nv);
    long long at = 0;
    auto take = [&](long long n) { const long long q = at; at = up(at + n, 256); return q; };
    p.xp = take(2ll * h->planes * rows * h->Dp);
    p.xscale = take(4 * M);
    if (!backward) {
        p.part = take(8ll * p.st.ns * M);
        p.hit = take(4 * M);
    } else {
        p.gtop = take(8);
        p.left_wanted = (want_x || want_w) && h->planes == 1 && p.copies == 1;
        p.targets_wanted = p.left_wanted && want_w;
        if (p.left_wanted) p.left = take(4 * M);
        if (p.targets_wanted) {
            p.sums = take(4ll * (M < h->V ? M : h->V) * h->D);
            p.slot = take(4ll * h->V);
        }
        p.g = take(2ll * h->planes * rows * p.Vc);
        if (want_b) p.db = take(4ll * 2 * p.st.nm * p.Vc);  // (two parts a tile of rows, or one of twice the pitch)
        if (want_x) {
            p.dx = split_of(p.copies * M, h->D, cdiv(nv, BK), h->planes, true);
            p.dxp = take(4ll * p.dx.z * M * h->D);
        }
        if (want_w) {  // the parts of a piece's dW and of the last, shorter one's
            long long most = 0;
            for (int n : {nv, h->V - (p.pieces - 1) * p.Vc}) {
                const DwPlan w = dw_plan(h, rows, n);
                for (int i = 0; i < 2; ++i)
                    if (w.n[i] && w.w[i].z > 1 && (long long)w.w[i].z * w.n[i] > most) most = (long long)w.w[i].z * w.n[i];
            }
            p.dwp = take(4ll * most * h->D);
        }
    }
    p.bytes = at;
    return p;
}

template <bool F16, bool SPLIT, bool GRAD> int launch_logits(const Streams &st, const LogitArgs &a, hipStream_t s) {
    const dim3 grid(a.nm * a.ns);
#define TSC_LOGITS(T1, T2)                                                                                                     \
    {                                                                                                                          \
        if (GRAD) hipLaunchKernelGGL((grad_logits_kernel<T1, F16, SPLIT>), grid, dim3(T1::NT), 0, s, a);                      \
        else hipLaunchKernelGGL((loss_logits_kernel<T2, F16, SPLIT>), grid, dim3(T2::NT), 0, s, a);                           \
    }
    if (st.s.kind == LARGE) TSC_LOGITS(TileLarge, TileLarge)
    else if (st.s.kind == MEDIUM) TSC_LOGITS(TileMedium, TileMedium)
    else TSC_LOGITS(TileWide, TileTall)
#undef TSC_LOGITS
    TSC_HIP_CHECK(hipGetLastError());
    return TSC_OK;
}
template <bool GRAD> int logits(const tsc_unembed *h, const Streams &st, const LogitArgs &a, hipStream_t s) {
    return h->elem == TSC_ELEM_F32    ? launch_logits<true, true, GRAD>(st, a, s)
           : h->elem == TSC_ELEM_BF16 ? launch_logits<false, false, GRAD>(st, a, s)
                                      : launch_logits<true, false, GRAD>(st, a, s);
}
LogitArgs logit_args(const tsc_unembed *h, const Plan &p, char *ws, int M, const long long *targets, long long ignore) {
    LogitArgs a{};
    a.W = {h->Wt, h->wt_ld, h->V};
    a.x = {(const short *)(ws + p.xp), (long long)h->planes * h->Dp, M};
    a.nk = h->Dp / BK;
    a.nm = p.st.nm; a.ns = p.st.ns; a.nv = p.st.nv; a.M = M; a.V = h->V;
    a.bias = h->bias32;
    a.wscale = h->planes == 2 ? h->wscale : nullptr;
    a.xscale = h->planes == 2 ? (const float *)(ws + p.xscale) : nullptr;
    a.targets = targets; a.ignore = ignore;
    return a;
}
// (elements of the operands; SCALED: the operand that is G, where it has two planes)
#define TSC_BY_ELEM(KERNEL, TILE, SCALED, ...)                                                                                  \
    {                                                                                                                           \
        if (elem == TSC_ELEM_F32) hipLaunchKernelGGL((KERNEL<TILE, __VA_ARGS__ true, 2, SCALED>), grid, dim3(TILE::NT), 0, s, q);     \
        else if (elem == TSC_ELEM_BF16) hipLaunchKernelGGL((KERNEL<TILE, __VA_ARGS__ false, 1, 0>), grid, dim3(TILE::NT), 0, s, q);   \
        else hipLaunchKernelGGL((KERNEL<TILE, __VA_ARGS__ true, 1, 0>), grid, dim3(TILE::NT), 0, s, q);                               \
    }
#define TSC_COMMA ,
int launch_dx(const Split &w, int elem, SumArgs &q, hipStream_t s) {
    q.per = w.per; q.ti = w.ti; q.tj = w.tj;
    const dim3 grid(w.ti * w.tj, w.z);
    if (w.s.kind == LARGE) TSC_BY_ELEM(sum_kernel, TileLarge, 1, false TSC_COMMA)
    else TSC_BY_ELEM(sum_kernel, TileMedium, 1, false TSC_COMMA)
    TSC_HIP_CHECK(hipGetLastError());
    return TSC_OK;
}
int launch_dw_parts(const Split &w, int elem, bool by_d, SumArgs &q, hipStream_t s) {
    q.per = w.per; q.ti = w.ti; q.tj = w.tj;
    const dim3 grid(w.ti * w.tj, w.z);
    if (w.s.kind == LARGE) {
        if (by_d) TSC_BY_ELEM(sum_kernel, TileLarge, 2, true TSC_COMMA) else TSC_BY_ELEM(sum_kernel, TileLarge, 1, true TSC_COMMA)
    } else {
        if (by_d) TSC_BY_ELEM(sum_kernel, TileMedium, 2, true TSC_COMMA) else TSC_BY_ELEM(sum_kernel, TileMedium, 1, true TSC_COMMA)
    }
    TSC_HIP_CHECK(hipGetLastError());
    return TSC_OK;
}
int launch_dw(const Split &w, int elem, bool by_d, OutArgs &q, hipStream_t s) {
    q.ti = w.ti; q.tj = w.tj;
    const dim3 grid(w.ti * w.tj);
    if (w.s.kind == LARGE) {
        if (by_d) TSC_BY_ELEM(out_kernel, TileLarge, 2, ) else TSC_BY_ELEM(out_kernel, TileLarge, 1, )
    } else {
        if (by_d) TSC_BY_ELEM(out_kernel, TileMedium, 2, ) else TSC_BY_ELEM(out_kernel, TileMedium, 1, )
    }
    TSC_HIP_CHECK(hipGetLastError());
    return TSC_OK;
}
#undef TSC_COMMA
#undef TSC_BY_ELEM

}  // namespace

namespace {
void pack_x(const tsc_unembed *h, const Plan &p, const TscRows &x, int M, const long long *targets, long long ignore, const float *g, char *ws,
            unsigned *gtop, hipStream_t s) {
    short *out = (short *)(ws + p.xp);
    float *xscale = (float *)(ws + p.xscale);
    const int n = p.Mp >= 16384 ? 4 : 1;  // (a full chip of waves first)
    const dim3 grid(cdiv(p.Mp, 4 * n));
    if (h->elem == TSC_ELEM_F32)
        hipLaunchKernelGGL((pack_x_kernel<float>), grid, dim3(256), 0, s, x, M, p.Mp, h->D, h->Dp, n, p.copies, targets, ignore, g, out, xscale, gtop);
    else
        hipLaunchKernelGGL((pack_x_kernel<short>), grid, dim3(256), 0, s, x, M, p.Mp, h->D, h->Dp, n, p.copies, targets, ignore, g, out, xscale, gtop);
}
}  // namespace

size_t tsc_unembed_workspace_(const tsc_unembed *h, long long M, int backward, int want_x, int want_w, int want_b) {
    return M < 1 ? 0 : (size_t)plan(h, M, backward, want_x, want_w, want_b).bytes;
}

int tsc_launch_unembed_loss(const tsc_unembed *h, const TscRows &x, int M, const long long *targets, long long ignore, float *loss,
                            float *lse, char *ws, hipStream_t s) {
    const int ordered = after_layout(h, s);
    if (ordered) return ordered;
    const Plan p = plan(h, M, false, false, false, false);
    LogitArgs a = logit_args(h, p, ws, M, targets, ignore);
    const bool one_stride = x.inner_stride * x.inner == x.outer_stride;
    if (h->elem != TSC_ELEM_F32 && one_stride && h->D % BK == 0 && x.inner_stride % 8 == 0 && x.inner_stride <= MAX_LD && (uintptr_t)x.data % 16 == 0)
        a.x = {(const short *)x.data, x.inner_stride, M};  // rows that a product can read where they are
    else
        pack_x(h, p, x, M, nullptr, ignore, nullptr, ws, nullptr, s);
    a.part = (float2 *)(ws + p.part);
    a.hit = (float *)(ws + p.hit);
    const int rc = logits<false>(h, p.st, a, s);
    if (rc) return rc;
    if (p.st.ns <= 16) hipLaunchKernelGGL((loss_kernel<true>), dim3(cdiv(M, 256)), dim3(256), 0, s, a.part, p.st.ns, M, h->V, a.hit, targets, ignore, loss, lse);
    else hipLaunchKernelGGL((loss_kernel<false>), dim3(cdiv(M, 4)), dim3(256), 0, s, a.part, p.st.ns, M, h->V, a.hit, targets, ignore, loss, lse);
    TSC_HIP_CHECK(hipGetLastError());
    return TSC_OK;
}

int tsc_launch_unembed_backward(const tsc_unembed *h, const float *g, const TscRows &x, int M, const long long *targets, long long ignore,
                                const float *lse, void *dx, void *dW, void *db, char *ws, hipStream_t s) {
    const bool f16 = h->elem != TSC_ELEM_BF16;
    if (M == 0) {
        auto zero = [&](void *p, int elem, long long n) {
            hipLaunchKernelGGL(zero_elem_kernel, dim3((int)(n < 1 << 24 ? cdiv(n, 256) : 1 << 16)), dim3(256), 0, s, p, elem, n);
        };
        if (dW) zero(dW, h->elem, (long long)h->D * h->V);
        if (db) zero(db, h->belem, h->V);
        TSC_HIP_CHECK(hipGetLastError());
        return TSC_OK;
    }
    const int ordered = after_layout(h, s);
    if (ordered) return ordered;
    const Plan p = plan(h, M, true, dx != nullptr, dW != nullptr, db != nullptr);
    short *xp = (short *)(ws + p.xp), *G = (short *)(ws + p.g);
    float *dxp = (float *)(ws + p.dxp);
    unsigned *gtop = f16 ? (unsigned *)(ws + p.gtop) : nullptr;
    if (gtop) hipLaunchKernelGGL(fill_kernel, dim3(1), dim3(256), 0, s, (float *)gtop, 0.f, 2ll);
    pack_x(h, p, x, M, targets, ignore, g, ws, gtop, s);
    LogitArgs a = logit_args(h, p, ws, M, targets, ignore);
    a.lse = lse; a.g = g; a.gtop = gtop; a.G = G; a.ldg = (long long)p.copies * p.Vc; a.rest = p.Vc;
    a.left = p.left_wanted ? (float *)(ws + p.left) : nullptr;
    a.Mp = dW ? p.Mp : M;  // (only dW's k-steps run over the rows behind M)
    a.x.ld *= p.copies;
    a.dbias = db ? (float *)(ws + p.db) : nullptr;
    const long long xld = (long long)h->planes * h->Dp;
    const int db_parts = p.st.nm * (p.st.s.kind == FEW ? 1 : 2);  // waves of a tile's rows
    for (int c = 0; c < p.pieces; ++c) {
        const int v0 = c * p.Vc, nv = h->V - v0 < p.Vc ? h->V - v0 : p.Vc;
        a.v0 = v0;
        a.nv = cdiv(nv, p.st.s.bj);
        a.ns = p.st.ns < a.nv ? p.st.ns : a.nv;
        int rc = logits<true>(h, p.st, a, s);
        if (rc) return rc;
        if (db) hipLaunchKernelGGL(dbias_kernel, dim3(cdiv(nv, 64)), dim3(1024), 0, s, a.dbias, db_parts, a.ldg, nv, gtop, h->belem, db, (long long)v0);
        if (dx) {
            SumArgs q{};
            q.A = {G, (long long)h->planes * p.Vc, p.copies * M};
            q.B = {h->Wd + (long long)h->planes * v0, h->wd_ld, h->D};
            q.nk = cdiv(nv, BK); q.I = M; q.J = h->D; q.add = c > 0; q.pair = p.copies == 2; q.out = dxp;
            Split w = p.dx;
            if (c > 0) w.per = cdiv(q.nk, w.z);  // the same parts, shorter
            rc = launch_dx(w, h->elem, q, s);
            if (rc) return rc;
        }
        if (dW) {
            const bool by_d = h->sv == 1;  // dW is dense in W's order: [D][V] or [V][D]
            float *sums = (float *)(ws + p.sums);
            int *slot = (int *)(ws + p.slot);
            if (p.targets_wanted) {
                auto launch = [&](auto *kernel) {
                    hipLaunchKernelGGL(kernel, dim3(cdiv(nv, TOKENS)), dim3(1024), 0, s, targets, ignore, a.left, xp, xld, M, h->D, v0, v0 + nv, sums, slot);
                };
                if (M <= h->V) f16 ? launch(target_rows_kernel<_Float16, false>) : launch(target_rows_kernel<__bf16, false>);
                else f16 ? launch(target_rows_kernel<_Float16, true>) : launch(target_rows_kernel<__bf16, true>);
            }
            const DwPlan parts = dw_plan(h, (long long)p.copies * p.Mp, nv);
            for (int i = 0, at = 0; i < 2 && parts.n[i]; at += parts.n[i++]) {
                const Split &w = parts.w[i];
                const Operand X = {xp, xld, h->D}, Gk = {G + (long long)h->planes * at, (long long)h->planes * p.Vc, parts.n[i]};
                const int I = by_d ? h->D : parts.n[i], J = by_d ? parts.n[i] : h->D;
                const long long first = by_d ? v0 + at : (long long)(v0 + at) * h->D, ld = by_d ? h->V : h->D;
                void *out = (char *)dW + first * (h->elem == TSC_ELEM_F32 ? 4 : 2);
                const Targets more = {sums, p.targets_wanted ? slot + v0 + at : nullptr, by_d};
                if (w.z == 1) {
                    OutArgs q{};
                    q.A = by_d ? X : Gk;
                    q.B = by_d ? Gk : X;
                    q.nk = p.copies * p.Mp / BK; q.I = I; q.J = J; q.gtop = gtop; q.ld = ld; q.out = out; q.more = more;
                    rc = launch_dw(w, h->elem, by_d, q, s);
                } else {
                    SumArgs q{};
                    q.A = by_d ? X : Gk;
                    q.B = by_d ? Gk : X;
                    q.nk = p.copies * p.Mp / BK; q.I = I; q.J = J; q.out = (float *)(ws + p.dwp);
                    rc = launch_dw_parts(w, h->elem, by_d, q, s);
                    if (!rc) {  // (many parts are of few elements: 63 of 311 x 137 25 us by single waves)
                        if (w.z >= 8) hipLaunchKernelGGL((join_kernel<true>), dim3(I, cdiv(J, 256)), dim3(256), 0, s, q.out, w.z, I, J, more, gtop, out, ld, h->elem);
                        else hipLaunchKernelGGL((join_kernel<false>), dim3(I, cdiv(J, 1024)), dim3(256), 0, s, q.out, w.z, I, J, more, gtop, out, ld, h->elem);
                    }
                }
                if (rc) return rc;
            }
        }
        TSC_HIP_CHECK(hipGetLastError());
    }
    if (dx) {
        const bool shared = p.dx.z >= 8;
        const dim3 grid(shared ? M : cdiv(M, 4), cdiv(h->D, 256));
        auto launch = [&](auto *kernel) {
            hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, dxp, p.dx.z, M, h->D, a.wscale, a.xscale, gtop, g, targets, ignore, a.left, h->Wt,
                               h->wt_ld, h->V, h->elem, dx);
        };
        shared ? launch(dx_kernel<true>) : launch(dx_kernel<false>);
    }
    TSC_HIP_CHECK(hipGetLastError());
    return TSC_OK;
}
