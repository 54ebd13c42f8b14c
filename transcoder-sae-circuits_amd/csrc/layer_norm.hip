// Layer norm over the last axis, forward and backward (gfx950).
//
//   mean = sum(x) / D        scale = sqrt(sum((x - mean)^2) / D + eps)        xh = (x - mean) / scale
//   y  = xh * w + b
//   dn = dy * w              dx = (dn - sum(dn)/D - xh * sum(dn xh)/D) / scale
//   dw = sum over rows of dy * xh          db = sum over rows of dy
//
// HBM-bound: one read of every operand and one write of the result, ~10 operations an element.  A row is held in the
// registers of TPR threads (NV 16-byte vectors each), so both passes over it (mean, then the squared deviations: no
// cancellation of two large sums) cost no second read.  All statistics and sums are fp32.  Thread groups walk the rows
// with the stride of the grid; backward they keep their part of dw and db in registers meanwhile.  The parts of a
// workgroup meet in LDS, those of the grid in the workspace, and a second launch adds them up in a fixed order, so results
// do not depend on timing.
#include <type_traits>

#include "tsc_internal.h"

namespace {

typedef _Float16 f16;
typedef __bf16 bf16;

template <class T> struct Elem;
template <> struct Elem<float> { static constexpr int VE = 4; };
template <> struct Elem<bf16> { static constexpr int VE = 8; };
template <> struct Elem<f16> { static constexpr int VE = 8; };

// 16 bytes of elements that are aligned to one element only: rows of an odd width start anywhere (the memory pipe takes
// any alignment; an aligned row costs the same instruction)
template <class T> struct __attribute__((packed, aligned(sizeof(T)))) Vec { T e[Elem<T>::VE]; };

template <class T> __device__ __forceinline__ float to_f(T v) { return (float)v; }

__device__ __forceinline__ float load_param(const void *p, int elem, long long i, float none) {
    if (!p) return none;
    if (elem == TSC_ELEM_F32) return ((const float *)p)[i];
    if (elem == TSC_ELEM_BF16) return (float)((const bf16 *)p)[i];
    return (float)((const f16 *)p)[i];
}
__device__ __forceinline__ void store_param(void *p, int elem, long long i, float v) {
    if (elem == TSC_ELEM_F32) ((float *)p)[i] = v;
    else if (elem == TSC_ELEM_BF16) ((bf16 *)p)[i] = (bf16)v;
    else ((f16 *)p)[i] = (f16)v;
}

__device__ __forceinline__ long long row_offset(const TscRows &r, long long row) {
    if (r.inner_stride * r.inner == r.outer_stride) return row * r.inner_stride;  // (uniform: one row stride)
    return (row / r.inner) * r.outer_stride + (row % r.inner) * r.inner_stride;
}

// Sum over groups of 2^k neighbouring lanes, the result in all of them: lane exchanges inside the vector unit, no LDS.
template <int N> __device__ __forceinline__ float lanes_sum(float v) {
    const auto dpp = [](float x, auto ctrl) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    if constexpr (N >= 2) v += dpp(v, std::integral_constant<int, 0xB1>());    // lane ^ 1
    if constexpr (N >= 4) v += dpp(v, std::integral_constant<int, 0x4E>());    // lane ^ 2
    if constexpr (N >= 8) v += dpp(v, std::integral_constant<int, 0x141>());   // 7 - lane: the other four
    if constexpr (N >= 16) v += dpp(v, std::integral_constant<int, 0x140>());  // 15 - lane: the other eight
    if constexpr (N >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (N >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}
// Sum over the TPR threads of a row.  TPR > 64: thread groups of NT / TPR rows of one workgroup meet at the same barriers;
// lds has a place for each of NT / 64 waves.
template <int TPR, int NT, int N> __device__ __forceinline__ void row_sum(float (&v)[N], float (*lds)[2]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lanes_sum<(TPR < 64 ? TPR : 64)>(v[i]);
    if constexpr (TPR > 64) {
        constexpr int NW = TPR / 64;
        const int w = threadIdx.x >> 6, first = w / NW * NW;
        __syncthreads();  // the last reduction's values are still being read
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) lds[w][i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = 0.f;
#pragma unroll
            for (int k = 0; k < NW; ++k) v[i] += lds[first + k][i];
        }
    }
}

// VE parameters from element i on (all within the row); `none` without parameters
template <int VE> __device__ __forceinline__ void load_params(const void *p, int elem, int i, float none, float (&v)[VE]) {
    if (!p) {
#pragma unroll
        for (int e = 0; e < VE; ++e) v[e] = none;
    } else if (elem == TSC_ELEM_F32) {
        struct __attribute__((packed, aligned(4))) P { float e[VE]; };
        const P x = *(const P *)((const float *)p + i);
#pragma unroll
        for (int e = 0; e < VE; ++e) v[e] = x.e[e];
    } else {
        struct __attribute__((packed, aligned(2))) P { unsigned short e[VE]; };
        const P x = *(const P *)((const unsigned short *)p + i);
#pragma unroll
        for (int e = 0; e < VE; ++e) v[e] = elem == TSC_ELEM_BF16 ? __uint_as_float((unsigned)x.e[e] << 16) : (float)__builtin_bit_cast(f16, x.e[e]);
    }
}

// A thread's elements of a row: vector j starts at element at(t, j), neighbouring threads' vectors are neighbours in memory.
// Vectors that would pass the row's end are moved back to end with it, so that a thread never takes single elements (one lane
// with a loop of its own cost the whole row a third of its time); the elements before `lo` are then another thread's, which
// only counts for the last vector.  Rows shorter than one vector are taken element by element.
template <class T, int NV, int TPR> struct Row {
    static constexpr int VE = Elem<T>::VE;
    int D, first[NV], lo;
    __device__ __forceinline__ Row(int D_, int t) : D(D_) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = (j * TPR + t) * VE;
            first[j] = D < VE ? 0 : i < D - VE ? i : D - VE;
            if (j == NV - 1) lo = D < VE ? (t ? VE : 0) : i - first[j];
        }
    }
    // does this thread own entry e of vector j
    __device__ __forceinline__ bool own(int j, int e) const { return j < NV - 1 || (e >= lo && e < D); }
    __device__ __forceinline__ void load(const T *p, Vec<T> (&v)[NV]) const {
        if (D >= VE) {
#pragma unroll
            for (int j = 0; j < NV; ++j) v[j] = *(const Vec<T> *)(p + first[j]);
        } else {
#pragma unroll
            for (int e = 0; e < VE; ++e) v[0].e[e] = p[e < D ? e : 0];
        }
    }
    __device__ __forceinline__ void store(T *p, int j, const float (&v)[VE]) const {  // (shared elements: the same value twice)
        if (D >= VE) {
            Vec<T> x;
#pragma unroll
            for (int e = 0; e < VE; ++e) x.e[e] = (T)v[e];
            if (j < NV - 1 || lo < VE) *(Vec<T> *)(p + first[j]) = x;
        } else {
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (own(j, e)) p[e] = (T)v[e];
        }
    }
    __device__ __forceinline__ void param(const void *p, int elem, int j, float none, float (&v)[VE]) const {
        if (D >= VE) {
            load_params<VE>(p, elem, first[j], none, v);
        } else {
#pragma unroll
            for (int e = 0; e < VE; ++e) v[e] = load_param(p, elem, e < D ? e : 0, none);
        }
    }
};

// The same elements for the backward pass, which has no registers for the moved vectors (1021 x 4099 bf16: 24 us with them
// against 19): the vector that would pass the row's end is taken element by element, zeros behind.
template <class T, int NV, int TPR> struct RowEnd {
    static constexpr int VE = Elem<T>::VE;
    static __device__ __forceinline__ int at(int t, int j) { return (j * TPR + t) * VE; }
    static __device__ __forceinline__ void load(const T *p, int n, int t, Vec<T> (&v)[NV]) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = at(t, j);
            if (i + VE <= n) {
                v[j] = *(const Vec<T> *)(p + i);
            } else {
#pragma unroll
                for (int e = 0; e < VE; ++e) v[j].e[e] = i + e < n ? p[i + e] : (T)0.f;
            }
        }
    }
    static __device__ __forceinline__ void store(T *p, int D, int i, const float (&v)[VE]) {
        if (i + VE <= D) {
            Vec<T> x;
#pragma unroll
            for (int e = 0; e < VE; ++e) x.e[e] = (T)v[e];
            *(Vec<T> *)(p + i) = x;
        } else {
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (i + e < D) p[i + e] = (T)v[e];
        }
    }
};

struct LnArgs {
    TscRows x, dy;
    const void *w, *b;
    int param_elem, D;
    long long rows;
    float eps;
    void *out;           // y or dx
    float *mean, *scale;
    float *part_w, *part_b;  // backward: [gridDim.x][D] or null
};

// Threads a row and 16-byte vectors a thread; thread groups of a workgroup take rows of their own.  The next row is read
// while this one is reduced.
// Measured (fresh inputs): 65536 x 768 bf16 37 us = 5.4 TB/s, fp32 68 us = 5.9 TB/s; 512 x 768 fp32 3.6 us, a launch's own time.
template <class T, int NV, int TPR, int NT> __global__ __launch_bounds__(NT) void ln_forward_kernel(const LnArgs a) {
    typedef Row<T, NV, TPR> R;
    constexpr int N = NV * R::VE, GROUPS = NT / TPR;
    __shared__ float red[16][2];
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const R r(a.D, t);
    const float inv = 1.f / (float)a.D;
    const long long step = (long long)gridDim.x * GROUPS, last = a.rows - 1;
    long long row = (long long)blockIdx.x * GROUPS + grp;
    Vec<T> next[NV];
    r.load((const T *)a.x.data + row_offset(a.x, row < last ? row : last), next);
    float w[NV][R::VE], b[NV][R::VE];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        r.param(a.w, a.param_elem, j, 1.f, w[j]);
        r.param(a.b, a.param_elem, j, 0.f, b[j]);
    }
    // (every thread group goes around equally often: the barriers of a wide row are the workgroup's)
    for (long long first = (long long)blockIdx.x * GROUPS; first < a.rows; first += step, row += step) {
        float x[N], s[1] = {0.f}, q[1] = {0.f};
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (float)next[i / R::VE].e[i % R::VE];
        if (first + step < a.rows) r.load((const T *)a.x.data + row_offset(a.x, row + step < last ? row + step : last), next);
#pragma unroll
        for (int i = 0; i < N; ++i) s[0] += r.own(i / R::VE, i % R::VE) ? x[i] : 0.f;
        row_sum<TPR, NT>(s, red);
        const float mean = s[0] * inv;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] -= mean;
            const float d = r.own(i / R::VE, i % R::VE) ? x[i] : 0.f;
            q[0] = fmaf(d, d, q[0]);
        }
        row_sum<TPR, NT>(q, red);
        const float scale = sqrtf(fmaf(q[0], inv, a.eps)), rs = 1.f / scale;
        if (row > last) continue;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float o[R::VE];
#pragma unroll
            for (int e = 0; e < R::VE; ++e) o[e] = fmaf(x[j * R::VE + e] * rs, w[j][e], b[j][e]);
            r.store((T *)a.out + row * a.D, j, o);
        }
        if (t == 0) {
            a.mean[row] = mean;
            a.scale[row] = scale;
        }
    }
}

// The row's elements stay as they were read and are widened in each of the two passes, and the weight lies in LDS (its place
// is needed for the sums only at the end), so that 16 waves a CU keep their rows and sums in registers.  At 16 elements a thread
// one or two of them do not fit: they are stored once and read back behind the rows, in the loop over them only for fp16 rows of
// more than 8192 elements (15 registers) and fp32 rows of more than 12288 (one).
// Measured: 65536 x 768 fp32 125 us = 4.8 TB/s, bf16 80 us = 3.8 TB/s; 16384 x 768 fp32 27 us and 4 for the sums' last step;
// 1021 x 4099 bf16 16 us.  Reading the next row ahead, as the forward pass does, changed nothing (and spills more with two vectors).
template <class T, int NV, int TPR, int NT> __global__ __launch_bounds__(NT) void ln_backward_kernel(const LnArgs a) {
    typedef RowEnd<T, NV, TPR> R;
    constexpr int N = NV * R::VE, GROUPS = NT / TPR;
    __shared__ float red[16][2];
    __shared__ __attribute__((aligned(16))) float part[(GROUPS > 1 ? NT / 2 : TPR) * N];
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR, D = a.D;
    const float inv = 1.f / (float)D;
    const long long step = (long long)gridDim.x * GROUPS, last = a.rows - 1;
    long long row = (long long)blockIdx.x * GROUPS + grp;
    if (grp == 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = R::at(t, j);
            float w[R::VE];
            if (i + R::VE <= D) {
                load_params<R::VE>(a.w, a.param_elem, i, 1.f, w);
            } else {
#pragma unroll
                for (int e = 0; e < R::VE; ++e) w[e] = i + e < D ? load_param(a.w, a.param_elem, i + e, 1.f) : 0.f;
            }
#pragma unroll
            for (int e = 0; e < R::VE; e += 4) *(float4 *)&part[((j * R::VE + e) / 4 * TPR + t) * 4] = make_float4(w[e], w[e + 1], w[e + 2], w[e + 3]);
        }
    }
    __syncthreads();
    float dw[N], db[N];
#pragma unroll
    for (int i = 0; i < N; ++i) dw[i] = db[i] = 0.f;
    // (every thread group goes around equally often: the barriers of a wide row are the workgroup's)
    for (long long first = (long long)blockIdx.x * GROUPS; first < a.rows; first += step, row += step) {
        const bool live = row <= last;
        const long long rc = live ? row : last;
        Vec<T> nx[NV], ny[NV];  // (a group without a row: zeros, which add nothing)
        R::load((const T *)a.x.data + row_offset(a.x, rc), live ? D : 0, t, nx);
        R::load((const T *)a.dy.data + row_offset(a.dy, rc), live ? D : 0, t, ny);
        const float mean = live ? a.mean[rc] : 0.f, rs = live ? 1.f / a.scale[rc] : 0.f;
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 w4 = *(const float4 *)&part[(i / 4 * TPR + t) * 4];
            const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // behind the row's end dy and w are 0: what is there adds nothing to the sums
                const int k = i + e;
                const float h = ((float)nx[k / R::VE].e[k % R::VE] - mean) * rs, g = (float)ny[k / R::VE].e[k % R::VE], dn = g * w[e];
                dw[k] = fmaf(g, h, dw[k]);
                db[k] += g;
                s[0] += dn;
                s[1] = fmaf(dn, h, s[1]);
            }
        }
        row_sum<TPR, NT>(s, red);
        s[0] *= inv;
        s[1] *= inv;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float o[R::VE];
#pragma unroll
            for (int i = 0; i < R::VE; i += 4) {
                const float4 w4 = *(const float4 *)&part[((j * R::VE + i) / 4 * TPR + t) * 4];
                const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float h = ((float)nx[j].e[i + e] - mean) * rs, dn = (float)ny[j].e[i + e] * w[e];
                    o[i + e] = (dn - fmaf(h, s[1], s[0])) * rs;
                }
            }
            if (live) R::store((T *)a.out + row * D, D, R::at(t, j), o);
        }
    }
    // the thread groups of the workgroup in halves (a fixed order), then one row of the workspace
    auto emit = [&](float (&v)[N], float *dst) {
        if constexpr (GROUPS > 1) {
#pragma unroll
            for (int h = GROUPS / 2; h > 0; h /= 2) {
                __syncthreads();
                if (grp >= h && grp < 2 * h) {
#pragma unroll
                    for (int i = 0; i < N; ++i) part[i * (NT / 2) + (grp - h) * TPR + t] = v[i];
                }
                __syncthreads();
                if (grp < h) {
#pragma unroll
                    for (int i = 0; i < N; ++i) v[i] += part[i * (NT / 2) + grp * TPR + t];
                }
            }
        }
        // (through LDS into the order of memory: a thread's vectors lie apart, and so would its stores; 1021 x 4099 bf16 16 us
        // against 19)
        __syncthreads();
        if (grp == 0) {
#pragma unroll
            for (int i = 0; i < N; i += 4)
                *(float4 *)&part[R::at(t, i / R::VE) + i % R::VE] = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < D; i += NT) dst[(long long)blockIdx.x * D + i] = part[i];
    };
    if (a.part_w) emit(dw, a.part_w);
    if (a.part_b) emit(db, a.part_b);
}

// Rows that no workgroup's registers hold: one workgroup a row, every pass reads the row again (from the caches).
template <class T> __global__ __launch_bounds__(1024) void ln_forward_wide_kernel(const LnArgs a) {
    __shared__ float red[16][2];
    const int t = threadIdx.x, D = a.D;
    const float inv = 1.f / (float)D;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x.data + row_offset(a.x, row);
        float s[1] = {0.f}, q[1] = {0.f};
        for (int i = t; i < D; i += 1024) s[0] += to_f(x[i]);
        row_sum<1024, 1024>(s, red);
        const float mean = s[0] * inv;
        for (int i = t; i < D; i += 1024) {
            const float d = to_f(x[i]) - mean;
            q[0] = fmaf(d, d, q[0]);
        }
        row_sum<1024, 1024>(q, red);
        const float scale = sqrtf(fmaf(q[0], inv, a.eps)), r = 1.f / scale;
        T *y = (T *)a.out + row * D;
        for (int i = t; i < D; i += 1024)
            y[i] = (T)fmaf((to_f(x[i]) - mean) * r, load_param(a.w, a.param_elem, i, 1.f), load_param(a.b, a.param_elem, i, 0.f));
        if (t == 0) {
            a.mean[row] = mean;
            a.scale[row] = scale;
        }
    }
}

template <class T> __global__ __launch_bounds__(1024) void ln_backward_wide_kernel(const LnArgs a) {
    __shared__ float red[16][2];
    const int t = threadIdx.x, D = a.D;
    const float inv = 1.f / (float)D;
    float *pw = a.part_w ? a.part_w + (long long)blockIdx.x * D : nullptr;
    float *pb = a.part_b ? a.part_b + (long long)blockIdx.x * D : nullptr;
    for (int i = t; i < D; i += 1024) {  // an element of the workspace row belongs to one thread throughout
        if (pw) pw[i] = 0.f;
        if (pb) pb[i] = 0.f;
    }
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x.data + row_offset(a.x, row), *dy = (const T *)a.dy.data + row_offset(a.dy, row);
        const float mean = a.mean[row], r = 1.f / a.scale[row];
        float s[2] = {0.f, 0.f};
        for (int i = t; i < D; i += 1024) {
            const float g = to_f(dy[i]), h = (to_f(x[i]) - mean) * r, dn = g * load_param(a.w, a.param_elem, i, 1.f);
            s[0] += dn;
            s[1] = fmaf(dn, h, s[1]);
            if (pw) pw[i] = fmaf(g, h, pw[i]);
            if (pb) pb[i] += g;
        }
        row_sum<1024, 1024>(s, red);
        s[0] *= inv;
        s[1] *= inv;
        T *dx = (T *)a.out + row * D;
        for (int i = t; i < D; i += 1024) {
            const float h = (to_f(x[i]) - mean) * r, dn = to_f(dy[i]) * load_param(a.w, a.param_elem, i, 1.f);
            dx[i] = (T)((dn - fmaf(h, s[1], s[0])) * r);
        }
    }
}

// Sums of the workspace rows, fixed order: 32 columns x 32 parts a workgroup.
__global__ __launch_bounds__(1024) void ln_reduce_kernel(const float *part_w, const float *part_b, int n_parts, int D, void *dw,
                                                         void *db, int elem) {
    __shared__ float red[32][33];
    const float *part = blockIdx.y == 0 ? part_w : part_b;
    void *out = blockIdx.y == 0 ? dw : db;
    if (!part) return;
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), p = threadIdx.x >> 5;
    float s = 0.f;
    if (c < D)
#pragma unroll 8
        for (int i = p; i < n_parts; i += 32) s += part[(long long)i * D + c];
    red[p][threadIdx.x & 31] = s;
    __syncthreads();
    if (p == 0 && c < D) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += red[i][threadIdx.x];
        store_param(out, elem, c, s);
    }
}

// zero rows: the gradients of the parameters are sums of nothing
__global__ void ln_zero_kernel(void *dw, void *db, int elem, int D) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= D) return;
    if (dw) store_param(dw, elem, i, 0.f);
    if (db) store_param(db, elem, i, 0.f);
}

constexpr int MAX_PARTS = 256;  // workgroups of a backward pass (one a CU, 16 waves) = rows of its workspace

struct Shape { int tpr, nv; };  // threads a row, 16-byte vectors a thread; nv 0: the wide kernels

// Of the shapes that hold the row in `most` vectors a thread, the one that leaves the fewest lanes without elements; the
// fewest vectors among equals (measured forward, bf16: 768 elements as 32 x 3 40 us against 52 as 64 x 2, 1600 as 256 x 1 31
// against 43 as 64 x 4).
template <class T> Shape pick(int D, int most) {
    const int vec = (D + Elem<T>::VE - 1) / Elem<T>::VE;
    Shape best{1024, 0};
    for (int tpr : {8, 32, 64, 256, 1024}) {
        const int nv = (vec + tpr - 1) / tpr;
        if (nv > most) continue;
        const int size = tpr * nv, least = best.tpr * best.nv;
        if (!best.nv || size < least || (size == least && nv < best.nv)) best = {tpr, nv};
    }
    return best;
}

#define TSC_LN(TPR, NV, NT)                                                                        \
    if (sh.tpr == TPR && sh.nv == NV)                                                              \
        hipLaunchKernelGGL((TSC_LN_KERNEL<T, NV, TPR, NT>), dim3(grid), dim3(NT), 0, s, a);          \
    else
#define TSC_LN_ALL(NV, NT) TSC_LN(8, NV, NT) TSC_LN(32, NV, NT) TSC_LN(64, NV, NT) TSC_LN(256, NV, NT) TSC_LN(1024, NV, 1024)

template <class T> int launch_forward(const LnArgs &a, hipStream_t s) {
    const Shape sh = pick<T>(a.D, 4);
    const int groups = sh.nv && sh.tpr < 256 ? 256 / sh.tpr : 1;
    const long long want = (a.rows + groups - 1) / groups;
    const int cap = sh.nv == 1 ? 2048 : sh.nv == 2 ? 1536 : 1024;  // what the kernel's registers let a chip hold
    const int grid = (int)(want < cap ? want : cap);
#define TSC_LN_KERNEL ln_forward_kernel
    TSC_LN_ALL(1, 256) TSC_LN_ALL(2, 256) TSC_LN_ALL(3, 256) TSC_LN_ALL(4, 256)
    hipLaunchKernelGGL((ln_forward_wide_kernel<T>), dim3(grid), dim3(1024), 0, s, a);
#undef TSC_LN_KERNEL
    TSC_HIP_CHECK(hipGetLastError());
    return TSC_OK;
}

template <class T> int launch_backward(const LnArgs &a, int *grid_out, hipStream_t s) {
    constexpr bool F32 = sizeof(T) == 4;
    const Shape sh = pick<T>(a.D, F32 ? 4 : 2);  // 16 elements a thread
    const int groups = sh.nv ? 1024 / sh.tpr : 1;
    const long long want = (a.rows + groups - 1) / groups;
    const int grid = *grid_out = (int)(want < MAX_PARTS ? want : MAX_PARTS);
#define TSC_LN_KERNEL ln_backward_kernel
    if constexpr (F32) {
        TSC_LN_ALL(3, 1024) TSC_LN_ALL(4, 1024) {}
    }
    TSC_LN_ALL(1, 1024) TSC_LN_ALL(2, 1024)
    if (!sh.nv) hipLaunchKernelGGL((ln_backward_wide_kernel<T>), dim3(grid), dim3(1024), 0, s, a);
#undef TSC_LN_KERNEL
    TSC_HIP_CHECK(hipGetLastError());
    return TSC_OK;
}
#undef TSC_LN_ALL
#undef TSC_LN

}  // namespace

size_t tsc_layer_norm_parts(long long rows) { return rows < MAX_PARTS ? (size_t)rows : (size_t)MAX_PARTS; }

int tsc_launch_layer_norm(int elem, const TscRows &x, long long rows, int D, const void *w, const void *b, int param_elem,
                          float eps, void *y, float *mean, float *scale, hipStream_t s) {
    LnArgs a{};
    a.x = x; a.w = w; a.b = b; a.param_elem = param_elem; a.D = D; a.rows = rows; a.eps = eps;
    a.out = y; a.mean = mean; a.scale = scale;
    if (elem == TSC_ELEM_F32) return launch_forward<float>(a, s);
    if (elem == TSC_ELEM_BF16) return launch_forward<bf16>(a, s);
    return launch_forward<f16>(a, s);
}

int tsc_launch_layer_norm_backward(int elem, const TscRows &dy, const TscRows &x, const float *mean, const float *scale,
                                   long long rows, int D, const void *w, int param_elem, void *dx, void *dw, void *db,
                                   float *workspace, hipStream_t s) {
    if (rows == 0) {
        if (dw || db) {
            hipLaunchKernelGGL(ln_zero_kernel, dim3((D + 255) / 256), dim3(256), 0, s, dw, db, param_elem, D);
            TSC_HIP_CHECK(hipGetLastError());
        }
        return TSC_OK;
    }
    LnArgs a{};
    a.x = x; a.dy = dy; a.w = w; a.param_elem = param_elem; a.D = D; a.rows = rows; a.out = dx;
    a.mean = (float *)mean; a.scale = (float *)scale;
    a.part_w = dw ? workspace : nullptr;
    a.part_b = db ? workspace + (dw ? tsc_layer_norm_parts(rows) * (size_t)D : 0) : nullptr;
    int grid = 0, rc;
    if (elem == TSC_ELEM_F32) rc = launch_backward<float>(a, &grid, s);
    else if (elem == TSC_ELEM_BF16) rc = launch_backward<bf16>(a, &grid, s);
    else rc = launch_backward<f16>(a, &grid, s);
    if (rc != TSC_OK || (!dw && !db)) return rc;
    hipLaunchKernelGGL(ln_reduce_kernel, dim3((D + 31) / 32, 2), dim3(1024), 0, s, a.part_w, a.part_b, grid, D, dw, db, param_elem);
    TSC_HIP_CHECK(hipGetLastError());
    return TSC_OK;
}
