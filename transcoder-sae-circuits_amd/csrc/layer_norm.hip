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
// with the stride of the grid and keep w and b (backward: w and their part of dw and db) in registers meanwhile; the
// parts of a workgroup meet in LDS, those of the grid in the workspace, and a second launch adds them up in a fixed
// order, so results do not depend on timing.
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

// Sum over the TPR threads of a row, the result in all of them.  TPR > 64: the row is a whole workgroup's.
template <int TPR> __device__ __forceinline__ void row_sum2(float &a, float &b, float (*lds)[2]) {
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) {
        a += __shfl_xor(a, o);
        b += __shfl_xor(b, o);
    }
    if constexpr (TPR > 64) {
        constexpr int NW = TPR / 64;
        const int w = threadIdx.x >> 6;
        __syncthreads();  // the last reduction's values are still being read
        if ((threadIdx.x & 63) == 0) lds[w][0] = a, lds[w][1] = b;
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) a += lds[i][0], b += lds[i][1];
    }
}

template <class T, int NV, int TPR> struct Row {
    static constexpr int VE = Elem<T>::VE;
    // element index of entry e of vector j of thread t: vectors of neighbouring threads are neighbours in memory
    static __device__ __forceinline__ int at(int t, int j) { return (j * TPR + t) * VE; }
    static __device__ __forceinline__ void load(const T *p, int D, int t, float (&v)[NV * VE]) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = at(t, j);
            if (i + VE <= D) {
                const Vec<T> x = *(const Vec<T> *)(p + i);
#pragma unroll
                for (int e = 0; e < VE; ++e) v[j * VE + e] = to_f(x.e[e]);
            } else {
#pragma unroll
                for (int e = 0; e < VE; ++e) v[j * VE + e] = i + e < D ? to_f(p[i + e]) : 0.f;
            }
        }
    }
    static __device__ __forceinline__ void store(T *p, int D, int t, const float (&v)[NV * VE]) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = at(t, j);
            if (i + VE <= D) {
                Vec<T> x;
#pragma unroll
                for (int e = 0; e < VE; ++e) x.e[e] = (T)v[j * VE + e];
                *(Vec<T> *)(p + i) = x;
            } else {
#pragma unroll
                for (int e = 0; e < VE; ++e)
                    if (i + e < D) p[i + e] = (T)v[j * VE + e];
            }
        }
    }
    static __device__ __forceinline__ void param(const void *p, int elem, int D, int t, float none, float (&v)[NV * VE]) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const int i = at(t, j) + e;
                v[j * VE + e] = i < D ? load_param(p, elem, i, none) : 0.f;
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

template <class T, int NV, int TPR>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void ln_forward_kernel(const LnArgs a) {
    typedef Row<T, NV, TPR> R;
    constexpr int N = NV * R::VE, NT = TPR > 256 ? TPR : 256, GROUPS = NT / TPR;
    __shared__ float red[16][2];
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR, D = a.D;
    const float inv = 1.f / (float)D;
    float w[N], b[N];
    R::param(a.w, a.param_elem, D, t, 1.f, w);
    R::param(a.b, a.param_elem, D, t, 0.f, b);
    for (long long row = (long long)blockIdx.x * GROUPS + grp; row < a.rows; row += (long long)gridDim.x * GROUPS) {
        float x[N];
        R::load((const T *)a.x.data + row_offset(a.x, row), D, t, x);
        float s = 0.f, unused = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) s += x[i];
        row_sum2<TPR>(s, unused, red);
        const float mean = s * inv;
        float q = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < R::VE; ++e) {
                const float d = R::at(t, j) + e < D ? x[j * R::VE + e] - mean : 0.f;
                x[j * R::VE + e] = d;
                q = fmaf(d, d, q);
            }
        row_sum2<TPR>(q, unused, red);
        const float scale = sqrtf(fmaf(q, inv, a.eps)), r = 1.f / scale;
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = fmaf(x[i] * r, w[i], b[i]);
        R::store((T *)a.out + row * D, D, t, x);
        if (t == 0) {
            a.mean[row] = mean;
            a.scale[row] = scale;
        }
    }
}

template <class T, int NV, int TPR>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void ln_backward_kernel(const LnArgs a) {
    typedef Row<T, NV, TPR> R;
    constexpr int N = NV * R::VE, NT = TPR > 256 ? TPR : 256, GROUPS = NT / TPR;
    __shared__ float red[16][2];
    __shared__ float part[GROUPS > 1 ? TPR * N : 1];
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR, D = a.D;
    const float inv = 1.f / (float)D;
    float w[N], dw[N], db[N];
    R::param(a.w, a.param_elem, D, t, 1.f, w);
#pragma unroll
    for (int i = 0; i < N; ++i) dw[i] = db[i] = 0.f;
    for (long long row = (long long)blockIdx.x * GROUPS + grp; row < a.rows; row += (long long)gridDim.x * GROUPS) {
        float x[N], dy[N];
        R::load((const T *)a.x.data + row_offset(a.x, row), D, t, x);
        R::load((const T *)a.dy.data + row_offset(a.dy, row), D, t, dy);
        const float mean = a.mean[row], r = 1.f / a.scale[row];
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {  // behind the row's end dy and w are 0: x = -mean there adds nothing
            x[i] = (x[i] - mean) * r;
            dw[i] = fmaf(dy[i], x[i], dw[i]);
            db[i] += dy[i];
            dy[i] *= w[i];
            s += dy[i];
            q = fmaf(dy[i], x[i], q);
        }
        row_sum2<TPR>(s, q, red);
        s *= inv;
        q *= inv;
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (dy[i] - fmaf(x[i], q, s)) * r;
        R::store((T *)a.out + row * D, D, t, x);
    }
    if (!a.part_w && !a.part_b) return;
    // the groups of the workgroup one after the other (a fixed order), then one row of the workspace
    auto emit = [&](float (&v)[N], float *dst) {
        if constexpr (GROUPS > 1) {
            for (int g = GROUPS - 1; g > 0; --g) {
                __syncthreads();
                if (grp == g) {
#pragma unroll
                    for (int i = 0; i < N; ++i) part[i * TPR + t] = v[i];
                }
                __syncthreads();
                if (grp == g - 1) {
#pragma unroll
                    for (int i = 0; i < N; ++i) v[i] += part[i * TPR + t];
                }
            }
        }
        if (grp == 0)
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < R::VE; ++e) {
                    const int i = R::at(t, j) + e;
                    if (i < D) dst[(long long)blockIdx.x * D + i] = v[j * R::VE + e];
                }
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
        float s = 0.f, q = 0.f, unused = 0.f;
        for (int i = t; i < D; i += 1024) s += to_f(x[i]);
        row_sum2<1024>(s, unused, red);
        const float mean = s * inv;
        for (int i = t; i < D; i += 1024) {
            const float d = to_f(x[i]) - mean;
            q = fmaf(d, d, q);
        }
        row_sum2<1024>(q, unused, red);
        const float scale = sqrtf(fmaf(q, inv, a.eps)), r = 1.f / scale;
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
        float s = 0.f, q = 0.f;
        for (int i = t; i < D; i += 1024) {
            const float g = to_f(dy[i]), h = (to_f(x[i]) - mean) * r, dn = g * load_param(a.w, a.param_elem, i, 1.f);
            s += dn;
            q = fmaf(dn, h, q);
            if (pw) pw[i] = fmaf(g, h, pw[i]);
            if (pb) pb[i] += g;
        }
        row_sum2<1024>(s, q, red);
        s *= inv;
        q *= inv;
        T *dx = (T *)a.out + row * D;
        for (int i = t; i < D; i += 1024) {
            const float h = (to_f(x[i]) - mean) * r, dn = to_f(dy[i]) * load_param(a.w, a.param_elem, i, 1.f);
            dx[i] = (T)((dn - fmaf(h, q, s)) * r);
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

constexpr int MAX_PARTS = 512;  // workgroups of a backward pass = rows of its workspace

struct Shape { int tpr, nv; };  // threads a row, 16-byte vectors a thread; nv 0: the wide kernels

template <class T> Shape pick(int D) {
    const int vec = (D + Elem<T>::VE - 1) / Elem<T>::VE;
    // the fewest threads that hold the row in at most four vectors each: short rows share a wave, and a thread has several
    // independent loads in flight
    for (int tpr : {8, 32, 64, 256, 1024})
        if (vec <= 4 * tpr) return {tpr, (vec + tpr - 1) / tpr};
    return {1024, 0};
}

template <class T, bool BWD> int launch(const LnArgs &a, int grid_cap, hipStream_t s, int *grid_out) {
    const Shape sh = pick<T>(a.D);
    const int groups = sh.nv && sh.tpr < 256 ? 256 / sh.tpr : 1;
    long long want = (a.rows + groups - 1) / groups;
    const int grid = (int)(want < grid_cap ? want : grid_cap);
    *grid_out = grid;
    const int nt = sh.tpr > 256 ? sh.tpr : 256;
#define TSC_LN(TPR, NV)                                                              \
    if (sh.tpr == TPR && sh.nv == NV) {                                              \
        if (BWD) hipLaunchKernelGGL((ln_backward_kernel<T, NV, TPR>), dim3(grid), dim3(nt), 0, s, a); \
        else hipLaunchKernelGGL((ln_forward_kernel<T, NV, TPR>), dim3(grid), dim3(nt), 0, s, a);      \
    } else
#define TSC_LN4(TPR) TSC_LN(TPR, 1) TSC_LN(TPR, 2) TSC_LN(TPR, 3) TSC_LN(TPR, 4)
    TSC_LN4(8) TSC_LN4(32) TSC_LN4(64) TSC_LN4(256) TSC_LN4(1024) {
        if (BWD) hipLaunchKernelGGL((ln_backward_wide_kernel<T>), dim3(grid), dim3(1024), 0, s, a);
        else hipLaunchKernelGGL((ln_forward_wide_kernel<T>), dim3(grid), dim3(1024), 0, s, a);
    }
#undef TSC_LN4
#undef TSC_LN
    TSC_HIP_CHECK(hipGetLastError());
    return TSC_OK;
}

}  // namespace

size_t tsc_layer_norm_parts(long long rows) { return rows < MAX_PARTS ? (size_t)rows : (size_t)MAX_PARTS; }

int tsc_launch_layer_norm(int elem, const TscRows &x, long long rows, int D, const void *w, const void *b, int param_elem,
                          float eps, void *y, float *mean, float *scale, hipStream_t s) {
    LnArgs a{};
    a.x = x; a.w = w; a.b = b; a.param_elem = param_elem; a.D = D; a.rows = rows; a.eps = eps;
    a.out = y; a.mean = mean; a.scale = scale;
    int grid;
    constexpr int CAP = 256 * 8;  // eight workgroups of four waves fill a CU
    if (elem == TSC_ELEM_F32) return launch<float, false>(a, CAP, s, &grid);
    if (elem == TSC_ELEM_BF16) return launch<bf16, false>(a, CAP, s, &grid);
    return launch<f16, false>(a, CAP, s, &grid);
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
    const int cap = dw || db ? MAX_PARTS : 256 * 8;
    if (elem == TSC_ELEM_F32) rc = launch<float, true>(a, cap, s, &grid);
    else if (elem == TSC_ELEM_BF16) rc = launch<bf16, true>(a, cap, s, &grid);
    else rc = launch<f16, true>(a, cap, s, &grid);
    if (rc != TSC_OK || (!dw && !db)) return rc;
    hipLaunchKernelGGL(ln_reduce_kernel, dim3((D + 31) / 32, 2), dim3(1024), 0, s, a.part_w, a.part_b, grid, D, dw, db, param_elem);
    TSC_HIP_CHECK(hipGetLastError());
    return TSC_OK;
}
