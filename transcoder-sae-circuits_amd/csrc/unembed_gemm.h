// The matrix product under the unembedding's cross entropy (unembed.hip): 16-bit operands, fp32 accumulation.
//
//   C[i][j] = sum_k A(i, k) * B(j, k)
//
// One workgroup computes a BI x BJ tile in k-steps of 64.  Both operand tiles of a k-step go global -> LDS by
// global_load_lds_dwordx4 (1 KiB a wave and instruction, no registers) into one of two buffers while the other one is
// multiplied; one barrier a k-step.  Operands come in two layouts:
//   row-major  A(i, k) = A[i * ld + k]: LDS rows of 128 bytes (64 k), a fragment is one ds_read_b128
//   k-major    A(i, k) = A[k * ld + i]: LDS rows of BI elements, a fragment is two transposing ds_read_b64_tr_b16
// 16-byte chunks are permuted through the source address of the copy (row-major: chunk ^ (row / 2) % 8; k-major: the
// 64-byte groups ^ k % 4), which spreads the lanes of a fragment read over the banks.
//
// fp32 operands are split into two fp16 planes: x / s = h1 + h2 / 2048, s a power of two that brings the largest magnitude
// into [2^13, 2^14).  h1 holds 11 bits, h2 the next 11 (and more where h1 is subnormal), so h1 + h2 / 2048 has 22 bits for
// values down to 2^-27 of the largest and a fixed 2^-49 of it below.  The product is three passes over k,
// (h2 h1' + h1 h2') / 2048 + h1 h1', the cross terms first; the dropped h2 h2' is 2^-24 of the product at most.  Every
// product of two fp16 values is exact in the matrix pipe, sums are fp32: the result carries the error of an fp32 product
// at a third of the 16-bit rate, which is 5 times the fp32 matrix rate.
#pragma once
#include "tsc_internal.h"

namespace unembed_gemm {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef const __attribute__((address_space(1))) void *gptr_t;
typedef __attribute__((address_space(3))) void *lptr_t;

constexpr int BK = 64;

template <int WI_, int WJ_, int VI_, int VJ_> struct Tile {  // 32 x 32 blocks of a wave, waves of a workgroup
    static constexpr int WI = WI_, WJ = WJ_, VI = VI_, VJ = VJ_, NW = VI * VJ, NT = 64 * NW;
    static constexpr int BI = VI * WI * 32, BJ = VJ * WJ * 32;
    static constexpr int PA = BI / 8 / NW, PB = BJ / 8 / NW;  // 1-KiB pieces of a k-step and wave
    static_assert(PA * NW * 8 == BI && PB * NW * 8 == BJ, "whole pieces a wave");
};
typedef Tile<4, 2, 2, 4> TileLarge;   // 256 x 256, 8 waves
typedef Tile<2, 2, 2, 2> TileMedium;  // 128 x 128, 4 waves
typedef Tile<1, 2, 4, 1> TileSkinny;  // 128 x 64, 4 waves: few tokens, the vocabulary streams

struct Operand {
    const short *p;
    long long ld;     // elements between rows (row-major) or between k (k-major)
    long long plane;  // elements from plane h1 to plane h2
    int rows;         // valid i (j); the tile's others read copies of valid ones
};

// k-steps [k0, k1) of every pass; passes 1 (16-bit operands) or 3 (split fp32)
template <class C, bool KMAJOR, bool F16> struct Gemm {
    static constexpr int ABYTES = C::BI * BK * 2, BBYTES = C::BJ * BK * 2, STAGE = ABYTES + BBYTES;
    static constexpr int LDS_BYTES = 2 * STAGE;

    template <int ROWS, int PIECES>
    static __device__ __forceinline__ void offsets(const Operand &o, int row0, unsigned (&off)[PIECES]) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
            const int piece = wave * PIECES + q;
            if (KMAJOR) {
                constexpr int CH = ROWS / 8;  // 16-byte chunks of a k
                const int at = piece * 64 + lane, k = at / CH, c = (at % CH) ^ (((k & 3) << 2) & (CH - 1));
                const int last = (o.rows + 7) / 8 * 8 - 8;
                const int i = row0 + c * 8 < last ? row0 + c * 8 : last;
                off[q] = (unsigned)(k * o.ld + i) * 2u;
            } else {
                const int r = piece * 8 + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
                const int i = row0 + r < o.rows ? row0 + r : o.rows - 1;
                off[q] = (unsigned)((i - row0) * (int)o.ld + c * 8) * 2u;  // relative to the tile's first row
            }
        }
    }
    template <int PIECES>
    static __device__ __forceinline__ void copy(const char *base, const unsigned (&off)[PIECES], char *lds) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int q = 0; q < PIECES; ++q)
            __builtin_amdgcn_global_load_lds((gptr_t)(base + (long long)(int)off[q]), (lptr_t)(lds + (wave * PIECES + q) * 1024), 16, 0, 0);
    }
    // fragment of 32 rows and 16 k (kk-th of the k-step): lane l holds row l % 32, k = 8 * (l / 32) + 0..7
    template <int ROWS> static __device__ __forceinline__ s16x8 fragment(const char *lds, int row0, int kk) {
        const int lane = threadIdx.x & 63;
        if constexpr (KMAJOR) {
            const int l = lane & 15, g = lane >> 4;
            const int i = row0 + (g & 1) * 16 + (l & 3) * 4, k = kk * 16 + (g >> 1) * 8 + (l >> 2);
            const int byte = k * ROWS * 2 + (((i >> 3) ^ (((k & 3) << 2) & (ROWS / 8 - 1))) << 4) + (i & 4) * 2;
            typedef __attribute__((address_space(3))) s16x4 *p4;
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(lptr_t)(lds + byte));
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(lptr_t)(lds + byte + 4 * ROWS * 2));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            const int li = lane & 31, lh = lane >> 5;
            return *(const s16x8 *)(lds + (row0 + li) * 128 + (((kk * 2 + lh) ^ ((li >> 1) & 7)) << 4));
        }
    }
    static __device__ __forceinline__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
        if constexpr (F16)
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }

    static __device__ __forceinline__ void run(const Operand &A, const Operand &B, int i0, int j0, int k0, int k1, int passes,
                                               char *lds, f32x16 (&acc)[C::WI][C::WJ]) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wi0 = (wave / C::VJ) * (C::WI * 32), wj0 = (wave % C::VJ) * (C::WJ * 32);
        unsigned offa[C::PA], offb[C::PB];
        offsets<C::BI, C::PA>(A, i0, offa);
        offsets<C::BJ, C::PB>(B, j0, offb);
#pragma unroll
        for (int a = 0; a < C::WI; ++a)
#pragma unroll
            for (int b = 0; b < C::WJ; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;
        const int n = k1 - k0, total = n * passes;
        auto base = [&](const Operand &o, int row0, int s, int second) {  // step s of the stream
            const int pass = passes == 1 ? 2 : s / n, k = k0 + (passes == 1 ? s : s % n);
            return (const char *)(o.p + (pass == second ? o.plane : 0) + (KMAJOR ? (long long)k * BK * o.ld : (long long)row0 * o.ld + (long long)k * BK));
        };
        auto issue = [&](int s) {
            char *dst = lds + (s & 1) * STAGE;
            copy<C::PA>(base(A, i0, s, 0), offa, dst);
            copy<C::PB>(base(B, j0, s, 1), offb, dst + ABYTES);
        };
        if (total > 0) issue(0);
        for (int s = 0; s < total; ++s) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();  // step s has arrived for everybody, and nobody reads the other buffer any more
            if (s + 1 < total) issue(s + 1);
            const char *la = lds + (s & 1) * STAGE, *lb = la + ABYTES;
            if (passes == 3 && s == 2 * n)
#pragma unroll
                for (int a = 0; a < C::WI; ++a)
#pragma unroll
                    for (int b = 0; b < C::WJ; ++b)
#pragma unroll
                        for (int r = 0; r < 16; ++r) acc[a][b][r] *= 1.f / 2048.f;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                s16x8 fa[C::WI], fb[C::WJ];
#pragma unroll
                for (int a = 0; a < C::WI; ++a) fa[a] = fragment<C::BI>(la, wi0 + a * 32, kk);
#pragma unroll
                for (int b = 0; b < C::WJ; ++b) fb[b] = fragment<C::BJ>(lb, wj0 + b * 32, kk);
#pragma unroll
                for (int a = 0; a < C::WI; ++a)
#pragma unroll
                    for (int b = 0; b < C::WJ; ++b) acc[a][b] = mfma(fa[a], fb[b], acc[a][b]);
            }
        }
    }
};

// Element r of a 32 x 32 block: row (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5), column lane & 31.
__device__ __forceinline__ int block_row(int r, int lh) { return (r & 3) + 8 * (r >> 2) + 4 * lh; }

}  // namespace unembed_gemm
