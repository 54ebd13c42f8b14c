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
typedef Tile<1, 2, 4, 1> TileTall;    // 128 x 64, 4 waves: few tokens, the vocabulary streams
typedef Tile<2, 1, 1, 4> TileWide;    // 64 x 128: the same with the operands exchanged

struct Operand {
    const short *p;
    long long ld;     // elements between rows (row-major) or between k (k-major)
    long long plane;  // elements from plane h1 to plane h2
    int rows;         // valid i (j); the tile's others read copies of valid ones
};

// One tile of a workgroup's stream: first rows of both operands.
struct TileAt {
    int i0, j0;
};

// The product of a stream of tiles.  All k-steps of all tiles of a workgroup form one stream: step s + 1 is in LDS and step
// s + 2 on its way while step s is multiplied, also across the end of a tile, so that only the first tile waits for memory.
//
//   step s:  MFMA k 0-15 | 16-31 | 32-47, each while the fragments of the next group are read
//            wait: own fragments of 48-63 are in registers, own copies of step s + 1 have landed; barrier
//            MFMA k 48-63 while the first fragments of step s + 1 are read and the copies of step s + 2 are issued
//
// Behind the barrier nobody reads the buffer of step s any more and everybody's part of step s + 1 is there.
template <class C, bool KMAJOR, bool F16> struct Gemm {
    static constexpr int ABYTES = C::BI * BK * 2, BBYTES = C::BJ * BK * 2, STAGE = ABYTES + BBYTES;
    static constexpr int LDS_BYTES = 2 * STAGE;

    // byte offsets of this lane's part of the PIECES 1-KiB pieces of this wave, relative to the tile's base
    template <int ROWS, int PIECES>
    static __device__ __forceinline__ void offsets(const Operand &o, int row0, unsigned (&off)[PIECES]) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
            const int piece = wave * PIECES + q;
            if (KMAJOR) {
                constexpr int CH = ROWS / 8;  // 16-byte chunks of a k
                const int at = piece * 64 + lane, k = at / CH, c = (at % CH) ^ (((k & 3) << 2) & (CH - 1));
                const int last = (o.rows + 7) / 8 * 8 - 8 - row0;
                const int i = c * 8 < last ? c * 8 : last;  // (last >= 0: a tile has at least one row)
                off[q] = (unsigned)(k * (int)o.ld + i) * 2u;
            } else {
                const int r = piece * 8 + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
                const int i = row0 + r < o.rows ? r : o.rows - 1 - row0;
                off[q] = (unsigned)(i * (int)o.ld + c * 8) * 2u;
            }
        }
    }
    static __device__ __forceinline__ const char *base(const Operand &o, int row0, int k0) {
        return (const char *)(o.p + (KMAJOR ? (long long)k0 * BK * o.ld + row0 : (long long)row0 * o.ld + (long long)k0 * BK));
    }
    static __device__ __forceinline__ long long step_bytes(const Operand &o) { return KMAJOR ? 2ll * BK * o.ld : 2ll * BK; }

    template <int ROWS> struct Frag {  // fragment reads of one operand: one LDS address for each of a step's four groups of 16 k
        unsigned at[4];
        __device__ __forceinline__ Frag(int row0, int extra) {
            const int lane = threadIdx.x & 63;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                if constexpr (KMAJOR) {
                    const int l = lane & 15, g = lane >> 4;
                    const int i = row0 + (g & 1) * 16 + (l & 3) * 4, k = kk * 16 + (g >> 1) * 8 + (l >> 2);
                    at[kk] = extra + k * ROWS * 2 + (((i >> 3) ^ (((k & 3) << 2) & (ROWS / 8 - 1))) << 4) + (i & 4) * 2;
                } else {
                    const int li = lane & 31, lh = lane >> 5;
                    at[kk] = extra + (row0 + li) * 128 + (((kk * 2 + lh) ^ ((li >> 1) & 7)) << 4);
                }
            }
        }
        // rows row0 + 32 * block of k group kk: lane l holds row l % 32, k = 8 * (l / 32) + 0..7
        template <int N> __device__ __forceinline__ void read(const char *lds, unsigned buf, int kk, s16x8 (&f)[N]) const {
            if constexpr (KMAJOR) {
                // the chunk permutation acts on the 64-byte groups, so a block's distance of 64 bytes is an exclusive or too
#pragma unroll
                for (int b = 0; b < N; ++b) {
                    typedef __attribute__((address_space(3))) s16x4 *p4;
                    const char *p = lds + (at[kk] ^ (b * 64)) + buf;
                    const s16x4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(lptr_t)p);
                    const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(lptr_t)(p + 4 * ROWS * 2));
                    f[b] = __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
                }
            } else {
                const char *p = lds + at[kk] + buf;
#pragma unroll
                for (int b = 0; b < N; ++b) f[b] = *(const s16x8 *)(p + b * 4096);
            }
        }
    };
    static __device__ __forceinline__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
        if constexpr (F16)
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }

    // tiles t = 0 .. n_tiles - 1 at tile(t); k-steps [k0, k1) in passes 1 (16-bit operands) or 3 (split fp32).
    // begin(t, acc) sets a tile's accumulators, done(t, acc) takes its sums.  LDS of the stages: lds[0 .. LDS_BYTES).
    template <class At, class Begin, class Done>
    static __device__ __forceinline__ void run(const Operand &A, const Operand &B, int n_tiles, At tile, int k0, int k1, int passes,
                                               char *lds, Begin begin, Done done) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int n = k1 - k0, total = n * passes;
        f32x16 acc[C::WI][C::WJ];
        if (n_tiles <= 0) return;
        if (n <= 0) {  // (a part of the k-steps behind their end)
            for (int t = 0; t < n_tiles; ++t) {
                begin(t, acc);
                done(t, acc);
            }
            return;
        }
        const Frag<C::BI> ra((wave / C::VJ) * (C::WI * 32), 0);
        const Frag<C::BJ> rb((wave % C::VJ) * (C::WJ * 32), ABYTES);
        unsigned offa[C::PA], offb[C::PB];
        // the producer: the next step to copy
        int pt = 0, pp = passes == 1 ? 2 : 0, ps = 0;  // tile, pass (0: h2 h1', 1: h1 h2', 2: h1 h1'), step of the pass
        unsigned pbuf = 0;
        const char *a0, *b0, *pa, *pb;
        const long long da = step_bytes(A), db = step_bytes(B);
        auto set_pass = [&]() {
            pa = a0 + (pp == 0 ? A.plane * 2 : 0);
            pb = b0 + (pp == 1 ? B.plane * 2 : 0);
        };
        auto set_tile = [&]() {
            const TileAt at = tile(pt);
            offsets<C::BI, C::PA>(A, at.i0, offa);
            offsets<C::BJ, C::PB>(B, at.j0, offb);
            a0 = base(A, at.i0, k0);
            b0 = base(B, at.j0, k0);
            set_pass();
        };
        auto piece = [&](int q) {
            char *dst = lds + pbuf + (q < C::PA ? (wave * C::PA + q) * 1024 : ABYTES + (wave * C::PB + q - C::PA) * 1024);
            const char *src = q < C::PA ? pa + offa[q < C::PA ? q : 0] : pb + offb[q < C::PA ? 0 : q - C::PA];
            __builtin_amdgcn_global_load_lds((gptr_t)src, (lptr_t)dst, 16, 0, 0);
        };
        auto advance = [&]() {
            pbuf ^= STAGE;
            if (++ps < n) {
                pa += da;
                pb += db;
                return;
            }
            if (pp < 2) {
                ps = 0;
                ++pp;
                set_pass();
            } else if (pt + 1 < n_tiles) {
                ps = 0;
                ++pt;
                pp = passes == 1 ? 2 : 0;
                set_tile();
            }  // else: the stream is at its end, its last step is copied again (twice, unread: no branch in the loop)
        };
        constexpr int P = C::PA + C::PB;
        set_tile();
#pragma unroll
        for (int q = 0; q < P; ++q) piece(q);
        advance();
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int q = 0; q < P; ++q) piece(q);
        advance();
        s16x8 fa[2][C::WI], fb[2][C::WJ];
        unsigned buf = 0;
        ra.read(lds, 0, 0, fa[0]);
        rb.read(lds, 0, 0, fb[0]);
        for (int t = 0; t < n_tiles; ++t) {
            begin(t, acc);
            for (int s = 0; s < total; ++s) {
                if (passes == 3 && s == 2 * n)
#pragma unroll
                    for (int a = 0; a < C::WI; ++a)
#pragma unroll
                        for (int b = 0; b < C::WJ; ++b)
#pragma unroll
                            for (int r = 0; r < 16; ++r) acc[a][b][r] *= 1.f / 2048.f;
#pragma unroll
                for (int kk = 0; kk < 3; ++kk) {
                    ra.read(lds, buf, kk + 1, fa[(kk + 1) & 1]);
                    rb.read(lds, buf, kk + 1, fb[(kk + 1) & 1]);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int a = 0; a < C::WI; ++a)
#pragma unroll
                        for (int b = 0; b < C::WJ; ++b) acc[a][b] = mfma(fa[kk & 1][a], fb[kk & 1][b], acc[a][b]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                buf ^= STAGE;
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                // (behind the last step of the last tile these fragments are not used)
                ra.read(lds, buf, 0, fa[0]);
                rb.read(lds, buf, 0, fb[0]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int a = 0; a < C::WI; ++a)
#pragma unroll
                    for (int b = 0; b < C::WJ; ++b) {
                        acc[a][b] = mfma(fa[1][a], fb[1][b], acc[a][b]);
                        __builtin_amdgcn_sched_barrier(0);
                        constexpr int G = C::WI * C::WJ;
#pragma unroll
                        for (int q = (a * C::WJ + b) * P / G; q < (a * C::WJ + b + 1) * P / G; ++q) piece(q);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                advance();
            }
            done(t, acc);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy may arrive in LDS that is somebody else's by then
    }
};

// Element r of a 32 x 32 block: row (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5), column lane & 31.
__device__ __forceinline__ int block_row(int r, int lh) { return (r & 3) + 8 * (r >> 2) + 4 * lh; }

}  // namespace unembed_gemm
